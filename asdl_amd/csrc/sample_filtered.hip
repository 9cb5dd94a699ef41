// One draw per row from softmax(logits / T) restricted by top-k, top-p and min-p, with one uniform number u per row.
// Classes are ordered by logit, the lowest index first among equals; with weights w = exp((x - max x) / T):
//   top-k  keeps the first k;  top-p  keeps a class while the weight in front of it is below p times the weight of what top-k kept;
//   min-p  keeps w >= min_p;   the draw is the first class, by index, at which the kept weight up to there exceeds u times all of it.
// A border between two classes is where a sum over up to all classes passes a number, so sums have to be the same whatever order
// they are formed in: a weight is an integer, w 2^s rounded, with s so large that the sum over all classes fits 63 bits (46 bits below
// the point for 50257 classes), and integers add exactly.  w itself is computed in double.
// The kept classes are those above a key (the logit's bits in an order that integers keep) and, of those equal to it, the ones up to an
// index.
#include <type_traits>
#include "elements.hpp"

namespace ak {

struct SfParams {
  const void* logits;
  const void* u;
  const float* temperatures;
  const int64_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  int64_t* targets;
  int* invalid;
  int64_t ld, first_row;
  double temperature, top_p, min_p;
  int64_t top_k;
  int classes, u_double, shift;
  float unit;             // a weight of 1 in sums of 32 bits over all classes; at most 2^22, so that its whole part stays in a float
};

__device__ __forceinline__ uint32_t sf_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);       // (-0 and 0 are equal)
  return b ^ ((b >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float sf_value(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// a b + c with c in scalar registers.  (The compiler takes the form that overwrites c, and copies it to vector registers every time: a
// third of the instructions of a weight.)
__device__ __forceinline__ double sf_fma(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// w = exp((x - top) / T) = 2^y in units of 2^-shift: y = (x - top) (log2 e / T) is split into the nearest integer and a rest f in
// [-1/2, 1/2], whose power is 1 + f q(f), q interpolated at the ten Chebyshev points (off by at most 6e-16; exactly 1 at f = 0).  The
// addition of 1.5 2^52 + shift rounds y and leaves the integer, plus shift, in the low word, which then goes to the exponent's place:
// no conversions, which run at a quarter of the rate.
struct SfWeight {
  double top, c, scale, round;
  __device__ __forceinline__ SfWeight(float top_, double c_, int shift)
      : top(top_), c(c_), scale(static_cast<double>(1ull << shift)), round(6755399441055744. + shift) {}
  __device__ __forceinline__ double scaled(float x) const {
    const double y = fmax((static_cast<double>(x) - top) * c, -1000.);           // (-inf and its NaN: 0 in the end)
    const double t = y + round, f = y - (t - round);
    double q = sf_fma(7.070977866508138e-09, f, 1.0205905413765595e-07);
    q = sf_fma(q, f, 1.3215451633221434e-06);
    q = sf_fma(q, f, 1.5252672924850737e-05);
    q = sf_fma(q, f, 0.00015403530424776529);
    q = sf_fma(q, f, 0.0013333558200794592);
    q = sf_fma(q, f, 0.009618129107618665);
    q = sf_fma(q, f, 0.05550410866465167);
    q = sf_fma(q, f, 0.24022650695910075);
    q = sf_fma(q, f, 0.6931471805599462);
    return __builtin_bit_cast(double, __builtin_bit_cast(u64, fma(q, f, 1.)) + (__builtin_bit_cast(u64, t) << 52));
  }
  // rounded to an integer by the addition of 2^52: the fraction's bits (scaled() is at most 2^51)
  static __device__ __forceinline__ u64 whole(double scaled) {
    return __builtin_bit_cast(u64, scaled + 4503599627370496.) & 0x000fffffffffffffull;
  }
  __device__ __forceinline__ u64 operator()(float x) const { return whole(scaled(x)); }
};

// What a row is drawn with.
struct SfFilter {
  double t, p, m, u;
  int64_t k;
  __device__ __forceinline__ SfFilter(const SfParams& q, int64_t row)
      : t(q.temperatures != nullptr ? static_cast<double>(q.temperatures[row]) : q.temperature),
        p(q.top_ps != nullptr ? static_cast<double>(q.top_ps[row]) : q.top_p),
        m(q.min_ps != nullptr ? static_cast<double>(q.min_ps[row]) : q.min_p),
        u(q.u_double ? static_cast<const double*>(q.u)[row] : static_cast<double>(static_cast<const float*>(q.u)[row])),
        k(q.top_ks != nullptr ? q.top_ks[row] : q.top_k) {}
  __device__ __forceinline__ bool good() const { return t >= 0. && p == p && m == m && u == u; }
  __device__ __forceinline__ double exponent() const { return t > 0. ? 1.4426950408889634 / t : INFINITY; }      // log2 e / T
  // temperatures so low that only the most probable class has weight (and the exponent would overflow) count as 0
  __device__ __forceinline__ bool greedy() const { return k == 1 || p <= 0. || !(exponent() < 1e300); }
  __device__ __forceinline__ double least(double scale) const { return (m < 1. ? m : 1.) * scale; }     // of the scaled weights
};

// u of `all` as an integer below it: the first class at which the kept weight exceeds it is drawn.
__device__ __forceinline__ u64 sf_target(double u, u64 all) {
  const double border = u > 0. ? u * static_cast<double>(all) : 0.;
  const u64 target = border < static_cast<double>(all) ? static_cast<u64>(border) : all - 1;
  return target < all ? target : all - 1;
}

// The weight in front of a class has to be below p times `all`: of integers, below that rounded up.
__device__ __forceinline__ u64 sf_border(double p, u64 all) {
  const double border = ceil(p * static_cast<double>(all));
  const u64 target = border < 1. ? 1 : border < static_cast<double>(all) ? static_cast<u64>(border) : all;
  return target < all ? target : all;
}

// The largest and smallest over a work group.
struct SfRange {
  float top, low, least;      // largest; smallest; smallest of the threads' largest ones
};
template <int WAVES>
__device__ __forceinline__ SfRange sf_range(SfRange r, SfRange* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    r.top = fmaxf(r.top, __shfl_xor(r.top, o));
    r.low = fminf(r.low, __shfl_xor(r.low, o));
    r.least = fminf(r.least, __shfl_xor(r.least, o));
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = r;
  __syncthreads();
  r = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    r.top = fmaxf(r.top, red[w].top);
    r.low = fminf(r.low, red[w].low);
    r.least = fminf(r.least, red[w].least);
  }
  return r;
}

// Sums of the threads before and of all threads.
template <int WAVES, typename A>
__device__ __forceinline__ void sf_scan(A own, A* red, A& before, A& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  A upto = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const A lower = __shfl_up(upto, o);
    if (lane >= o) upto += lower;
  }
  __syncthreads();
  if (lane == 63) red[wave] = upto;
  __syncthreads();
  before = upto - own;
  total = 0;
#pragma unroll 4              // (all 16 at once take registers that the passes need)
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
}

// (up to kSfSteps steps of a group a wave's loads are one after the other; sums are kept for every step of every wave)
constexpr int kSfBins = 2048, kSfListed = 2048, kSfSteps = 128;

template <int CELLS>
struct SfShared {
  u64 bins[kSfBins];
  u64 order[kSfListed];                 // listed classes: key, 2^32 - 1 - index; the later class has the smaller number
  u64 cells[CELLS];
  u64 red[16];
  double red_double[16];
  SfRange range[16];
  u64 above;
  int where, until, listed, gathered, found;
  uint32_t found_key, lowest, highest;
  int found_index;
  u64 found_order;
};

__device__ __forceinline__ u64 sf_order(uint32_t key, int c) { return static_cast<u64>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(c)); }
__device__ __forceinline__ uint32_t sf_order_key(u64 o) { return static_cast<uint32_t>(o >> 32); }
__device__ __forceinline__ int sf_order_class(u64 o) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(o)); }

// The first `count` numbers in falling order: a bitonic network over the power of two above (numbers of 0 are added).
template <int NT>
__device__ __forceinline__ void sf_sort(u64* order, int count) {
  const int tid = threadIdx.x;
  int n = 2;
  while (n < count) n *= 2;
  __syncthreads();
  for (int i = count + tid; i < n; i += NT) order[i] = 0;
  __syncthreads();
  for (int size = 2; size <= n; size *= 2)
    for (int gap = size / 2; gap > 0; gap /= 2) {
      for (int t = tid; t < n / 2; t += NT) {
        const int i = 2 * t - (t & (gap - 1));
        const u64 a = order[i], b = order[i + gap];
        if ((a < b) == ((i & size) == 0)) {
          order[i] = b;
          order[i + gap] = a;
        }
      }
      __syncthreads();
    }
}

// A row in vectors of E elements, step after step 64 U neighbouring ones a wave; the last n % E classes are a step of their own, one for
// each of the first threads.  U is 1 up to kSfSteps steps.  Every pass reads the row again, from the caches but for the first one;
// the next step is on its way, of fp32 the next two.  (With four of bfloat16 a draw of 8 rows takes 10% longer and one of 4096 as long; fp32,
// 4096 rows, top-p 0.9: 488 us with one, 458 with two, 451 with four, which cost 256 rows 55 us for 53.)
template <typename T, int NT>
struct SfRow {
  static constexpr int E = 16 / sizeof(T), AHEAD = sizeof(T) == 4 ? 2 : 1;
  const T* __restrict__ x;
  int whole, rest, run, steps;         // run: U E classes
  __device__ __forceinline__ SfRow(const T* __restrict__ x_, int n) : x(x_), whole(n / E * E), rest(n % E) {
    const int vectors = n / E, most = NT * kSfSteps;
    run = vectors > most ? (vectors + most - 1) / most * E : E;
    const int64_t all = static_cast<int64_t>(NT) * run;
    steps = static_cast<int>((whole + all - 1) / all);
  }
  // fn(values, first class) for neighbouring classes of this thread (E of them, or one), done(step) behind every step, for all threads
  template <typename Fn, typename Done>
  __device__ __forceinline__ void each(Fn&& fn, Done&& done) const {
    const int tid = static_cast<int>(threadIdx.x);
    if (run == E) {
      Some<T, E> ahead[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        ahead[i].clear();
        if ((i * NT + tid) * E < whole) ahead[i].load(x + (i * NT + tid) * E);
      }
      for (int v = 0; v < steps; v += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int at = ((v + i) * NT + tid) * E, later = at + AHEAD * NT * E;
          float value[E];
#pragma unroll
          for (int e = 0; e < E; ++e) value[e] = ahead[i].get(e);
          if (later < whole) ahead[i].load(x + later);
          if (at < whole) fn(value, at);
          if (v + i < steps) done(v + i);
          if constexpr (AHEAD > 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      const int64_t wave_first = (tid & ~63) * static_cast<int64_t>(run) + (tid & 63) * E;
      for (int v = 0; v < steps; ++v) {
        const int64_t first = v * static_cast<int64_t>(NT) * run + wave_first;
        for (int j = 0; j < run / E; ++j) {
          const int64_t at = first + j * 64 * E;
          if (at >= whole) break;
          Some<T, E> some;
          some.load(x + at);
          float value[E];
#pragma unroll
          for (int e = 0; e < E; ++e) value[e] = some.get(e);
          fn(value, static_cast<int>(at));
        }
        done(v);
      }
    }
    if (tid < rest) {
      const float value[1] = {static_cast<float>(x[whole + tid])};
      fn(value, whole + tid);
    }
    done(steps);
  }
  template <typename Fn>
  __device__ __forceinline__ void each(Fn&& fn) const {
    each(fn, [](int) {});
  }
  // the cell (step and wave) of a class
  __device__ __forceinline__ int cell(int c) const { return c < whole ? c / run / 64 : steps * (NT / 64); }
  // fn(value, class) for the classes of lane `lane` of a cell: wave `wave` of step `step`
  template <typename Fn>
  __device__ __forceinline__ void each_of_cell(int step, int wave, int lane, Fn&& fn) const {
    const bool of_rest = step == steps;
    const int64_t begin = of_rest ? whole + lane : (static_cast<int64_t>(step) * NT + wave * 64 + lane) * run;
    const int64_t end = of_rest ? begin + (lane < rest ? 1 : 0) : begin + run < whole ? begin + run : whole;
    for (int64_t c = begin; c < end; ++c) fn(static_cast<float>(x[c]), static_cast<int>(c));
  }
};

// One work group per row, in passes over it: the range, with top-k along with the counts of 2048 bins of logits, which say in what bin the
// border lies.  Where the classes up to this bin are at most kSfListed, the next pass lists them in the LDS, and the draw is among them.
// With top-p alone a pass adds the classes' weights to bins, about, and says where the border will be, and one with exact weights sums
// those in front of it by cells (a step of a wave), lists those about it and finds it among them; the draw is in the cell at which the
// sums pass the number.  Where min-p seems to decide before top-p does, a pass sums what it keeps and all, exactly; if these sums say so,
// the draw is among those, else top-p's pass follows.  Without top-k and top-p one pass sums all.  Where a list does not hold the classes of a border's bin (thousands of equal
// or nearly equal ones), the border is narrowed by bins of their keys to a class.
// What bounds it: 4096 rows of 50257 fp32 classes (823 MB; 161 us to read them once at the rate of a large copy; normal logits of deviation
// 2) take 241 us with T = 0 and 258 with top-k 40 (two reads, 6.4 TB/s), 326 without filters, 322 with min-p 0.05, 426 with top-p 0.9 and
// min-p 0.05, and 450 with top-p 0.9, of which 80% are vector instructions, 66 a class, most of them for the exact weights.  8 rows take 10 us with T = 0, 22 with top-k 40 and 42 with top-p 0.9: one CU a row and the barriers
// between the passes.
template <typename T, int NT>
static __global__ __launch_bounds__(NT, 4) void sf_row_kernel(SfParams p) {
  constexpr int WAVES = NT / 64, CELLS = (kSfSteps + 1) * WAVES;
  using Row = SfRow<T, NT>;
  __shared__ SfShared<CELLS> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.classes;
  const int64_t row_index = p.first_row + blockIdx.x;
  const Row row(static_cast<const T*>(p.logits) + row_index * p.ld, n);
  const SfFilter filter(p, row_index);

  // Bins of logits: number round(x a) - round(top a), a < 0, that is 0 for the largest and more for smaller ones.
  float a = 0.f, base = 0.f;
  auto bin_at = [&](float v) { return rintf(v * a) - base; };
  auto bin_of = [&](float v) { return static_cast<int>(__builtin_amdgcn_fmed3f(bin_at(v), 0.f, static_cast<float>(kSfBins - 1))); };
  uint32_t* const counts = reinterpret_cast<uint32_t*>(sh.bins);
  auto clear_bins = [&] {
    __syncthreads();
    for (int b = tid; b < kSfBins; b += NT) sh.bins[b] = 0;
    __syncthreads();
  };

  // The range; for top-k in the same pass, before the top is known, the counts of bins that are T / 32 wide (or 1 / 64), whose numbers are
  // taken modulo 2048.  They serve if the row's finite logits span no more than these 64 T.  (4096 rows of 50257 classes, top-k 40: 279 us
  // for 356 with a pass of their own; for top-p, whose sums are dearer and whose bins hold more classes to put in order, nothing is won.)
  const bool by_k = filter.k > 0 && filter.k < n;
  bool early = by_k && filter.good() && !filter.greedy();
  if (early) {
    a = static_cast<float>(-32. / (filter.t < 0.5 ? 0.5 : filter.t));
    early = a < -1e-30f;
  }
  SfRange range{-INFINITY, INFINITY, 0.f};
  bool bad = !filter.good();
  if (early) {
    clear_bins();
    row.each([&](const auto& v, int) {
#pragma unroll
      for (const float x : v) {
        bad = bad || !(x < INFINITY);
        range.top = fmaxf(range.top, x);
        if (x > -INFINITY) {
          range.low = fminf(range.low, x);
          // (the sum with 1.5 2^23 holds the integer in its low bits)
          atomicAdd(counts + (__builtin_bit_cast(uint32_t, rintf(x * a) + 12582912.f) & (kSfBins - 1)), 1u);
        }
      }
    });
  } else {
    row.each([&](const auto& v, int) {
#pragma unroll
      for (const float x : v) {
        bad = bad || !(x < INFINITY);
        range.top = fmaxf(range.top, x);
        range.low = fminf(range.low, x);
      }
    });
  }
  range.least = range.top;
  bad = __syncthreads_or(bad) != 0;
  range = sf_range<WAVES>(range, sh.range);
  const float top = range.top;
  if (bad || top == -INFINITY) {
    if (tid == 0) {
      p.targets[row_index] = -1;
      if (p.invalid != nullptr) *p.invalid = 1;
    }
    return;
  }
  if (filter.greedy()) {
    int best = 0x7fffffff;
    row.each([&](const auto& v, int at) {
      int c = at;
      for (const float x : v) {
        best = x == top && c < best ? c : best;
        ++c;
      }
    });
    if (tid == 0) sh.where = 0x7fffffff;
    __syncthreads();
    if (best != 0x7fffffff) atomicMin(&sh.where, best);
    __syncthreads();
    if (tid == 0) p.targets[row_index] = sh.where;
    return;
  }

  const SfWeight weight(top, filter.exponent(), p.shift);
  const double least = filter.least(weight.scale);
  auto drawn = [&](double w) -> u64 { return w < least ? 0 : SfWeight::whole(w); };
  float border_value = -INFINITY;    // kept: above the value, and equal to it up to the index
  int border_index = -1;
  // (bit by bit: no branches)
  auto kept = [&](float v, int c) -> bool { return (v > border_value) | ((v == border_value) & (c <= border_index)); };
  const float lightest = static_cast<float>(static_cast<double>(top) - 37. * filter.t);      // weights of classes below round to 0
  int start = 0;                     // the place of bin 0
  if (early) {
    early = fabsf(top * a) < 4e6f && fabsf(range.low * a) < 4e6f && rintf(range.low * a) - rintf(top * a) < static_cast<float>(kSfBins);
    base = rintf(top * a);
    start = static_cast<int>(early ? base : 0.f) & (kSfBins - 1);
  }
  auto set_bins = [&](float low) {
    const float s = static_cast<float>(kSfBins - 2) / (top - low);
    a = top > low && s < INFINITY ? -s : 0.f;
    base = rintf(top * a);
    start = 0;
  };
  // The first bin at which the sum reaches `target` (made from the sum of all): its number and the sum in front of it in `sh`.
  // False if none does.
  auto cross = [&](const auto* bins, auto&& make_target, u64& target) {
    constexpr int PER = kSfBins / NT;
    __syncthreads();
    u64 own = 0, before, total;
#pragma unroll
    for (int b = 0; b < PER; ++b) own += bins[(start + tid * PER + b) & (kSfBins - 1)];
    sf_scan<WAVES>(own, sh.red, before, total);
    target = make_target(total);
    if (before < target && before + own >= target) {
      int b = tid * PER;
      for (; before + bins[(start + b) & (kSfBins - 1)] < target; ++b) before += bins[(start + b) & (kSfBins - 1)];
      sh.where = b;
      sh.above = before;
    }
    __syncthreads();
    return total >= target;
  };
  bool full = false;                 // the list, as far as this wave knows
  auto clear_list = [&] {
    __syncthreads();
    full = false;
    if (tid == 0) {
      sh.listed = 0;
      sh.lowest = 0xffffffffu;
      sh.highest = 0;
    }
    __syncthreads();
  };
  // Lists the wanted of neighbouring classes; one addition to the counter a wave, and none once the list is full.
  auto list = [&](const auto& want, const auto& v, int at) {
    constexpr int N = sizeof(v) / sizeof(float);
    u64 mask[N];
    int count = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      mask[e] = __ballot(want[e] && !full);
      count += __popcll(mask[e]);
    }
    if (count == 0) return;
    int base = 0;
    if (lane == __ffsll(__ballot(true)) - 1) base = atomicAdd(&sh.listed, count);
    base = __builtin_amdgcn_readfirstlane(base);
    full = base + count > kSfListed;
    if (full) return;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (want[e]) sh.order[base + __popcll(mask[e] & ((1ull << lane) - 1))] = sf_order(sf_key(v[e]), at + e);
      base += __popcll(mask[e]);
    }
  };
  // Of `count` numbers, fn(number, its weight as worth(number), the weight in front of it).  (Weights are made twice: kept they take
  // registers that the passes need.)
  auto each_of = [&](const u64* numbers, int count, auto&& worth, auto&& fn) {
    const int per = (count + NT - 1) / NT, from = tid * per, to = from + per < count ? from + per : count;
    u64 own = 0, before, total;
#pragma unroll 1
    for (int j = from; j < to; ++j) own += worth(numbers[j]);
    sf_scan<WAVES>(own, sh.red, before, total);
#pragma unroll 1
    for (int j = from; j < to; ++j) {
      const u64 w = worth(numbers[j]);
      fn(numbers[j], w, before);
      before += w;
    }
  };
  // The class of index order at which the sums of the cells exceed `target`: its cell in sh.where, the sum in front in sh.above.
  auto cell_of = [&](auto&& make_target, u64& target) {
    __syncthreads();
    const int cells = (row.steps + 1) * WAVES, per = (cells + NT - 1) / NT;
    u64 own = 0, before, all;
    for (int i = 0; i < per; ++i)
      if (tid * per + i < cells) own += sh.cells[tid * per + i];
    sf_scan<WAVES>(own, sh.red, before, all);
    target = make_target(all);
    if (before <= target && before + own > target) {
      int i = tid * per;
      for (; before + sh.cells[i] <= target; ++i) before += sh.cells[i];
      sh.where = i;
      sh.above = before;
    }
    __syncthreads();
  };
  // In that cell (by one wave): found(class) for the class at which `value`s exceed the target.
  auto class_of = [&](u64 target, auto&& value, auto&& found) {
    if (wave != 0) return;
    const int step = sh.where / WAVES, of_wave = sh.where % WAVES;
    u64 mine = 0;
    row.each_of_cell(step, of_wave, lane, [&](float v, int c) { mine += value(v, c); });
    u64 upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 lower = __shfl_up(upto, o);
      if (lane >= o) upto += lower;
    }
    u64 from = sh.above + upto - mine;
    if (from <= target && from + mine > target)
      row.each_of_cell(step, of_wave, lane, [&](float v, int c) {
        const u64 w = value(v, c);
        if (from <= target && from + w > target) found(c);
        from += w;
      });
  };
  u64 sum = 0;
  auto to_cell = [&](int step) {
    const u64 s = wave_sum(sum);
    if (lane == 0) sh.cells[step * WAVES + wave] = s;
    sum = 0;
  };
  // The border in bin sh.where, `target` counts (weights) from the top, as a value and an index: of the classes in(value, class) in
  // this bin.  Where they are too many for the list, bins of equal parts of their keys take the place of the bin, until it is few
  // enough classes or one key, whose classes are counted by index.
  auto narrow = [&](u64 target, auto&& in, auto&& worth) {
    const int bin = sh.where;
    u64 above = sh.above;
    uint32_t low = 0, high = 0xffffffffu;
    for (;;) {
      uint32_t least_key = 0xffffffffu, most_key = 0;
      clear_list();
      row.each([&](const auto& v, int at) {
        constexpr int N = sizeof(v) / sizeof(float);
        bool want[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t kk = sf_key(v[e]);
          want[e] = kk >= low && kk <= high && bin_of(v[e]) == bin && in(v[e], at + e);
          least_key = want[e] && kk < least_key ? kk : least_key;
          most_key = want[e] && kk > most_key ? kk : most_key;
        }
        list(want, v, at);
      });
      if (most_key >= least_key) {
        atomicMin(&sh.lowest, least_key);
        atomicMax(&sh.highest, most_key);
      }
      __syncthreads();
      const int count = sh.listed;
      low = sh.lowest;
      high = sh.highest;
      if (count <= kSfListed) {
        sf_sort<NT>(sh.order, count);
        each_of(sh.order, count, [&](u64 o) { return worth(sf_value(sf_order_key(o))); }, [&](u64 o, u64 w, u64 before) {
          if (above + before < target && above + before + w >= target) {
            sh.found_key = sf_order_key(o);
            sh.found_index = sf_order_class(o);
          }
        });
        break;
      }
      if (low == high) {
        const u64 w = worth(sf_value(low)), nth = (target - above + w - 1) / w - 1;
        auto equal = [&](float v, int c) -> u64 { return sf_key(v) == low && in(v, c) ? 1 : 0; };
        row.each([&](const auto& v, int at) {
          int c = at;
          for (const float x : v) sum += equal(x, c++);
        }, to_cell);
        u64 unused;
        cell_of([&](u64) { return nth; }, unused);
        class_of(nth, equal, [&](int c) {
          sh.found_key = low;
          sh.found_index = c;
        });
        break;
      }
      const int bits = 32 - __clz(high - low), shift = bits > 11 ? bits - 11 : 0;
      clear_bins();
      row.each([&](const auto& v, int at) {
        int c = at;
        for (const float x : v) {
          const uint32_t kk = sf_key(x);
          if (kk >= low && kk <= high && bin_of(x) == bin && in(x, c)) {
            const u64 w = worth(x);
            if (w != 0) atomicAdd(sh.bins + ((high - kk) >> shift), w);
          }
          ++c;
        }
      });
      u64 left;
      cross(sh.bins, [&](u64) { return target - above; }, left);
      above += sh.above;
      high -= static_cast<uint32_t>(sh.where) << shift;
      const uint32_t span = (1u << shift) - 1;
      low = high - low > span ? high - span : low;
    }
    __syncthreads();
    border_value = sf_value(sh.found_key);
    border_index = sh.found_index;
  };
  // The draw among up to 64 listed classes by one wave, one class a lane: lanes change places, by counting how many are in front of each,
  // to the order of the filters and then to that of the indices.
  auto draw_of_wave = [&](int count) {
    auto moved = [&](u64 v, int to) {
      const uint32_t low = __builtin_amdgcn_ds_permute(to * 4, static_cast<int>(v)), high = __builtin_amdgcn_ds_permute(to * 4, static_cast<int>(v >> 32));
      return static_cast<u64>(high) << 32 | low;
    };
    auto of_lane = [](u64 v, int j) {
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(v), j), high = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), j);
      return static_cast<u64>(high) << 32 | low;
    };
    auto upto = [&](u64 w) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const u64 lower = __shfl_up(w, o);
        if (lane >= o) w += lower;
      }
      return w;
    };
    const u64 listed = lane < count ? sh.order[lane] : 0;
    int rank = lane < count ? 0 : lane;
    for (int j = 0; j < count; ++j) rank += (of_lane(listed, j) > listed) & (lane < count) ? 1 : 0;
    const u64 o = moved(listed, rank);
    const double w = weight.scaled(sf_value(sf_order_key(o)));
    bool keep = (lane < filter.k) & (lane < count);
    if (filter.p < 1.) {
      const u64 own = keep ? SfWeight::whole(w) : 0, sum = upto(own), border = sf_border(filter.p, of_lane(sum, 63));
      keep = keep & (sum - own < border);
    }
    const int c = lane < count ? sf_order_class(o) : 0x40000000 + lane;
    rank = 0;
    for (int j = 0; j < 64; ++j) rank += __builtin_amdgcn_readlane(c, j) < c ? 1 : 0;
    const u64 own = moved(keep ? drawn(w) : 0, rank), sum = upto(own), target = sf_target(filter.u, of_lane(sum, 63));
    const int by_index = __builtin_amdgcn_ds_permute(rank * 4, c);
    if (sum - own <= target && sum > target) p.targets[row_index] = by_index;
  };
  // The draw among the listed classes: of those in bin `bin` the first `need` are kept, and all in front of this bin.  Each of the
  // three borders (top-k's, top-p's, the drawn class) is first a bin, of logits or of indices, and only its few classes are put in order.
  auto draw_listed = [&](int bin, int need) {
    __syncthreads();
    const int count = sh.listed;
    if (count <= 64) {
      if (wave == 0) draw_of_wave(count);
      return;
    }
    const int rounds = (count + NT - 1) / NT;
    uint32_t own = 0;                               // bit by bit: a class of this thread is kept
    for (int q = 0; q < rounds; ++q) own |= q * NT + tid < count ? 1u << q : 0;
    auto each_own = [&](auto&& fn) {
      for (int q = 0; q < rounds; ++q)
        if ((own >> q & 1) != 0) fn(q, sh.order[q * NT + tid]);
    };
    auto logit = [](u64 o) { return sf_value(sf_order_key(o)); };
    // those wanted, as numbers in falling order in place of the bins
    auto gather = [&](auto&& want, auto&& number) {
      __syncthreads();
      if (tid == 0) sh.gathered = 0;
      __syncthreads();
      for (int q = 0; q < rounds; ++q) {
        const u64 o = sh.order[q * NT + tid];
        const bool in = (own >> q & 1) != 0 && want(o);
        const u64 mask = __ballot(in);
        if (mask == 0) continue;
        int base = 0;
        const int leader = __ffsll(mask) - 1;
        if (lane == leader) base = atomicAdd(&sh.gathered, __popcll(mask));
        base = __builtin_amdgcn_readlane(base, leader);
        if (in) sh.bins[base + __popcll(mask & ((1ull << lane) - 1))] = number(o);
      }
      __syncthreads();
      const int found = sh.gathered;
      sf_sort<NT>(sh.bins, found);
      return found;
    };
    auto same = [](u64 o) { return o; };
    auto keep_from = [&](u64 border) {
      each_own([&](int q, u64 o) { own &= o >= border ? ~0u : ~(1u << q); });
    };
    gather([&](u64 o) { return bin_of(logit(o)) == bin; }, same);
    keep_from(sh.bins[need - 1]);
    if (filter.p < 1.) {
      clear_bins();
      each_own([&](int, u64 o) { atomicAdd(sh.bins + bin_of(logit(o)), weight(logit(o))); });
      u64 target;
      cross(sh.bins, [&](u64 all) { return sf_border(filter.p, all); }, target);
      const int p_bin = sh.where;
      const u64 above = sh.above;
      const int found = gather([&](u64 o) { return bin_of(logit(o)) == p_bin; }, same);
      each_of(sh.bins, found, [&](u64 o) { return weight(logit(o)); }, [&](u64 o, u64 w, u64 before) {
        if (above + before < target && above + before + w >= target) sh.found_order = o;
      });
      __syncthreads();
      keep_from(sh.found_order);
    }
    clear_bins();
    const int bits = 32 - __clz(n - 1), part = bits > 11 ? bits - 11 : 0;
    auto worth = [&](u64 o) { return drawn(weight.scaled(logit(o))); };
    each_own([&](int, u64 o) { atomicAdd(sh.bins + (sf_order_class(o) >> part), worth(o)); });
    u64 target;                                     // (the sum exceeds one number: reaches the next)
    cross(sh.bins, [&](u64 all) { return sf_target(filter.u, all) + 1; }, target);
    const int drawn_part = sh.where;
    const u64 above = sh.above;
    auto turned = [](u64 o) { return o << 32 | o >> 32; };      // the index in front, the lowest first
    const int found = gather([&](u64 o) { return sf_order_class(o) >> part == drawn_part; }, turned);
    each_of(sh.bins, found, [&](u64 o) { return worth(turned(o)); }, [&](u64 o, u64 w, u64 before) {
      if (above + before < target && above + before + w >= target) p.targets[row_index] = sf_order_class(turned(o));
    });
  };

  auto value = [&](float v, int c) -> u64 { return kept(v, c) ? drawn(weight.scaled(v)) : 0; };
  auto draw_cells = [&] {
    u64 target;
    cell_of([&](u64 all) { return sf_target(filter.u, all); }, target);
    class_of(target, value, [&](int c) { p.targets[row_index] = c; });
  };

  if (by_k) {
    float low = range.low;
    for (bool counted = early;; counted = false) {
      if (!counted) {
        // Of as many classes as there are threads, the largest of each thread's, none is below the least of them.  A class further down
        // than 37 T has no weight, kept or not: masks of -inf or of the type's lowest value do not take the bins away from the others.
        low = fmaxf(filter.k <= NT ? range.least : range.low, lightest);
        set_bins(low);
        clear_bins();
        row.each([&](const auto& v, int) {
          for (const float x : v)
            if (x >= low) atomicAdd(counts + bin_of(x), 1u);
        });
      }
      u64 target;
      if (!cross(counts, [&](u64) { return static_cast<u64>(filter.k); }, target)) break;        // all that have weight are kept
      const int bin = sh.where;
      const u64 above = sh.above;
      if (above + counts[(start + bin) & (kSfBins - 1)] <= kSfListed) {
        start = 0;
        clear_list();
        row.each([&](const auto& v, int at) {
          constexpr int N = sizeof(v) / sizeof(float);
          bool want[N];
#pragma unroll
          for (int e = 0; e < N; ++e) want[e] = v[e] >= low && bin_of(v[e]) <= bin;
          list(want, v, at);
        });
        return draw_listed(bin, static_cast<int>(target - above));
      }
      if (counted) continue;
      narrow(target, [&](float v, int) { return v >= low; }, [](float) -> u64 { return 1; });
      break;
    }
  }
  if (filter.p < 1.) {
    // Where the border will be, from 32-bit sums: a weight in its bin, of unit 1 in the middle, is taken as a straight line over the bin
    // (a chord of 2^-drop, off by 4e-5 at most).  (Additions of fp32 numbers in the LDS take three times as long as all the rest of the
    // pass.)
    set_bins(fmaxf(range.low, lightest));
    clear_bins();
    uint32_t* const sums = counts;
    const float drop = a < 0.f ? static_cast<float>(filter.exponent() / -static_cast<double>(a)) : 0.f;
    const float up = exp2f(0.5f * drop), down = exp2f(-0.5f * drop);
    const float middle = 0.5f * (up + down) * p.unit + 8388608.f, slope = (down - up) * p.unit;      // (2^23: as above)
    auto share = [&](float v) {
      const float place = __builtin_fmaf(v, a, -rintf(v * a));       // (one rounding: v * a may be large)
      return __builtin_bit_cast(uint32_t, __builtin_fmaf(place, slope, middle)) - 0x4b000000u;
    };
    auto add_sums = [&](auto all) {        // all: every class is kept (of -inf, in the last bin, nothing is taken)
      row.each([&](const auto& v, int at) {
        int c = at;
        for (const float x : v) {
          if (decltype(all)::value ? x > -INFINITY : kept(x, c)) atomicAdd(sums + bin_of(x), share(x));
          ++c;
        }
      });
    };
    const bool unrestricted = border_index < 0;
    if (unrestricted) add_sums(std::true_type{});
    else add_sums(std::false_type{});
    __syncthreads();
    {
      constexpr int PER_BINS = kSfBins / NT;
      double own[PER_BINS], sum_of = 0., before, total;
#pragma unroll
      for (int q = 0; q < PER_BINS; ++q)
        sum_of += own[q] = static_cast<double>(sums[tid * PER_BINS + q]) * static_cast<double>(exp2f(-drop * static_cast<float>(tid * PER_BINS + q)));
      sf_scan<WAVES>(sum_of, sh.red_double, before, total);
      // Where min-p seems to keep less than top-p would, its classes are summed at once (256 requests with filters of their own: 55 us for
      // 69).  These sums are estimates, whose error grows with |logit| / T (the product with a is rounded) and with the number of classes
      // (unit); 1e-3 is a margin that usually does.  What they say is proved below, as the border's bins are.
      const int least_bin = filter.m > 0. ? bin_of(top + static_cast<float>(filter.t) * __log2f(static_cast<float>(filter.m)) * 0.693147f) + 1 : kSfBins;
      if (tid == 0) {
        sh.where = sh.until = kSfBins - 1;
        sh.found = 0;
      }
      __syncthreads();
      const double border = filter.p * total, margin = 1e-4 * total;
#pragma unroll
      for (int q = 0; q < PER_BINS; ++q) {
        if (before <= border && before + own[q] > border) {
          const int bin = tid * PER_BINS + q;
          sh.where = border - before < margin && bin > 0 ? bin - 1 : bin;
          sh.until = before + own[q] - border < margin && bin < kSfBins - 1 ? bin + 1 : bin;
        }
        before += own[q];
        if (tid * PER_BINS + q == least_bin && before < (filter.p - 1e-3) * total) sh.found = 1;
      }
      clear_list();
    }
    if (sh.found != 0) {
      // Exact sums of what min-p keeps, by cells, and of all.  Where the one is at most top-p's border, so is the weight in front of each of
      // its classes: top-p keeps them all, and the draw is among them.
      u64 own_kept = 0, own_all = 0;
      row.each(
          [&](const auto& v, int at) {
            int c = at;
            for (const float x : v) {
              const double w = weight.scaled(x);
              const u64 whole = kept(x, c++) ? SfWeight::whole(w) : 0;
              own_all += whole;
              sum += w < least ? 0 : whole;
            }
          },
          [&](int step) {
            own_kept += sum;
            to_cell(step);
          });
      const u64 by_least = group_sum<WAVES>(own_kept, sh.red), all = group_sum<WAVES>(own_all, sh.red);
      if (by_least <= sf_border(filter.p, all)) return draw_cells();
    }
    // One pass with exact weights: of the bins in front of the border's (and of a neighbour, where the border is near its edge), by
    // cells; of all others; the classes of these bins.
    const float from_bin = sh.where > 0 ? static_cast<float>(sh.where) : -INFINITY, to_bin = sh.until < kSfBins - 1 ? static_cast<float>(sh.until) : INFINITY;
    u64 own_all = 0, own_above = 0;
    auto add_weights = [&](auto every) {
      row.each(
          [&](const auto& v, int at) {
            constexpr int N = sizeof(v) / sizeof(float);
            bool want[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float bin = bin_at(v[e]);
              const bool in = decltype(every)::value ? true : kept(v[e], at + e);
              const u64 w = in ? weight(v[e]) : 0;
              const bool front = bin < from_bin;
              sum += front ? w : 0;
              own_all += w;
              want[e] = in & !front & (bin <= to_bin);
            }
            list(want, v, at);
          },
          [&](int step) {
            own_above += sum;
            to_cell(step);
          });
    };
    if (unrestricted) add_weights(std::true_type{});
    else add_weights(std::false_type{});
    const u64 above = group_sum<WAVES>(own_above, sh.red), all = group_sum<WAVES>(own_all, sh.red), target = sf_border(filter.p, all);
    const int count = sh.listed;
    if (tid == 0) sh.found = 0;
    if (count <= kSfListed && above < target) {
      sf_sort<NT>(sh.order, count);
      each_of(sh.order, count, [&](u64 o) { return weight(sf_value(sf_order_key(o))); }, [&](u64 o, u64 w, u64 before) {
        if (above + before >= target) return;
        const int c = sf_order_class(o);
        if (w != 0) atomicAdd(sh.cells + row.cell(c), w);
        if (above + before + w >= target) {
          sh.found_key = sf_order_key(o);
          sh.found_index = c;
          sh.found = 1;
        }
      });
    }
    __syncthreads();
    if (sh.found) {
      border_value = sf_value(sh.found_key);
      border_index = sh.found_index;
      if (weight.scaled(border_value) >= least) return draw_cells();       // (else the cells hold what min-p leaves out)
    } else {
      // The border was not there, or the classes too many: the weights of bins, and the border's bin in parts.
      clear_bins();
      row.each([&](const auto& v, int at) {
        int c = at;
        for (const float x : v) {
          if (kept(x, c)) {
            const u64 w = weight(x);
            if (w != 0) atomicAdd(sh.bins + bin_of(x), w);
          }
          ++c;
        }
      });
      u64 same;
      cross(sh.bins, [&](u64) { return target; }, same);
      narrow(target, kept, weight);
    }
  }
  row.each([&](const auto& v, int at) {
    int c = at;
    for (const float x : v) sum += value(x, c++);
  }, to_cell);
  draw_cells();
}

// A group's threads: few where the rows are many, since the waves of small groups, four groups on a CU, wait for each other less
// (4096 rows of 50257 bfloat16 classes, top-k 40: 190 us with 256 threads, 225 with 512), many where they do not fill the card (256 such
// rows: 45, 33 and 33 us with 256, 512 and 1024; top-p 0.9 of 128 fp32 rows: 69, 49 and 46), not many for few classes (256 rows of 5000: 18
// us with 512 and 20 with 1024; of 1000: 18.7 with 256 and 19.7 with 1024), and enough for kSfSteps steps (512 rows of 250000: 265 us in
// steps, 754 in longer runs).
template <typename T>
static int sf_launch(SfParams p, int64_t rows, hipStream_t s) {
  int threads = p.classes <= 2048 || rows >= 1024 ? 256 : p.classes <= 8192 || rows > 256 ? 512 : 1024;
  while (threads < 1024 && p.classes >= threads * kSfSteps * SfRow<T, 512>::E) threads *= 2;
  constexpr int64_t kMost = 1 << 22;                   // rows of a launch: the threads of one are counted in 32 bits
  for (p.first_row = 0; p.first_row < rows; p.first_row += kMost) {
    const dim3 grid(static_cast<unsigned>(rows - p.first_row < kMost ? rows - p.first_row : kMost));
    if (threads == 256) hipLaunchKernelGGL((sf_row_kernel<T, 256>), grid, dim3(256), 0, s, p);
    else if (threads == 512) hipLaunchKernelGGL((sf_row_kernel<T, 512>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((sf_row_kernel<T, 1024>), grid, dim3(1024), 0, s, p);
    const int rc = check_launch();
    if (rc != AK_OK) return rc;
  }
  return AK_OK;
}

}  // namespace ak

extern "C" int ak_sample_filtered(const void* logits, int dtype, int64_t rows, int64_t classes, int64_t ld, const void* u, int u_is_double,
                                  double temperature, const float* temperatures, int64_t top_k, const int64_t* top_ks, double top_p,
                                  const float* top_ps, double min_p, const float* min_ps, int64_t* targets, int* invalid, ak_stream_t stream) {
  using namespace ak;
  if (rows < 0 || classes <= 0 || (rows > 1 && ld < classes) || !is_element_type(dtype)) return AK_ERR_ARG;
  if (temperatures == nullptr && !(temperature >= 0.)) return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (logits == nullptr || u == nullptr || targets == nullptr) return AK_ERR_ARG;
  if (classes > (1 << 30) || rows > 0x7fffffff) return AK_ERR_TOO_LARGE;
  int bits = 0;
  while ((1ll << bits) < classes) ++bits;
  const int shift = 62 - bits < 51 ? 62 - bits : 51;
  const SfParams p{logits, u, temperatures, top_ks, top_ps, min_ps, targets, invalid, ld, 0, temperature, top_p, min_p, top_k,
                   static_cast<int>(classes), u_is_double, shift, static_cast<float>(1u << (bits > 9 ? 31 - bits : 22))};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto type) {
    return sf_launch<typename decltype(type)::type>(p, rows, s);
  });
}
