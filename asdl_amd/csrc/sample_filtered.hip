// One draw per row from softmax(logits / T) restricted by top-k, top-p and min-p, with one uniform number u per row.
// Classes are ordered by logit, the lowest index first among equals; with weights w = exp((x - max x) / T):
//   top-k  keeps the first k;  top-p  keeps a class while the weight in front of it is below p times the weight of what top-k kept;
//   min-p  keeps w >= min_p;   the draw is the first class, by index, at which the kept weight up to there exceeds u times all of it.
// A border between two classes is where a sum over up to all classes passes a number, so sums have to be the same whatever order
// they are formed in: a weight is an integer, w 2^s rounded, with s so large that the sum over all classes fits 63 bits (46 bits below
// the point for 50257 classes), and integers add exactly.  w itself is computed in double.
// The kept classes are those above a key (the logit's bits in an order that integers keep) and, of those equal to it, the ones up to an
// index.
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
  int64_t ld;
  double temperature, top_p, min_p;
  int64_t top_k;
  int classes, u_double, shift;
};

__device__ __forceinline__ uint32_t sf_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);       // (-0 and 0 are equal)
  return b ^ ((b >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float sf_value(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// w = exp((x - top) / T) = 2^y in units of 2^-shift: y = (x - top) (log2 e / T) is split into the nearest integer and a rest in
// [-1/2, 1/2], whose power is 1 + f q(f), q interpolated at the ten Chebyshev points (off by at most 6e-16; exactly 1 at f = 0).
struct SfWeight {
  double top, c, scale;
  int shift;
  __device__ __forceinline__ double scaled(float x) const {
    double y = (static_cast<double>(x) - top) * c;
    y = fmax(y, -2000.);
    if (x == -INFINITY) y = -2000.;                      // (also where c is 0)
    const double whole = rint(y), f = y - whole;
    double q = 7.070977866508138e-09;
    q = fma(q, f, 1.0205905413765595e-07);
    q = fma(q, f, 1.3215451633221434e-06);
    q = fma(q, f, 1.5252672924850737e-05);
    q = fma(q, f, 0.00015403530424776529);
    q = fma(q, f, 0.0013333558200794592);
    q = fma(q, f, 0.009618129107618665);
    q = fma(q, f, 0.05550410866465167);
    q = fma(q, f, 0.24022650695910075);
    q = fma(q, f, 0.6931471805599462);
    return ldexp(fma(q, f, 1.), static_cast<int>(whole) + shift);
  }
  // rounded to an integer by the addition of 2^52 (scaled() is at most that)
  static __device__ __forceinline__ u64 whole(double scaled) {
    return __builtin_bit_cast(u64, scaled + 4503599627370496.) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ u64 operator()(float x) const { return whole(scaled(x)); }
};

struct SfShared {
  u64 mass[256];
  uint32_t count[256];
  u64 red[16];
  int red_int[16];
  u64 above;
  uint32_t digit;
  int found;
};

// The first bin from the top at which the sum of `v` reaches `target`; one wave, lane l has bins 255 - 4 l ... 252 - 4 l.
__device__ __forceinline__ void sf_crossing(const u64* v, u64 target, uint32_t& digit, u64& above) {
  const int lane = threadIdx.x & 63;
  u64 own[4], sum = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += own[e] = v[255 - 4 * lane - e];
  u64 upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 before = __shfl_up(upto, o);
    if (lane >= o) upto += before;
  }
  u64 at = upto - sum;
  if (at < target && upto >= target) {
    int e = 0;
    while (at + own[e] < target) at += own[e++];
    digit = 255 - 4 * lane - e;
    above = at;
  }
}

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

__device__ __forceinline__ void sf_no_distribution(const SfParams& p, int64_t row) {
  p.targets[row] = -1;
  if (p.invalid != nullptr) *p.invalid = 1;
}

// A row of any length and any distribution that is not greedy, read from memory in every step.  The key at which a sum of counts or
// weights from the top reaches a number is found digit by digit, 8 bits of it a step, from histograms.
template <typename T, int NT>
__device__ __forceinline__ void sf_general(const SfParams& p, int64_t row, const SfFilter& filter, float top, SfShared& sh) {
  constexpr int WAVES = NT / 64;
  u64* bins = sh.mass;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.classes;
  const T* __restrict__ x = static_cast<const T*>(p.logits) + row * p.ld;
  const int64_t k = filter.k;
  const double top_p = filter.p;
  const SfWeight weight{static_cast<double>(top), filter.exponent(), static_cast<double>(1ull << p.shift), p.shift};
  uint32_t key = 0;           // classes above it are kept, and the first `ties` equal to it
  uint32_t ties = 0xffffffffu, equal = 0;
  // The digits of the key at which the count (by weight: the weight) from the top reaches `target`; `floor_key`, `floor_ties`:
  // classes below are out, and of those equal so many are in.
  auto select = [&](bool by_weight, u64 target, uint32_t floor_key, uint32_t floor_ties, uint32_t& out_key, u64& above_all, uint32_t& out_equal) {
    uint32_t prefix = 0;
    u64 above = 0;
    for (int at = 24; at >= 0; at -= 8) {
      for (int b = tid; b < 256; b += NT) {
        bins[b] = 0;
        sh.count[b] = 0;
      }
      __syncthreads();
      for (int c = tid; c < n; c += NT) {
        const float v = static_cast<float>(x[c]);
        const uint32_t kk = sf_key(v);
        if (at < 24 && (kk >> (at + 8)) != prefix) continue;
        if (kk < floor_key || (kk == floor_key && floor_ties != 0xffffffffu)) continue;
        atomicAdd(&sh.count[kk >> at & 255], 1u);
        if (by_weight) atomicAdd(&bins[kk >> at & 255], weight(v));
      }
      __syncthreads();
      if (tid == 0 && floor_ties != 0xffffffffu && (at == 24 || (floor_key >> (at + 8)) == prefix)) {
        sh.count[floor_key >> at & 255] += floor_ties;
        bins[floor_key >> at & 255] += floor_ties * weight(sf_value(floor_key));
      }
      __syncthreads();
      if (!by_weight) {
        for (int b = tid; b < 256; b += NT) bins[b] = sh.count[b];
        __syncthreads();
      }
      if (wave == 0) sf_crossing(bins, target - above, sh.digit, sh.above);
      __syncthreads();
      above += sh.above;
      prefix = prefix << 8 | sh.digit;
      out_equal = sh.count[sh.digit];
      __syncthreads();
    }
    out_key = prefix;
    above_all = above;
  };

  if (k > 0 && k < n) {
    u64 above;
    select(false, static_cast<u64>(k), 0, 0xffffffffu, key, above, equal);
    ties = static_cast<uint32_t>(static_cast<u64>(k) - above);
    if (ties >= equal) ties = 0xffffffffu;
  }
  auto in_k = [&](uint32_t kk) { return kk > key || (kk == key && ties == 0xffffffffu); };
  if (top_p < 1.) {
    u64 all = 0;
    for (int c = tid; c < n; c += NT) {
      const float v = static_cast<float>(x[c]);
      if (in_k(sf_key(v))) all += weight(v);
    }
    all = group_sum<WAVES>(all, sh.red);
    if (ties != 0xffffffffu) all += ties * weight(sf_value(key));
    const u64 target = sf_border(top_p, all);
    uint32_t key2;
    u64 above;
    select(true, target, key, ties, key2, above, equal);
    const u64 w = weight(sf_value(key2));
    const u64 need = w == 0 ? equal : (target - above + w - 1) / w;
    key = key2;
    ties = need >= equal ? (ties != 0xffffffffu && equal == ties ? ties : 0xffffffffu) : static_cast<uint32_t>(need);
  }

  // the index behind which classes equal to the key are out
  int last_tie = 0x7fffffff;
  if (ties != 0xffffffffu) {
    uint32_t before = 0;
    for (int c0 = 0; c0 < n; c0 += NT) {
      const int c = c0 + tid;
      const bool is = c < n && sf_key(static_cast<float>(x[c])) == key;
      const u64 mask = __ballot(is);
      if (lane == 0) sh.red_int[wave] = __popcll(mask);
      __syncthreads();
      uint32_t rank = before + __popcll(mask & ((1ull << lane) - 1)), sum = 0;
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) rank += sh.red_int[w];
        sum += sh.red_int[w];
      }
      if (is && rank == ties - 1) sh.found = c;
      before += sum;
      __syncthreads();
      if (before >= ties) break;
    }
    last_tie = sh.found;
  }
  auto kept = [&](int c) -> u64 {
    const float v = static_cast<float>(x[c]);
    const uint32_t kk = sf_key(v);
    if (kk < key || (kk == key && c > last_tie)) return 0;
    const double w = weight.scaled(v);
    return w < filter.least(weight.scale) ? 0 : SfWeight::whole(w);
  };
  u64 all = 0;
  for (int c = tid; c < n; c += NT) all += kept(c);
  all = group_sum<WAVES>(all, sh.red);
  const u64 target = sf_target(filter.u, all);
  u64 before = 0;
  for (int c0 = 0; c0 < n; c0 += NT) {
    const int c = c0 + tid;
    const u64 w = c < n ? kept(c) : 0;
    u64 upto = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 lower = __shfl_up(upto, o);
      if (lane >= o) upto += lower;
    }
    __syncthreads();
    if (lane == 63) sh.red[wave] = upto;
    __syncthreads();
    u64 sum = 0;
    for (int v = 0; v < WAVES; ++v) {
      if (v < wave) upto += sh.red[v];
      sum += sh.red[v];
    }
    upto += before;
    if (upto > target && upto - w <= target) p.targets[row] = c;
    before += sum;
    if (before > target) return;
  }
}

// The largest and smallest over a work group.
struct SfRange {
  float top, low, least;      // largest; smallest finite one; smallest of the lanes' largest ones
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
template <int WAVES>
__device__ __forceinline__ void sf_scan(u64 own, u64* red, u64& before, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 upto = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 lower = __shfl_up(upto, o);
    if (lane >= o) upto += lower;
  }
  __syncthreads();
  if (lane == 63) red[wave] = upto;
  __syncthreads();
  before = upto - own;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
}

constexpr int kSfBins = 2048, kSfCandidates = 1024, kSfMostSteps = 64;

template <int CELLS>
struct SfRowShared {
  u64 bins[kSfBins];
  u64 weight[kSfCandidates];
  uint32_t key[kSfCandidates];
  int index[kSfCandidates];
  u64 cells[CELLS];
  u64 red[16];
  SfRange range[16];
  u64 above;
  int where, candidates, found_index;
  uint32_t found_key;
};

// A row in vectors of E elements, step after step NT of them: class (step NT + thread) E + e; the last n % E classes are a step of
// their own, one for each of the first threads.  Held in registers, or read in every pass.
template <typename T, int NT, int V, bool HELD>
struct SfRow {
  static constexpr int E = 16 / sizeof(T);
  const T* __restrict__ x;
  int whole, rest, steps;
  Some<T, E> held[HELD ? V : 1];
  T last;
  __device__ __forceinline__ SfRow(const T* __restrict__ x_, int n) : x(x_), whole(n / E * E), rest(n % E), steps(HELD ? V : (n / E + NT - 1) / NT) {
    if constexpr (HELD) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        held[v].clear();
        if ((v * NT + static_cast<int>(threadIdx.x)) * E < whole) held[v].load(x + (v * NT + threadIdx.x) * E);
      }
    }
    last = static_cast<T>(0.f);
    if (static_cast<int>(threadIdx.x) < rest) last = x[whole + threadIdx.x];
  }
  // fn(value, class) for the classes of this thread, done(step) behind every step
  template <typename Fn, typename Done>
  __device__ __forceinline__ void each(Fn&& fn, Done&& done) const {
    if constexpr (HELD) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int at = (v * NT + static_cast<int>(threadIdx.x)) * E;
        if (at < whole)
#pragma unroll
          for (int e = 0; e < E; ++e) fn(held[v].get(e), at + e);
        done(v);
      }
    } else {
      for (int v = 0; v < steps; ++v) {
        const int at = (v * NT + static_cast<int>(threadIdx.x)) * E;
        if (at < whole) {
          Some<T, E> some;
          some.load(x + at);
#pragma unroll
          for (int e = 0; e < E; ++e) fn(some.get(e), at + e);
        }
        done(v);
      }
    }
    if (static_cast<int>(threadIdx.x) < rest) fn(static_cast<float>(last), whole + static_cast<int>(threadIdx.x));
    done(steps);
  }
  template <typename Fn>
  __device__ __forceinline__ void each(Fn&& fn) const {
    each(fn, [](int) {});
  }
  // the cell (step and wave) of a class
  __device__ __forceinline__ int cell(int c) const { return c < whole ? c / (NT * E) * (NT / 64) + c % (NT * E) / (64 * E) : steps * (NT / 64); }
};

// One work group per row, in three or four passes over it: the range; with top-k the counts of 2048 bins between its ends, which say in
// what bin the border lies; with top-p the weights of such bins; the kept weight of every cell (a step of a wave).  The classes of a
// border's bin are listed and ranked by counting; more than kSfCandidates of them go to sf_general.
template <typename T, int NT, int V, bool HELD>
static __global__ __launch_bounds__(NT) void sf_row_kernel(SfParams p) {
  constexpr int WAVES = NT / 64, CELLS = ((HELD ? V : kSfMostSteps) + 1) * WAVES;
  using Row = SfRow<T, NT, V, HELD>;
  constexpr int E = Row::E;
  __shared__ SfRowShared<CELLS> sh;
  __shared__ SfShared general;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.classes;
  const int64_t row_index = blockIdx.x;
  const Row row(static_cast<const T*>(p.logits) + row_index * p.ld, n);
  const SfFilter filter(p, row_index);

  SfRange range{-INFINITY, INFINITY, 0.f};
  int bad = filter.good() ? 0 : 1;
  row.each([&](float v, int) {
    bad |= v < INFINITY ? 0 : 1;
    range.top = fmaxf(range.top, v);
    range.low = fminf(range.low, v > -INFINITY ? v : INFINITY);
  });
  range.least = range.top;
  bad = __syncthreads_or(bad);
  range = sf_range<WAVES>(range, sh.range);
  const float top = range.top;
  if (bad != 0 || top == -INFINITY) {
    if (tid == 0) sf_no_distribution(p, row_index);
    return;
  }
  if (filter.greedy()) {
    int best = 0x7fffffff;
    row.each([&](float v, int c) { best = v == top && c < best ? c : best; });
    if (tid == 0) sh.where = 0x7fffffff;
    __syncthreads();
    if (best != 0x7fffffff) atomicMin(&sh.where, best);
    __syncthreads();
    if (tid == 0) p.targets[row_index] = sh.where;
    return;
  }

  uint32_t key = 0;                  // kept: above the key, and equal to it up to the index
  int last = 0x7fffffff;
  float scale = 0.f;
  auto kept = [&](uint32_t kk, int c) { return kk > key || (kk == key && c <= last); };
  auto bin_of = [&](float v) {       // the same or a later bin for a smaller logit
    const float b = (top - v) * scale;
    return b < static_cast<float>(kSfBins - 1) ? static_cast<int>(b) : kSfBins - 1;
  };
  auto set_scale = [&](float low) {
    const float s = static_cast<float>(kSfBins - 1) / (top - low);
    scale = top > low && s < INFINITY ? s : 0.f;
  };
  auto clear_bins = [&] {
    for (int b = tid; b < kSfBins; b += NT) sh.bins[b] = 0;
    if (tid == 0) sh.candidates = 0;
    __syncthreads();
  };
  // The first bin at which the sum reaches `target` (made from the sum of all bins); false if it does not.
  auto cross = [&](auto value, auto make_target, u64& target) {
    constexpr int PER = kSfBins / NT;
    u64 own = 0, before, total;
#pragma unroll
    for (int b = 0; b < PER; ++b) own += value(tid * PER + b);
    sf_scan<WAVES>(own, sh.red, before, total);
    target = make_target(total);
    if (before < target && before + own >= target) {
      int b = tid * PER;
      for (u64 v = value(b); before + v < target; v = value(++b)) before += v;
      sh.where = b;
      sh.above = before;
    }
    __syncthreads();
    return total >= target;
  };
  auto list = [&](uint32_t kk, int c, u64 w) {
    const int i = atomicAdd(&sh.candidates, 1);
    if (i < kSfCandidates) {
      sh.key[i] = kk;
      sh.index[i] = c;
      sh.weight[i] = w;
    }
  };

  if (filter.k > 0 && filter.k < n) {
    // of as many classes as there are threads, the largest of each thread's, none is below the least of them
    const float low = filter.k <= NT && range.least > -INFINITY ? range.least : range.low;
    set_scale(low);
    clear_bins();
    uint32_t* counts = reinterpret_cast<uint32_t*>(sh.bins);
    row.each([&](float v, int) {
      if (v >= low) atomicAdd(counts + bin_of(v), 1u);
    });
    __syncthreads();
    u64 target;
    if (cross([&](int b) { return static_cast<u64>(counts[b]); }, [&](u64) { return static_cast<u64>(filter.k); }, target)) {
      const int border = sh.where;
      row.each([&](float v, int c) {
        if (v >= low && bin_of(v) == border) list(sf_key(v), c, 0);
      });
      __syncthreads();
      const int count = sh.candidates;
      if (count > kSfCandidates) return sf_general<T, NT>(p, row_index, filter, top, general);
      const int nth = static_cast<int>(target - sh.above) - 1;
      for (int j = tid; j < count; j += NT) {
        const uint32_t kk = sh.key[j];
        const int c = sh.index[j];
        int rank = 0;
        for (int i = 0; i < count; ++i) rank += sh.key[i] > kk || (sh.key[i] == kk && sh.index[i] < c) ? 1 : 0;
        if (rank == nth) {
          sh.found_key = kk;
          sh.found_index = c;
        }
      }
      __syncthreads();
      key = sh.found_key;
      last = sh.found_index;
    }
    __syncthreads();
  }

  const SfWeight weight{static_cast<double>(top), filter.exponent(), static_cast<double>(1ull << p.shift), p.shift};
  const double least = filter.least(weight.scale);
  auto drawn = [&](double w) -> u64 { return w < least ? 0 : SfWeight::whole(w); };
  u64 sum = 0;
  auto to_cell = [&](int step) {
    const u64 s = wave_sum(sum);
    if (lane == 0) sh.cells[step * WAVES + wave] = s;
    sum = 0;
  };
  if (filter.p < 1.) {
    // (weights of classes further down than 37 T round to 0)
    set_scale(fmaxf(range.low, static_cast<float>(static_cast<double>(top) - 37. * filter.t)));
    clear_bins();
    row.each([&](float v, int c) {
      if (kept(sf_key(v), c)) {
        const u64 w = weight(v);
        if (w != 0) atomicAdd(sh.bins + bin_of(v), w);
      }
    });
    __syncthreads();
    u64 target;
    cross([&](int b) { return sh.bins[b]; }, [&](u64 total) { return sf_border(filter.p, total); }, target);
    const int border = sh.where;
    const u64 above = sh.above;
    row.each(
        [&](float v, int c) {
          const int b = bin_of(v);
          if (b > border || !kept(sf_key(v), c)) return;
          const double w = weight.scaled(v);
          if (b < border) sum += drawn(w);
          else if (const u64 whole = SfWeight::whole(w); whole != 0) list(sf_key(v), c, whole);
        },
        to_cell);
    __syncthreads();
    const int count = sh.candidates;
    if (count > kSfCandidates) return sf_general<T, NT>(p, row_index, filter, top, general);
    for (int j = tid; j < count; j += NT) {
      const uint32_t kk = sh.key[j];
      const int c = sh.index[j];
      u64 before = above;
      for (int i = 0; i < count; ++i)
        if (sh.key[i] > kk || (sh.key[i] == kk && sh.index[i] < c)) before += sh.weight[i];
      if (before < target && before + sh.weight[j] >= target) {
        sh.found_key = kk;
        sh.found_index = c;
      }
    }
    __syncthreads();
    key = sh.found_key;
    last = sh.found_index;
    for (int j = tid; j < count; j += NT)
      if (kept(sh.key[j], sh.index[j])) {
        const u64 w = drawn(weight.scaled(sf_value(sh.key[j])));
        if (w != 0) atomicAdd(sh.cells + row.cell(sh.index[j]), w);
      }
  } else {
    row.each([&](float v, int c) { if (kept(sf_key(v), c)) sum += drawn(weight.scaled(v)); }, to_cell);
  }
  __syncthreads();

  // the cell in which the draw lies, then the class
  const int cells = (row.steps + 1) * WAVES, per = (cells + NT - 1) / NT;
  u64 own = 0, before, all;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < cells) own += sh.cells[tid * per + i];
  sf_scan<WAVES>(own, sh.red, before, all);
  const u64 target = sf_target(filter.u, all);
  if (before <= target && before + own > target) {
    int i = tid * per;
    for (; before + sh.cells[i] <= target; ++i) before += sh.cells[i];
    sh.where = i;
    sh.above = before;
  }
  __syncthreads();
  if (wave != 0) return;
  const int step = sh.where / WAVES, of_wave = sh.where % WAVES;
  const int at = step < row.steps ? (step * NT + of_wave * 64 + lane) * E : row.whole + lane;
  const int count = step < row.steps ? (at < row.whole ? E : 0) : lane < row.rest ? 1 : 0;
  u64 w[E], mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = 0;
    if (e < count) {
      const float v = static_cast<float>(row.x[at + e]);
      if (kept(sf_key(v), at + e)) w[e] = drawn(weight.scaled(v));
    }
    mine += w[e];
  }
  u64 upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 lower = __shfl_up(upto, o);
    if (lane >= o) upto += lower;
  }
  u64 from = sh.above + upto - mine;
  if (from <= target && from + mine > target) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (from <= target && from + w[e] > target) p.targets[row_index] = at + e;
      from += w[e];
    }
  }
}

// Rows beyond the steps of the kernel above.
template <typename T>
static __global__ __launch_bounds__(1024) void sf_long_kernel(SfParams p) {
  __shared__ SfShared sh;
  __shared__ SfRange red[16];
  __shared__ int first;
  const int64_t row = blockIdx.x;
  const T* __restrict__ x = static_cast<const T*>(p.logits) + row * p.ld;
  const SfFilter filter(p, row);
  SfRange range{-INFINITY, 0.f, 0.f};
  int bad = filter.good() ? 0 : 1;
  for (int c = threadIdx.x; c < p.classes; c += 1024) {
    const float v = static_cast<float>(x[c]);
    bad |= v < INFINITY ? 0 : 1;
    range.top = fmaxf(range.top, v);
  }
  if (threadIdx.x == 0) first = 0x7fffffff;
  bad = __syncthreads_or(bad);
  range = sf_range<16>(range, red);
  if (bad != 0 || range.top == -INFINITY) {
    if (threadIdx.x == 0) sf_no_distribution(p, row);
    return;
  }
  if (!filter.greedy()) return sf_general<T, 1024>(p, row, filter, range.top, sh);
  for (int c = threadIdx.x; c < p.classes; c += 1024)
    if (static_cast<float>(x[c]) == range.top) {
      atomicMin(&first, c);
      break;
    }
  __syncthreads();
  if (threadIdx.x == 0) p.targets[row] = first;
}

template <typename T>
static void sf_launch(const SfParams& p, int64_t rows, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const dim3 grid(static_cast<unsigned>(rows));
  if (p.classes <= 2048) hipLaunchKernelGGL((sf_row_kernel<T, 256, 1, false>), grid, dim3(256), 0, s, p);
  else if (p.classes / E <= kSfMostSteps * 1024) hipLaunchKernelGGL((sf_row_kernel<T, 1024, 1, false>), grid, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL(sf_long_kernel<T>, grid, dim3(1024), 0, s, p);
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
  const int shift = 62 - bits < 52 ? 62 - bits : 52;
  const SfParams p{logits, u, temperatures, top_ks, top_ps, min_ps, targets, invalid, ld, temperature, top_p, min_p, top_k,
                   static_cast<int>(classes), u_is_double, shift};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto type) {
    sf_launch<typename decltype(type)::type>(p, rows, s);
    return check_launch();
  });
}
