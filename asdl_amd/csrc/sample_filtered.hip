// One draw per row from softmax(logits / T) restricted by top-k, top-p and min-p, with one uniform number u per row.
// Classes are ordered by logit, the lowest index first among equals; with weights w = exp((x - max x) / T):
//   top-k  keeps the first k;  top-p  keeps a class while the weight in front of it is below p times the weight of what top-k kept;
//   min-p  keeps w >= min_p;   the draw is the first class, by index, at which the kept weight up to there exceeds u times all of it.
// A border between two classes is where a sum over up to all classes passes a number, so sums have to be the same whatever order
// they are formed in: a weight is an integer, w 2^s rounded, with s so large that the sum over all classes fits 63 bits (46 bits below
// the point for 50257 classes), and integers add exactly.  w itself is computed in double.
// The kept classes are those above a key (the logit's bits in an order that integers keep) and the first few equal to it: the key is
// found digit by digit from histograms of counts or weights.
#include "elements.hpp"

namespace ak {

typedef unsigned long long u64;

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

struct SfWeight {
  double top, inv_t, scale;
  __device__ __forceinline__ double real(float x) const { return x == -INFINITY ? 0. : exp((static_cast<double>(x) - top) * inv_t); }
  __device__ __forceinline__ u64 operator()(float x) const { return static_cast<u64>(real(x) * scale + 0.5); }
};

struct SfShared {
  u64 mass[256];
  uint32_t count[256];
  u64 red[16];
  int red_int[16];
  float red_float[16];
  u64 above;
  uint32_t digit, ties;
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

template <typename T, int NT>
static __global__ __launch_bounds__(NT) void sf_kernel(SfParams p) {
  constexpr int WAVES = NT / 64;
  __shared__ SfShared sh;
  __shared__ u64 bins[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.classes;
  const int64_t row = blockIdx.x;
  const T* __restrict__ x = static_cast<const T*>(p.logits) + row * p.ld;
  const double t = p.temperatures != nullptr ? static_cast<double>(p.temperatures[row]) : p.temperature;
  const double top_p = p.top_ps != nullptr ? static_cast<double>(p.top_ps[row]) : p.top_p;
  const double min_p = p.min_ps != nullptr ? static_cast<double>(p.min_ps[row]) : p.min_p;
  int64_t k = p.top_ks != nullptr ? p.top_ks[row] : p.top_k;
  if (t == 0.) k = 1;
  const double u = p.u_double ? static_cast<const double*>(p.u)[row] : static_cast<double>(static_cast<const float*>(p.u)[row]);

  float top = -INFINITY;
  int bad = t >= 0. && top_p == top_p && min_p == min_p && u == u ? 0 : 1;
  for (int c = tid; c < n; c += NT) {
    const float v = static_cast<float>(x[c]);
    bad |= v < INFINITY ? 0 : 1;
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) sh.red_float[wave] = top;
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sh.red_float[w]);
  if (bad != 0 || top == -INFINITY) {       // no distribution, or no number to draw with
    if (tid == 0) {
      p.targets[row] = -1;
      if (p.invalid != nullptr) *p.invalid = 1;
    }
    return;
  }
  SfWeight weight{static_cast<double>(top), t == 0. ? 1. : 1. / t, static_cast<double>(1ull << p.shift)};

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
  if (top_p < 1. && k != 1) {
    u64 all = 0;
    for (int c = tid; c < n; c += NT) {
      const float v = static_cast<float>(x[c]);
      if (in_k(sf_key(v))) all += weight(v);
    }
    all = group_sum<WAVES>(all, sh.red);
    if (ties != 0xffffffffu) all += ties * weight(sf_value(key));
    // in front of a class less than p all: of integers, less than that rounded up
    const double border = top_p > 0. ? ceil(top_p * static_cast<double>(all)) : 0.;
    u64 target = border < 1. ? 1 : static_cast<u64>(border);
    if (target > all) target = all;
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
    if (min_p > 0. && v != top && weight.real(v) < min_p) return 0;
    return weight(v);
  };
  u64 all = 0;
  for (int c = tid; c < n; c += NT) all += kept(c);
  all = group_sum<WAVES>(all, sh.red);
  const double border = u > 0. ? u * static_cast<double>(all) : 0.;
  u64 target = border >= static_cast<double>(all) ? all - 1 : static_cast<u64>(border);
  if (target >= all) target = all - 1;
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
    using T = typename decltype(type)::type;
    if (classes <= 2048) hipLaunchKernelGGL((sf_kernel<T, 256>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((sf_kernel<T, 1024>), dim3(static_cast<unsigned>(rows)), dim3(1024), 0, s, p);
    return check_launch();
  });
}
