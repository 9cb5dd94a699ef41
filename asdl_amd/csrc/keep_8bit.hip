// Activations kept in 8 bits between the passes, and what the backward pass makes of them.
// A block of 128 features of a row shares a power of two: e is the least integer with max |x| 2^-e <= 448, clamped to -127 .. 127, and a
// value is kept as the nearest e4m3 number (4 bits of exponent, 3 of fraction, ties to even) of x 2^-e, which stands for code 2^e.  Scaling by a
// power of two rounds nothing, and a floating code loses no accuracy by it: the largest code of a block is above 224, so normal codes (from
// 2^-6 on, off by at most 2^-4 of themselves) reach down to 2^-13.8 of its largest value, to 2^-14.8 at best; what is smaller is off by at
// most 2^(e - 10).  Infinities and NaN are kept as NaN and do not count for e; what would be rounded to 2^128 is kept as 1.875 2^127.
//   gelu:    y = x P(x) and the kept x in one pass;  dx = g (P(x') + x' P'(x')) with the kept x', P the normal distribution or its
//            approximation by tanh
//   linear:  dw = g^T x',  db = sum g.  x' is a bfloat16 number exactly, so the products are exact and their sums fp32: g in
//            bfloat16 as it is, in fp16 and fp32 as two and three bfloat16 pieces that add up to it exactly
// The elementwise passes are bound by the memory (gelu of 8192 x 4096 bf16 36 us each way, 4.7 TB/s), the products by the matrix cores (16384
// rows of 4096 to 4096 bf16 400 to 435 us, 1.3 PFLOP/s at the power limit; of 768 to 2304 from 8192 rows 39 us, too few tiles).
#include <algorithm>
#include "column_sums.hpp"
#include "half_product.hpp"

namespace ak {

constexpr int kKeepBlock = 128, kKeepLanes = 16, kKeepEach = 8;      // a block is 16 lanes of 8 elements
constexpr float kKeepLargest = 448.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true)));
}
// The largest over 16 neighbouring lanes, in each of them (the moves of lanes_sum()).
__device__ __forceinline__ uint32_t lanes16_max(uint32_t v) {
  v = max_dpp<0xB1>(v);
  v = max_dpp<0x4E>(v);
  v = max_dpp<0x141>(v);
  return max_dpp<0x140>(v);
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

constexpr uint32_t kInfinityBits = 0x7f800000u;

__device__ __forceinline__ int keep_exponent(float most) {
  if (most == 0.f) return -127;
  const int e = __builtin_amdgcn_frexp_expf(most) - 1;                       // most = m 2^e, 1 <= m < 2
  const float m = 2.f * __builtin_amdgcn_frexp_mantf(most);
  return max(-127, min(127, e - 8 + (m > kKeepLargest / 256.f ? 1 : 0)));
}

// The exponent of a block whose lanes have x each, and the codes of x.  The largest magnitude is the largest pattern of bits; infinities and
// NaN, and e = 120, which is that of values from 1.75 2^127 on, the largest of which would be rounded to 2^128 (they are kept as
// 240 2^120), are seen to where a block has them.
__device__ __forceinline__ u32x2 keep_codes(float (&x)[kKeepEach], int& exponent) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < kKeepEach; ++e) most = max(most, magnitude_bits(x[e]));
  most = lanes16_max(most);
  float v[kKeepEach];
  if (most >= kInfinityBits) {
    most = 0;
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) most = max(most, magnitude_bits(x[e]) < kInfinityBits ? magnitude_bits(x[e]) : 0u);
    most = lanes16_max(most);
  }
  exponent = keep_exponent(__builtin_bit_cast(float, most));
  const float scale = ldexpf(1.f, -exponent);
#pragma unroll
  for (int e = 0; e < kKeepEach; ++e) v[e] = x[e] * scale;
  if (exponent >= 120) {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) v[e] = fabsf(v[e]) > 240.f ? copysignf(240.f, v[e]) : v[e];
  }
  u32x2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], w, true);
    o[h] = static_cast<uint32_t>(w);
  }
#pragma unroll
  for (int e = 0; e < kKeepEach; ++e)
    if (magnitude_bits(x[e]) >= kInfinityBits) o[e >> 2] |= 0x7fu << 8 * (e & 3);
  return o;
}

__device__ __forceinline__ void keep_values(u32x2 codes, int e, float (&x)[kKeepEach]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float scale = ldexpf(1.f, e);            // (2^-127 is a number, too: products with it are exact)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[h]), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[h]), true);
    x[4 * h] = lo[0] * scale;
    x[4 * h + 1] = lo[1] * scale;
    x[4 * h + 2] = hi[0] * scale;
    x[4 * h + 3] = hi[1] * scale;
  }
}

enum { kGeluExact = 0, kGeluTanh = 1 };

// P(x), and with SLOPE P'(x).
// Exact: P(-|x|) = exp(-x^2 / 2) t q(t), t = 1 / (1 + 0.3 |x|), with a polynomial fitted to half the scaled complementary error
// function of |x| / sqrt(2) over t = 1 ... 1 / 5.2 at least relative error (1.5e-7; its steps in fp32 4.5e-7).  The
// exponential is that of P'; its rounded argument is off by up to 1.5 x^2 2^-24, and the tail by as much of itself (measured 2.6e-6 at |x| = 4 to 8,
// 7.8e-6 at 8 to 13; next to P = 1 nothing of it is seen).  (The library's erfc: gelu of 8192 x 4096 bf16 56 us each way, which is the
// arithmetic's time.)
template <int KIND, bool SLOPE>
__device__ __forceinline__ void gelu_share(float x, float& below, float& slope) {
  if constexpr (KIND == kGeluExact) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, fabsf(x), 1.f));
    const float bell = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
    constexpr float q[8] = {0.11962930113077164f, 0.12075396627187729f,  0.09991341084241867f,  0.12856192886829376f,
                            -0.05368424206972122f, 0.20635418593883514f, -0.15720349550247192f, 0.03567487746477127f};
    float v = q[7];
#pragma unroll
    for (int k = 6; k >= 0; --k) v = __builtin_fmaf(v, t, q[k]);
    v *= t * bell;
    below = x < 0.f ? v : 1.f - v;
    if constexpr (SLOPE) slope = 0.39894228040143268f * bell;
  } else {
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
    // (beyond 20 the share is 0 or 1; the cube of a large number is no float32.  A NaN stays.)
    x = fabsf(x) > 20.f ? copysignf(20.f, x) : x;
    const float x2 = x * x;
    const float e = __builtin_amdgcn_exp2f(x * -2.3022081984803314f * __builtin_fmaf(0.044715f, x2, 1.f));       // exp(-2 u)
    below = __builtin_amdgcn_rcpf(1.f + e);
    // P (1 - P) = P e P; e is infinite where P is 0
    if constexpr (SLOPE) slope = e < INFINITY ? below * (e * below) * 1.5957691216057308f * __builtin_fmaf(0.134145f, x2, 1.f) : 0.f;
  }
}

struct Keep {
  const void* x;           // the activations, or the gradient of the result on the way back
  void* y;                 // the result, or the gradient of the activations
  uint8_t* codes;          // [rows][F]
  int8_t* exponents;       // [rows][blocks]
  int64_t ldx, rows;
  int F, blocks;
};

// The elements of a lane: eight, fewer at the end of a row.  A work group has 16 blocks, one after the other over the rows.
struct KeepPlace {
  int64_t row, block;
  int c, count;
  __device__ __forceinline__ explicit KeepPlace(const Keep& p) {
    const uint32_t b = static_cast<uint32_t>(p.blocks);
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (256 / kKeepLanes), row0 = first / b;      // (the same for all lanes)
    const uint32_t at = static_cast<uint32_t>(first - row0 * b) + threadIdx.x / kKeepLanes, down = at / b;
    row = static_cast<int64_t>(row0 + down);
    block = at - down * b;
    c = static_cast<int>(block) * kKeepBlock + static_cast<int>(threadIdx.x % kKeepLanes) * kKeepEach;
    count = row < p.rows ? min(max(p.F - c, 0), kKeepEach) : 0;
  }
};

template <typename T>
__device__ __forceinline__ void keep_load(const T* __restrict__ p, int count, float (&x)[kKeepEach]) {
  if (count == kKeepEach) {
    Some<T, kKeepEach> v;
    v.load(p);
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) x[e] = v.get(e);
  } else {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) x[e] = e < count ? static_cast<float>(p[e]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void keep_store(T* __restrict__ p, int count, const float (&x)[kKeepEach]) {
  if (count == kKeepEach) {
    Some<T, kKeepEach> v;
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) v.set(e, x[e]);
    v.store(p);
  } else {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e)
      if (e < count) p[e] = static_cast<T>(x[e]);
  }
}

// KIND -1: the kept values alone
template <typename T, int KIND>
static __global__ __launch_bounds__(256) void keep_kernel(Keep p) {
  const KeepPlace at(p);
  float x[kKeepEach];
  keep_load(static_cast<const T*>(p.x) + at.row * p.ldx + at.c, at.count, x);
  int exponent;
  const u32x2 codes = keep_codes(x, exponent);
  if (at.count == 0) return;
  uint8_t* __restrict__ to = p.codes + at.row * p.F + at.c;
  if (at.count == kKeepEach) {
    __builtin_memcpy(to, &codes, 8);
  } else {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e)
      if (e < at.count) to[e] = static_cast<uint8_t>(codes[e >> 2] >> 8 * (e & 3));
  }
  if (threadIdx.x % kKeepLanes == 0) p.exponents[at.row * p.blocks + at.block] = static_cast<int8_t>(exponent);
  if constexpr (KIND >= 0) {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) {
      float below, slope;
      gelu_share<KIND, false>(x[e], below, slope);
      x[e] = x[e] * below;
    }
    keep_store(static_cast<T*>(p.y) + at.row * p.F + at.c, at.count, x);
  }
}

__device__ __forceinline__ u32x2 keep_fetch(const uint8_t* __restrict__ from, int count) {
  u32x2 codes = {0, 0};
  if (count == kKeepEach) {
    __builtin_memcpy(&codes, from, 8);
  } else {
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e)
      if (e < count) codes[e >> 2] |= static_cast<uint32_t>(from[e]) << 8 * (e & 3);
  }
  return codes;
}

// KIND -1: y = the kept values (pitch ldy, zeros up to it); else y = x (P + x' P')
template <typename T, int KIND>
__device__ __forceinline__ void keep_back(const Keep& p, int64_t ldy, int padded) {
  const KeepPlace at(p);
  if (at.row >= p.rows) return;
  float x[kKeepEach] = {};
  if (at.count > 0) {
    const int exponent = p.exponents[at.row * p.blocks + at.block];
    keep_values(keep_fetch(p.codes + at.row * p.F + at.c, at.count), exponent, x);
  }
  if constexpr (KIND >= 0) {
    if (at.count == 0) return;
    float g[kKeepEach];
    keep_load(static_cast<const T*>(p.x) + at.row * p.ldx + at.c, at.count, g);
#pragma unroll
    for (int e = 0; e < kKeepEach; ++e) {
      float below, slope;
      gelu_share<KIND, true>(x[e], below, slope);
      x[e] = g[e] * (below + x[e] * slope);
    }
    keep_store(static_cast<T*>(p.y) + at.row * ldy + at.c, at.count, x);
  } else {
    const int count = min(max(padded - at.c, 0), kKeepEach);
    if (count > 0) keep_store(static_cast<T*>(p.y) + at.row * ldy + at.c, count, x);
  }
}

template <typename T, int KIND>
static __global__ __launch_bounds__(256) void keep_back_kernel(Keep p, int64_t ldy, int padded) {
  keep_back<T, KIND>(p, ldy, padded);
}

// What a weight gradient's product needs: the kept values as bfloat16, and the chunks of g's column sums, by work groups behind them.
// (This and the totals in one launch, where each had its own: the bias's gradient of 2304 outputs from 8192 rows 10.5 -> 1.7 us.)
template <typename T>
static __global__ __launch_bounds__(256) void keep_prepare_kernel(Keep p, int64_t ldx, uint32_t front, const T* __restrict__ g, int64_t ldg, int64_t rows,
                                                                  int64_t cols, int64_t rows_per_chunk, float* __restrict__ part) {
  __shared__ float joined[8][kColumnsPerGroup];
  if (blockIdx.x < front) return keep_back<__bf16, -1>(p, ldx, static_cast<int>(ldx));
  const uint32_t at = blockIdx.x - front, groups = static_cast<uint32_t>((cols + kColumnsPerGroup - 1) / kColumnsPerGroup);
  column_chunk(g, ldg, rows, cols, rows_per_chunk, part, at % groups, at / groups, joined);
}

// The totals of the splits' sums and, by work groups behind them, of the columns' chunks.
template <typename O>
static __global__ __launch_bounds__(256) void keep_totals_kernel(const float* __restrict__ sum, int64_t ld, int64_t stride, int splits, int64_t rows,
                                                                 int cols, O* __restrict__ dw, uint32_t front, const float* __restrict__ part, int chunks,
                                                                 O* __restrict__ db) {
  if (blockIdx.x < front) hp_total_part(sum, ld, stride, splits, rows, cols, 1.f, nullptr, dw, blockIdx.x, front);
  else column_total(part, rows, chunks, 1.f, nullptr, db, blockIdx.x - front);
}

// ---- host side
struct KeepPlan {
  int pieces, splits;
  int64_t ldf, ldg, ld_sum;
};

inline KeepPlan keep_plan(int dtype, int64_t rows, int64_t F, int64_t out) {
  KeepPlan p;
  p.pieces = dtype == AK_BF16 ? 1 : dtype == AK_F16 ? 2 : 3;
  p.ldf = align_up(F, 8);
  p.ldg = align_up(out, 8);
  p.ld_sum = align_up(F, 4);
  p.splits = 1;
  if (F == 0) return p;          // (sums of columns alone)
  if (hp_wide(F, out)) return p;          // (129 tiles of 256 and more: two splits of them would not run at once)
  const int64_t tiles = ((F + 127) / 128) * ((out + 127) / 128);
  const int64_t s = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / tiles, rows / 256), 64));
  const int64_t per = align_up((rows + s - 1) / s, 32);
  p.splits = static_cast<int>((rows + per - 1) / per);
  return p;
}

struct KeepSpace {
  __bf16 *x, *g;
  float *sum, *columns;
  size_t bytes;
};

inline KeepSpace keep_space(const KeepPlan& p, int64_t rows, int64_t out, bool weight, bool copy, bool bias, void* ws) {
  Carver c{static_cast<unsigned char*>(ws)};
  KeepSpace s = {};
  if (weight) s.x = c.take<__bf16>(rows * p.ldf);
  if (weight && copy) s.g = c.take<__bf16>(p.pieces * rows * p.ldg);
  if (weight && p.splits > 1) s.sum = c.take<float>(p.splits * out * p.ld_sum);
  if (bias) s.columns = c.take<float>(static_cast<int64_t>(column_sums_ws_bytes(rows, out) / sizeof(float)));
  s.bytes = c.used;
  return s;
}

inline int keep_check(int dtype, int64_t ld, int64_t rows, int64_t F) {
  if (!is_element_type(dtype) || rows < 0 || F <= 0 || ld < F) return AK_ERR_ARG;
  if (F > (1ll << 24) || rows > (1ll << 31) || rows * ((F + kKeepBlock - 1) / kKeepBlock) > (1ll << 34)) return AK_ERR_TOO_LARGE;
  return AK_OK;
}

inline dim3 keep_grid(const Keep& p) {
  return dim3(static_cast<unsigned>((p.rows * p.blocks + 256 / kKeepLanes - 1) / (256 / kKeepLanes)));
}

// launch(a piece of the rows) for all of them, in pieces of 2^27 blocks, 2^31 threads; x and y: bytes of an element, ldy: pitch of y.
// The last piece is left to the caller.
template <typename F>
inline Keep keep_pieces(Keep p, int64_t x, int64_t y, int64_t ldy, F&& launch) {
  const int64_t most = (1ll << 27) / p.blocks;             // (at most 2^17 blocks a row)
  while (p.rows > most) {
    Keep piece = p;
    piece.rows = most;
    launch(piece);
    if (p.x != nullptr) p.x = static_cast<const char*>(p.x) + most * p.ldx * x;
    if (p.y != nullptr) p.y = static_cast<char*>(p.y) + most * ldy * y;
    p.codes += most * p.F;
    p.exponents += most * p.blocks;
    p.rows -= most;
  }
  return p;
}

}  // namespace ak

extern "C" int ak_quantize_8bit(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t width, int gelu, void* y, uint8_t* codes, int8_t* exponents,
                                ak_stream_t stream) {
  using namespace ak;
  const int rc = keep_check(dtype, ldx, rows, width);
  if (rc != AK_OK) return rc;
  if (gelu < -1 || gelu > kGeluTanh) return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (x == nullptr || codes == nullptr || exponents == nullptr || (gelu >= 0 && y == nullptr)) return AK_ERR_ARG;
  const Keep p{x, y, codes, exponents, ldx, rows, static_cast<int>(width), static_cast<int>((width + kKeepBlock - 1) / kKeepBlock)};
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](const Keep& q) {
      if (gelu == kGeluExact) hipLaunchKernelGGL((keep_kernel<T, kGeluExact>), keep_grid(q), dim3(256), 0, s, q);
      else if (gelu == kGeluTanh) hipLaunchKernelGGL((keep_kernel<T, kGeluTanh>), keep_grid(q), dim3(256), 0, s, q);
      else hipLaunchKernelGGL((keep_kernel<T, -1>), keep_grid(q), dim3(256), 0, s, q);
    };
    launch(keep_pieces(p, sizeof(T), sizeof(T), width, launch));
    return check_launch();
  });
}

extern "C" int ak_dequantize_8bit(const uint8_t* codes, const int8_t* exponents, int64_t rows, int64_t width, int gelu, const void* g, int64_t ldg,
                                  void* y, int dtype, ak_stream_t stream) {
  using namespace ak;
  const int rc = keep_check(dtype, gelu >= 0 ? ldg : width, rows, width);
  if (rc != AK_OK) return rc;
  if (gelu < -1 || gelu > kGeluTanh) return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (codes == nullptr || exponents == nullptr || y == nullptr || (gelu >= 0 && g == nullptr)) return AK_ERR_ARG;
  const int F = static_cast<int>(width);
  const Keep p{g, y, const_cast<uint8_t*>(codes), const_cast<int8_t*>(exponents), ldg, rows, F, (F + kKeepBlock - 1) / kKeepBlock};
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](const Keep& q) {
      if (gelu == kGeluExact) hipLaunchKernelGGL((keep_back_kernel<T, kGeluExact>), keep_grid(q), dim3(256), 0, s, q, width, F);
      else if (gelu == kGeluTanh) hipLaunchKernelGGL((keep_back_kernel<T, kGeluTanh>), keep_grid(q), dim3(256), 0, s, q, width, F);
      else hipLaunchKernelGGL((keep_back_kernel<T, -1>), keep_grid(q), dim3(256), 0, s, q, width, F);
    };
    launch(keep_pieces(p, sizeof(T), sizeof(T), width, launch));
    return check_launch();
  });
}

extern "C" size_t ak_weight_grad_8bit_ws_bytes(int dtype, int64_t rows, int64_t width, int64_t out) {
  if (!ak::is_element_type(dtype) || rows <= 0 || width < 0 || out <= 0 || rows > (1ll << 30) || width > (1 << 20) || out > (1 << 20)) return 0;
  return ak::keep_space(ak::keep_plan(dtype, rows, width, out), rows, out, width > 0, true, true, nullptr).bytes;
}

extern "C" size_t ak_weight_grad_8bit_ws_bytes_of(const void* g, int dtype, int64_t ldg, int64_t rows, int64_t width, int64_t out, int gradients) {
  if (ak_weight_grad_8bit_ws_bytes(dtype, rows, width, out) == 0) return 0;
  return ak::keep_space(ak::keep_plan(dtype, rows, width, out), rows, out, (gradients & 1) != 0, dtype != AK_BF16 || !ak::hp_aligned(g, ldg, out),
                        (gradients & 2) != 0, nullptr).bytes;
}

extern "C" int ak_weight_grad_8bit(const void* g, int dtype, int64_t ldg, const uint8_t* codes, const int8_t* exponents, int64_t rows, int64_t width,
                                   int64_t out, void* dw, void* db, int grad_dtype, void* ws, size_t ws_bytes, ak_stream_t stream) {
  using namespace ak;
  int rc = keep_check(dtype, ldg, rows, out);
  if (rc != AK_OK) return rc;
  if (!is_element_type(grad_dtype) || width < 0 || (dw != nullptr && width == 0) || rows == 0) return AK_ERR_ARG;
  if (rows > (1ll << 30) || width > (1 << 20) || out > (1 << 20) || ldg > (1ll << 24)) return AK_ERR_TOO_LARGE;
  if (dw == nullptr && db == nullptr) return AK_OK;
  if (g == nullptr || (dw != nullptr && (codes == nullptr || exponents == nullptr))) return AK_ERR_ARG;
  const KeepPlan plan = keep_plan(dtype, rows, width, out);
  const bool copy = dtype != AK_BF16 || !hp_aligned(g, ldg, out);
  const KeepSpace s = keep_space(plan, rows, out, dw != nullptr, copy, db != nullptr, ws);
  if (ws == nullptr || ws_bytes < s.bytes) return AK_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int F = static_cast<int>(width), chunks = column_chunks(rows);
  if (dw == nullptr)
    return with_type(grad_dtype, [&](auto o) {
      using O = typename decltype(o)::type;
      return with_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        return column_sums(static_cast<const T*>(g), ldg, rows, out, 1.f, nullptr, static_cast<O*>(db), s.columns, st);
      });
    });
  const Keep all{nullptr, s.x, const_cast<uint8_t*>(codes), const_cast<int8_t*>(exponents), 0, rows, F, (F + kKeepBlock - 1) / kKeepBlock};
  const Keep k = keep_pieces(all, 0, sizeof(__bf16), plan.ldf, [&](const Keep& q) {
    hipLaunchKernelGGL((keep_back_kernel<__bf16, -1>), keep_grid(q), dim3(256), 0, st, q, plan.ldf, static_cast<int>(plan.ldf));
  });
  const unsigned front = keep_grid(k).x;
  const int64_t behind = db != nullptr ? chunks * ((out + kColumnsPerGroup - 1) / kColumnsPerGroup) : 0;         // (at most 2^18: fits the launch)
  with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    hipLaunchKernelGGL(keep_prepare_kernel<T>, dim3(front + static_cast<unsigned>(behind)), dim3(256), 0, st, k, plan.ldf, front, static_cast<const T*>(g), ldg,
                       rows, out, (rows + chunks - 1) / chunks, s.columns);
    return AK_OK;
  });
  const __bf16* from = static_cast<const __bf16*>(g);
  int64_t ld = ldg;
  rc = check_launch();
  if (rc == AK_OK && copy) {
    rc = dtype == AK_BF16  ? hp_pad(from, ldg, rows, out, s.g, plan.ldg, st)
         : dtype == AK_F16 ? hp_pieces<2>(static_cast<const _Float16*>(g), ldg, rows, out, s.g, plan.ldg, st)
                           : hp_pieces<3>(static_cast<const float*>(g), ldg, rows, out, s.g, plan.ldg, st);
    from = s.g;
    ld = plan.pieces * plan.ldg;
  }
  if (rc != AK_OK) return rc;
  return with_type(grad_dtype, [&](auto o) {
    using O = typename decltype(o)::type;
    // i features, j outputs, k rows
    auto products = [&](auto cfg) {
      using Cfg = decltype(cfg);
      HpProblem q = hp_problem<Cfg>(hp_operand(s.x, plan.ldf, rows, width, false), hp_operand(from, ld, rows, out, false), width, out, rows, plan.splits);
      if (Cfg::PIECES) q.pieces = hp_pieces_of_b(plan.pieces, plan.ldg);
      if constexpr (Cfg::BI == 128)
        if (plan.splits > 1) return hp_launch<Cfg, __bf16, HpSum>(q, HpSum::Params{s.sum, plan.ld_sum, out * plan.ld_sum, F, static_cast<int>(out), 1}, st);
      return hp_launch<Cfg, __bf16, HpStore<O>>(q, typename HpStore<O>::Params{static_cast<O*>(dw), width, F, static_cast<int>(out), 1.f, nullptr}, st);
    };
    auto of_form = [&](auto pieces) {
      constexpr bool P = decltype(pieces)::value;
      return hp_wide(width, out) ? products(HpWide<false, false, P>{}) : products(HpSmall<false, false, P>{});
    };
    const int done = plan.pieces > 1 ? of_form(std::true_type{}) : of_form(std::false_type{});
    const unsigned sums = plan.splits > 1 ? hp_total_groups(out, plan.ld_sum) : 0, groups = sums + (db != nullptr ? static_cast<unsigned>((out + 255) / 256) : 0);
    if (done != AK_OK || groups == 0) return done;
    hipLaunchKernelGGL(keep_totals_kernel<O>, dim3(groups), dim3(256), 0, st, s.sum, plan.ld_sum, out * plan.ld_sum, plan.splits, out, F, static_cast<O*>(dw),
                       sums, s.columns, chunks, static_cast<O*>(db));
    return check_launch();
  });
}
