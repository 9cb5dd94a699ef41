// Softmax cross entropy of a linear layer, in pieces of the classes, without its logits:
//   s = h w^T + b,  lse_n = log sum_v exp s_nv,  loss_n = lse_n - s_n,t(n)  (0 for an ignored row)
//   back, with c_n the gradient of loss_n (0 for an ignored row):
//   d_nv = c_n (exp(s_nv - lse_n) - [v = t(n)]),  dh = d w,  dw = d^T h,  db_v = sum_n d_nv
// Forward, the product's tiles leave the largest logit and the sum of exponentials of their classes for each row, and the target's
// logit; a second launch joins them.  Backward, the logits of a piece of the classes are formed again (2 N V D operations more than
// with kept logits, which would be written, read and written again: 1.6 GB in fp32 for 8192 rows of 50257 classes), and become the piece
// of d in their tile's epilogue; both gradients are products with it.
// 16-bit operands: fp32 sums.  d is rounded to the operands' type, which the matrix cores need and which is what a framework's own
// backward pass in that type has; it holds c_n over the largest |c_n| (fp16: times 2^14, so that shares of the classes down to
// 2^-28 are normal numbers), and the products' epilogues put that factor back: where all c_n are alike, the target's entry of a row that is
// far from sure, -1 + exp(..), is rounded by next to nothing, where a power of two in its place would round all of these alike by up to 2^-9
// (error of dh of 8192 x 768 x 50257, bf16: 0.0030 -> 0.0018 of its size).
// fp32 operands: three bf16 pieces each, six of their products a product (half_product.hpp), through the same tiles; d in three pieces, too.
// Bound by the matrix cores at the device's power limit where rows are many (both ways, on several cards: 8192 x 768 x 50257 bf16 2.5 to
// 2.65 ms, 1.0 PFLOP/s of the four products; 4096 x 2048 x 128000 fp16 7.4 to 8.1 ms, 1.1 PFLOP/s), by the memory where they are few
// (4 rows of 50257 x 768, forward alone: 21 us, 3.7 TB/s).
#include <algorithm>
#include "column_sums.hpp"
#include "half_product.hpp"

namespace ak {

// What the matrix cores take of an operand type: the element and how many of them a value is.
template <typename E>
struct LceKind {
  using type = E;
  static constexpr int pieces = 1;
};
template <>
struct LceKind<float> {
  using type = __bf16;
  static constexpr int pieces = 3;
};

enum { kLossNone = 0, kLossSum = 1, kLossMean = 2 };

typedef float floatx2 __attribute__((ext_vector_type(2)));

// (largest, sum of exp(s - largest)) of two sets of classes together; -inf and 0 of an empty one.
__device__ __forceinline__ floatx2 lce_join2(floatx2 a, floatx2 b) {
  const float m = fmaxf(a[0], b[0]);
  // (m is -inf where nothing is there; a NaN is in the sums)
  const float base = m == -INFINITY ? 0.f : m;
  return floatx2{m, a[1] * __expf(a[0] - base) + b[1] * __expf(b[0] - base)};
}

struct LceRows {
  const int64_t* targets;
  const float* bias;       // fp32, or null
  int64_t ignore;
  int rows, classes;
};

constexpr float kLog2e = 1.44269504088896340736f;

// exp(s - shift) = exp(s) * rest, a fused multiplication and addition and the power of two an element: the product of the shift is rounded
// to float32 (2^-24 of a shift of 60 is 4e-6), and what that loses, exact by a fused operation, is a factor that all elements share.
// From 2^20 on (all classes of a tile masked by a type's lowest value, -1e10, -1e30) that factor would be no number or the product
// infinite: the difference itself goes into the power there.  That is one more operation an element, for waves that have such a row;
// the other rows of theirs subtract 0, so that their bits are the same beside it.
struct Shifted {
  float from, by, rest;
  __device__ __forceinline__ explicit Shifted(float shift) {
    const bool near = fabsf(shift) < 0x1p20f;           // (neither infinite nor NaN)
    from = near ? 0.f : shift;
    by = near ? shift * kLog2e : 0.f;
    rest = near ? __builtin_amdgcn_exp2f(-__builtin_fmaf(shift, kLog2e, -by)) : 1.f;
  }
  __device__ __forceinline__ bool far() const { return __any(from != 0.f); }
  template <bool FAR>
  __device__ __forceinline__ float exp(float s) const {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(FAR ? s - from : s, kLog2e, -by));
  }
};

// What a tile's sums become: the bias is added, and classes behind the last are -inf.  Most tiles have neither.  (c0: first class of the
// product, i_tile: first one of the tile behind it)
template <class Cfg>
__device__ __forceinline__ void lce_scores(const LceRows& r, floatx16 (&acc)[Cfg::FR][Cfg::FC], int i_tile, int c0, int wr) {
  const int first = c0 + i_tile;
  if (r.bias == nullptr && first + Cfg::BI <= r.classes) return;
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int c = first + 32 * (Cfg::FR * wr + a) + 8 * (x >> 2) + 4 * g + (x & 3);
      const float shift = r.bias != nullptr && c < r.classes ? r.bias[c] : 0.f;
#pragma unroll
      for (int b = 0; b < Cfg::FC; ++b) acc[a][b][x] = c < r.classes ? acc[a][b][x] + shift : -INFINITY;
    }
}

// Tiles of the forward pass: i classes, j rows.
struct LceStats {
  struct Params {
    LceRows r;
    floatx2* part;         // [tile of classes][rows]
    float* at_target;      // [rows]
  };
  template <class Cfg>
  static __device__ __forceinline__ void run(const Params& e, floatx16 (&acc)[Cfg::FR][Cfg::FC], int ti, int tj, int, int wr, int wc,
                                             AK_LDS unsigned char* lds) {
    AK_LDS floatx2* joined = reinterpret_cast<AK_LDS floatx2*>(lds);       // [WR][BJ]
    const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
    const int i0 = ti * Cfg::BI + 32 * Cfg::FR * wr + 4 * g;
    __syncthreads();                           // everybody has read the last panels
    lce_scores<Cfg>(e.r, acc, ti * Cfg::BI, 0, wr);
#pragma unroll
    for (int b = 0; b < Cfg::FC; ++b) {
      const int jl = 32 * Cfg::FC * wc + 32 * b + l32, j = tj * Cfg::BJ + jl;
      const int64_t target = j < e.r.rows ? e.r.targets[j] : -1;
      const int64_t at = target - i0;      // 32 a + 8 q + k where this lane has the target's logit
      float m = -INFINITY;
#pragma unroll
      for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
        for (int x = 0; x < 16; ++x) m = fmaxf(m, acc[a][b][x]);
      const Shifted by(m == -INFINITY ? 0.f : m);
      float s = 0.f;
      auto add = [&](auto far) {
#pragma unroll
        for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
          for (int x = 0; x < 16; ++x) s += by.exp<decltype(far)::value>(acc[a][b][x]);
      };
      if (by.far()) add(std::true_type{});
      else add(std::false_type{});
      s *= by.rest;
      if (__any(at >= 0 && at < 32 * Cfg::FR)) {
#pragma unroll
        for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (at == 32 * a + 8 * (x >> 2) + (x & 3) && target < e.r.classes) e.at_target[j] = acc[a][b][x];
      }
      floatx2 ms = {m, s};
      ms = lce_join2(ms, floatx2{__shfl_xor(m, 32), __shfl_xor(s, 32)});
      if (g == 0) joined[wr * Cfg::BJ + jl] = ms;
    }
    __syncthreads();
    for (int jl = threadIdx.x; jl < Cfg::BJ; jl += Cfg::THREADS) {
      const int j = tj * Cfg::BJ + jl;
      if (j >= e.r.rows) continue;
      floatx2 ms = joined[jl];
#pragma unroll
      for (int w = 1; w < Cfg::WR; ++w) ms = lce_join2(ms, joined[w * Cfg::BJ + jl]);
      e.part[static_cast<int64_t>(ti) * e.r.rows + j] = ms;
    }
  }
};

// Tiles of a piece of d: i classes from c0 on, j rows; d[j][i - c0], zeros up to a multiple of eight classes.
template <typename E>
struct LceGrad {
  using M = typename LceKind<E>::type;
  struct Params {
    LceRows r;
    const float* lse;
    const float* share;    // c_n over the largest, times 2^14 for fp16
    M* d;                  // a row: its pieces side by side
    int64_t ldd, pitch;    // elements between rows, between pieces
    int c0, width;         // classes of the piece, a multiple of eight (those from r.classes on are zeros)
  };
  template <class Cfg>
  static __device__ __forceinline__ void run(const Params& e, floatx16 (&acc)[Cfg::FR][Cfg::FC], int ti, int tj, int, int wr, int wc,
                                             AK_LDS unsigned char* lds) {
    lce_scores<Cfg>(e.r, acc, ti * Cfg::BI, e.c0, wr);
    const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
    const int i0 = ti * Cfg::BI + 32 * Cfg::FR * wr + 4 * g, j0 = tj * Cfg::BJ + 32 * Cfg::FC * wc + l32;
#pragma unroll
    for (int b = 0; b < Cfg::FC; ++b) {
      const int j = j0 + 32 * b;
      const bool in = j < e.r.rows;
      const float share = in ? e.share[j] : 0.f, lse = in ? e.lse[j] : 0.f;
      const Shifted by(lse);
      const float times = share * by.rest;
      const int64_t at = in && share != 0.f ? e.r.targets[j] - e.c0 - i0 : -1;
      // (ignored rows: 0, whatever their scores; the share of a class of no probability: 0)
      auto shares = [&](auto far) {
#pragma unroll
        for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[a][b][x] = share != 0.f ? by.exp<decltype(far)::value>(acc[a][b][x]) * times : 0.f;
      };
      if (by.far()) shares(std::true_type{});
      else shares(std::false_type{});
      if (__any(at >= 0 && at < 32 * Cfg::FR)) {
#pragma unroll
        for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (at == 32 * a + 8 * (x >> 2) + (x & 3)) acc[a][b][x] -= share;
      }
    }
    if constexpr (LceKind<E>::pieces == 1) {
      hp_store_rows<Cfg>(lds, ti, tj, wr, wc, [&](int a, int b, int x) { return acc[a][b][x]; }, e.d, e.ldd, e.width, e.r.rows);
    } else {
#pragma unroll
      for (int k = 0; k < LceKind<E>::pieces; ++k) {
        hp_eights<Cfg, M>(ti, tj, wr, wc, [&](int a, int b, int x) { return acc[a][b][x]; },
                          [&](int i, int j, u32x4 v) {
                            if (j < e.r.rows && i < e.width) __builtin_memcpy(e.d + static_cast<int64_t>(j) * e.ldd + k * e.pitch + i, &v, 16);
                          });
#pragma unroll
        for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
          for (int b = 0; b < Cfg::FC; ++b)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const float v = acc[a][b][x];
              acc[a][b][x] = fabsf(v) < INFINITY ? v - static_cast<float>(static_cast<M>(v)) : 0.f;
            }
      }
    }
  }
};

// Eight consecutive k of a row on their way to the matrix instruction 16 x 16 x 32.
template <typename E>
struct LceEight {
  E v[8];
  __device__ __forceinline__ void load(const E* p) { __builtin_memcpy(v, p, sizeof(v)); }
  // n of them, zeros behind: all eight loaded (the row's end, and the next row's beginning) unless that is behind the matrix
  __device__ __forceinline__ void some(const E* p, int n, const E* end) {
    if (n > 0 && end - p >= 8) {
      load(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? v[e] : static_cast<E>(0.f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : static_cast<E>(0.f);
    }
  }
};

// BELOW, float32: numbers below kHpLarge; the largest there are, to `most`.
template <bool BELOW, typename E>
__device__ __forceinline__ floatx4 lce_mma(const LceEight<E>& a, const LceEight<E>& b, floatx4 c, float& most) {
  if constexpr (__is_same(E, float)) {
    __bf16 pa[8][3], pb[8][3];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hp_split<3, BELOW>(a.v[e], pa[e]);
      hp_split<3, BELOW>(b.v[e], pb[e]);
      if constexpr (BELOW) most = fmaxf(most, fmaxf(fabsf(a.v[e]), fabsf(b.v[e])));
    }
    constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int t = 0; t < 6; ++t) {
      bf16x8 x, y;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = pa[e][A[t]];
        y[e] = pb[e][B[t]];
      }
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
    return c;
  } else if constexpr (__is_same(E, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// A few rows: a wave (and work group: the device is filled evenly) takes 16 classes, weights straight to the matrix instruction
// (16 x 16 x 32).  A lane has 32 consecutive k of every 128 of one class: what the four lanes of a class read at once is a part of each
// 128-byte line, all of it in four loads.  The order of k is the same for both operands.
template <typename E, int NB>
static __global__ __launch_bounds__(64) void lce_few_kernel(const E* __restrict__ h, int64_t ldh, const E* __restrict__ w, int64_t ldw, int D,
                                                             LceRows r, floatx2* __restrict__ part, float* __restrict__ at_target) {
  const int lane = threadIdx.x, quarter = lane >> 4, l16 = lane & 15;
  const int c0 = blockIdx.x * 16;
  const E* __restrict__ wr = w + static_cast<int64_t>(min(c0 + l16, r.classes - 1)) * ldw + 32 * quarter;
  const E* hr[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) hr[b] = h + static_cast<int64_t>(min(16 * b + l16, r.rows - 1)) * ldh + 32 * quarter;
  floatx4 acc[NB];
  float most = 0.f;
  auto products = [&](auto below) {
    constexpr bool BELOW = decltype(below)::value;
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int whole = D / 128 * 128;
    LceEight<E> wn[4];
    if (whole > 0)
#pragma unroll
      for (int e = 0; e < 4; ++e) wn[e].load(wr + 8 * e);
    for (int k = 0; k < whole; k += 128) {
      LceEight<E> wc[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) wc[e] = wn[e];
      if (k + 128 < whole)
#pragma unroll
        for (int e = 0; e < 4; ++e) wn[e].load(wr + k + 128 + 8 * e);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          LceEight<E> x;
          x.load(hr[b] + k + 8 * e);
          acc[b] = lce_mma<BELOW>(wc[e], x, acc[b], most);
        }
    }
    if (whole < D) {
      const E *w_end = w + static_cast<int64_t>(r.classes - 1) * ldw + D, *h_end = h + static_cast<int64_t>(r.rows - 1) * ldh + D;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = D - whole - 32 * quarter - 8 * e;
        LceEight<E> a, x;
        a.some(wr + whole + 8 * e, n, w_end);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          x.some(hr[b] + whole + 8 * e, n, h_end);
          acc[b] = lce_mma<BELOW>(a, x, acc[b], most);
        }
      }
    }
  };
  products(std::true_type{});
  // (once more, slower, where a wave has met one: infinities, and what bf16 rounds to them)
  if constexpr (__is_same(E, float))
    if (__any(most >= kHpLarge)) products(std::false_type{});
  // acc[b][x]: class c0 + 4 quarter + x, row 16 b + l16
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int j = 16 * b + l16;
    const int64_t target = j < r.rows ? r.targets[j] : -1;
    float m = -INFINITY, v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = c0 + 4 * quarter + x;
      v[x] = c < r.classes ? acc[b][x] + (r.bias != nullptr ? r.bias[c] : 0.f) : -INFINITY;
      if (c == target && c < r.classes) at_target[j] = v[x];
      m = fmaxf(m, v[x]);
    }
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) s += __expf(v[x] - base);
    floatx2 ms = {m, s};
    ms = lce_join2(ms, floatx2{__shfl_xor(ms[0], 16), __shfl_xor(ms[1], 16)});
    ms = lce_join2(ms, floatx2{__shfl_xor(ms[0], 32), __shfl_xor(ms[1], 32)});
    if (quarter == 0 && j < r.rows) part[static_cast<int64_t>(blockIdx.x) * r.rows + j] = ms;
  }
}

__device__ __forceinline__ void lce_row(const LceRows& r, int j, floatx2 ms, const float* __restrict__ at_target, float* __restrict__ losses,
                                        float* __restrict__ lse) {
  const int64_t target = r.targets[j];
  const float l = __logf(ms[1]);
  lse[j] = ms[0] + l;
  // (a target that is no class and not the ignored one: NaN)
  losses[j] = target == r.ignore ? 0.f : target < 0 || target >= r.classes ? NAN : ms[0] - at_target[j] + l;
}

// lse and loss of 64 rows from the parts of all classes, a sixteenth of them a wave.
static __global__ __launch_bounds__(1024) void lce_rows_kernel(LceRows r, const floatx2* __restrict__ part, int parts, const float* __restrict__ at_target,
                                                               float* __restrict__ losses, float* __restrict__ lse) {
  __shared__ floatx2 joined[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + lane;
  floatx2 ms = {-INFINITY, 0.f};
  if (j < r.rows) {
#pragma unroll 4
    for (int t = wave; t < parts; t += 16) ms = lce_join2(ms, part[static_cast<int64_t>(t) * r.rows + j]);
  }
  joined[wave][lane] = ms;
  __syncthreads();
  if (wave != 0 || j >= r.rows) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) ms = lce_join2(ms, joined[k][lane]);
  lce_row(r, j, ms, at_target, losses, lse);
}

// A row a work group, for few rows of many parts.
static __global__ __launch_bounds__(512) void lce_row_kernel(LceRows r, const floatx2* __restrict__ part, int parts, const float* __restrict__ at_target,
                                                             float* __restrict__ losses, float* __restrict__ lse) {
  __shared__ floatx2 joined[8];
  const int j = blockIdx.x;
  floatx2 ms = {-INFINITY, 0.f};
#pragma unroll 8
  for (int t = threadIdx.x; t < parts; t += 512) ms = lce_join2(ms, part[static_cast<int64_t>(t) * r.rows + j]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ms = lce_join2(ms, floatx2{__shfl_xor(ms[0], o), __shfl_xor(ms[1], o)});
  if ((threadIdx.x & 63) == 0) joined[threadIdx.x >> 6] = ms;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) ms = lce_join2(ms, joined[w]);
  lce_row(r, j, ms, at_target, losses, lse);
}

// The sum or mean over the rows, in double.
static __global__ __launch_bounds__(1024) void lce_total_kernel(LceRows r, const float* __restrict__ losses, int reduction, float* __restrict__ loss) {
  __shared__ double red[16];
  __shared__ u64 count_of[16];
  double s = 0.;
  u64 count = 0;
  for (int j = threadIdx.x; j < r.rows; j += 1024) {
    s += losses[j];
    count += r.targets[j] != r.ignore ? 1 : 0;
  }
  s = group_sum<16>(s, red);
  count = group_sum<16>(count, count_of);
  if (threadIdx.x == 0) *loss = static_cast<float>(reduction == kLossMean ? s / static_cast<double>(count) : s);
}

// share[n] = c_n / most 2^lift, unit = most 2^-lift, with the largest finite |c_n| for most (plain: 1).
static __global__ __launch_bounds__(1024) void lce_shares_kernel(LceRows r, const float* __restrict__ g, int reduction, int plain, int lift,
                                                                 float* __restrict__ share, float* __restrict__ unit) {
  __shared__ float red[16];
  __shared__ u64 count_of[16];
  float common = 0.f;
  if (reduction != kLossNone) {
    u64 count = 0;
    if (reduction == kLossMean) {
      for (int j = threadIdx.x; j < r.rows; j += 1024) count += r.targets[j] != r.ignore ? 1 : 0;
      count = group_sum<16>(count, count_of);
    } else {
      count = 1;
    }
    common = count == 0 ? 0.f : *g / static_cast<float>(count);
  }
  float most = 1.f;
  if (!plain) {
    most = fabsf(common);
    if (reduction == kLossNone) {
      most = 0.f;
      for (int j = threadIdx.x; j < r.rows; j += 1024) most = fmaxf(most, r.targets[j] != r.ignore && fabsf(g[j]) < INFINITY ? fabsf(g[j]) : 0.f);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 16; ++w) most = fmaxf(most, red[w]);
    }
    most = most > 0.f && most < INFINITY ? fmaxf(most, 0x1p-100f) : 1.f;      // (the unit is a normal number)
  }
  if (threadIdx.x == 0) *unit = ldexpf(most, -lift);
  for (int j = threadIdx.x; j < r.rows; j += 1024) {
    const int64_t target = r.targets[j];
    const float c = reduction == kLossNone ? g[j] : common;
    share[j] = target == r.ignore ? 0.f : target < 0 || target >= r.classes ? NAN : ldexpf(c / most, lift);
  }
}

template <typename T>
static __global__ __launch_bounds__(256) void lce_bias_kernel(const T* __restrict__ x, int n, float* __restrict__ out) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = static_cast<float>(x[i]);
}

// ---- host side
constexpr int64_t kLcePieceBytes = 512ll << 20;       // of d
// Rows that lce_few_kernel() takes rather than the tiles; copied: the tiles want copies of the operands first, of another pitch or in pieces.
// (50257 x 768: bf16 4 rows 21 us, 16 rows 26 us, the tiles of 128 24 us for any number of these, but 103083 x 302 with copies 58 us, 10 rows
// without 25 us, 120757 x 461 80 us either way for 17 rows; fp32 55 us for up to 16, 75 us for 32 and 114 us for 64 rows, by the tiles 172 us.)
inline int64_t lce_few_rows(int dtype, bool copied) { return dtype == AK_F32 ? 64 : copied ? 16 : 8; }

constexpr int64_t kLcePartBytes = 512ll << 20;        // of the forward pass's sums of tiles

// Sizes that both the workspace query and the launches use.
constexpr int64_t kLceSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
constexpr double kLceSumUs = 6. / 4.5e6;                  // of an element of a split's sum

struct LcePlan {
  int64_t N, V, D;
  int k;                   // 16-bit pieces of a value
  bool few;                // the forward pass of few rows
  int64_t part, rows;      // classes of a part of the forward pass; rows that it takes at a time
  int64_t piece, pieces;   // classes of a piece, a multiple of 256 (the last may have fewer)
  int64_t ldp;             // row pitch of padded operands
  bool wide;               // tiles of 256 in the gradients' products
  int splits, splits_dw;   // of the contractions over a piece's classes, over the rows
  int64_t ld_sum;          // row pitch of the fp32 sums of dh
};

inline LcePlan lce_plan(int dtype, int64_t N, int64_t V, int64_t D, bool backward, bool copied) {
  LcePlan p = {};
  p.N = N; p.V = V; p.D = D;
  p.k = dtype == AK_F32 ? 3 : 1;
  p.few = !backward && N <= lce_few_rows(dtype, copied);
  p.part = p.few ? 16 : hp_wide(V, N) ? 256 : hp_tiny(V, N) ? 64 : 128;
  // (at least 256 rows: 2^20 tiles at most, far from the 2^23 whose threads 32 bits count)
  p.rows = std::min(N, std::max<int64_t>(kLcePartBytes / (((V + p.part - 1) / p.part) * static_cast<int64_t>(sizeof(float) * 2)) / 256 * 256, 256));
  // (at most 2^24: 32 rows of d within 32-bit byte offsets)
  const int64_t fit = std::min<int64_t>(std::max<int64_t>(kLcePieceBytes / (N * p.k * 2) / 256 * 256, 256), 1 << 24);
  p.pieces = (V + fit - 1) / fit;
  p.piece = align_up((V + p.pieces - 1) / p.pieces, 256);
  p.pieces = (V + p.piece - 1) / p.piece;
  p.ldp = align_up(D, 8);
  p.ld_sum = align_up(D, 4);
  if (!backward) return p;
  // The gradients' products of a piece, in one launch: the tiles of 256 or 128 and the splits of either contraction that are least in an
  // estimate of the time: k-tiles of 0.82 us, or of 0.6 us where two small ones share a CU, over as many work groups as run at once, the
  // longest first; what the last of them wait for; and the sums of the splits, written and read.  (With 8 splits of the classes at most,
  // none of the rows and tiles of 256 wherever they fill the device: 10 rows of 103083 classes of 302 210 us, with up to 64 34 us;
  // 2987 x 2680 x 1600 in fp32 487 us, with three splits of the rows 362 us.)
  const int64_t k = std::min(p.piece, V), k_dw = (N + 31) / 32, k_dh = (align_up(k, 8) + 31) / 32, products = p.k == 1 ? 1 : 6;
  double least = 1e30;
  for (const int64_t tile : {256, 128}) {
    const int64_t across = (D + tile - 1) / tile, of_dw = across * ((k + tile - 1) / tile), of_dh = across * ((N + tile - 1) / tile);
    const int64_t places = tile == 256 ? 256 : 512;
    const double share = static_cast<double>(of_dw * k_dw + of_dh * k_dh) / places;
    for (const int64_t w : kLceSplits) {
      if (w > 1 && (k_dw / w < 4 || of_dw * w > 2 * places)) break;
      for (const int64_t h : kLceSplits) {
        if (h > 1 && k_dh / h < 4) break;
        const double of_w = (k_dw + w - 1) / w, of_h = (k_dh + h - 1) / h;
        const double longest = std::max(of_w, of_h), tiles = std::max(longest, share + longest / 8 + std::min(of_w, of_h) / 2);
        const double sums = static_cast<double>(h) * N * D + (w > 1 ? static_cast<double>(w) * k * D : 0.);
        const double us = tiles * products * (tile == 256 ? 0.82 : 0.6) + sums * kLceSumUs + (w > 1 ? 5. : 0.);
        if (us < least) {
          least = us;
          p.wide = tile == 256;
          p.splits_dw = static_cast<int>(w);
          p.splits = static_cast<int>(h);
        }
      }
    }
  }
  auto whole = [](int64_t n, int splits) {           // splits of whole k-tiles
    const int64_t per = align_up((n + splits - 1) / splits, 32);
    return static_cast<int>((n + per - 1) / per);
  };
  p.splits = whole(align_up(k, 8), p.splits);
  p.splits_dw = whole(N, p.splits_dw);
  return p;
}

struct LceSpace {
  unsigned char *h, *w;    // padded operands, or operands in pieces
  float* bias;
  floatx2* part;
  float *at_target, *losses;
  // backward
  float *share, *unit;
  unsigned char* d;
  float *sum, *sum_dw, *columns;
  size_t bytes;
};

// What a call makes in its workspace beside what all calls do: copies of operands, sums of the gradients that are asked for.
struct LceNeeds {
  bool h, w, bias;         // copied
  bool dh, dw, db;
};

inline LceSpace lce_space(const LcePlan& p, bool backward, const LceNeeds& need, void* ws) {
  Carver c{static_cast<unsigned char*>(ws)};
  LceSpace s = {};
  if (need.h) s.h = c.take<unsigned char>(p.N * p.ldp * p.k * 2);
  if (need.w) s.w = c.take<unsigned char>(p.V * p.ldp * p.k * 2);
  if (need.bias) s.bias = c.take<float>(p.V);
  if (!backward) {
    s.part = c.take<floatx2>((p.V + p.part - 1) / p.part * p.rows);
    s.at_target = c.take<float>(p.rows);
    s.losses = c.take<float>(p.N);
  } else {
    s.share = c.take<float>(p.N);
    s.unit = c.take<float>(1);
    s.d = c.take<unsigned char>(p.N * p.piece * p.k * 2);
    if (need.dh) s.sum = c.take<float>(static_cast<int64_t>(p.splits) * p.N * p.ld_sum);
    if (need.dw && p.splits_dw > 1) s.sum_dw = c.take<float>(p.splits_dw * std::min(p.piece, p.V) * p.ld_sum);
    if (need.db) s.columns = c.take<float>(static_cast<int64_t>(column_sums_ws_bytes(p.N, p.k * p.piece) / sizeof(float)));
  }
  s.bytes = c.used;
  return s;
}

struct LceCall {
  const void* h; int64_t ldh;
  const void* w; int64_t ldw;
  const void* bias; int bias_dtype;
  LceRows r;
  int64_t D;
  int dtype;
  hipStream_t stream;
};

// Operands as the panels need them: copied where their pitch or alignment is another, or in pieces.
template <typename E>
inline int lce_operands(LceCall& c, const LcePlan& p, const LceSpace& s) {
  auto as_needed = [&](const void*& x, int64_t& ld, int64_t rows, unsigned char* to) {
    if (to == nullptr) return AK_OK;
    const E* from = static_cast<const E*>(x);
    const int64_t from_ld = ld;
    x = to;
    ld = p.k * p.ldp;
    if constexpr (__is_same(E, float)) return hp_pieces<3>(from, from_ld, rows, p.D, reinterpret_cast<__bf16*>(to), p.ldp, c.stream);
    else return hp_pad(from, from_ld, rows, p.D, reinterpret_cast<E*>(to), p.ldp, c.stream);
  };
  const int rc = as_needed(c.h, c.ldh, p.N, s.h);
  return rc != AK_OK ? rc : as_needed(c.w, c.ldw, p.V, s.w);
}

inline int lce_bias(LceCall& c, const LcePlan& p, const LceSpace& s) {
  if (c.bias == nullptr) return AK_OK;
  if (c.bias_dtype == AK_F32) {
    c.r.bias = static_cast<const float*>(c.bias);
    return AK_OK;
  }
  c.r.bias = s.bias;
  return with_type(c.bias_dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    hipLaunchKernelGGL(lce_bias_kernel<T>, dim3(static_cast<unsigned>((p.V + 255) / 256)), dim3(256), 0, c.stream, static_cast<const T*>(c.bias),
                       static_cast<int>(p.V), s.bias);
    return check_launch();
  });
}

// losses and lse of all rows
template <typename E>
inline int lce_forward(LceCall c, const LcePlan& p, const LceSpace& s, float* losses, float* lse) {
  if (p.few) {
    const int64_t groups = (p.V + 15) / 16;
    auto go = [&](auto nb) {
      hipLaunchKernelGGL((lce_few_kernel<E, decltype(nb)::value>), dim3(static_cast<unsigned>(groups)), dim3(64), 0, c.stream, static_cast<const E*>(c.h),
                         c.ldh, static_cast<const E*>(c.w), c.ldw, static_cast<int>(p.D), c.r, s.part, s.at_target);
      hipLaunchKernelGGL(lce_row_kernel, dim3(static_cast<unsigned>(p.N)), dim3(512), 0, c.stream, c.r, s.part, static_cast<int>(groups), s.at_target, losses, lse);
      return check_launch();
    };
    if constexpr (__is_same(E, float)) {
      if (p.N > 32) return go(std::integral_constant<int, 4>{});
      if (p.N > 16) return go(std::integral_constant<int, 2>{});
    }
    return go(std::integral_constant<int, 1>{});
  }
  const int rc = lce_operands<E>(c, p, s);
  if (rc != AK_OK) return rc;
  using M = typename LceKind<E>::type;
  constexpr bool PIECES = LceKind<E>::pieces > 1;
  const HpOperand A = hp_operand(c.w, c.ldw, p.V, p.D, true);
  for (int64_t n = 0; n < p.N; n += p.rows) {
    LceRows r = c.r;
    r.targets += n;
    r.rows = static_cast<int>(std::min(p.N - n, p.rows));
    const HpOperand B = hp_operand(static_cast<const M*>(c.h) + n * c.ldh, c.ldh, r.rows, p.D, true);
    auto go = [&](auto cfg) {
      using Cfg = decltype(cfg);
      HpProblem q = hp_problem<Cfg>(A, B, p.V, r.rows, align_up(p.D, 8));
      if (PIECES) q.pieces = hp_six(p.ldp, p.ldp);
      const int done = hp_launch<Cfg, M, LceStats>(q, LceStats::Params{r, s.part, s.at_target}, c.stream);
      if (done != AK_OK) return done;
      hipLaunchKernelGGL(lce_rows_kernel, dim3(static_cast<unsigned>((r.rows + 63) / 64)), dim3(1024), 0, c.stream, r, s.part, q.tiles_i, s.at_target, losses + n,
                         lse + n);
      return check_launch();
    };
    const int done = hp_form<true, true, PIECES>(p.V, p.N, go);
    if (done != AK_OK) return done;
  }
  return AK_OK;
}

struct LceGrads {
  void *dh, *dw, *db;
  int db_dtype;
};

template <typename E>
inline int lce_backward(LceCall c, const float* lse, const LcePlan& p, const LceSpace& s, const LceGrads& out) {
  using M = typename LceKind<E>::type;
  constexpr bool PIECES = LceKind<E>::pieces > 1;
  int rc = lce_operands<E>(c, p, s);
  if (rc != AK_OK) return rc;
  M* d = reinterpret_cast<M*>(s.d);
  const int64_t ldd = p.k * p.piece;
  for (int64_t k = 0; k < p.pieces; ++k) {
    const int64_t c0 = k * p.piece, width = std::min(p.piece, p.V - c0), padded = align_up(width, 8);
    const M* w = static_cast<const M*>(c.w) + c0 * c.ldw;
    auto grad = [&](auto cfg) {
      using Cfg = decltype(cfg);
      HpProblem q = hp_problem<Cfg>(hp_operand(w, c.ldw, width, p.D, true), hp_operand(c.h, c.ldh, p.N, p.D, true), padded, p.N, align_up(p.D, 8));
      if (PIECES) q.pieces = hp_six(p.ldp, p.ldp);
      typename LceGrad<E>::Params e{c.r, lse, s.share, d, ldd, p.piece, static_cast<int>(c0), static_cast<int>(padded)};
      return hp_launch<Cfg, M, LceGrad<E>>(q, e, c.stream);
    };
    rc = hp_form<true, true, PIECES>(padded, p.N, grad);
    if (rc != AK_OK) return rc;
    // dw: i features, j classes, k rows.  dh: i features, j rows, k classes (a shorter last piece has no more splits)
    auto gradients = [&](auto dw_cfg, auto dh_cfg) {
      using W = decltype(dw_cfg);
      using H = decltype(dh_cfg);
      HpProblem qw = hp_problem<W>(hp_operand(c.h, c.ldh, p.N, p.D, false), hp_operand(d, ldd, p.N, padded, false), p.D, width, p.N, p.splits_dw);
      HpProblem qh = hp_problem<H>(hp_operand(w, c.ldw, width, p.D, false), hp_operand(d, ldd, p.N, padded, true), p.D, p.N, padded, p.splits);
      if (PIECES) qw.pieces = qh.pieces = hp_six(p.ldp, p.piece);
      E* dw = static_cast<E*>(out.dw) + c0 * p.D;
      const int D = static_cast<int>(p.D), classes = static_cast<int>(width);
      const HpSum::Params eh{s.sum, p.ld_sum, p.N * p.ld_sum, D, static_cast<int>(p.N), k == 0};
      if (out.dw == nullptr) return hp_launch<H, M, HpSum>(qh, eh, c.stream);
      if (p.splits_dw == 1) {
        const typename HpStore<E>::Params ew{dw, p.D, D, classes, 1.f, s.unit};
        if (out.dh == nullptr) return hp_launch<W, M, HpStore<E>>(qw, ew, c.stream);
        return hp_launch_both<W, HpStore<E>, H, HpSum, M>(qw, ew, qh, eh, c.stream);
      }
      const HpSum::Params ew{s.sum_dw, p.ld_sum, width * p.ld_sum, D, classes, 1};
      const int done = out.dh == nullptr ? hp_launch<W, M, HpSum>(qw, ew, c.stream) : hp_launch_both<W, HpSum, H, HpSum, M>(qw, ew, qh, eh, c.stream);
      return done != AK_OK ? done : hp_total(s.sum_dw, p.ld_sum, width * p.ld_sum, p.splits_dw, width, D, 1.f, s.unit, dw, c.stream);
    };
    if (out.dh != nullptr || out.dw != nullptr)
      rc = p.wide ? gradients(HpWide<false, false, PIECES>{}, HpWide<false, true, PIECES>{})
                  : gradients(HpSmall<false, false, PIECES>{}, HpSmall<false, true, PIECES>{});
    if (rc == AK_OK && out.db != nullptr)
      rc = with_type(out.db_dtype, [&](auto t) {
        using O = typename decltype(t)::type;
        return column_sums(d, ldd, p.N, width, 1.f, s.unit, static_cast<O*>(out.db) + c0, s.columns, c.stream, p.k, p.piece);
      });
    if (rc != AK_OK) return rc;
  }
  if (out.dh == nullptr) return AK_OK;
  return hp_total(s.sum, p.ld_sum, p.N * p.ld_sum, p.splits, p.N, static_cast<int>(p.D), 1.f, s.unit, static_cast<E*>(out.dh), c.stream);
}

inline int lce_check(const void* h, int64_t ldh, const void* w, int64_t ldw, const void* bias, int bias_dtype, const int64_t* targets, int64_t rows,
                     int64_t classes, int64_t width, int dtype, int reduction) {
  if (h == nullptr || w == nullptr || targets == nullptr || rows < 0 || classes <= 0 || width <= 0 || ldh < width || ldw < width) return AK_ERR_ARG;
  if (!is_element_type(dtype) || (bias != nullptr && bias_dtype != AK_F32 && bias_dtype != dtype)) return AK_ERR_ARG;
  if (reduction < kLossNone || reduction > kLossMean) return AK_ERR_ARG;
  // counts in 32 bits; 256 rows of a panel within 32-bit byte offsets
  if (rows > (1 << 28) || classes > (1 << 28) || width > (1 << 20) || ldh > (1 << 21) || ldw > (1 << 21)) return AK_ERR_TOO_LARGE;
  return AK_OK;
}

}  // namespace ak

extern "C" size_t ak_linear_cross_entropy_ws_bytes(int dtype, int64_t rows, int64_t classes, int64_t width, int backward) {
  if (!ak::is_element_type(dtype) || rows <= 0 || classes <= 0 || width <= 0 || rows > (1 << 28) || classes > (1 << 28) || width > (1 << 20)) return 0;
  // enough for operands of any alignment
  auto bytes = [&](bool copied) {
    const ak::LcePlan p = ak::lce_plan(dtype, rows, classes, width, backward != 0, copied);
    return ak::lce_space(p, backward != 0, {copied && !p.few, copied && !p.few, true, true, true, true}, nullptr).bytes;
  };
  return backward != 0 ? bytes(true) : std::max(bytes(false), bytes(true));
}

namespace ak {

// Plan and workspace of a call.
struct LceLayout {
  LcePlan plan;
  LceSpace space;
};

inline LceLayout lce_layout(const void* h, int dtype, int64_t ldh, const void* w, int64_t ldw, bool narrow_bias, int64_t rows, int64_t classes, int64_t width,
                            bool backward, bool dh, bool dw, bool db, void* ws) {
  const bool copy_h = dtype == AK_F32 || !hp_aligned(h, ldh, width), copy_w = dtype == AK_F32 || !hp_aligned(w, ldw, width);
  const LcePlan p = lce_plan(dtype, rows, classes, width, backward, copy_h || copy_w);
  return LceLayout{p, lce_space(p, backward, {!p.few && copy_h, !p.few && copy_w, narrow_bias, dh, dw, db}, ws)};
}

}  // namespace ak

extern "C" size_t ak_linear_cross_entropy_ws_bytes_of(const void* h, int dtype, int64_t ldh, const void* w, int64_t ldw, int bias_dtype, int64_t rows,
                                                      int64_t classes, int64_t width, int gradients) {
  if (ak_linear_cross_entropy_ws_bytes(dtype, rows, classes, width, 0) == 0) return 0;
  return ak::lce_layout(h, dtype, ldh, w, ldw, bias_dtype >= 0 && bias_dtype != AK_F32, rows, classes, width, gradients != 0, (gradients & 1) != 0,
                        (gradients & 2) != 0, (gradients & 4) != 0, nullptr).space.bytes;
}

extern "C" int ak_linear_cross_entropy(const void* h, int dtype, int64_t ldh, const void* w, int64_t ldw, const void* bias, int bias_dtype,
                                       const int64_t* targets, int64_t rows, int64_t classes, int64_t width, int64_t ignore_index, int reduction,
                                       float* loss, float* lse, void* ws, size_t ws_bytes, ak_stream_t stream) {
  using namespace ak;
  int rc = lce_check(h, ldh, w, ldw, bias, bias_dtype, targets, rows, classes, width, dtype, reduction);
  if (rc != AK_OK) return rc;
  if (rows == 0) return reduction == kLossNone ? AK_OK : AK_ERR_ARG;
  if (loss == nullptr || lse == nullptr) return AK_ERR_ARG;
  const LceLayout layout = lce_layout(h, dtype, ldh, w, ldw, bias != nullptr && bias_dtype != AK_F32, rows, classes, width, false, false, false, false, ws);
  const LcePlan& p = layout.plan;
  const LceSpace& s = layout.space;
  if (ws == nullptr || ws_bytes < s.bytes) return AK_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LceCall c{h, ldh, w, ldw, bias, bias_dtype, LceRows{targets, nullptr, ignore_index, static_cast<int>(rows), static_cast<int>(classes)}, width, dtype, st};
  rc = lce_bias(c, p, s);
  if (rc != AK_OK) return rc;
  float* losses = reduction == kLossNone ? loss : s.losses;
  rc = with_type(dtype, [&](auto t) { return lce_forward<typename decltype(t)::type>(c, p, s, losses, lse); });
  if (rc != AK_OK) return rc;
  if (reduction != kLossNone) hipLaunchKernelGGL(lce_total_kernel, dim3(1), dim3(1024), 0, st, c.r, losses, reduction, loss);
  return check_launch();
}

extern "C" int ak_linear_cross_entropy_backward(const float* g, const void* h, int dtype, int64_t ldh, const void* w, int64_t ldw, const void* bias,
                                                int bias_dtype, const int64_t* targets, const float* lse, int64_t rows, int64_t classes, int64_t width,
                                                int64_t ignore_index, int reduction, void* dh, void* dw, void* db, void* ws, size_t ws_bytes,
                                                ak_stream_t stream) {
  using namespace ak;
  int rc = lce_check(h, ldh, w, ldw, bias, bias_dtype, targets, rows, classes, width, dtype, reduction);
  if (rc != AK_OK) return rc;
  if (g == nullptr || lse == nullptr || rows == 0) return AK_ERR_ARG;
  if (dh == nullptr && dw == nullptr && db == nullptr) return AK_OK;
  const LceLayout layout = lce_layout(h, dtype, ldh, w, ldw, bias != nullptr && bias_dtype != AK_F32, rows, classes, width, true, dh != nullptr, dw != nullptr,
                                      db != nullptr, ws);
  const LcePlan& p = layout.plan;
  const LceSpace& s = layout.space;
  if (ws == nullptr || ws_bytes < s.bytes) return AK_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LceCall c{h, ldh, w, ldw, bias, bias_dtype, LceRows{targets, nullptr, ignore_index, static_cast<int>(rows), static_cast<int>(classes)}, width, dtype, st};
  rc = lce_bias(c, p, s);
  if (rc != AK_OK) return rc;
  hipLaunchKernelGGL(lce_shares_kernel, dim3(1), dim3(1024), 0, st, c.r, g, reduction, dtype == AK_F32 ? 1 : 0, dtype == AK_F16 ? 14 : 0, s.share, s.unit);
  const LceGrads out{dh, dw, db, bias == nullptr ? dtype : bias_dtype};
  return with_type(dtype, [&](auto t) { return lce_backward<typename decltype(t)::type>(c, lse, p, s, out); });
}
