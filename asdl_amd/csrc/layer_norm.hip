// Layer norm over the last axis, its backward pass, and the unit-wise Fisher blocks of its weight and bias.
//   forward:  m = mean x, r = (mean (x - m)^2 + eps)^(-1/2), h = (x - m) r, y = h w + b;  m and r are kept for the way back
//   backward: dx = r (g w - mean(g w) - h mean(g w h)),  dw = sum_rows g h,  db = sum_rows g,
//             blocks[f] = beta blocks[f] + alpha sum_rows [[(g h)^2, g^2 h], [g^2 h, g^2]]
// The mean of what is left after the first mean is taken off corrects it by what its sum had rounded away (rows of equal values give
// h = 0 whatever their size), and the variance is the mean of centred squares, no difference of large sums.  Everything is fp32,
// rounded when it is stored.
// Each way reads its operands once and writes its result once.  8192 rows of 768 fp32 features with Fisher blocks: 10.9 us forward
// (50 MB, 4.6 TB/s), 16.3 us backward (75 MB, 4.6 TB/s) and 3.9 us for the sums of the partial rows, bfloat16 ones with half the bytes 8.4 us
// forward and 15.7 us for both launches backward (14.7 without the blocks), which is not the memory's time; 16384 rows of 4096 bfloat16 ones: 130 us
// both ways (671 MB, 5.2 TB/s, the rate of a large copy).  A few rows cost the launch, 5 to 6 us a call.
#include "elements.hpp"

namespace ak {

struct LnForward {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int64_t ldx, ldy, rows, F;
  float eps;
};

struct LnBackward {
  const void* g;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* w;
  void* dx;
  float* part;             // [chunks][sums][F]
  int64_t ldg, ldx, lddx, rows, F, rows_per_chunk;
};

// L lanes hold a row in registers: V vectors of E elements a lane and, where F is no multiple of E, one of the last F % E elements
// each for the first lanes (a loop over the elements of a last vector, with a condition each, cost more code than all the rest).
template <int L, int V, int E_>
struct LnLayout {
  static constexpr int E = E_, N = E * V + 1, most = L * V * E;       // values a lane, features
  int lane, whole, rest;
  __device__ __forceinline__ LnLayout(int64_t F)
      : lane(threadIdx.x % L), whole(static_cast<int>(F) / E * E), rest(static_cast<int>(F) % E) {}
  __device__ __forceinline__ int at(int v) const { return (v * L + lane) * E; }
  __device__ __forceinline__ bool has(int i) const { return i < N - 1 ? at(i / E) < whole : lane < rest; }
};

// A lane's part of a row or of a weight on its way: 0 where it has none.
template <typename T, typename Layout, int V>
struct LnSlice {
  static constexpr int E = Layout::E;
  Some<T, E> v[V];
  T last;
  __device__ __forceinline__ void load(const Layout& at, const T* __restrict__ p) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i].clear();
      if (at.at(i) < at.whole) v[i].load(p + at.at(i));
    }
    last = static_cast<T>(0.f);
    if (at.lane < at.rest) last = p[at.whole + at.lane];
  }
  __device__ __forceinline__ float get(int i) const { return i < E * V ? v[i / E].get(i % E) : static_cast<float>(last); }
  __device__ __forceinline__ void set(int i, float x) {
    if (i < E * V) v[i / E].set(i % E, x);
    else last = static_cast<T>(x);
  }
  __device__ __forceinline__ void store(const Layout& at, T* __restrict__ p) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (at.at(i) < at.whole) v[i].store(p + at.at(i));
    if (at.lane < at.rest) p[at.whole + at.lane] = last;
  }
};

// The type of the weights is a template parameter, not a branch on a code: such a branch inside the per-lane conditions of load() left the
// register pair of the lane's column offset undefined on one of its ways, and the addresses made from it faulted.
template <typename W, int V, typename Layout>
__device__ __forceinline__ void ln_vector(const Layout& at, const void* p, float none, float (&out)[Layout::N]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < Layout::N; ++i) out[i] = none;
    return;
  }
  LnSlice<W, Layout, V> some;
  some.load(at, static_cast<const W*>(p));
#pragma unroll
  for (int i = 0; i < Layout::N; ++i) out[i] = some.get(i);
}

// Sums of K values over the lanes of a row.  L > 64: through `red` (K words a wave) with barriers, which the whole work group passes.
template <int L, int K>
__device__ __forceinline__ void ln_row_sums(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lanes_sum<(L < 64 ? L : 64)>(v[k]);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = red[first * K + k];
#pragma unroll
      for (int w = 1; w < W; ++w) s += red[(first + w) * K + k];
      v[k] = s;
    }
  }
}

// Bound by the memory: the weights stay in registers over the rows of a lane group, and the next row is on its way while one is
// computed.  (A work group per row that reads it three more times from the caches: 44 us for 2048 rows of 8192, here 16.)
template <typename X, typename Y, typename W, int L, int V, int THREADS>
static __global__ __launch_bounds__(THREADS) void ln_forward_rows_kernel(LnForward p) {
  using Layout = LnLayout<L, V, 16 / sizeof(X)>;
  constexpr int N = Layout::N, GROUPS = THREADS / L;
  __shared__ float red[THREADS / 64];
  const Layout at(p.F);
  const int group = threadIdx.x / L;
  const float n = static_cast<float>(p.F);
  float w[N], b[N];
  ln_vector<W, V>(at, p.w, 1.f, w);
  ln_vector<W, V>(at, p.b, 0.f, b);
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS;
  LnSlice<X, Layout, V> next;
  auto fetch = [&](int64_t row) { next.load(at, static_cast<const X*>(p.x) + (row < p.rows ? row : 0) * p.ldx); };
  fetch(base + group);
  for (; base < p.rows; base += step) {
    const int64_t row = base + group;
    float c[N], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) s[0] += c[i] = next.get(i);
    if (base + step < p.rows) fetch(row + step);
    ln_row_sums<L>(s, red);
    const float m0 = s[0] / n;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s[0] += c[i] = at.has(i) ? c[i] - m0 : 0.f;
    ln_row_sums<L>(s, red);
    const float m = m0 + s[0] / n, shift = m - m0;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = at.has(i) ? c[i] - shift : 0.f;
      s[0] += c[i] * c[i];
    }
    ln_row_sums<L>(s, red);
    const float r = 1.f / sqrtf(s[0] / n + p.eps);
    if (row < p.rows) {
      LnSlice<Y, Layout, V> out;
#pragma unroll
      for (int i = 0; i < N; ++i) out.set(i, c[i] * r * w[i] + b[i]);
      out.store(at, static_cast<Y*>(p.y) + row * p.ldy);
      if (at.lane == 0) {
        p.mean[row] = m;
        p.rstd[row] = r;
      }
    }
  }
}

// A lane keeps the sums of its columns over its rows: SUMS 0 none, 2 dw and db, 5 with the three products of the Fisher blocks.  At the
// end the groups of a work group are added through the LDS, one partial row per work group in `part`.
template <typename X, typename G, typename W, int L, int V, int THREADS, int SUMS>
static __global__ __launch_bounds__(THREADS) void ln_backward_fused_kernel(LnBackward p) {
  using Layout = LnLayout<L, V, 16 / sizeof(X)>;
  constexpr int N = Layout::N, GROUPS = THREADS / L;
  __shared__ float red[2 * THREADS / 64];
  alignas(16) __shared__ float joined[SUMS > 0 && GROUPS > 1 ? GROUPS * Layout::most : 4];
  const Layout at(p.F);
  const int group = threadIdx.x / L;
  const float n = static_cast<float>(p.F);
  float w[N], sums[SUMS > 0 ? SUMS : 1][N];
  ln_vector<W, V>(at, p.w, 1.f, w);
#pragma unroll
  for (int q = 0; q < SUMS; ++q)
#pragma unroll
    for (int i = 0; i < N; ++i) sums[q][i] = 0.f;
  LnSlice<X, Layout, V> next_x;
  LnSlice<G, Layout, V> next_g;
  float next_m, next_r;
  auto fetch = [&](int64_t row) {
    row = row < p.rows ? row : 0;
    next_x.load(at, static_cast<const X*>(p.x) + row * p.ldx);
    next_g.load(at, static_cast<const G*>(p.g) + row * p.ldg);
    next_m = p.mean[row];
    next_r = p.rstd[row];
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS;
  fetch(base + group);
  for (; base < p.rows; base += step) {
    const int64_t row = base + group;
    const float m = next_m, r = next_r;
    float h[N], g[N], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      g[i] = next_g.get(i);
      h[i] = at.has(i) ? (next_x.get(i) - m) * r : 0.f;
    }
    if (base + step < p.rows) fetch(row + step);
    if (SUMS > 0 && row < p.rows) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float gh = g[i] * h[i];
        sums[0][i] += gh;
        sums[1][i] += g[i];
        if constexpr (SUMS == 5) {
          sums[2][i] += gh * gh;
          sums[3][i] += gh * g[i];
          sums[4][i] += g[i] * g[i];
        }
      }
    }
    if (p.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        g[i] *= w[i];
        s[0] += g[i];
        s[1] += g[i] * h[i];
      }
      ln_row_sums<L>(s, red);
      const float a = s[0] / n, t = s[1] / n;
      if (row < p.rows) {
        LnSlice<X, Layout, V> out;
#pragma unroll
        for (int i = 0; i < N; ++i) out.set(i, r * (g[i] - a - h[i] * t));
        out.store(at, static_cast<X*>(p.dx) + row * p.lddx);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < SUMS; ++q) {
    float* part = p.part + (static_cast<int64_t>(blockIdx.x) * SUMS + q) * p.F;
    LnSlice<float, Layout, V> out;
#pragma unroll
    for (int i = 0; i < N; ++i) out.set(i, sums[q][i]);
    if constexpr (GROUPS == 1) {
      out.store(at, part);
    } else {
      __syncthreads();
      out.store(at, joined + group * Layout::most);
      __syncthreads();
      for (int f = threadIdx.x; f < static_cast<int>(p.F); f += THREADS) {
        float s = joined[f];
#pragma unroll 8
        for (int k = 1; k < GROUPS; ++k) s += joined[k * Layout::most + f];
        part[f] = s;
      }
    }
  }
}

// Rows of more than 8192 features: one work group per row, which is read four times, from the caches but for the first, an element a
// load.  4096 rows of 16384 bfloat16 features: 214 us forward, 246 us backward (1.3 and 1.6 TB/s); 2048 of fp32 ones: 119 and 172 us.
template <typename X, typename Y, typename W>
static __global__ __launch_bounds__(256) void ln_forward_kernel(LnForward p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const X* __restrict__ x = static_cast<const X*>(p.x) + row * p.ldx;
  Y* __restrict__ y = static_cast<Y*>(p.y) + row * p.ldy;
  const float n = static_cast<float>(p.F);
  float s = 0.f;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) s += static_cast<float>(x[f]);
  float m = group_sum<4>(s, red) / n;
  s = 0.f;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) s += static_cast<float>(x[f]) - m;
  m += group_sum<4>(s, red) / n;
  s = 0.f;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    const float c = static_cast<float>(x[f]) - m;
    s += c * c;
  }
  const float r = 1.f / sqrtf(group_sum<4>(s, red) / n + p.eps);
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    float v = (static_cast<float>(x[f]) - m) * r;
    if (p.w != nullptr) v *= static_cast<float>(static_cast<const W*>(p.w)[f]);
    if (p.b != nullptr) v += static_cast<float>(static_cast<const W*>(p.b)[f]);
    y[f] = static_cast<Y>(v);
  }
  if (threadIdx.x == 0) {
    p.mean[row] = m;
    p.rstd[row] = r;
  }
}

template <typename X, typename G, typename W>
static __global__ __launch_bounds__(256) void ln_backward_rows_kernel(LnBackward p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const X* __restrict__ x = static_cast<const X*>(p.x) + row * p.ldx;
  const G* __restrict__ g = static_cast<const G*>(p.g) + row * p.ldg;
  X* __restrict__ dx = static_cast<X*>(p.dx) + row * p.lddx;
  const float n = static_cast<float>(p.F), m = p.mean[row], r = p.rstd[row];
  float s = 0.f, t = 0.f;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    const float gw = static_cast<float>(g[f]) * (p.w != nullptr ? static_cast<float>(static_cast<const W*>(p.w)[f]) : 1.f);
    s += gw;
    t += gw * ((static_cast<float>(x[f]) - m) * r);
  }
  s = group_sum<4>(s, red) / n;
  t = group_sum<4>(t, red) / n;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    const float gw = static_cast<float>(g[f]) * (p.w != nullptr ? static_cast<float>(static_cast<const W*>(p.w)[f]) : 1.f);
    dx[f] = static_cast<X>(r * (gw - s - (static_cast<float>(x[f]) - m) * r * t));
  }
}

// Sums over the rows of a chunk, a thread per column: dw, db and with BLOCKS the three products.  grid (columns / 256, chunks)
template <typename X, typename G, bool BLOCKS>
static __global__ __launch_bounds__(256) void ln_backward_columns_kernel(LnBackward p) {
  const int64_t f = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, chunk = blockIdx.y;
  if (f >= p.F) return;
  const int64_t r0 = chunk * p.rows_per_chunk, r1 = r0 + p.rows_per_chunk < p.rows ? r0 + p.rows_per_chunk : p.rows;
  float dw = 0.f, db = 0.f, ww = 0.f, wb = 0.f, bb = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float g = static_cast<float>(static_cast<const G*>(p.g)[row * p.ldg + f]);
    const float h = (static_cast<float>(static_cast<const X*>(p.x)[row * p.ldx + f]) - p.mean[row]) * p.rstd[row];
    const float gh = g * h;
    dw += gh;
    db += g;
    if constexpr (BLOCKS) {
      ww += gh * gh;
      wb += gh * g;
      bb += g * g;
    }
  }
  float* out = p.part + chunk * (BLOCKS ? 5 : 2) * p.F + f;
  out[0] = dw;
  out[p.F] = db;
  if constexpr (BLOCKS) {
    out[2 * p.F] = ww;
    out[3 * p.F] = wb;
    out[4 * p.F] = bb;
  }
}

// Sums of the partial rows, in a fixed order: 32 of the `sums` x F columns x 32 lanes of partial rows a work group.
template <typename W>
static __global__ __launch_bounds__(1024) void ln_backward_finish_kernel(const float* __restrict__ part, int64_t chunks, int64_t F, int sums,
                                                                         W* dw, W* db, float* blocks, float alpha, float beta) {
  __shared__ float red[32][33];
  const int column = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + column, width = F * sums;
  float s = 0.f;
  if (at < width) {
#pragma unroll 4
    for (int64_t c = lane; c < chunks; c += 32) s += part[c * width + at];
  }
  red[lane][column] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || at >= width) return;
  float total = 0.f;
#pragma unroll
  for (int l = 0; l < 32; ++l) total += red[l][column];
  const int q = static_cast<int>(at / F);
  const int64_t f = at - q * F;
  if (q == 0) {
    if (dw != nullptr) dw[f] = static_cast<W>(total);
  } else if (q == 1) {
    if (db != nullptr) db[f] = static_cast<W>(total);
  } else {
    float* out = blocks + 4 * f + (q == 2 ? 0 : q == 3 ? 1 : 3);
    out[0] = alpha * total + (beta != 0.f ? beta * out[0] : 0.f);
    if (q == 3) out[1] = alpha * total + (beta != 0.f ? beta * out[1] : 0.f);
  }
}

// Lanes of a row and elements a lane, by the features: a row lies in registers up to 8192 of them.  As few lanes as hold the row, since
// lanes without elements cost as much as others, and one wave rather than several where its registers hold the row, since sums over
// several waves wait at barriers.  Both ways, bfloat16, us forward / backward:
//   65536 rows of 96: 16 lanes 9.2 / 13.9, 64 lanes 28.6 / 29.6;          8192 of 768: 64 lanes 8.3 / 15.2, 256 lanes 17.6 / 19.8
//   8192 of 1600: 64 lanes 12.5 / 25.2, 256 lanes 18.7 / 21.5 (8 elements) and 22.0 / 30.0 (16)
// The backward pass of 2048 features would take twice the accumulators that a wave has registers for.  fn(lanes, elements) as integral
// constants; false for more features.
template <int I>
struct LnInt {
  static constexpr int value = I;
};
template <bool FORWARD, typename Fn>
static bool ln_layout(int64_t F, Fn&& fn) {
  if (F <= 128) fn(LnInt<16>{}, LnInt<8>{});
  else if (F <= 512) fn(LnInt<64>{}, LnInt<8>{});
  else if (F <= 1024) fn(LnInt<64>{}, LnInt<16>{});
  else if (F <= 2048) fn(LnInt<(FORWARD ? 64 : 256)>{}, LnInt<(FORWARD ? 32 : 8)>{});
  else if (F <= 4096) fn(LnInt<256>{}, LnInt<16>{});
  else if (F <= 8192) fn(LnInt<512>{}, LnInt<16>{});
  else return false;
  return true;
}

// Work groups that keep their weights over several rows, and partial rows of the backward pass: more of them hide more of the memory's
// time, fewer load and add less.  Both ways, us for 8192 x 768 with blocks / 1000 x 1021 / 16384 x 4096 bfloat16: 30.3 / 20.0 / 139.0; with 512
// work groups forward and 256 partial rows 31.1 / 19.6 / 146.9, with 4096 and 768 31.3 / 19.0 / 142.9, with 1024 and 1024 30.4 / 19.6 / 149.1.
constexpr int kLnForwardBlocks = 1024;
constexpr int kLnMostChunks = 512;

// Work groups (of 512 threads) of the backward pass, one partial row each: what the registers of its accumulators let run at once, 256 with
// the five sums of the blocks (with 512: 34.9 us both ways at 8192 x 768, with 256 30.3).
static int64_t ln_backward_blocks(int64_t rows, int64_t F, bool blocks) {
  int groups = 0;
  if (!ln_layout<false>(F, [&](auto lanes, auto) { groups = 512 / decltype(lanes)::value; })) {
    const int64_t per = (rows + kLnMostChunks - 1) / kLnMostChunks;          // chunks of 16 rows at least
    return (rows + (per < 16 ? 16 : per) - 1) / (per < 16 ? 16 : per);
  }
  const int64_t need = (rows + groups - 1) / groups, most = blocks ? 256 : kLnMostChunks;
  return need < most ? need : most;
}

}  // namespace ak

extern "C" int ak_layer_norm(const void* x, int x_dtype, int64_t ldx, const void* weight, const void* bias, int w_dtype, int64_t rows,
                             int64_t F, float eps, void* y, int y_dtype, int64_t ldy, float* mean, float* rstd, ak_stream_t stream) {
  using namespace ak;
  if (rows < 0 || F <= 0 || ldx < F || ldy < F || !(eps >= 0.f) || !is_element_type(x_dtype) || (y_dtype != x_dtype && y_dtype != AK_F32) ||
      (w_dtype != x_dtype && w_dtype != AK_F32))
    return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (x == nullptr || y == nullptr || mean == nullptr || rstd == nullptr) return AK_ERR_ARG;
  if (rows > 0x7fffffff || F > (1 << 30)) return AK_ERR_UNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const LnForward p{x, weight, bias, y, mean, rstd, ldx, ldy, rows, F, eps};
  return with_type(x_dtype, [&](auto xt) {
    using X = typename decltype(xt)::type;
    auto launch = [&](auto yt, auto wt) {
      using Y = typename decltype(yt)::type;
      using W = typename decltype(wt)::type;
      const bool held = ln_layout<true>(F, [&](auto lanes, auto elements) {
        constexpr int L = decltype(lanes)::value, V = decltype(elements)::value * static_cast<int>(sizeof(X)) / 16;
        constexpr int threads = L > 256 ? L : 256;
        const int64_t need = (rows + threads / L - 1) / (threads / L);
        hipLaunchKernelGGL((ln_forward_rows_kernel<X, Y, W, L, V, threads>), dim3(static_cast<unsigned>(need < kLnForwardBlocks ? need : kLnForwardBlocks)),
                           dim3(threads), 0, s, p);
      });
      if (!held) hipLaunchKernelGGL((ln_forward_kernel<X, Y, W>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
    };
    if (y_dtype == x_dtype) w_dtype == x_dtype ? launch(Type<X>{}, Type<X>{}) : launch(Type<X>{}, Type<float>{});
    else w_dtype == x_dtype ? launch(Type<float>{}, Type<X>{}) : launch(Type<float>{}, Type<float>{});
    return check_launch();
  });
}

extern "C" size_t ak_layer_norm_backward_ws_bytes(int64_t rows, int64_t F, int with_blocks) {
  if (rows <= 0 || F <= 0) return 0;
  return static_cast<size_t>(ak::ln_backward_blocks(rows, F, with_blocks != 0)) * F * (with_blocks ? 5 : 2) * sizeof(float);
}

extern "C" int ak_layer_norm_backward(const void* g, int g_dtype, int64_t ldg, const void* x, int x_dtype, int64_t ldx, const float* mean,
                                      const float* rstd, const void* weight, int w_dtype, int64_t rows, int64_t F, void* dx, int64_t lddx,
                                      void* dw, void* db, float* blocks, float alpha, float beta, void* ws, size_t ws_bytes,
                                      ak_stream_t stream) {
  using namespace ak;
  if (rows < 0 || F <= 0 || ldg < F || ldx < F || (dx != nullptr && lddx < F) || !is_element_type(x_dtype) ||
      (g_dtype != x_dtype && g_dtype != AK_F32) || (w_dtype != x_dtype && w_dtype != AK_F32))
    return AK_ERR_ARG;
  if (rows > 0 && (g == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)) return AK_ERR_ARG;
  if (rows > 0x7fffffff || F > (1 << 30)) return AK_ERR_UNSUPPORTED;
  const int sums = blocks != nullptr ? 5 : dw != nullptr || db != nullptr ? 2 : 0;
  if (sums > 0 && rows > 0 && (ws == nullptr || ws_bytes < ak_layer_norm_backward_ws_bytes(rows, F, blocks != nullptr))) return AK_ERR_WORKSPACE;
  if (sums > 0 && F > (1 << 24)) return AK_ERR_UNSUPPORTED;         // (a launch's threads are counted in 32 bits)
  if (sums == 0 && (dx == nullptr || rows == 0)) return AK_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(ws);
  const int64_t chunks = rows > 0 ? ln_backward_blocks(rows, F, blocks != nullptr) : 0;
  if (rows > 0) {
    const LnBackward p{g, x, mean, rstd, weight, dx, part, ldg, ldx, lddx, rows, F, (rows + chunks - 1) / chunks};
    const int rc = with_type(x_dtype, [&](auto xt) {
      using X = typename decltype(xt)::type;
      auto launch = [&](auto gt, auto wt) {
        using G = typename decltype(gt)::type;
        using W = typename decltype(wt)::type;
        const dim3 grid(static_cast<unsigned>(chunks));
        const bool held = ln_layout<false>(F, [&](auto lanes, auto elements) {
          constexpr int L = decltype(lanes)::value, V = decltype(elements)::value * static_cast<int>(sizeof(X)) / 16;
          if (sums == 5) hipLaunchKernelGGL((ln_backward_fused_kernel<X, G, W, L, V, 512, 5>), grid, dim3(512), 0, s, p);
          else if (sums == 2) hipLaunchKernelGGL((ln_backward_fused_kernel<X, G, W, L, V, 512, 2>), grid, dim3(512), 0, s, p);
          else hipLaunchKernelGGL((ln_backward_fused_kernel<X, G, W, L, V, 512, 0>), grid, dim3(512), 0, s, p);
        });
        if (held) return;
        if (dx != nullptr) hipLaunchKernelGGL((ln_backward_rows_kernel<X, G, W>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
        const dim3 columns(static_cast<unsigned>((F + 255) / 256), static_cast<unsigned>(chunks));
        if (sums == 5) hipLaunchKernelGGL((ln_backward_columns_kernel<X, G, true>), columns, dim3(256), 0, s, p);
        else if (sums == 2) hipLaunchKernelGGL((ln_backward_columns_kernel<X, G, false>), columns, dim3(256), 0, s, p);
      };
      if (g_dtype == x_dtype) w_dtype == x_dtype ? launch(Type<X>{}, Type<X>{}) : launch(Type<X>{}, Type<float>{});
      else w_dtype == x_dtype ? launch(Type<float>{}, Type<X>{}) : launch(Type<float>{}, Type<float>{});
      return check_launch();
    });
    if (rc != AK_OK) return rc;
  }
  if (sums == 0) return AK_OK;
  return with_type(w_dtype, [&](auto wt) {
    using W = typename decltype(wt)::type;
    hipLaunchKernelGGL(ln_backward_finish_kernel<W>, dim3(static_cast<unsigned>((F * sums + 31) / 32)), dim3(1024), 0, s, part, chunks, F, sums,
                       static_cast<W*>(dw), static_cast<W*>(db), blocks, alpha, beta);
    return check_launch();
  });
}
