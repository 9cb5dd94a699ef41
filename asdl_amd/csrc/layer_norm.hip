// Layer norm over the last axis, its backward pass, and the unit-wise Fisher blocks of its weight and bias.
//   forward:  m = mean x, r = (mean (x - m)^2 + eps)^(-1/2), h = (x - m) r, y = h w + b;  m and r are kept for the way back
//   backward: dx = r (g w - mean(g w) - h mean(g w h)),  dw = sum_rows g h,  db = sum_rows g,
//             blocks[f] = beta blocks[f] + alpha sum_rows [[(g h)^2, g^2 h], [g^2 h, g^2]]
// The mean of what is left after the first mean is taken off corrects it by what its sum had rounded away (rows of equal values give
// h = 0 whatever their size), and the variance is the mean of centred squares, no difference of large sums.  Everything is fp32,
// rounded when it is stored.
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
  int w_dtype;
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
  int w_dtype;
};

// One work group per row, the row read four times.
template <typename X, typename Y>
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
    if (p.w != nullptr) v *= load_as_float(p.w, p.w_dtype, f);
    if (p.b != nullptr) v += load_as_float(p.b, p.w_dtype, f);
    y[f] = static_cast<Y>(v);
  }
  if (threadIdx.x == 0) {
    p.mean[row] = m;
    p.rstd[row] = r;
  }
}

template <typename X, typename G>
static __global__ __launch_bounds__(256) void ln_backward_rows_kernel(LnBackward p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const X* __restrict__ x = static_cast<const X*>(p.x) + row * p.ldx;
  const G* __restrict__ g = static_cast<const G*>(p.g) + row * p.ldg;
  X* __restrict__ dx = static_cast<X*>(p.dx) + row * p.lddx;
  const float n = static_cast<float>(p.F), m = p.mean[row], r = p.rstd[row];
  float s = 0.f, t = 0.f;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    const float gw = static_cast<float>(g[f]) * (p.w != nullptr ? load_as_float(p.w, p.w_dtype, f) : 1.f);
    s += gw;
    t += gw * ((static_cast<float>(x[f]) - m) * r);
  }
  s = group_sum<4>(s, red) / n;
  t = group_sum<4>(t, red) / n;
  for (int64_t f = threadIdx.x; f < p.F; f += 256) {
    const float gw = static_cast<float>(g[f]) * (p.w != nullptr ? load_as_float(p.w, p.w_dtype, f) : 1.f);
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

// Sums of the chunks, in a fixed order.  64 columns x 16 lanes of chunks a work group.
static __global__ __launch_bounds__(1024) void ln_backward_finish_kernel(const float* __restrict__ part, int64_t chunks, int64_t F, int sums,
                                                                         void* dw, void* db, int w_dtype, float* blocks, float alpha, float beta) {
  __shared__ float red[5][16][64];
  const int fl = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * 64 + fl;
  for (int q = 0; q < sums; ++q) {
    float s = 0.f;
    if (f < F)
      for (int64_t c = lane; c < chunks; c += 16) s += part[(c * sums + q) * F + f];
    red[q][lane][fl] = s;
  }
  __syncthreads();
  if (lane >= sums || f >= F) return;
  float total = 0.f;
#pragma unroll
  for (int l = 0; l < 16; ++l) total += red[lane][l][fl];
  if (lane == 0) {
    if (dw != nullptr) store_from_float(dw, w_dtype, f, total);
  } else if (lane == 1) {
    if (db != nullptr) store_from_float(db, w_dtype, f, total);
  } else {
    float* out = blocks + 4 * f + (lane == 2 ? 0 : lane == 3 ? 1 : 3);
    out[0] = alpha * total + (beta != 0.f ? beta * out[0] : 0.f);
    if (lane == 3) out[1] = alpha * total + (beta != 0.f ? beta * out[1] : 0.f);
  }
}

constexpr int64_t kLnMostChunks = 256;

static int64_t ln_rows_per_chunk(int64_t rows) {
  const int64_t per = (rows + kLnMostChunks - 1) / kLnMostChunks;
  return per < 16 ? 16 : per;
}

static int64_t ln_chunks(int64_t rows) {
  const int64_t per = ln_rows_per_chunk(rows);
  return (rows + per - 1) / per;
}

}  // namespace ak

extern "C" int ak_layer_norm(const void* x, int x_dtype, int64_t ldx, const void* weight, const void* bias, int w_dtype, int64_t rows,
                             int64_t F, float eps, void* y, int y_dtype, int64_t ldy, float* mean, float* rstd, ak_stream_t stream) {
  using namespace ak;
  if (rows < 0 || F <= 0 || ldx < F || ldy < F || !(eps >= 0.f) || !is_element_type(x_dtype) || (y_dtype != x_dtype && y_dtype != AK_F32) ||
      !is_element_type(w_dtype))
    return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (x == nullptr || y == nullptr || mean == nullptr || rstd == nullptr) return AK_ERR_ARG;
  if (rows > 0x7fffffff || F > (1 << 30)) return AK_ERR_UNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const LnForward p{x, weight, bias, y, mean, rstd, ldx, ldy, rows, F, w_dtype, eps};
  return with_type(x_dtype, [&](auto xt) {
    using X = typename decltype(xt)::type;
    if (y_dtype == x_dtype) hipLaunchKernelGGL((ln_forward_kernel<X, X>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((ln_forward_kernel<X, float>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
    return check_launch();
  });
}

extern "C" size_t ak_layer_norm_backward_ws_bytes(int64_t rows, int64_t F, int with_blocks) {
  if (rows <= 0 || F <= 0) return 0;
  return static_cast<size_t>(ak::ln_chunks(rows)) * F * (with_blocks ? 5 : 2) * sizeof(float);
}

extern "C" int ak_layer_norm_backward(const void* g, int g_dtype, int64_t ldg, const void* x, int x_dtype, int64_t ldx, const float* mean,
                                      const float* rstd, const void* weight, int w_dtype, int64_t rows, int64_t F, void* dx, int64_t lddx,
                                      void* dw, void* db, float* blocks, float alpha, float beta, void* ws, size_t ws_bytes,
                                      ak_stream_t stream) {
  using namespace ak;
  if (rows < 0 || F <= 0 || ldg < F || ldx < F || (dx != nullptr && lddx < F) || !is_element_type(x_dtype) ||
      (g_dtype != x_dtype && g_dtype != AK_F32) || !is_element_type(w_dtype))
    return AK_ERR_ARG;
  if (rows > 0 && (g == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)) return AK_ERR_ARG;
  if (rows > 0x7fffffff || F > (1 << 30)) return AK_ERR_UNSUPPORTED;
  const bool sums = dw != nullptr || db != nullptr || blocks != nullptr;
  if (sums && rows > 0 && (ws == nullptr || ws_bytes < ak_layer_norm_backward_ws_bytes(rows, F, blocks != nullptr))) return AK_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(ws);
  const int64_t chunks = rows > 0 ? ln_chunks(rows) : 0;
  if (rows > 0) {
    const LnBackward p{g, x, mean, rstd, weight, dx, part, ldg, ldx, lddx, rows, F, ln_rows_per_chunk(rows), w_dtype};
    const int rc = with_type(x_dtype, [&](auto xt) {
      using X = typename decltype(xt)::type;
      auto launch = [&](auto gt) {
        using G = typename decltype(gt)::type;
        if (dx != nullptr) hipLaunchKernelGGL((ln_backward_rows_kernel<X, G>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, p);
        const dim3 grid(static_cast<unsigned>((F + 255) / 256), static_cast<unsigned>(chunks));
        if (blocks != nullptr) hipLaunchKernelGGL((ln_backward_columns_kernel<X, G, true>), grid, dim3(256), 0, s, p);
        else if (sums) hipLaunchKernelGGL((ln_backward_columns_kernel<X, G, false>), grid, dim3(256), 0, s, p);
      };
      if (g_dtype == x_dtype) launch(Type<X>{});
      else launch(Type<float>{});
      return check_launch();
    });
    if (rc != AK_OK) return rc;
  }
  if (sums)
    hipLaunchKernelGGL(ln_backward_finish_kernel, dim3(static_cast<unsigned>((F + 63) / 64)), dim3(1024), 0, s, part, chunks, F,
                       blocks != nullptr ? 5 : 2, dw, db, w_dtype, blocks, alpha, beta);
  return check_launch();
}
