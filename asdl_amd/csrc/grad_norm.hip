// The norm of many tensors as one vector, and copies of them (or themselves) scaled down to a largest norm.
//   n = (sum x^2)^(1/2), sum |x| or max |x| over all elements;  c = min(1, max_norm / (n + 1e-6));  out = c x
// Sums are double: no square of an fp32 value overflows or vanishes there, and 2^53 of them lose nothing that a float holds.  Every
// launch has its tensors' addresses in the kernel arguments: nothing is uploaded, so a captured graph needs no memory of the host.
// Partial sums are added in a fixed order by every work group that needs the norm; no atomics.
// Bound by the memory: the norm reads all elements once, clipping reads them again and writes them.  1.26 GB of fp32 gradients: 209 us the
// norm (6.0 TB/s, part of it from the 256 MB cache), 690 us with clipped copies (5.5 TB/s for two reads and a write: the second read is not
// to be had for less where the gradients do not fit the cache); 105 MB: 21 and 52 us; a few small tensors: 9 us, two launches.
#include "elements.hpp"

namespace ak {

// Measured for 1.26 GB / 105 MB / 2.7 MB, norm and clipped copies: 209, 690 / 20.8, 52.5 / 9.3, 9.4 us.  One load ahead: 221, 706 / 23.5, 54.8 /
// 10.7, 12.9; eight: 206, 695 / 21.6, 52.4 / 11.4, 11.2.  Chunks of 4096: 211, 688 / 21.8, 53.2 / 10.5, 12.4; of 65536: 209, 700 / 20.9, 50.9 /
// 10.2, 14.5.  2048 work groups: 213, 694 / 23.1, 53.0 / 10.3, 11.1.
constexpr int kGnThreads = 256;
constexpr int kGnBlocks = 1024;            // work groups of all norm launches of a call: so many partial sums
constexpr int64_t kGnChunk = 16384;        // elements
constexpr int kGnAhead = 4;                // 16-byte loads a thread has on their way
constexpr int kGnNormTensors = 180, kGnClipTensors = 130;      // whose tables fit 4 KB of kernel arguments

struct GnNormTable {
  const void* src[kGnNormTensors];
  int64_t size[kGnNormTensors];            // elements * 4 + type of the source
  int first[kGnNormTensors];               // chunks of the tensors before
  int count, chunks;
};

struct GnClipTable {
  const void* src[kGnClipTensors];
  void* dst[kGnClipTensors];
  int64_t size[kGnClipTensors];            // elements * 16 + type of the result * 4 + type of the source
  int first[kGnClipTensors];
  int count, chunks;
};
static_assert(sizeof(GnNormTable) + 64 <= 4096 && sizeof(GnClipTable) + 64 <= 4096, "kernel arguments");

// The tensor that a chunk belongs to: the last one whose first chunk is not behind it.
template <typename Table>
__device__ __forceinline__ int gn_find(const Table& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Types in the tables: 0 fp32, 1 bf16, 2 fp16.  fn(Type<T>{}), the same for all lanes.
template <typename Fn>
__device__ __forceinline__ void gn_with_type(int type, Fn&& fn) {
  if (type == 0) fn(Type<float>{});
  else if (type == 1) fn(Type<__bf16>{});
  else fn(Type<_Float16>{});
}

// KIND 0: sum x^2, 1: sum |x|, 2: max |x| (as the bits of a float's magnitude: NaN is above all numbers)
template <int KIND>
__device__ __forceinline__ double gn_join(double a, double b) {
  if constexpr (KIND < 2) return a + b;
  return a != a || a > b ? a : b;
}

template <int KIND>
__device__ __forceinline__ double gn_take(double a, float x) {
  if constexpr (KIND == 0) return fma(static_cast<double>(x), static_cast<double>(x), a);
  if constexpr (KIND == 1) return a + fabs(static_cast<double>(x));
  return gn_join<2>(fabs(static_cast<double>(x)), a);
}

template <int KIND>
__device__ __forceinline__ double gn_group(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = gn_join<KIND>(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kGnThreads / 64; ++w) v = gn_join<KIND>(v, red[w]);
  return v;
}

template <int KIND>
static __global__ __launch_bounds__(kGnThreads) void gn_partial_kernel(GnNormTable t, double* __restrict__ part) {
  __shared__ double red[kGnThreads / 64];
  double acc = 0.;
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int i = gn_find(t, chunk);
    const int64_t n = t.size[i] >> 2, from = (chunk - t.first[i]) * kGnChunk, to = from + kGnChunk < n ? from + kGnChunk : n;
    const int type = static_cast<int>(t.size[i] & 3);
    gn_with_type(type, [&](auto xt) {
      using X = typename decltype(xt)::type;
      constexpr int E = 16 / sizeof(X), STEP = kGnThreads * E;
      const X* __restrict__ x = static_cast<const X*>(t.src[i]) + from;
      const int count = static_cast<int>(to - from), mine = static_cast<int>(threadIdx.x) * E;
      int at = mine;
      for (; at + (kGnAhead - 1) * STEP + E <= count; at += kGnAhead * STEP) {
        Some<X, E> some[kGnAhead];
#pragma unroll
        for (int a = 0; a < kGnAhead; ++a) some[a].load(x + at + a * STEP);
#pragma unroll
        for (int a = 0; a < kGnAhead; ++a)
#pragma unroll
          for (int e = 0; e < E; ++e) acc = gn_take<KIND>(acc, some[a].get(e));
      }
      for (; at < count; at += STEP)
        for (int e = at; e < at + E && e < count; ++e) acc = gn_take<KIND>(acc, static_cast<float>(x[e]));
    });
  }
  acc = gn_group<KIND>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int KIND>
__device__ __forceinline__ double gn_norm(const double* __restrict__ part, int parts, double* red) {
  double v = 0.;
  for (int i = threadIdx.x; i < parts; i += kGnThreads) v = gn_join<KIND>(v, part[i]);
  v = gn_group<KIND>(v, red);
  return KIND == 0 ? sqrt(v) : v;
}

template <int KIND>
static __global__ __launch_bounds__(kGnThreads) void gn_finish_kernel(const double* __restrict__ part, int parts, float* norm) {
  __shared__ double red[kGnThreads / 64];
  const double n = gn_norm<KIND>(part, parts, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

template <int KIND>
static __global__ __launch_bounds__(kGnThreads) void gn_clip_kernel(GnClipTable t, const double* __restrict__ part, int parts, double max_norm,
                                                                    float* norm) {
  __shared__ double red[kGnThreads / 64];
  const double n = gn_norm<KIND>(part, parts, red);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const double most = max_norm / (n + 1e-6);
  const float c = static_cast<float>(most > 1. ? 1. : most);           // (NaN stays)
  // (from the end, which the pass before has read last and the caches may hold: 690 us for 696 from the start)
  for (int chunk = t.chunks - 1 - static_cast<int>(blockIdx.x); chunk >= 0; chunk -= gridDim.x) {
    const int i = gn_find(t, chunk);
    if (c == 1.f && t.src[i] == t.dst[i]) continue;
    const int64_t n_el = t.size[i] >> 4, from = (chunk - t.first[i]) * kGnChunk, to = from + kGnChunk < n_el ? from + kGnChunk : n_el;
    const int type = static_cast<int>(t.size[i] & 3), to_type = static_cast<int>(t.size[i] >> 2 & 3);
    gn_with_type(type, [&](auto xt) {
      using X = typename decltype(xt)::type;
      auto scale = [&](auto yt) {
        using Y = typename decltype(yt)::type;
        constexpr int E = 16 / sizeof(X), STEP = kGnThreads * E;
        const X* x = static_cast<const X*>(t.src[i]) + from;         // (may be y)
        Y* y = static_cast<Y*>(t.dst[i]) + from;
        const int count = static_cast<int>(to - from);
        int at = static_cast<int>(threadIdx.x) * E;
        for (; at + (kGnAhead - 1) * STEP + E <= count; at += kGnAhead * STEP) {
          Some<X, E> some[kGnAhead];
#pragma unroll
          for (int a = 0; a < kGnAhead; ++a) some[a].load(x + at + a * STEP);
#pragma unroll
          for (int a = 0; a < kGnAhead; ++a) {
            Some<Y, E> out;
#pragma unroll
            for (int e = 0; e < E; ++e) out.set(e, c * some[a].get(e));
            out.store(y + at + a * STEP);
          }
        }
        for (; at < count; at += STEP)
          for (int e = at; e < at + E && e < count; ++e) y[e] = static_cast<Y>(c * static_cast<float>(x[e]));
      };
      if (to_type == type) scale(Type<X>{});
      else scale(Type<float>{});
    });
  }
}

static int gn_type(int dtype) { return dtype == AK_F32 ? 0 : dtype == AK_BF16 ? 1 : 2; }

static int64_t gn_chunks(int64_t n) { return (n + kGnChunk - 1) / kGnChunk; }

// Every launch of the partial sums gets its share of kGnBlocks work groups by its chunks, and one at least.
static int gn_blocks(int64_t chunks, int64_t all) {
  const int64_t share = all <= kGnBlocks ? chunks : (chunks * kGnBlocks + all - 1) / all;
  return static_cast<int>(share < 1 ? 1 : share > chunks ? chunks : share);
}

static int gn_check(const int64_t* items, int count, int kind, bool clip) {
  if (items == nullptr && count > 0) return AK_ERR_ARG;
  if (count < 0 || kind < 0 || kind > 2) return AK_ERR_ARG;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t* r = items + 5 * static_cast<int64_t>(i);
    if (r[2] < 0 || !is_element_type(static_cast<int>(r[3])) || (r[2] > 0 && r[0] == 0)) return AK_ERR_ARG;
    if (clip && ((r[2] > 0 && r[1] == 0) || (r[4] != r[3] && r[4] != AK_F32))) return AK_ERR_ARG;
    if (r[2] > (1ll << 45)) return AK_ERR_TOO_LARGE;
    chunks += gn_chunks(r[2]);
  }
  return chunks > 0x3fffffff ? AK_ERR_TOO_LARGE : AK_OK;
}

// fn(first item, one behind the last, their chunks) for runs of at most `most` tensors that are not empty
template <typename Fn>
static void gn_runs(const int64_t* items, int count, int most, Fn&& fn) {
  int from = 0;
  while (from < count) {
    int to = from, held = 0;
    int64_t chunks = 0;
    for (; to < count; ++to) {
      const int64_t n = items[5 * static_cast<int64_t>(to) + 2];
      if (n == 0) continue;
      if (held == most) break;
      ++held;
      chunks += gn_chunks(n);
    }
    if (held > 0) fn(from, to, chunks);
    from = to;
  }
}

template <int KIND>
static int gn_run(const int64_t* items, int count, bool clip, double max_norm, float* norm, double* part, hipStream_t s) {
  int64_t all = 0;
  for (int i = 0; i < count; ++i) all += gn_chunks(items[5 * static_cast<int64_t>(i) + 2]);
  int parts = 0;
  gn_runs(items, count, kGnNormTensors, [&](int from, int to, int64_t chunks) {
    GnNormTable t;
    t.count = 0;
    t.chunks = 0;
    for (int i = from; i < to; ++i) {
      const int64_t* r = items + 5 * static_cast<int64_t>(i);
      if (r[2] == 0) continue;
      t.src[t.count] = reinterpret_cast<const void*>(r[0]);
      t.size[t.count] = r[2] * 4 + gn_type(static_cast<int>(r[3]));
      t.first[t.count++] = t.chunks;
      t.chunks += static_cast<int>(gn_chunks(r[2]));
    }
    const int blocks = gn_blocks(chunks, all);
    hipLaunchKernelGGL(gn_partial_kernel<KIND>, dim3(blocks), dim3(kGnThreads), 0, s, t, part + parts);
    parts += blocks;
  });
  bool first = true;
  if (clip) {
    gn_runs(items, count, kGnClipTensors, [&](int from, int to, int64_t chunks) {
      GnClipTable t;
      t.count = 0;
      t.chunks = 0;
      for (int i = from; i < to; ++i) {
        const int64_t* r = items + 5 * static_cast<int64_t>(i);
        if (r[2] == 0) continue;
        t.src[t.count] = reinterpret_cast<const void*>(r[0]);
        t.dst[t.count] = reinterpret_cast<void*>(r[1]);
        t.size[t.count] = r[2] * 16 + gn_type(static_cast<int>(r[4])) * 4 + gn_type(static_cast<int>(r[3]));
        t.first[t.count++] = t.chunks;
        t.chunks += static_cast<int>(gn_chunks(r[2]));
      }
      const int blocks = static_cast<int>(chunks < 4 * kGnBlocks ? chunks : 4 * kGnBlocks);
      hipLaunchKernelGGL(gn_clip_kernel<KIND>, dim3(blocks), dim3(kGnThreads), 0, s, t, part, parts, max_norm, first ? norm : nullptr);
      first = false;
    });
  }
  if (first) hipLaunchKernelGGL(gn_finish_kernel<KIND>, dim3(1), dim3(kGnThreads), 0, s, part, parts, norm);
  return check_launch();
}

}  // namespace ak

extern "C" size_t ak_grad_norm_ws_bytes(int count) {
  return count < 0 ? 0 : (ak::kGnBlocks + static_cast<size_t>(count) / ak::kGnNormTensors + 1) * 2 * sizeof(double);
}

static int ak_grad_norm_checked(const int64_t* items, int count, int kind, bool clip, double max_norm, float* norm, void* ws, size_t ws_bytes,
                                ak_stream_t stream) {
  const int rc = ak::gn_check(items, count, kind, clip);
  if (rc != AK_OK) return rc;
  if (norm == nullptr) return AK_ERR_ARG;
  if (ws == nullptr || ws_bytes < ak_grad_norm_ws_bytes(count)) return AK_ERR_WORKSPACE;
  double* part = static_cast<double*>(ws);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (kind == 0) return ak::gn_run<0>(items, count, clip, max_norm, norm, part, s);
  if (kind == 1) return ak::gn_run<1>(items, count, clip, max_norm, norm, part, s);
  return ak::gn_run<2>(items, count, clip, max_norm, norm, part, s);
}

extern "C" int ak_grad_norm(const int64_t* items, int count, int kind, float* norm, void* ws, size_t ws_bytes, ak_stream_t stream) {
  return ak_grad_norm_checked(items, count, kind, false, 0., norm, ws, ws_bytes, stream);
}

extern "C" int ak_clip_grad_norm(const int64_t* items, int count, int kind, double max_norm, float* norm, void* ws, size_t ws_bytes,
                                 ak_stream_t stream) {
  if (!(max_norm >= 0.)) return AK_ERR_ARG;
  return ak_grad_norm_checked(items, count, kind, true, max_norm, norm, ws, ws_bytes, stream);
}
