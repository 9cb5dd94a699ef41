// Sums of the columns of a matrix of any element type in fp32, in two launches whose order of additions is fixed: chunks of rows, then
// the chunks.  Bound by the memory: the matrix is read once.
#pragma once
#include "elements.hpp"

namespace ak {

constexpr int kColumnsPerGroup = 256, kColumnChunks = 64;

// A work group's chunk of 256 columns: a thread has eight columns and every eighth row of it.
template <typename T>
__device__ __forceinline__ void column_chunk(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t cols, int64_t rows_per_chunk,
                                             float* __restrict__ part, int64_t group, int64_t chunk, float (*joined)[kColumnsPerGroup]) {
  const int lane = threadIdx.x & 31, row_of = threadIdx.x >> 5;
  const int64_t c = group * kColumnsPerGroup + 8 * lane;
  const int64_t r0 = chunk * rows_per_chunk, r1 = r0 + rows_per_chunk < rows ? r0 + rows_per_chunk : rows;
  float s[8] = {};
  if (c + 8 <= cols) {
#pragma unroll 4
    for (int64_t r = r0 + row_of; r < r1; r += 8) {
      Some<T, 8> v;
      v.load(x + r * ld + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += v.get(e);
    }
  } else {
    for (int64_t r = r0 + row_of; r < r1; r += 8)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) s[e] += static_cast<float>(x[r * ld + c + e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) joined[row_of][8 * lane + e] = s[e];
  __syncthreads();
  const int64_t col = group * kColumnsPerGroup + threadIdx.x;
  if (col >= cols) return;
  float t = joined[0][threadIdx.x];
#pragma unroll
  for (int k = 1; k < 8; ++k) t += joined[k][threadIdx.x];
  part[chunk * cols + col] = t;
}

// grid (columns / 256, chunks, pieces); the last piece's chunks are the first.
template <typename T>
static __global__ __launch_bounds__(256) void column_chunks_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                                   int64_t rows_per_chunk, int64_t pitch, float* __restrict__ part) {
  __shared__ float joined[8][kColumnsPerGroup];
  column_chunk(x + (gridDim.z - 1 - blockIdx.z) * pitch, ld, rows, cols, rows_per_chunk, part + static_cast<int64_t>(blockIdx.z) * gridDim.y * cols, blockIdx.x,
               blockIdx.y, joined);
}

template <typename T>
__device__ __forceinline__ void column_total(const float* __restrict__ part, int64_t cols, int chunks, float scale, const float* __restrict__ factor,
                                             T* __restrict__ out, int64_t group) {
  const int64_t c = group * 256 + threadIdx.x;
  if (c >= cols) return;
  float t = 0.f;
#pragma unroll 8
  for (int k = 0; k < chunks; ++k) t += part[k * cols + c];
  out[c] = static_cast<T>(t * (factor != nullptr ? scale * *factor : scale));
}

template <typename T>
static __global__ __launch_bounds__(256) void column_total_kernel(const float* __restrict__ part, int64_t cols, int chunks, float scale,
                                                                  const float* __restrict__ factor, T* __restrict__ out) {
  column_total(part, cols, chunks, scale, factor, out, blockIdx.x);
}

inline int column_chunks(int64_t rows) {
  const int64_t c = (rows + 63) / 64;
  return static_cast<int>(c < 1 ? 1 : c > kColumnChunks ? kColumnChunks : c);
}

inline size_t column_sums_ws_bytes(int64_t rows, int64_t cols) { return static_cast<size_t>(column_chunks(rows)) * cols * sizeof(float); }

// out[c] = scale * factor * sum over rows and pieces of x[r][piece * pitch + c]; `part`: column_sums_ws_bytes of pieces * cols columns
template <typename T, typename O>
inline int column_sums(const T* x, int64_t ld, int64_t rows, int64_t cols, float scale, const float* factor, O* out, float* part, hipStream_t s, int pieces = 1,
                       int64_t pitch = 0) {
  if (cols <= 0) return AK_OK;
  if (cols > (1ll << 30)) return AK_ERR_TOO_LARGE;
  const int chunks = column_chunks(rows);
  const int64_t per = (rows + chunks - 1) / chunks;
  const unsigned groups = static_cast<unsigned>((cols + 255) / 256);
  hipLaunchKernelGGL(column_chunks_kernel<T>, dim3(groups, static_cast<unsigned>(chunks), static_cast<unsigned>(pieces)), dim3(256), 0, s, x, ld, rows, cols,
                     per, pitch, part);
  hipLaunchKernelGGL(column_total_kernel<O>, dim3(groups), dim3(256), 0, s, part, cols, pieces * chunks, scale, factor, out);
  return check_launch();
}

}  // namespace ak
