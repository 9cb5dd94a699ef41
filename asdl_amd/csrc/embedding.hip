// Rows of a table by token, times a factor, and the gradient of the table:
//   y_n = c E[t(n)],   dE[v] = beta dE[v] + c * (sum of g_n over n with t(n) = v, in ascending order of n)
// The gradient goes by tokens in sorted order, so that every row of it is written once and no addition depends on the order in which work
// groups run (atomics on the 3 KB rows of a frequent token would also wait for each other: a twentieth of a text is its commonest token).
//   sort:   a work group per range of rows reads all tokens, counts those in front of its range and those of each row, and puts the
//           positions of its own in order: a stable counting sort without a word between work groups, one launch.  Of more tokens than
//           kEmbScan that costs more than two further launches, which bring the tokens into ranges first (131072 tokens: 116 -> 36 us)
//   sums:   a wave per chunk of sorted positions and 1 KB of columns; runs of equal tokens inside a chunk are written, parts of runs that
//           cross its ends go to the workspace; other waves write the rows that no token names
//   joins:  the parts of a run, in order
// Bound by the memory: the gradients are read once, the table's gradient is written once (131072 tokens of 131072 x 1024 bf16: lookup 80 to 87 us,
// sort 34, sums 127, 4.2 TB/s, joins 13), few tokens by the launches (4.5 us each).
#include <algorithm>
#include "elements.hpp"

namespace ak {

constexpr int kEmbBins = 1024, kEmbWaves = 16;        // keys of a sorting work group at most, its waves
constexpr int64_t kEmbScan = 16384;
constexpr int kEmbChunk = 4096;                      // tokens of a chunk
#define AK_LDS __attribute__((address_space(3)))

template <typename I>
struct Tokens {
  const I* p;
  int64_t count;
  int rows;
  int64_t padding;         // a token that takes no gradient; -1: none
  __device__ __forceinline__ int64_t at(int64_t n) const { return static_cast<int64_t>(p[n]); }
  // (positions behind the last, tokens that name no row and the padding: -1)
  __device__ __forceinline__ int named(int64_t n) const {
    if (n >= count) return -1;
    const int64_t t = at(n);
    return t >= 0 && t < rows && t != padding ? static_cast<int>(t) : -1;
  }
};

// L lanes copy a row, V elements (16 bytes) at a time.
template <typename T, typename O, typename I, int L>
static __global__ __launch_bounds__(256) void emb_rows_kernel(Tokens<I> t, const T* __restrict__ table, int64_t ld, int D, float scale, O* __restrict__ out) {
  constexpr int V = 16 / sizeof(T);
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (n >= t.count) return;
  const int64_t token = t.at(n);
  O* __restrict__ to = out + n * D;
  if (token < 0 || token >= t.rows) {
    for (int c = threadIdx.x % L; c < D; c += L) to[c] = static_cast<O>(NAN);
    return;
  }
  const T* __restrict__ from = table + token * ld;
  const int whole = D / V * V;
#pragma unroll 4
  for (int c = (threadIdx.x % L) * V; c < whole; c += L * V) {
    Some<T, V> v;
    Some<O, V> o;
    v.load(from + c);
#pragma unroll
    for (int e = 0; e < V; ++e) o.set(e, v.get(e) * scale);
    o.store(to + c);
  }
  const int c = whole + threadIdx.x % L;
  if (c < D && threadIdx.x % L < V) to[c] = static_cast<O>(static_cast<float>(from[c]) * scale);
}

// What a sorting work group goes through and where it puts it.  A key below 0 is not its own.
//   ALL     the text; keys are the rows of its range (one launch: every work group reads the whole text)
//   CHUNK   its chunk of the text; keys are the ranges of rows
//   RANGE   what CHUNK has put into its range; keys are the rows of it
enum EmbSort { kSortAll, kSortChunk, kSortRange };

template <typename I>
struct EmbSorted {
  Tokens<I> t;
  int bins, ranges, chunk, chunks;       // rows of a range, tokens of a chunk
  int* counts;                           // [chunk][range]
  int* firsts;                           // first sorted position of each range, and behind the last
  int *token, *place;                    // tokens and their positions by range
  int *starts, *order, *sorted;          // first sorted position of each row's tokens; position in the text and token of each
};

// Tokens of each range in a chunk.
template <typename I>
static __global__ __launch_bounds__(1024) void emb_count_kernel(EmbSorted<I> p) {
  __shared__ int count[kEmbBins];
  for (int i = threadIdx.x; i < kEmbBins; i += 1024) count[i] = 0;
  __syncthreads();
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * p.chunk;
  for (int i = threadIdx.x; i < p.chunk; i += 1024) {
    const int v = p.t.named(n0 + i);
    if (v >= 0) atomicAdd(&count[v / p.bins], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.ranges; i += 1024) p.counts[blockIdx.x * p.ranges + i] = count[i];
}

// A stable counting sort by one work group: every wave goes through a part of its own, twice, counting keys and then placing them.
template <typename I, int MODE>
static __global__ __launch_bounds__(64 * kEmbWaves) void emb_sort_kernel(EmbSorted<I> p) {
  __shared__ int count[kEmbWaves][kEmbBins];
  __shared__ int sums[kEmbWaves], below_of[kEmbWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = MODE == kSortChunk ? p.ranges : p.bins, v0 = MODE == kSortChunk ? 0 : blockIdx.x * p.bins, v1 = min(v0 + p.bins, p.t.rows);
  static_assert(kEmbBins <= 64 * kEmbWaves, "a key a thread");
  if (threadIdx.x < keys)
#pragma unroll
    for (int w = 0; w < kEmbWaves; ++w) count[w][threadIdx.x] = 0;
  // what there is to go through; the sorted position of the first
  int64_t begin = 0, end = p.t.count;
  int first = 0;
  if constexpr (MODE == kSortChunk) {
    begin = static_cast<int64_t>(blockIdx.x) * p.chunk;
    end = begin + p.chunk < p.t.count ? begin + p.chunk : p.t.count;
  }
  if constexpr (MODE == kSortRange) {
    begin = first = p.firsts[blockIdx.x];
    end = p.firsts[blockIdx.x + 1];
  }
  __syncthreads();
  const int64_t part = (end - begin + 64 * kEmbWaves - 1) / (64 * kEmbWaves) * 64, n0 = begin + wave * part, n1 = n0 + part < end ? n0 + part : end;
  constexpr int U = 8;
  // f(key, token, position in the text) of 64 positions at a time; whole waves
  auto each = [&](auto&& f) {
    for (int64_t n = n0; n < n1; n += 64 * U) {
      int v[U], at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t m = n + 64 * u + lane;
        if constexpr (MODE == kSortRange) {
          v[u] = m < n1 ? p.token[m] : -1;
          at[u] = m < n1 ? p.place[m] : 0;
        } else {
          v[u] = m < n1 ? p.t.named(m) : -1;
          at[u] = static_cast<int>(m);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int key = v[u] - v0;
        if constexpr (MODE == kSortChunk) key = v[u] >= 0 ? v[u] / p.bins : -1;
        else if (v[u] < v0 || v[u] >= v1) key = -1;
        f(key, v[u], at[u]);
      }
    }
  };
  int below = 0;
  each([&](int key, int token, int) {
    if constexpr (MODE == kSortAll) below += token >= 0 && token < v0 ? 1 : 0;
    if (key >= 0) atomicAdd(&count[wave][key], 1);
  });
  if constexpr (MODE == kSortAll) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
    if (lane == 0) below_of[wave] = below;
  }
  __syncthreads();
  if constexpr (MODE == kSortAll)
#pragma unroll
    for (int w = 0; w < kEmbWaves; ++w) first += below_of[w];
  // thread i: key i; places of the waves' tokens of that key from the exclusive sums over keys and waves
  int mine = 0, earlier = 0;             // of this key: tokens behind it that count for the next key, tokens in front of this work group's
  if constexpr (MODE == kSortChunk) {
    if (threadIdx.x < keys)
#pragma unroll 8
      for (int c = 0; c < p.chunks; ++c) {
        const int n = p.counts[c * p.ranges + threadIdx.x];
        mine += n;
        earlier += c < static_cast<int>(blockIdx.x) ? n : 0;
      }
  } else if (threadIdx.x < keys) {
#pragma unroll
    for (int w = 0; w < kEmbWaves; ++w) mine += count[w][threadIdx.x];
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int at = first + incl - mine;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) at += w < wave ? sums[w] : 0;
  if (threadIdx.x < keys) {
    if constexpr (MODE != kSortChunk) {
      const int v = v0 + threadIdx.x;
      if (v < v1) {
        p.starts[v] = at;
        if (v == p.t.rows - 1) p.starts[p.t.rows] = at + mine;
      }
    }
    if constexpr (MODE == kSortChunk)
      if (blockIdx.x == 0) {
        p.firsts[threadIdx.x] = at;
        if (static_cast<int>(threadIdx.x) == keys - 1) p.firsts[keys] = at + mine;
      }
    at += earlier;
#pragma unroll
    for (int w = 0; w < kEmbWaves; ++w) {
      const int c = count[w][threadIdx.x];
      count[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  AK_LDS volatile int* next = (AK_LDS volatile int*)count[wave];
  const int bits = 32 - __builtin_clz(keys | 1);
  each([&](int key, int token, int at_text) {
    u64 same = __ballot(key >= 0);
    if (same == 0) return;
    for (int b = 0; b < bits; ++b) {             // the lanes whose key has the same bits
      const bool bit = (key >> b & 1) != 0;
      const u64 set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    if (key < 0) return;
    const int base = next[key], rank = __popcll(same & ((1ull << lane) - 1));
    const int to = base + rank;
    if constexpr (MODE == kSortChunk) {
      p.token[to] = token;
      p.place[to] = at_text;
    } else {
      p.sorted[to] = token;
      p.order[to] = at_text;
    }
    if (rank == 0) next[key] = base + __popcll(same);
  });
}

struct EmbSums {
  const int *starts, *order, *sorted;
  const void* g;
  void* out;
  int2* joins;             // [chunks] token and chunks of the run that begins in a chunk and ends in a later one; no chunks: none
  float *lead, *trail;     // [chunks][ldp] parts of runs that began in front of a chunk; that begin in it and go on behind it
  int64_t ldg, ldo, ldp;
  int rows, D, chunk, chunks, slabs, rows_of;        // rows_of: rows that a wave looks through for those without a token
  float scale, beta;
};

// out <- beta*out + scale*sum, one lane's E columns from c on
template <typename O, int E>
__device__ __forceinline__ void emb_write(const EmbSums& p, int row, int c, const float (&sum)[E]) {
  O* __restrict__ to = static_cast<O*>(p.out) + static_cast<int64_t>(row) * p.ldo + c;
  if (c + E <= p.D) {
    Some<O, E> o;
    if (p.beta != 0.f) {
      o.load(to);
#pragma unroll
      for (int e = 0; e < E; ++e) o.set(e, p.beta * o.get(e) + p.scale * sum[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) o.set(e, p.scale * sum[e]);
    }
    o.store(to);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < p.D) to[e] = static_cast<O>(p.beta != 0.f ? p.beta * static_cast<float>(to[e]) + p.scale * sum[e] : p.scale * sum[e]);
  }
}

template <typename G, typename O>
static __global__ __launch_bounds__(256) void emb_sums_kernel(EmbSums p) {
  constexpr int E = 16 / sizeof(G), U = 8;
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t units = static_cast<int64_t>(p.chunks) * p.slabs;
  if (unit >= units) {
    // its rows that have no token
    const int64_t v0 = (unit - units) * p.rows_of;
    if (v0 >= p.rows) return;
    const int64_t v = v0 + lane;
    u64 none = __ballot(lane < p.rows_of && v < p.rows && p.starts[v < p.rows ? v : 0] == p.starts[v < p.rows ? v + 1 : 0]);
    if (p.beta == 1.f) return;
    const float zero[E] = {};
    while (none != 0) {
      const int row = static_cast<int>(v0) + __builtin_ctzll(none);
      for (int c = lane * E; c < p.D; c += 64 * E) emb_write<O, E>(p, row, c, zero);
      none &= none - 1;
    }
    return;
  }
  const int chunk = static_cast<int>(unit / p.slabs), slab = static_cast<int>(unit - static_cast<int64_t>(chunk) * p.slabs);
  const int total = p.starts[p.rows];
  const int p0 = chunk * p.chunk, p1 = min(p0 + p.chunk, total);
  if (p0 >= p1) {
    if (slab == 0 && lane == 0) p.joins[chunk] = int2{0, 0};
    return;
  }
  const int c = slab * 64 * E + lane * E;
  const bool has = c < p.D, full = c + E <= p.D;
  const int my_row = p0 + lane < p1 ? p.order[p0 + lane] : 0;
  const int my_token = p0 + lane < p1 ? p.sorted[p0 + lane] : -1;
  const int before = p0 > 0 ? p.sorted[p0 - 1] : -1, behind = p1 < total ? p.sorted[p1] : -1;
  float sum[E] = {};
  auto flush = [&](int token, bool first, bool last) {
    if (!has) return;
    const bool from = first && token == before, on = last && token == behind;
    if (!from && !on) {
      emb_write<O, E>(p, token, c, sum);
      return;
    }
    float* __restrict__ to = (from ? p.lead : p.trail) + chunk * p.ldp + c;       // (ldp holds whole vectors)
#pragma unroll
    for (int e = 0; e < E; ++e) to[e] = sum[e];
  };
  if (slab == 0 && lane == 0) {
    const int last = p.sorted[p1 - 1];
    int2 join = {last, 0};
    if (last == behind && p.starts[last] >= p0) join.y = (p.starts[last + 1] - 1) / p.chunk - chunk + 1;
    p.joins[chunk] = join;
  }
  int token = __builtin_amdgcn_readlane(my_token, 0);
  bool first = true;
  for (int i = 0; i < p1 - p0; i += U) {
    Some<G, E> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].clear();
      if (i + u < p1 - p0) {
        const G* __restrict__ from = static_cast<const G*>(p.g) + static_cast<int64_t>(__builtin_amdgcn_readlane(my_row, i + u)) * p.ldg + c;
        if (full) {
          v[u].load(from);
        } else if (has) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (c + e < p.D) v[u].v[e] = from[e];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= p1 - p0) continue;
      const int next = __builtin_amdgcn_readlane(my_token, i + u);
      if (next != token) {
        flush(token, first, false);
        first = false;
        token = next;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] += v[u].get(e);
    }
  }
  flush(token, first, true);
}

// Parts k0 .. k1 - 1 of the run that begins in a chunk, four columns from c on.
__device__ __forceinline__ floatx4 emb_parts(const EmbSums& p, int chunk, int k0, int k1, int c) {
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = k0; k < k1; ++k) sum += *reinterpret_cast<const floatx4*>((k == 0 ? p.trail : p.lead) + static_cast<int64_t>(chunk + k) * p.ldp + c);
  return sum;
}

// Runs that begin in a chunk and end in a later one, 256 columns at a time.  The first work groups take the long ones: a run of more than
// 16 chunks begins in no more than one of 16 neighbouring chunks; four waves take a quarter of its parts each.  Behind them, a wave
// takes the run of a chunk alone.  (All four waves for every run: 17 us for 131072 tokens of 1024 columns, most of it waves that wait.)
constexpr int kEmbLong = 16;

template <typename O>
static __global__ __launch_bounds__(256) void emb_joins_kernel(EmbSums p, int long_groups, int column_blocks) {
  __shared__ floatx4 joined[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (static_cast<int>(blockIdx.x) < long_groups) {
    const int first = static_cast<int>(blockIdx.x) / column_blocks * kEmbLong, c = static_cast<int>(blockIdx.x) % column_blocks * 256 + 4 * lane;
    int2 mine = {0, 0};
    if (lane < kEmbLong && first + lane < p.chunks) mine = p.joins[first + lane];
    const u64 runs = __ballot(mine.y > kEmbLong);          // (the same in every wave)
    if (runs == 0) return;
    const int at = __builtin_ctzll(runs), token = __builtin_amdgcn_readlane(mine.x, at), parts = __builtin_amdgcn_readlane(mine.y, at), per = (parts + 3) / 4;
    joined[wave][lane] = c < p.D ? emb_parts(p, first + at, wave * per, min((wave + 1) * per, parts), c) : floatx4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (wave != 0 || c >= p.D) return;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ((joined[0][lane][e] + joined[1][lane][e]) + joined[2][lane][e]) + joined[3][lane][e];
    emb_write<O, 4>(p, token, c, v);
    return;
  }
  const int64_t unit = static_cast<int64_t>(blockIdx.x - long_groups) * 4 + wave;
  const int64_t chunk = unit / column_blocks;
  const int c = static_cast<int>(unit - chunk * column_blocks) * 256 + 4 * lane;
  if (chunk >= p.chunks || c >= p.D) return;
  const int2 join = p.joins[chunk];
  if (join.y == 0 || join.y > kEmbLong) return;
  const floatx4 sum = emb_parts(p, static_cast<int>(chunk), 0, join.y, c);
  const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
  emb_write<O, 4>(p, join.x, c, v);
}

// Sorted positions of a chunk: enough chunks for 32 waves a CU, few enough for little to be joined.
inline int emb_chunk(int64_t tokens, int64_t D, int elements) {
  const int64_t slabs = (D + 64 * elements - 1) / (64 * elements), want = tokens * slabs / 8192;
  return want <= 8 ? 8 : want <= 16 ? 16 : want <= 32 ? 32 : 64;
}

template <typename F>
inline int with_tokens(int type, F&& f) {
  switch (type) {
    case AK_I64: return f(Type<int64_t>{});
    case AK_I32: return f(Type<int32_t>{});
    default: return AK_ERR_ARG;
  }
}

struct EmbSpace {
  int *starts, *order, *sorted, *token, *place, *counts, *firsts;
  int bins, ranges, cut, cuts;           // rows of a range; tokens of a chunk of the sort, or all of them at once: cuts == 0
  int2* joins;
  float *lead, *trail;
  int chunk, chunks;
  int64_t ldp;
  size_t bytes;
};

inline EmbSpace emb_space(int64_t tokens, int64_t rows, int64_t D, int elements, void* ws) {
  unsigned char* base = static_cast<unsigned char*>(ws);
  size_t used = 0;
  auto take = [&](int64_t words) {
    void* at = base != nullptr ? base + used : nullptr;
    used += static_cast<size_t>((words * 4 + 255) / 256 * 256);
    return at;
  };
  EmbSpace s = {};
  s.chunk = emb_chunk(tokens, D, elements);
  s.chunks = static_cast<int>((tokens + s.chunk - 1) / s.chunk);
  s.ldp = (D + 7) / 8 * 8;
  s.starts = static_cast<int*>(take(rows + 1));
  s.order = static_cast<int*>(take(tokens));
  s.sorted = static_cast<int*>(take(tokens));
  // 256 ranges where they hold the table; tokens by range first where there are many, and few enough ranges
  s.bins = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + 255) / 256, kEmbBins)));
  s.ranges = static_cast<int>((rows + s.bins - 1) / s.bins);
  s.cut = static_cast<int>(std::max<int64_t>(kEmbChunk, (tokens + 255) / 256));
  s.cuts = tokens > kEmbScan && s.ranges <= kEmbBins ? static_cast<int>((tokens + s.cut - 1) / s.cut) : 0;
  if (s.cuts > 0) {
    s.token = static_cast<int*>(take(tokens));
    s.place = static_cast<int*>(take(tokens));
    s.counts = static_cast<int*>(take(static_cast<int64_t>(s.ranges) * s.cuts));
    s.firsts = static_cast<int*>(take(s.ranges + 1));
  }
  s.joins = static_cast<int2*>(take(2 * static_cast<int64_t>(s.chunks)));
  s.lead = static_cast<float*>(take(s.chunks * s.ldp));
  s.trail = static_cast<float*>(take(s.chunks * s.ldp));
  s.bytes = used;
  return s;
}

inline int emb_check(int token_type, int64_t tokens, int64_t rows, int64_t D, int64_t ld) {
  if ((token_type != AK_I64 && token_type != AK_I32) || tokens < 0 || rows < 0 || D <= 0 || ld < D) return AK_ERR_ARG;
  if (tokens > (1ll << 30) || rows > (1ll << 30) || D > (1ll << 24)) return AK_ERR_TOO_LARGE;
  return AK_OK;
}

}  // namespace ak

extern "C" int ak_embedding(const void* tokens, int token_type, int64_t count, const void* table, int dtype, int64_t ld, int64_t rows, int64_t width,
                            float scale, void* out, int out_dtype, ak_stream_t stream) {
  using namespace ak;
  const int rc = emb_check(token_type, count, rows, width, ld);
  if (rc != AK_OK) return rc;
  if (!is_element_type(dtype) || (out_dtype != dtype && out_dtype != AK_F32)) return AK_ERR_ARG;
  if (count == 0) return AK_OK;
  if (tokens == nullptr || out == nullptr || (table == nullptr && rows > 0)) return AK_ERR_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    auto go = [&](auto o) {
      using O = typename decltype(o)::type;
      return with_tokens(token_type, [&](auto i) {
        using I = typename decltype(i)::type;
        auto launch = [&](auto lanes) {
          constexpr int L = decltype(lanes)::value;
          constexpr int64_t kMost = 1ll << 25;       // tokens of a launch: 2^31 threads of 64 a token
          for (int64_t n = 0; n < count; n += kMost) {
            const Tokens<I> tk{static_cast<const I*>(tokens) + n, std::min(count - n, kMost), static_cast<int>(rows), -1};
            hipLaunchKernelGGL((emb_rows_kernel<T, O, I, L>), dim3(static_cast<unsigned>((tk.count + 256 / L - 1) / (256 / L))), dim3(256), 0, s, tk,
                               static_cast<const T*>(table), ld, static_cast<int>(width), scale, static_cast<O*>(out) + n * width);
          }
          return check_launch();
        };
        // as many lanes as a row has vectors, 8 to 64
        const int64_t vectors = (width + 16 / static_cast<int64_t>(sizeof(T)) - 1) / (16 / static_cast<int64_t>(sizeof(T)));
        return vectors <= 8 ? launch(std::integral_constant<int, 8>{}) : vectors <= 32 ? launch(std::integral_constant<int, 32>{})
                                                                                       : launch(std::integral_constant<int, 64>{});
      });
    };
    if (out_dtype == dtype) return go(t);
    return go(Type<float>{});
  });
}

extern "C" size_t ak_embedding_backward_ws_bytes(int64_t count, int64_t rows, int64_t width) {
  if (count < 0 || rows < 0 || width <= 0 || count > (1ll << 30) || rows > (1ll << 30) || width > (1ll << 24)) return 0;
  return std::max(ak::emb_space(count, rows, width, 4, nullptr).bytes, ak::emb_space(count, rows, width, 8, nullptr).bytes);
}

extern "C" int ak_embedding_backward(const void* g, int dtype, int64_t ldg, const void* tokens, int token_type, int64_t count, int64_t rows,
                                     int64_t width, float scale, int64_t padding, float beta, void* out, int out_dtype, int64_t ldo, void* ws,
                                     size_t ws_bytes, ak_stream_t stream) {
  using namespace ak;
  int rc = emb_check(token_type, count, rows, width, ldo);
  if (rc != AK_OK) return rc;
  if (!is_element_type(dtype) || !is_element_type(out_dtype) || ldg < width) return AK_ERR_ARG;
  if (rows == 0) return AK_OK;
  if (out == nullptr || (count > 0 && (g == nullptr || tokens == nullptr))) return AK_ERR_ARG;
  if (ws == nullptr || ws_bytes < ak_embedding_backward_ws_bytes(count, rows, width)) return AK_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int elements = dtype == AK_F32 ? 4 : 8;
  const EmbSpace s = emb_space(count, rows, width, elements, ws);
  rc = with_tokens(token_type, [&](auto i) {
    using I = typename decltype(i)::type;
    const Tokens<I> tk{static_cast<const I*>(tokens), count, static_cast<int>(rows), padding};
    const EmbSorted<I> q{tk, s.bins, s.ranges, s.cut, s.cuts, s.counts, s.firsts, s.token, s.place, s.starts, s.order, s.sorted};
    const dim3 ranges(static_cast<unsigned>(s.ranges)), cuts(static_cast<unsigned>(s.cuts)), threads(64 * kEmbWaves);
    if (s.cuts == 0) {
      hipLaunchKernelGGL((emb_sort_kernel<I, kSortAll>), ranges, threads, 0, st, q);
    } else {
      hipLaunchKernelGGL(emb_count_kernel<I>, cuts, dim3(1024), 0, st, q);
      hipLaunchKernelGGL((emb_sort_kernel<I, kSortChunk>), cuts, threads, 0, st, q);
      hipLaunchKernelGGL((emb_sort_kernel<I, kSortRange>), ranges, threads, 0, st, q);
    }
    return check_launch();
  });
  if (rc != AK_OK) return rc;
  EmbSums p;
  p.starts = s.starts; p.order = s.order; p.sorted = s.sorted;
  p.g = g; p.out = out; p.joins = s.joins; p.lead = s.lead; p.trail = s.trail;
  p.ldg = ldg; p.ldo = ldo; p.ldp = s.ldp;
  p.rows = static_cast<int>(rows); p.D = static_cast<int>(width);
  p.chunk = s.chunk; p.chunks = s.chunks;
  p.slabs = static_cast<int>((width + 64 * elements - 1) / (64 * elements));
  // (64 rows a wave leave most of the device idle where rows are few and long: 2365 of 3265 columns 58 -> 10 us)
  p.rows_of = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(64, rows / 8192)));
  p.scale = scale; p.beta = beta;
  const int64_t units = static_cast<int64_t>(p.chunks) * p.slabs + (rows + p.rows_of - 1) / p.rows_of;
  if (!fits_a_launch((units + 3) / 4, 256)) return AK_ERR_TOO_LARGE;
  return with_type(out_dtype, [&](auto o) {
    using O = typename decltype(o)::type;
    const int64_t column_blocks = (width + 255) / 256, longs = (p.chunks + kEmbLong - 1) / kEmbLong * column_blocks, shorts = (p.chunks * column_blocks + 3) / 4;
    if (!fits_a_launch(longs + shorts, 256)) return AK_ERR_TOO_LARGE;
    const int done = with_type(dtype, [&](auto t) {
      using G = typename decltype(t)::type;
      hipLaunchKernelGGL((emb_sums_kernel<G, O>), dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, st, p);
      return check_launch();
    });
    if (done != AK_OK || p.chunks < 2) return done;
    hipLaunchKernelGGL(emb_joins_kernel<O>, dim3(static_cast<unsigned>(longs + shorts)), dim3(256), 0, st, p, static_cast<int>(longs),
                       static_cast<int>(column_blocks));
    return check_launch();
  });
}
