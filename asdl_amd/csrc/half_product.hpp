// Products of 16-bit matrices (bf16 or fp16, fp32 sums) on the matrix cores, for operators whose epilogue is their own:
//   D[i][j] = sum_k A[i][k] B[k][j]
// Either operand lies in memory with its contraction index along the rows ("by k": row i or j holds its k values) or across them ("by
// row": row k holds all i or j).  A work group has one BI x BJ tile of D; a lane of a wave has, for every 32 x 32 block, one column j and
// 16 rows i, four of them consecutive: an epilogue that writes D transposed writes four neighbouring elements, one that reduces over i
// stays in the lane.
// Panels of 32 k go from memory to the LDS without passing registers (syrk_dtl_tile.hpp: load_to_lds), Cfg::STAGES of them in flight.  Both
// kinds of panel are blocks of 2 KB, 32 rows of 64 bytes:
//   by k:   [32 i][32 k], 16-byte chunks of a row exchanged by (row / 4) % 4, so that the 16 rows a ds_read_b128 serves at once lie in
//           different banks; the exchange is made on the memory side of the load, within the 64 bytes of a row
//   by row: [32 k][32 i], read by ds_read_b64_tr_b16
// The base of an operand's descriptor moves with the k-tile (scalar arithmetic), so offsets of a lane are constants and no size of the
// contraction is too large for them; what lies outside the matrix reads as zero: rows beyond it by the number of records or an offset
// beyond it, the last k by a comparison.
#pragma once
#include <algorithm>
#include <atomic>
#include "elements.hpp"
#include "syrk_dtl_tile.hpp"

namespace ak {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename E>
__device__ __forceinline__ floatx16 hp_mfma(short8v a, short8v b, floatx16 c) {
  if constexpr (sizeof(E) == 2 && __is_same(E, __bf16))
    return mfma_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct HpOperand {
  const void* p;           // 16-byte aligned
  int64_t ld;              // bytes between rows, a multiple of 16
  int rows;                // by k: rows i (or j) there are
  int cols;                // by row: elements of a row, a multiple of 8 (what lies behind the matrix is not stored)
  int64_t k;               // k there are (by row: rows; a contraction that is longer takes zeros)
};

// Operands in pieces that add up to their values, side by side in a row: D is the sum of the products of `count` pairs of them, one after
// the other in the contraction.  fp32 values are three bf16 pieces exactly, of whose nine products the six that matter are taken (the others are
// below 2^-24 of the product), the smallest first.
struct HpPieces {
  int count;
  int a[6], b[6];          // bytes from a row's first piece
};

struct HpProblem {
  HpOperand A, B;
  HpPieces pieces;         // of a configuration with PIECES
  int64_t K, k_per_split;  // k_per_split a multiple of 32
  int tiles_i, tiles_j, splits;
};

template <int WR_, int WC_, int FR_, int FC_, bool A_BY_K_, bool B_BY_K_, int STAGES_, bool PIECES_ = false>
struct HpCfg {
  static constexpr int WR = WR_, WC = WC_, FR = FR_, FC = FC_, NW = WR * WC, THREADS = 64 * NW, STAGES = STAGES_;
  static constexpr bool A_BY_K = A_BY_K_, B_BY_K = B_BY_K_, PIECES = PIECES_;
  static constexpr int BI = 32 * FR * WR, BJ = 32 * FC * WC, BK = 32;
  static constexpr int BLOCK = 2048, PANEL_A = BI * 64, PANEL_B = BJ * 64, STAGE = PANEL_A + PANEL_B, LDS_BYTES = STAGES * STAGE;
  static constexpr int LDS_ALL = LDS_BYTES > BJ * (BI * 2 + 16) ? LDS_BYTES : BJ * (BI * 2 + 16);        // or a tile of 16-bit rows
  static constexpr int IA = BI / 16 / NW, IB = BJ / 16 / NW, LPT = IA + IB;      // wave-wide loads of a k-tile, per wave
  static_assert(BI / 16 % NW == 0 && BJ / 16 % NW == 0 && LDS_ALL <= 160 * 1024, "loads split evenly, panels fit the LDS");
};

// What one wave loads of an operand: N wave-wide loads a k-tile.
template <bool BY_K, int N>
struct HpLoader {
  uint64_t base;           // of the next k-tile
  int64_t step, left;      // bytes to the k-tile behind it; k from there to the end
  uint32_t off[N];
  int64_t ld;
  int k_of_lane, first;

  __device__ __forceinline__ void init(const HpOperand& o, int wave, int lane, int at0, int64_t k0, int64_t k_count) {
    ld = o.ld;
    left = k_count < o.k - k0 ? k_count : o.k - k0;
    if constexpr (BY_K) {
      const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
      base = reinterpret_cast<uint64_t>(o.p) + static_cast<uint64_t>(at0) * o.ld + static_cast<uint64_t>(k0) * 2;
      step = 64;
      k_of_lane = 8 * chunk;
      first = wave * N * 1024;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = 16 * (wave * N + i) + (lane >> 2);
        off[i] = at0 + row < o.rows ? static_cast<uint32_t>(row) * static_cast<uint32_t>(o.ld) + 16u * chunk : kDtlOob;
      }
    } else {
      const int half = wave & 1, cb = (wave >> 1) * N, row = 16 * half + (lane >> 2);
      base = reinterpret_cast<uint64_t>(o.p) + static_cast<uint64_t>(k0) * o.ld;
      step = 32 * o.ld;
      first = cb * 2048 + half * 1024;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int col = at0 + 32 * (cb + i) + 8 * (lane & 3);
        off[i] = col < o.cols ? static_cast<uint32_t>(row) * static_cast<uint32_t>(o.ld) + 2u * static_cast<uint32_t>(col) : kDtlOob;
      }
    }
  }

  // Load i of the k-tile that base stands at, to the panel at `lds`.
  __device__ __forceinline__ void load(int i, uint32_t lds) const {
    u32x4 rsrc;
    rsrc[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base));
    rsrc[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base >> 32) & 0xffffu);
    rsrc[3] = 0x00020000u;
    uint32_t at = off[i];
    if constexpr (BY_K) {
      rsrc[2] = kDtlRange;
      if (k_of_lane >= left) at = kDtlOob;
    } else {
      // rows of the tile that exist, in bytes: an offset into a row behind them is at least that
      const int64_t bytes = (left < 32 ? (left < 0 ? 0 : left) : 32) * ld;
      rsrc[2] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bytes));
    }
    load_to_lds<true>(rsrc, lds + first + i * (BY_K ? 1024 : 2048), at);
  }

  __device__ __forceinline__ void next() {
    base += step;
    left -= 32;
  }
  // Back by `tiles` k-tiles and on by `bytes`: to the start of another piece.
  __device__ __forceinline__ void again(int tiles, int64_t bytes) {
    base += static_cast<uint64_t>(bytes - tiles * step);
    left += 32 * static_cast<int64_t>(tiles);
  }
};

// Offsets of a lane's fragments within the blocks of a panel: of the first and of the second 16 k of a k-tile.
template <bool BY_K>
__device__ __forceinline__ int hp_fragment(int lane, int kk) {
  const int g = lane >> 5, l32 = lane & 31, j16 = lane & 15, hl = (lane >> 4) & 1;
  if constexpr (BY_K) return l32 * 64 + (((2 * kk + g) ^ ((l32 >> 2) & 3)) << 4);
  return (16 * kk + 8 * g + (j16 >> 2)) * 64 + hl * 32 + (j16 & 3) * 8;
}

template <bool BY_K>
__device__ __forceinline__ short8v hp_read(AK_LDS const unsigned char* q) {
  if constexpr (BY_K) return *reinterpret_cast<AK_LDS const short8v*>(q);
  const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AK_LDS short4v*)(q));
  const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AK_LDS short4v*)(q + 256));
  return short8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Tiles in groups of eight along i, so that the tiles an XCD works on at a time share panels in its L2.
__device__ __forceinline__ void hp_place(int id, int tiles_i, int tiles_j, int& ti, int& tj) {
  constexpr int GROUP = 8;
  const int per = GROUP * tiles_j, group = id / per, i0 = group * GROUP, height = min(GROUP, tiles_i - i0), rest = id - group * per;
  ti = i0 + rest % height;
  tj = rest / height;
}

// One tile of D.  The loop alone sustains 1.3 PFLOP/s (512 k-tiles of 256 x 256, both operands by row, bf16), where the device is at its
// power limit (1.9 GHz, the matrix cores busy for 66 % of the cycles; fp16 operands 1.5 GHz and 71 %).  A work group that goes on to another
// tile, with its loads running on into that one under the epilogue, was not faster: 649 -> 626 us for the 6304 tiles of 24 k-tiles of
// a 50257-class forward pass, but 1982 -> 2068 us for 8000 of 64.
template <class Cfg, typename E, class Epilogue>
__device__ __forceinline__ void hp_run(const HpProblem& p, const typename Epilogue::Params& e, uint32_t block, uint32_t blocks) {
  constexpr int FR = Cfg::FR, FC = Cfg::FC, S = Cfg::STAGES, LPT = Cfg::LPT;
  extern __shared__ __attribute__((aligned(1024))) unsigned char hp_smem[];
  AK_LDS unsigned char* lds = (AK_LDS unsigned char*)hp_smem;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / Cfg::WC, wc = wave % Cfg::WC;
  const int tiles = p.tiles_i * p.tiles_j, id = static_cast<int>(xcd_contiguous_id(block, blocks)), split = id / tiles;
  int ti, tj;
  hp_place(id - split * tiles, p.tiles_i, p.tiles_j, ti, tj);
  const int64_t k0 = split * p.k_per_split, k_count = p.K - k0 < p.k_per_split ? p.K - k0 : p.k_per_split;
  HpLoader<Cfg::A_BY_K, Cfg::IA> la;
  HpLoader<Cfg::B_BY_K, Cfg::IB> lb;
  la.init(p.A, wave, lane, ti * Cfg::BI, k0, k_count);
  lb.init(p.B, wave, lane, tj * Cfg::BJ, k0, k_count);
  const int nk = static_cast<int>((k_count + 31) / 32);        // k-tiles (of a piece)
  int piece = 0, left_of_piece = nk;
  if constexpr (Cfg::PIECES) {
    la.base += p.pieces.a[0];
    lb.base += p.pieces.b[0];
  }
  auto load_next = [&]() {
    la.next();
    lb.next();
    if constexpr (Cfg::PIECES) {
      if (--left_of_piece == 0 && piece + 1 < p.pieces.count) {
        la.again(nk, p.pieces.a[piece + 1] - p.pieces.a[piece]);
        lb.again(nk, p.pieces.b[piece + 1] - p.pieces.b[piece]);
        ++piece;
        left_of_piece = nk;
      }
    }
  };
  auto load_one = [&](int l, int stage) {
    const uint32_t at = lds0 + stage * Cfg::STAGE;
    if (l < Cfg::IA) la.load(l, at);
    else lb.load(l - Cfg::IA, at + Cfg::PANEL_A);
  };
  const int fa_off[2] = {hp_fragment<Cfg::A_BY_K>(lane, 0), hp_fragment<Cfg::A_BY_K>(lane, 1)};
  const int fb_off[2] = {hp_fragment<Cfg::B_BY_K>(lane, 0), hp_fragment<Cfg::B_BY_K>(lane, 1)};
  AK_LDS const unsigned char* pa = lds + wr * FR * Cfg::BLOCK;
  AK_LDS const unsigned char* pb = lds + Cfg::PANEL_A + wc * FC * Cfg::BLOCK;
  // fragment u of 16 k, in the order in which the matrix instructions want them: a0, b0 .. b(FC-1), a1 .. a(FR-1)
  auto read_unit = [&](short8v (&fa)[FR], short8v (&fb)[FC], int stage, int kk, int u) {
    const int s = stage * Cfg::STAGE;
    if (u == 0 || u > FC) fa[u == 0 ? 0 : u - FC] = hp_read<Cfg::A_BY_K>(pa + s + (u == 0 ? 0 : u - FC) * Cfg::BLOCK + fa_off[kk]);
    else fb[u - 1] = hp_read<Cfg::B_BY_K>(pb + s + (u - 1) * Cfg::BLOCK + fb_off[kk]);
  };
  floatx16 acc[FR][FC];
#pragma unroll
  for (int a = 0; a < FR; ++a)
#pragma unroll
    for (int b = 0; b < FC; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  const int steps = Cfg::PIECES ? nk * p.pieces.count : nk;
#pragma unroll
  for (int t = 0; t < S - 1; ++t) {              // k-tiles behind the last load zeros: the counts stay uniform
#pragma unroll
    for (int l = 0; l < LPT; ++l) load_one(l, t);
    load_next();
  }
  if constexpr (Cfg::NW == 8) {
    // Two groups of four waves, one wave of each on every SIMD, take turns: while one reads the LDS and asks for a k-tile further
    // ahead, the other has the matrix cores, and a barrier changes their parts.  A wave's fragments of a k-tile have arrived before
    // its turn, its loads of the next one before the barrier in front of it.  (With reads and loads spread between the matrix instructions
    // of the same wave, as below: 8192 x 768 x 50257 bf16 622 -> 616 us, 4096 x 2048 x 128000 fp16 2010 -> 1934 us.)
    const bool second = wave >= 4;
    wait_vmcnt<(S - 2) * LPT>();                 // this wave's loads of the first k-tile have landed
    __syncthreads();                             // ... and everybody's
    if (second) asm volatile("s_barrier" ::: "memory");
    int rd = 0, to = S - 1;
    for (int kt = 0; kt < steps; ++kt) {
      short8v fa[2][FR], fb[2][FC];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int u = 0; u < FR + FC; ++u) read_unit(fa[kk], fb[kk], rd, kk, u);
#pragma unroll
      for (int l = 0; l < LPT; ++l) load_one(l, to);
      load_next();
      rd = (rd + 1 == S) ? 0 : rd + 1;
      to = (to + 1 == S) ? 0 : to + 1;
      // own loads of the next k-tile have landed, own fragments have arrived
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LPT) : "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int a = 0; a < FR; ++a)
#pragma unroll
          for (int b = 0; b < FC; ++b) acc[a][b] = hp_mfma<E>(fa[kk][a], fb[kk][b], acc[a][b]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_barrier" ::: "memory");
    }
    if (!second) asm volatile("s_barrier" ::: "memory");
  } else {
    // Four waves, two work groups a CU.  The matrix instructions of 16 k, with the reads of the next 16 and (NLOAD) the loads of a k-tile
    // further ahead spread between them.
    auto half_step = [&](auto loads_tag, const short8v (&ca)[FR], const short8v (&cb)[FC], short8v (&na)[FR], short8v (&nb)[FC], int stage,
                         int kk, int to) {
      constexpr int NLOAD = decltype(loads_tag)::value, NM = FR * FC, NS = NLOAD + FR + FC;
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const int a = m / FC, b = m % FC;
        acc[a][b] = hp_mfma<E>(ca[a], cb[b], acc[a][b]);
#pragma unroll
        for (int s = (m * NS) / NM; s < ((m + 1) * NS) / NM; ++s) {
          __builtin_amdgcn_sched_barrier(0);
          if (s < NLOAD) load_one(s, to);
          else read_unit(na, nb, stage, kk, s - NLOAD);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    wait_vmcnt<(S - 2) * LPT>();                   // this wave's loads of the first k-tile have landed
    __syncthreads();                               // ... and everybody's
    short8v fa0[FR], fb0[FC], fa1[FR], fb1[FC];
#pragma unroll
    for (int u = 0; u < FR + FC; ++u) read_unit(fa0, fb0, 0, 0, u);
    int rd = 0, to = S - 1;
    for (int kt = 0; kt < steps; ++kt) {
      half_step(std::integral_constant<int, 0>{}, fa0, fb0, fa1, fb1, rd, 1, 0);
      wait_vmcnt<(S - 3) * LPT>();                 // own loads of the next k-tile have landed
      __syncthreads();                             // everybody's have; nobody reads the k-tile before this one any more
      rd = (rd + 1 == S) ? 0 : rd + 1;
      half_step(std::integral_constant<int, LPT>{}, fa1, fb1, fa0, fb0, rd, 0, to);
      load_next();
      to = (to + 1 == S) ? 0 : to + 1;
    }
  }
  wait_vmcnt<0>();                               // the loads of zeros have landed before the LDS is used again
  Epilogue::template run<Cfg>(e, acc, ti, tj, split, wr, wc, lds);
}

template <class Cfg, typename E, class Epilogue>
static __global__ __launch_bounds__(Cfg::THREADS, 2) void hp_kernel(HpProblem p, typename Epilogue::Params e) {
  hp_run<Cfg, E, Epilogue>(p, e, blockIdx.x, gridDim.x);
}

// Two products in one launch, the first work groups to the first: what one leaves of the device the other fills.
template <class Cfg1, class Epilogue1, class Cfg2, class Epilogue2, typename E>
static __global__ __launch_bounds__(Cfg1::THREADS, 2) void hp_both_kernel(HpProblem p1, typename Epilogue1::Params e1, uint32_t blocks1, HpProblem p2,
                                                                            typename Epilogue2::Params e2, uint32_t blocks2, int second_first) {
  static_assert(Cfg1::THREADS == Cfg2::THREADS && Cfg1::LDS_ALL == Cfg2::LDS_ALL, "one launch");
  const uint32_t front = second_first ? blocks2 : blocks1;
  const bool in_front = blockIdx.x < front;
  const uint32_t block = in_front ? blockIdx.x : blockIdx.x - front;
  if (in_front == (second_first != 0)) hp_run<Cfg2, E, Epilogue2>(p2, e2, block, blocks2);
  else hp_run<Cfg1, E, Epilogue1>(p1, e1, block, blocks1);
}

// f(i, j, values of rows i .. i + 3) for a lane's part of the tile.
template <class Cfg, typename F>
__device__ __forceinline__ void hp_quads(floatx16 (&acc)[Cfg::FR][Cfg::FC], int ti, int tj, int wr, int wc, F&& f) {
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int i0 = ti * Cfg::BI + 32 * Cfg::FR * wr + 4 * g, j0 = tj * Cfg::BJ + 32 * Cfg::FC * wc + l32;
#pragma unroll
  for (int b = 0; b < Cfg::FC; ++b)
#pragma unroll
    for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        f(i0 + 32 * a + 8 * q, j0 + 32 * b, floatx4{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]});
}

// f(i, j, eight values of rows i .. i + 7, as 16-bit elements of type T) for a lane's part of the tile, whose halves exchange their
// quads of two neighbouring blocks of eight rows for that: 16-byte stores.  make(a, b, x): the value of register x of block (a, b).
template <class Cfg, typename T, typename Make, typename F>
__device__ __forceinline__ void hp_eights(int ti, int tj, int wr, int wc, Make&& make, F&& f) {
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int i0 = ti * Cfg::BI + 32 * Cfg::FR * wr + 8 * g, j0 = tj * Cfg::BJ + 32 * Cfg::FC * wc + l32;
  typedef T vec2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int b = 0; b < Cfg::FC; ++b)
#pragma unroll
    for (int a = 0; a < Cfg::FR; ++a)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        u32x4 out;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const vec2 lo = {static_cast<T>(make(a, b, 4 * q + 2 * h)), static_cast<T>(make(a, b, 4 * q + 2 * h + 1))};
          const vec2 hi = {static_cast<T>(make(a, b, 4 * q + 4 + 2 * h)), static_cast<T>(make(a, b, 4 * q + 5 + 2 * h))};
          // lower lanes: (own quad of the first block, the upper lanes' of it); upper lanes: (the lower lanes' of the second block, own)
          const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi), false, false);
          out[h] = both[0];
          out[2 + h] = both[1];
        }
        f(i0 + 32 * a + 8 * q, j0 + 32 * b, out);
      }
}

// Up to eight 16-bit elements of a row that ends at element `end`.
template <typename T>
__device__ __forceinline__ void hp_store8(T* __restrict__ row, int i, int end, u32x4 v) {
  if (i + 8 <= end) {
    __builtin_memcpy(row + i, &v, 16);
  } else {
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (i + k < end) row[i + k] = __builtin_bit_cast(T, static_cast<unsigned short>(v[k >> 1] >> 16 * (k & 1)));
  }
}

// out[j][i] = make(block a, b, register x) for a tile, as 16-bit elements, j < J, i < I, through the LDS: a wave writes whole rows of
// the tile, 512 bytes each, where stores straight from the accumulators are 32 bytes of 32 rows and keep the loads behind them waiting (the
// piece of d of 4096 x 64000 fp16, beside the forward pass's tiles of the same products, which write nothing: 1.20 times their time,
// 1.10 through the LDS).  Rows in the LDS are 16 bytes longer than in the tile, so that the banks of 16 rows differ.
template <class Cfg, typename T, typename Make>
__device__ __forceinline__ void hp_store_rows(AK_LDS unsigned char* lds, int ti, int tj, int wr, int wc, Make&& make, T* __restrict__ out, int64_t ldo, int I, int J) {
  constexpr int PITCH = Cfg::BI * 2 + 16, LANES = Cfg::BI / 8, ROWS = Cfg::THREADS / LANES;
  static_assert(Cfg::BJ * PITCH <= Cfg::LDS_ALL, "the tile fits the LDS");
  __syncthreads();                               // the panels have been read
  hp_eights<Cfg, T>(0, 0, wr, wc, make, [&](int i, int j, u32x4 v) { *reinterpret_cast<AK_LDS u32x4*>(lds + j * PITCH + 2 * i) = v; });
  __syncthreads();
  const int i = ti * Cfg::BI + 8 * (static_cast<int>(threadIdx.x) % LANES), row = static_cast<int>(threadIdx.x) / LANES;
  if (i >= I) return;
  const int rows = min(Cfg::BJ, J - tj * Cfg::BJ);
  T* __restrict__ to = out + static_cast<int64_t>(tj) * Cfg::BJ * ldo;
  AK_LDS const unsigned char* from = lds + 16 * (static_cast<int>(threadIdx.x) % LANES);
#pragma unroll 4
  for (int r = row; r < rows; r += ROWS) hp_store8(to + r * ldo, i, I, *reinterpret_cast<AK_LDS const u32x4*>(from + r * PITCH));
}

// out[j][i] = scale * D[i][j] as T
template <typename T>
struct HpStore {
  struct Params {
    T* out;
    int64_t ldo;
    int I, J;
    float scale;
    const float* factor;     // optional further one, on the device
  };
  template <class Cfg>
  static __device__ __forceinline__ void run(const Params& e, floatx16 (&acc)[Cfg::FR][Cfg::FC], int ti, int tj, int, int wr, int wc,
                                             AK_LDS unsigned char*) {
    const float s = e.factor != nullptr ? e.scale * *e.factor : e.scale;
    if constexpr (sizeof(T) == 2) {
      hp_eights<Cfg, T>(ti, tj, wr, wc, [&](int a, int b, int x) { return acc[a][b][x] * s; },
                        [&](int i, int j, u32x4 v) {
                          if (j < e.J && i < e.I) hp_store8(e.out + static_cast<int64_t>(j) * e.ldo, i, e.I, v);
                        });
    } else {
      hp_quads<Cfg>(acc, ti, tj, wr, wc, [&](int i, int j, floatx4 v) {
        if (j >= e.J || i >= e.I) return;
        T* __restrict__ to = e.out + static_cast<int64_t>(j) * e.ldo + i;
        v *= s;
        if (i + 4 <= e.I) {
          __builtin_memcpy(to, &v, 16);
        } else {
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (i + k < e.I) to[k] = v[k];
        }
      });
    }
  }
};

// sum[split][j][i] = or += D[i][j], fp32
struct HpSum {
  struct Params {
    float* sum;
    int64_t ldo, stride;     // elements between rows, between splits; rows are whole multiples of four
    int I, J, first;         // first: set, else add
  };
  template <class Cfg>
  static __device__ __forceinline__ void run(const Params& e, floatx16 (&acc)[Cfg::FR][Cfg::FC], int ti, int tj, int split, int wr, int wc,
                                             AK_LDS unsigned char*) {
    float* __restrict__ sum = e.sum + split * e.stride;
    const bool first = e.first != 0;
    hp_quads<Cfg>(acc, ti, tj, wr, wc, [&](int i, int j, floatx4 v) {
      if (j >= e.J || i >= e.I) return;
      floatx4* to = reinterpret_cast<floatx4*>(sum + static_cast<int64_t>(j) * e.ldo + i);
      *to = first ? v : *to + v;
    });
  }
};

// dst[row][c] = T(scale * factor * sum over the splits of sum[split][row][c])
template <typename T>
__device__ __forceinline__ void hp_total_part(const float* __restrict__ sum, int64_t ld, int64_t stride, int splits, int64_t rows, int cols, float scale,
                                              const float* __restrict__ factor, T* __restrict__ dst, int64_t group, int64_t groups) {
  const int64_t n = rows * ld;
  const float u = factor != nullptr ? scale * *factor : scale;
  for (int64_t i = 4 * (group * 256 + threadIdx.x); i < n; i += 4 * groups * 256) {
    const int64_t row = i / ld;
    const int c = static_cast<int>(i - row * ld);
    floatx4 t = *reinterpret_cast<const floatx4*>(sum + i);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) t += *reinterpret_cast<const floatx4*>(sum + s * stride + i);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < cols) dst[row * cols + c + k] = static_cast<T>(t[k] * u);
  }
}

template <typename T>
static __global__ __launch_bounds__(256) void hp_total_kernel(const float* __restrict__ sum, int64_t ld, int64_t stride, int splits, int64_t rows,
                                                              int cols, float scale, const float* __restrict__ factor, T* __restrict__ dst) {
  hp_total_part(sum, ld, stride, splits, rows, cols, scale, factor, dst, blockIdx.x, gridDim.x);
}

inline unsigned hp_total_groups(int64_t rows, int64_t ld) { return static_cast<unsigned>(std::min<int64_t>((rows * ld + 1023) / 1024, 8192)); }

template <typename T>
inline int hp_total(const float* sum, int64_t ld, int64_t stride, int splits, int64_t rows, int cols, float scale, const float* factor, T* dst,
                    hipStream_t stream) {
  hipLaunchKernelGGL(hp_total_kernel<T>, dim3(hp_total_groups(rows, ld)), dim3(256), 0, stream, sum, ld, stride, splits, rows, cols, scale, factor, dst);
  return check_launch();
}

// Rows at a pitch of ldo elements, zeros behind them: what the panels' loads need where an operand has another pitch or alignment.
template <typename T>
static __global__ __launch_bounds__(256) void hp_pad_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols, T* __restrict__ out, int ldo) {
  // eight columns a thread
  const int per = ldo / 8;
  const int64_t n = rows * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per;
    const int c = static_cast<int>(i - row * per) * 8;
    const T* __restrict__ from = x + row * ld + c;
    Some<T, 8> v;
    v.clear();
    if (c + 8 <= cols) {
      v.load(from);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) v.v[e] = from[e];
    }
    v.store(out + row * ldo + c);
  }
}

template <typename T>
inline int hp_pad(const T* x, int64_t ld, int64_t rows, int64_t cols, T* out, int64_t ldo, hipStream_t stream) {
  const int64_t groups = (rows * (ldo / 8) + 255) / 256;
  hipLaunchKernelGGL(hp_pad_kernel<T>, dim3(static_cast<unsigned>(groups < 1 ? 1 : groups < 16384 ? groups : 16384)), dim3(256), 0, stream, x, ld, rows,
                     static_cast<int>(cols), out, static_cast<int>(ldo));
  return check_launch();
}

// From here on the bf16 number nearest to a float32 number is infinite: the first of its pieces is the largest finite one.
constexpr float kHpLarge = 0x1.ffp127f;

// x in bf16 pieces that add up to it exactly (fp16: two, fp32: three), side by side in rows of PIECES * ldo, zeros behind the columns.
// BELOW: |x| is known to be below kHpLarge, or x is NaN.
template <int PIECES, bool BELOW = false>
__device__ __forceinline__ void hp_split(float x, __bf16 (&piece)[PIECES]) {
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    if constexpr (BELOW) {
      piece[k] = static_cast<__bf16>(x);
      x -= static_cast<float>(piece[k]);
    } else {
      const bool finite = fabsf(x) < INFINITY;
      piece[k] = static_cast<__bf16>(k == 0 && finite ? __builtin_amdgcn_fmed3f(x, -0x1.fep127f, 0x1.fep127f) : x);
      x = finite ? x - static_cast<float>(piece[k]) : 0.f;          // (infinities and NaN in the first piece alone)
    }
  }
}

template <typename T, int PIECES>
static __global__ __launch_bounds__(256) void hp_pieces_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols, __bf16* __restrict__ out, int ldo) {
  // eight columns a thread
  const int per = ldo / 8;
  const int64_t n = rows * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per;
    const int c = static_cast<int>(i - row * per) * 8;
    const T* __restrict__ from = x + row * ld + c;
    Some<T, 8> v;
    v.clear();
    if (c + 8 <= cols) {
      v.load(from);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) v.v[e] = from[e];
    }
    Some<__bf16, 8> o[PIECES];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      __bf16 piece[PIECES];
      hp_split(v.get(e), piece);
#pragma unroll
      for (int k = 0; k < PIECES; ++k) o[k].v[e] = piece[k];
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) o[k].store(out + (row * PIECES + k) * ldo + c);
  }
}

template <int PIECES, typename T>
inline int hp_pieces(const T* x, int64_t ld, int64_t rows, int64_t cols, __bf16* out, int64_t ldo, hipStream_t stream) {
  const int64_t groups = (rows * (ldo / 8) + 255) / 256;
  hipLaunchKernelGGL((hp_pieces_kernel<T, PIECES>), dim3(static_cast<unsigned>(groups < 1 ? 1 : groups < 16384 ? groups : 16384)), dim3(256), 0, stream, x, ld,
                     rows, static_cast<int>(cols), out, static_cast<int>(ldo));
  return check_launch();
}

// Both operands fp32: the six products.  pa, pb: elements between the pieces of a row.
inline HpPieces hp_six(int64_t pa, int64_t pb) {
  static constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
  HpPieces p = {6, {}, {}};
  for (int i = 0; i < 6; ++i) {
    p.a[i] = static_cast<int>(A[i] * pa * 2);
    p.b[i] = static_cast<int>(B[i] * pb * 2);
  }
  return p;
}

// B alone in pieces.
inline HpPieces hp_pieces_of_b(int count, int64_t pb) {
  HpPieces p = {count, {}, {}};
  for (int i = 0; i < count; ++i) p.b[i] = static_cast<int>((count - 1 - i) * pb * 2);
  return p;
}

// 16-bit elements whose rows the panels' loads can read where they lie.
inline bool hp_aligned(const void* x, int64_t ld, int64_t cols) {
  return cols % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

inline int64_t align_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// rows x cols, row pitch ld elements
inline HpOperand hp_operand(const void* p, int64_t ld, int64_t rows, int64_t cols, bool by_k) {
  return HpOperand{p, ld * 2, static_cast<int>(rows), static_cast<int>(align_up(cols, 8)), by_k ? align_up(cols, 8) : rows};
}

// An I x J result; the contraction in (at most) `splits` parts.
template <class Cfg>
inline HpProblem hp_problem(const HpOperand& A, const HpOperand& B, int64_t I, int64_t J, int64_t K, int splits = 1) {
  HpProblem p = {};
  p.A = A; p.B = B;
  p.K = K;
  p.k_per_split = align_up((K + splits - 1) / splits, 32);
  p.tiles_i = static_cast<int>((I + Cfg::BI - 1) / Cfg::BI);
  p.tiles_j = static_cast<int>((J + Cfg::BJ - 1) / Cfg::BJ);
  p.splits = static_cast<int>((K + p.k_per_split - 1) / p.k_per_split);
  return p;
}

// Consecutive parts of a workspace, each at a multiple of 256 bytes (without a base: their size).
struct Carver {
  unsigned char* base;
  size_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* at = base != nullptr ? reinterpret_cast<T*>(base + used) : nullptr;
    used += static_cast<size_t>(align_up(count * static_cast<int64_t>(sizeof(T)), 256));
    return at;
  }
};

template <bool A_BY_K, bool B_BY_K, bool PIECES = false>
using HpWide = HpCfg<2, 4, 4, 2, A_BY_K, B_BY_K, 4, PIECES>;      // 256 x 256
template <bool A_BY_K, bool B_BY_K, bool PIECES = false>
using HpSmall = HpCfg<2, 2, 2, 2, A_BY_K, B_BY_K, 4, PIECES>;     // 128 x 128
template <bool A_BY_K, bool B_BY_K, bool PIECES = false>
using HpTiny = HpCfg<2, 2, 1, 1, A_BY_K, B_BY_K, 4, PIECES>;      // 64 x 64

// 256 x 256 tiles, but for results that 128 x 128 ones of at most one place each cover: two of those take 0.83 of the time of one wide
// tile on a CU (1000 x 10007 x 513 in six products: 632 small tiles 126 us, 160 wide ones 97 us).
inline bool hp_wide(int64_t I, int64_t J) { return ((I + 127) / 128) * ((J + 127) / 128) > 512; }
// Tiles of 64 where those of 128 are for at most half of the CUs (533 x 865 x 2971, 35 tiles of 128: bf16 48 -> 37 us, six products 186 ->
// 126 us; 1024 x 2048 x 768, 128 of them: 14.2 -> 13.0 us, 59 -> 55 us).
inline bool hp_tiny(int64_t I, int64_t J) { return ((I + 127) / 128) * ((J + 127) / 128) <= 128; }

// go(the tile form for a product whose contraction is in one piece)
template <bool A_BY_K, bool B_BY_K, bool PIECES, typename F>
inline int hp_form(int64_t I, int64_t J, F&& go) {
  return hp_wide(I, J) ? go(HpWide<A_BY_K, B_BY_K, PIECES>{}) : hp_tiny(I, J) ? go(HpTiny<A_BY_K, B_BY_K, PIECES>{}) : go(HpSmall<A_BY_K, B_BY_K, PIECES>{});
}

// The device's LDS is more than a kernel has without asking; once a kernel and device.
template <typename Kernel>
inline int hp_ask_lds(Kernel kernel, int bytes, std::atomic<uint64_t>& known) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return AK_ERR_LAUNCH;
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (known.load(std::memory_order_relaxed) & bit) != 0) return AK_OK;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return AK_ERR_LAUNCH;
  if (device < 64) known.fetch_or(bit, std::memory_order_relaxed);
  return AK_OK;
}

inline int64_t hp_blocks(const HpProblem& p) { return static_cast<int64_t>(p.tiles_i) * p.tiles_j * p.splits; }

template <class Cfg, typename E, class Epilogue>
inline int hp_launch(const HpProblem& p, const typename Epilogue::Params& e, hipStream_t stream) {
  const int64_t blocks = hp_blocks(p);
  if (blocks <= 0) return AK_OK;
  if (!fits_a_launch(blocks, Cfg::THREADS)) return AK_ERR_TOO_LARGE;
  auto kernel = hp_kernel<Cfg, E, Epilogue>;
  static std::atomic<uint64_t> known{0};
  const int rc = hp_ask_lds(kernel, Cfg::LDS_ALL, known);
  if (rc != AK_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(Cfg::THREADS), Cfg::LDS_ALL, stream, p, e);
  return check_launch();
}

// The product whose work groups take longer goes first.
template <class Cfg1, class Epilogue1, class Cfg2, class Epilogue2, typename E>
inline int hp_launch_both(const HpProblem& p1, const typename Epilogue1::Params& e1, const HpProblem& p2, const typename Epilogue2::Params& e2,
                          hipStream_t stream) {
  const int64_t b1 = hp_blocks(p1), b2 = hp_blocks(p2);
  if (!fits_a_launch(b1 + b2, Cfg1::THREADS)) return AK_ERR_TOO_LARGE;
  auto kernel = hp_both_kernel<Cfg1, Epilogue1, Cfg2, Epilogue2, E>;
  static std::atomic<uint64_t> known{0};
  const int rc = hp_ask_lds(kernel, Cfg1::LDS_ALL, known);
  if (rc != AK_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(b1 + b2)), dim3(Cfg1::THREADS), Cfg1::LDS_ALL, stream, p1, e1, static_cast<uint32_t>(b1), p2, e2,
                     static_cast<uint32_t>(b2), p2.k_per_split > p1.k_per_split ? 1 : 0);
  return check_launch();
}

}  // namespace ak
