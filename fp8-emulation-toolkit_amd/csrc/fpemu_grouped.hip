// fpemu_grouped.hip -- matrix products by group: each run of rows offsets[g] .. offsets[g + 1] of one matrix is multiplied
// by its own weight matrix (the experts of a model, each seeing the tokens routed to it), and the gradients of both sides.
// How many rows a group has is known on the device only: the grid covers the largest number of tiles that M rows in G
// groups can need, and each workgroup finds its group and rows from the offsets.
//   y  = x W_g       rows of one group x columns of W_g, contraction over K
//   dx = dy W_g^T    the same product with the other weight layout
//   dW_g = x_g^T dy_g   contraction over the group's rows: both operands have it in their slow dimension
// 16-bit storage: v_mfma_f32_32x32x16, fp32 sums.  fp32 storage: v_mfma_f32_32x32x2_f32, the k-ascending fmaf chain.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <type_traits>

#include "../../include/fpemu_hip.h"
#include "fpemu_common.hpp"

using namespace fpemu;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

int fail(int code, const char *who, const char *what) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  fpemu_set_error_(msg);
  return code;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- which rows a workgroup works on -----------------------------------------------------------------------------------
struct RowTile {
  int64_t first, end;   // rows [first, end) of the tile
  int group;            // -1: rows of no group (zeros)
};

__device__ __forceinline__ int64_t row_at(const int32_t *offsets, int64_t g, int64_t M) {
  const int64_t o = offsets[g];
  return o < 0 ? 0 : o > M ? M : o;
}

// Tiles of BM rows are numbered group after group, then the rows before the first and behind the last group.  64 groups at a
// time, one per lane: tiles per group and a prefix sum over the wave; a ballot finds the group that holds a tile.
template <int BM> struct TileMap {
  const int32_t *offsets;
  int64_t groups, M;
  uint32_t grouped, heads, tails;   // tiles of the groups, before the first, behind the last
  int64_t head, tail;

  struct Lane { int64_t lo, hi; uint32_t mine, inc; };
  __device__ __forceinline__ Lane scan(int64_t g0) const {
    const unsigned lane = threadIdx.x & 63u;
    Lane l{0, 0, 0, 0};
    if (g0 + lane < groups) {
      l.lo = row_at(offsets, g0 + lane, M);
      l.hi = row_at(offsets, g0 + lane + 1, M);
    }
    l.inc = l.mine = l.hi > l.lo ? (uint32_t)((l.hi - l.lo + BM - 1) / BM) : 0u;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)l.inc, off, 64);
      if ((int)lane >= off) l.inc += o;
    }
    return l;
  }
  __device__ __forceinline__ TileMap(const int32_t *o, int64_t g, int64_t m) : offsets(o), groups(g), M(m), grouped(0) {
    for (int64_t g0 = 0; g0 < groups; g0 += 64) grouped += (uint32_t)__shfl((int)scan(g0).inc, 63, 64);
    head = row_at(offsets, 0, M);
    tail = row_at(offsets, groups, M);
    heads = (uint32_t)((head + BM - 1) / BM);
    tails = (uint32_t)((M - tail + BM - 1) / BM);
  }
  __device__ __forceinline__ uint32_t tiles() const { return __builtin_amdgcn_readfirstlane(grouped + heads + tails); }
  __device__ __forceinline__ RowTile find(uint32_t tile) const {
    RowTile r;
    uint32_t before = 0;
    for (int64_t g0 = 0; tile < grouped && g0 < groups; g0 += 64) {
      const Lane l = scan(g0);
      const uint32_t all = (uint32_t)__shfl((int)l.inc, 63, 64);
      if (tile < before + all) {
        const int at = __ffsll((unsigned long long)__ballot(before + l.inc > tile)) - 1;
        const uint32_t start = before + (uint32_t)__shfl((int)(l.inc - l.mine), at, 64);
        const int64_t lo = __shfl((long long)l.lo, at, 64), hi = __shfl((long long)l.hi, at, 64);
        r.first = lo + (int64_t)(tile - start) * BM;
        r.end = r.first + BM < hi ? r.first + BM : hi;
        r.group = (int)(g0 + at);
        return r;
      }
      before += all;
    }
    const uint32_t t = tile - grouped;
    r.group = -1;
    r.first = t < heads ? (int64_t)t * BM : tail + (int64_t)(t - heads) * BM;
    const int64_t end = t < heads ? head : M;
    r.end = r.first + BM < end ? r.first + BM : end;
    return r;
  }
};

// ---- any sizes, any alignment: 128 x 128 tiles, elements staged one by one --------------------------------------------------
constexpr int GT = 128;
template <int DT> struct Gen {
  static constexpr int BK = DT == FPEMU_F32 ? 16 : 32;
  static constexpr int LD = DT == FPEMU_F32 ? BK + 1 : BK + 8;
};

// element (r, k) of an operand: p[r * ld + k], or p[k * ld + r] where the contraction is its slow dimension (COL)
template <int DT, bool COL>
__device__ __forceinline__ void stage(typename Storage<DT>::elem *lds, const typename Storage<DT>::elem *p, int64_t ld, int64_t r0,
                                      int64_t rend, int64_t k0, int64_t kend, typename Storage<DT>::elem pad) {
  constexpr int BK = Gen<DT>::BK, LD = Gen<DT>::LD;
  for (int i = threadIdx.x; i < GT * BK; i += 256) {
    const int r = COL ? i % GT : i / BK, k = COL ? i / GT : i % BK;
    const int64_t gr = r0 + r, gk = k0 + k;
    lds[r * LD + k] = gr < rend && gk < kend ? (COL ? p[gk * ld + gr] : p[gr * ld + gk]) : pad;
  }
}

template <int DT, bool A_COL, bool B_COL>
__device__ __forceinline__ void tile_product(const typename Storage<DT>::elem *a, int64_t lda, int64_t ar0, int64_t arend,
                                             const typename Storage<DT>::elem *b, int64_t ldb, int64_t br0, int64_t brend, int64_t k0,
                                             int64_t kend, f32x16 (&acc)[2][2]) {
  using elem = typename Storage<DT>::elem;
  constexpr int BK = Gen<DT>::BK, LD = Gen<DT>::LD;
  __shared__ __attribute__((aligned(16))) elem as[GT * LD];
  __shared__ __attribute__((aligned(16))) elem bs[GT * LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  elem apad = 0, bpad = 0;
  if constexpr (DT == FPEMU_F32) apad = -0.0f;   // products of the ragged end are -0: they leave any chain as it is
  for (int64_t k = k0; k < kend; k += BK) {
    stage<DT, A_COL>(as, a, lda, ar0, arend, k, kend, apad);
    stage<DT, B_COL>(bs, b, ldb, br0, brend, k, kend, bpad);
    __syncthreads();
    if constexpr (DT == FPEMU_F32) {
#pragma unroll
      for (int kk = 0; kk < BK; kk += 2) {
        float av[2], bv[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          av[i] = as[(wr + i * 32 + (lane & 31)) * LD + kk + (lane >> 5)];
          bv[i] = bs[(wc + i * 32 + (lane & 31)) * LD + kk + (lane >> 5)];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(av[i], bv[j], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < BK; kk += 16) {
        u32x4 av[2], bv[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          av[i] = *(const u32x4 *)&as[(wr + i * 32 + (lane & 31)) * LD + kk + (lane >> 5) * 8];
          bv[i] = *(const u32x4 *)&bs[(wc + i * 32 + (lane & 31)) * LD + kk + (lane >> 5) * 8];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            if constexpr (DT == FPEMU_BF16)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, av[i]), __builtin_bit_cast(bf16x8, bv[j]),
                                                                  acc[i][j], 0, 0, 0);
            else
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, av[i]), __builtin_bit_cast(f16x8, bv[j]),
                                                                 acc[i][j], 0, 0, 0);
          }
      }
    }
    __syncthreads();
  }
}

template <int DT>
__device__ __forceinline__ void tile_store(typename Storage<DT>::elem *c, int64_t ldc, int64_t r0, int64_t rend, int64_t c0, int64_t cend,
                                           const f32x16 (&acc)[2][2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t col = c0 + wc + j * 32 + (lane & 31);
      if (col >= cend) continue;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int64_t row = r0 + wr + i * 32 + (e / 4) * 8 + (lane >> 5) * 4 + (e & 3);
        if (row >= rend) continue;
        const float v = acc[i][j][e] + 0.0f;   // the chain's -0 is written as the c-model writes it
        if constexpr (DT == FPEMU_F32) c[row * ldc + col] = v;
        else c[row * ldc + col] = (typename Storage<DT>::elem)store_elem16<DT>(v);
      }
    }
}

template <int DT, bool W_TRANS>
__global__ __launch_bounds__(256) void grouped_any_kernel(typename Storage<DT>::elem *y, const typename Storage<DT>::elem *x,
                                                          const typename Storage<DT>::elem *w, const int32_t *offsets, int64_t M,
                                                          int64_t N, int64_t K, int64_t groups, uint32_t col_tiles) {
  const TileMap<GT> map(offsets, groups, M);
  if (blockIdx.x / col_tiles >= map.tiles()) return;
  const RowTile r = map.find(blockIdx.x / col_tiles);
  const int64_t c0 = (int64_t)(blockIdx.x % col_tiles) * GT;
  f32x16 acc[2][2] = {};
  if (r.group >= 0) {
    const typename Storage<DT>::elem *wg = w + (int64_t)r.group * K * N;
    tile_product<DT, false, !W_TRANS>(x, K, r.first, r.end, wg, W_TRANS ? K : N, c0, N, 0, K, acc);
  }
  tile_store<DT>(y, N, r.first, r.end, c0, N, acc);
}

template <int DT>
__global__ __launch_bounds__(256) void grouped_wgrad_any_kernel(typename Storage<DT>::elem *dw, const typename Storage<DT>::elem *a,
                                                                const typename Storage<DT>::elem *b, const int32_t *offsets,
                                                                int64_t M, int64_t P, int64_t Q, uint32_t ptiles, uint32_t qtiles) {
  const uint32_t g = blockIdx.x / (ptiles * qtiles), t = blockIdx.x % (ptiles * qtiles);
  const int64_t p0 = (int64_t)(t / qtiles) * GT, q0 = (int64_t)(t % qtiles) * GT;
  const int64_t lo = row_at(offsets, g, M), hi = row_at(offsets, (int64_t)g + 1, M);
  f32x16 acc[2][2] = {};
  tile_product<DT, true, true>(a, P, p0, P, b, Q, q0, Q, lo, hi, acc);
  tile_store<DT>(dw + (int64_t)g * P * Q, Q, p0, P, q0, Q, acc);
}

// ---- 16-bit storage in whole 16-byte vectors: tiles fed by loads that go straight to LDS ----------------------------------
// A tile of BM rows x BN columns, 64 deep in k per stage; while one stage is multiplied the next ones are on their way.
// A stage row of 64 k is 128 bytes, a whole cache line: with 32 deep stages every line was fetched twice (it had left the
// 32 KB L1 before its second half was asked for), and the tiles then ran at the rate of the L2, not of the matrix cores.
// An operand whose contraction is contiguous lies in LDS as rows of 128 bytes and is read 16 bytes a lane; one whose
// contraction is its slow dimension lies as it is in memory and is read through the transposing LDS read (of 16 lanes, lane
// i gets column i of 4 k-rows).  The loads write LDS linearly, so the bank swizzle is applied to the global address a lane
// fetches and undone where the fragment is read.
// Waves: WM x WN over the tile.
constexpr int FK = 64;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(const lds_char *)p; }

// 16 bytes per lane from base + off into LDS at `lds` + 16 * lane.  (Writing M0 needs a wait state before its use.)
__device__ __forceinline__ void load_to_lds(uint32_t lds, const void *base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() {   // all but the last N loads have arrived, all LDS reads too
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}

template <int BM_, int BN_, int WM_, int WN_, int STAGES_> struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr int THREADS = WM * WN * 64;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;   // matrix tiles of a wave
  static constexpr int A_BYTES = BM * FK * 2, B_BYTES = BN * FK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int OUT_LD = BN + 8;   // elements; the finished tile goes through LDS to be stored in whole rows
  static constexpr int OUT = BM * OUT_LD * 2, LDS = STAGES * STAGE > OUT ? STAGES * STAGE : OUT;
};

// One operand's tile: EXT entries (rows of a row operand, columns of a COL operand) x FK of the contraction.
template <bool COL, int EXT, int THREADS> struct Panel {
  static constexpr int LOADS = EXT * FK * 2 / 16 / THREADS;   // per thread and stage
  static_assert(LOADS * THREADS * 16 == EXT * FK * 2, "whole vectors per thread");
  const char *base;      // uniform: the tile's first element at the stage's first k
  int64_t step;          // bytes from stage to stage
  uint32_t off[LOADS];   // per thread: byte offsets of its vectors in the tile

  // entries beyond `lim` are fetched from inside (they only feed results that are not stored)
  __device__ __forceinline__ void set(const void *p, int64_t ld, int lim) {
    base = (const char *)p;
    step = (COL ? ld : 1) * FK * 2;
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      int outer, k;
      place(j, outer, k);
      if (COL) off[j] = (uint32_t)(k * ld + (outer + 8 <= lim ? outer : lim - 8)) * 2u;
      else off[j] = (uint32_t)((outer < lim ? outer : lim - 1) * ld + k) * 2u;
    }
  }
  // entry and k of the first element of this thread's vector j
  __device__ __forceinline__ static void place(int j, int &outer, int &k) {
    const int id = j * THREADS + (int)threadIdx.x;
    if (COL) {
      constexpr int PER = EXT / 8;
      k = id / PER;
      outer = ((id % PER) ^ swizzle_col(k)) * 8;
    } else {
      outer = id / 8;
      k = ((id & 7) ^ swizzle_row(outer)) * 8;
    }
  }
  // in vectors of 16 bytes: 16 rows that are read together lie in 16 different places of 256 bytes
  __device__ __forceinline__ static int swizzle_row(int row) { return (row >> 1) & 7; }
  // four k-rows of a transposing read go to different banks
  __device__ __forceinline__ static int swizzle_col(int k) { return EXT >= 128 ? (k & 3) * 4 : EXT >= 64 ? (k & 1) * 4 : 0; }
  __device__ __forceinline__ void fetch(uint32_t wave_lds, int j) const {   // wave_lds: where the wave's first vector goes
    load_to_lds(wave_lds + (uint32_t)(j * THREADS * 16), base, off[j]);
  }
  // the last, partial stage: `left` of the contraction, zeros behind
  __device__ __forceinline__ void fetch_tail(char *lds, int left) const {
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      int outer, k;
      place(j, outer, k);
      u32x4 v = {0u, 0u, 0u, 0u};
      if (k < left) v = *(const u32x4 *)(base + off[j]);
      *(u32x4 *)(lds + (j * THREADS + (int)threadIdx.x) * 16) = v;
    }
  }
  // Where a lane finds its fragments in the tile: a matrix operand of 32 entries, 16 of k: lane l has entry l % 32,
  // k = (l / 32) * 8 + 0..7.  The places for the four k-steps of a stage are kept; further entries are a constant away.
  uint32_t frag[COL ? 1 : 4];
  __device__ __forceinline__ void set_fragments(int at) {
    const int lane = threadIdx.x & 63;
    if constexpr (COL) {
      const int i = lane & 15, g = lane >> 4, k = (g >> 1) * 8 + (i >> 2), col = at + (g & 1) * 16 + (i & 3) * 4;
      frag[0] = (uint32_t)(k * (EXT * 2) + (((col >> 3) ^ swizzle_col(k)) * 16) + (col & 7) * 2);
    } else {
      const int row = at + (lane & 31);
#pragma unroll
      for (int s = 0; s < 4; s++) frag[s] = (uint32_t)(row * (FK * 2) + (((s * 2 + (lane >> 5)) ^ swizzle_row(row)) * 16));
    }
  }
  // the operand `tile` tiles of 32 entries further on, k-step `step` (both known at compile time), of the stage at `lds`
  __device__ __forceinline__ u32x4 fragment(const char *lds, int tile, int step) const {
    if constexpr (COL) {
      u32x4 r;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        // entries 32 further on are 4 vectors away: an exclusive or where the swizzle may touch the same bits
        const uint32_t where = (frag[0] ^ (uint32_t)(tile * 64)) + (uint32_t)((step * 16 + h * 4) * (EXT * 2));
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + where));
        const uint2 w = __builtin_bit_cast(uint2, v);
        r[2 * h] = w.x;
        r[2 * h + 1] = w.y;
      }
      return r;
    } else {
      return *(const u32x4 *)(lds + frag[step] + (uint32_t)(tile * 32 * FK * 2));
    }
  }
};

template <int DT> __device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == FPEMU_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// acc[i][j]: entries wa + 32 i of A (its columns) and wb + 32 j of B (its rows): a lane holds 4 neighbours along B.
// idle: this wave's part of the tile has no rows (it still loads and waits with the others).
template <int DT, class S, bool A_COL, bool B_COL>
__device__ __forceinline__ void fast_product(char *smem, Panel<A_COL, S::BM, S::THREADS> &a, Panel<B_COL, S::BN, S::THREADS> &b, int full,
                                             int left, bool idle, f32x16 (&acc)[S::TM][S::TN]) {
  using PA = Panel<A_COL, S::BM, S::THREADS>;
  using PB = Panel<B_COL, S::BN, S::THREADS>;
  constexpr int AHEAD = S::STAGES - 1, LOADS = PA::LOADS + PB::LOADS, STEPS = FK / 16, TILES = S::TM * S::TN;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem) + (threadIdx.x & ~63u) * 16u);
  const int stages = full + (left ? 1 : 0);
  int put = 0, get = 0;   // bytes: the stage being filled, the stage being read
  auto load = [&](int j) {
    if (j < PA::LOADS) a.fetch(lds0 + put, j);
    else b.fetch(lds0 + put + S::A_BYTES, j - PA::LOADS);
  };
  auto filled = [&]() {
    put = put + S::STAGE == S::STAGES * S::STAGE ? 0 : put + S::STAGE;
    a.base += a.step;
    b.base += b.step;
  };
  // The loads of a stage are spread over the matrix instructions of three steps (slots 0 .. 3 TILES): issued in one go they
  // fill the memory pipeline's queue and every wave stands before it with its matrix instructions undone.
  auto loads_at = [&](int slot) {
#pragma unroll
    for (int j = 0; j < LOADS; j++)
      if (j * 3 * TILES / LOADS == slot) load(j);
  };
  auto tail = [&](int t) {   // stages that are not whole: the partial one, or nothing
    if (t == full && left) {
      a.fetch_tail(smem + put, left);
      b.fetch_tail(smem + put + S::A_BYTES, left);
    }
    filled();
  };
  // Stage t is here once all loads but those of the stages behind it have arrived, for every wave.
  auto arrive = [&](int t) {
    if (t + AHEAD - 1 < full) wait_loads<(AHEAD - 1) * LOADS>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
  };
  u32x4 av[2][S::TM], bv[2][S::TN];
  auto read = [&](int set, int step) {
    const char *sa = smem + get, *sb = sa + S::A_BYTES;
#pragma unroll
    for (int j = 0; j < S::TN; j++) bv[set][j] = b.fragment(sb, j, step);
#pragma unroll
    for (int i = 0; i < S::TM; i++) av[set][i] = a.fragment(sa, i, step);
  };
  // One stage.  The fragments of the next step are read while the current one's are multiplied; the step that ends a stage
  // waits for the next stage first, so the barrier and the first reads of a stage hide behind matrix instructions too.
  auto stage = [&](auto works, int t, bool loads_now, bool loads_next) {
    constexpr bool WORKS = decltype(works)::value;
#pragma unroll
    for (int step = 0; step < STEPS; step++) {
      const int set = step & 1, next = set ^ 1;
      const bool ends = step + 1 == STEPS;
      if (!ends) {
        if (WORKS) read(next, step + 1);
      } else if (t + 1 < stages) {
        arrive(t + 1);
        get = get + S::STAGE == S::STAGES * S::STAGE ? 0 : get + S::STAGE;
        if (WORKS) read(next, 0);
        if (!loads_next) tail(t + 1 + AHEAD);
      }
      const bool loads = ends ? loads_next : loads_now && step < 2;
      const int slot0 = ends ? 0 : (step + 1) * TILES;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < S::TM; i++)
#pragma unroll
        for (int j = 0; j < S::TN; j++) {
          if (WORKS) acc[i][j] = mfma16<DT>(bv[set][j], av[set][i], acc[i][j]);
          if (loads) {
            loads_at(slot0 + i * S::TN + j);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      if (loads_now && step == 1) filled();
    }
  };
#pragma unroll
  for (int t = 0; t < AHEAD; t++) {
    if (t < full) {
#pragma unroll
      for (int j = 0; j < LOADS; j++) load(j);
      filled();
    } else {
      tail(t);
    }
  }
  auto run = [&](auto works) {
    arrive(0);
    if (decltype(works)::value) read(0, 0);
    if (AHEAD < full) {
#pragma unroll
      for (int slot = 0; slot < TILES; slot++) loads_at(slot);
    } else {
      tail(AHEAD);
    }
    int t = 0;
    for (; t + 1 + AHEAD < full; t++) stage(works, t, true, true);
    for (; t < stages; t++) stage(works, t, t + AHEAD < full, false);
  };
  if (idle) run(std::false_type());   // the same waits and barriers
  else run(std::true_type());
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();   // the stages are free
}

// The tile through LDS to memory in whole rows; rows < rlim, columns < clim (a multiple of 8).
template <int DT, class S>
__device__ __forceinline__ void fast_store(char *smem, uint16_t *c, int64_t ldc, int rlim, int clim, int wa, int wb,
                                           const f32x16 (&acc)[S::TM][S::TN]) {
  const int lane = threadIdx.x & 63;
  uint16_t *t = (uint16_t *)smem;
#pragma unroll
  for (int i = 0; i < S::TM; i++)
#pragma unroll
    for (int j = 0; j < S::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int row = wa + i * 32 + (lane & 31), col = wb + j * 32 + (e / 4) * 8 + (lane >> 5) * 4;
        const uint2 v = {pack_pair16<DT>(acc[i][j][e], acc[i][j][e + 1]), pack_pair16<DT>(acc[i][j][e + 2], acc[i][j][e + 3])};
        *(uint2 *)(t + row * S::OUT_LD + col) = v;
      }
  __syncthreads();
  constexpr int PER = S::BN / 8;
  const int col = (threadIdx.x % PER) * 8;
  if (col < clim)
    for (int row = threadIdx.x / PER; row < rlim; row += S::THREADS / PER)
      *(u32x4 *)(c + row * ldc + col) = *(const u32x4 *)(t + row * S::OUT_LD + col);
}

// Workgroup b runs on XCD b % 8: each XCD gets an eighth of the tiles, one after the other, so that neighbours share rows of
// x and a group's weights in its L2.
constexpr uint32_t NO_TILE = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t xcd_tile(uint32_t b, uint32_t tiles) {
  const uint32_t share = (tiles + 7u) / 8u, at = b >> 3;
  const uint32_t id = (b & 7u) * share + at;
  return at < share && id < tiles ? id : NO_TILE;
}

// Row and column tile of number id: bands of four row tiles, down the band first, so that the tiles an XCD works on at one
// time are about as high as wide and share what they read.
__device__ __forceinline__ void banded(uint32_t id, uint32_t row_tiles, uint32_t col_tiles, uint32_t &row, uint32_t &col) {
  const uint32_t band = id / (4u * col_tiles), in = id - band * 4u * col_tiles;
  const uint32_t high = row_tiles - band * 4u < 4u ? row_tiles - band * 4u : 4u;
  row = band * 4u + in % high;
  col = in / high;
}

template <class S> struct WaveAt {   // a wave's part of the tile; waves that share a SIMD (w, w + 4) differ in their rows
  int wa, wb;
  __device__ __forceinline__ WaveAt() {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    wb = (wave % S::WN) * (S::BN / S::WN);
    wa = (wave / S::WN) * (S::BM / S::WM);
  }
};

template <int DT, bool W_TRANS, class S>
__global__ __launch_bounds__(S::THREADS) void grouped_fast_kernel(uint16_t *y, const uint16_t *x, const uint16_t *w, const int32_t *offsets,
                                                                  int64_t M, int64_t N, int64_t K, int64_t groups, uint32_t col_tiles) {
  __shared__ __attribute__((aligned(16))) char smem[S::LDS];
  const TileMap<S::BM> map(offsets, groups, M);
  const uint32_t id = xcd_tile(blockIdx.x, map.tiles() * col_tiles);
  if (id == NO_TILE) return;
  uint32_t row_tile, col_tile;
  banded(id, map.tiles(), col_tiles, row_tile, col_tile);
  const RowTile r = map.find(row_tile);
  const int64_t first = __builtin_amdgcn_readfirstlane((int)r.first), c0 = (int64_t)col_tile * S::BN;
  const int group = __builtin_amdgcn_readfirstlane(r.group), rows = __builtin_amdgcn_readfirstlane((int)(r.end - r.first));
  const int cols = (int)(N - c0 < S::BN ? N - c0 : S::BN);
  const WaveAt<S> at;
  f32x16 acc[S::TM][S::TN] = {};
  if (group >= 0) {
    const uint16_t *wg = w + (int64_t)group * K * N;
    Panel<false, S::BM, S::THREADS> a;
    Panel<!W_TRANS, S::BN, S::THREADS> b;
    a.set(x + first * K, K, rows);
    b.set(W_TRANS ? wg + c0 * K : wg + c0, W_TRANS ? K : N, cols);
    a.set_fragments(at.wa);
    b.set_fragments(at.wb);
    fast_product<DT, S, false, !W_TRANS>(smem, a, b, (int)(K / FK), (int)(K % FK), at.wa >= rows || at.wb >= cols, acc);
  }
  fast_store<DT, S>(smem, y + first * N + c0, N, rows, cols, at.wa, at.wb, acc);
}

template <int DT, class S>
__global__ __launch_bounds__(S::THREADS) void grouped_wgrad_fast_kernel(uint16_t *dw, const uint16_t *a, const uint16_t *b,
                                                                        const int32_t *offsets, int64_t M, int64_t P, int64_t Q,
                                                                        uint32_t ptiles, uint32_t qtiles, uint32_t tiles) {
  __shared__ __attribute__((aligned(16))) char smem[S::LDS];
  const uint32_t id = xcd_tile(blockIdx.x, tiles);
  if (id == NO_TILE) return;
  const uint32_t g = id / (ptiles * qtiles);
  uint32_t pt, qt;
  banded(id % (ptiles * qtiles), ptiles, qtiles, pt, qt);
  const int64_t p0 = (int64_t)pt * S::BM, q0 = (int64_t)qt * S::BN;
  const int64_t lo = row_at(offsets, g, M), hi = row_at(offsets, (int64_t)g + 1, M);
  const int plim = (int)(P - p0 < S::BM ? P - p0 : S::BM), qlim = (int)(Q - q0 < S::BN ? Q - q0 : S::BN);
  const WaveAt<S> at;
  f32x16 acc[S::TM][S::TN] = {};
  if (hi > lo) {
    Panel<true, S::BM, S::THREADS> pa;
    Panel<true, S::BN, S::THREADS> pb;
    pa.set(a + lo * P + p0, P, plim);
    pb.set(b + lo * Q + q0, Q, qlim);
    pa.set_fragments(at.wa);
    pb.set_fragments(at.wb);
    fast_product<DT, S, true, true>(smem, pa, pb, (int)((hi - lo) / FK), (int)((hi - lo) % FK), at.wa >= plim || at.wb >= qlim, acc);
  }
  fast_store<DT, S>(smem, dw + (int64_t)g * P * Q + p0 * Q + q0, Q, plim, qlim, at.wa, at.wb, acc);
}

using Large = Shape<256, 256, 2, 4, 2>;
using Medium = Shape<128, 128, 2, 2, 2>;

// Whole 16-byte vectors everywhere, and offsets within a tile that fit 32 bits.
bool fast_rows(const void *p, int64_t ld) { return (uintptr_t)p % 16u == 0 && ld % 8 == 0 && ld <= 1 << 21; }

int check_grouped(const char *who, const void *c, const void *a, const void *b, const int32_t *offsets, int64_t M, int64_t N, int64_t K,
                  int64_t groups, int dtype) {
  if (dtype < FPEMU_F32 || dtype > FPEMU_BF16) return fail(FPEMU_EINVAL, who, "bad dtype id");
  if (M < 0 || N < 0 || K < 0 || groups < 1) return fail(FPEMU_EINVAL, who, "sizes are not negative, and there is a group at least");
  if (M > 0x7FFFFFFFll || N > 0x7FFFFFFFll || K > 0x7FFFFFFFll || groups > 0x7FFFFFFFll)
    return fail(FPEMU_EINVAL, who, "a size is over 2^31 - 1");
  if (offsets == nullptr) return fail(FPEMU_EINVAL, who, "null offsets");
  if (((uintptr_t)offsets) % 4u) return fail(FPEMU_EALIGN, who, "offsets not aligned");
  for (const void *p : {c, a, b})
    if ((uintptr_t)p % elem_size(dtype)) return fail(FPEMU_EALIGN, who, "buffer not aligned to its element size");
  return FPEMU_OK;
}

int launched(const char *who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FPEMU_OK : fail((int)e, who, hipGetErrorString(e));
}

template <int DT>
void run_grouped(void *y, const void *x, const void *w, const int32_t *offsets, int64_t M, int64_t N, int64_t K, int64_t groups,
                 int w_trans, unsigned blocks, uint32_t cols, hipStream_t s) {
  using elem = typename Storage<DT>::elem;
  if (w_trans)
    grouped_any_kernel<DT, true><<<blocks, 256, 0, s>>>((elem *)y, (const elem *)x, (const elem *)w, offsets, M, N, K, groups, cols);
  else
    grouped_any_kernel<DT, false><<<blocks, 256, 0, s>>>((elem *)y, (const elem *)x, (const elem *)w, offsets, M, N, K, groups, cols);
}

}  // namespace

extern "C" int fpemu_grouped_gemm(void *y, const void *x, const void *w, const int32_t *offsets, int64_t M, int64_t N, int64_t K,
                                  int64_t groups, int dtype, int w_trans, void *stream) {
  const char *who = "fpemu_grouped_gemm";
  if (const int rc = check_grouped(who, y, x, w, offsets, M, N, K, groups, dtype)) return rc;
  if (M == 0 || N == 0) return FPEMU_OK;
  if (y == nullptr || (K > 0 && (x == nullptr || w == nullptr))) return fail(FPEMU_EINVAL, who, "null buffer");
  const int64_t cols = ceil_div(N, GT), rows = ceil_div(M, GT) + groups + 2;   // every group may end in a partial tile
  if (rows * cols > 0x7FFFFFFFll) return fail(FPEMU_EINVAL, who, "too many tiles for one launch");
  hipStream_t s = (hipStream_t)stream;
  if (dtype != FPEMU_F32 && K > 0 && fast_rows(y, N) && fast_rows(x, K) && fast_rows(w, N)) {
    static const char *force = getenv("FPEMU_GROUPED_SHAPE");
    auto shape = [&](auto tag) {
      using S = decltype(tag);
      const int64_t ct = ceil_div(N, S::BN), rt = ceil_div(M, S::BM) + groups + 2;
      if (rt * ct > 0x7FFFFFF0ll) return false;
      const unsigned blocks = (unsigned)(ceil_div(rt * ct, 8) * 8);
      auto go = [&](auto kernel) {
        kernel<<<blocks, S::THREADS, 0, s>>>((uint16_t *)y, (const uint16_t *)x, (const uint16_t *)w, offsets, M, N, K, groups, (uint32_t)ct);
      };
      if (dtype == FPEMU_F16) w_trans ? go(grouped_fast_kernel<FPEMU_F16, true, S>) : go(grouped_fast_kernel<FPEMU_F16, false, S>);
      else w_trans ? go(grouped_fast_kernel<FPEMU_BF16, true, S>) : go(grouped_fast_kernel<FPEMU_BF16, false, S>);
      return true;
    };
    const int f = force ? atoi(force) : -1;
    const bool done = f == 0 ? shape(Large()) : f == 1 ? shape(Medium()) : M >= 512 * groups ? shape(Large()) : shape(Medium());
    if (done) return launched(who);
  }
  const unsigned blocks = (unsigned)(rows * cols);
  if (dtype == FPEMU_F32) run_grouped<FPEMU_F32>(y, x, w, offsets, M, N, K, groups, w_trans, blocks, (uint32_t)cols, s);
  else if (dtype == FPEMU_F16) run_grouped<FPEMU_F16>(y, x, w, offsets, M, N, K, groups, w_trans, blocks, (uint32_t)cols, s);
  else run_grouped<FPEMU_BF16>(y, x, w, offsets, M, N, K, groups, w_trans, blocks, (uint32_t)cols, s);
  return launched(who);
}

extern "C" int fpemu_grouped_gemm_wgrad(void *dw, const void *a, const void *b, const int32_t *offsets, int64_t M, int64_t P, int64_t Q,
                                        int64_t groups, int dtype, void *stream) {
  const char *who = "fpemu_grouped_gemm_wgrad";
  if (const int rc = check_grouped(who, dw, a, b, offsets, M, P, Q, groups, dtype)) return rc;
  if (P == 0 || Q == 0) return FPEMU_OK;
  if (dw == nullptr || (M > 0 && (a == nullptr || b == nullptr))) return fail(FPEMU_EINVAL, who, "null buffer");
  const int64_t pt = ceil_div(P, GT), qt = ceil_div(Q, GT);
  if (pt * qt > 0x7FFFFFFFll / groups) return fail(FPEMU_EINVAL, who, "too many tiles for one launch");
  hipStream_t s = (hipStream_t)stream;
  if (dtype != FPEMU_F32 && M > 0 && fast_rows(dw, Q) && fast_rows(a, P) && fast_rows(b, Q)) {
    static const char *force = getenv("FPEMU_GROUPED_SHAPE");
    auto shape = [&](auto tag) {
      using S = decltype(tag);
      const int64_t pf = ceil_div(P, S::BM), qf = ceil_div(Q, S::BN), tiles = pf * qf * groups;   // no more than the ones above
      const unsigned blocks = (unsigned)(ceil_div(tiles, 8) * 8);
      auto go = [&](auto kernel) {
        kernel<<<blocks, S::THREADS, 0, s>>>((uint16_t *)dw, (const uint16_t *)a, (const uint16_t *)b, offsets, M, P, Q, (uint32_t)pf,
                                             (uint32_t)qf, (uint32_t)tiles);
      };
      if (dtype == FPEMU_F16) go(grouped_wgrad_fast_kernel<FPEMU_F16, S>);
      else go(grouped_wgrad_fast_kernel<FPEMU_BF16, S>);
    };
    const int f = force ? atoi(force) : -1;
    if (f == 0) shape(Large());
    else shape(Medium());
    return launched(who);
  }
  const unsigned blocks = (unsigned)(pt * qt * groups);
  if (dtype == FPEMU_F32)
    grouped_wgrad_any_kernel<FPEMU_F32><<<blocks, 256, 0, s>>>((float *)dw, (const float *)a, (const float *)b, offsets, M, P, Q, (uint32_t)pt, (uint32_t)qt);
  else if (dtype == FPEMU_F16)
    grouped_wgrad_any_kernel<FPEMU_F16><<<blocks, 256, 0, s>>>((uint16_t *)dw, (const uint16_t *)a, (const uint16_t *)b, offsets, M, P, Q, (uint32_t)pt, (uint32_t)qt);
  else
    grouped_wgrad_any_kernel<FPEMU_BF16><<<blocks, 256, 0, s>>>((uint16_t *)dw, (const uint16_t *)a, (const uint16_t *)b, offsets, M, P, Q, (uint32_t)pt, (uint32_t)qt);
  return launched(who);
}
