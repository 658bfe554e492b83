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
  int group;            // -1: rows of no group (zeros), -2: nothing to do
};

__device__ __forceinline__ int64_t row_at(const int32_t *offsets, int64_t g, int64_t M) {
  const int64_t o = offsets[g];
  return o < 0 ? 0 : o > M ? M : o;
}

// Tile number `tile` of BM rows: group after group, then the rows before the first and behind the last group.  64 groups at
// a time, one per lane: tiles per group, a prefix sum over the wave, a ballot for the group that holds the tile.
template <int BM> __device__ __forceinline__ RowTile find_rows(const int32_t *offsets, int64_t groups, int64_t M, uint32_t tile) {
  const unsigned lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (int64_t g0 = 0; g0 < groups; g0 += 64) {
    const int64_t g = g0 + lane;
    int64_t lo = 0, hi = 0;
    if (g < groups) {
      lo = row_at(offsets, g, M);
      hi = row_at(offsets, g + 1, M);
    }
    const uint32_t mine = hi > lo ? (uint32_t)((hi - lo + BM - 1) / BM) : 0u;
    uint32_t inc = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)inc, off, 64);
      if ((int)lane >= off) inc += o;
    }
    const uint32_t all = (uint32_t)__shfl((int)inc, 63, 64);
    if (tile < before + all) {
      const int at = __ffsll((unsigned long long)__ballot(before + inc > tile)) - 1;
      const uint32_t start = before + (uint32_t)__shfl((int)(inc - mine), at, 64);
      const int64_t glo = __shfl((long long)lo, at, 64), ghi = __shfl((long long)hi, at, 64);
      RowTile r;
      r.first = glo + (int64_t)(tile - start) * BM;
      r.end = r.first + BM < ghi ? r.first + BM : ghi;
      r.group = (int)(g0 + at);
      return r;
    }
    before += all;
  }
  const int64_t head = row_at(offsets, 0, M), tail = row_at(offsets, groups, M);
  uint32_t t = tile - before;
  const uint32_t heads = (uint32_t)((head + BM - 1) / BM), tails = (uint32_t)((M - tail + BM - 1) / BM);
  RowTile r;
  r.group = -1;
  if (t < heads) {
    r.first = (int64_t)t * BM;
    r.end = r.first + BM < head ? r.first + BM : head;
  } else if (t - heads < tails) {
    r.first = tail + (int64_t)(t - heads) * BM;
    r.end = r.first + BM < M ? r.first + BM : M;
  } else {
    r.first = r.end = 0;
    r.group = -2;
  }
  return r;
}

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
  const RowTile r = find_rows<GT>(offsets, groups, M, blockIdx.x / col_tiles);
  if (r.group == -2) return;
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

// ---- 16-bit storage in whole 16-byte vectors: 128 x 256 tiles fed by loads that go straight to LDS -------------------------
// 4 waves, each 64 x 128 of the tile as 2 x 4 matrix tiles (128 accumulators); 32 deep in k, three LDS stages of 24 KB, so
// two stages are in flight while one is multiplied and two workgroups share a CU: one's barrier and LDS reads hide behind
// the other's matrix instructions.  A wave reads (64 + 128) x 32 bytes from LDS for 8 matrix instructions of 32 cycles, three
// quarters of what LDS delivers.  An operand whose contraction is contiguous lies in LDS as rows of 64 bytes and is read 16
// bytes a lane; one whose contraction is its slow dimension lies as it is in memory and is read through the transposing
// LDS read (lane i of 16 gets column i of 4 k-rows).  The stages are written linearly by the loads, so the bank swizzle is
// applied to the global address a lane fetches and undone where the fragment is read.
constexpr int FM = 128, FN = 256, FK = 32, STAGES = 3;
constexpr int A_BYTES = FM * FK * 2, B_BYTES = FN * FK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int OUT_LD = FN + 8;   // elements; the finished tile goes through LDS to be stored in whole rows
static_assert(FM * OUT_LD * 2 <= STAGES * STAGE_BYTES, "the tile fits where the stages were");

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(const lds_char *)p; }

// 16 bytes per lane from base + off into LDS at `lds` + 16 * lane.  (Writing M0 needs a wait state before its use.)
__device__ __forceinline__ void load_to_lds(uint32_t lds, const void *base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() {   // all but the last N loads have arrived, all LDS reads too
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}

// One operand's tile: EXT entries (rows of a row operand, columns of a COL operand) x FK of the contraction.
template <bool COL, int EXT> struct Panel {
  static constexpr int LOADS = EXT * FK * 2 / 16 / 256;   // per thread and stage
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
    const int id = j * 256 + (int)threadIdx.x;
    if (COL) {
      constexpr int PER = EXT / 8;
      k = id / PER;
      outer = ((id % PER) ^ swizzle_col(k)) * 8;
    } else {
      outer = id / 4;
      k = ((id & 3) ^ ((outer >> 1) & 3)) * 8;
    }
  }
  __device__ __forceinline__ static int swizzle_col(int k) { return (k & 3) * 4; }   // in vectors of 16 bytes
  __device__ __forceinline__ void fetch(uint32_t lds) const {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x & ~63u) * 16u);   // the wave's first vector
#pragma unroll
    for (int j = 0; j < LOADS; j++) load_to_lds(to + (uint32_t)j * 4096u, base, off[j]);
  }
  // the last, partial stage: `left` of the contraction, zeros behind
  __device__ __forceinline__ void fetch_tail(char *lds, int left) const {
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      int outer, k;
      place(j, outer, k);
      u32x4 v = {0u, 0u, 0u, 0u};
      if (k < left) v = *(const u32x4 *)(base + off[j]);
      *(u32x4 *)(lds + (j * 256 + (int)threadIdx.x) * 16) = v;
    }
  }
  // matrix operand of 32 entries from `at`, 16 of k from kk: lane l has entry l % 32, k = kk + (l / 32) * 8 + 0..7
  __device__ __forceinline__ static u32x4 fragment(const char *lds, int at, int kk) {
    const int lane = threadIdx.x & 63;
    if constexpr (COL) {
      const int i = lane & 15, g = lane >> 4;
      const int col = at + (g & 1) * 16 + (i & 3) * 4;
      u32x4 r;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = kk + (g >> 1) * 8 + h * 4 + (i >> 2);
        const int where = k * (EXT * 2) + (((col >> 3) ^ swizzle_col(k)) * 16) + (col & 7) * 2;
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + where));
        const uint2 w = __builtin_bit_cast(uint2, v);
        r[2 * h] = w.x;
        r[2 * h + 1] = w.y;
      }
      return r;
    } else {
      const int row = at + (lane & 31), c = (kk >> 3) + (lane >> 5);
      return *(const u32x4 *)(lds + row * (FK * 2) + ((c ^ ((row >> 1) & 3)) * 16));
    }
  }
};

template <int DT> __device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == FPEMU_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// acc[i][j]: entries wa + 32 i of A (its columns) and wb + 32 j of B (its rows): a lane holds 4 neighbours along B
template <int DT, bool A_COL, bool B_COL>
__device__ __forceinline__ void fast_product(char *smem, Panel<A_COL, FM> &a, Panel<B_COL, FN> &b, int full, int left, f32x16 (&acc)[2][4]) {
  constexpr int LOADS = Panel<A_COL, FM>::LOADS + Panel<B_COL, FN>::LOADS;
  const int wave = threadIdx.x >> 6, wa = (wave >> 1) * 64, wb = (wave & 1) * 128;
  const uint32_t lds0 = lds_address(smem);
  const int stages = full + (left ? 1 : 0);
  auto fetch = [&](int t) {
    const int at = (t % STAGES) * STAGE_BYTES;
    if (t < full) {
      a.fetch(lds0 + at);
      b.fetch(lds0 + at + A_BYTES);
    } else if (t < stages) {
      a.fetch_tail(smem + at, left);
      b.fetch_tail(smem + at + A_BYTES, left);
    }
    a.base += a.step;
    b.base += b.step;
  };
  fetch(0);
  fetch(1);
  for (int t = 0; t < stages; t++) {
    if (t + 1 < full) wait_loads<LOADS>();   // stage t + 1 may still be on its way
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    fetch(t + 2);                            // into the stage that everybody has read
    const char *sa = smem + (t % STAGES) * STAGE_BYTES, *sb = sa + A_BYTES;
#pragma unroll
    for (int kk = 0; kk < FK; kk += 16) {
      u32x4 av[2], bv[4];
#pragma unroll
      for (int i = 0; i < 2; i++) av[i] = Panel<A_COL, FM>::fragment(sa, wa + i * 32, kk);
#pragma unroll
      for (int j = 0; j < 4; j++) bv[j] = Panel<B_COL, FN>::fragment(sb, wb + j * 32, kk);
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = mfma16<DT>(bv[j], av[i], acc[i][j]);
    }
  }
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();   // the stages are free
}

// The tile through LDS to memory in rows of 512 bytes; rows < rlim, columns < clim (a multiple of 8).
template <int DT> __device__ __forceinline__ void fast_store(char *smem, uint16_t *c, int64_t ldc, int rlim, int clim, const f32x16 (&acc)[2][4]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wa = (wave >> 1) * 64, wb = (wave & 1) * 128;
  uint16_t *t = (uint16_t *)smem;
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int row = wa + i * 32 + (lane & 31), col = wb + j * 32 + (e / 4) * 8 + (lane >> 5) * 4;
        const uint2 v = {pack_pair16<DT>(acc[i][j][e], acc[i][j][e + 1]), pack_pair16<DT>(acc[i][j][e + 2], acc[i][j][e + 3])};
        *(uint2 *)(t + row * OUT_LD + col) = v;
      }
  __syncthreads();
  const int col = (threadIdx.x & 31) * 8;
  if (col < clim)
    for (int row = threadIdx.x >> 5; row < FM && row < rlim; row += 8)
      *(u32x4 *)(c + row * ldc + col) = *(const u32x4 *)(t + row * OUT_LD + col);
}

// Tiles of one XCD follow each other: neighbours share rows of x and a group's weights in its L2.  grid: a multiple of 8.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b) { return (b & 7u) * (gridDim.x >> 3) + (b >> 3); }

template <int DT, bool W_TRANS>
__global__ __launch_bounds__(256, 2) void grouped_fast_kernel(uint16_t *y, const uint16_t *x, const uint16_t *w, const int32_t *offsets,
                                                              int64_t M, int64_t N, int64_t K, int64_t groups, uint32_t col_tiles) {
  __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE_BYTES];
  const uint32_t id = xcd_order(blockIdx.x);
  const RowTile r = find_rows<FM>(offsets, groups, M, id / col_tiles);
  if (r.group == -2) return;
  const int64_t first = __builtin_amdgcn_readfirstlane((int)r.first), c0 = (int64_t)(id % col_tiles) * FN;
  const int group = __builtin_amdgcn_readfirstlane(r.group), rows = __builtin_amdgcn_readfirstlane((int)(r.end - r.first));
  const int cols = (int)(N - c0 < FN ? N - c0 : FN);
  f32x16 acc[2][4] = {};
  if (group >= 0) {
    const uint16_t *wg = w + (int64_t)group * K * N;
    Panel<false, FM> a;
    Panel<!W_TRANS, FN> b;
    a.set(x + first * K, K, rows);
    b.set(W_TRANS ? wg + c0 * K : wg + c0, W_TRANS ? K : N, cols);
    fast_product<DT, false, !W_TRANS>(smem, a, b, (int)(K / FK), (int)(K % FK), acc);
  }
  fast_store<DT>(smem, y + first * N + c0, N, rows, cols, acc);
}

template <int DT>
__global__ __launch_bounds__(256, 2) void grouped_wgrad_fast_kernel(uint16_t *dw, const uint16_t *a, const uint16_t *b, const int32_t *offsets,
                                                                    int64_t M, int64_t P, int64_t Q, uint32_t ptiles, uint32_t qtiles,
                                                                    uint32_t tiles) {
  __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE_BYTES];
  const uint32_t id = xcd_order(blockIdx.x);
  if (id >= tiles) return;
  const uint32_t g = id / (ptiles * qtiles), t = id % (ptiles * qtiles);
  const int64_t p0 = (int64_t)(t / qtiles) * FM, q0 = (int64_t)(t % qtiles) * FN;
  const int64_t lo = row_at(offsets, g, M), hi = row_at(offsets, (int64_t)g + 1, M);
  const int plim = (int)(P - p0 < FM ? P - p0 : FM), qlim = (int)(Q - q0 < FN ? Q - q0 : FN);
  f32x16 acc[2][4] = {};
  if (hi > lo) {
    Panel<true, FM> pa;
    Panel<true, FN> pb;
    pa.set(a + lo * P + p0, P, plim);
    pb.set(b + lo * Q + q0, Q, qlim);
    fast_product<DT, true, true>(smem, pa, pb, (int)((hi - lo) / FK), (int)((hi - lo) % FK), acc);
  }
  fast_store<DT>(smem, dw + (int64_t)g * P * Q + p0 * Q + q0, Q, plim, qlim, acc);
}

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
    const int64_t ct = ceil_div(N, FN), rt = ceil_div(M, FM) + groups + 2;
    if (rt * ct < 0x7FFFFFF0ll) {
      const unsigned blocks = (unsigned)(ceil_div(rt * ct, 8) * 8);
      auto go = [&](auto kernel) {
        kernel<<<blocks, 256, 0, s>>>((uint16_t *)y, (const uint16_t *)x, (const uint16_t *)w, offsets, M, N, K, groups, (uint32_t)ct);
      };
      if (dtype == FPEMU_F16) w_trans ? go(grouped_fast_kernel<FPEMU_F16, true>) : go(grouped_fast_kernel<FPEMU_F16, false>);
      else w_trans ? go(grouped_fast_kernel<FPEMU_BF16, true>) : go(grouped_fast_kernel<FPEMU_BF16, false>);
      return launched(who);
    }
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
    const int64_t pf = ceil_div(P, FM), qf = ceil_div(Q, FN), tiles = pf * qf * groups;   // no more than the ones above
    const unsigned blocks = (unsigned)(ceil_div(tiles, 8) * 8);
    auto go = [&](auto kernel) {
      kernel<<<blocks, 256, 0, s>>>((uint16_t *)dw, (const uint16_t *)a, (const uint16_t *)b, offsets, M, P, Q, (uint32_t)pf, (uint32_t)qf,
                                    (uint32_t)tiles);
    };
    if (dtype == FPEMU_F16) go(grouped_wgrad_fast_kernel<FPEMU_F16>);
    else go(grouped_wgrad_fast_kernel<FPEMU_BF16>);
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
