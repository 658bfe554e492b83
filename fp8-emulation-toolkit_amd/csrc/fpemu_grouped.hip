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

// Workgroup b runs on XCD b % 8.  In one run: each XCD gets an eighth of the tiles, one after the other, so that neighbours
// share rows of x and a group's weights in its L2.  In turns of TURN tiles: where tiles cost what their group has rows, every
// XCD gets its part of every group (16 groups, the largest 2.5 times the mean, weight gradient of 2048 x 4096: 362 -> 295 us).
constexpr uint32_t NO_TILE = 0xFFFFFFFFu, TURN = 8;
__device__ __forceinline__ uint32_t xcd_tile(uint32_t b, uint32_t tiles) {
  const uint32_t share = (tiles + 7u) / 8u, at = b >> 3, id = (b & 7u) * share + at;
  return at < share && id < tiles ? id : NO_TILE;
}
__device__ __forceinline__ uint32_t xcd_turn(uint32_t b, uint32_t tiles) {
  const uint32_t at = b >> 3, id = (at / TURN * 8u + (b & 7u)) * TURN + at % TURN;
  return id < tiles ? id : NO_TILE;
}

// Row and column tile of number id: bands of four row tiles, down the band first, so that the tiles an XCD works on at one
// time are about as high as wide and share what they read.
__device__ __forceinline__ void banded(uint32_t id, uint32_t row_tiles, uint32_t col_tiles, uint32_t &row, uint32_t &col) {
  const uint32_t band = id / (4u * col_tiles), in = id - band * 4u * col_tiles;
  const uint32_t high = row_tiles - band * 4u < 4u ? row_tiles - band * 4u : 4u;
  row = band * 4u + in % high;
  col = in / high;
}

// ---- any storage, sizes and alignment: tiles staged through registers ----------------------------------------------------------------
// fp32 is bound by its matrix instructions (64 cycles each), so staging through registers feeds it: the vectors of the next two
// stages are on their way to registers while the current one is multiplied; then the next one is written to the other LDS
// buffer.
// The same kernel takes 16-bit operands whose rows are not whole 16-byte vectors: global loads need no more than element
// alignment, and vectors that reach over an edge are put together element by element.
// Measured, fp32: 2051 rows, 8 uneven groups, 768 x 1000: y 62, dx 57, dW 49 us (56 TFLOP/s: 64 x 64 tiles, each a chain over all
// of k, 2.3 of them for a CU; the matrix units are busy 43 to 56 % of the time); 4096^3 113 to 136 TFLOP/s.
// A stage is 128 bytes deep in k (64 16-bit or 32 fp32 elements).  LDS holds it as described for the tiles further down.
typedef uint32_t vec_any __attribute__((ext_vector_type(4), aligned(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

// in vectors of 16 bytes: 16 rows that are read together lie in 16 different places of 256 bytes
__device__ __forceinline__ int swizzle_row(int row) { return (row >> 1) & 7; }
// four 16-bit k-rows of a transposing read, or the two fp32 k-rows of a matrix instruction, go to different banks
template <int ES, int EXT> __device__ __forceinline__ int swizzle_col(int k) {
  return ES == 4 ? (k & 1) * 8 : EXT >= 128 ? (k & 3) * 4 : (k & 1) * 4;
}

// element (r, k) of an operand: p[r * ld + k], or p[k * ld + r] where the contraction is its slow dimension (COL)
template <int DT, bool COL, int EXT> struct Staged {
  using elem = typename Storage<DT>::elem;
  static constexpr int ES = (int)sizeof(elem), V = 16 / ES, FK = 128 / ES, LOADS = EXT * 128 / 16 / 256;
  static constexpr int BYTES = EXT * 128;
  const elem *base;   // the tile's first element at the stage's first k
  int64_t ld, step;
  int lim;            // entries of the tile
  elem pad;           // what a load behind the contraction yields
  u32x4 v[2][LOADS];  // two stages

  __device__ __forceinline__ void set(const elem *p, int64_t ld_, int lim_, elem pad_) {
    base = p;
    ld = ld_;
    lim = lim_;
    pad = pad_;
    step = (COL ? ld : 1) * FK;
  }
  __device__ __forceinline__ static void place(int j, int &outer, int &k) {
    const int id = j * 256 + (int)threadIdx.x;
    if (COL) {
      constexpr int PER = EXT / V;
      k = id / PER;
      outer = ((id % PER) ^ swizzle_col<ES, EXT>(k)) * V;
    } else {
      outer = id / 8;
      k = ((id & 7) ^ swizzle_row(outer)) * V;
    }
  }
  // every vector of a whole stage is whole
  __device__ __forceinline__ bool plain() const { return !COL || lim >= EXT; }
  // the next stage, of which `left` k are there
  template <bool PLAIN> __device__ __forceinline__ void load(int set, int64_t left) {
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      int outer, k;
      place(j, outer, k);
      const int r = PLAIN && COL ? outer : outer < lim ? outer : lim - 1;   // entries beyond the tile's only feed results that
      const elem *p = COL ? base + k * ld + r : base + r * ld + k;          // are not stored
      if constexpr (PLAIN) {
        v[set][j] = *(const vec_any *)p;
      } else {
        const int have = COL ? (k < left ? (lim - r < V ? lim - r : V) : 0) : left - k >= V ? V : (int)(left - k);
        if (have >= V) {
          v[set][j] = *(const vec_any *)p;
        } else {
          elem e[V];
#pragma unroll
          for (int i = 0; i < V; i++) e[i] = i < have ? p[i] : pad;
          __builtin_memcpy(&v[set][j], e, 16);
        }
      }
    }
    base += step;
  }
  __device__ __forceinline__ void put(char *lds, int set) const {
#pragma unroll
    for (int j = 0; j < LOADS; j++) *(u32x4 *)(lds + (j * 256 + (int)threadIdx.x) * 16) = v[set][j];
  }
  // 16-bit: a matrix operand of 32 entries from `at`, k-step of 16.  fp32: the operands of two matrix instructions, k-step of
  // 4: the k of lane half h are 0 + h and 2 + h, a row's four come as one vector and pick() takes the lane's two.
  __device__ __forceinline__ static u32x4 fragment(const char *lds, int at, int step) {
    const int lane = threadIdx.x & 63;
    u32x4 r = {0u, 0u, 0u, 0u};
    if constexpr (!COL) {
      const int row = at + (lane & 31), c = DT == FPEMU_F32 ? step : step * 2 + (lane >> 5);
      r = *(const u32x4 *)(lds + row * 128 + ((c ^ swizzle_row(row)) * 16));
    } else if constexpr (DT == FPEMU_F32) {
      const int col = at + (lane & 31);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int k = step * 4 + i * 2 + (lane >> 5);
        r[i] = *(const uint32_t *)(lds + k * (EXT * 4) + (((col >> 2) ^ swizzle_col<4, EXT>(k)) * 16) + (col & 3) * 4);
      }
    } else {
      const int i = lane & 15, g = lane >> 4, col = at + (g & 1) * 16 + (i & 3) * 4;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = step * 16 + (g >> 1) * 8 + h * 4 + (i >> 2);
        const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(
            lds + k * (EXT * 2) + (((col >> 3) ^ swizzle_col<2, EXT>(k)) * 16) + (col & 7) * 2));
        const uint2 w = __builtin_bit_cast(uint2, t);
        r[2 * h] = w.x;
        r[2 * h + 1] = w.y;
      }
    }
    return r;
  }
  __device__ __forceinline__ static float pick(u32x4 r, int i) {
    if constexpr (COL) return u2f(r[i]);
    else return u2f((threadIdx.x & 32u) ? r[2 * i + 1] : r[2 * i]);
  }
};

template <int DT> __device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == FPEMU_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int BM_, int BN_> struct AnyShape {   // 4 waves: 2 x 2 over the tile, side by side over one of 32 rows
  static constexpr int BM = BM_, BN = BN_, WM = BM >= 64 ? 2 : 1, WN = 4 / WM, TM = BM / WM / 32, TN = BN / WN / 32;
  __device__ __forceinline__ static int row() { return (int)(threadIdx.x >> 6) / WN * (BM / WM); }
  __device__ __forceinline__ static int col() { return (int)(threadIdx.x >> 6) % WN * (BN / WN); }
};

// acc[i][j] of a wave: rows S::row() + 32 i of A, columns S::col() + 32 j of B; k of them, ascending
template <int DT, class S, bool A_COL, bool B_COL>
__device__ __forceinline__ void any_product(char *smem, Staged<DT, A_COL, S::BM> &a, Staged<DT, B_COL, S::BN> &b, int64_t k,
                                            f32x16 (&acc)[S::TM][S::TN]) {
  using SA = Staged<DT, A_COL, S::BM>;
  using SB = Staged<DT, B_COL, S::BN>;
  constexpr int STEPS = DT == FPEMU_F32 ? SA::FK / 4 : SA::FK / 16, STAGE = SA::BYTES + SB::BYTES;
  const int wr = S::row(), wc = S::col();
  char *now = smem, *then = smem + STAGE;
  auto multiply = [&]() {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      u32x4 av[S::TM], bv[S::TN];
#pragma unroll
      for (int i = 0; i < S::TM; i++) av[i] = SA::fragment(now, wr + i * 32, s);
#pragma unroll
      for (int j = 0; j < S::TN; j++) bv[j] = SB::fragment(now + SA::BYTES, wc + j * 32, s);
      if constexpr (DT == FPEMU_F32) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < S::TM; i++)
#pragma unroll
            for (int j = 0; j < S::TN; j++)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(SA::pick(av[i], h), SB::pick(bv[j], h), acc[i][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < S::TM; i++)
#pragma unroll
          for (int j = 0; j < S::TN; j++) acc[i][j] = mfma16<DT>(av[i], bv[j], acc[i][j]);
      }
    }
  };
  auto load = [&](auto plain, int set, int64_t left) {
    a.template load<decltype(plain)::value>(set, left);
    b.template load<decltype(plain)::value>(set, left);
  };
  // one stage: `set` holds the next one, the one after it is loaded into the other set
  auto stage = [&](auto plain, int set, int64_t left) {
    if (decltype(plain)::value || left > 2 * SA::FK) load(plain, set ^ 1, left - 2 * SA::FK);
    multiply();
    if (left > SA::FK) {
      a.put(then, set);
      b.put(then + SA::BYTES, set);
    }
    __syncthreads();
    char *t = now;
    now = then;
    then = t;
  };
  load(std::false_type(), 0, k);
  if (k > SA::FK) load(std::false_type(), 1, k - SA::FK);
  a.put(now, 0);
  b.put(now + SA::BYTES, 0);
  __syncthreads();
  int64_t left = k;
  if (a.plain() && b.plain()) {
    for (; left >= 4 * SA::FK; left -= 2 * SA::FK) {   // the stages two and three ahead are whole
      stage(std::true_type(), 1, left);
      stage(std::true_type(), 0, left - SA::FK);
    }
  }
  for (; left > 0; left -= 2 * SA::FK) {
    stage(std::false_type(), 1, left);
    if (left > SA::FK) stage(std::false_type(), 0, left - SA::FK);
  }
}

template <int DT, class S>
__device__ __forceinline__ void any_store(typename Storage<DT>::elem *c, int64_t ldc, int rlim, int clim,
                                          const f32x16 (&acc)[S::TM][S::TN]) {
  const int lane = threadIdx.x & 63, wr = S::row(), wc = S::col();
#pragma unroll
  for (int i = 0; i < S::TM; i++)
#pragma unroll
    for (int j = 0; j < S::TN; j++) {
      const int col = wc + j * 32 + (lane & 31);
      if (col >= clim) continue;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int row = wr + i * 32 + (e / 4) * 8 + (lane >> 5) * 4 + (e & 3);
        if (row >= rlim) continue;
        const float v = acc[i][j][e] + 0.0f;   // the chain's -0 is written as the c-model writes it
        if constexpr (DT == FPEMU_F32) c[row * ldc + col] = v;
        else c[row * ldc + col] = (typename Storage<DT>::elem)store_elem16<DT>(v);
      }
    }
}

// Behind the contraction A's filler is -0 and B's +0 in fp32: products of -0, the one value that leaves any chain as it is.
template <int DT> __device__ __forceinline__ typename Storage<DT>::elem a_pad() {
  if constexpr (DT == FPEMU_F32) return -0.0f;
  else return 0;
}

template <int DT, bool W_TRANS, class S>
__global__ __launch_bounds__(256, 2) void grouped_any_kernel(typename Storage<DT>::elem *y, const typename Storage<DT>::elem *x,
                                                             const typename Storage<DT>::elem *w, const int32_t *offsets, int64_t M,
                                                             int64_t N, int64_t K, int64_t groups, uint32_t col_tiles) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (S::BM + S::BN) * 128];
  const TileMap<S::BM> map(offsets, groups, M);
  const uint32_t id = xcd_tile(blockIdx.x, map.tiles() * col_tiles);
  if (id == NO_TILE) return;
  uint32_t row_tile, col_tile;
  banded(id, map.tiles(), col_tiles, row_tile, col_tile);
  const RowTile r = map.find(row_tile);
  const int64_t c0 = (int64_t)col_tile * S::BN;
  const int rows = (int)(r.end - r.first), cols = (int)(N - c0 < S::BN ? N - c0 : S::BN);
  f32x16 acc[S::TM][S::TN] = {};
  if (r.group >= 0) {
    const typename Storage<DT>::elem *wg = w + (int64_t)r.group * K * N;
    Staged<DT, false, S::BM> a;
    Staged<DT, !W_TRANS, S::BN> b;
    a.set(x + r.first * K, K, rows, a_pad<DT>());
    b.set(W_TRANS ? wg + c0 * K : wg + c0, W_TRANS ? K : N, cols, 0);
    any_product<DT, S, false, !W_TRANS>(smem, a, b, K, acc);
  }
  any_store<DT, S>(y + r.first * N + c0, N, rows, cols, acc);
}

template <int DT, class S>
__global__ __launch_bounds__(256, 2) void grouped_wgrad_any_kernel(typename Storage<DT>::elem *dw, const typename Storage<DT>::elem *a,
                                                                   const typename Storage<DT>::elem *b, const int32_t *offsets,
                                                                   int64_t M, int64_t P, int64_t Q, uint32_t ptiles, uint32_t qtiles,
                                                                   uint32_t tiles) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (S::BM + S::BN) * 128];
  const uint32_t id = xcd_turn(blockIdx.x, tiles);
  if (id == NO_TILE) return;
  const uint32_t g = id / (ptiles * qtiles);
  uint32_t pt, qt;
  banded(id % (ptiles * qtiles), ptiles, qtiles, pt, qt);
  const int64_t p0 = (int64_t)pt * S::BM, q0 = (int64_t)qt * S::BN;
  const int64_t lo = row_at(offsets, g, M), hi = row_at(offsets, (int64_t)g + 1, M);
  const int plim = (int)(P - p0 < S::BM ? P - p0 : S::BM), qlim = (int)(Q - q0 < S::BN ? Q - q0 : S::BN);
  f32x16 acc[S::TM][S::TN] = {};
  if (hi > lo) {
    Staged<DT, true, S::BM> sa;
    Staged<DT, true, S::BN> sb;
    sa.set(a + lo * P + p0, P, plim, a_pad<DT>());
    sb.set(b + lo * Q + q0, Q, qlim, 0);
    any_product<DT, S, true, true>(smem, sa, sb, hi - lo, acc);
  }
  any_store<DT, S>(dw + (int64_t)g * P * Q + p0 * Q + q0, Q, plim, qlim, acc);
}

// ---- 16-bit storage in whole 16-byte vectors: tiles fed by loads that go straight to LDS -----------------------------------
// A tile of BM rows x BN columns, 64 deep in k per stage; while one stage is multiplied the next ones are on their way.
// A stage row of 64 k is 128 bytes, a whole cache line: with 32 deep stages every line was fetched twice (it had left the
// 32 KB L1 before its second half was asked for), and the tiles then ran at the rate of the L2, not of the matrix cores.
// An operand whose contraction is contiguous lies in LDS as rows of 128 bytes and is read 16 bytes a lane; one whose
// contraction is its slow dimension lies as it is in memory and is read through the transposing LDS read (of 16 lanes, lane
// i gets column i of 4 k-rows).  The loads write LDS linearly, so the bank swizzle is applied to the global address a lane
// fetches and undone where the fragment is read.
// Waves: WM x WN over the tile.
// Bound by the matrix cores (by the clock they hold on data that is not zero) where K is long, by a tile's start and end (about
// 10 us of a 256 x 256 tile) where it is not, by the weights' bytes for few rows.  Measured: 8192^3 bf16 1330 to 1380 TFLOP/s,
// fp16 1240 to 1270; 16381 rows, 16 uneven groups, 2048 x 4096 fp16 296 us (930); 8197 rows, 16 groups, 1024 x 2816 bf16, y, dx and
// dW 203 us (700; 68, 75 and 63 alone); 64 rows, 32 groups of which 26 have rows, 2048 x 1408 39 us with their 152 MB of weights
// from memory (3.9 TB/s), 25 us with them in the cache.  The matrix units are busy 57 % of the time in the first of these, 34 to 41 %
// in the second; one workgroup fills a CU's LDS, so nothing runs while its tile starts or ends.
constexpr int FK = 64;

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
  static constexpr int OUT = 32 * TN * 64;   // a wave's 32 finished rows on their way to memory
  static constexpr int LDS = STAGES * STAGE + WM * WN * OUT;
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
      outer = ((id % PER) ^ swizzle_col<2, EXT>(k)) * 8;
    } else {
      outer = id / 8;
      k = ((id & 7) ^ swizzle_row(outer)) * 8;
    }
  }
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
      frag[0] = (uint32_t)(k * (EXT * 2) + (((col >> 3) ^ swizzle_col<2, EXT>(k)) * 16) + (col & 7) * 2);
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

// acc[i][j]: entries wa + 32 i of A (its columns) and wb + 32 j of B (its rows): a lane holds 4 neighbours along B.
// idle: this wave's part of the tile has no rows (it still loads and waits with the others).
template <int DT, class S, bool A_COL, bool B_COL>
__device__ __forceinline__ void fast_product(char *smem, Panel<A_COL, S::BM, S::THREADS> &a, Panel<B_COL, S::BN, S::THREADS> &b, int full,
                                             int left, bool idle, f32x16 (&acc)[S::TM][S::TN]) {
  using PA = Panel<A_COL, S::BM, S::THREADS>;
  using PB = Panel<B_COL, S::BN, S::THREADS>;
  constexpr int AHEAD = S::STAGES - 1, LOADS = PA::LOADS + PB::LOADS, STEPS = FK / 16, TILES = S::TM * S::TN, SPREAD = 2,
                LATE = TILES / 2, SLOTS = SPREAD * TILES - LATE;
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
  // The loads of a stage are spread over the matrix instructions of a step and a half (slots 0 .. SLOTS): issued in one go
  // they fill the memory pipeline's queue and every wave stands before it with its matrix instructions undone; spread
  // wider, the last ones arrive late (8192^3, bf16: 1119 TFLOP/s in one go, 1274 over three steps, 1346 like this).
  auto loads_at = [&](int slot) {
#pragma unroll
    for (int j = 0; j < LOADS; j++)
      if (j * SLOTS / LOADS == slot) load(j);
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
  // waits for the next stage half way, so the barrier and the first reads of a stage hide behind matrix instructions too.
  auto stage = [&](auto works, int t, bool loads_now, bool loads_next) {
    constexpr bool WORKS = decltype(works)::value;
#pragma unroll
    for (int step = 0; step < STEPS; step++) {
      const int set = step & 1, next = set ^ 1;
      const bool ends = step + 1 == STEPS;
      if (!ends && WORKS) read(next, step + 1);
      const bool loads = ends ? loads_next : loads_now && step + 1 < SPREAD;
      const int slot0 = ends ? 0 : (step + 1) * TILES;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < TILES; m++) {
        if (ends && m == LATE) {
          if (t + 1 < stages) {
            arrive(t + 1);
            get = get + S::STAGE == S::STAGES * S::STAGE ? 0 : get + S::STAGE;
            if (WORKS) read(next, 0);
            if (!loads_next) tail(t + 1 + AHEAD);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        const int i = m / S::TN, j = m % S::TN;
        if (WORKS) acc[i][j] = mfma16<DT>(bv[set][j], av[set][i], acc[i][j]);
        if (loads) {
          loads_at(ends ? m - LATE : slot0 - LATE + m);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (loads_now && step + 2 == SPREAD) filled();
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
      for (int slot = 0; slot < TILES - LATE; slot++) loads_at(slot);
    } else {
      tail(AHEAD);
    }
    int t = 0;
    for (; t + 1 + AHEAD < full; t++) stage(works, t, true, true);
    for (; t < stages; t++) stage(works, t, t + AHEAD < full, false);
  };
  if (idle) run(std::false_type());   // the same waits and barriers
  else run(std::true_type());
}

template <class S> struct WaveAt {   // a wave's part of the tile; waves that share a SIMD (w, w + 4) differ in their rows
  int wa, wb;
  __device__ __forceinline__ WaveAt() {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    wb = (wave % S::WN) * (S::BN / S::WN);
    wa = (wave / S::WN) * (S::BM / S::WM);
  }
};

// A wave's part of the finished tile, 32 rows at a time through LDS of its own, to memory in rows of TN * 64 bytes; rows < rlim,
// columns < clim (a multiple of 8) of the tile.  stream: past the caches.
template <int DT, class S>
__device__ __forceinline__ void fast_store(char *smem, uint16_t *c, int64_t ldc, int rlim, int clim, bool stream, const WaveAt<S> &at,
                                           const f32x16 (&acc)[S::TM][S::TN]) {
  constexpr int PER = S::TN * 4;   // vectors of a row
  const int lane = threadIdx.x & 63;
  char *lds = smem + S::STAGES * S::STAGE + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * S::OUT;
  auto place = [](int row, int vec) { return row * (PER * 16) + ((vec ^ (PER == 8 ? (row >> 1) & 7 : (row >> 2) & 3)) * 16); };
#pragma unroll
  for (int i = 0; i < S::TM; i++) {
#pragma unroll
    for (int j = 0; j < S::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const uint2 v = {pack_pair16<DT>(acc[i][j][e], acc[i][j][e + 1]), pack_pair16<DT>(acc[i][j][e + 2], acc[i][j][e + 3])};
        *(uint2 *)(lds + place(lane & 31, j * 4 + e / 4) + (lane >> 5) * 8) = v;
      }
    asm volatile("" : : : "memory");   // one wave's LDS operations are in order: its lanes see each other's writes
#pragma unroll
    for (int r = 0; r < 32; r += 64 / PER) {
      const int row = r + lane / PER, vec = lane % PER;
      const u32x4 v = *(const u32x4 *)(lds + place(row, vec));
      const int orow = at.wa + i * 32 + row, ocol = at.wb + vec * 8;
      if (orow < rlim && ocol < clim) {
        u32x4 *to = (u32x4 *)(c + orow * ldc + ocol);
        if (stream) {   // fenced off: the compiler would make one ordinary store of the two
          asm volatile("" : : : "memory");
          __builtin_nontemporal_store(v, to);
          asm volatile("" : : : "memory");
        } else {
          *to = v;
        }
      }
    }
    asm volatile("" : : : "memory");
  }
}

template <int DT, bool W_TRANS, class S>
__global__ __launch_bounds__(S::THREADS) void grouped_fast_kernel(uint16_t *y, const uint16_t *x, const uint16_t *w, const int32_t *offsets,
                                                                  int64_t M, int64_t N, int64_t K, int64_t groups, uint32_t col_tiles, bool stream) {
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
  fast_store<DT, S>(smem, y + first * N + c0, N, rows, cols, stream, at, acc);
}

template <int DT, class S>
__global__ __launch_bounds__(S::THREADS) void grouped_wgrad_fast_kernel(uint16_t *dw, const uint16_t *a, const uint16_t *b,
                                                                        const int32_t *offsets, int64_t M, int64_t P, int64_t Q,
                                                                        uint32_t ptiles, uint32_t qtiles, uint32_t tiles, bool stream) {
  __shared__ __attribute__((aligned(16))) char smem[S::LDS];
  const uint32_t id = xcd_turn(blockIdx.x, tiles);
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
  fast_store<DT, S>(smem, dw + (int64_t)g * P * Q + p0 * Q + q0, Q, plim, qlim, stream, at, acc);
}

using Large = Shape<256, 256, 2, 4, 2>;
using Medium = Shape<128, 128, 2, 2, 2>;
using Little = Shape<64, 64, 2, 2, 2>;

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

// A shape's tiles cost nearly the same whether their rows are filled or not, so the large one needs groups of some rows, and tiles
// for half of the CUs.  bf16, us with 256 x 256 / 128 x 128 tiles, groups alike (and uneven, the largest twice the mean),
// operands in the caches: 16 groups of about 1024 rows, 2048 x 4096: 233 / 307 (257 / 314); of 512, 1024 x 2816 (352 large
// tiles): 54 / 53 (52 / 66), 2816 x 1024 (128): 54 / 45 (55 / 72); 8 of 256, 768 x 1024 (32): 19 / 10; 32 of 2 rows, 2048 x
// 1408: 37 / 28.
constexpr int64_t kLargeRows = 256, kLargeTiles = 128;
bool large_tiles(int64_t rows_per_group, int64_t tiles) { return rows_per_group >= kLargeRows && tiles >= kLargeTiles; }

// Fewer 128 x 128 tiles than CUs: 64 x 64 ones.  bf16, us with 128 / 64: 4 groups of 75, 512 x 1024 (24 tiles): 8.5 / 7.4; 8 of
// 256, 768 x 1024 (128): 10.4 / 8.6; 16 of 256, 1024 x 1024 (256): 17.4 / 18.8, uneven 17.2 / 24.2.
// Through registers (`any`) below two tiles a CU, because the longest group's tiles are what the others wait for.  fp32, us
// with 128 / 64, groups alike, then uneven: 8 groups of 256, 768 x 1000, y (128 tiles): 90 / 51, 91 / 63, dW (384): 48 / 46,
// 63 / 44; 16 of 256, 1024 x 1024 (256): 86 / 85, 148 / 104; 8 of 768, 1024 x 1024 (384): 149 / 126, 149 / 142; and from there on
// 16 of 512, 768 x 1024 (512): 116 / 127, 171 / 140; 8 of 1024, 768 x 2048 (1024): 225 / 247, 278 / 258.
constexpr int64_t kLittleTiles = 256;
bool little_tiles(int64_t row_tiles, int64_t col_tiles, bool any) { return row_tiles * col_tiles < (any ? 2 : 1) * kLittleTiles; }

// Results of more than 64 MB (16-bit, whole vectors) are stored past the caches, which keep the operands instead.  bf16, us in
// the cache / past it, and with an elementwise pass over the result behind: y of 23 MB 35 / 34, 43 / 46; 46 MB 69 / 69, 82 / 85;
// 134 MB 306 / 300, 347 / 339; dW of 46 MB 47 / 41, 66 / 68; 92 MB 80 / 63, 118 / 119; 185 MB 52 / 41, 154 / 141; 268 MB
// 292 / 275, 426 / 406.
constexpr int64_t kStreamBytes = 64ll << 20;
bool streams(int64_t bytes) { return bytes > kStreamBytes; }

// Groups of few rows, staged through registers: tiles of 32 rows leave fewer matrix instructions to rows that are not there.
// fp32, 32 groups, 2048 x 1408, us with 64 x 64 / 32 x 128 tiles: 2 rows a group 129 / 95 (weights transposed 147 / 106), 32 rows
// 133 / 95 (152 / 110), 38 rows 135 / 137 (151 / 158), 64 rows 139 / 142 (154 / 161).  bf16 at 2047 x 1409: 2 rows 62 / 72
// (43 / 39), 32 rows 61 / 73 (42 / 40).
bool flat_tiles(int64_t rows, int64_t groups) { return rows <= 32 * groups; }

template <int DT>
bool run_grouped(void *y, const void *x, const void *w, const int32_t *offsets, int64_t M, int64_t N, int64_t K, int64_t groups,
                 int w_trans, hipStream_t s) {
  using elem = typename Storage<DT>::elem;
  auto go = [&](int64_t bm, int64_t bn, int threads, auto kernel, auto... more) {
    const int64_t cols = ceil_div(N, bn), rows = ceil_div(M, bm) + groups + 2;   // every group may end in a partial tile
    if (rows * cols > 0x7FFFFFF0ll) return false;
    kernel<<<(unsigned)(ceil_div(rows * cols, 8) * 8), threads, 0, s>>>((elem *)y, (const elem *)x, (const elem *)w, offsets, M, N, K, groups,
                                                                        (uint32_t)cols, more...);
    return true;
  };
  if constexpr (DT != FPEMU_F32) {
    if (K > 0 && fast_rows(y, N) && fast_rows(x, K) && fast_rows(w, N)) {
      const bool stream = streams(2 * M * N);
      if (large_tiles(M / groups, ceil_div(M, Large::BM) * ceil_div(N, Large::BN))) {
        if (w_trans ? go(Large::BM, Large::BN, Large::THREADS, grouped_fast_kernel<DT, true, Large>, stream)
                    : go(Large::BM, Large::BN, Large::THREADS, grouped_fast_kernel<DT, false, Large>, stream))
          return true;
      }
      if (little_tiles(ceil_div(M, Medium::BM), ceil_div(N, Medium::BN), false))
        return w_trans ? go(Little::BM, Little::BN, Little::THREADS, grouped_fast_kernel<DT, true, Little>, stream)
                       : go(Little::BM, Little::BN, Little::THREADS, grouped_fast_kernel<DT, false, Little>, stream);
      return w_trans ? go(Medium::BM, Medium::BN, Medium::THREADS, grouped_fast_kernel<DT, true, Medium>, stream)
                     : go(Medium::BM, Medium::BN, Medium::THREADS, grouped_fast_kernel<DT, false, Medium>, stream);
    }
  }
  auto any = [&](auto shape) {
    using S = decltype(shape);
    return w_trans ? go(S::BM, S::BN, 256, grouped_any_kernel<DT, true, S>) : go(S::BM, S::BN, 256, grouped_any_kernel<DT, false, S>);
  };
  if (flat_tiles(M, groups)) return any(AnyShape<32, 128>());
  return little_tiles(ceil_div(M, 128), ceil_div(N, 128), true) ? any(AnyShape<64, 64>()) : any(AnyShape<128, 128>());
}

template <int DT>
bool run_wgrad(void *dw, const void *a, const void *b, const int32_t *offsets, int64_t M, int64_t P, int64_t Q, int64_t groups,
               hipStream_t s) {
  using elem = typename Storage<DT>::elem;
  auto go = [&](int64_t bm, int64_t bn, int threads, auto kernel, auto... more) {
    const int64_t pt = ceil_div(P, bm), qt = ceil_div(Q, bn);
    if (pt * qt > 0x7FFFFF00ll / groups) return false;
    const int64_t tiles = pt * qt * groups;
    kernel<<<(unsigned)(ceil_div(tiles, 8 * TURN) * 8 * TURN), threads, 0, s>>>((elem *)dw, (const elem *)a, (const elem *)b, offsets, M, P, Q, (uint32_t)pt,
                                                                  (uint32_t)qt, (uint32_t)tiles, more...);
    return true;
  };
  if constexpr (DT != FPEMU_F32) {
    if (M > 0 && fast_rows(dw, Q) && fast_rows(a, P) && fast_rows(b, Q)) {
      const bool stream = streams(2 * P * Q * groups);
      if (large_tiles(M / groups, ceil_div(P, Large::BM) * ceil_div(Q, Large::BN) * groups))
        return go(Large::BM, Large::BN, Large::THREADS, grouped_wgrad_fast_kernel<DT, Large>, stream);
      if (little_tiles(ceil_div(P, Medium::BM) * groups, ceil_div(Q, Medium::BN), false))
        return go(Little::BM, Little::BN, Little::THREADS, grouped_wgrad_fast_kernel<DT, Little>, stream);
      return go(Medium::BM, Medium::BN, Medium::THREADS, grouped_wgrad_fast_kernel<DT, Medium>, stream);
    }
  }
  if (little_tiles(ceil_div(P, 128) * groups, ceil_div(Q, 128), true)) return go(64, 64, 256, grouped_wgrad_any_kernel<DT, AnyShape<64, 64>>);
  return go(128, 128, 256, grouped_wgrad_any_kernel<DT, AnyShape<128, 128>>);
}

}  // namespace

extern "C" int fpemu_grouped_gemm(void *y, const void *x, const void *w, const int32_t *offsets, int64_t M, int64_t N, int64_t K,
                                  int64_t groups, int dtype, int w_trans, void *stream) {
  const char *who = "fpemu_grouped_gemm";
  if (const int rc = check_grouped(who, y, x, w, offsets, M, N, K, groups, dtype)) return rc;
  if (M == 0 || N == 0) return FPEMU_OK;
  if (y == nullptr || (K > 0 && (x == nullptr || w == nullptr))) return fail(FPEMU_EINVAL, who, "null buffer");
  hipStream_t s = (hipStream_t)stream;
  const bool done = dtype == FPEMU_F32   ? run_grouped<FPEMU_F32>(y, x, w, offsets, M, N, K, groups, w_trans, s)
                    : dtype == FPEMU_F16 ? run_grouped<FPEMU_F16>(y, x, w, offsets, M, N, K, groups, w_trans, s)
                                         : run_grouped<FPEMU_BF16>(y, x, w, offsets, M, N, K, groups, w_trans, s);
  return done ? launched(who) : fail(FPEMU_EINVAL, who, "too many tiles for one launch");
}

extern "C" int fpemu_grouped_gemm_wgrad(void *dw, const void *a, const void *b, const int32_t *offsets, int64_t M, int64_t P, int64_t Q,
                                        int64_t groups, int dtype, void *stream) {
  const char *who = "fpemu_grouped_gemm_wgrad";
  if (const int rc = check_grouped(who, dw, a, b, offsets, M, P, Q, groups, dtype)) return rc;
  if (P == 0 || Q == 0) return FPEMU_OK;
  if (dw == nullptr || (M > 0 && (a == nullptr || b == nullptr))) return fail(FPEMU_EINVAL, who, "null buffer");
  hipStream_t s = (hipStream_t)stream;
  const bool done = dtype == FPEMU_F32   ? run_wgrad<FPEMU_F32>(dw, a, b, offsets, M, P, Q, groups, s)
                    : dtype == FPEMU_F16 ? run_wgrad<FPEMU_F16>(dw, a, b, offsets, M, P, Q, groups, s)
                                         : run_wgrad<FPEMU_BF16>(dw, a, b, offsets, M, P, Q, groups, s);
  return done ? launched(who) : fail(FPEMU_EINVAL, who, "too many tiles for one launch");
}
