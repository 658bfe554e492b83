// fpemu_train.hip -- operators of a language model's training step that run beside the emulated cast: rows in the
// order of their group (a router's experts, a vocabulary's entries), the scaled embedding lookup with the gradient of
// its table, and the norm and clipping of a whole list of gradients.  Sums are held in 32 bits (table gradient) or
// 64 bits (norms; squares of 16-bit values are added in fours in 32 bits first) and rounded once, when they are stored.  No floating-point atomics: every sum has one fixed order,
// so a call repeated on the same inputs gives the same bits.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/fpemu_hip.h"
#include "fpemu_common.hpp"

using namespace fpemu;

namespace {

int fail(int code, const char *who, const char *what) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  fpemu_set_error_(msg);
  return code;
}

int launched(const char *who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FPEMU_OK : fail((int)e, who, hipGetErrorString(e));
}

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// ---- rows in the order of their group -----------------------------------------------------------------------------
// A stable counting sort by digits of the group id, least significant digit first (one pass up to 511 groups, two up to
// 2^18 - 1, ...).  A row outside [0, groups) has the key `groups` and so ends up behind every group.  The rank of a row among
// the equal digits before it is found wave by wave: ballots over the digit's bits give the lanes with the same digit, one
// LDS counter per (wave, digit) carries the count from round to round.  The chain of rounds is what a small sort takes
// (ballots, an LDS atomic and a shuffle each), so a workgroup is as wide as it can be: 16 waves, four rounds at most.
// Measured: 1031 ids in 64 groups 4.5 us (one launch); 65536 ids in 30522 groups 34 us of kernels (two digits: count 3.8 and
// place 10.5 us each on 16 workgroups, latency; offsets 5.2, a binary search an entry); 2^20 ids in 256 groups 22 us (count 4.8,
// scan 4.2, place 13.3: its 4-byte stores leave in the order of the lanes, not of the digits).
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kSortRounds = 4;
constexpr int kSortTile = kSortThreads * kSortRounds;   // 4096 rows per workgroup
constexpr int kMaxBits = 9;                             // digits of at most 512 values: 32 KB of counters
constexpr int kMaxBins = 1 << kMaxBits;
constexpr unsigned kSelfSum = 32;                       // up to this many tiles a tile adds up the counts before it by itself
constexpr int kMaxPasses = 4;

struct SortPlan {
  int bits, passes, shift[kMaxPasses], width[kMaxPasses];
};

SortPlan sort_plan(uint64_t groups) {
  SortPlan p;
  p.bits = 1;
  while (p.bits < 32 && ((uint64_t)1 << p.bits) <= groups) p.bits++;   // keys 0 .. groups
  p.passes = (p.bits + kMaxBits - 1) / kMaxBits;
  for (int i = 0, at = 0; i < p.passes; i++) {
    const int w = (p.bits - at + (p.passes - i) - 1) / (p.passes - i);
    p.shift[i] = at;
    p.width[i] = w;
    at += w;
  }
  return p;
}

// Memory that a sort's kernels clear beside their own work, in workgroups behind the sort's: a table's gradient is cleared
// while its tokens are sorted (the sort keeps a few CUs busy, the stores the memory).  `stream`: past the caches.
typedef uint32_t vec_a2 __attribute__((ext_vector_type(4), aligned(2)));   // rows of odd widths: element-aligned only
struct Fill {
  char *p;
  uint64_t bytes;          // even
  uint64_t first, last;    // this launch's share, in pieces of kFillPiece
  bool stream;
};
constexpr uint64_t kFillPiece = 128 << 10;   // of one workgroup

__device__ __forceinline__ void fill_piece(const Fill &f, uint64_t piece) {
  const uint64_t at = (f.first + piece) * kFillPiece, end = at + kFillPiece < f.bytes ? at + kFillPiece : f.bytes;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  uint64_t i = at + threadIdx.x * 16u;
  if (f.stream) {
#pragma unroll 4
    for (; i + 16 <= end; i += kSortThreads * 16u) __builtin_nontemporal_store(zero, (vec_a2 *)(f.p + i));
  } else {
#pragma unroll 4
    for (; i + 16 <= end; i += kSortThreads * 16u) *(vec_a2 *)(f.p + i) = zero;
  }
  for (; i < end; i += 2) *(uint16_t *)(f.p + i) = 0;   // the thread whose vector reaches over the end
}

__device__ __forceinline__ uint32_t key_of(const void *ids, int wide, uint64_t i, uint32_t groups) {
  if (wide) {
    const uint64_t v = ((const uint64_t *)ids)[i];
    return v < groups ? (uint32_t)v : groups;
  }
  const uint32_t v = ((const uint32_t *)ids)[i];
  return v < groups ? v : groups;
}

// rank of each of the lane's rows among the rows of its wave with the same digit before it; cnt: the wave's counters
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[kSortRounds], unsigned valid, int rounds, int bits, uint32_t *cnt,
                                           uint32_t (&rank)[kSortRounds]) {
  const unsigned lane = threadIdx.x & 63u;
  const uint64_t below = ((uint64_t)1 << lane) - 1u;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    if (r >= rounds) break;
    const bool ok = (valid >> r) & 1u;
    uint64_t same = __ballot(ok);
    for (int b = 0; b < bits; b++) {
      const bool bit = (digit[r] >> b) & 1u;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const uint32_t before = (uint32_t)__popcll(same & below);
    uint32_t base = 0;
    if (ok && before == 0) base = atomicAdd(&cnt[digit[r]], (uint32_t)__popcll(same));
    const int leader = ok ? __ffsll((unsigned long long)same) - 1 : (int)lane;
    rank[r] = (uint32_t)__shfl((int)base, leader, 64) + before;
  }
}

// exclusive sum over the first `bins` entries of v (LDS), all threads of the workgroup; tmp: kSortWaves words
__device__ __forceinline__ void exclusive_bins(uint32_t *v, int bins, uint32_t *tmp) {
  static_assert(kMaxBins <= kSortThreads, "a thread per digit");
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const int at = (int)threadIdx.x;
  const uint32_t x = at < bins ? v[at] : 0u;
  uint32_t inc = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)inc, off, 64);
    if ((int)lane >= off) inc += o;
  }
  if (lane == 63u) tmp[wave] = inc;
  __syncthreads();
  uint32_t run = inc - x;
  for (unsigned w = 0; w < wave; w++) run += tmp[w];
  if (at < bins) v[at] = run;
  __syncthreads();
}

// Up to kSortTile rows: every pass inside one workgroup, rows exchanged through LDS.  keys_out (or NULL): the sorted keys;
// offsets (or NULL): with one pass they are the counters' sums.
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const void *ids, int wide, uint32_t n, uint32_t groups,
                                                                  SortPlan plan, int32_t *order, uint32_t *keys_out,
                                                                  int32_t *offsets, Fill fill) {
  __shared__ uint32_t cnt[kSortWaves * kMaxBins];
  __shared__ uint32_t skey[kSortTile];
  __shared__ uint16_t spos[kSortTile];
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t tmp[kSortWaves];
  if (blockIdx.x > 0) return fill_piece(fill, blockIdx.x - 1u);
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const int rounds = (int)((n + kSortThreads - 1u) / kSortThreads);
  const uint32_t mine = wave * 64u * (uint32_t)rounds + lane;   // the wave's rows are neighbours
  uint32_t key[kSortRounds], pos[kSortRounds], digit[kSortRounds], rank[kSortRounds];
  unsigned valid = 0;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    const uint32_t i = mine + (uint32_t)r * 64u;
    pos[r] = i;
    key[r] = 0;
    if (r < rounds && i < n) {
      key[r] = key_of(ids, wide, i, groups);
      valid |= 1u << r;
    }
  }
  for (int p = 0; p < plan.passes; p++) {
    const int bins = 1 << plan.width[p];
    for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; r++) digit[r] = (key[r] >> plan.shift[p]) & (uint32_t)(bins - 1);
    wave_ranks(digit, valid, rounds, plan.width[p], cnt + wave * bins, rank);
    __syncthreads();
    if ((int)threadIdx.x < bins) {
      const int d = (int)threadIdx.x;
      uint32_t run = 0;
#pragma unroll
      for (int w = 0; w < kSortWaves; w++) {
        const uint32_t c = cnt[w * bins + d];
        cnt[w * bins + d] = run;
        run += c;
      }
      base[d] = run;
    }
    __syncthreads();
    exclusive_bins(base, bins, tmp);
    const bool last = p + 1 == plan.passes;
    if (last && offsets != nullptr && plan.passes == 1)
      for (uint32_t g = threadIdx.x; g <= groups; g += kSortThreads) offsets[g] = (int32_t)base[g];
#pragma unroll
    for (int r = 0; r < kSortRounds; r++) {
      if (!((valid >> r) & 1u)) continue;
      const uint32_t to = base[digit[r]] + cnt[wave * bins + digit[r]] + rank[r];
      if (last) {
        order[to] = (int32_t)pos[r];
        if (keys_out != nullptr) keys_out[to] = key[r];
      } else {
        skey[to] = key[r];
        spos[to] = (uint16_t)pos[r];
      }
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (int r = 0; r < kSortRounds; r++) {
        const uint32_t i = mine + (uint32_t)r * 64u;
        if ((valid >> r) & 1u) {
          key[r] = skey[i];
          pos[r] = spos[i];
        }
      }
    }
  }
}

// rows (key, position) of a pass: the first pass reads the ids, later ones what the pass before wrote
struct SortIn {
  const void *ids;        // first pass
  const uint32_t *keys;   // later passes
  const int32_t *pos;
  int wide;
};

__device__ __forceinline__ uint32_t sort_key(const SortIn &in, uint64_t i, uint32_t groups) {
  return in.keys != nullptr ? in.keys[i] : key_of(in.ids, in.wide, i, groups);
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortIn in, uint32_t n, uint32_t groups, int shift, int width,
                                                                  uint32_t tiles, uint32_t *counts, Fill fill) {
  __shared__ uint32_t cnt[kMaxBins];
  if (blockIdx.x >= tiles) return fill_piece(fill, blockIdx.x - tiles);
  const int bins = 1 << width;
  for (int i = threadIdx.x; i < bins; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  const uint64_t first = (uint64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    const uint64_t i = first + (uint64_t)r * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&cnt[(sort_key(in, i, groups) >> shift) & (uint32_t)(bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[(uint64_t)d * tiles + blockIdx.x] = cnt[d];   // [digit][tile]
}

// counts[digit][tile] -> the rows of that digit in the tiles before; totals[digit].  A wave per digit.
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t *counts, uint32_t tiles, int bins, uint32_t *totals) {
  const int d = (int)(blockIdx.x * 4u + (threadIdx.x >> 6));
  const unsigned lane = threadIdx.x & 63u;
  if (d >= bins) return;
  uint32_t run = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += 64u) {
    const uint32_t t = t0 + lane;
    const uint32_t c = t < tiles ? counts[(uint64_t)d * tiles + t] : 0u;
    uint32_t inc = c;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)inc, off, 64);
      if ((int)lane >= off) inc += o;
    }
    if (t < tiles) counts[(uint64_t)d * tiles + t] = run + inc - c;
    run += (uint32_t)__shfl((int)inc, 63, 64);
  }
  if (lane == 0) totals[d] = run;
}

__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(SortIn in, uint32_t n, uint32_t groups, int shift, int width,
                                                                  uint32_t tiles, const uint32_t *counts,
                                                                  const uint32_t *totals, uint32_t *keys_out, int32_t *pos_out,
                                                                  int32_t *offsets, Fill fill) {
  __shared__ uint32_t cnt[kSortWaves * kMaxBins];
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t tmp[kSortWaves];
  if (blockIdx.x >= tiles) return fill_piece(fill, blockIdx.x - tiles);
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const int bins = 1 << width;
  uint32_t key[kSortRounds], pos[kSortRounds], digit[kSortRounds], rank[kSortRounds];
  unsigned valid = 0;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    const uint64_t i = (uint64_t)blockIdx.x * kSortTile + wave * (64u * kSortRounds) + (uint32_t)r * 64u + lane;
    key[r] = pos[r] = 0;
    if (i < n) {
      key[r] = sort_key(in, i, groups);
      pos[r] = in.pos != nullptr ? (uint32_t)in.pos[i] : (uint32_t)i;
      valid |= 1u << r;
    }
    digit[r] = (key[r] >> shift) & (uint32_t)(bins - 1);
  }
  // per digit (a thread each): rows of the tiles before this one, and all rows
  const int d = (int)threadIdx.x;
  uint32_t own = 0, all = 0;
  if (d < bins) {
    if (totals != nullptr) {
      own = counts[(uint64_t)d * tiles + blockIdx.x];
      all = totals[d];
    } else {
#pragma unroll 8
      for (uint32_t t = 0; t < tiles; t++) {
        const uint32_t c = counts[(uint64_t)d * tiles + t];
        own += t < blockIdx.x ? c : 0u;
        all += c;
      }
    }
    base[d] = all;
  }
  for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  wave_ranks(digit, valid, kSortRounds, width, cnt + wave * bins, rank);
  exclusive_bins(base, bins, tmp);   // its barriers also stand between the ranks and the counters' sums
  if (offsets != nullptr && blockIdx.x == 0)
    for (uint32_t g = threadIdx.x; g <= groups; g += kSortThreads) offsets[g] = (int32_t)base[g];
  if (d < bins) {
    uint32_t run = base[d] + own;
#pragma unroll
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = cnt[w * bins + d];
      cnt[w * bins + d] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    if (!((valid >> r) & 1u)) continue;
    const uint32_t to = cnt[wave * bins + digit[r]] + rank[r];
    pos_out[to] = (int32_t)pos[r];
    if (keys_out != nullptr) keys_out[to] = key[r];
  }
}

// offsets[g] = the first sorted row whose key is at least g, g = 0 .. groups
__global__ __launch_bounds__(256) void sort_offsets_kernel(const uint32_t *keys, uint32_t n, uint32_t groups, int32_t *offsets) {
  const uint64_t g = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (g > groups) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2u;
    if (keys[mid] < (uint32_t)g) lo = mid + 1u;
    else hi = mid;
  }
  offsets[g] = (int32_t)lo;
}

__global__ __launch_bounds__(kSortThreads) void fill_kernel(Fill fill) { fill_piece(fill, blockIdx.x); }

// workspace of the sort, in words: [sorted keys][keys a][pos a] + counts + totals (passes alternate between a and the results)
struct SortSpace {
  uint64_t keys, keys_a, pos_a, counts, totals, words;
};

SortSpace sort_space(uint64_t n, uint64_t groups, bool with_keys) {
  const SortPlan plan = sort_plan(groups);
  const uint64_t tiles = ceil_div(n, kSortTile);
  SortSpace s{};
  uint64_t at = 0;
  auto take = [&](uint64_t words) { const uint64_t o = at; at += (words + 3) / 4 * 4; return o; };
  if (plan.passes > 1 || with_keys) s.keys = take(n);
  if (tiles > 1) {
    if (plan.passes > 1) {
      s.keys_a = take(n);
      s.pos_a = take(n);
    }
    s.counts = take(tiles * kMaxBins);
    s.totals = take(kMaxBins);
  }
  s.words = at;
  return s;
}

// order[n]; offsets[groups + 1] or NULL; with_keys: the sorted keys at ws + sort_space().keys; fill: cleared on the way
int sort_rows(const char *who, const void *ids, int wide, uint64_t n, uint64_t groups, int32_t *order, int32_t *offsets, bool with_keys,
              uint32_t *ws, Fill fill, hipStream_t stream) {
  const SortPlan plan = sort_plan(groups);
  const SortSpace sp = sort_space(n, groups, with_keys);
  const uint32_t n32 = (uint32_t)n, g32 = (uint32_t)groups;
  const uint32_t tiles = (uint32_t)ceil_div(n, kSortTile);
  const uint64_t pieces = ceil_div(fill.bytes, kFillPiece);
  // the share of launch i of `of` launches that clear something
  auto share = [&](int i, int of) {
    fill.first = pieces * (uint64_t)i / (uint64_t)of;
    fill.last = pieces * (uint64_t)(i + 1) / (uint64_t)of;
    return (unsigned)(fill.last - fill.first);
  };
  if (n == 0) {
    if (pieces > 0) {
      const unsigned blocks = share(0, 1);
      fill_kernel<<<blocks, kSortThreads, 0, stream>>>(fill);
    }
    if (offsets != nullptr) {
      const Fill zero{(char *)offsets, 4 * (groups + 1), 0, 0, false};
      fill_kernel<<<(unsigned)ceil_div(zero.bytes, kFillPiece), kSortThreads, 0, stream>>>(zero);
    }
    return launched(who);
  }
  uint32_t *sorted = plan.passes > 1 || with_keys ? ws + sp.keys : nullptr;
  if (tiles == 1) {
    const unsigned more = share(0, 1);
    sort_small_kernel<<<1 + more, kSortThreads, 0, stream>>>(ids, wide, n32, g32, plan, order, sorted, offsets, fill);
  } else {
    SortIn in{ids, nullptr, nullptr, wide};
    for (int p = 0; p < plan.passes; p++) {
      const bool other = (plan.passes - 1 - p) & 1;   // passes alternate so that the last one writes the results
      uint32_t *keys = other ? ws + sp.keys_a : sorted;
      int32_t *pos = other ? (int32_t *)(ws + sp.pos_a) : order;
      unsigned more = share(2 * p, 2 * plan.passes);
      sort_count_kernel<<<tiles + more, kSortThreads, 0, stream>>>(in, n32, g32, plan.shift[p], plan.width[p], tiles, ws + sp.counts, fill);
      const uint32_t *totals = nullptr;
      if (tiles > kSelfSum) {
        const int bins = 1 << plan.width[p];
        sort_scan_kernel<<<(unsigned)ceil_div(bins, 4), 256, 0, stream>>>(ws + sp.counts, tiles, bins, ws + sp.totals);
        totals = ws + sp.totals;
      }
      more = share(2 * p + 1, 2 * plan.passes);
      sort_place_kernel<<<tiles + more, kSortThreads, 0, stream>>>(in, n32, g32, plan.shift[p], plan.width[p], tiles, ws + sp.counts, totals,
                                                                   keys, pos, plan.passes == 1 ? offsets : nullptr, fill);
      in.keys = keys;
      in.pos = pos;
    }
  }
  if (plan.passes > 1 && offsets != nullptr)
    sort_offsets_kernel<<<(unsigned)ceil_div(groups + 1, 256), 256, 0, stream>>>(sorted, n32, g32, offsets);
  return launched(who);
}

int check_ids(const char *who, const void *ids, int id_bytes, uint64_t n, uint64_t groups) {
  if (id_bytes != 4 && id_bytes != 8) return fail(FPEMU_EINVAL, who, "ids are 4- or 8-byte integers");
  if (n > 0x7FFFFFFFull) return fail(FPEMU_EINVAL, who, "more than 2^31 - 1 rows");
  if (groups < 1 || groups > 0x7FFFFFFEull) return fail(FPEMU_EINVAL, who, "the number of groups is between 1 and 2^31 - 2");
  if (n > 0 && ids == nullptr) return fail(FPEMU_EINVAL, who, "null ids");
  if (((uintptr_t)ids) % (unsigned)id_bytes) return fail(FPEMU_EALIGN, who, "ids not aligned to their size");
  return FPEMU_OK;
}

// ---- vectors of 16 bytes at any element address ----------------------------------------------------------------------
template <int DT> struct Elems {
  static constexpr int V = DT == FPEMU_F32 ? 4 : 8;
  using elem = typename Storage<DT>::elem;
  __device__ static __forceinline__ void unpack(u32x4 v, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (DT == FPEMU_F32) f[j] = u2f(v[j]);
      else {
        f[2 * j] = load_elem16<DT>(v[j] & 0xFFFFu);
        f[2 * j + 1] = load_elem16<DT>(v[j] >> 16);
      }
    }
  }
  __device__ static __forceinline__ u32x4 pack(const float (&f)[V]) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (DT == FPEMU_F32) v[j] = f2u(f[j]);
      else v[j] = pack_pair16<DT>(f[2 * j], f[2 * j + 1]);
    }
    return v;
  }
  __device__ static __forceinline__ float one(const elem *p) {
    if constexpr (DT == FPEMU_F32) return *p;
    else return load_elem16<DT>(*p);
  }
  __device__ static __forceinline__ void put(elem *p, float f) {
    if constexpr (DT == FPEMU_F32) *p = f;
    else *p = (elem)store_elem16<DT>(f);
  }
};

// V elements from column c of a row of `width`: a vector where they all exist, element by element at the row's end
template <int DT> __device__ __forceinline__ void load_cols(const typename Elems<DT>::elem *row, uint64_t c, uint64_t width,
                                                            float (&f)[Elems<DT>::V]) {
  if (c + Elems<DT>::V <= width) {
    Elems<DT>::unpack(*(const vec_a2 *)(row + c), f);
  } else {
#pragma unroll
    for (int j = 0; j < Elems<DT>::V; j++) f[j] = c + j < width ? Elems<DT>::one(row + c + j) : 0.f;
  }
}
template <int DT> __device__ __forceinline__ void store_cols(typename Elems<DT>::elem *row, uint64_t c, uint64_t width,
                                                             const float (&f)[Elems<DT>::V]) {
  if (c + Elems<DT>::V <= width) {
    *(vec_a2 *)(row + c) = Elems<DT>::pack(f);
  } else {
#pragma unroll
    for (int j = 0; j < Elems<DT>::V; j++)
      if (c + j < width) Elems<DT>::put(row + c + j, f[j]);
  }
}

// ---- embedding --------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t id_at(const void *ids, int wide, uint64_t i) {
  return wide ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
}

// out[t] = scale * weight[ids[t]]: 2^lg_tpr threads a row, R rows a thread (their loads are in flight together).  A row whose
// id is outside the table reads nothing of it and is NaN.  Bound by memory (each row read and written once): 32768 rows of 2048
// bf16 in 42 us, 6.4 TB/s (of 134 MB read 86 miss the L2s: frequent tokens' rows).  One row a thread
// where the launch is short (one token: 1.4 us).
template <int DT, int R>
__global__ __launch_bounds__(256) void embedding_kernel(const void *weight, const void *ids, int wide, void *out, uint64_t n,
                                                        uint64_t vocab, uint64_t width, float scale, int lg_tpr) {
  using E = Elems<DT>;
  const uint64_t rows = 256u >> lg_tpr;
  const uint64_t t0 = (uint64_t)blockIdx.x * rows * R + (threadIdx.x >> lg_tpr);
  const typename E::elem *src[R];
  bool known[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint64_t t = t0 + r * rows;
    const int64_t id = t < n ? id_at(ids, wide, t) : 0;
    known[r] = id >= 0 && (uint64_t)id < vocab;
    src[r] = (const typename E::elem *)weight + (known[r] ? (uint64_t)id : 0u) * width;
  }
  const uint64_t step = (uint64_t)E::V << lg_tpr;
  for (uint64_t c = (uint64_t)(threadIdx.x & ((1u << lg_tpr) - 1u)) * E::V; c < width; c += step) {
    if (c + E::V <= width) {
      u32x4 v[R];
#pragma unroll
      for (int r = 0; r < R; r++) v[r] = *(const vec_a2 *)(src[r] + c);
#pragma unroll
      for (int r = 0; r < R; r++) {
        const uint64_t t = t0 + r * rows;
        if (t >= n) continue;
        float f[E::V];
        E::unpack(v[r], f);
#pragma unroll
        for (int j = 0; j < E::V; j++) f[j] = known[r] ? f[j] * scale : u2f(0x7FC00000u);
        *(vec_a2 *)((typename E::elem *)out + t * width + c) = E::pack(f);
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; r++) {
        const uint64_t t = t0 + r * rows;
        if (t >= n) continue;
        for (uint64_t j = c; j < width; j++)
          E::put((typename E::elem *)out + t * width + j, known[r] ? E::one(src[r] + j) * scale : u2f(0x7FC00000u));
      }
    }
  }
}

// Gradient of the table from the sorted tokens; the table is zero when these kernels run.  The sorted positions are cut into
// chunks.  A wave takes the runs (tokens of one entry) that begin in its chunk, to their ends, and writes their rows; a chunk
// that an earlier run fills is summed by a wave of its own first (a frequent token's run is long: its chunks go to many
// waves), so behind its own chunk a run is a list of chunk sums and the tokens of the chunk that it ends in.
// 64 lanes take 16 bytes of the row each; a wave loads the rows of eight tokens before it adds the first.  In a row that is
// not whole vectors the last lane's vector begins earlier and shares columns with its neighbour's, which writes the same
// values there; only rows shorter than a vector (WHOLE false) go element by element.
// Bound by rows read at random, 4 KB at a time, with the cleared table on its way out.  Measured: 32768 tokens, entry v about as often as
// 1 / (v + 1), 131072 x 2048 bf16: chunks 15 us, runs 41 us, behind a sort of 94 us that clears 537 MB meanwhile (5.7 TB/s); 1024
// tokens, 30522 x 768 fp32: 3.9 and 5.6 us, behind 14 us for sort and clearing.
constexpr uint32_t kSub = 16;    // positions looked at together: their keys and tokens lie in the wave's lanes
constexpr int kRows = 8;

struct Tokens {
  const void *dout;
  const uint32_t *keys;     // sorted; entries outside the table have the key `vocab`
  const int32_t *order;
  uint32_t n, vocab, padding, chunk;
  uint32_t cols;            // waves side by side over a row
  uint64_t width;
  bool stream;              // rows are read past the caches
};

// A wave's chunk and its part of the row: the waves of one row lie side by side, so that they ask for its memory together.
struct WaveChunk {
  uint32_t chunk, col;
  __device__ __forceinline__ explicit WaveChunk(uint32_t cols) {
    const uint32_t wave = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    chunk = wave / cols;
    col = wave - chunk * cols;
  }
};

// One look at kSub positions from `base`: keys and tokens in the lanes, which positions are there, begin a run, count.
struct Look {
  uint32_t key, pos, there, starts, counts;
  __device__ __forceinline__ Look(const Tokens &t, uint32_t base) {
    const uint32_t lane = threadIdx.x & 63u, i = base + lane;
    const bool here = lane < kSub && i < t.n;
    key = here ? t.keys[i] : 0xFFFFFFFFu;
    pos = here ? (uint32_t)t.order[i] : 0u;
    const uint32_t before = here && i > 0 ? t.keys[i - 1] : 0xFFFFFFFFu;
    there = (uint32_t)__ballot(here);
    starts = (uint32_t)__ballot(here && key != before);
    counts = (uint32_t)__ballot(here && key < t.vocab && key != t.padding);
  }
};

// V columns of a row from c on
template <int DT, bool WHOLE> struct Columns {
  using E = Elems<DT>;
  uint64_t c;      // the lane's first column
  bool mine;       // lanes behind the row's end do column 0's work and store nothing
  __device__ __forceinline__ Columns(uint32_t col, uint64_t width) {
    c = ((uint64_t)col * 64u + (threadIdx.x & 63u)) * E::V;
    mine = c < width;
    if (!mine) c = 0;
    else if (WHOLE && c + E::V > width) c = width - E::V;
  }
  template <bool STREAM> __device__ __forceinline__ u32x4 load(const typename E::elem *row, uint64_t width) const {
    if constexpr (WHOLE && STREAM) return __builtin_nontemporal_load((const vec_a2 *)(row + c));
    if constexpr (WHOLE) return *(const vec_a2 *)(row + c);
    typename E::elem e[E::V];
#pragma unroll
    for (int j = 0; j < E::V; j++) e[j] = c + j < width ? row[c + j] : (typename E::elem)0;
    return __builtin_bit_cast(u32x4, e);
  }
  __device__ __forceinline__ void store(typename E::elem *row, uint64_t width, const float (&f)[E::V]) const {
    if constexpr (WHOLE) *(vec_a2 *)(row + c) = E::pack(f);
    else store_cols<DT>(row, c, width, f);
  }
  // fp32 sums of the same columns
  __device__ __forceinline__ void load_sum(const float *row, uint64_t width, float (&f)[E::V]) const {
#pragma unroll
    for (int j = 0; j < E::V; j++) f[j] = WHOLE || c + j < width ? row[c + j] : 0.f;
  }
  __device__ __forceinline__ void store_sum(float *row, uint64_t width, const float (&f)[E::V]) const {
#pragma unroll
    for (int j = 0; j < E::V; j++)
      if (WHOLE || c + j < width) row[c + j] = f[j];
  }
};

// adds the rows of the positions in `take` of one look, in order; flush(j) runs before position j is added
template <int DT, bool WHOLE, class F>
__device__ __forceinline__ void add_rows(const Tokens &t, const Look &look, uint32_t take, const Columns<DT, WHOLE> &at,
                                         float (&acc)[Elems<DT>::V], F &&flush) {
  using E = Elems<DT>;
#pragma unroll
  for (uint32_t j0 = 0; j0 < kSub; j0 += kRows) {
    if (!((take | look.starts) >> j0 & ((1u << kRows) - 1u))) continue;
    u32x4 v[kRows];
    auto load_rows = [&](auto stream) {
#pragma unroll
      for (uint32_t u = 0; u < kRows; u++) {   // positions that are not taken load row 0 and are not added
        const uint32_t row = (take >> (j0 + u)) & 1u ? (uint32_t)__builtin_amdgcn_readlane((int)look.pos, (int)(j0 + u)) : 0u;
        v[u] = at.template load<decltype(stream)::value>((const typename E::elem *)t.dout + (uint64_t)row * t.width, t.width);
      }
    };
    if (WHOLE && t.stream) load_rows(std::true_type());
    else load_rows(std::false_type());
#pragma unroll
    for (uint32_t u = 0; u < kRows; u++) {
      flush(j0 + u);
      if ((take >> (j0 + u)) & 1u) {
        float f[E::V];
        E::unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < E::V; e++) acc[e] += f[e];
      }
    }
  }
}

template <int DT, bool WHOLE> __global__ __launch_bounds__(256) void embedding_chunks_kernel(Tokens t, float *sums) {
  const WaveChunk wave(t.cols);
  const uint64_t first = (uint64_t)wave.chunk * t.chunk;
  if (first == 0 || first + t.chunk > t.n) return;
  const uint32_t key = t.keys[first - 1];
  if (key != t.keys[first + t.chunk - 1] || key >= t.vocab || key == t.padding) return;   // not inside one run
  const Columns<DT, WHOLE> at(wave.col, t.width);
  float acc[Elems<DT>::V] = {};
  for (uint32_t base = 0; base < t.chunk; base += kSub) {
    const Look look(t, (uint32_t)first + base);
    add_rows<DT, WHOLE>(t, look, look.there, at, acc, [](uint32_t) {});
  }
  if (at.mine) at.store_sum(sums + (uint64_t)wave.chunk * t.width, t.width, acc);
}

template <int DT, bool WHOLE>
__global__ __launch_bounds__(256) void embedding_runs_kernel(Tokens t, const float *sums, void *dweight, float scale) {
  using E = Elems<DT>;
  const WaveChunk wave(t.cols);
  const uint64_t first = (uint64_t)wave.chunk * t.chunk;
  if (first >= t.n) return;
  const Columns<DT, WHOLE> at(wave.col, t.width);
  float acc[E::V] = {};
  bool open = false;      // a run of this chunk is being added up
  uint32_t entry = 0;
  auto close = [&]() {
    if (open && at.mine) {
      float out[E::V];
#pragma unroll
      for (int j = 0; j < E::V; j++) out[j] = acc[j] * scale;
      at.store((typename E::elem *)dweight + (uint64_t)entry * t.width, t.width, out);
    }
#pragma unroll
    for (int j = 0; j < E::V; j++) acc[j] = 0.f;
  };
  for (uint32_t base = 0; base < t.chunk && first + base < t.n; base += kSub) {
    const Look look(t, (uint32_t)(first + base));
    // positions before the first run that begins here belong to an earlier chunk's, unless one of ours is open
    const uint32_t ours = open ? ~0u : look.starts ? ~((look.starts & (0u - look.starts)) - 1u) : 0u;
    add_rows<DT, WHOLE>(t, look, look.counts & ours, at, acc, [&](uint32_t j) {
      if (!((look.starts >> j) & 1u)) return;
      close();
      open = (look.counts >> j) & 1u;
      entry = (uint32_t)__builtin_amdgcn_readlane((int)look.key, (int)j);
    });
  }
  // The last run goes on: 64 chunks at a time, a lane asks of each whether the run fills it; their sums, eight loads at once.
  uint64_t next = first + t.chunk;
  bool filled = open;
  while (filled && next < t.n) {
    const uint64_t mine = next + (uint64_t)(threadIdx.x & 63u) * t.chunk;
    const uint64_t fills = __ballot(mine + t.chunk <= t.n && t.keys[mine + t.chunk - 1] == entry);   // sorted: so is all before it
    const int count = ~fills ? __ffsll((unsigned long long)~fills) - 1 : 64;
    const float *row = sums + next / t.chunk * t.width;
    for (int i = 0; i < count; i += kRows) {
      float f[kRows][E::V];
#pragma unroll
      for (int u = 0; u < kRows; u++) at.load_sum(row + (uint64_t)(i + u < count ? i + u : i) * t.width, t.width, f[u]);
#pragma unroll
      for (int u = 0; u < kRows; u++)
        if (i + u < count) {
#pragma unroll
          for (int e = 0; e < E::V; e++) acc[e] += f[u][e];
        }
    }
    next += (uint64_t)count * t.chunk;
    filled = count == 64;
  }
  for (uint64_t end = next + t.chunk; open && next < t.n && next < end; next += kSub) {   // and the chunk that it ends in
    Look look(t, (uint32_t)next);
    const uint32_t same = (uint32_t)__ballot(look.key == entry) & look.there;
    if (!same) break;
    look.starts = 0;
    add_rows<DT, WHOLE>(t, look, same, at, acc, [](uint32_t) {});
  }
  close();
}

// The table's gradient and the tokens' rows go through the 256 MB cache before the memory where the next reader can find them
// there, past it where they are more: then the rows do not wait for cleared lines to be written back, nor that reader.  us
// through / past the cache, an elementwise pass over the gradient included, by MB of table and rows: 106 69 / 75, 135 86 / 91,
// 168 110 / 110, 208 158 / 146, 250 128 / 119, 266 201 / 194, 671 448 / 434 (and 164 / 142 without that pass, which alone loses
// from streaming up to 266 MB of table with few rows: 46 / 59).
constexpr uint64_t kStreamBytes = 192ull << 20;
bool streams(uint64_t bytes) { return bytes > kStreamBytes; }

uint32_t chunk_of(uint64_t n) {
  uint32_t c = kSub;
  while ((uint64_t)c * 4096u < n) c *= 2u;   // at most 4096 chunk sums for one entry
  return c;
}

// ---- norm and clipping of a list of gradients -----------------------------------------------------------------------------
// One pass of partial sums, one workgroup that joins them in order, one pass that scales; each is bound by memory.  Measured:
// 182 M bf16 gradients, norm 68 us (5.3 TB/s), scaled into fp32 in 176 us (6.2 TB/s); 3.5 M fp32 elements in 51 tensors that
// need no clipping: 5.9 + 2.2 + 3.2 us, launches.
constexpr int kGrads = 128;              // tensors per launch (the table travels in the kernel arguments)
constexpr unsigned kNormBlocks = 2048;   // workgroups (= partial sums) per launch

struct GradTable {
  const void *in[kGrads];
  void *out[kGrads];
  uint64_t n[kGrads];
  uint32_t end[kGrads];    // chunks of tensors 0 .. i
  uint8_t in_dt[kGrads], out_dt[kGrads];
  int count;
  uint32_t chunk;          // elements of one workgroup's step
};

// tensor of chunk c (uniform), and c becomes the chunk within it
__device__ __forceinline__ int grad_of(const GradTable &tab, uint32_t &c) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (c < tab.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  c -= lo ? tab.end[lo - 1] : 0u;
  return lo;
}

template <int ORDER> __device__ __forceinline__ double norm_join(double a, double b) {
  if constexpr (ORDER == FPEMU_NORM_INF) return (b > a || b != b) ? b : a;   // a NaN stays
  else return a + b;
}
template <int ORDER> __device__ __forceinline__ double norm_add(double acc, float x) {
  if constexpr (ORDER == FPEMU_NORM_2) return fma((double)x, (double)x, acc);
  else return norm_join<ORDER>(acc, (double)fabsf(x));
}

// f(vector index) for this thread's whole vectors of `m` elements, four at a time, so that four loads are in flight
template <int V, class F4, class F1> __device__ __forceinline__ void each_vector(uint32_t m, F4 &&four, F1 &&one) {
  const uint32_t vecs = m / V;
  uint32_t i = threadIdx.x;
  for (; i + 768u < vecs; i += 1024u) four(i);
  for (; i < vecs; i += 256u) one(i);
}

template <int ORDER, int DT> __device__ __forceinline__ double norm_chunk(const void *in, uint32_t m, double acc) {
  using E = Elems<DT>;
  const typename E::elem *p = (const typename E::elem *)in;
  double a[4] = {acc, 0.0, 0.0, 0.0};
  auto add = [&](u32x4 v) {
    float f[E::V];
    E::unpack(v, f);
    if constexpr (ORDER == FPEMU_NORM_2 && DT != FPEMU_F32) {
      // squares of 16-bit values are exact in fp32; four of them are added there (two roundings at most, 2^-24 each)
      // before 64 bits take over.  bf16 squares outside fp32's range go one by one.
      float q[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float *g = f + 4 * h;
        q[h] = __builtin_fmaf(g[0], g[0], g[1] * g[1]) + __builtin_fmaf(g[2], g[2], g[3] * g[3]);
      }
      const float low = q[0] < q[1] ? q[0] : q[1], all = q[0] + q[1];
      const bool zeros = ((v[0] | v[1] | v[2] | v[3]) & 0x7FFF7FFFu) == 0;
      if (DT == FPEMU_F16 || zeros || (low > 0x1p-90f && all < 0x1p126f)) {
        a[0] += (double)q[0];
        a[1] += (double)q[1];
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < E::V; j++) a[j & 3] = norm_add<ORDER>(a[j & 3], f[j]);
  };
  each_vector<E::V>(
      m,
      [&](uint32_t i) {
        u32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = *(const vec_a2 *)(p + (i + u * 256u) * E::V);
#pragma unroll
        for (int u = 0; u < 4; u++) add(v[u]);
      },
      [&](uint32_t i) { add(*(const vec_a2 *)(p + i * E::V)); });
  for (uint32_t i = m / E::V * E::V + threadIdx.x; i < m; i += 256u) a[0] = norm_add<ORDER>(a[0], E::one(p + i));
  return norm_join<ORDER>(norm_join<ORDER>(a[0], a[1]), norm_join<ORDER>(a[2], a[3]));
}

// elements of chunk c of a tensor of n, and where it begins
__device__ __forceinline__ uint32_t chunk_size(const GradTable &tab, uint64_t n, uint32_t c, uint64_t &first) {
  first = (uint64_t)c * tab.chunk;
  return n - first < tab.chunk ? (uint32_t)(n - first) : tab.chunk;
}

template <int ORDER> __device__ __forceinline__ double block_join(double acc, double *tmp) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc = norm_join<ORDER>(acc, __shfl_xor(acc, off, 64));
  if ((threadIdx.x & 63u) == 0) tmp[threadIdx.x >> 6] = acc;
  __syncthreads();
  double all = tmp[0];
  for (unsigned w = 1; w < blockDim.x / 64u; w++) all = norm_join<ORDER>(all, tmp[w]);
  return all;
}

template <int ORDER> __global__ __launch_bounds__(256) void norm_kernel(GradTable tab, uint32_t chunks, double *partial) {
  __shared__ double tmp[4];
  double acc = 0.0;
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    uint32_t c = i;
    const int t = grad_of(tab, c);
    uint64_t first;
    const uint32_t m = chunk_size(tab, tab.n[t], c, first);
    if (tab.in_dt[t] == FPEMU_F32) acc = norm_chunk<ORDER, FPEMU_F32>((const float *)tab.in[t] + first, m, acc);
    else if (tab.in_dt[t] == FPEMU_F16) acc = norm_chunk<ORDER, FPEMU_F16>((const uint16_t *)tab.in[t] + first, m, acc);
    else acc = norm_chunk<ORDER, FPEMU_BF16>((const uint16_t *)tab.in[t] + first, m, acc);
  }
  const double all = block_join<ORDER>(acc, tmp);
  if (threadIdx.x == 0) partial[blockIdx.x] = all;
}

template <int ORDER> __global__ __launch_bounds__(1024) void norm_finish_kernel(const double *partial, uint32_t count, double *sum) {
  __shared__ double tmp[16];
  double acc = 0.0;
  for (uint32_t i = threadIdx.x; i < count; i += 1024u) acc = norm_join<ORDER>(acc, partial[i]);
  const double all = block_join<ORDER>(acc, tmp);
  if (threadIdx.x == 0) *sum = all;
}

// Every store of a wave is one run of 1 KB: 16 bytes a lane on the output's side, which is 8 on the side of 16-bit gradients
// that become fp32 ones.
template <int DI, int DO> __device__ __forceinline__ void clip_chunk(const void *in, void *out, uint64_t first, uint32_t m, float coef) {
  using E = Elems<DI>;
  using O = Elems<DO>;
  typedef uint32_t half_a2 __attribute__((ext_vector_type(2), aligned(2)));
  constexpr int V = O::V;   // elements of a lane's step
  const typename E::elem *p = (const typename E::elem *)in + first;
  typename O::elem *q = (typename O::elem *)out + first;
  auto get = [&](uint32_t i) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if constexpr (DI == DO) {
      v = *(const vec_a2 *)(p + i * V);
    } else {
      const half_a2 h = *(const half_a2 *)(p + i * V);
      v[0] = h[0];
      v[1] = h[1];
    }
    return v;
  };
  auto put = [&](uint32_t i, u32x4 v) {
    float f[E::V], g[V];
    E::unpack(v, f);
#pragma unroll
    for (int j = 0; j < V; j++) g[j] = f[j] * coef;
    __builtin_nontemporal_store((u32x4)O::pack(g), (vec_a2 *)(q + i * V));
  };
  each_vector<V>(
      m,
      [&](uint32_t i) {
        u32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = get(i + u * 256u);
#pragma unroll
        for (int u = 0; u < 4; u++) put(i + u * 256u, v[u]);
      },
      [&](uint32_t i) { put(i, get(i)); });
  for (uint32_t i = m / V * V + threadIdx.x; i < m; i += 256u) O::put(q + i, E::one(p + i) * coef);
}

// coef = min(1, max_norm / (norm + 1e-6)), a NaN norm gives a NaN coefficient.  Gradients that stay in place and keep
// their value (coef = 1) are not touched.
__global__ __launch_bounds__(256) void clip_kernel(GradTable tab, uint32_t chunks, int order, const double *sum, float max_norm,
                                                   float *norm_out) {
  const double s = *sum;
  const float norm = (float)(order == FPEMU_NORM_2 ? sqrt(s) : s);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float raw = max_norm / (norm + 1e-6f);
  const float coef = raw > 1.0f ? 1.0f : raw;
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    uint32_t c = chunks - 1u - i;   // backwards: what the norm read last is the likeliest to be cached still
    const int t = grad_of(tab, c);
    const void *in = tab.in[t];
    void *out = tab.out[t];
    if (coef == 1.0f && in == out) continue;
    uint64_t first;
    const uint32_t m = chunk_size(tab, tab.n[t], c, first);
    const int di = tab.in_dt[t], dout = tab.out_dt[t];
    if (di == FPEMU_F32) clip_chunk<FPEMU_F32, FPEMU_F32>(in, out, first, m, coef);
    else if (di == FPEMU_F16 && dout == FPEMU_F16) clip_chunk<FPEMU_F16, FPEMU_F16>(in, out, first, m, coef);
    else if (di == FPEMU_F16) clip_chunk<FPEMU_F16, FPEMU_F32>(in, out, first, m, coef);
    else if (dout == FPEMU_BF16) clip_chunk<FPEMU_BF16, FPEMU_BF16>(in, out, first, m, coef);
    else clip_chunk<FPEMU_BF16, FPEMU_F32>(in, out, first, m, coef);
  }
}

__global__ void norm_value_kernel(int order, const double *sum, float *norm) {
  *norm = (float)(order == FPEMU_NORM_2 ? sqrt(*sum) : *sum);
}

int check_grads(const char *who, const fpemu_grad_t *grads, uint64_t count, int order, bool with_out) {
  if (count > 0 && grads == nullptr) return fail(FPEMU_EINVAL, who, "null gradient table");
  if (order != FPEMU_NORM_INF && order != FPEMU_NORM_1 && order != FPEMU_NORM_2)
    return fail(FPEMU_EINVAL, who, "the norm's order is 1, 2 or infinity");
  for (uint64_t i = 0; i < count; i++) {
    const fpemu_grad_t &g = grads[i];
    if (g.in_dtype < FPEMU_F32 || g.in_dtype > FPEMU_BF16) return fail(FPEMU_EINVAL, who, "bad dtype id");
    if (g.n > ((uint64_t)1 << 40)) return fail(FPEMU_EINVAL, who, "more than 2^40 elements in one tensor");
    if (g.n == 0) continue;
    if (g.in == nullptr) return fail(FPEMU_EINVAL, who, "null buffer");
    if ((uintptr_t)g.in % elem_size(g.in_dtype)) return fail(FPEMU_EALIGN, who, "buffer not aligned to its element size");
    if (!with_out) continue;
    if (g.out_dtype != g.in_dtype && g.out_dtype != FPEMU_F32)
      return fail(FPEMU_EINVAL, who, "clipped gradients have the gradient's type or are fp32");
    if (g.out == nullptr) return fail(FPEMU_EINVAL, who, "null output");
    if ((uintptr_t)g.out % elem_size(g.out_dtype)) return fail(FPEMU_EALIGN, who, "output not aligned to its element size");
    const uintptr_t a = (uintptr_t)g.in, b = (uintptr_t)g.out;
    const uint64_t na = g.n * elem_size(g.in_dtype), nb = g.n * elem_size(g.out_dtype);
    if (!(a == b && g.in_dtype == g.out_dtype) && a < b + nb && b < a + na)
      return fail(FPEMU_EINVAL, who, "a gradient and its clipped form overlap without being the same buffer");
  }
  return FPEMU_OK;
}

// the next launch's table, from grads[at]; returns where the one after begins.  Steps of 8192 elements, two batches of four
// loads a thread: 182 M bf16 gradients into fp32 ones take 187 us so, from before the first launch to behind the second, 197 with
// steps of 16384, 218 with 65536.
uint64_t fill_table(const fpemu_grad_t *grads, uint64_t count, uint64_t at, GradTable &tab, uint64_t &chunks) {
  tab.count = 0;
  uint64_t elems = 0;
  for (; at < count && tab.count < kGrads; at++) {
    if (grads[at].n == 0) continue;
    const int i = tab.count++;
    tab.in[i] = grads[at].in;
    tab.out[i] = grads[at].out;
    tab.n[i] = grads[at].n;
    tab.in_dt[i] = (uint8_t)grads[at].in_dtype;
    tab.out_dt[i] = (uint8_t)grads[at].out_dtype;
    elems += grads[at].n;
  }
  tab.chunk = 8192;
  while (elems / tab.chunk > 0x3FFFFFFFull) tab.chunk *= 2;
  chunks = 0;
  for (int i = 0; i < tab.count; i++) {
    chunks += ceil_div(tab.n[i], tab.chunk);
    tab.end[i] = (uint32_t)chunks;
  }
  return at;
}

}  // namespace

extern "C" {

uint64_t fpemu_group_rows_workspace_bytes(uint64_t n, uint64_t groups) {
  if (n > 0x7FFFFFFFull || groups < 1 || groups > 0x7FFFFFFEull) return 0;
  return 4u * sort_space(n, groups, false).words;
}

int fpemu_group_rows(const void *ids, int id_bytes, uint64_t n, uint64_t groups, int32_t *order, int32_t *offsets, void *ws,
                     uint64_t ws_bytes, void *stream) {
  const char *who = "fpemu_group_rows";
  if (const int rc = check_ids(who, ids, id_bytes, n, groups)) return rc;
  if ((n > 0 && order == nullptr) || offsets == nullptr) return fail(FPEMU_EINVAL, who, "null output");
  const uint64_t need = fpemu_group_rows_workspace_bytes(n, groups);
  if (need > 0 && (ws == nullptr || ws_bytes < need)) return fail(FPEMU_EINVAL, who, "workspace too small");
  if ((uintptr_t)ws % 16u || (uintptr_t)order % 4u || (uintptr_t)offsets % 4u)
    return fail(FPEMU_EALIGN, who, "workspace (16 bytes) or output (4 bytes) not aligned");
  return sort_rows(who, ids, id_bytes == 8, n, groups, order, offsets, false, (uint32_t *)ws, Fill{}, (hipStream_t)stream);
}

static int check_embedding(const char *who, const void *a, const void *b, uint64_t n, uint64_t width, int dtype) {
  if (dtype < FPEMU_F32 || dtype > FPEMU_BF16) return fail(FPEMU_EINVAL, who, "bad dtype id");
  if (width > ((uint64_t)1 << 31)) return fail(FPEMU_EINVAL, who, "rows of more than 2^31 elements");
  if (width == 0) return FPEMU_OK;
  if (a == nullptr || (n > 0 && b == nullptr)) return fail(FPEMU_EINVAL, who, "null buffer");
  if ((uintptr_t)a % elem_size(dtype) || (uintptr_t)b % elem_size(dtype))
    return fail(FPEMU_EALIGN, who, "buffer not aligned to its element size");
  return FPEMU_OK;
}

int fpemu_embedding(const void *weight, const void *ids, int id_bytes, void *out, uint64_t n, uint64_t vocab, uint64_t width,
                    int dtype, float scale, void *stream) {
  const char *who = "fpemu_embedding";
  if (const int rc = check_ids(who, ids, id_bytes, n, vocab)) return rc;
  if (const int rc = check_embedding(who, weight, out, n, width, dtype)) return rc;
  if (n == 0 || width == 0) return FPEMU_OK;
  const uint64_t vecs = ceil_div(width, vec_elems(dtype));
  int lg = 0;
  while (lg < 8 && ((uint64_t)1 << lg) < vecs) lg++;
  const uint64_t rows = 256u >> lg;   // of a workgroup, times 1 or 4: four only where enough workgroups are left
  const bool four = n >= rows * 4 * 1024;
  const unsigned blocks = (unsigned)ceil_div(n, four ? rows * 4 : rows);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { kernel<<<blocks, 256, 0, s>>>(weight, ids, id_bytes == 8, out, n, vocab, width, scale, lg); };
  if (dtype == FPEMU_F32) four ? go(embedding_kernel<FPEMU_F32, 4>) : go(embedding_kernel<FPEMU_F32, 1>);
  else if (dtype == FPEMU_F16) four ? go(embedding_kernel<FPEMU_F16, 4>) : go(embedding_kernel<FPEMU_F16, 1>);
  else four ? go(embedding_kernel<FPEMU_BF16, 4>) : go(embedding_kernel<FPEMU_BF16, 1>);
  return launched(who);
}

// words before the chunk sums: the sort's and the order
static uint64_t embedding_words(uint64_t n, uint64_t vocab) {
  const uint64_t words = sort_space(n, vocab, true).words + n;
  return (words + 3) / 4 * 4;
}

uint64_t fpemu_embedding_grad_workspace_bytes(uint64_t n, uint64_t vocab, uint64_t width) {
  if (n > 0x7FFFFFFFull || vocab < 1 || vocab > 0x7FFFFFFEull || width > ((uint64_t)1 << 31)) return 0;
  return 4u * (embedding_words(n, vocab) + n / chunk_of(n) * width);
}

int fpemu_embedding_grad(const void *dout, const void *ids, int id_bytes, void *dweight, uint64_t n, uint64_t vocab,
                         uint64_t width, int dtype, float scale, int64_t padding, void *ws, uint64_t ws_bytes, void *stream) {
  const char *who = "fpemu_embedding_grad";
  if (const int rc = check_ids(who, ids, id_bytes, n, vocab)) return rc;
  if (const int rc = check_embedding(who, dweight, dout, n, width, dtype)) return rc;
  if (width == 0) return FPEMU_OK;
  if (n > 0 && (ws == nullptr || ws_bytes < fpemu_embedding_grad_workspace_bytes(n, vocab, width)))
    return fail(FPEMU_EINVAL, who, "workspace too small");
  if ((uintptr_t)ws % 16u) return fail(FPEMU_EALIGN, who, "workspace not aligned to 16 bytes");
  const uint64_t cols = ceil_div(width, 64u * vec_elems(dtype));
  if (cols > 65535u) return fail(FPEMU_EINVAL, who, "table too wide for one launch");
  const uint64_t bytes = vocab * width * elem_size(dtype);
  if (ceil_div(bytes, kFillPiece) > 0x7FFFFFFFull) return fail(FPEMU_EINVAL, who, "table too large for one launch");
  hipStream_t s = (hipStream_t)stream;
  const bool past = streams(bytes + n * width * elem_size(dtype));
  uint32_t *words = (uint32_t *)ws;
  const SortSpace sp = sort_space(n, vocab, true);
  int32_t *order = (int32_t *)(words + sp.words);
  float *sums = (float *)(words + embedding_words(n, vocab));
  if (const int rc = sort_rows(who, ids, id_bytes == 8, n, vocab, order, nullptr, true, words, Fill{(char *)dweight, bytes, 0, 0, past}, s)) return rc;
  if (n == 0) return FPEMU_OK;
  const uint32_t chunk = chunk_of(n);
  const Tokens t{dout, words + sp.keys, order, (uint32_t)n, (uint32_t)vocab, padding >= 0 && (uint64_t)padding < vocab ? (uint32_t)padding : 0xFFFFFFFFu,
                 chunk, (uint32_t)cols, width, past};
  const unsigned grid = (unsigned)ceil_div(ceil_div(n, chunk) * cols, 4);   // at most 4096 chunks, 65535 parts of a row
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const bool whole = width >= (uint64_t)Elems<DT>::V;
    if (n > chunk) {
      if (whole) embedding_chunks_kernel<DT, true><<<grid, 256, 0, s>>>(t, sums);
      else embedding_chunks_kernel<DT, false><<<grid, 256, 0, s>>>(t, sums);
    }
    if (whole) embedding_runs_kernel<DT, true><<<grid, 256, 0, s>>>(t, sums, dweight, scale);
    else embedding_runs_kernel<DT, false><<<grid, 256, 0, s>>>(t, sums, dweight, scale);
  };
  if (dtype == FPEMU_F32) go(std::integral_constant<int, FPEMU_F32>());
  else if (dtype == FPEMU_F16) go(std::integral_constant<int, FPEMU_F16>());
  else go(std::integral_constant<int, FPEMU_BF16>());
  return launched(who);
}

uint64_t fpemu_grad_norm_workspace_bytes(uint64_t count) { return 8u * kNormBlocks * (ceil_div(count, kGrads) + 1u); }

int fpemu_grad_norm_multi(const fpemu_grad_t *grads, uint64_t count, int order, double *sum, float *norm, void *ws,
                          uint64_t ws_bytes, void *stream) {
  const char *who = "fpemu_grad_norm_multi";
  if (const int rc = check_grads(who, grads, count, order, false)) return rc;
  if (sum == nullptr || ws == nullptr || ws_bytes < fpemu_grad_norm_workspace_bytes(count))
    return fail(FPEMU_EINVAL, who, "null sum or workspace too small");
  if ((uintptr_t)sum % 8u || (uintptr_t)ws % 8u || (uintptr_t)norm % 4u) return fail(FPEMU_EALIGN, who, "sum, norm or workspace not aligned");
  hipStream_t s = (hipStream_t)stream;
  double *partial = (double *)ws;
  uint32_t used = 0;
  GradTable tab{};
  for (uint64_t at = 0; at < count;) {
    uint64_t chunks;
    at = fill_table(grads, count, at, tab, chunks);
    if (chunks == 0) continue;
    const unsigned blocks = chunks < kNormBlocks ? (unsigned)chunks : kNormBlocks;
    if (order == FPEMU_NORM_2) norm_kernel<FPEMU_NORM_2><<<blocks, 256, 0, s>>>(tab, (uint32_t)chunks, partial + used);
    else if (order == FPEMU_NORM_1) norm_kernel<FPEMU_NORM_1><<<blocks, 256, 0, s>>>(tab, (uint32_t)chunks, partial + used);
    else norm_kernel<FPEMU_NORM_INF><<<blocks, 256, 0, s>>>(tab, (uint32_t)chunks, partial + used);
    used += blocks;
  }
  if (order == FPEMU_NORM_2) norm_finish_kernel<FPEMU_NORM_2><<<1, 1024, 0, s>>>(partial, used, sum);
  else if (order == FPEMU_NORM_1) norm_finish_kernel<FPEMU_NORM_1><<<1, 1024, 0, s>>>(partial, used, sum);
  else norm_finish_kernel<FPEMU_NORM_INF><<<1, 1024, 0, s>>>(partial, used, sum);
  if (norm != nullptr) norm_value_kernel<<<1, 1, 0, s>>>(order, sum, norm);
  return launched(who);
}

int fpemu_clip_multi(const fpemu_grad_t *grads, uint64_t count, int order, const double *sum, float max_norm, float *norm,
                     void *stream) {
  const char *who = "fpemu_clip_multi";
  if (const int rc = check_grads(who, grads, count, order, true)) return rc;
  if (sum == nullptr) return fail(FPEMU_EINVAL, who, "null sum");
  if (!(max_norm >= 0.0f)) return fail(FPEMU_EINVAL, who, "max_norm is not negative and not NaN");
  if ((uintptr_t)sum % 8u || (uintptr_t)norm % 4u) return fail(FPEMU_EALIGN, who, "sum or norm not aligned");
  hipStream_t s = (hipStream_t)stream;
  GradTable tab{};
  bool told = false;
  for (uint64_t at = 0; at < count;) {
    uint64_t chunks;
    at = fill_table(grads, count, at, tab, chunks);
    if (chunks == 0) continue;
    const unsigned blocks = chunks < 0x7FFFFFFFull ? (unsigned)chunks : 0x7FFFFFFFu;
    clip_kernel<<<blocks, 256, 0, s>>>(tab, (uint32_t)chunks, order, sum, max_norm, told ? nullptr : norm);
    told = true;
  }
  if (!told && norm != nullptr) norm_value_kernel<<<1, 1, 0, s>>>(order, sum, norm);
  return launched(who);
}

}  // extern "C"
