// fpemu_train.hip -- operators of a language model's training step that run beside the emulated cast: rows in the
// order of their group (a router's experts, a vocabulary's entries), the scaled embedding lookup with the gradient of
// its table, and the norm and clipping of a whole list of gradients.  Sums are held in 32 bits (table gradient) or
// 64 bits (norms) and rounded once, when they are stored.  No floating-point atomics: every sum has one fixed order,
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
// A stable counting sort by digits of the group id, least significant digit first (one pass up to 1024 keys, two up to
// 2^20, ...).  A row outside [0, groups) has the key `groups` and so ends up behind every group.  The rank of a row
// among the equal digits before it is found wave by wave: ballots over the digit's bits give the lanes with the same
// digit, one LDS counter per (wave, digit) carries the count from round to round.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64, kSortRounds = 8;
constexpr int kSortTile = kSortThreads * kSortRounds;   // 4096 rows per workgroup
constexpr int kMaxBits = 10;                            // digits of at most 1024 values: 32 KB of counters
constexpr int kMaxBins = 1 << kMaxBits;
constexpr unsigned kSelfSum = 32;                       // up to this many tiles a tile adds up the counts before it by itself

struct SortPlan {
  int bits, passes, shift[4], width[4];
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

__device__ __forceinline__ uint32_t key_of(const void *ids, int wide, uint64_t i, uint32_t groups) {
  if (wide) {
    const uint64_t v = ((const uint64_t *)ids)[i];
    return v < groups ? (uint32_t)v : groups;
  }
  const uint32_t v = ((const uint32_t *)ids)[i];
  return v < groups ? v : groups;
}

// rank of each of the lane's rows among the rows of its wave with the same digit before it; cnt: the wave's counters
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[kSortRounds], unsigned valid, int bits, uint32_t *cnt,
                                           uint32_t (&rank)[kSortRounds]) {
  const unsigned lane = threadIdx.x & 63u;
  const uint64_t below = ((uint64_t)1 << lane) - 1u;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
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
  constexpr int PER = kMaxBins / kSortThreads;   // 2
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t x[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int at = (int)threadIdx.x * PER + i;
    x[i] = at < bins ? v[at] : 0u;
    sum += x[i];
  }
  uint32_t inc = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)inc, off, 64);
    if ((int)lane >= off) inc += o;
  }
  if (lane == 63u) tmp[wave] = inc;
  __syncthreads();
  uint32_t run = inc - sum;
  for (unsigned w = 0; w < wave; w++) run += tmp[w];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int at = (int)threadIdx.x * PER + i;
    if (at < bins) v[at] = run;
    run += x[i];
  }
  __syncthreads();
}

// Up to kSortTile rows: every pass inside one workgroup, rows exchanged through LDS.  keys_out: the sorted keys
// (passes > 1 only; the offsets are searched in them); with one pass the offsets are the counters' sums.
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const void *ids, int wide, uint32_t n, uint32_t groups,
                                                                  SortPlan plan, int32_t *order, uint32_t *keys_out,
                                                                  int32_t *offsets) {
  __shared__ uint32_t cnt[kSortWaves * kMaxBins];
  __shared__ uint32_t skey[kSortTile];
  __shared__ uint16_t spos[kSortTile];
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t tmp[kSortWaves];
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t key[kSortRounds], pos[kSortRounds], digit[kSortRounds], rank[kSortRounds];
  unsigned valid = 0;
#pragma unroll
  for (int r = 0; r < kSortRounds; r++) {
    const uint32_t i = wave * (64u * kSortRounds) + (uint32_t)r * 64u + lane;
    pos[r] = i;
    key[r] = 0;
    if (i < n) {
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
    wave_ranks(digit, valid, plan.width[p], cnt + wave * bins, rank);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
      uint32_t run = 0;
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
        const uint32_t i = wave * (64u * kSortRounds) + (uint32_t)r * 64u + lane;
        if (i < n) {
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
                                                                  uint32_t tiles, uint32_t *counts) {
  __shared__ uint32_t cnt[kMaxBins];
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
                                                                  int32_t *offsets) {
  __shared__ uint32_t cnt[kSortWaves * kMaxBins];
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t tmp[kSortWaves];
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
  for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  wave_ranks(digit, valid, width, cnt + wave * bins, rank);
  __syncthreads();
  // per digit: rows before this tile's (own[]), and all rows (base[], turned into the digit's start below)
  constexpr int PER = kMaxBins / kSortThreads;
  uint32_t own[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int d = (int)threadIdx.x + j * kSortThreads;
    own[j] = 0;
    if (d < bins) {
      if (totals != nullptr) {
        own[j] = counts[(uint64_t)d * tiles + blockIdx.x];
        base[d] = totals[d];
      } else {
        uint32_t all = 0, before = 0;
        for (uint32_t t = 0; t < tiles; t++) {
          const uint32_t c = counts[(uint64_t)d * tiles + t];
          before += t < blockIdx.x ? c : 0u;
          all += c;
        }
        own[j] = before;
        base[d] = all;
      }
    }
  }
  __syncthreads();
  exclusive_bins(base, bins, tmp);
  if (offsets != nullptr && blockIdx.x == 0)
    for (uint32_t g = threadIdx.x; g <= groups; g += kSortThreads) offsets[g] = (int32_t)base[g];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int d = (int)threadIdx.x + j * kSortThreads;
    if (d < bins) {
      uint32_t run = base[d] + own[j];
      for (int w = 0; w < kSortWaves; w++) {
        const uint32_t c = cnt[w * bins + d];
        cnt[w * bins + d] = run;
        run += c;
      }
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

__global__ __launch_bounds__(256) void zero_words_kernel(int32_t *p, uint64_t n) {
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (i < n) p[i] = 0;
}

// workspace of the sort, in words: [keys a][pos a][keys b] + counts + totals (passes alternate between a and b; the last
// pass writes its positions to `order`)
struct SortSpace {
  uint64_t keys_a, pos_a, keys_b, counts, totals, words;
};

SortSpace sort_space(uint64_t n, uint64_t groups) {
  const SortPlan plan = sort_plan(groups);
  const uint64_t tiles = ceil_div(n, kSortTile);
  SortSpace s{};
  uint64_t at = 0;
  auto take = [&](uint64_t words) { const uint64_t o = at; at += (words + 3) / 4 * 4; return o; };
  if (plan.passes > 1) s.keys_b = take(n);
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

// order[n], offsets[groups + 1]; ws of sort_space().words words
int sort_rows(const char *who, const void *ids, int wide, uint64_t n, uint64_t groups, int32_t *order, int32_t *offsets,
              uint32_t *ws, hipStream_t stream) {
  const SortPlan plan = sort_plan(groups);
  const SortSpace sp = sort_space(n, groups);
  const uint32_t n32 = (uint32_t)n, g32 = (uint32_t)groups;
  if (n == 0) {
    zero_words_kernel<<<(unsigned)ceil_div(groups + 1, 256), 256, 0, stream>>>(offsets, groups + 1);
    return launched(who);
  }
  const uint32_t tiles = (uint32_t)ceil_div(n, kSortTile);
  const uint32_t *sorted = nullptr;
  if (tiles == 1) {
    uint32_t *keys = plan.passes > 1 ? ws + sp.keys_b : nullptr;
    sort_small_kernel<<<1, kSortThreads, 0, stream>>>(ids, wide, n32, g32, plan, order, keys, offsets);
    sorted = keys;
  } else {
    SortIn in{ids, nullptr, nullptr, wide};
    for (int p = 0; p < plan.passes; p++) {
      const bool last = p + 1 == plan.passes;
      // the last pass's keys go to b (only the offsets read them); the ones before alternate so that they end in a
      uint32_t *keys = plan.passes == 1 ? nullptr : ws + (((plan.passes - 1 - p) & 1) ? sp.keys_a : sp.keys_b);
      int32_t *pos = last || ((plan.passes - 1 - p) & 1) == 0 ? order : (int32_t *)(ws + sp.pos_a);
      sort_count_kernel<<<tiles, kSortThreads, 0, stream>>>(in, n32, g32, plan.shift[p], plan.width[p], tiles, ws + sp.counts);
      const uint32_t *totals = nullptr;
      if (tiles > kSelfSum) {
        const int bins = 1 << plan.width[p];
        sort_scan_kernel<<<(unsigned)ceil_div(bins, 4), 256, 0, stream>>>(ws + sp.counts, tiles, bins, ws + sp.totals);
        totals = ws + sp.totals;
      }
      sort_place_kernel<<<tiles, kSortThreads, 0, stream>>>(in, n32, g32, plan.shift[p], plan.width[p], tiles, ws + sp.counts,
                                                            totals, keys, pos, plan.passes == 1 ? offsets : nullptr);
      in.keys = keys;
      in.pos = pos;
      sorted = keys;
    }
  }
  if (plan.passes > 1)
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
typedef uint32_t vec_a2 __attribute__((ext_vector_type(4), aligned(2)));   // rows of odd widths: element-aligned only

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

// out[t] = scale * weight[ids[t]]: 2^lg_tpr threads a row.  A row whose id is outside the table reads nothing and is NaN.
template <int DT>
__global__ __launch_bounds__(256) void embedding_kernel(const void *weight, const void *ids, int wide, void *out, uint64_t n,
                                                        uint64_t vocab, uint64_t width, float scale, int lg_tpr) {
  using E = Elems<DT>;
  const uint64_t t = (uint64_t)blockIdx.x * (256u >> lg_tpr) + (threadIdx.x >> lg_tpr);
  if (t >= n) return;
  const int64_t id = id_at(ids, wide, t);
  const bool known = id >= 0 && (uint64_t)id < vocab;
  const typename E::elem *src = (const typename E::elem *)weight + (known ? (uint64_t)id : 0u) * width;
  typename E::elem *dst = (typename E::elem *)out + t * width;
  const uint64_t step = (uint64_t)E::V << lg_tpr;
  for (uint64_t c = (uint64_t)(threadIdx.x & ((1u << lg_tpr) - 1u)) * E::V; c < width; c += step) {
    float f[E::V];
    if (known) {
      load_cols<DT>(src, c, width, f);
#pragma unroll
      for (int j = 0; j < E::V; j++) f[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < E::V; j++) f[j] = u2f(0x7FC00000u);
    }
    store_cols<DT>(dst, c, width, f);
  }
}

// Gradient of the table from the sorted tokens.  The sorted positions are cut into chunks of `chunk`; a chunk that lies
// inside one entry's run is summed by embedding_chunks_kernel (a frequent token's run is long: its chunks go to many
// workgroups), and an entry's row is the sum of its chunks' sums and of the tokens at its two ends.
template <int DT>
__global__ __launch_bounds__(64) void embedding_chunks_kernel(const void *dout, const void *ids, int wide, const int32_t *order,
                                                              uint32_t n, uint64_t width, uint32_t chunk, float *sums) {
  using E = Elems<DT>;
  const uint32_t first = blockIdx.x * chunk;
  if ((uint64_t)first + chunk > n) return;
  if (id_at(ids, wide, (uint64_t)order[first]) != id_at(ids, wide, (uint64_t)order[first + chunk - 1u])) return;
  const uint64_t c = ((uint64_t)blockIdx.y * 64u + threadIdx.x) * E::V;
  if (c >= width) return;
  float acc[E::V] = {};
#pragma unroll 4
  for (uint32_t i = 0; i < chunk; i++) {
    float f[E::V];
    load_cols<DT>((const typename E::elem *)dout + (uint64_t)order[first + i] * width, c, width, f);
#pragma unroll
    for (int j = 0; j < E::V; j++) acc[j] += f[j];
  }
  float *row = sums + (uint64_t)blockIdx.x * width;
#pragma unroll
  for (int j = 0; j < E::V; j++)
    if (c + j < width) row[c + j] = acc[j];
}

template <int DT>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const void *dout, const int32_t *order, const int32_t *offsets,
                                                             const float *sums, void *dweight, uint64_t vocab, uint64_t width,
                                                             uint32_t chunk, float scale, int64_t padding) {
  using E = Elems<DT>;
  const uint64_t v = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
  if (v >= vocab) return;
  const uint64_t c = ((uint64_t)blockIdx.y * 64u + (threadIdx.x & 63u)) * E::V;
  if (c >= width) return;
  uint32_t i = (uint32_t)offsets[v];
  const uint32_t end = (int64_t)v == padding ? i : (uint32_t)offsets[v + 1];
  float acc[E::V] = {};
  while (i < end) {
    if (i % chunk == 0 && i + chunk <= end) {
      const float *row = sums + (uint64_t)(i / chunk) * width;
#pragma unroll
      for (int j = 0; j < E::V; j++)
        if (c + j < width) acc[j] += row[c + j];
      i += chunk;
    } else {
      float f[E::V];
      load_cols<DT>((const typename E::elem *)dout + (uint64_t)order[i] * width, c, width, f);
#pragma unroll
      for (int j = 0; j < E::V; j++) acc[j] += f[j];
      i++;
    }
  }
#pragma unroll
  for (int j = 0; j < E::V; j++) acc[j] *= scale;
  store_cols<DT>((typename E::elem *)dweight + v * width, c, width, acc);
}

uint32_t chunk_of(uint64_t n) {
  uint32_t c = 32;
  while ((uint64_t)c * 2048u < n) c *= 2u;   // at most 2048 chunk sums for one entry
  return c;
}

// ---- norm and clipping of a list of gradients -----------------------------------------------------------------------------
constexpr int kGrads = 128;              // tensors per launch (the table travels in the kernel arguments)
constexpr uint64_t kGradChunk = 16384;   // elements of one workgroup's step
constexpr unsigned kNormBlocks = 1024;   // workgroups (= partial sums) per launch

struct GradTable {
  const void *in[kGrads];
  void *out[kGrads];
  uint64_t n[kGrads];
  uint32_t end[kGrads];    // chunks of tensors 0 .. i
  uint8_t in_dt[kGrads], out_dt[kGrads];
  int count;
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

template <int ORDER, int DT> __device__ __forceinline__ double norm_chunk(const void *in, uint64_t n, uint32_t chunk, double acc) {
  using E = Elems<DT>;
  const typename E::elem *p = (const typename E::elem *)in + (uint64_t)chunk * kGradChunk;
  const uint64_t left = n - (uint64_t)chunk * kGradChunk;
  const uint32_t m = left < kGradChunk ? (uint32_t)left : (uint32_t)kGradChunk;
  double a[4] = {acc, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (uint32_t c = threadIdx.x * E::V; c < m; c += 256u * E::V) {
    float f[E::V];
    load_cols<DT>(p, c, m, f);
#pragma unroll
    for (int j = 0; j < E::V; j++) a[j & 3] = norm_add<ORDER>(a[j & 3], f[j]);
  }
  return norm_join<ORDER>(norm_join<ORDER>(a[0], a[1]), norm_join<ORDER>(a[2], a[3]));
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
    if (tab.in_dt[t] == FPEMU_F32) acc = norm_chunk<ORDER, FPEMU_F32>(tab.in[t], tab.n[t], c, acc);
    else if (tab.in_dt[t] == FPEMU_F16) acc = norm_chunk<ORDER, FPEMU_F16>(tab.in[t], tab.n[t], c, acc);
    else acc = norm_chunk<ORDER, FPEMU_BF16>(tab.in[t], tab.n[t], c, acc);
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

template <int DI, int DO> __device__ __forceinline__ void clip_chunk(const void *in, void *out, uint64_t n, uint32_t chunk, float coef) {
  using E = Elems<DI>;
  using O = Elems<DO>;
  const typename E::elem *p = (const typename E::elem *)in + (uint64_t)chunk * kGradChunk;
  typename O::elem *q = (typename O::elem *)out + (uint64_t)chunk * kGradChunk;
  const uint64_t left = n - (uint64_t)chunk * kGradChunk;
  const uint32_t m = left < kGradChunk ? (uint32_t)left : (uint32_t)kGradChunk;
#pragma unroll 4
  for (uint32_t c = threadIdx.x * E::V; c < m; c += 256u * E::V) {
    float f[E::V];
    load_cols<DI>(p, c, m, f);
#pragma unroll
    for (int j = 0; j < E::V; j++) f[j] *= coef;
    if constexpr (DI == DO) {
      store_cols<DO>(q, c, m, f);
    } else {   // 16-bit gradients into fp32 ones: two vectors
#pragma unroll
      for (int h = 0; h < E::V; h += O::V) {
        float g[O::V];
#pragma unroll
        for (int j = 0; j < O::V; j++) g[j] = f[h + j];
        if (c + h < m) store_cols<DO>(q, c + h, m, g);
      }
    }
  }
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
    const int di = tab.in_dt[t], dout = tab.out_dt[t];
    if (di == FPEMU_F32) clip_chunk<FPEMU_F32, FPEMU_F32>(in, out, tab.n[t], c, coef);
    else if (di == FPEMU_F16 && dout == FPEMU_F16) clip_chunk<FPEMU_F16, FPEMU_F16>(in, out, tab.n[t], c, coef);
    else if (di == FPEMU_F16) clip_chunk<FPEMU_F16, FPEMU_F32>(in, out, tab.n[t], c, coef);
    else if (dout == FPEMU_BF16) clip_chunk<FPEMU_BF16, FPEMU_BF16>(in, out, tab.n[t], c, coef);
    else clip_chunk<FPEMU_BF16, FPEMU_F32>(in, out, tab.n[t], c, coef);
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
    if (g.n > ((uint64_t)1 << 45)) return fail(FPEMU_EINVAL, who, "more than 2^45 elements in one tensor");
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

// the next launch's table, from grads[at]; returns where the one after begins
uint64_t fill_table(const fpemu_grad_t *grads, uint64_t count, uint64_t at, GradTable &tab, uint64_t &chunks) {
  tab.count = 0;
  chunks = 0;
  for (; at < count && tab.count < kGrads; at++) {
    if (grads[at].n == 0) continue;
    const uint64_t c = ceil_div(grads[at].n, kGradChunk);
    if (chunks + c > 0xFFFFFFFFull) break;
    chunks += c;
    const int i = tab.count++;
    tab.in[i] = grads[at].in;
    tab.out[i] = grads[at].out;
    tab.n[i] = grads[at].n;
    tab.end[i] = (uint32_t)chunks;
    tab.in_dt[i] = (uint8_t)grads[at].in_dtype;
    tab.out_dt[i] = (uint8_t)grads[at].out_dtype;
  }
  return at;
}

}  // namespace

extern "C" {

uint64_t fpemu_group_rows_workspace_bytes(uint64_t n, uint64_t groups) {
  if (n > 0x7FFFFFFFull || groups < 1 || groups > 0x7FFFFFFEull) return 0;
  return 4u * sort_space(n, groups).words;
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
  return sort_rows(who, ids, id_bytes == 8, n, groups, order, offsets, (uint32_t *)ws, (hipStream_t)stream);
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
  const unsigned blocks = (unsigned)ceil_div(n, 256u >> lg);
  const int wide = id_bytes == 8;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == FPEMU_F32) embedding_kernel<FPEMU_F32><<<blocks, 256, 0, s>>>(weight, ids, wide, out, n, vocab, width, scale, lg);
  else if (dtype == FPEMU_F16) embedding_kernel<FPEMU_F16><<<blocks, 256, 0, s>>>(weight, ids, wide, out, n, vocab, width, scale, lg);
  else embedding_kernel<FPEMU_BF16><<<blocks, 256, 0, s>>>(weight, ids, wide, out, n, vocab, width, scale, lg);
  return launched(who);
}

// words before the chunk sums: the sort's, the order, the offsets
static uint64_t embedding_words(uint64_t n, uint64_t vocab) {
  const uint64_t words = sort_space(n, vocab).words + n + vocab + 1;
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
  if (ws == nullptr || ws_bytes < fpemu_embedding_grad_workspace_bytes(n, vocab, width))
    return fail(FPEMU_EINVAL, who, "workspace too small");
  if ((uintptr_t)ws % 16u) return fail(FPEMU_EALIGN, who, "workspace not aligned to 16 bytes");
  const int wide = id_bytes == 8;
  hipStream_t s = (hipStream_t)stream;
  uint32_t *words = (uint32_t *)ws;
  int32_t *order = (int32_t *)(words + sort_space(n, vocab).words), *offsets = order + n;
  float *sums = (float *)(words + embedding_words(n, vocab));
  if (const int rc = sort_rows(who, ids, wide, n, vocab, order, offsets, words, s)) return rc;
  const uint32_t chunk = chunk_of(n);
  const unsigned cols = (unsigned)ceil_div(width, 64u * vec_elems(dtype));
  if (cols > 65535u || vocab > 0x7FFFFFFFull) return fail(FPEMU_EINVAL, who, "table too wide for one launch");
  const dim3 cgrid((unsigned)(n / chunk), cols), rgrid((unsigned)ceil_div(vocab, 4), cols);
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (cgrid.x > 0)
      embedding_chunks_kernel<DT><<<cgrid, 64, 0, s>>>(dout, ids, wide, order, (uint32_t)n, width, chunk, sums);
    embedding_rows_kernel<DT><<<rgrid, 256, 0, s>>>(dout, order, offsets, sums, dweight, vocab, width, chunk, scale, padding);
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
