// Embedding lookup with scaling and its gradient for gfx950.
//
//   rows[i] = scale * table[ids[i]]          d_table[v] = scale * sum over { i : ids[i] = v } of d_out[i]
//
// The batch gathers of DiffGraph-Rec/Model.py:101-105 and what autograd forms for them, for tables of any width in fp32,
// bf16 or fp16.  The gradient is formed token by token, never by atomics on the rows: the (id, position) pairs are
// sorted by id -- stably, so a token's positions stay in order -- and each run of equal ids is summed in fp32 in that
// order, whole runs by the lanes that meet them, runs that cross from one chunk of the sorted list into the next through
// partial sums added chunk by chunk.  Every output row is written once, by one owner: the same bits on every run.
#include "dg_internal.h"
#include "dg_types.h"

namespace {

// ---- lookup ---------------------------------------------------------------------------------------------------------
// GL lanes per row, VEC elements per lane and step.  An id outside the table gathers nothing: its row is NaN.  One read and
// one write, bound by memory: 65536 rows of 1024 bf16 in 43 us (6.2 TB/s read and written); 6144 of 128 fp32 in 3.2 us, a
// launch's latency and a row's.
template <typename T, int VEC, int GL>
__global__ __launch_bounds__(256) void embedding_lookup_kernel(const T *__restrict__ table, int64_t n_rows, int64_t stride, int dim,
                                                               const void *__restrict__ ids, int ids64, int64_t n_ids, float scale,
                                                               T *__restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * (256 / GL) + threadIdx.x / GL;
  if (i >= n_ids) return;
  const int64_t id = ids64 ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
  const bool ok = (uint64_t)id < (uint64_t)n_rows;
  const T *src = table + (ok ? id : 0) * stride;
  T *dst = out + i * dim;
  for (int c = (threadIdx.x % GL) * VEC; c < dim; c += GL * VEC) {
    float f[VEC];
    if (ok) {
      dg_load_unaligned<VEC>(src + c, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = __builtin_nanf("");
    }
    dg_store_unaligned<VEC>(dst + c, f);
  }
}

// ---- stable radix sort of (id, position) ------------------------------------------------------------------------------
// Passes over at most kMaxDigit bits, low digit first; ids that take no gradient (outside the table, the padding id) get
// the key n_rows, behind all others.  A pass: digit counts per block, per-digit scans over the blocks, stable scatter.
// Bound by launches and by the latency of a block's few dependent steps, not by its bytes: 65536 ids of 18 bits take two
// passes of 4.8 + 9.1 us for 1 MB.
constexpr int kMaxDigit = 10, kWaves = 4;
constexpr int kSelfScan = 64;     // up to so many blocks a scatter adds their counts up itself (one launch less)

struct key_source {
  const void *ids;      // first pass: the caller's ids
  int ids64;
  int64_t padding;
  uint32_t n_rows;
  const uint32_t *keys, *pos;   // later passes
};

// N entries, `step` apart, all on their way at once (an entry behind the list: some other one, to be left aside).
template <int N>
__device__ __forceinline__ void load_keys(const key_source &s, int64_t first, int step, int64_t n, uint32_t (&key)[N], uint32_t (&pos)[N]) {
  if (s.keys) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t i = min(first + e * step, n - 1);
      key[e] = s.keys[i];
      pos[e] = s.pos[i];
    }
    return;
  }
  int64_t id[N];
  if (s.ids64) {
#pragma unroll
    for (int e = 0; e < N; ++e) id[e] = ((const int64_t *)s.ids)[min(first + e * step, n - 1)];
  } else {
    int32_t low[N];
#pragma unroll
    for (int e = 0; e < N; ++e) low[e] = ((const int32_t *)s.ids)[min(first + e * step, n - 1)];
#pragma unroll
    for (int e = 0; e < N; ++e) id[e] = low[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    key[e] = ((uint64_t)id[e] >= (uint64_t)s.n_rows || id[e] == s.padding) ? s.n_rows : (uint32_t)id[e];
    pos[e] = (uint32_t)(first + e * step);
  }
}

// counts[digit][block], or [block][digit] where the scatter adds the blocks up itself
template <int IPT>
__global__ __launch_bounds__(256) void radix_count_kernel(key_source s, int64_t n, int shift, int bits, int n_blocks, int by_block,
                                                          uint32_t *__restrict__ counts, uint32_t *__restrict__ n_crossing) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *n_crossing = 0;
  __shared__ uint32_t hist[1 << kMaxDigit];
  const int bins = 1 << bits;
  for (int d = threadIdx.x; d < bins; d += 256) hist[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (256 * IPT);
  uint32_t key[IPT], pos[IPT];
  load_keys<IPT>(s, base + threadIdx.x, 256, n, key, pos);
#pragma unroll
  for (int r = 0; r < IPT; ++r)
    if (base + r * 256 + threadIdx.x < n) atomicAdd(&hist[(key[r] >> shift) & (bins - 1)], 1u);   // (whole numbers: any order)
  __syncthreads();
  if (by_block) {
    for (int d = threadIdx.x; d < bins; d += 256) counts[(size_t)blockIdx.x * bins + d] = hist[d];
  } else {
    for (int d = threadIdx.x; d < bins; d += 256) counts[(size_t)d * n_blocks + blockIdx.x] = hist[d];
  }
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o);
    if ((int)(threadIdx.x & 63) >= o) v += u;
  }
  return v;
}

// Exclusive sum of one value per thread over the 256 threads; `total` gets the sum.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t *wave_sums, uint32_t &total) {
  const uint32_t inc = wave_inclusive(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) wave_sums[threadIdx.x >> 6] = inc;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += wave_sums[w];
    total += wave_sums[w];
  }
  return before + inc - v;
}

// One block per digit: counts[digit][*] becomes its exclusive scan over the blocks, totals[digit] the sum.
__global__ __launch_bounds__(256) void radix_scan_kernel(uint32_t *__restrict__ counts, int n_blocks, uint32_t *__restrict__ totals) {
  __shared__ uint32_t wave_sums[4];
  uint32_t *row = counts + (size_t)blockIdx.x * n_blocks, carry = 0;
  for (int b = 0; b < n_blocks; b += 256) {
    const int i = b + threadIdx.x;
    const uint32_t v = i < n_blocks ? row[i] : 0;
    uint32_t total;
    const uint32_t ex = block_exclusive(v, wave_sums, total);
    if (i < n_blocks) row[i] = carry + ex;
    carry += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <int PER>
__device__ __forceinline__ void sum_blocks(const uint32_t *__restrict__ counts, int bins, int n_blocks, uint32_t (&all)[4],
                                           uint32_t (&before)[4]) {
#pragma unroll 16
  for (int b = 0; b < n_blocks; ++b) {
    uint32_t c[PER];
    const uint32_t *src = counts + (size_t)b * bins;       // (bins and the digit are multiples of PER)
    if constexpr (PER == 1) c[0] = *src;
    if constexpr (PER == 2) { const uint2 v = *reinterpret_cast<const uint2 *>(src); c[0] = v.x; c[1] = v.y; }
    if constexpr (PER == 4) { const uint4 v = *reinterpret_cast<const uint4 *>(src); c[0] = v.x; c[1] = v.y; c[2] = v.z; c[3] = v.w; }
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      all[q] += c[q];
      before[q] += b < (int)blockIdx.x ? c[q] : 0;
    }
  }
}

template <int IPT>
__global__ __launch_bounds__(256) void radix_scatter_kernel(key_source s, int64_t n, int shift, int bits, int n_blocks,
                                                            const uint32_t *__restrict__ counts, const uint32_t *__restrict__ totals,
                                                            uint32_t *__restrict__ keys_out, uint32_t *__restrict__ pos_out) {
  __shared__ uint32_t seen[kWaves][1 << kMaxDigit];   // items of a digit met so far, per wave
  __shared__ uint32_t base[1 << kMaxDigit];
  __shared__ uint32_t wave_sums[4];
  const int bins = 1 << bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int d = threadIdx.x; d < bins; d += 256)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) seen[w][d] = 0;
  // a thread takes bins / 256 neighbouring digits: their entries, and those of the blocks before this one
  const int per = max(1, bins >> 8), d0 = threadIdx.x * per;
  uint32_t all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0}, sum = 0, total;
  if (d0 < bins) {
    if (totals) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < per) {
          all[q] = totals[d0 + q];
          before[q] = counts[(size_t)(d0 + q) * n_blocks + blockIdx.x];
        }
    } else if (per == 1) {
      sum_blocks<1>(counts + d0, bins, n_blocks, all, before);
    } else if (per == 2) {
      sum_blocks<2>(counts + d0, bins, n_blocks, all, before);
    } else {
      sum_blocks<4>(counts + d0, bins, n_blocks, all, before);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) sum += all[q];
  uint32_t at = block_exclusive(sum, wave_sums, total);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (q < per && d0 < bins) {
      base[d0 + q] = at + before[q];
      at += all[q];
    }
  __syncthreads();
  uint32_t key[IPT], pos[IPT], rank[IPT];
  const int64_t first = (int64_t)blockIdx.x * (256 * IPT) + wave * (64 * IPT);   // a wave's items are neighbours
  load_keys<IPT>(s, first + lane, 64, n, key, pos);
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const bool in = first + r * 64 + lane < n;
    const uint32_t d = (key[r] >> shift) & (bins - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? set : ~set;
    }
    const uint32_t below = __popcll(same & ((1ull << lane) - 1));
    const uint32_t before = in ? seen[wave][d] : 0;
    rank[r] = before + below;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");         // (a wave's LDS accesses stay in order)
    if (in && (same >> lane) == 1) seen[wave][d] = before + below + 1;   // the digit's last lane
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 256) {
    uint32_t at = base[d];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = seen[w][d];
      seen[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    if (first + r * 64 + lane >= n) continue;
    const uint32_t to = seen[wave][(key[r] >> shift) & (bins - 1)] + rank[r];
    keys_out[to] = key[r];
    pos_out[to] = pos[r];
  }
}

// ---- the same order for short lists, in one launch ---------------------------------------------------------------------
// An entry's place is the number of entries before it: those of a smaller key, and those of its own key that come earlier.
// Every workgroup places 32 entries by comparing them with all n (staged in LDS, four keys a read, 32 slices of threads):
// n^2 comparisons of two instructions each over the whole chip.  The whole gradient, 64 columns of 60000 rows: 14.1 us at
// 2048 ids, 18.9 us at 8192 against 23.4 and 28.6 us by the radix passes (launches and their latencies); 33.4 against
// 31.2 us at 12000, so longer lists go by those.
constexpr int kRankMax = 8192, kRankTokens = 32, kRankSlices = 1024 / kRankTokens;

__global__ __launch_bounds__(1024) void rank_sort_kernel(key_source s, int n, uint32_t *__restrict__ keys_out,
                                                         uint32_t *__restrict__ pos_out, uint32_t *__restrict__ n_crossing) {
  __shared__ alignas(16) uint32_t stage[kRankMax];
  __shared__ uint32_t part[kRankSlices][kRankTokens + 1];
  if (blockIdx.x == 0 && threadIdx.x == 0) *n_crossing = 0;
  const int i0 = blockIdx.x * kRankTokens, t = threadIdx.x % kRankTokens, slice = threadIdx.x / kRankTokens, i = i0 + t;
  constexpr int PER = kRankMax / 1024;
  uint32_t own[1], pos[1], k[PER], unused[PER], rank = 0, r4[4] = {0, 0, 0, 0};
  load_keys<1>(s, i, 0, n, own, pos);
  load_keys<PER>(s, threadIdx.x, 1024, n, k, unused);
#pragma unroll
  for (int e = 0; e < PER; ++e)                             // (behind the list: smaller than no key)
    stage[e * 1024 + threadIdx.x] = e * 1024 + (int)threadIdx.x < n ? k[e] : 0xffffffffu;
  __syncthreads();
  const uint32_t key = own[0];
  auto below = [&](int from, int to, uint32_t top) {
#pragma unroll 4
    for (int q = from + slice * 4; q < to; q += 4 * kRankSlices) {
      const uint4 v = *reinterpret_cast<const uint4 *>(&stage[q]);
      r4[0] += v.x < top;                                   // (four chains: each step is a compare and an add with carry)
      r4[1] += v.y < top;
      r4[2] += v.z < top;
      r4[3] += v.w < top;
    }
  };
  // an earlier entry of the same key counts, a later one does not; the workgroup's own entries are taken as later ones ...
  below(0, i0, key + 1);
  below(i0, n, key);
  if (slice < t && stage[i0 + slice] == key) ++rank;        // ... but for these
  part[slice][t] = rank + r4[0] + r4[1] + r4[2] + r4[3];
  __syncthreads();
  if (threadIdx.x >= kRankTokens || i >= n) return;
  uint32_t to = 0;
#pragma unroll
  for (int q = 0; q < kRankSlices; ++q) to += part[q][t];
  keys_out[to] = key;
  pos_out[to] = pos[0];
}

// ---- sums over the runs of equal ids ----------------------------------------------------------------------------------
// GL lanes take `chunk` consecutive entries of the sorted list for their GL * VEC columns (blockIdx.y: the column block),
// eight rows on their way at a time.  A run that lies inside the chunk is written to its row; a run that comes from the
// chunk before leaves its part in slab[chunk][0], one that starts here and goes on in slab[chunk][1], and is listed for the
// launch behind (the list's order does not matter: its entries are independent of each other).
// The blocks behind those of the chunks write the rows that no id names: zeros.  They wait on memory alone, the chunks'
// blocks mostly on the latency of their rows, so the two share the launch.  Bound by memory where the list is long: 65536
// rows of 1024 bf16 into 131072, 402 MB in 90 us (4.5 TB/s); by latency where it is short: 6144 of 128 fp32 into 63114,
// 35 MB in 10.5 us, of which the zeros alone take 7.7.
constexpr int kZeroRows = 64, kMarkMax = 16384;

// First place in keys[lo, hi) that is not below `key`.
__device__ __forceinline__ int64_t lower_bound(const uint32_t *__restrict__ keys, int64_t lo, int64_t hi, uint32_t key) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// The same by a whole wave, 64 probes a step.
__device__ __forceinline__ int64_t wave_lower_bound(const uint32_t *__restrict__ keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  const int lane = threadIdx.x & 63;
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) >> 6, at = lo + lane * step;
    const int below = __popcll(__ballot(at < hi && keys[at] < key));    // (the first ones: the keys ascend)
    if (below == 0) return lo;
    hi = min(hi, lo + below * step);
    lo = lo + (below - 1) * step + 1;
  }
  return lo;
}

template <typename T, int VEC, int GL>
__device__ __forceinline__ void zero_unnamed_rows(int64_t block, const uint32_t *__restrict__ keys, int64_t n, uint32_t n_rows, int dim,
                                                  T *__restrict__ d_table) {
  __shared__ uint8_t named[kZeroRows];
  __shared__ int64_t ends[2];
  const int64_t r0 = block * kZeroRows;
  const int rows = (int)min((int64_t)kZeroRows, (int64_t)n_rows - r0);
  if (threadIdx.x < kZeroRows) named[threadIdx.x] = 0;
  if (threadIdx.x < 128) {
    const int64_t at = wave_lower_bound(keys, n, (uint32_t)(r0 + (threadIdx.x >= 64 ? rows : 0)));
    if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  const int64_t lo = ends[0], hi = ends[1];
  if (hi - lo <= kMarkMax) {
    for (int64_t i = lo + threadIdx.x; i < hi; i += 256) named[keys[i] - r0] = 1;
  } else if ((int)threadIdx.x < rows) {                     // long runs: look for each row instead of reading them all
    const uint32_t row = (uint32_t)r0 + threadIdx.x;
    const int64_t at = lower_bound(keys, lo, hi, row);
    named[threadIdx.x] = at < hi && keys[at] == row;
  }
  __syncthreads();
  const int steps = dim / VEC, g = threadIdx.x / GL, l = threadIdx.x % GL;
  float zero[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) zero[v] = 0.f;
  for (int r = g; r < rows; r += 256 / GL) {
    if (named[r]) continue;
    T *dst = d_table + (r0 + r) * dim;
    for (int c = l; c < steps; c += GL) dg_store_unaligned<VEC>(dst + c * VEC, zero);
  }
}

template <typename T, int VEC, int GL>
__global__ __launch_bounds__(256) void embedding_runs_kernel(const T *__restrict__ d_out, int64_t stride, int dim,
                                                             const uint32_t *__restrict__ keys, const uint32_t *__restrict__ pos,
                                                             int64_t n, uint32_t n_rows, int chunk, unsigned chunk_blocks, float scale,
                                                             T *__restrict__ d_table, float *__restrict__ slab,
                                                             uint32_t *__restrict__ crossing, uint32_t *__restrict__ n_crossing) {
  if (blockIdx.x >= chunk_blocks) {
    const int64_t block = (int64_t)(blockIdx.x - chunk_blocks) * gridDim.y + blockIdx.y;
    if (block * kZeroRows < n_rows) zero_unnamed_rows<T, VEC, GL>(block, keys, n, n_rows, dim, d_table);
    return;
  }
  const int64_t c = (int64_t)blockIdx.x * (256 / GL) + threadIdx.x / GL;
  const int64_t b = c * chunk, e = min(b + chunk, n);
  if (b >= n) return;
  const int col = (blockIdx.y * GL + threadIdx.x % GL) * VEC;
  const bool live = col < dim;
  uint32_t cur = keys[b];
  bool open = b > 0 && keys[b - 1] == cur;    // the run began before this chunk
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  auto flush = [&](bool goes_on) {
    if (!live || cur >= n_rows) return;
    if (open || goes_on) {
      dg_store_unaligned<VEC>(slab + (size_t)(2 * c + (open ? 0 : 1)) * dim + col, acc);
      if (!open && col == 0 && crossing) crossing[atomicAdd(n_crossing, 1u)] = (uint32_t)c;
    } else {
      float f[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) f[v] = acc[v] * scale;
      dg_store_unaligned<VEC>(d_table + (size_t)cur * dim + col, f);
    }
  };
  constexpr int U = 8;
  for (int64_t i = b; i < e; i += U) {
    alignas(16) uint32_t k[U], p[U];          // (the lists reach to a multiple of 8 entries, whatever the ends hold)
#pragma unroll
    for (int u = 0; u < U; u += 4) {
      *reinterpret_cast<uint4 *>(k + u) = *reinterpret_cast<const uint4 *>(keys + i + u);
      *reinterpret_cast<uint4 *>(p + u) = *reinterpret_cast<const uint4 *>(pos + i + u);
    }
    if (k[0] >= n_rows) break;                // no gradient from here on
    dg_vec<T, VEC> row[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (live && i + u < e) row[u] = dg_load_raw<VEC, 2>(d_out + (int64_t)p[u] * stride + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= e) break;
      if (k[u] != cur) {
        flush(false);
        cur = k[u];
        open = false;
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
      }
      if (live) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += dg_widen(row[u].v[v]);
      }
    }
  }
  flush(e < n && keys[e] == cur);
}

// Long lists: the parts that chunks left are first added up over kFold neighbouring chunks, as if those were one.  A run that
// begins and ends among them is written to its row, one that crosses their border leaves its part in their two places of the
// next slab (and is listed).  16 lanes take 64 columns; the parts of eight chunks are on their way at a time.
// A million ids that are all the same, 64 columns: 140 us against 532 us without; 2048 chunks of 65536 ids that fall off like
// one over their rank, 1024 columns: 18 against 13 us, so shorter lists go without.
constexpr int kFold = 16, kFoldMin = 2048;
template <typename T>
__global__ __launch_bounds__(256) void embedding_fold_kernel(const uint32_t *__restrict__ keys, int64_t n, uint32_t n_rows, int dim, int chunk,
                                                             int64_t n_chunks, float scale, const float *__restrict__ slab,
                                                             T *__restrict__ d_table, float *__restrict__ next_slab,
                                                             uint32_t *__restrict__ crossing, uint32_t *__restrict__ n_crossing) {
  const int64_t f = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), c0 = f * kFold, c1 = min(c0 + kFold, n_chunks);
  if (c0 >= n_chunks) return;
  const int col = blockIdx.y * 64 + (threadIdx.x & 15) * 4, live = max(0, min(4, dim - col));
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  bool from_before = true;                                  // the run at hand began before these chunks
  auto load = [&](int64_t place, float (&v)[4]) {
    const float *src = slab + (size_t)place * dim + col;
    if (live == 4) {
      dg_load_unaligned<4>(src, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = e < live ? src[e] : 0.f;
    }
  };
  auto leave = [&](uint32_t key, bool goes_on) {
    if (from_before || goes_on) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < live) next_slab[(size_t)(2 * f + (from_before ? 0 : 1)) * dim + col + e] = acc[e];
      if (!from_before && col == 0) crossing[atomicAdd(n_crossing, 1u)] = (uint32_t)f;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < live) d_table[(size_t)key * dim + col + e] = dg_round<T>(acc[e] * scale);
    }
  };
  constexpr int U = 8;
  for (int64_t c = c0; c < c1; c += U) {
    uint32_t before[U], first[U], last[U], after[U];
    float head[U][4], tail[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t b = min(c + u, c1 - 1) * chunk, e = min(b + chunk, n);
      before[u] = b ? keys[b - 1] : n_rows;
      first[u] = keys[b];
      last[u] = keys[e - 1];
      after[u] = e < n ? keys[e] : n_rows;                  // (n_rows: the key of what takes no gradient, and leaves no part)
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = 2 * min(c + u, c1 - 1);
      if (before[u] == first[u] && first[u] < n_rows) load(at, head[u]);
      if (last[u] == after[u] && last[u] < n_rows) load(at + 1, tail[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u >= c1) break;
      const bool open = before[u] == first[u] && first[u] < n_rows, goes_on = last[u] == after[u] && last[u] < n_rows;
      const bool through = open && goes_on && first[u] == last[u];      // nothing but the run at hand in this chunk
      if (open) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += head[u][e];
        if (!through) leave(first[u], false);
      }
      if (goes_on && !through) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = tail[u][e];
        from_before = false;
      }
      if (c + u == c1 - 1 && goes_on) leave(last[u], true);
    }
  }
}

// The runs that cross from chunk to chunk (or from fold to fold), 64 columns of one at a time: 16 strands of every 16th
// part, the strands added in order.  A workgroup takes every so many of them from the list.  Bound by the latency of its
// dependent steps (list, key, end of the run, parts): 4.1 us behind 6144 ids, 13.8 us behind 65536 of 1024 columns.
constexpr int kCrossCols = 64;
template <typename T>
__global__ __launch_bounds__(256) void embedding_crossing_kernel(const uint32_t *__restrict__ keys, int64_t n, int dim, int chunk,
                                                                 float scale, const float *__restrict__ slab,
                                                                 const uint32_t *__restrict__ crossing,
                                                                 const uint32_t *__restrict__ n_crossing, T *__restrict__ d_table) {
  __shared__ float part[16][kCrossCols];
  __shared__ int64_t last_chunk;
  const int64_t blocks = (dim + kCrossCols - 1) / kCrossCols, items = (int64_t)*n_crossing * blocks;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t c = crossing[item / blocks];
    const int col = (int)(item % blocks) * kCrossCols + 4 * l;
    const uint32_t key = keys[(c + 1) * chunk];             // (it goes on there)
    __syncthreads();
    if (threadIdx.x < 64) {                                 // the last chunk that begins with the run
      int64_t last = c + 1;
      for (;;) {
        const int64_t j = last + 1 + (threadIdx.x & 63);
        const int more = __popcll(__ballot(j * chunk < n && keys[min(j * chunk, n - 1)] == key));
        last += more;
        if (more < 64) break;
      }
      if (threadIdx.x == 0) last_chunk = last;
    }
    __syncthreads();
    const int64_t last = last_chunk;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int64_t k = c + g; k <= last; k += 16) {
      const float *src = slab + (size_t)(2 * k + (k == c ? 1 : 0)) * dim + col;
      if (col + 4 <= dim) {
        float f[4];
        dg_load_unaligned<4>(src, f);
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[v] += f[v];
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (col + v < dim) acc[v] += src[v];
      }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) part[g][4 * l + v] = acc[v];
    __syncthreads();
    const int o = (int)(item % blocks) * kCrossCols + threadIdx.x;
    if (threadIdx.x < kCrossCols && o < dim) {
      float t = part[0][threadIdx.x];
      for (int q = 1; q < 16; ++q) t += part[q][threadIdx.x];
      d_table[(size_t)key * dim + o] = dg_round<T>(t * scale);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
int type_size(int dtype) { return dtype == DG_F32 ? 4 : (dtype == DG_BF16 || dtype == DG_F16) ? 2 : 0; }
constexpr int kMaxIpt = 16;
int items_per_thread(int64_t n) { return n <= 256 * 256 * 4 ? 4 : kMaxIpt; }

// Entries of a chunk: as many as leave some 4096 waves (16 a CU), 8 to 256.  Short chunks are more loads on their way at
// once, and more partial sums (65536 x 1024 bf16: 16 entries 118 us, 32: 103, 64: 114 for the runs and those that cross).
int chunk_of(int64_t n, int dim, int elem) {
  const int lanes = (dim * elem + 15) / 16;
  int c = 8;
  while (c < 256 && (n / c * lanes > 4096 * 64 || (c < 16 && n / c > 2048))) c <<= 1;
  return c;
}

struct grad_plan {
  int64_t n_blocks, n_chunks, folds;   // (folds: 0 where the chunks' parts are added up at once)
  int ipt, chunk, passes, bits;     // bits of the id's range
  bool ranked;
  size_t keys, pos, counts, totals, crossing, slab, folded, bytes;   // offsets (two key and position lists)
};

grad_plan plan_of(int64_t n_ids, int64_t n_rows, int dim, int elem) {
  grad_plan p;
  p.ipt = items_per_thread(n_ids);
  p.n_blocks = (n_ids + 256 * p.ipt - 1) / (256 * p.ipt);
  p.chunk = chunk_of(n_ids, dim, elem);
  p.n_chunks = (n_ids + p.chunk - 1) / p.chunk;
  p.bits = 1;
  while (p.bits < 32 && (n_rows >> p.bits) != 0) ++p.bits;     // keys 0 .. n_rows
  p.passes = (p.bits + kMaxDigit - 1) / kMaxDigit;
  p.ranked = n_ids <= kRankMax;
  const size_t list = ((size_t)n_ids * 4 + 255) & ~(size_t)255;   // (a multiple of 8 entries)
  size_t at = 0;
  const int lists = p.ranked ? 1 : 2;
  p.keys = at; at += lists * list;
  p.pos = at; at += lists * list;
  p.counts = at; at += p.ranked ? 0 : (((size_t)p.n_blocks << kMaxDigit) * 4 + 255) & ~(size_t)255;
  p.totals = at; at += p.ranked ? 0 : (size_t)4 << kMaxDigit;
  p.crossing = at; at += ((size_t)p.n_chunks * 4 + 4 + 255) & ~(size_t)255;    // their number, then the chunks
  p.slab = at; at += ((size_t)p.n_chunks * 2 * dim * 4 + 255) & ~(size_t)255;
  p.folds = p.n_chunks > kFoldMin ? (p.n_chunks + kFold - 1) / kFold : 0;
  p.folded = at; at += (size_t)p.folds * 2 * dim * 4;
  p.bytes = at;
  return p;
}

int lanes_for(int steps) { return steps > 32 ? 64 : steps > 16 ? 32 : 16; }

template <typename T, int VEC, int GL>
int lookup_as(const void *table, int64_t n_rows, int64_t stride, int dim, const void *ids, int ids64, int64_t n, float scale, void *out,
              hipStream_t stream) {
  constexpr int64_t kMost = (int64_t)(1 << 22) * (256 / GL);      // (2^30 threads a launch: 2^32 are its limit)
  for (int64_t first = 0; first < n; first += kMost) {
    const int64_t some = n - first < kMost ? n - first : kMost;
    hipLaunchKernelGGL((embedding_lookup_kernel<T, VEC, GL>), dim3((unsigned)((some + 256 / GL - 1) / (256 / GL))), dim3(256), 0, stream,
                       (const T *)table, n_rows, stride, dim, (const char *)ids + first * (ids64 ? 8 : 4), ids64, some, scale,
                       (T *)out + first * dim);
    DG_HIP(hipGetLastError());
  }
  return 0;
}

template <typename T, int VEC, int GL>
int grad_as(const grad_plan &p, const void *d_out, int64_t stride, const uint32_t *keys, const uint32_t *pos, int64_t n, int64_t n_rows,
            int dim, float scale, void *d_table, float *slab, float *folded, uint32_t *crossing, hipStream_t stream) {
  const unsigned chunk_blocks = (unsigned)((p.n_chunks + 256 / GL - 1) / (256 / GL));
  const int cols = (dim + GL * VEC - 1) / (GL * VEC);
  const int64_t zero_blocks = (n_rows + kZeroRows - 1) / kZeroRows;
  const dim3 grid(chunk_blocks + (unsigned)((zero_blocks + cols - 1) / cols), cols);
  hipLaunchKernelGGL((embedding_runs_kernel<T, VEC, GL>), grid, dim3(256), 0, stream, (const T *)d_out, stride, dim, keys, pos, n,
                     (uint32_t)n_rows, p.chunk, chunk_blocks, scale, (T *)d_table, slab, p.folds ? nullptr : crossing + 1, crossing);
  DG_HIP(hipGetLastError());
  if (p.n_chunks < 2) return 0;      // nothing to cross into
  const unsigned col_blocks = (unsigned)((dim + kCrossCols - 1) / kCrossCols);
  if (p.folds) {
    hipLaunchKernelGGL((embedding_fold_kernel<T>), dim3((unsigned)((p.folds + 15) / 16), col_blocks), dim3(256), 0, stream, keys, n,
                       (uint32_t)n_rows, dim, p.chunk, p.n_chunks, scale, slab, (T *)d_table, folded, crossing + 1, crossing);
    DG_HIP(hipGetLastError());
  }
  const int64_t items = (p.folds ? p.folds : p.n_chunks) * col_blocks;
  hipLaunchKernelGGL((embedding_crossing_kernel<T>), dim3((unsigned)(items < 2048 ? items : 2048)), dim3(256), 0, stream, keys, n, dim,
                     p.folds ? p.chunk * kFold : p.chunk, scale, p.folds ? folded : slab, crossing + 1, crossing, (T *)d_table);
  DG_HIP(hipGetLastError());
  return 0;
}

// The widest loads, of up to 16 bytes, that cut a row into whole ones, and the lanes a row takes.
#define DG_BY_LANES(FN, T, VEC, dim, ...)                   \
  switch (lanes_for((dim) / (VEC))) {                       \
    case 64: return FN<T, VEC, 64>(__VA_ARGS__);            \
    case 32: return FN<T, VEC, 32>(__VA_ARGS__);            \
    default: return FN<T, VEC, 16>(__VA_ARGS__);            \
  }
#define DG_BY_WIDTH(FN, T, dim, ...)                                                          \
  if ((dim) % (16 / (int)sizeof(T)) == 0) { DG_BY_LANES(FN, T, 16 / (int)sizeof(T), dim, __VA_ARGS__) } \
  if ((dim) % (8 / (int)sizeof(T)) == 0) { DG_BY_LANES(FN, T, 8 / (int)sizeof(T), dim, __VA_ARGS__) }   \
  if (sizeof(T) == 2 && (dim) % 2 == 0) { DG_BY_LANES(FN, T, 2, dim, __VA_ARGS__) }           \
  DG_BY_LANES(FN, T, 1, dim, __VA_ARGS__)
#define DG_BY_TYPE(FN, dtype, dim, ...)                     \
  switch (dtype) {                                          \
    case DG_F32: DG_BY_WIDTH(FN, float, dim, __VA_ARGS__)   \
    case DG_BF16: DG_BY_WIDTH(FN, dg_bf16, dim, __VA_ARGS__) \
    default: DG_BY_WIDTH(FN, dg_f16, dim, __VA_ARGS__)      \
  }

int check_sizes(const char *what, int64_t n_ids, int64_t n_rows, int dim, int dtype) {
  if (!type_size(dtype)) return dg_fail(DG_ERR_ARG, "%s: unknown element type %d", what, dtype);
  if (n_ids < 0 || n_rows <= 0 || dim <= 0) return dg_fail(DG_ERR_ARG, "%s: bad sizes", what);
  if (n_ids > 0x7fffffff || n_rows > 0x7ffffffe) return dg_fail(DG_ERR_SIZE, "%s: at most 2^31 - 1 ids and 2^31 - 2 rows", what);
  if (dim > (1 << 20)) return dg_fail(DG_ERR_DIM, "%s: rows of more than 2^20 elements", what);
  return 0;
}

}  // namespace

extern "C" int dg_embedding_lookup(const void *table, int64_t n_rows, int64_t row_stride, int32_t dim, int32_t dtype, const void *ids,
                                   int32_t ids_are_64, int64_t n_ids, float scale, void *out, void *stream) {
  if (const int rc = check_sizes("dg_embedding_lookup", n_ids, n_rows, dim, dtype)) return rc;
  if (n_ids == 0) return 0;
  if (!table || !ids || !out) return dg_fail(DG_ERR_ARG, "dg_embedding_lookup: NULL argument");
  if (row_stride < 0) return dg_fail(DG_ERR_ARG, "dg_embedding_lookup: negative row stride");
  DG_BY_TYPE(lookup_as, dtype, dim, table, n_rows, row_stride, dim, ids, ids_are_64, n_ids, scale, out, (hipStream_t)stream)
}

extern "C" size_t dg_embedding_grad_workspace(int64_t n_ids, int64_t n_rows, int32_t dim) {
  if (n_ids < 0 || n_rows <= 0 || dim <= 0) return 0;
  return plan_of(n_ids, n_rows, dim, 2).bytes;      // (of 16-bit rows: the shorter chunks, the larger workspace)
}

extern "C" int dg_embedding_grad(const void *d_out, int64_t row_stride, const void *ids, int32_t ids_are_64, int64_t n_ids, int64_t n_rows,
                                 int32_t dim, int32_t dtype, float scale, int64_t padding_idx, void *d_table, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  if (const int rc = check_sizes("dg_embedding_grad", n_ids, n_rows, dim, dtype)) return rc;
  if (!d_table || (n_ids && (!d_out || !ids || !workspace))) return dg_fail(DG_ERR_ARG, "dg_embedding_grad: NULL argument");
  if (row_stride < 0) return dg_fail(DG_ERR_ARG, "dg_embedding_grad: negative row stride");
  if (n_rows > (1 << 29)) return dg_fail(DG_ERR_SIZE, "dg_embedding_grad: at most 2^29 rows");      // (4 threads a row, 2^32 in all)
  const grad_plan p = plan_of(n_ids, n_rows, dim, type_size(dtype));
  if (n_ids && (workspace_bytes < p.bytes || ((uintptr_t)workspace & 15)))
    return dg_fail(DG_ERR_SIZE, "dg_embedding_grad: a 16-byte aligned workspace of %zu bytes is needed, got %zu", p.bytes, workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  char *ws = (char *)workspace;
  const size_t list = p.ranked ? 0 : (p.pos - p.keys) / 2;
  uint32_t *keys[2] = {(uint32_t *)(ws + p.keys), (uint32_t *)(ws + p.keys + list)};
  uint32_t *pos[2] = {(uint32_t *)(ws + p.pos), (uint32_t *)(ws + p.pos + list)};
  uint32_t *counts = (uint32_t *)(ws + p.counts), *totals = (uint32_t *)(ws + p.totals);
  uint32_t *crossing = (uint32_t *)(ws + p.crossing);
  int at = 0;
  if (n_ids && p.ranked) {
    const key_source s = {ids, ids_are_64, padding_idx, (uint32_t)n_rows, nullptr, nullptr};
    hipLaunchKernelGGL(rank_sort_kernel, dim3((unsigned)((n_ids + kRankTokens - 1) / kRankTokens)), dim3(1024), 0, st, s, (int)n_ids, keys[0],
                       pos[0], crossing);
    DG_HIP(hipGetLastError());
  } else if (n_ids) {
    key_source s = {ids, ids_are_64, padding_idx, (uint32_t)n_rows, nullptr, nullptr};
    for (int pass = 0, shift = 0; pass < p.passes; ++pass) {
      const int bits = (p.bits - shift + (p.passes - pass) - 1) / (p.passes - pass);
      const dim3 grid((unsigned)p.n_blocks);
      const int nb = (int)p.n_blocks, by_block = nb <= kSelfScan;
      const uint32_t *sums = by_block ? nullptr : totals;
      if (p.ipt == 4) hipLaunchKernelGGL((radix_count_kernel<4>), grid, dim3(256), 0, st, s, n_ids, shift, bits, nb, by_block, counts, crossing);
      else hipLaunchKernelGGL((radix_count_kernel<kMaxIpt>), grid, dim3(256), 0, st, s, n_ids, shift, bits, nb, by_block, counts, crossing);
      if (!by_block) hipLaunchKernelGGL(radix_scan_kernel, dim3(1u << bits), dim3(256), 0, st, counts, nb, totals);
      if (p.ipt == 4) hipLaunchKernelGGL((radix_scatter_kernel<4>), grid, dim3(256), 0, st, s, n_ids, shift, bits, nb, counts, sums, keys[at], pos[at]);
      else hipLaunchKernelGGL((radix_scatter_kernel<kMaxIpt>), grid, dim3(256), 0, st, s, n_ids, shift, bits, nb, counts, sums, keys[at], pos[at]);
      DG_HIP(hipGetLastError());
      s.keys = keys[at];
      s.pos = pos[at];
      at ^= 1;
      shift += bits;
    }
    at ^= 1;
  }
  DG_BY_TYPE(grad_as, dtype, dim, p, d_out, row_stride, keys[at], pos[at], n_ids, n_rows, dim, scale, d_table,
             (float *)(ws + p.slab), (float *)(ws + p.folded), crossing, st)
}
