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
// GL lanes per row, VEC elements per lane and step.  An id outside the table gathers nothing: its row is NaN.
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
      dg_load<VEC>(src + c, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = __builtin_nanf("");
    }
    dg_store<VEC>(dst + c, f);
  }
}

// ---- stable radix sort of (id, position) ------------------------------------------------------------------------------
// Passes over at most kMaxDigit bits, low digit first; ids that take no gradient (outside the table, the padding id) get
// the key n_rows, behind all others.  A pass: digit counts per block, per-digit scans over the blocks, stable scatter.
constexpr int kMaxDigit = 10, kWaves = 4;

struct key_source {
  const void *ids;      // first pass: the caller's ids
  int ids64;
  int64_t padding;
  uint32_t n_rows;
  const uint32_t *keys, *pos;   // later passes
};

__device__ __forceinline__ void load_key(const key_source &s, int64_t i, uint32_t &key, uint32_t &pos) {
  if (s.keys) {
    key = s.keys[i];
    pos = s.pos[i];
    return;
  }
  const int64_t id = s.ids64 ? ((const int64_t *)s.ids)[i] : (int64_t)((const int32_t *)s.ids)[i];
  key = ((uint64_t)id >= (uint64_t)s.n_rows || id == s.padding) ? s.n_rows : (uint32_t)id;
  pos = (uint32_t)i;
}

// counts[digit][block]
template <int IPT>
__global__ __launch_bounds__(256) void radix_count_kernel(key_source s, int64_t n, int shift, int bits, int n_blocks,
                                                          uint32_t *__restrict__ counts) {
  __shared__ uint32_t hist[1 << kMaxDigit];
  const int bins = 1 << bits;
  for (int d = threadIdx.x; d < bins; d += 256) hist[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (256 * IPT);
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const int64_t i = base + r * 256 + threadIdx.x;
    if (i < n) {
      uint32_t key, pos;
      load_key(s, i, key, pos);
      atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);   // (whole numbers: any order gives the same counts)
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 256) counts[(size_t)d * n_blocks + blockIdx.x] = hist[d];
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
  uint32_t carry = 0;
  for (int d0 = 0; d0 < bins; d0 += 256) {
    const int d = d0 + threadIdx.x;
    uint32_t total;
    const uint32_t ex = block_exclusive(d < bins ? totals[d] : 0, wave_sums, total);
    if (d < bins) base[d] = carry + ex + counts[(size_t)d * n_blocks + blockIdx.x];
    carry += total;
  }
  __syncthreads();
  uint32_t key[IPT], pos[IPT], rank[IPT];
  const int64_t first = (int64_t)blockIdx.x * (256 * IPT) + wave * (64 * IPT);   // a wave's items are neighbours
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const int64_t i = first + r * 64 + lane;
    key[r] = 0; pos[r] = 0;
    if (i < n) load_key(s, i, key[r], pos[r]);
  }
  volatile uint32_t *mine = seen[wave];
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
    const uint32_t before = in ? mine[d] : 0;
    rank[r] = before + below;
    __builtin_amdgcn_wave_barrier();
    if (in && (same >> lane) == 1) mine[d] = before + below + 1;   // the digit's last lane
    __builtin_amdgcn_wave_barrier();
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

// ---- sums over the runs of equal ids ----------------------------------------------------------------------------------
// GL lanes take `chunk` consecutive entries of the sorted list for their GL * VEC columns (blockIdx.y: the column block).
// A run that lies inside the chunk is written to its row; a run that comes from the chunk before leaves its part in
// slab[chunk][0], one that starts here and goes on in slab[chunk][1].
template <typename T, int VEC, int GL>
__global__ __launch_bounds__(256) void embedding_runs_kernel(const T *__restrict__ d_out, int64_t stride, int dim,
                                                             const uint32_t *__restrict__ keys, const uint32_t *__restrict__ pos,
                                                             int64_t n, uint32_t n_rows, int chunk, float scale,
                                                             T *__restrict__ d_table, float *__restrict__ slab) {
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
      dg_store<VEC>(slab + (size_t)(2 * c + (open ? 0 : 1)) * dim + col, acc);
    } else {
      float f[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) f[v] = acc[v] * scale;
      dg_store<VEC>(d_table + (size_t)cur * dim + col, f);
    }
  };
  constexpr int U = 4;
  for (int64_t i = b; i < e; i += U) {
    uint32_t k[U];
    float row[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = min(i + u, e - 1);
      k[u] = keys[j];
      if (live) dg_load<VEC>(d_out + (int64_t)pos[j] * stride + col, row[u]);
    }
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
        for (int v = 0; v < VEC; ++v) acc[v] += row[u][v];
      }
    }
  }
  flush(e < n && keys[e] == cur);
}

// First place in keys[0, n) that is not below `key`.
__device__ __forceinline__ int64_t lower_bound(const uint32_t *__restrict__ keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Blocks [0, n_chunks): the run that starts in chunk c and goes on behind it -- its parts, chunk after chunk (256 / GL
// strands of every so many chunks, added strand by strand).  The blocks behind them: rows that no id names become zero.
constexpr int kZeroRows = 64;
template <typename T, int VEC, int GL>
__global__ __launch_bounds__(256) void embedding_finish_kernel(const uint32_t *__restrict__ keys, int64_t n, uint32_t n_rows, int dim,
                                                               int chunk, int64_t n_chunks, float scale,
                                                               const float *__restrict__ slab, T *__restrict__ d_table) {
  __shared__ float part[256 / GL][GL * VEC];
  __shared__ uint8_t named[kZeroRows];
  if ((int64_t)blockIdx.x >= n_chunks) {
    const int64_t r0 = ((int64_t)blockIdx.x - n_chunks) * kZeroRows;
    if (threadIdx.x < kZeroRows) {
      const int64_t row = r0 + threadIdx.x;
      bool is = true;
      if (row < n_rows) {
        const int64_t at = lower_bound(keys, n, (uint32_t)row);
        is = at < n && keys[at] == (uint32_t)row;
      }
      named[threadIdx.x] = is;
    }
    __syncthreads();
    const int steps = (dim + VEC - 1) / VEC;
    float zero[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) zero[v] = 0.f;
    for (int64_t q = threadIdx.x; q < (int64_t)kZeroRows * steps; q += 256) {
      const int r = (int)(q / steps), c = (int)(q % steps) * VEC;
      if (!named[r]) dg_store<VEC>(d_table + (r0 + r) * dim + c, zero);
    }
    return;
  }
  const int64_t c = blockIdx.x, b = c * chunk, e = min(b + chunk, n);
  const uint32_t key = keys[e - 1];
  if (key >= n_rows || e >= n || keys[e] != key) return;             // nothing goes on behind this chunk
  if (keys[b] == key && b > 0 && keys[b - 1] == key) return;         // ... or it began before it
  const int64_t end = lower_bound(keys, n, key + 1), last = (end - 1) / chunk;
  const int g = threadIdx.x / GL, l = threadIdx.x % GL;
  for (int c0 = 0; c0 < dim; c0 += GL * VEC) {
    const int col = c0 + l * VEC;
    float acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
    if (col < dim) {
      for (int64_t k = c + g; k <= last; k += 256 / GL) {
        float f[VEC];
        dg_load<VEC>(slab + (size_t)(2 * k + (k == c ? 1 : 0)) * dim + col, f);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += f[v];
      }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) part[g][l * VEC + v] = acc[v];
    __syncthreads();
    if (g == 0 && col < dim) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float t = part[0][l * VEC + v];
        for (int k = 1; k < 256 / GL; ++k) t += part[k][l * VEC + v];
        acc[v] = t * scale;
      }
      dg_store<VEC>(d_table + (size_t)key * dim + col, acc);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
constexpr int kMaxIpt = 16;
int items_per_thread(int64_t n) { return n <= 256 * 256 * 4 ? 4 : kMaxIpt; }

// Entries of a chunk: short ones while the list is short (every CU gets some), longer ones as it grows.
int chunk_of(int64_t n, int dim) {
  int c = 8;
  while (c < 256 && n / c > 4096) c <<= 1;
  return c;
}

struct grad_plan {
  int64_t n_blocks, n_chunks;
  int ipt, chunk, passes, bits;     // bits of the id's range
  size_t keys, pos, counts, totals, slab, bytes;   // offsets (two key and position lists)
};

grad_plan plan_of(int64_t n_ids, int64_t n_rows, int dim) {
  grad_plan p;
  p.ipt = items_per_thread(n_ids);
  p.n_blocks = (n_ids + 256 * p.ipt - 1) / (256 * p.ipt);
  p.chunk = chunk_of(n_ids, dim);
  p.n_chunks = (n_ids + p.chunk - 1) / p.chunk;
  p.bits = 1;
  while (p.bits < 32 && (n_rows >> p.bits) != 0) ++p.bits;     // keys 0 .. n_rows
  p.passes = (p.bits + kMaxDigit - 1) / kMaxDigit;
  const size_t list = ((size_t)n_ids * 4 + 255) & ~(size_t)255;
  size_t at = 0;
  p.keys = at; at += 2 * list;
  p.pos = at; at += 2 * list;
  p.counts = at; at += (((size_t)p.n_blocks << kMaxDigit) * 4 + 255) & ~(size_t)255;
  p.totals = at; at += (size_t)4 << kMaxDigit;
  p.slab = at; at += (size_t)p.n_chunks * 2 * dim * 4;
  p.bytes = at;
  return p;
}

bool aligned(const void *p, int64_t stride, int dim, int elem) {
  return ((uintptr_t)p | (uintptr_t)(stride * elem) | (uintptr_t)((int64_t)dim * elem)) % 16 == 0;
}

int lanes_for(int steps) { return steps > 32 ? 64 : steps > 16 ? 32 : 16; }

template <typename T, int VEC, int GL>
int lookup_as(const void *table, int64_t n_rows, int64_t stride, int dim, const void *ids, int ids64, int64_t n, float scale, void *out,
              hipStream_t stream) {
  const int64_t blocks = (n + 256 / GL - 1) / (256 / GL);
  if (blocks > 0x7fffffff) return dg_fail(DG_ERR_SIZE, "dg_embedding_lookup: too many ids");
  hipLaunchKernelGGL((embedding_lookup_kernel<T, VEC, GL>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T *)table, n_rows, stride,
                     dim, ids, ids64, n, scale, (T *)out);
  DG_HIP(hipGetLastError());
  return 0;
}

template <typename T, int VEC, int GL>
int grad_as(const grad_plan &p, const void *d_out, int64_t stride, const uint32_t *keys, const uint32_t *pos, int64_t n, int64_t n_rows,
            int dim, float scale, void *d_table, float *slab, hipStream_t stream) {
  if (n > 0) {
    const int64_t blocks = (p.n_chunks + 256 / GL - 1) / (256 / GL);
    const int cols = (dim + GL * VEC - 1) / (GL * VEC);
    hipLaunchKernelGGL((embedding_runs_kernel<T, VEC, GL>), dim3((unsigned)blocks, cols), dim3(256), 0, stream, (const T *)d_out, stride,
                       dim, keys, pos, n, (uint32_t)n_rows, p.chunk, scale, (T *)d_table, slab);
    DG_HIP(hipGetLastError());
  }
  const int64_t blocks = p.n_chunks + (n_rows + kZeroRows - 1) / kZeroRows;
  hipLaunchKernelGGL((embedding_finish_kernel<T, VEC, GL>), dim3((unsigned)blocks), dim3(256), 0, stream, keys, n, (uint32_t)n_rows, dim,
                     p.chunk, p.n_chunks, scale, slab, (T *)d_table);
  DG_HIP(hipGetLastError());
  return 0;
}

// The widest load that rows of this width and alignment allow (16 bytes, or one element), and the lanes a row takes.
#define DG_BY_LANES(FN, T, VEC, steps, ...)                 \
  switch (lanes_for(steps)) {                               \
    case 64: return FN<T, VEC, 64>(__VA_ARGS__);            \
    case 32: return FN<T, VEC, 32>(__VA_ARGS__);            \
    default: return FN<T, VEC, 16>(__VA_ARGS__);            \
  }
#define DG_BY_TYPE(FN, dtype, wide, dim, ...)                                              \
  switch (dtype) {                                                                         \
    case DG_F32:                                                                           \
      if (wide) { DG_BY_LANES(FN, float, 4, ((dim) + 3) / 4, __VA_ARGS__) }                \
      DG_BY_LANES(FN, float, 1, dim, __VA_ARGS__)                                          \
    case DG_BF16:                                                                          \
      if (wide) { DG_BY_LANES(FN, dg_bf16, 8, ((dim) + 7) / 8, __VA_ARGS__) }              \
      DG_BY_LANES(FN, dg_bf16, 1, dim, __VA_ARGS__)                                        \
    default:                                                                               \
      if (wide) { DG_BY_LANES(FN, dg_f16, 8, ((dim) + 7) / 8, __VA_ARGS__) }               \
      DG_BY_LANES(FN, dg_f16, 1, dim, __VA_ARGS__)                                         \
  }

int type_size(int dtype) { return dtype == DG_F32 ? 4 : (dtype == DG_BF16 || dtype == DG_F16) ? 2 : 0; }

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
  const int z = type_size(dtype);
  const bool wide = aligned(table, row_stride, dim, z) && aligned(out, dim, dim, z);
  DG_BY_TYPE(lookup_as, dtype, wide, dim, table, n_rows, row_stride, dim, ids, ids_are_64, n_ids, scale, out, (hipStream_t)stream)
}

extern "C" size_t dg_embedding_grad_workspace(int64_t n_ids, int64_t n_rows, int32_t dim) {
  if (n_ids < 0 || n_rows <= 0 || dim <= 0) return 0;
  return plan_of(n_ids, n_rows, dim).bytes;
}

extern "C" int dg_embedding_grad(const void *d_out, int64_t row_stride, const void *ids, int32_t ids_are_64, int64_t n_ids, int64_t n_rows,
                                 int32_t dim, int32_t dtype, float scale, int64_t padding_idx, void *d_table, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  if (const int rc = check_sizes("dg_embedding_grad", n_ids, n_rows, dim, dtype)) return rc;
  if (!d_table || (n_ids && (!d_out || !ids || !workspace))) return dg_fail(DG_ERR_ARG, "dg_embedding_grad: NULL argument");
  if (row_stride < 0) return dg_fail(DG_ERR_ARG, "dg_embedding_grad: negative row stride");
  const grad_plan p = plan_of(n_ids, n_rows, dim);
  if (n_ids && (workspace_bytes < p.bytes || ((uintptr_t)workspace & 15)))
    return dg_fail(DG_ERR_SIZE, "dg_embedding_grad: a 16-byte aligned workspace of %zu bytes is needed, got %zu", p.bytes, workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  char *ws = (char *)workspace;
  const size_t list = (p.pos - p.keys) / 2;
  uint32_t *keys[2] = {(uint32_t *)(ws + p.keys), (uint32_t *)(ws + p.keys + list)};
  uint32_t *pos[2] = {(uint32_t *)(ws + p.pos), (uint32_t *)(ws + p.pos + list)};
  uint32_t *counts = (uint32_t *)(ws + p.counts), *totals = (uint32_t *)(ws + p.totals);
  int at = 0;
  if (n_ids) {
    key_source s = {ids, ids_are_64, padding_idx, (uint32_t)n_rows, nullptr, nullptr};
    for (int pass = 0, shift = 0; pass < p.passes; ++pass) {
      const int bits = (p.bits - shift + (p.passes - pass) - 1) / (p.passes - pass);
      const dim3 grid((unsigned)p.n_blocks);
      if (p.ipt == 4)
        hipLaunchKernelGGL((radix_count_kernel<4>), grid, dim3(256), 0, st, s, n_ids, shift, bits, (int)p.n_blocks, counts);
      else
        hipLaunchKernelGGL((radix_count_kernel<kMaxIpt>), grid, dim3(256), 0, st, s, n_ids, shift, bits, (int)p.n_blocks, counts);
      hipLaunchKernelGGL(radix_scan_kernel, dim3(1u << bits), dim3(256), 0, st, counts, (int)p.n_blocks, totals);
      if (p.ipt == 4)
        hipLaunchKernelGGL((radix_scatter_kernel<4>), grid, dim3(256), 0, st, s, n_ids, shift, bits, (int)p.n_blocks, counts, totals, keys[at], pos[at]);
      else
        hipLaunchKernelGGL((radix_scatter_kernel<kMaxIpt>), grid, dim3(256), 0, st, s, n_ids, shift, bits, (int)p.n_blocks, counts, totals, keys[at], pos[at]);
      DG_HIP(hipGetLastError());
      s.keys = keys[at];
      s.pos = pos[at];
      at ^= 1;
      shift += bits;
    }
    at ^= 1;
  }
  const int z = type_size(dtype);
  const bool wide = (!n_ids || aligned(d_out, row_stride, dim, z)) && aligned(d_table, dim, dim, z);
  DG_BY_TYPE(grad_as, dtype, wide, dim, p, d_out, row_stride, keys[at], pos[at], n_ids, n_rows, dim, scale, d_table,
             (float *)(ws + p.slab), st)
}
