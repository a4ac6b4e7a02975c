// Penalties, biases and masks on a table of scores [rows][items] for gfx950: what lies between t.mm(usr, itm^T) and
// t.topk in DiffGraph-Rec/main.py:157-158 (there: the training items' mask), and what a service puts there.
//
//   had      = how often item v occurs in the row's history (a CSR row of item ids in any order, repeats counted)
//   s        = had ? (s > 0 ? s / repetition : s * repetition) - (frequency * had + presence) : s
//   s        = s + bias[v]
//   out      = masked ? fill : s          masked: the row's mask has no bit for v, or `exclude` and had
//
// One pass: a workgroup takes one row's tile of items, counts the history's entries that fall into it in LDS (whole
// numbers: any order of the atomics gives the same counts) and streams the tile through registers, in fp32, rounded once.
// Bound by the table's read and write; the counts cost an LDS word per item, the history a read per tile from the L2.
// 4096 x 65537 bf16 with 300 entries of history a row: 1.08 GB in 250 us (4.3 TB/s, a copy's rate is 4.7; traced: 266); 1024 x 31232 fp32:
// 256 MB in 44 us; one row of 31232: 4.8 us, a launch and three dependent loads.  Several rows or tiles a workgroup (fewer,
// longer ones) were measured and no faster.
#include "dg_internal.h"
#include "dg_types.h"

namespace {

constexpr int kTile = 4096;

struct score_args {
  const void *scores;
  void *out;
  int64_t stride, out_stride, first_row;
  int items;
  const int32_t *rowptr, *col;
  const int64_t *hist_rows;
  int64_t n_hist, n_col;
  const float *repetition, *frequency, *presence;
  float repetition_all, frequency_all, presence_all;
  const float *bias;
  int64_t bias_stride;
  const uint8_t *allowed;
  const int32_t *allowed_rows;
  int64_t allowed_stride;   // bytes between two masks
  int32_t n_masks;
  int32_t exclude;
  float fill;
};

template <typename T, int VEC>
__global__ __launch_bounds__(256) void adjust_scores_kernel(score_args a) {
  __shared__ alignas(16) uint32_t had[kTile];
  const int64_t row = a.first_row + blockIdx.y;
  const int c0 = blockIdx.x * kTile, width = min(kTile, a.items - c0);
  int64_t begin = 0, end = 0;
  if (a.rowptr) {
    const int64_t h = a.hist_rows ? a.hist_rows[row] : row;
    if ((uint64_t)h < (uint64_t)a.n_hist) {                 // (no such history: empty)
      begin = max((int64_t)a.rowptr[h], (int64_t)0);
      end = min((int64_t)a.rowptr[h + 1], a.n_col);
    }
  }
  const bool any = begin < end;
  // the tile's scores are asked for first: they arrive while the history is counted
  const T *src = (const T *)a.scores + row * a.stride + c0;
  T *dst = (T *)a.out + row * a.out_stride + c0;
  constexpr int N = kTile / (256 * VEC);
  dg_vec<T, VEC> held[N];
#pragma unroll
  for (int v = 0; v < N; ++v) {
    const int c = (v * 256 + threadIdx.x) * VEC;
    if (c + VEC <= width) held[v] = dg_load_raw<VEC, 2>(src + c);
  }
  if (any) {
    for (int i = 4 * threadIdx.x; i < kTile; i += 1024) *reinterpret_cast<uint4 *>(&had[i]) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    constexpr int U = 8;                                    // entries on their way at a time
    for (int64_t i = begin + threadIdx.x; i < end; i += 256 * U) {
      uint32_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = (uint32_t)a.col[min(i + 256 * u, end - 1)] - (uint32_t)c0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + 256 * u < end && c[u] < (uint32_t)width) atomicAdd(&had[c[u]], 1u);   // (entries outside [0, items) are in no tile)
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float fre = a.frequency ? a.frequency[row] : a.frequency_all;
  const float pre = a.presence ? a.presence[row] : a.presence_all;
  const uint8_t *mask = nullptr;
  if (a.allowed) {
    const int64_t m = a.allowed_rows ? a.allowed_rows[row] : a.n_masks == 1 ? 0 : row;
    if ((uint64_t)m < (uint64_t)a.n_masks) mask = a.allowed + m * a.allowed_stride;
  }
  const float *bias = a.bias ? a.bias + row * a.bias_stride : nullptr;
#pragma unroll
  for (int v = 0; v < N; ++v) {
    const int c = (v * 256 + threadIdx.x) * VEC;
    if (c >= width) break;
    const bool whole = c + VEC <= width;
    float s[VEC], more[VEC] = {};
    if (whole) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] = dg_widen(held[v].v[e]);
      if (bias) dg_load_unaligned<VEC>(bias + c0 + c, more);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[e] = c + e < width ? dg_widen(src[c + e]) : 0.f;
        if (bias && c + e < width) more[e] = bias[c0 + c + e];
      }
    }
    const uint32_t bits = mask ? mask[(c0 + c) >> 3] >> ((c0 + c) & 7) : ~0u;     // (VEC divides 8: one byte holds them)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t n = any ? had[c + e] : 0;
      if (n) s[e] = (s[e] > 0.f ? s[e] / rep : s[e] * rep) - (fre * (float)n + pre);
      if (bias) s[e] += more[e];
      if (!((bits >> e) & 1) || (a.exclude && n)) s[e] = a.fill;
    }
    if (whole) {
      dg_store_unaligned<VEC>(dst + c, s);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e < width) dst[c + e] = dg_round<T>(s[e]);
    }
  }
}

}  // namespace

extern "C" int dg_adjust_scores(const dg_score_task *t, void *stream) {
  if (!t) return dg_fail(DG_ERR_ARG, "dg_adjust_scores: NULL task");
  if (t->dtype != DG_F32 && t->dtype != DG_BF16 && t->dtype != DG_F16)
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: unknown element type %d", t->dtype);
  if (t->n_rows < 0 || t->n_items < 0) return dg_fail(DG_ERR_ARG, "dg_adjust_scores: bad sizes");
  if (t->n_rows == 0 || t->n_items == 0) return 0;
  if (!t->scores || !t->out) return dg_fail(DG_ERR_ARG, "dg_adjust_scores: NULL argument");
  if (t->n_rows > 1 && (t->row_stride < 0 || t->out_stride < t->n_items))
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: rows of the output overlap, or a negative row stride");
  if (t->n_rows > 1 && t->scores == t->out && t->row_stride != t->out_stride)
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: the output overlaps the scores with another row stride");
  if ((t->hist_rowptr != nullptr) != (t->hist_col != nullptr) || (!t->hist_rowptr && t->hist_rows))
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: a history needs row offsets and item ids");
  if (t->hist_rowptr && (t->n_hist < 0 || t->n_hist_items < 0 || (!t->hist_rows && t->n_hist < t->n_rows)))
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: %lld histories for %d rows", (long long)t->n_hist, t->n_rows);
  if (!t->repetition && !(t->repetition_all > 0.f)) return dg_fail(DG_ERR_ARG, "dg_adjust_scores: the repetition penalty must be positive");
  const int64_t words = ((int64_t)t->n_items + 31) / 32;
  if (t->allowed && (t->n_masks < 1 || t->mask_words < words))
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: a mask has at least %lld words, got %lld", (long long)words, (long long)t->mask_words);
  if (t->allowed && !t->allowed_rows && t->n_masks != 1 && t->n_masks < t->n_rows)
    return dg_fail(DG_ERR_ARG, "dg_adjust_scores: %d masks for %d rows", t->n_masks, t->n_rows);
  if (t->bias && t->bias_stride < 0) return dg_fail(DG_ERR_ARG, "dg_adjust_scores: negative bias stride");
  score_args a = {t->scores, t->out, t->row_stride, t->out_stride, 0, t->n_items, t->hist_rowptr, t->hist_col, t->hist_rows, t->n_hist,
                  t->n_hist_items, t->repetition, t->frequency, t->presence, t->repetition_all, t->frequency_all, t->presence_all, t->bias,
                  t->bias_stride, (const uint8_t *)t->allowed, t->allowed_rows, t->mask_words * 4, t->n_masks, t->exclude, t->fill};
  const int tiles = (int)(((int64_t)t->n_items + kTile - 1) / kTile);
  for (int64_t r0 = 0; r0 < t->n_rows; r0 += 65535) {    // (the grid's second axis holds that many)
    const dim3 grid(tiles, (unsigned)(t->n_rows - r0 < 65535 ? t->n_rows - r0 : 65535));
    score_args b = a;
    b.first_row = r0;
    if (t->dtype == DG_F32) hipLaunchKernelGGL((adjust_scores_kernel<float, 4>), grid, dim3(256), 0, (hipStream_t)stream, b);
    else if (t->dtype == DG_BF16) hipLaunchKernelGGL((adjust_scores_kernel<dg_bf16, 8>), grid, dim3(256), 0, (hipStream_t)stream, b);
    else hipLaunchKernelGGL((adjust_scores_kernel<dg_f16, 8>), grid, dim3(256), 0, (hipStream_t)stream, b);
    DG_HIP(hipGetLastError());
  }
  return 0;
}
