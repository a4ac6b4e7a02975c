// Activation checkpoints in 8 bits and the backward pass of a dense layer out of them, for gfx950.
//
// Kept of x [n][k]: one byte per element and one scale per group of 32 columns of a row, the smallest power of two with
// (largest of the group) <= 127 scale (int8) or 448 scale (e4m3), so that no code saturates and the codes' values,
//   x^ = code * scale,   code = x / scale rounded to the nearest code (ties to even),
// are exact in bf16: at most seven (int8) or four (e4m3) significant bits.  A group that holds an infinity or a NaN stands
// for NaN as a whole.
// Four rows lie together, byte by byte: code (r, c) at (r / 4) 4 pitch + 4 c + r mod 4, and behind all codes the scale of
// (r, g) at (r / 4) 4 groups + 4 g + r mod 4.  A thread of the product, which needs four rows of a few columns, then has
// them in one load, a column's four codes in one word, and the rows' scales in another.
//
// The layer's backward (nn.Linear with tanh behind it: DiffGraph-Rec/Model.py:228-233) out of the codes of its input x
// and, with tanh, of its output y:
//   d_z = d_y (1 - y^ y^)      d_w = d_z^T . x^      d_b = column sums of d_z
// The product runs on the bf16 matrix instruction: x^ is exact there, and d_z (fp32) is cut into bf16 numbers that add up
// to it bit by bit -- three where d_z has 24 bits (fp32, and every type under tanh), two for fp16 as it came (11 bits), one
// for bf16 as it came -- with sums in fp32.  Rows are cut into strips whose partial results a second launch adds in strip
// order: the same bits on every run.
#include "dg_internal.h"
#include "dg_types.h"

namespace {

constexpr int kGroup = 32, kLowest = -110;      // columns per scale; smallest exponent (code values stay normal in bf16)
constexpr uint32_t kNoNumber = 255;             // scale byte of a group that stands for NaN

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- codes ------------------------------------------------------------------------------------------------------
// Scale byte (exponent + 127) of a group whose largest magnitude has the bits `top`.
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return kNoNumber;
  const int e = (int)(top >> 23) - 127;                                  // top = (1 + m / 2^23) 2^e
  const uint32_t m = top & 0x7fffffu;
  const int s = FMT == DG_E4M3 ? e - 8 + (m > 0x600000u)                 // 448 = 1.75 * 2^8
                               : e - 6 + (m > 0x7e0000u);                // 127 = 1.984375 * 2^6
  return (uint32_t)(max(s, kLowest) + 127);
}

// Four rows' codes of a column.
template <int FMT>
__device__ __forceinline__ uint32_t encode_rows(float q0, float q1, float q2, float q3) {
  if constexpr (FMT == DG_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q0, q1, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q2, q3, w, true);
  } else {
    return ((uint32_t)(int)rintf(q0) & 255u) | ((uint32_t)(int)rintf(q1) & 255u) << 8 | ((uint32_t)(int)rintf(q2) & 255u) << 16 |
           (uint32_t)(int)rintf(q3) << 24;
  }
}

// Four rows' scales: a scale byte is the exponent field of its fp32 value (255: infinity, times code 0 = NaN).
__device__ __forceinline__ void scales_of(uint32_t w, float (&s)[4]) {
  s[0] = __uint_as_float((w << 23) & 0x7f800000u);
  s[1] = __uint_as_float((w << 15) & 0x7f800000u);
  s[2] = __uint_as_float((w << 7) & 0x7f800000u);
  s[3] = __uint_as_float((w >> 1) & 0x7f800000u);
}

template <int FMT>
__device__ __forceinline__ void decode_rows(uint32_t w, const float (&s)[4], float (&f)[4]) {
  if constexpr (FMT == DG_E4M3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = a[0] * s[0]; f[1] = a[1] * s[1]; f[2] = b[0] * s[2]; f[3] = b[1] * s[3];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = (float)(int8_t)(w >> (8 * q)) * s[q];
  }
}

// A thread takes four rows of C columns (16 bytes of each), 32 / C neighbouring lanes a group; a quad of rows takes `lanes`
// = 32 / C ceil(k / 32) of them.  One read of x, 4 C bytes written a thread: bound by memory (1e6 rows of 128 fp32: 5.7 TB/s).
template <typename T, int FMT, int C>
__global__ __launch_bounds__(256) void checkpoint8_kernel(const T *__restrict__ x, int64_t stride, int64_t n, int k, int pitch,
                                                          int lanes, int quads_per_block, uint8_t *__restrict__ codes,
                                                          uint8_t *__restrict__ scales) {
  constexpr int SHARE = kGroup / C;
  const int r = threadIdx.x / min(lanes, 256);
  const int64_t quad = (int64_t)blockIdx.x * quads_per_block + r, row = quad * 4;
  if (r >= quads_per_block || row >= n) return;
  for (int u = threadIdx.x - r * min(lanes, 256); u < lanes; u += 256) {
    const int c = u * C;
    float f[4][C];
    uint32_t byte[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const T *src = x + min(row + q, n - 1) * stride + c;      // (behind the last row: its values, cleared below)
      if (c + C <= k) {
        dg_load_unaligned<C>(src, f[q]);
      } else {
#pragma unroll
        for (int e = 0; e < C; ++e) f[q][e] = c + e < k ? dg_widen(src[e]) : 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < C; ++e) top = max(top, __float_as_uint(f[q][e]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < SHARE; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
      byte[q] = scale_byte<FMT>(row + q < n ? top : 0);
      const bool none = byte[q] == kNoNumber || row + q >= n;
      const float inv = __uint_as_float((254u - (none ? 0 : byte[q])) << 23);
#pragma unroll
      for (int e = 0; e < C; ++e) f[q][e] = none ? 0.f : f[q][e] * inv;
    }
    if (c < pitch) {
      u32x4 *to = reinterpret_cast<u32x4 *>(codes + quad * 4 * pitch + 4 * c);
#pragma unroll
      for (int h = 0; h < C / 4; ++h) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = encode_rows<FMT>(f[0][4 * h + e], f[1][4 * h + e], f[2][4 * h + e], f[3][4 * h + e]);
        to[h] = w;
      }
    }
    if (u % SHARE == 0)
      *reinterpret_cast<uint32_t *>(scales + quad * 4 * (lanes / SHARE) + 4 * (u / SHARE)) = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
  }
}

// The same the other way round, four columns a lane: bound by memory (1e6 rows of 128 to fp32: 5.9 TB/s; 4097 x 333
// fp16 in 3.4 us, mostly a launch's latency).
template <typename T, int FMT>
__global__ __launch_bounds__(256) void checkpoint8_values_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                                 int64_t n, int k, int pitch, int lanes, int quads_per_block,
                                                                 T *__restrict__ out) {
  const int r = threadIdx.x / min(lanes, 256);
  const int64_t quad = (int64_t)blockIdx.x * quads_per_block + r, row = quad * 4;
  if (r >= quads_per_block || row >= n) return;
  for (int u = threadIdx.x - r * min(lanes, 256); u < lanes; u += 256) {
    const int c = u * 4;
    if (c >= k) continue;
    const u32x4 w = *reinterpret_cast<const u32x4 *>(codes + quad * 4 * pitch + 4 * c);
    float s[4], f[4][4];
    scales_of(*reinterpret_cast<const uint32_t *>(scales + quad * (lanes >> 1) + (u >> 3) * 4), s);
#pragma unroll
    for (int e = 0; e < 4; ++e) decode_rows<FMT>(w[e], s, f[e]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (row + q >= n) break;
      T *dst = out + (row + q) * k + c;
      const float v[4] = {f[0][q], f[1][q], f[2][q], f[3][q]};
      if (c + 4 <= k) {
        dg_store_unaligned<4>(dst, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < k) dst[e] = dg_round<T>(v[e]);
      }
    }
  }
}

// ---- the layer's backward -----------------------------------------------------------------------------------------
struct back_args {
  const void *d_y;
  int64_t d_stride;
  const uint8_t *x, *x_scales, *y, *y_scales;
  int x_pitch, x_groups, y_pitch, y_groups;
  int64_t n;
  int k, m;
  int strips, tiles_m, tiles_n;
  void *d_z;            // contiguous [n][m], written under tanh
  float *part, *part_b; // [strip][tile_m][tile_n][BM][BN], [strip][tiles_m * BM]
};

__device__ __forceinline__ uint32_t high_halves(float a, float b) {   // bf16(a) | bf16(b) << 16, by truncation
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// W neighbouring elements through a buffer descriptor: beyond its end they read as zeros.
template <int BYTES>
__device__ __forceinline__ auto load_bytes(__amdgpu_buffer_rsrc_t r, uint32_t at) {
  if constexpr (BYTES == 16) return __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
  else if constexpr (BYTES == 8) return __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
  else if constexpr (BYTES == 4) return __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
  else if constexpr (BYTES == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
  else return __builtin_amdgcn_raw_buffer_load_b8(r, at, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void *base, int64_t offset, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)base + offset), 0, bytes, 0x00020000);
}

// What a thread holds of a block of rows until it lays them down: four rows of WA columns of d_y (and of the codes of y),
// four rows of WB columns of the codes of x, a word a column, and the four rows' scales.
template <typename T, int WA, int WB>
struct back_regs {
  dg_vec<T, WA> d[4];
  uint32_t y[WA], ys, x[WB], xs;
};

// A workgroup sums one strip of rows -- every so many blocks of 32, so that all workgroups together read on through the
// memory -- for a BM x BN tile of d_w, a block a step: its threads load quads of rows x a few
// columns, form d_z, cut it, and lay both operands down in LDS with eight rows of a column in 16 bytes -- what a lane of
// the matrix instruction takes -- transposing in their registers.  A column c of a tile of B sits in slot
// (c mod W) 32 + c / W, W = B / 32, so that neighbouring lanes write neighbouring slots; results are kept in slot order
// until the second launch.  Two buffers in LDS and two steps on their way in registers: one barrier a step, and the conversion of
// the next step runs beside the matrix instructions of this one.  A block's rows end with their descriptors: rows behind
// the last one, and whole blocks behind it, come as zeros, with no branch round a load.
// Bound by memory for few columns (1e6 rows, 128 -> 64, fp32, tanh: 710 MB in 135 us, 5.3 TB/s), for many by conversion,
// LDS and matrix instructions that overlap in part (16384 rows, 1000 -> 1000, bf16, with the strips' sums: 58 us, 565 TFLOP/s;
// some 24, 20 and 14 us of vector, LDS and matrix cycles on a SIMD; under tanh, three bf16 numbers a d_z: 140 us).  Paths of
// their own for odd widths and for the tiles that form no column sums: 57 us, not kept.
// NARROW: d_y has one column (a load of two would leave its row).
template <typename T, int FMT, bool TANH, int PIECES, int BM, int BN, bool NARROW>
__global__ __launch_bounds__(256) void checkpoint8_backward_kernel(back_args a) {
  constexpr int BK = 32, WA = BM / 32, WB = BN / 32, WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32, Z = sizeof(T);
  constexpr bool RAW = PIECES == 1 && Z == 2 && !TANH;                 // bf16 as it came
  struct buffer {
    u32x4 a[PIECES][BK / 8][BM], b[BK / 8][BN];
  };
  __shared__ buffer lds[2];
  const int tiles = a.tiles_m * a.tiles_n;
  // an eighth of the (strip, tile) pairs to each XCD, strip by strip: the tiles of a strip, which read the same rows, share an L2
  const int64_t per = gridDim.x >> 3, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  const int strip = (int)(item / tiles), tile = (int)(item % tiles);
  if (strip >= a.strips) return;
  const int m0 = tile / a.tiles_n * BM, n0 = tile % a.tiles_n * BN;
  const bool first_n = n0 == 0;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  // (half a wave writes both halves of 16 slots: 256 bytes on end, every bank once)
  const int cw = (tid & 15) | ((tid >> 1) & 16), rq = ((tid >> 5) & 6) | ((tid >> 4) & 1), steps = (int)(((a.n + BK - 1) / BK - strip + a.strips - 1) / a.strips);
  // columns behind the last one: some other column's values, in rows or columns of the tile that nobody keeps
  const int ca = min(m0 + cw * WA, a.m - 1) / WA * WA, cb = min(n0 + cw * WB, a.k - 1) / WB * WB;
  // the last columns of an odd width are read from further left, and moved into place when they are laid down
  const bool odd = a.m % WA != 0;
  const int from = odd && !NARROW ? min(ca, a.m - WA) : ca, shift = ca - from;
  const uint32_t r0 = rq * 4, d_pitch = (uint32_t)a.d_stride * Z;
  const uint32_t at_d = r0 * d_pitch + from * Z, at_y = r0 * a.y_pitch + 4 * ca, at_ys = r0 * a.y_groups + ca / kGroup * 4;
  const uint32_t at_x = r0 * a.x_pitch + 4 * cb, at_xs = r0 * a.x_groups + cb / kGroup * 4;

  float sums[WA];
#pragma unroll
  for (int j = 0; j < WA; ++j) sums[j] = 0.f;
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  auto fetch = [&](back_regs<T, WA, WB> &g, int step) {
    const int64_t base = ((int64_t)step * a.strips + strip) * BK;
    const int left = (int)max((int64_t)0, min((int64_t)BK, a.n - base));
    const auto d = rows_at(a.d_y, base * d_pitch, left ? (left - 1) * (int)d_pitch + a.m * Z : 0);
    const int kept = (left + 3) & ~3;                                   // (whole quads of rows; those behind the last: zeros)
    const auto x = rows_at(a.x, base * a.x_pitch, kept * a.x_pitch), xs = rows_at(a.x_scales, base * a.x_groups, kept * a.x_groups);
    const auto y = rows_at(a.y, base * a.y_pitch, kept * a.y_pitch), ys = rows_at(a.y_scales, base * a.y_groups, kept * a.y_groups);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (!NARROW) {
        const auto w = load_bytes<WA * Z>(d, at_d + q * d_pitch);
        __builtin_memcpy(&g.d[q], &w, WA * Z);
      } else {
        const auto w = load_bytes<Z>(d, at_d + q * d_pitch);
        __builtin_memcpy(&g.d[q].v[0], &w, Z);
        g.d[q].v[1] = g.d[q].v[0];
      }
    }
    if (TANH) {
      const auto w = load_bytes<4 * WA>(y, at_y);
      __builtin_memcpy(g.y, &w, 4 * WA);
      g.ys = load_bytes<4>(ys, at_ys);
    }
    const auto w = load_bytes<4 * WB>(x, at_x);
    __builtin_memcpy(g.x, &w, 4 * WB);
    g.xs = load_bytes<4>(xs, at_xs);
  };

  auto lay_down = [&](const back_regs<T, WA, WB> &g, int step, buffer &to) {
    float d[4][WA];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < WA; ++j) d[q][j] = dg_widen(g.d[q].v[j]);
    if (odd) {
#pragma unroll
      for (int by = WA / 2; by; by >>= 1)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j + by < WA; ++j) {
            const float here = d[q][j], there = d[q][j + by];
            d[q][j] = (shift & by) ? there : here;
          }
    }
    if (TANH) {
      const int64_t base = ((int64_t)step * a.strips + strip) * BK;
      float s[4], y[4];
      scales_of(g.ys, s);
#pragma unroll
      for (int j = 0; j < WA; ++j) {
        decode_rows<FMT>(g.y[j], s, y);
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q][j] *= 1.f - y[q] * y[q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (first_n && base + r0 + q < a.n && m0 + cw * WA < a.m) {
          T *dst = (T *)a.d_z + (base + r0 + q) * a.m + ca;
          if (!odd) {
            dg_store_unaligned<WA>(dst, d[q]);
          } else {
#pragma unroll
            for (int j = 0; j < WA; ++j)
              if (ca + j < a.m) dst[j] = dg_round<T>(d[q][j]);
          }
        }
      }
    }
    if (first_n) {
#pragma unroll
      for (int j = 0; j < WA; ++j) sums[j] += (d[0][j] + d[1][j]) + (d[2][j] + d[3][j]);
    }
    if (RAW && !odd) {                                                 // two halves of a word, rows paired column by column
#pragma unroll
      for (int j = 0; j < WA; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) __builtin_memcpy(&w[q], &g.d[q].v[j & ~1], 4);
        const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
        const u32x2 p = {__builtin_amdgcn_perm(w[1], w[0], pick), __builtin_amdgcn_perm(w[3], w[2], pick)};
        reinterpret_cast<u32x2 *>(&to.a[0][rq >> 1][j * 32 + cw])[rq & 1] = p;
      }
    } else {
#pragma unroll
      for (int j = 0; j < WA; ++j) {
        float v[4] = {d[0][j], d[1][j], d[2][j], d[3][j]};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const u32x2 w = {high_halves(v[0], v[1]), high_halves(v[2], v[3])};
          reinterpret_cast<u32x2 *>(&to.a[p][rq >> 1][j * 32 + cw])[rq & 1] = w;
          if (p + 1 < PIECES) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] -= __uint_as_float(__float_as_uint(v[q]) & 0xffff0000u);   // (exact)
          }
        }
      }
    }
    float s[4], x[4];
    scales_of(g.xs, s);
#pragma unroll
    for (int j = 0; j < WB; ++j) {
      decode_rows<FMT>(g.x[j], s, x);
      const u32x2 w = {high_halves(x[0], x[1]), high_halves(x[2], x[3])};
      reinterpret_cast<u32x2 *>(&to.b[rq >> 1][j * 32 + cw])[rq & 1] = w;
    }
  };

  auto multiply = [&](const buffer &from) {
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const int k8 = kk * 2 + (lane >> 5);
      bf16x8 fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = __builtin_bit_cast(bf16x8, from.b[k8][wn + j * 32 + (lane & 31)]);
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const bf16x8 fa = __builtin_bit_cast(bf16x8, from.a[p][k8][wm + i * 32 + (lane & 31)]);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb[j], acc[i][j], 0, 0, 0);
        }
    }
  };

  // Step i is multiplied out of buffer i mod 2 while step i + 1 is laid down in the other and step i + 3 is asked for.
  back_regs<T, WA, WB> g0, g1;
  fetch(g0, 0);
  fetch(g1, 1);
  lay_down(g0, 0, lds[0]);
  fetch(g0, 2);
  __syncthreads();
  for (int i = 0; i < steps; i += 2) {
    lay_down(g1, i + 1, lds[1]);
    fetch(g1, i + 3);
    multiply(lds[0]);
    __syncthreads();
    lay_down(g0, i + 2, lds[0]);
    fetch(g0, i + 4);
    multiply(lds[1]);
    __syncthreads();
  }

  float *part = a.part + ((size_t)strip * tiles + tile) * (BM * BN);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        part[(size_t)(wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * BN + wn + j * 32 + (lane & 31)] = acc[i][j][e];
  if (!first_n) return;
  float *col_sums = reinterpret_cast<float *>(&lds[0]);               // [8][BM]; the last step's readers are past their barrier
#pragma unroll
  for (int j = 0; j < WA; ++j) col_sums[rq * BM + cw * WA + j] = sums[j];
  __syncthreads();
  for (int c = tid; c < BM; c += 256) {
    float s = 0.f;
    for (int q = 0; q < 8; ++q) s += col_sums[q * BM + c];
    a.part_b[(size_t)strip * (a.tiles_m * BM) + m0 + c] = s;
  }
}

// Adds the strips' parts: 2^log_strands strands of every so many strips each, the strands in order.  A block takes
// 1024 >> log_strands neighbouring values: of a tile (in slot order), or -- the blocks behind them -- of the column sums.
// Bound by its read: 8 strips of 1024 x 1024 (34 MB) in 8.7 us.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void checkpoint8_reduce_kernel(const float *__restrict__ part, const float *__restrict__ part_b,
                                                                 int strips, int log_strands, int tiles_m, int tiles_n, int m, int k,
                                                                 T *__restrict__ d_w, T *__restrict__ d_b) {
  __shared__ alignas(16) float strand[1024];
  const int tiles = tiles_m * tiles_n, per = 1024 >> log_strands, strands = 1 << log_strands, lanes = per / 4;
  const unsigned blocks_w = (unsigned)tiles * (BM * BN / per);
  const bool bias = blockIdx.x >= blocks_w;
  const size_t at = (size_t)(bias ? blockIdx.x - blocks_w : blockIdx.x) * per;
  const size_t step = bias ? (size_t)tiles_m * BM : (size_t)tiles * BM * BN;
  const int g = threadIdx.x / lanes, l = threadIdx.x % lanes;
  const float *src = (bias ? part_b : part) + at + 4 * l;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (at + 4 * l < step) {
#pragma unroll 4
    for (int s = g; s < strips; s += strands) {
      float f[4];
      dg_load<4>(src + s * step, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) strand[g * per + 4 * l + e] = acc[e];
  __syncthreads();
  for (int v = threadIdx.x; v < per; v += 256) {
    float s = strand[v];
    for (int q = 1; q < strands; ++q) s += strand[q * per + v];
    if (bias) {
      if (at + v < (size_t)m) d_b[at + v] = dg_round<T>(s);
      continue;
    }
    const int tile = (int)(at / (BM * BN)), in = (int)(at % (BM * BN)) + v, i = in / BN, j = in % BN;
    const int o = tile / tiles_n * BM + i % 32 * (BM / 32) + i / 32, c = tile % tiles_n * BN + j % 32 * (BN / 32) + j / 32;
    if (o < m && c < k) d_w[(size_t)o * k + c] = dg_round<T>(s);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------
int type_size(int dtype) { return dtype == DG_F32 ? 4 : (dtype == DG_BF16 || dtype == DG_F16) ? 2 : 0; }
int pitch_of(int k) { return (k + 15) / 16 * 16; }
int groups_of(int k) { return (k + kGroup - 1) / kGroup; }

int check_sizes(const char *what, int64_t n, int64_t k, int fmt) {
  if (fmt != DG_INT8 && fmt != DG_E4M3) return dg_fail(DG_ERR_ARG, "%s: unknown 8-bit format %d", what, fmt);
  if (n < 0 || k <= 0) return dg_fail(DG_ERR_ARG, "%s: bad sizes", what);
  if (k > (1 << 20) || n > 0x7fffffff) return dg_fail(DG_ERR_SIZE, "%s: at most 2^31 - 1 rows of 2^20 columns", what);
  return 0;
}

int64_t quads_of(int64_t n) { return (n + 3) / 4; }
size_t scales_at(int64_t n, int k) { return (size_t)quads_of(n) * 4 * pitch_of(k); }

constexpr int64_t kMostBlocks = 0xffffff;       // of 256 threads: a launch has fewer than 2^32 (2^35 elements fit for any k)

struct row_grid {
  int lanes, quads_per_block;
  int64_t blocks;
};
row_grid rows_of(int64_t n, int k, int columns) {
  row_grid g;
  g.lanes = kGroup / columns * groups_of(k);
  g.quads_per_block = g.lanes >= 256 ? 1 : 256 / g.lanes;
  g.blocks = (quads_of(n) + g.quads_per_block - 1) / g.quads_per_block;
  return g;
}

// Tiles of 128 columns, or 64 where that leaves fewer of them empty; strips so that at most 512 workgroups run, two a CU and
// all at once (one more than 512, 63114 rows, 136 -> 128, fp32, tanh: 47 against 36 us; 1024, 1e6 rows, 128 -> 64: 153 against
// 141, for the partial sums they add), of at least 128 rows each (64 rows, 8192 x 256 x 256: 29 against 26 us), and 256 with
// the largest tile, whose partial sums cost the most (8192 rows, 200 -> 128, bf16: 12.8 us against 16.3 with 128; 512 x 1024 x
// 1024: 16.3 against 19.7).
int side_of(int columns) { return (columns + 127) / 128 * 2 > (columns + 63) / 64 ? 64 : 128; }
struct back_plan {
  int bm, bn, tiles_m, tiles_n, strips;
  size_t part, part_b, bytes;
};
back_plan plan_of(int64_t n, int k, int m) {
  back_plan p;
  p.bm = side_of(m);
  p.bn = m == 1 ? 128 : side_of(k);
  p.tiles_m = (m + p.bm - 1) / p.bm;
  p.tiles_n = (k + p.bn - 1) / p.bn;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  const int64_t least = p.bm * p.bn == 128 * 128 ? 256 : 128, most = (n + least - 1) / least;
  int64_t strips = tiles < 512 ? 512 / tiles : 1;
  strips = strips < most ? strips : most;
  p.strips = (int)strips;
  p.part = 0;
  p.part_b = (size_t)p.strips * tiles * p.bm * p.bn * 4;
  p.bytes = p.part_b + (size_t)p.strips * p.tiles_m * p.bm * 4 + 256;
  return p;
}

template <typename T, int FMT, bool TANH, int PIECES, int BM, int BN, bool NARROW>
int back_as(const back_plan &p, const back_args &a, T *d_w, T *d_b, hipStream_t stream) {
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, blocks = (p.strips * tiles + 7) / 8 * 8;
  int log_strands = 0;
  while (log_strands < 6 && (2 << log_strands) <= p.strips) ++log_strands;
  const int per = 1024 >> log_strands;
  const int64_t sums = tiles * (BM * BN / per) + ((int64_t)p.tiles_m * BM + per - 1) / per;
  if (blocks > kMostBlocks || sums > kMostBlocks) return dg_fail(DG_ERR_SIZE, "dg_checkpoint8_backward: a weight of %d x %d is too large", a.m, a.k);
  if (p.strips) {
    hipLaunchKernelGGL((checkpoint8_backward_kernel<T, FMT, TANH, PIECES, BM, BN, NARROW>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    DG_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL((checkpoint8_reduce_kernel<T, BM, BN>), dim3((unsigned)sums), dim3(256), 0, stream, a.part, a.part_b, p.strips,
                     log_strands, p.tiles_m, p.tiles_n, a.m, a.k, d_w, d_b);
  DG_HIP(hipGetLastError());
  return 0;
}

template <typename T, int FMT, bool TANH, int PIECES>
int back_tiles(const back_plan &p, const back_args &a, void *d_w, void *d_b, hipStream_t stream) {
  if (a.m == 1) return back_as<T, FMT, TANH, PIECES, 64, 128, true>(p, a, (T *)d_w, (T *)d_b, stream);
  if (p.bm == 128) {
    if (p.bn == 128) return back_as<T, FMT, TANH, PIECES, 128, 128, false>(p, a, (T *)d_w, (T *)d_b, stream);
    return back_as<T, FMT, TANH, PIECES, 128, 64, false>(p, a, (T *)d_w, (T *)d_b, stream);
  }
  if (p.bn == 128) return back_as<T, FMT, TANH, PIECES, 64, 128, false>(p, a, (T *)d_w, (T *)d_b, stream);
  return back_as<T, FMT, TANH, PIECES, 64, 64, false>(p, a, (T *)d_w, (T *)d_b, stream);
}

// PLAIN: the bf16 numbers that hold a value of T; three hold an fp32 value, as d_z is under tanh whatever the type.
template <typename T, int PLAIN>
int back_forms(int fmt, bool tanh, const back_plan &p, const back_args &a, void *d_w, void *d_b, hipStream_t stream) {
  if (fmt == DG_E4M3)
    return tanh ? back_tiles<T, DG_E4M3, true, 3>(p, a, d_w, d_b, stream) : back_tiles<T, DG_E4M3, false, PLAIN>(p, a, d_w, d_b, stream);
  return tanh ? back_tiles<T, DG_INT8, true, 3>(p, a, d_w, d_b, stream) : back_tiles<T, DG_INT8, false, PLAIN>(p, a, d_w, d_b, stream);
}

}  // namespace

extern "C" size_t dg_checkpoint8_bytes(int64_t n, int32_t k) {
  if (n < 0 || n > 0x7fffffff || k <= 0 || k > (1 << 20)) return 0;
  return scales_at(n, k) + (size_t)quads_of(n) * 4 * groups_of(k);
}

// FN(element type, format) for a pair of them.
#define DG_BY_TYPE_AND_FORMAT(FN, dtype, format)   \
  if (format == DG_E4M3) {                         \
    if (dtype == DG_F32) FN(float, DG_E4M3);       \
    else if (dtype == DG_BF16) FN(dg_bf16, DG_E4M3); \
    else FN(dg_f16, DG_E4M3);                      \
  } else {                                         \
    if (dtype == DG_F32) FN(float, DG_INT8);       \
    else if (dtype == DG_BF16) FN(dg_bf16, DG_INT8); \
    else FN(dg_f16, DG_INT8);                      \
  }

extern "C" int dg_checkpoint8(const void *x, int64_t row_stride, int64_t n, int32_t k, int32_t dtype, int32_t format, void *kept,
                              void *stream) {
  if (const int rc = check_sizes("dg_checkpoint8", n, k, format)) return rc;
  if (!type_size(dtype)) return dg_fail(DG_ERR_ARG, "dg_checkpoint8: unknown element type %d", dtype);
  if (row_stride < 0) return dg_fail(DG_ERR_ARG, "dg_checkpoint8: negative row stride");
  if (n == 0) return 0;
  if (!x || !kept) return dg_fail(DG_ERR_ARG, "dg_checkpoint8: NULL argument");
  if ((uintptr_t)kept & 15) return dg_fail(DG_ERR_ARG, "dg_checkpoint8: the kept bytes must be 16-byte aligned");
  const row_grid g = rows_of(n, k, 16 / type_size(dtype));
  if (g.blocks > kMostBlocks) return dg_fail(DG_ERR_SIZE, "dg_checkpoint8: %lld rows of %d columns are too many", (long long)n, k);
  uint8_t *codes = (uint8_t *)kept, *scales = codes + scales_at(n, k);
#define DG_KEEP(T, F)                                                                                                               \
  hipLaunchKernelGGL((checkpoint8_kernel<T, F, 16 / sizeof(T)>), dim3((unsigned)g.blocks), dim3(256), 0, (hipStream_t)stream, (const T *)x, row_stride, n, k, \
                     pitch_of(k), g.lanes, g.quads_per_block, codes, scales)
  DG_BY_TYPE_AND_FORMAT(DG_KEEP, dtype, format)
#undef DG_KEEP
  DG_HIP(hipGetLastError());
  return 0;
}

extern "C" int dg_checkpoint8_values(const void *kept, int64_t n, int32_t k, int32_t format, int32_t dtype, void *out, void *stream) {
  if (const int rc = check_sizes("dg_checkpoint8_values", n, k, format)) return rc;
  if (!type_size(dtype)) return dg_fail(DG_ERR_ARG, "dg_checkpoint8_values: unknown element type %d", dtype);
  if (n == 0) return 0;
  if (!kept || !out) return dg_fail(DG_ERR_ARG, "dg_checkpoint8_values: NULL argument");
  if ((uintptr_t)kept & 15) return dg_fail(DG_ERR_ARG, "dg_checkpoint8_values: the kept bytes must be 16-byte aligned");
  const row_grid g = rows_of(n, k, 4);
  if (g.blocks > kMostBlocks) return dg_fail(DG_ERR_SIZE, "dg_checkpoint8_values: %lld rows of %d columns are too many", (long long)n, k);
  const uint8_t *codes = (const uint8_t *)kept, *scales = codes + scales_at(n, k);
#define DG_READ(T, F)                                                                                                           \
  hipLaunchKernelGGL((checkpoint8_values_kernel<T, F>), dim3((unsigned)g.blocks), dim3(256), 0, (hipStream_t)stream, codes, scales, n, k, \
                     pitch_of(k), g.lanes, g.quads_per_block, (T *)out)
  DG_BY_TYPE_AND_FORMAT(DG_READ, dtype, format)
#undef DG_READ
  DG_HIP(hipGetLastError());
  return 0;
}

extern "C" size_t dg_checkpoint8_backward_workspace(int64_t n, int32_t k, int32_t m) {
  if (n < 0 || k <= 0 || m <= 0 || n > 0x7fffffff || k > (1 << 20) || m > (1 << 20)) return 0;
  return plan_of(n, k, m).bytes;
}

extern "C" int dg_checkpoint8_backward(const void *d_y, int64_t row_stride, int64_t n, int32_t m, int32_t k, int32_t dtype, int32_t format,
                                       const void *x_kept, const void *y_kept, void *d_z, void *d_w, void *d_b, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  if (const int rc = check_sizes("dg_checkpoint8_backward", n, k, format)) return rc;
  if (const int rc = check_sizes("dg_checkpoint8_backward", n, m, format)) return rc;
  if (!type_size(dtype)) return dg_fail(DG_ERR_ARG, "dg_checkpoint8_backward: unknown element type %d", dtype);
  const bool tanh = y_kept != nullptr;
  if (!d_w || !d_b || !workspace || (n && (!d_y || !x_kept || (tanh && !d_z))))
    return dg_fail(DG_ERR_ARG, "dg_checkpoint8_backward: NULL argument");
  if (((uintptr_t)x_kept | (uintptr_t)y_kept | (uintptr_t)workspace) & 15)
    return dg_fail(DG_ERR_ARG, "dg_checkpoint8_backward: kept bytes and workspace must be 16-byte aligned");
  if (row_stride > (1 << 24)) return dg_fail(DG_ERR_SIZE, "dg_checkpoint8_backward: rows of d_y more than 2^24 elements apart");
  if (row_stride < m) return dg_fail(DG_ERR_ARG, "dg_checkpoint8_backward: rows of d_y overlap");
  const back_plan p = plan_of(n, k, m);
  if (workspace_bytes < p.bytes)
    return dg_fail(DG_ERR_SIZE, "dg_checkpoint8_backward: workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
  const uint8_t *x = (const uint8_t *)x_kept, *y = (const uint8_t *)y_kept;
  back_args a = {d_y, row_stride, x, x + scales_at(n, k), y, tanh ? y + scales_at(n, m) : nullptr,
                 pitch_of(k), groups_of(k), pitch_of(m), groups_of(m), n, k, m, p.strips, p.tiles_m, p.tiles_n, d_z,
                 (float *)workspace, (float *)((char *)workspace + p.part_b)};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DG_F32) return back_forms<float, 3>(format, tanh, p, a, d_w, d_b, st);
  if (dtype == DG_BF16) return back_forms<dg_bf16, 1>(format, tanh, p, a, d_w, d_b, st);
  return back_forms<dg_f16, 2>(format, tanh, p, a, d_w, d_b, st);
}
