// Block quantisation to 8-bit floating point (pgv_f8_quantize): every value is read once, its block's maximum is found in
// registers, and the byte and the scale are written - of the matrix, and on request of its transpose and its column sums.
//
// Bound by memory: R C (element size + 1 or 2) bytes.  Two kernels:
//   quant_rows   blocks of 128 along a row, no transpose: 16 lanes x 8 values per block, the maximum by DPP inside the 16
//                lanes, no LDS.  Units (block, row) run over the rows first so that neighbouring units write neighbouring
//                scales ([K/128][R]: a product reads the scales of a tile's rows at one K as one line).
//   quant_tile   one 128 x 128 tile per workgroup of 256: a thread holds 8 x 8 values, so a column's maximum and an 8-byte
//                piece of the transpose are in its registers; the transpose leaves through a 17 KB LDS image.
#include "f8_common.h"

namespace {

constexpr int UNITS = 4;   // blocks in flight per 16 lanes

template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ldx, int R, int C, int Kb,
                                                         uint8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t units = (int64_t)R * Kb, Kp = (int64_t)Kb * F8B;
  const int l16 = threadIdx.x & 15;
  const int64_t u0 = (int64_t)blockIdx.x * (16 * UNITS) + (threadIdx.x >> 4);
  float v[UNITS][8];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int64_t u = u0 + 16 * i;
    if (u < units) {
      const int kb = (int)(u / R), r = (int)(u - (int64_t)kb * R), c = kb * F8B + l16 * 8;
      f8_load8<VEC>(x + r * ldx + c, C - c, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int64_t u = u0 + 16 * i;
    if (u >= units) continue;
    const int kb = (int)(u / R), r = (int)(u - (int64_t)kb * R), c = kb * F8B + l16 * 8;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, f8_abs_bits(v[i][j]));
    m = f8_max16(m);
    float s, inv;
    f8_scale<FMT>(m, s, inv);
    i32x2 o;
    o.x = f8_pack4<FMT>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
    o.y = f8_pack4<FMT>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
    *reinterpret_cast<i32x2*>(q + r * Kp + c) = o;
    if (l16 == 0) scale[u] = s;
  }
}

constexpr int TP = 132;   // bytes per row of the transposed image: 33 dwords, so that 8-byte pieces 8 rows apart spread over the banks

// ROWS / TRANS: which of q / qt is written.  TILE: one scale for the whole tile, else one per row (q) and per column (qt).
template <typename T, int FMT, bool TILE, bool VEC>
__global__ __launch_bounds__(256) void quant_tile_kernel(const T* __restrict__ x, int64_t ldx, int R, int C, int Kb, int Rb,
                                                         uint8_t* __restrict__ q, float* __restrict__ scale,
                                                         uint8_t* __restrict__ qt, float* __restrict__ scale_t,
                                                         float* __restrict__ colpart) {
  __shared__ __attribute__((aligned(16))) uint8_t img[F8B * TP];
  __shared__ uint32_t red[4][F8B];
  __shared__ float sums[4][F8B];
  __shared__ float inv_t[F8B];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = tid & 15, g = tid >> 4;
  const int kb = blockIdx.x % Kb, rb = blockIdx.x / Kb;
  const int r0 = rb * F8B + g * 8, c0 = kb * F8B + l16 * 8;   // this thread's 8 x 8 values
  const int64_t Kp = (int64_t)Kb * F8B, Rp = (int64_t)Rb * F8B;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (r0 + i < R)
      f8_load8<VEC>(x + (r0 + i) * ldx + c0, C - c0, v[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
  }
  float s, inv;
  if constexpr (TILE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, f8_abs_bits(v[i][j]));
    m = f8_max16(m);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
    if (lane == 0) red[wave][0] = m;
    __syncthreads();
    m = max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0]));
    f8_scale<FMT>(m, s, inv);
    if (tid == 0) {
      if (q) scale[(int64_t)rb * Kb + kb] = s;
      if (qt) scale_t[(int64_t)kb * Rb + rb] = s;
    }
  }
  if (q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (!TILE) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, f8_abs_bits(v[i][j]));
        m = f8_max16(m);
        f8_scale<FMT>(m, s, inv);
      }
      if (r0 + i < R) {
        i32x2 o;
        o.x = f8_pack4<FMT>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        o.y = f8_pack4<FMT>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        *reinterpret_cast<i32x2*>(q + (r0 + i) * Kp + c0) = o;
        if (!TILE && l16 == 0) scale[(int64_t)kb * R + r0 + i] = s;
      }
    }
  }
  if (!qt && !colpart) return;   // (uniform over the grid)
  // maxima and sums of the columns: 8 rows in the thread, 4 threads of the wave, 4 waves
  if (!TILE || colpart) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t m = 0;
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, f8_abs_bits(v[i][j])), t += v[i][j];
      if (!TILE) {
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if (lane < 16) red[wave][l16 * 8 + j] = m;
      }
      if (colpart) {
        t += __shfl_xor(t, 16, 64);
        t += __shfl_xor(t, 32, 64);
        if (lane < 16) sums[wave][l16 * 8 + j] = t;
      }
    }
    __syncthreads();
    if (tid < F8B) {
      const int c = kb * F8B + tid;
      if (!TILE) {
        const uint32_t m = max(max(red[0][tid], red[1][tid]), max(red[2][tid], red[3][tid]));
        float sc, iv;
        f8_scale<FMT>(m, sc, iv);
        inv_t[tid] = iv;
        if (qt && c < C) scale_t[(int64_t)rb * C + c] = sc;
      }
      if (colpart && c < C) colpart[(int64_t)rb * C + c] = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
    }
    __syncthreads();
  }
  if (!qt) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float iv = TILE ? inv : inv_t[l16 * 8 + j];
    int* d = reinterpret_cast<int*>(img + (l16 * 8 + j) * TP + g * 8);
    d[0] = f8_pack4<FMT>(v[0][j] * iv, v[1][j] * iv, v[2][j] * iv, v[3][j] * iv);
    d[1] = f8_pack4<FMT>(v[4][j] * iv, v[5][j] * iv, v[6][j] * iv, v[7][j] * iv);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int cl = (tid >> 3) + 32 * i, c = kb * F8B + cl;
    if (c < C) {
      const int* sp = reinterpret_cast<const int*>(img + cl * TP + (tid & 7) * 16);
      i32x4 o = {sp[0], sp[1], sp[2], sp[3]};
      *reinterpret_cast<i32x4*>(qt + c * Rp + rb * F8B + (tid & 7) * 16) = o;
    }
  }
}

// column sums from the per-tile partial sums: 32 columns x 8 interleaved chains of tiles, then their sum
__global__ __launch_bounds__(256) void colsum_parts_kernel(const float* __restrict__ part, int Rb, int C,
                                                           float* __restrict__ out) {
  __shared__ double red[8][32];
  const int l = threadIdx.x & 31, ph = threadIdx.x >> 5, c = blockIdx.x * 32 + l;
  double t = 0.0;
  if (c < C)
#pragma unroll 4
    for (int r = ph; r < Rb; r += 8) t += (double)part[(int64_t)r * C + c];
  red[ph][l] = t;
  __syncthreads();
  if (threadIdx.x < 32 && c < C) {
    for (int i = 1; i < 8; ++i) t += red[i][l];
    out[c] = (float)t;
  }
}

template <typename T, int FMT>
int launch(const T* x, int64_t R, int64_t C, int64_t ldx, int block, uint8_t* q, float* scale, uint8_t* qt, float* scale_t,
           float* colsum, float* part, hipStream_t st) {
  const int Kb = (int)pgv_cdiv(C, F8B), Rb = (int)pgv_cdiv(R, F8B);
  const bool vec = ((uintptr_t)x % 16) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  if (block == PGV_F8_ROWS && !qt && !colsum) {
    const int64_t grid = pgv_cdiv(R * Kb, 16 * UNITS);
    if (vec)
      quant_rows_kernel<T, FMT, true><<<dim3((unsigned)grid), 256, 0, st>>>(x, ldx, (int)R, (int)C, Kb, q, scale);
    else
      quant_rows_kernel<T, FMT, false><<<dim3((unsigned)grid), 256, 0, st>>>(x, ldx, (int)R, (int)C, Kb, q, scale);
  } else {
    const dim3 grid((unsigned)((int64_t)Kb * Rb));
#define PGV_TILE(TILE, VEC) \
  quant_tile_kernel<T, FMT, TILE, VEC><<<grid, 256, 0, st>>>(x, ldx, (int)R, (int)C, Kb, Rb, q, scale, qt, scale_t, part)
    if (block == PGV_F8_TILES)
      vec ? PGV_TILE(true, true) : PGV_TILE(true, false);
    else
      vec ? PGV_TILE(false, true) : PGV_TILE(false, false);
#undef PGV_TILE
    if (colsum) colsum_parts_kernel<<<dim3((unsigned)pgv_cdiv(C, 32)), 256, 0, st>>>(part, Rb, (int)C, colsum);
  }
  PGV_CHECK_LAUNCH("pgv_f8_quantize");
  return PGV_OK;
}

}  // namespace

extern "C" int64_t pgv_f8_quantize_workspace(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? 4 * pgv_cdiv(rows, F8B) * cols : 0;
}

extern "C" int pgv_f8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int block, int fmt, void* q,
                               float* scale, void* qt, float* scale_t, float* colsum, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  PGV_CHECK_ARG(f8_dt_ok(dtype), "pgv_f8_quantize: unknown element type %d", dtype);
  PGV_CHECK_ARG(block == PGV_F8_ROWS || block == PGV_F8_TILES, "pgv_f8_quantize: unknown block kind %d", block);
  PGV_CHECK_ARG(fmt == PGV_F8_E4M3 || fmt == PGV_F8_E5M2, "pgv_f8_quantize: unknown 8-bit format %d", fmt);
  PGV_CHECK_ARG(rows >= 0 && cols >= 0 && rows <= PGV_F8_MAX_EXTENT && cols <= PGV_F8_MAX_EXTENT && ldx >= cols,
                "pgv_f8_quantize: bad extents %lld x %lld (row stride %lld)", (long long)rows, (long long)cols, (long long)ldx);
  PGV_CHECK_ARG((q == nullptr) == (scale == nullptr) && (qt == nullptr) == (scale_t == nullptr),
                "pgv_f8_quantize: bytes and scales come together");
  PGV_CHECK_ARG(q || qt || colsum, "pgv_f8_quantize: nothing to write");
  PGV_CHECK_ARG(((uintptr_t)q % 16) == 0 && ((uintptr_t)qt % 16) == 0, "pgv_f8_quantize: outputs must be 16-byte aligned");
  PGV_CHECK_ARG(pgv_cdiv(rows, F8B) * pgv_cdiv(cols, F8B) <= (1ll << 24), "pgv_f8_quantize: matrix too large");
  if (rows == 0 || cols == 0) {
    PGV_CHECK_ARG(!colsum || cols == 0, "pgv_f8_quantize: column sums of an empty matrix");
    return PGV_OK;
  }
  PGV_CHECK_ARG(x != nullptr, "pgv_f8_quantize: null input");
  if (colsum && (!workspace || workspace_bytes < pgv_f8_quantize_workspace(rows, cols))) {
    pgv_set_error("pgv_f8_quantize: column sums need a workspace of %lld bytes", (long long)pgv_f8_quantize_workspace(rows, cols));
    return PGV_E_WORKSPACE;
  }
  float* part = colsum ? (float*)workspace : nullptr;
  hipStream_t st = pgv_stream(stream);
#define PGV_CALL(T, FMT) \
  launch<T, FMT>((const T*)x, rows, cols, ldx, block, (uint8_t*)q, scale, (uint8_t*)qt, scale_t, colsum, part, st)
  if (fmt == PGV_F8_E4M3)
    return dtype == PGV_DT_F32 ? PGV_CALL(float, PGV_F8_E4M3) : dtype == PGV_DT_BF16 ? PGV_CALL(__bf16, PGV_F8_E4M3) : PGV_CALL(_Float16, PGV_F8_E4M3);
  return dtype == PGV_DT_F32 ? PGV_CALL(float, PGV_F8_E5M2) : dtype == PGV_DT_BF16 ? PGV_CALL(__bf16, PGV_F8_E5M2) : PGV_CALL(_Float16, PGV_F8_E5M2);
#undef PGV_CALL
}
