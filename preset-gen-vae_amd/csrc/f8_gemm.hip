// Products of block-scaled 8-bit operands (pgv_f8_matmul, pgv_f8_linear):
//   C[m][n] = sum over blocks b of 128  sa[m][b] sb[n][b] * sum_{k in b} a[m][k] b[n][k]   (+ bias[n])
// on v_mfma_f32_16x16x128_f8f6f4: ONE instruction is one block of the reduction for a 16 x 16 tile, so a partial product leaves
// the matrix pipe exactly where its scales change; it is scaled in fp32 on the vector pipe (one fma per element and block
// against 32 matrix cycles per instruction) and summed in fp32.  The second factor's rows (n) are the instruction's rows and
// the first factor's (m) its columns: a lane then owns ONE m - its scale is one register - and four neighbouring n - one store.
// The order of k inside a block is free as long as both operands use the same: every lane reads 32 consecutive bytes.
//
// Three kernels:
//   skinny  few rows (m): bound by reading b once.  No LDS on the way in: b goes from memory straight into the fragment
//           registers, the reduction is spread over the 8 waves of a workgroup and over workgroups, the partial sums meet in
//           LDS.  The fused form also quantises the rows of a in registers: a lane's 32 values of a block are in its
//           fragment, the block's maximum is two shuffles away.
//   tile    everything else: BM x BN x 128-byte stages in LDS, filled by LDS-DMA, double buffered.
//   join    adds the fp32 partial results of a reduction that was split over workgroups, in the order of the splits.
#include "f8_common.h"

namespace {

// ---- one block of the reduction for a 16 x 16 tile ------------------------------------------------------------------------
// F32 = false: v_mfma_f32_16x16x128_f8f6f4.  Its sum of 128 products is not a 32-bit one: against 64 bits the results are off
// by 1.4e-5 (e4m3) and 1.1e-5 (e5m2) of their norm, and v_mfma_f32_16x16x32_fp8_fp8 gives the same values.  That is a
// hundredth of what rounding to bfloat16 costs and less than a tenth of what float16 does, so it serves the 16-bit outputs.
// F32 = true (float32 outputs): the bytes are widened to bfloat16, exactly, and multiplied by v_mfma_f32_16x16x32_bf16, whose
// sums are 32-bit ones (1e-7): twice the matrix cycles, and 16 conversions per fragment.
template <bool F32>
struct frag {
  i32x8 v;
};
template <>
struct frag<true> {
  bf16x8 v[4];
};

template <int FMT, bool F32>
__device__ __forceinline__ frag<F32> make_frag(i32x8 x) {
  frag<F32> r;
  if constexpr (!F32) {
    r.v = x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x2 lo = FMT == PGV_F8_E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + h], 1.f, false)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x[2 * i + h], 1.f, false);
        const bf16x2 hi = FMT == PGV_F8_E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + h], 1.f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x[2 * i + h], 1.f, true);
        r.v[i][4 * h] = lo[0], r.v[i][4 * h + 1] = lo[1], r.v[i][4 * h + 2] = hi[0], r.v[i][4 * h + 3] = hi[1];
      }
    }
  }
  return r;
}

// cbsz / blgp select the formats of the instruction's first / second operand (0 e4m3, 1 e5m2); b is always e4m3
template <int FA, bool F32>
__device__ __forceinline__ f32x4 mfma128(const frag<F32>& b_rows, const frag<F32>& a_cols) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
  if constexpr (!F32) {
    d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b_rows.v, a_cols.v, d, 0, FA, 0, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b_rows.v[i], a_cols.v[i], d, 0, 0, 0);
  }
  return d;
}

__device__ __forceinline__ i32x8 cat8(i32x4 lo, i32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// ---- skinny -------------------------------------------------------------------------------------------------------------
constexpr int SW = 8;   // waves per workgroup

struct skinny_args {
  int M, N, K, Kb, splits;
  const void* a;          // 8-bit rows [M][Kp], or (fused) the values [M][lda]
  int64_t lda;
  const float* sa;        // [Kb][M] (8-bit rows)
  const uint8_t* b;       // [N][Kp]
  const float* sb;        // [ceil(N/128)][Kb]
  const float* bias;
  void* out;
  int out_dt;
  float* part;            // [splits][M][N] when splits > 1
};

// 32 consecutive values of a row, as they lie in memory (VEC: 16-byte aligned), then as 32 bytes + their block's scale
template <typename T>
struct raw32 {
  T v[32];
};
template <typename T, bool VEC>
__device__ __forceinline__ raw32<T> load32(const T* __restrict__ p, int n) {
  raw32<T> r;
  constexpr int E = 16 / sizeof(T);
  typedef T te __attribute__((ext_vector_type(E)));
  if (VEC && n >= 32) {
#pragma unroll
    for (int i = 0; i < 32 / E; ++i) {
      const te t = reinterpret_cast<const te*>(p)[i];
#pragma unroll
      for (int j = 0; j < E; ++j) r.v[i * E + j] = t[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ i32x8 quant_frag(const raw32<T>& r, float& scale) {
  i32x8 f;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, f8_abs_bits((float)r.v[i]));
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  float inv;
  f8_scale<PGV_F8_E4M3>(m, scale, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = f8_pack4<PGV_F8_E4M3>((float)r.v[4 * i] * inv, (float)r.v[4 * i + 1] * inv, (float)r.v[4 * i + 2] * inv,
                                 (float)r.v[4 * i + 3] * inv);
  return f;
}

// T = uint8_t: a is 8-bit rows of format FA; else its values are quantised here (e4m3).  MF x NF tiles of 16 x 16 per wave;
// U blocks of the reduction are requested before the first is used: a wave has few of them, so their latencies must overlap.
template <typename T, int FA, bool F32, bool VEC, int MF, int NF, int U>
__global__ __launch_bounds__(64 * SW) void skinny_kernel(skinny_args p) {
  constexpr bool Q = sizeof(T) == 1;
  constexpr int GRP = NF * MF < 4 ? NF * MF : 4;   // tiles that meet in LDS at a time
  __shared__ __attribute__((aligned(16))) float lds[SW * GRP * 256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NF), m0 = blockIdx.y * (16 * MF), split = blockIdx.z;
  const int kb0 = (int)((int64_t)p.Kb * split / p.splits), kb1 = (int)((int64_t)p.Kb * (split + 1) / p.splits);
  const int64_t Kp = (int64_t)p.Kb * F8B;
  const uint8_t* bp[NF];
  const float* sbp[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = min(n0 + 16 * f + l16, p.N - 1);
    bp[f] = p.b + n * Kp + g * 32;
    sbp[f] = p.sb + (int64_t)(min(n0 + 16 * f, p.N - 1) / F8B) * p.Kb;
  }
  f32x4 acc[NF][MF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[f][i] = {0.f, 0.f, 0.f, 0.f};
  for (int kbase = kb0 + wave; kbase < kb1; kbase += SW * U) {
    i32x8 b8[U][NF], a8[U][Q ? MF : 1];
    raw32<T> av[U][Q ? 1 : MF];
    float sb[U][NF], sa[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a block past the end is read as the last one and takes no part)
      const int kb = min(kbase + u * SW, kb1 - 1);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const i32x4* s = reinterpret_cast<const i32x4*>(bp[f] + (int64_t)kb * F8B);
        b8[u][f] = cat8(s[0], s[1]);
        sb[u][f] = sbp[f][kb];
      }
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const int mc = min(m0 + 16 * i + l16, p.M - 1);
        if constexpr (Q) {
          const i32x4* s = reinterpret_cast<const i32x4*>((const uint8_t*)p.a + mc * Kp + (int64_t)kb * F8B + g * 32);
          a8[u][i] = cat8(s[0], s[1]);
          sa[u][i] = p.sa[(int64_t)kb * p.M + mc];
        } else {
          const int k = kb * F8B + g * 32;
          av[u][i] = load32<T, VEC>((const T*)p.a + mc * p.lda + k, p.K - k);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kbase + u * SW >= kb1) break;
      frag<F32> bf[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) bf[f] = make_frag<PGV_F8_E4M3, F32>(b8[u][f]);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        frag<F32> af;
        if constexpr (Q)
          af = make_frag<FA, F32>(a8[u][i]);
        else
          af = make_frag<PGV_F8_E4M3, F32>(quant_frag(av[u][i], sa[u][i]));
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const f32x4 d = mfma128<FA, F32>(bf[f], af);
          const float s = sa[u][i] * sb[u][f];
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[f][i][j] = fmaf(d[j], s, acc[f][i][j]);
        }
      }
    }
  }
  // the waves' sums meet, GRP tiles at a time: image [wave][tile][m 16][n 16]
#pragma unroll
  for (int t0 = 0; t0 < NF * MF; t0 += GRP) {
    if (t0) __syncthreads();
#pragma unroll
    for (int t = 0; t < GRP; ++t) {
      const int f = (t0 + t) / MF, i = (t0 + t) % MF;
      if (t0 + t < NF * MF) *reinterpret_cast<f32x4*>(&lds[((wave * GRP + t) * 16 + l16) * 16 + 4 * g]) = acc[f][i];
    }
    __syncthreads();
    for (int e = tid; e < GRP * 256; e += 64 * SW) {
      const int t = e >> 8, f = (t0 + t) / MF, i = (t0 + t) % MF;
      const int m = m0 + 16 * i + ((e >> 4) & 15), n = n0 + 16 * f + (e & 15);
      if (t0 + t < NF * MF && m < p.M && n < p.N) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < SW; ++w) s += lds[w * GRP * 256 + e];
        const int64_t o = (int64_t)m * p.N + n;
        if (p.splits > 1)
          p.part[(int64_t)split * p.M * p.N + o] = s;
        else
          f8_store(p.out, p.out_dt, o, s + (p.bias ? p.bias[n] : 0.f));
      }
    }
  }
}

// ---- join ---------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int64_t MN, int N,
                                                   const float* __restrict__ bias, void* out, int out_dt) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= MN) return;
  float s = 0.f;
  for (int z = 0; z < splits; ++z) s += part[z * MN + i];
  f8_store(out, out_dt, i, s + (bias ? bias[i % N] : 0.f));
}

// ---- tile ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p;
}

// descriptor of "the bytes [p, p + bytes)": reads beyond it fetch nothing
__device__ __forceinline__ i32x4 make_rsrc(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;
  i32x4 r;
  r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xFFFF);
  r.z = __builtin_amdgcn_readfirstlane((int)bytes);
  r.w = 0x00020000;
  return r;
}

// 1 KB from memory into LDS: 64 lanes x 16 bytes, destination m0 + 16 * lane.  Inline asm: the compiler orders every later LDS
// read behind the builtin's load with vmcnt(0), which would serialise the stage in flight with the stage being multiplied; the
// kernel waits by hand before the barrier that publishes a stage.  No register is written.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_1k(i32x4 rsrc, unsigned lds, unsigned voff, unsigned soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void dma_wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

struct tile_args {
  int M, N, Kb, splits, tiles_m, tiles_n;
  const uint8_t* a;   // [M][Kp]
  const float* sa;    // [Kb][M]
  const uint8_t* b;   // [N][Kp]
  const float* sb;    // tiles: [ceil(N/128)][Kb]; rows: [Kb][N]
  const float* bias;
  void* out;
  int out_dt;
  float* part;
};

// A stage in LDS is rows of 128 bytes; the 16-byte piece c of row r sits at piece c ^ (r & 7), so that the eight rows of a
// fragment read (same c) fall into different banks.  LDS-DMA writes lane by lane, so the permutation is applied to the
// address each lane fetches from.
template <int BM, int BN, int WM, int WN, bool BROW, int FA, bool F32>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void tile_kernel(tile_args p) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, MF = WM / 16, NF = WN / 16;
  constexpr int STAGE = (BM + BN) * F8B, PIECES = (BM + BN) / 8;
  static_assert(PIECES % NW == 0 && (BM / 8) % (PIECES / NW) == 0, "a wave fills pieces of one operand only");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x, split = blockIdx.y;
  const int m0 = (tile % p.tiles_m) * BM, n0 = (tile / p.tiles_m) * BN;
  const int wm = (wave / NWN) * WM, wn = (wave % NWN) * WN;
  const int kb0 = (int)((int64_t)p.Kb * split / p.splits), kb1 = (int)((int64_t)p.Kb * (split + 1) / p.splits);
  const uint32_t Kp = (uint32_t)p.Kb * F8B;
  // this wave's share of a stage: pieces of 8 rows
  constexpr int PW = PIECES / NW;
  const bool fills_a = wave * PW < BM / 8;
  const int piece0 = fills_a ? wave * PW : wave * PW - BM / 8;
  const int rows_a = min(BM, p.M - m0), rows_b = min(BN, p.N - n0);
  const i32x4 rsrc = fills_a ? make_rsrc(p.a + (int64_t)m0 * Kp, rows_a * Kp) : make_rsrc(p.b + (int64_t)n0 * Kp, rows_b * Kp);
  // (the row is in the checked part of the address: a row beyond the matrix is beyond the descriptor by itself, whatever K)
  unsigned voff[PW];
#pragma unroll
  for (int j = 0; j < PW; ++j)
    voff[j] = ((unsigned)(piece0 + j) * 8u + (unsigned)(lane >> 3)) * Kp + (unsigned)(((lane & 7) ^ (lane >> 3)) * 16);
  const unsigned dst0 = lds_addr(lds8) + (unsigned)(wave * PW) * 1024u;
  auto fill = [&](int kb, int stage) {
#pragma unroll
    for (int j = 0; j < PW; ++j)
      dma_1k(rsrc, dst0 + stage * STAGE + j * 1024u, voff[j], (unsigned)kb * F8B);
  };
  // scales: sa one float per lane and column tile; sb one per wave (tiles) or four per lane and row tile (rows)
  const float* sap[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) sap[i] = p.sa + min(m0 + wm + 16 * i + l16, p.M - 1);
  f32x4 acc[NF][MF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[f][i] = {0.f, 0.f, 0.f, 0.f};
  float sav[MF], sbt = 0.f, sbr[BROW ? NF : 1][4];
  auto scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < MF; ++i) sav[i] = sap[i][(int64_t)kb * p.M];
    if constexpr (BROW) {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j) sbr[f][j] = p.sb[(int64_t)kb * p.N + min(n0 + wn + 16 * f + 4 * g + j, p.N - 1)];
    } else {
      sbt = p.sb[(int64_t)(min(n0 + wn, p.N - 1) / F8B) * p.Kb + kb];
    }
  };
  if (kb0 < kb1) {
    fill(kb0, 0);
    dma_wait_all();
  }
  __syncthreads();
  for (int kb = kb0; kb < kb1; ++kb) {
    const int stage = (kb - kb0) & 1;
    scales(kb);
    if (kb + 1 < kb1) fill(kb + 1, stage ^ 1);
    const uint8_t* A = lds8 + stage * STAGE;
    const uint8_t* B = A + BM * F8B;
    frag<F32> bf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const uint8_t* row = B + (wn + 16 * f + l16) * F8B;
      bf[f] = make_frag<PGV_F8_E4M3, F32>(cat8(*reinterpret_cast<const i32x4*>(row + ((2 * g) ^ (l16 & 7)) * 16),
                                               *reinterpret_cast<const i32x4*>(row + ((2 * g + 1) ^ (l16 & 7)) * 16)));
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const uint8_t* row = A + (wm + 16 * i + l16) * F8B;
      const frag<F32> af = make_frag<FA, F32>(cat8(*reinterpret_cast<const i32x4*>(row + ((2 * g) ^ (l16 & 7)) * 16),
                                                   *reinterpret_cast<const i32x4*>(row + ((2 * g + 1) ^ (l16 & 7)) * 16)));
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const f32x4 d = mfma128<FA, F32>(bf[f], af);
        if constexpr (BROW) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[f][i][j] = fmaf(d[j], sav[i] * sbr[f][j], acc[f][i][j]);
        } else {
          const float s = sav[i] * sbt;
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[f][i][j] = fmaf(d[j], s, acc[f][i][j]);
        }
      }
    }
    dma_wait_all();
    __syncthreads();
  }
  const bool quad = (p.N & 3) == 0;
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = n0 + wn + 16 * f + 4 * g;
    f32x4 bv = {0.f, 0.f, 0.f, 0.f};
    if (p.bias && p.splits == 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) bv[j] = n + j < p.N ? p.bias[n + j] : 0.f;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int m = m0 + wm + 16 * i + l16;
      if (m >= p.M || n >= p.N) continue;
      const int64_t o = (int64_t)m * p.N + n;
      void* out = p.splits > 1 ? (void*)(p.part + (int64_t)split * p.M * p.N) : p.out;
      const int dt = p.splits > 1 ? PGV_DT_F32 : p.out_dt;
      const f32x4 v = acc[f][i] + bv;
      if (quad)
        f8_store4(out, dt, o, v);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) f8_store(out, dt, o + j, v[j]);
    }
  }
}

template <int BM, int BN, int WM, int WN, bool BROW, int FA, bool F32>
int launch_tile(tile_args p, hipStream_t st) {
  p.tiles_m = (int)pgv_cdiv(p.M, BM);
  p.tiles_n = (int)pgv_cdiv(p.N, BN);
  constexpr int lds = 2 * (BM + BN) * F8B;
  auto k = tile_kernel<BM, BN, WM, WN, BROW, FA, F32>;
  static const hipError_t once = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (once != hipSuccess) {
    pgv_set_error("pgv_f8_matmul: %d bytes of LDS refused: %s", lds, hipGetErrorString(once));
    return PGV_E_LAUNCH;
  }
  k<<<dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits), (BM / WM) * (BN / WN) * 64, lds, st>>>(p);
  return PGV_OK;
}

template <typename T, int FA, bool F32, bool VEC, int MF, int NF, int U>
void launch_skinny(const skinny_args& p, hipStream_t st) {
  skinny_kernel<T, FA, F32, VEC, MF, NF, U>
      <<<dim3((unsigned)pgv_cdiv(p.N, 16 * NF), (unsigned)pgv_cdiv(p.M, 16 * MF), (unsigned)p.splits), 64 * SW, 0, st>>>(p);
}

// ---- which kernel, and how the reduction is split: a function of the sizes alone -------------------------------------------
struct plan {
  bool skinny;
  int mf, nf;       // skinny
  int splits;
};

plan make_plan(int64_t M, int64_t N, int64_t Kb, int b_block) {
  plan q = {};
  q.skinny = M <= 64 && b_block == PGV_F8_TILES;
  int64_t wgs;
  int64_t most;
  if (q.skinny) {
    q.mf = M <= 16 ? 1 : M <= 32 ? 2 : M <= 48 ? 3 : 4;
    q.nf = 1;
    wgs = pgv_cdiv(N, 16 * q.nf);
    most = Kb / (2 * SW);
  } else {
    wgs = pgv_cdiv(M, 128) * pgv_cdiv(N, 128);
    most = Kb / 4;
  }
  int64_t s = wgs >= 256 ? 1 : 512 / wgs;
  q.splits = (int)(s < 1 ? 1 : s > most ? (most < 1 ? 1 : most) : s);
  return q;
}

int check_shape(const char* who, int64_t M, int64_t N, int64_t K) {
  PGV_CHECK_ARG(M >= 0 && N >= 0 && K >= 0 && M <= PGV_F8_MAX_EXTENT && N <= PGV_F8_MAX_EXTENT && K <= PGV_F8_MAX_K,
                "%s: bad extents M=%lld N=%lld K=%lld", who, (long long)M, (long long)N, (long long)K);
  PGV_CHECK_ARG(pgv_cdiv(M, 128) * pgv_cdiv(N, 128) <= (1ll << 24), "%s: output too large", who);
  return PGV_OK;
}

int run_join(const plan& pl, int64_t M, int64_t N, const float* part, const float* bias, void* out, int out_dt, hipStream_t st) {
  if (pl.splits > 1)
    join_kernel<<<dim3((unsigned)pgv_cdiv(M * N, 256)), 256, 0, st>>>(part, pl.splits, M * N, (int)N, bias, out, out_dt);
  return PGV_OK;
}

template <int FA, bool F32>
int run_matmul(int64_t M, int64_t N, int64_t K, const void* a, const float* sa, const void* b, const float* sb, int b_block,
               const float* bias, void* out, int out_dt, float* part, hipStream_t st) {
  const int Kb = (int)pgv_cdiv(K, F8B);
  const plan pl = make_plan(M, N, Kb, b_block);
  if (pl.skinny) {
    skinny_args p = {(int)M, (int)N, (int)K, Kb, pl.splits, a, 0, sa, (const uint8_t*)b, sb, bias, out, out_dt, part};
    if (pl.mf == 1)
      launch_skinny<uint8_t, FA, F32, true, 1, 1, 4>(p, st);
    else if (pl.mf == 2)
      launch_skinny<uint8_t, FA, F32, true, 2, 1, 4>(p, st);
    else if (pl.mf == 3)
      launch_skinny<uint8_t, FA, F32, true, 3, 1, 3>(p, st);
    else
      launch_skinny<uint8_t, FA, F32, true, 4, 1, 2>(p, st);
  } else {
    tile_args p = {(int)M, (int)N, Kb, pl.splits, 0, 0, (const uint8_t*)a, sa, (const uint8_t*)b, sb, bias, out, out_dt, part};
    const int rc = b_block == PGV_F8_ROWS ? launch_tile<128, 128, 64, 64, true, FA, F32>(p, st) : launch_tile<128, 128, 64, 64, false, FA, F32>(p, st);
    if (rc != PGV_OK) return rc;
  }
  run_join(pl, M, N, part, bias, out, out_dt, st);
  PGV_CHECK_LAUNCH("pgv_f8_matmul");
  return PGV_OK;
}

}  // namespace

extern "C" int64_t pgv_f8_matmul_workspace(int64_t M, int64_t N, int64_t K, int b_block) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const plan pl = make_plan(M, N, pgv_cdiv(K, F8B), b_block);
  return pl.splits > 1 ? 4 * M * N * pl.splits : 0;
}

extern "C" int pgv_f8_matmul(int64_t M, int64_t N, int64_t K, const void* a, const float* a_scale, int a_fmt, const void* b,
                             const float* b_scale, int b_block, const float* bias, void* out, int out_dtype, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const int rc = check_shape("pgv_f8_matmul", M, N, K);
  if (rc != PGV_OK) return rc;
  PGV_CHECK_ARG(a_fmt == PGV_F8_E4M3 || a_fmt == PGV_F8_E5M2, "pgv_f8_matmul: unknown 8-bit format %d", a_fmt);
  PGV_CHECK_ARG(b_block == PGV_F8_ROWS || b_block == PGV_F8_TILES, "pgv_f8_matmul: unknown block kind %d", b_block);
  PGV_CHECK_ARG(f8_dt_ok(out_dtype), "pgv_f8_matmul: unknown output type %d", out_dtype);
  if (M == 0 || N == 0) return PGV_OK;
  PGV_CHECK_ARG(K > 0 && a && a_scale && b && b_scale && out, "pgv_f8_matmul: null operand or empty reduction");
  PGV_CHECK_ARG((uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0 && (uintptr_t)out % 16 == 0,
                "pgv_f8_matmul: operands and output must be 16-byte aligned");
  const int64_t need = pgv_f8_matmul_workspace(M, N, K, b_block);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    pgv_set_error("pgv_f8_matmul: workspace of %lld bytes needed", (long long)need);
    return PGV_E_WORKSPACE;
  }
#define PGV_MM(FA, F32) \
  run_matmul<FA, F32>(M, N, K, a, a_scale, b, b_scale, b_block, bias, out, out_dtype, (float*)workspace, pgv_stream(stream))
  if (out_dtype == PGV_DT_F32) return a_fmt == PGV_F8_E4M3 ? PGV_MM(PGV_F8_E4M3, true) : PGV_MM(PGV_F8_E5M2, true);
  return a_fmt == PGV_F8_E4M3 ? PGV_MM(PGV_F8_E4M3, false) : PGV_MM(PGV_F8_E5M2, false);
#undef PGV_MM
}

// How many rows the skinny kernel quantises by itself: every workgroup repeats that work for its 16 columns.
static constexpr int64_t FUSED_ROWS = 16;

extern "C" int pgv_f8_linear_fused(int64_t M, int b_block) { return M <= FUSED_ROWS && b_block == PGV_F8_TILES; }

extern "C" int pgv_f8_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* b, const float* b_scale,
                             int b_block, int64_t N, const float* bias, void* xq, float* x_scale, void* out, int out_dtype,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_shape("pgv_f8_linear", M, N, K);
  if (rc != PGV_OK) return rc;
  if (M == 0 || N == 0) return PGV_OK;
  if (!pgv_f8_linear_fused(M, b_block)) {
    PGV_CHECK_ARG(xq && x_scale, "pgv_f8_linear: %lld rows need buffers for the quantised rows", (long long)M);
    const int rq = pgv_f8_quantize(x, dtype, M, K, ldx, PGV_F8_ROWS, PGV_F8_E4M3, xq, x_scale, nullptr, nullptr, nullptr, nullptr, 0, stream);
    if (rq != PGV_OK) return rq;
    return pgv_f8_matmul(M, N, K, xq, x_scale, PGV_F8_E4M3, b, b_scale, b_block, bias, out, out_dtype, workspace, workspace_bytes, stream);
  }
  PGV_CHECK_ARG(f8_dt_ok(dtype) && f8_dt_ok(out_dtype), "pgv_f8_linear: unknown element type %d / %d", dtype, out_dtype);
  PGV_CHECK_ARG(K > 0 && x && b && b_scale && out && ldx >= K, "pgv_f8_linear: null operand, empty reduction or bad row stride");
  PGV_CHECK_ARG((uintptr_t)b % 16 == 0, "pgv_f8_linear: the weight must be 16-byte aligned");
  const int Kb = (int)pgv_cdiv(K, F8B);
  const plan pl = make_plan(M, N, Kb, b_block);
  const int64_t need = pgv_f8_matmul_workspace(M, N, K, b_block);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    pgv_set_error("pgv_f8_linear: workspace of %lld bytes needed", (long long)need);
    return PGV_E_WORKSPACE;
  }
  hipStream_t st = pgv_stream(stream);
  skinny_args p = {(int)M, (int)N, (int)K, Kb, pl.splits, x, ldx, nullptr, (const uint8_t*)b, b_scale, bias, out, out_dtype, (float*)workspace};
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * f8_dt_size(dtype)) % 16 == 0;
#define PGV_SK2(T, F32) \
  (vec ? launch_skinny<T, 0, F32, true, 1, 1, sizeof(T) == 4 ? 2 : 4>(p, st) : launch_skinny<T, 0, F32, false, 1, 1, 1>(p, st))
#define PGV_SK(T) (out_dtype == PGV_DT_F32 ? PGV_SK2(T, true) : PGV_SK2(T, false))
  if (dtype == PGV_DT_F32)
    PGV_SK(float);
  else if (dtype == PGV_DT_BF16)
    PGV_SK(__bf16);
  else
    PGV_SK(_Float16);
#undef PGV_SK2
#undef PGV_SK
  run_join(pl, M, N, (const float*)workspace, bias, out, out_dtype, st);
  PGV_CHECK_LAUNCH("pgv_f8_linear");
  return PGV_OK;
}
