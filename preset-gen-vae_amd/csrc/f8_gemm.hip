// Products of block-scaled 8-bit operands (pgv_f8_matmul, pgv_f8_linear):
//   C[m][n] = sum over blocks b of 128  sa[m][b] sb[n][b] * sum_{k in b} a[m][k] b[n][k]   (+ bias[n])
// on v_mfma_f32_16x16x128_f8f6f4: ONE instruction is one block of the reduction for a 16 x 16 tile, so a partial product leaves
// the matrix pipe exactly where its scales change; it is scaled in fp32 on the vector pipe (one fma per element and block
// against 32 matrix cycles per instruction) and summed in fp32.  The second factor's rows (n) are the instruction's rows and
// the first factor's (m) its columns: a lane then owns ONE m - its scale is one register - and four neighbouring n - one store.
// The order of k inside a block is free as long as both operands use the same: every lane reads 32 consecutive bytes.
//
// Three kernels:
//   skinny  few rows (m): bound by reading b once.  b goes from memory straight into the fragment registers, the reduction is
//           spread over the 8 waves of a workgroup and over workgroups, the partial sums meet in LDS.  The fused form also
//           quantises the rows of a.
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

// first of n things that part k of `parts` takes (32-bit: n parts < 2^31 here, a 64-bit division is 100 instructions)
__device__ __forceinline__ int split_at(int n, int k, int parts) { return parts == 1 ? k * n : (int)((unsigned)n * (unsigned)k / (unsigned)parts); }

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

// lanes of a wave have exchanged data through LDS: what they wrote before is seen after (the LDS serves a wave in order; this
// keeps the compiler's order too)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// T = uint8_t: a is 8-bit rows of format FA; else its values are quantised here (e4m3), by every wave for its own blocks: 16
// lanes x 8 values make a block, four blocks of a row at a time, and the bytes change lanes through LDS (a lane of the matrix
// instruction takes 32 neighbours).  No barrier: a wave reads what it wrote.  For one row that is 16 times less work than
// quantising in the fragment layout, where 15 of 16 rows are none.
// MF tiles of 16 x 16 per wave; U blocks of the reduction are requested before the first is used: a wave has few of them, so
// their latencies must overlap.
template <typename T, int FA, bool F32, bool VEC, int MF, int U>
__global__ __launch_bounds__(64 * SW) void skinny_kernel(skinny_args p) {
  constexpr bool Q = sizeof(T) == 1;
  static_assert(Q || (MF == 1 && U == 4), "the fused form holds 16 rows and four blocks");
  constexpr int ROW = 128 + 16;                     // bytes of a row of the exchange image: 16-byte pieces of 8 rows in 8 banks
  constexpr int XCH = Q ? 0 : U * (16 * ROW + 64);  // a wave's image: U blocks of 16 rows, U x 16 scales
  constexpr int SUM = MF * 256 * (int)sizeof(float);
  __shared__ __attribute__((aligned(16))) uint8_t lds[SW * (XCH > SUM ? XCH : SUM)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, split = blockIdx.z;
  const int kb0 = split_at(p.Kb, split, p.splits), kb1 = split_at(p.Kb, split + 1, p.splits);
  const int64_t Kp = (int64_t)p.Kb * F8B;
  const uint8_t* bp = p.b + min(n0 + l16, p.N - 1) * Kp + g * 32;
  const float* sbp = p.sb + (int64_t)(n0 / F8B) * p.Kb;
  uint8_t* img = lds + wave * XCH;
  float* img_s = reinterpret_cast<float*>(img + U * 16 * ROW);
  f32x4 acc[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) acc[i] = {0.f, 0.f, 0.f, 0.f};
  for (int kbase = kb0 + wave; kbase < kb1; kbase += SW * U) {
    i32x8 b8[U], a8[U][Q ? MF : 1];
    float sb[U], sa[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a block past the end is read as the last one and takes no part)
      const int kb = min(kbase + u * SW, kb1 - 1);
      const i32x4* s = reinterpret_cast<const i32x4*>(bp + (int64_t)kb * F8B);
      b8[u] = cat8(s[0], s[1]);
      sb[u] = sbp[kb];
      if constexpr (Q)
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          const int mc = min(16 * i + l16, p.M - 1);
          const i32x4* t = reinterpret_cast<const i32x4*>((const uint8_t*)p.a + mc * Kp + (int64_t)kb * F8B + g * 32);
          a8[u][i] = cat8(t[0], t[1]);
          sa[u][i] = p.sa[(int64_t)kb * p.M + mc];
        }
    }
    if constexpr (!Q) {
      const int k = min(kbase + g * SW, kb1 - 1) * F8B + l16 * 8;
      const T* x = (const T*)p.a + k;
#pragma unroll 2
      for (int m = 0; m < p.M; ++m) {
        float v[8], sc, inv;
        f8_load8<VEC>(x + m * p.lda, p.K - k, v);
        uint32_t t = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) t = max(t, f8_abs_bits(v[j]));
        f8_scale<PGV_F8_E4M3>(f8_max16(t), sc, inv);
        i32x2 o;
        o.x = f8_pack4<PGV_F8_E4M3>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        o.y = f8_pack4<PGV_F8_E4M3>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *reinterpret_cast<i32x2*>(img + (g * 16 + m) * ROW + l16 * 8) = o;
        if (l16 == 0) img_s[g * 16 + m] = sc;
      }
      wave_sync();
      // (lanes of rows that are none read whatever the image holds: their columns of the product are not stored)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const i32x4* t = reinterpret_cast<const i32x4*>(img + (u * 16 + l16) * ROW + g * 32);
        a8[u][0] = cat8(t[0], t[1]);
        sa[u][0] = img_s[u * 16 + l16];
      }
      wave_sync();   // (the next blocks go into the same image)
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kbase + u * SW >= kb1) break;
      const frag<F32> bf = make_frag<PGV_F8_E4M3, F32>(b8[u]);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const f32x4 d = mfma128<FA, F32>(bf, make_frag<FA, F32>(a8[u][i]));
        const float s = sa[u][i] * sb[u];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(d[j], s, acc[i][j]);
      }
    }
  }
  // the waves' sums meet: image [wave][tile][m 16][n 16]
  if constexpr (!Q) __syncthreads();   // (over the exchange images)
  float* sum = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < MF; ++i) *reinterpret_cast<f32x4*>(&sum[((wave * MF + i) * 16 + l16) * 16 + 4 * g]) = acc[i];
  __syncthreads();
  for (int e = tid; e < MF * 256; e += 64 * SW) {
    const int m = e >> 4, n = n0 + (e & 15);
    if (m >= p.M || n >= p.N) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < SW; ++w) s += sum[w * MF * 256 + e];
    const int64_t o = (int64_t)m * p.N + n;
    if (p.splits > 1)
      p.part[(int64_t)split * p.M * p.N + o] = s;
    else
      f8_store(p.out, p.out_dt, o, s + (p.bias ? p.bias[n] : 0.f));
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

// From memory into LDS, 16 or 4 bytes per lane: destination m0 + 16 (4) * lane.  Inline asm: the compiler orders every later
// LDS read behind the builtin's load with vmcnt(0), which would serialise the stages in flight with the stage being
// multiplied; the kernel counts its own loads (they are the only vector memory operations of the loop) and waits by hand before
// the barrier that publishes a stage.  No register is written.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_16(i32x4 rsrc, unsigned lds, unsigned voff, unsigned soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}
__device__ __forceinline__ void dma_4(i32x4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

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

// Which tile a workgroup takes.  Consecutive workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own: an XCD
// gets a contiguous run of tiles, in bands of 4 tile columns (n) and down the rows (m) within a band, so that the 32 tiles it
// works on at a time share 8 panels of a and 4 of b.
__device__ __forceinline__ void tile_of(const tile_args& p, int wg, int& tm, int& tn) {
  const int total = p.tiles_m * p.tiles_n, per = total >> 3, extra = total & 7, xcd = wg & 7, idx = wg >> 3;
  const int t = xcd * per + min(xcd, extra) + idx;   // (workgroup wg exists only if idx < per + (xcd < extra))
  const int band = 4 * p.tiles_m, b = t / band, r = t - b * band, width = min(4, p.tiles_n - 4 * b);
  tm = r / width;
  tn = 4 * b + (r - tm * width);
}

// A stage in LDS is rows of 128 bytes (BM of a, BN of b), then 256 bytes of scales per wave.  The 16-byte piece c of row r sits
// at piece c ^ (r & 7) ^ (r >> 3 & 1), so that the 16 rows of a fragment read (same c) fall into different halves of different
// banks (without the last term: 3.3 conflict cycles per read, the product 3 % slower); LDS-DMA writes lane by lane, so the
// permutation is applied to the address each lane fetches from.  S stages: S - 1 are in flight or complete while
// one is multiplied.  Every wave issues PW + 1 loads per stage: its pieces of 8 rows, and one of the scales.
template <int BM, int BN, int WM, int WN, int S, bool BROW, int FA, bool F32>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, (BM / WM) * (BN / WN) == 4 ? 2 : 1) void tile_kernel(tile_args p) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, MF = WM / 16, NF = WN / 16;
  constexpr int ROWS = (BM + BN) * F8B, STAGE = ROWS + NW * 256, PIECES = (BM + BN) / 8, PW = PIECES / NW;
  static_assert(PIECES % NW == 0, "every wave fills as many pieces");
  static_assert(BM / 64 + BN / 64 <= NW && BN % 64 == 0 && WN <= F8B && F8B % WN == 0, "one load of scales per wave");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int split = blockIdx.y;
  int tm, tn;
  tile_of(p, blockIdx.x, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int wm = (wave / NWN) * WM, wn = (wave % NWN) * WN;
  const int kb0 = split_at(p.Kb, split, p.splits), kb1 = split_at(p.Kb, split + 1, p.splits);
  const uint32_t Kp = (uint32_t)p.Kb * F8B;
  const int rows_a = min(BM, p.M - m0), rows_b = min(BN, p.N - n0);
  const i32x4 rsrc_a = make_rsrc(p.a + (int64_t)m0 * Kp, rows_a * Kp), rsrc_b = make_rsrc(p.b + (int64_t)n0 * Kp, rows_b * Kp);
  // (the row is in the checked part of the address: a row beyond the matrix is beyond the descriptor by itself, whatever K)
  unsigned voff[PW];
#pragma unroll
  for (int j = 0; j < PW; ++j) {
    const int piece = wave * PW + j;
    voff[j] = ((unsigned)(piece < BM / 8 ? piece : piece - BM / 8) * 8u + (unsigned)(lane >> 3)) * Kp +
              (unsigned)(((lane & 7) ^ (lane >> 3) ^ (piece & 1)) * 16);
  }
  // scales: waves 0 .. BM/64 - 1 fetch sa of 64 rows each, the following ones sb of 64 rows each (or the tiles' sb, one lane
  // each); waves with neither fetch nothing (an empty descriptor), so that all count alike
  const float* sp;
  int sstep, svalid;
  unsigned svoff = (unsigned)lane * 4u;
  if (wave < BM / 64) {
    sp = p.sa + (int64_t)kb0 * p.M + m0 + wave * 64;
    sstep = p.M;
    svalid = min(64, max(0, p.M - m0 - wave * 64)) * 4;
  } else if (BROW) {
    const int w = wave - BM / 64;
    sp = p.sb + (int64_t)kb0 * p.N + n0 + w * 64;
    sstep = p.N;
    svalid = w < BN / 64 ? min(64, max(0, p.N - n0 - w * 64)) * 4 : 0;
  } else {
    constexpr int T = BN > F8B ? BN / F8B : 1;
    sp = p.sb + (int64_t)(n0 / F8B) * p.Kb + kb0;
    sstep = 1;
    const int have = min(T, (p.N - n0 + F8B - 1) / F8B);
    svalid = wave == BM / 64 ? ((have - 1) * p.Kb + 1) * 4 : 0;
    svoff = lane < have ? (unsigned)lane * (unsigned)p.Kb * 4u : 0xfffffff0u;
  }
  const unsigned lds0 = lds_addr(lds8);
  auto fill = [&](int kb, int stage) {
    const unsigned base = lds0 + (unsigned)stage * STAGE;
#pragma unroll
    for (int j = 0; j < PW; ++j)
      dma_16(wave * PW + j < BM / 8 ? rsrc_a : rsrc_b, base + (unsigned)(wave * PW + j) * 1024u, voff[j], (unsigned)kb * F8B);
    dma_4(make_rsrc(sp + (int64_t)(kb - kb0) * sstep, (uint32_t)svalid), base + ROWS + (unsigned)wave * 256u, svoff);
  };
  f32x4 acc[NF][MF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[f][i] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (kb0 + s < kb1) fill(kb0 + s, s);
  int stage = 0;
  for (int kb = kb0; kb < kb1; ++kb) {
    if (kb + S - 2 < kb1)
      vm_wait<(S - 2) * (PW + 1)>();
    else
      vm_wait<0>();
    lds_barrier();   // stage kb is complete, and nobody reads stage kb - 1 any more
    if (kb + S - 1 < kb1) fill(kb + S - 1, stage == 0 ? S - 1 : stage - 1);
    const uint8_t* A = lds8 + stage * STAGE;
    const uint8_t* B = A + BM * F8B;
    const float* sA = reinterpret_cast<const float*>(A + ROWS) + wm + l16;
    const float* sB = reinterpret_cast<const float*>(A + ROWS) + BM;
    frag<F32> bf[NF];
    f32x4 sbr[BROW ? NF : 1];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const uint8_t* row = B + (wn + 16 * f + l16) * F8B;
      bf[f] = make_frag<PGV_F8_E4M3, F32>(cat8(*reinterpret_cast<const i32x4*>(row + ((2 * g) ^ (l16 & 7) ^ (l16 >> 3)) * 16),
                                               *reinterpret_cast<const i32x4*>(row + ((2 * g + 1) ^ (l16 & 7) ^ (l16 >> 3)) * 16)));
      if constexpr (BROW) sbr[f] = *reinterpret_cast<const f32x4*>(sB + wn + 16 * f + 4 * g);
    }
    const float sbt = BROW ? 1.f : sB[wn / F8B];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const uint8_t* row = A + (wm + 16 * i + l16) * F8B;
      const frag<F32> af = make_frag<FA, F32>(cat8(*reinterpret_cast<const i32x4*>(row + ((2 * g) ^ (l16 & 7) ^ (l16 >> 3)) * 16),
                                                   *reinterpret_cast<const i32x4*>(row + ((2 * g + 1) ^ (l16 & 7) ^ (l16 >> 3)) * 16)));
      const float s = sA[16 * i] * sbt;
      f32x4 d[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) d[f] = mfma128<FA, F32>(bf[f], af);
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[f][i][j] = fmaf(d[f][j], BROW ? s * sbr[BROW ? f : 0][j] : s, acc[f][i][j]);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
  }
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
      if (n + 4 <= p.N)
        f8_store4(out, dt, o, v);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) f8_store(out, dt, o + j, v[j]);
    }
  }
}

template <int BM, int BN, int WM, int WN, int S, bool BROW, int FA, bool F32>
int launch_tile(tile_args p, hipStream_t st) {
  p.tiles_m = (int)pgv_cdiv(p.M, BM);
  p.tiles_n = (int)pgv_cdiv(p.N, BN);
  constexpr int threads = (BM / WM) * (BN / WN) * 64, lds = S * ((BM + BN) * F8B + threads * 4);
  auto k = tile_kernel<BM, BN, WM, WN, S, BROW, FA, F32>;
  static std::atomic<uint64_t> done{0};
  const int rc = f8_allow_lds((const void*)k, lds, done, "pgv_f8_matmul");
  if (rc != PGV_OK) return rc;
  k<<<dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits), threads, lds, st>>>(p);
  return PGV_OK;
}

template <typename T, int FA, bool F32, bool VEC, int MF, int U>
void launch_skinny(const skinny_args& p, hipStream_t st) {
  skinny_kernel<T, FA, F32, VEC, MF, U><<<dim3((unsigned)pgv_cdiv(p.N, 16), 1, (unsigned)p.splits), 64 * SW, 0, st>>>(p);
}

// ---- which kernel, and how the reduction is split: a function of the sizes alone -------------------------------------------
struct plan {
  bool skinny;
  int mf;      // skinny: tiles of 16 rows
  int tile;    // tile: 256, 128 or 64 rows and columns
  int splits;
};

// Tile sizes (8 waves of 128 x 64, 8 of 32 x 64, 4 of 32 x 32): the larger ones read their operands less often and are faster
// per workgroup slot - 4096 cubed into bfloat16: 73 / 83 / 130 us - but fill the device later - 2048 cubed: 38 / 19 / 24 us,
// 1024 x 1024 x 8192: 110 / 50 / 28 us - and a lone workgroup per CU does not hide its first and last blocks - 1024 x 25024 x 256
// into float32: 41 / 33 / 47 us.  256: one workgroup per CU, 3.5 times the work of a 128 one at its rate; 128 and 64:
// two per CU.
// Skinny: b is read by 16 rows at a time and a by every workgroup; from 17 rows on the 64 x 64 tiles take over where there are
// enough of them (64 x 16384 x 4096: 18 us against 40; 64 x 4096 x 4096: 15 against 14).
// Splits of the reduction: only while workgroups are missing, and with 12 blocks at least each - a join costs 4 us and its
// reads (256 x 1024 x 25024 into float32: 124 us unsplit, 31 us with 8 splits; 100 x 4096 x 4096: 15.8 us unsplit, 15.6 with 2);
// skinny from 17 instructions per wave on, with 8 each (37 x 1024 x 24576: 45 us unsplit, 16.7 with 8; 17 x 2048 x 8192: 11 us
// unsplit, 13.5 with 2).
plan make_plan(int64_t M, int64_t N, int64_t Kb, int b_block) {
  plan q = {};
  q.skinny = b_block == PGV_F8_TILES && (M <= 16 || (M <= 64 && N <= 8192));
  int64_t wgs, most;
  if (q.skinny) {
    q.mf = (int)pgv_cdiv(M, 16);
    wgs = pgv_cdiv(N, 16);
    const int64_t work = pgv_cdiv(Kb, SW) * q.mf;   // instructions of a wave
    most = work <= 16 ? 1 : pgv_cdiv(work, 8) < Kb / (2 * SW) ? pgv_cdiv(work, 8) : Kb / (2 * SW);
  } else {
    const int64_t t256 = pgv_cdiv(M, 256) * pgv_cdiv(N, 256), t128 = pgv_cdiv(M, 128) * pgv_cdiv(N, 128);
    q.tile = t128 < 256 ? 64 : Kb >= 8 && 7 * pgv_cdiv(t256, 256) <= 4 * pgv_cdiv(t128, 512) ? 256 : 128;
    wgs = pgv_cdiv(M, q.tile) * pgv_cdiv(N, q.tile);
    most = Kb / 12;
  }
  const int64_t s = wgs >= 256 ? 1 : 512 / wgs;
  q.splits = (int)(s < 1 || most < 1 ? 1 : s > most ? most : s);
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
      launch_skinny<uint8_t, FA, F32, true, 1, 4>(p, st);
    else if (pl.mf == 2)
      launch_skinny<uint8_t, FA, F32, true, 2, 4>(p, st);
    else if (pl.mf == 3)
      launch_skinny<uint8_t, FA, F32, true, 3, 3>(p, st);
    else
      launch_skinny<uint8_t, FA, F32, true, 4, 2>(p, st);
  } else {
    tile_args p = {(int)M, (int)N, Kb, pl.splits, 0, 0, (const uint8_t*)a, sa, (const uint8_t*)b, sb, bias, out, out_dt, part};
#define PGV_TL(...) (b_block == PGV_F8_ROWS ? launch_tile<__VA_ARGS__, true, FA, F32>(p, st) : launch_tile<__VA_ARGS__, false, FA, F32>(p, st))
    const int rc = pl.tile == 256 ? PGV_TL(256, 256, 128, 64, 2) : pl.tile == 128 ? PGV_TL(128, 128, 32, 64, 2) : PGV_TL(64, 64, 32, 32, 4);
#undef PGV_TL
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

// How many rows the skinny kernel quantises by itself: every workgroup repeats that work for its 16 columns (8 rows x 16384 x
// 4096: 21 us, as much as in two launches; 16 rows: 29 against 23).
static constexpr int64_t FUSED_ROWS = 8;

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
#define PGV_SK2(T, F32) (vec ? launch_skinny<T, 0, F32, true, 1, 4>(p, st) : launch_skinny<T, 0, F32, false, 1, 4>(p, st))
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
