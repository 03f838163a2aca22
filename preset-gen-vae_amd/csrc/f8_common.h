// Shared helpers of the 8-bit (OCP e4m3 / e5m2) operand kernels: element types, conversion, the scale of a block.
#pragma once
#include <atomic>
#include "pgv_common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int F8B = PGV_F8_BLOCK;           // values per block along the reduction

template <int FMT>
__device__ __forceinline__ constexpr float f8_max() {
  return FMT == PGV_F8_E4M3 ? 448.f : 57344.f;
}

// Four scaled values -> four bytes, round to nearest even (v_cvt_pk_fp8_f32 / v_cvt_pk_bf8_f32: OCP formats on gfx950,
// checked byte by byte against the CPU's rounding in tests/test_gpu_fp8.py).
template <int FMT>
__device__ __forceinline__ int f8_pack4(float a, float b, float c, float d) {
  int r = 0;
  if constexpr (FMT == PGV_F8_E4M3) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return r;
}

// Block maxima travel as the bits of |x|: for non-negative floats the integer order is the float order with NaN above
// infinity, so one integer maximum also carries "this block holds a NaN or an infinity".
__device__ __forceinline__ uint32_t f8_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int CTRL>
__device__ __forceinline__ uint32_t f8_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
// maximum over a row of 16 lanes, in every lane of it
__device__ __forceinline__ uint32_t f8_max16(uint32_t v) {
  v = max(v, f8_dpp<0xB1>(v));    // quad_perm [1,0,3,2]
  v = max(v, f8_dpp<0x4E>(v));    // quad_perm [2,3,0,1]
  v = max(v, f8_dpp<0x141>(v));   // row_half_mirror
  v = max(v, f8_dpp<0x140>(v));   // row_mirror
  return v;
}

// scale = amax / F and inv = F / amax, amax at least 2^-100 (an empty block keeps finite factors and bytes of zero); a
// block that is not finite gets NaN for both, so whatever reads it shows it.  Both quotients are correctly rounded - the
// stored pair is the definition, not an approximation of it: a quotient from a correctly rounded reciprocal plus one residual
// step is (Markstein), and all 2^23 mantissas were compared with IEEE division.  15 instructions against 24.
template <int FMT>
__device__ __forceinline__ void f8_scale(uint32_t bits, float& scale, float& inv) {
  constexpr float F = f8_max<FMT>(), RF = 1.f / F;
  const float a = fmaxf(__uint_as_float(bits), 0x1p-100f);
  const float q = a * RF;
  float s = fmaf(fmaf(-q, F, a), RF, q);
  const float m = __builtin_amdgcn_frexp_mantf(a);   // [0.5, 1): its reciprocal cannot leave the normal range
  const float y0 = __builtin_amdgcn_rcpf(m);
  const float y = fmaf(fmaf(-m, y0, 1.f), y0, y0);
  const float t = F * y;
  float v = __builtin_amdgcn_ldexpf(fmaf(fmaf(-t, m, F), y, t), -__builtin_amdgcn_frexp_expf(a));
  const bool bad = bits >= 0x7f800000u;
  scale = bad ? __uint_as_float(0x7fc00000u) : s;
  inv = bad ? __uint_as_float(0x7fc00000u) : v;
}

// a vector at an address that is a multiple of AL bytes only
template <typename V, int AL>
struct __attribute__((packed, aligned(AL), may_alias)) at_align {
  V v;
};

// 8 consecutive values as floats, of which the first n exist (0 beyond).  VEC: p is 16-byte aligned; otherwise whole pieces are
// the same loads at the alignment of a value.
template <int AL, typename T>
__device__ __forceinline__ void f8_load8_vec(const T* __restrict__ p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const at_align<f32x4, AL>* q = reinterpret_cast<const at_align<f32x4, AL>*>(p);
    const f32x4 a = q[0].v, b = q[1].v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 a = reinterpret_cast<const at_align<t8, AL>*>(p)->v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void f8_load8(const T* __restrict__ p, int n, float (&v)[8]) {
  if (n >= 8) {
    f8_load8_vec<VEC ? 16 : (int)sizeof(T)>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}

// one value of the output type, rounded once
__device__ __forceinline__ void f8_store(void* out, int dt, int64_t i, float v) {
  if (dt == PGV_DT_F32)
    reinterpret_cast<float*>(out)[i] = v;
  else if (dt == PGV_DT_BF16)
    reinterpret_cast<__bf16*>(out)[i] = (__bf16)v;
  else
    reinterpret_cast<_Float16*>(out)[i] = (_Float16)v;
}
// four neighbours, at any multiple of a value
__device__ __forceinline__ void f8_store4(void* out, int dt, int64_t i, f32x4 v) {
  if (dt == PGV_DT_F32) {
    reinterpret_cast<at_align<f32x4, 4>*>(reinterpret_cast<float*>(out) + i)->v = v;
  } else if (dt == PGV_DT_BF16) {
    bf16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (__bf16)v[j];
    reinterpret_cast<at_align<bf16x4, 2>*>(reinterpret_cast<__bf16*>(out) + i)->v = o;
  } else {
    f16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (_Float16)v[j];
    reinterpret_cast<at_align<f16x4, 2>*>(reinterpret_cast<_Float16*>(out) + i)->v = o;
  }
}

// Raises a kernel's dynamic LDS limit, once per device (`done`: the kernel's own bit set of devices).
static inline int f8_allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done, const char* who) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e == hipSuccess && (done.load(std::memory_order_relaxed) & bit)) return PGV_OK;
  if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    pgv_set_error("%s: %d bytes of LDS refused: %s", who, bytes, hipGetErrorString(e));
    return PGV_E_LAUNCH;
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return PGV_OK;
}

static inline int f8_dt_size(int dt) { return dt == PGV_DT_F32 ? 4 : 2; }
static inline bool f8_dt_ok(int dt) { return dt == PGV_DT_F32 || dt == PGV_DT_BF16 || dt == PGV_DT_F16; }
