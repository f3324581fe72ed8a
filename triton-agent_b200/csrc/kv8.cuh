// Codes of the 8-bit KV cache: element types and their exact conversions.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "sm100.cuh"

namespace b200 {

using e4m3_t = __nv_fp8_e4m3;

// 32 bytes of one lane as one store (whole sectors; dst 32-byte aligned).
__device__ __forceinline__ void stg256(void* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Largest code magnitude.
template <typename KV>
__host__ __device__ constexpr float kv8_max() {
  return std::is_same<KV, int8_t>::value ? 127.0f : 448.0f;
}

// Four codes (lowest byte first) as fp32.  int8: a byte with its sign bit
// flipped, placed below the exponent of 2^23, is 2^23 + 128 + code.
template <typename KV>
__device__ __forceinline__ void kv8_to_f32x4(uint32_t w, float* f) {
  if constexpr (std::is_same<KV, int8_t>::value) {
    const uint32_t u = w ^ 0x80808080u;
    f[0] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)) - 8388736.0f;
    f[1] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)) - 8388736.0f;
    f[2] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)) - 8388736.0f;
    f[3] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)) - 8388736.0f;
  } else {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  }
}

// The codes of w as f16 pairs, exactly: bytes 0 and 1, bytes 2 and 3.  int8: a
// byte with its sign bit flipped, below the exponent of 2^10, is 1024 + 128 +
// code; one packed subtraction takes the rest off.  e4m3: the hardware
// conversion, NaN codes included.
template <typename KV>
__device__ __forceinline__ void kv8_in_order(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same<KV, int8_t>::value) {
    const uint32_t u = w ^ 0x80808080u, off = 0x64806480u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&off));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  }
}

// D = A B + C on 16 x 8 x 32 tiles of bytes: A signed codes, B signed or unsigned.
// The first form starts all of D at one word (no register has to be set first).
#define B200_MMA8(TYPES, CLIST, ...)                                                                          \
  asm volatile("mma.sync.aligned.m16n8k32.row.col." TYPES " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " CLIST ";" \
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                               \
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), __VA_ARGS__)
template <bool UB>
__device__ __forceinline__ void mma8_start(int32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                           int32_t c) {
  if constexpr (UB) B200_MMA8("s32.s8.u8.s32", "{%10,%10,%10,%10}", "r"(c));
  else B200_MMA8("s32.s8.s8.s32", "{%10,%10,%10,%10}", "r"(c));
}
template <bool UB>
__device__ __forceinline__ void mma8_add(int32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const int32_t c0 = d[0], c1 = d[1], c2 = d[2], c3 = d[3];
  if constexpr (UB) B200_MMA8("s32.s8.u8.s32", "{%10,%11,%12,%13}", "r"(c0), "r"(c1), "r"(c2), "r"(c3));
  else B200_MMA8("s32.s8.s8.s32", "{%10,%11,%12,%13}", "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
#undef B200_MMA8

// Sums below 2^22 start at the bit pattern of 1.5 * 2^23, whose low bits they
// then count: a value is one exact subtraction, without the conversion pipe.
constexpr int32_t kAccStart = 0x4B400000;
__device__ __forceinline__ void acc_values(int32_t a, int32_t b, float& x, float& y) {
  x = -12582912.0f, y = -12582912.0f;
  sm100::fadd2_acc(x, y, __int_as_float(a), __int_as_float(b));
}

// Two 16 x 16 byte matrices, transposed: lane (r, q) gets rows 4q..4q+3 of
// columns r and r + 8 of the first (lanes 0-15 give its row addresses) and of the second.
__device__ __forceinline__ void ldsm_x2_t8(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// The scales of a key and its value as the attention kernels use them: the
// logit factor ks, log2 vs and 1 / vs.  A value scale below 2^-100 (a slot
// never written holds 0) counts as 2^-100; NaN stays NaN.
__device__ __forceinline__ void kv8_value_scale(float vs, float& lvs, float& ivs) {
  constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(vs) : "f"(kTiny));
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lvs) : "f"(vs));
  asm("rcp.approx.f32 %0, %1;" : "=f"(ivs) : "f"(vs));
}

}  // namespace b200
