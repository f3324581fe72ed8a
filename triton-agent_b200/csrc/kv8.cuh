// Codes of the 8-bit KV cache: element types and their exact conversions.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

using e4m3_t = __nv_fp8_e4m3;

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

// The codes of w as f16 pairs, exactly: bytes 0 and 2, bytes 1 and 3.  int8: a
// byte with its sign bit flipped, below the exponent of 2^10, is 1024 + 128 +
// code; one packed subtraction takes the rest off.  (The shift of the odd bytes
// as a high multiplication, to relieve the integer pipe, was slower: decode of 64
// sequences 126 -> 144 us.)  e4m3: the hardware conversion, NaN codes included.
template <typename KV>
__device__ __forceinline__ void kv8_pairs(uint32_t w, uint32_t& even, uint32_t& odd) {
  if constexpr (std::is_same<KV, int8_t>::value) {
    const uint32_t e = (w & 0x00ff00ffu) ^ 0x64806480u;
    const uint32_t o = __byte_perm(w ^ 0x80808080u, 0x64646464u, 0x4341);
    const uint32_t off = 0x64806480u;
    const __half2 de = __hsub2(*reinterpret_cast<const __half2*>(&e), *reinterpret_cast<const __half2*>(&off));
    const __half2 d1 = __hsub2(*reinterpret_cast<const __half2*>(&o), *reinterpret_cast<const __half2*>(&off));
    even = *reinterpret_cast<const uint32_t*>(&de);
    odd = *reinterpret_cast<const uint32_t*>(&d1);
  } else {
    const uint32_t p = __byte_perm(w, 0, 0x3120);
    const __half2_raw e = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(p & 0xffffu), __NV_E4M3);
    const __half2_raw o = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(p >> 16), __NV_E4M3);
    even = *reinterpret_cast<const uint32_t*>(&e);
    odd = *reinterpret_cast<const uint32_t*>(&o);
  }
}

// The codes of w in order: bytes 0 and 1, bytes 2 and 3.
template <typename KV>
__device__ __forceinline__ void kv8_in_order(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same<KV, int8_t>::value) {
    uint32_t e, o;
    kv8_pairs<KV>(w, e, o);
    lo = __byte_perm(e, o, 0x5410);
    hi = __byte_perm(e, o, 0x7632);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  }
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
