// The 8-bit paged KV cache: layout, element types and what its kernels share.
//
// codes [pages][2][Hkv][P][128] (K, then V) one byte each, scales f32 [pages][2][Hkv], optional
// sums f32 [pages][Hkv][P]; value = code * scale.  P tokens of one head and side are one run of
// P * 128 bytes with one scale, so a run is the unit of quantisation and of the copies.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace kv8 {

constexpr int kD = 128;

enum Kind { kInt8 = 0, kE4m3 = 1 };

template <int kKind>
__host__ __device__ constexpr float code_max() {
  return kKind == kInt8 ? 127.0f : 448.0f;
}

// Value over its scale -> code, to nearest even within the finite range; NaN -> 0.
template <int kKind>
__device__ __forceinline__ uint32_t encode(float x) {
  x = x == x ? x : 0.f;
  x = fminf(fmaxf(x, -code_max<kKind>()), code_max<kKind>());
  if (kKind == kInt8) return static_cast<uint32_t>(__float2int_rn(x)) & 0xffu;
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
// The four codes of a word as numbers.  int8: a byte with its sign bit flipped, as the low mantissa of
// 2^23, is 2^23 + 128 + code (the integer conversion would take the slow unit).
template <int kKind>
__device__ __forceinline__ void decode4(uint32_t w, float* f) {
  if (kKind == kInt8) {
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 | e)) - 8388736.f;
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 t = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * e)), __NV_E4M3)));
      f[2 * e] = t.x;
      f[2 * e + 1] = t.y;
    }
  }
}

// Host checks shared by the entry points.
inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool valid_cache(int dtype, int64_t num_pages, int Hkv, int D, int page) {
  return (dtype == kInt8 || dtype == kE4m3) && D == kD && Hkv > 0 && Hkv <= 1024 && num_pages > 0 &&
         (page == 16 || page == 32 || page == 64 || page == 128) &&
         // rows of 128 bytes are counted in 32 bits (256 GB of codes)
         num_pages <= 0x7fffffffll / (2ll * Hkv * page);
}

}  // namespace kv8
