// Device helpers of the kernels that write e4m3 values with block scales.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

namespace tb200 {

constexpr uint32_t kSfAtom = 512;            // scale factors of 128 rows x one K block (block-scaled MMA)

// four e4m3 bytes, round-to-nearest, saturating
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// byte offset of row r's four slice bytes inside a scale atom
__host__ __device__ __forceinline__ uint32_t sf_row_offset(int r) { return static_cast<uint32_t>((r & 31) * 16 + (r >> 5) * 4); }

// Smallest power of two s with amax / s <= 448, as its UE8M0 byte (s = 2^(byte - 127)), and 1 / s.
__device__ __forceinline__ uint32_t pow2_scale(float amax, float* inv) {
    int e = 0;
    if (amax > 0.f) {
        const uint32_t bits = __float_as_uint(amax * (1.0f / 448.0f));
        e = static_cast<int>((bits >> 23) & 0xFF) - 127 + ((bits & 0x7FFFFFu) != 0u ? 1 : 0);
        e = max(-126, min(e, 126));
    }
    *inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    return static_cast<uint32_t>(e + 127);
}

// The same without the rounding of the product: the power of two s that a kept activation is divided by (s and 1 / s are
// returned as floats).  448 = 1.75 * 2^8, so the fraction of amax alone decides.  x / s is then exact, and so is q * s in fp32 and bf16.
__device__ __forceinline__ float2 exact_pow2_scale(float amax) {
    int e = 0;
    if (amax > 0.f) {
        const uint32_t bits = __float_as_uint(amax);
        e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
        e = max(-126, min(e, 126));
    }
    return make_float2(__uint_as_float(static_cast<uint32_t>(127 + e) << 23), __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
}

// eight e4m3 bytes -> floats
__device__ __forceinline__ void unpack_e4m3x8(uint2 q, float2 (&f)[4]) {
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        f[i] = __half22float2(*reinterpret_cast<const __half2*>(&h));
    }
}

}  // namespace tb200
