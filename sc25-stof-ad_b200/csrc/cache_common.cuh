// What the kernels of the paged 8-bit cache share: entry types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace stof {

// Two entries (the low 16 bits of `w`) as fp16 numbers; both types' entries are exact in fp16.
template <bool E4M3>
__device__ __forceinline__ uint32_t entries_to_half2(uint32_t w);
template <>
__device__ __forceinline__ uint32_t entries_to_half2<true>(uint32_t w) {
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(w));
    return h;
}
// int8: 1024 + (entry + 128) is the fp16 number with the biased byte as its low mantissa bits
template <>
__device__ __forceinline__ uint32_t entries_to_half2<false>(uint32_t w) {
    const uint32_t biased = __byte_perm(w ^ 0x8080u, 0x64646464u, 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool E4M3>
constexpr float entry_max() { return E4M3 ? 448.0f : 127.0f; }

// round(a * inv), round(b * inv) as two entries in the low 16 bits
template <bool E4M3>
__device__ __forceinline__ uint32_t quantise2(float a, float b, float inv) {
    const float most = entry_max<E4M3>();
    a *= inv;
    b *= inv;
    if constexpr (E4M3) {
        return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    } else {
        const int x = __float2int_rn(fminf(fmaxf(a, -most), most)), y = __float2int_rn(fminf(fmaxf(b, -most), most));
        return (static_cast<uint32_t>(x) & 0xFFu) | ((static_cast<uint32_t>(y) & 0xFFu) << 8);
    }
}

template <bool BF16>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

}  // namespace stof
