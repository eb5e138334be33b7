// What the kernels of the paged 8-bit cache share: entry types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace stof {

// Four entries as fp16 numbers (exact for both types): the first two and the last two.
template <bool E4M3>
__device__ __forceinline__ void entries_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // 1024 + (entry + 128) is the fp16 number with the biased byte as its low mantissa bits
        const uint32_t biased = w ^ 0x80808080u;
        const __half2 off(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(biased, 0x64646464u, 0x4140), b = __byte_perm(biased, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// 1 / x to a unit in the last place
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
