// What the kernels of the paged 8-bit cache share: entry types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "stof_ptx.cuh"

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

// A cap whose inverse and multiples stay inside fp32: scores capped to 1e-30 are all alike, and 1e30 caps none that are told apart
inline float usable_cap(float cap) { return cap > 0.f ? (cap < 1e-30f ? 1e-30f : cap > 1e30f ? 1e30f : cap) : 0.f; }

// A finite bias stays finite in units of log2: keys masked by fp32's lowest value are still visible, and a row that sees no others is a softmax
// over them (those beyond 2.3e38 count as alike).  A NaN stays.
__device__ __forceinline__ float finite_or_nan(float x) {
    float y;
    asm("{\n\t.reg .f32 a;\n\tmax.NaN.f32 a, %1, 0fFF7FFFFF;\n\tmin.NaN.f32 %0, a, 0f7F7FFFFF;\n\t}" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x to a unit in the last place
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh(u) = 1 - 2 / (1 + e^(2u)), which is off by 1e-7: of the value only where that is not small.  Up to 0.35 an odd polynomial, off by 2.9e-6 of
// the value (weighted least squares moved towards the minimax one; a cap of 1e6 beside scores of 1 would leave them no digits otherwise).
__device__ __forceinline__ float tanh_near_zero(float u) {
    const float w = u * u;
    return u * fmaf(w, fmaf(w, 0.1239503026008606f, -0.33290955424308777f), 0.9999971389770508f);
}
__device__ __forceinline__ float tanh_any(float u) {
    const float far = fmaf(-2.f, fast_reciprocal(1.f + fast_exp2(u * 2.8853900817779268f)), 1.f);
    return fabsf(u) <= 0.35f ? tanh_near_zero(u) : far;
}

template <bool E4M3>
constexpr float entry_max() { return E4M3 ? 448.0f : 127.0f; }

// round(x * inv) of four numbers as entries
template <bool E4M3>
__device__ __forceinline__ uint32_t quantise4(float2 x, float2 y, float inv) {
    x.x *= inv;
    x.y *= inv;
    y.x *= inv;
    y.y *= inv;
    if constexpr (E4M3) {
        uint32_t w;
        asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\tmov.b32 %0, {a, b};\n\t}"
            : "=r"(w) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
        return w;
    } else {
        // next to 1.5 * 2^23 the numbers are integers: the sum is rounded to one, its low byte is the entry (a conversion takes four times as long)
        auto whole = [](float v) { return __float_as_uint(fminf(fmaxf(v, -127.f), 127.f) + 12582912.f); };
        return __byte_perm(__byte_perm(whole(x.x), whole(x.y), 0x0040), __byte_perm(whole(y.x), whole(y.y), 0x0040), 0x5410);
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
