// Device helpers of the microscaled 4-bit format.
//
// A block is 32 neighbouring elements: 16 code bytes (element 2i in the low half of byte i; a code is the sign bit 8 and the
// index of the magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6) and a scale byte s that stands for 2^(s - 127), 255 for NaN. For a block
// whose largest magnitude is a, s = max(0, floor(log2 a) - 2 + 127): the largest element then lies in [4, 8) times the scale,
// and what rounds beyond 6 is held as 6. Scaling by a power of two is exact, so an element is rounded once, to the nearest
// value, ties to the even code; reading back is exact in fp32. gfx950 converts both ways in one instruction for two elements,
// with the scale given as a float of which it takes the exponent bits: s << 23 for every s (0 stands for 2^-127 there, 255
// gives NaN), checked over all codes and scales on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

namespace mg {

typedef float mx_v2f __attribute__((ext_vector_type(2)));
typedef __bf16 mx_v2bf __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float mx4_scale(uint32_t s) { return __uint_as_float(s << 23); }

// The scale byte of a block from the largest of its elements' bit patterns without sign (as integers, so that a NaN or an
// infinity anywhere is seen): a block with one is NaN as a whole.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax) {
    const int s = (int)(amax >> 23) - 2;
    return amax >= 0x7f800000u ? 255u : (uint32_t)(s > 0 ? s : 0);
}

// Eight elements to a word of codes, element e in bits 4e .. 4e + 3.
__device__ __forceinline__ uint32_t mx4_pack8(const float x[8], float scale) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}
__device__ __forceinline__ void mx4_unpack8(uint32_t w, float scale, float x[8]) {
    const mx_v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}

// Eight consecutive elements of a row as floats, and back. Beyond `left` elements: zero, and not stored. Sixteen bytes at a time with
// the element's alignment alone, which global memory takes (2445 fp32 rows of 6371 quantised and read back: element by element
// 71 us).
template <int N>
struct Raw16;
template <>
struct Raw16<2> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2), may_alias));
};
template <>
struct Raw16<4> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4), may_alias));
};
template <class T>
__device__ __forceinline__ void real_load8(const T* p, int left, float x[8]) {
    using R = typename Raw16<sizeof(T)>::type;
    if (left >= 8) {
        constexpr int n = sizeof(T) / 2;
        R r[n];
#pragma unroll
        for (int i = 0; i < n; i++) r[i] = ((const R*)p)[i];
        T t[8];
        __builtin_memcpy(t, r, sizeof(t));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = e < left ? (float)p[e] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void real_store8(T* p, int left, const float x[8]) {
    using R = typename Raw16<sizeof(T)>::type;
    if (left >= 8) {
        constexpr int n = sizeof(T) / 2;
        R r[n];
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = (T)x[e];
        __builtin_memcpy(r, t, sizeof(t));
#pragma unroll
        for (int i = 0; i < n; i++) ((R*)p)[i] = r[i];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) p[e] = (T)x[e];
    }
}

// Four neighbouring elements of a row from floats, `left` of which exist, with the element's alignment alone.
template <class T, class V>
__device__ __forceinline__ void real_store4(T* p, const V& v, int left) {
    typedef uint32_t R4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
    typedef uint32_t R2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
    using R = std::conditional_t<sizeof(T) == 4, R4, R2>;
    T t[4];
#pragma unroll
    for (int r = 0; r < 4; r++) t[r] = (T)v[r];
    if (left >= 4) {
        R w;
        __builtin_memcpy(&w, t, sizeof(t));
        *(R*)p = w;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r < left) p[r] = t[r];
    }
}

// Four lanes hold a block, eight elements each: its scale byte (in all four) and each lane's word of codes.
__device__ __forceinline__ uint32_t mx4_block(const float x[8], uint32_t& s) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    // lanes 1 0 3 2, then 2 3 0 1 of each four
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    s = mx4_scale_byte(m);
    return mx4_pack8(x, mx4_scale(s));
}

// Allows a kernel dynamic LDS above the default limit, once per device.
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& allowed) {
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (allowed.load() & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) allowed |= bit;
    return e;
}

// Calls f with a null pointer of the element type's C++ type.
template <class F>
auto by_real(int type, F&& f) {
    switch (type) {
        case 0: return f((float*)nullptr);
        case 1: return f((_Float16*)nullptr);
        default: return f((__bf16*)nullptr);
    }
}

}  // namespace mg
