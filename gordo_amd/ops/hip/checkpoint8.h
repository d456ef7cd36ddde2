// 8-bit activation codes, shared by the kernels that write and that read them.
//
// 32 consecutive values (the last group of a row may be shorter) share one
// scale, a power of two 2^e with e = max(floor(log2 max|v|) - 6, -126), kept as
// the byte e + 127. code = clamp(rint(v / 2^e), -127, 127). A power of two
// costs up to one of the eight bits against max|v|/127, and buys exactness:
// v / 2^e and code * 2^e are exact in 32 bits, and code * 2^e has at most seven
// significant bits, so it is exact in bf16 and fp16 too and goes into a matrix
// product without a rounding of its own. |code * 2^e - v| <= max|v| / 127, or 2^-127
// where that is more (groups below 2^-120, whose e has no further to go).
// Byte 255: a value of the group was not finite; the whole group restores as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <cstdint>
#include <type_traits>

#define C8_GROUP 32

// ---- element types by storage: unsigned short bits for bf16 / fp16 -----------
struct C8Bf16 {
    typedef unsigned short store;
    static __device__ __forceinline__ float up(store u) { return __uint_as_float((unsigned int)u << 16); }
    static __device__ __forceinline__ store down(float f) {
        union { __bf16 h; unsigned short u; } c;
        c.h = (__bf16)f;
        return c.u;
    }
};
struct C8Fp16 {
    typedef unsigned short store;
    static __device__ __forceinline__ float up(store u) {
        union { unsigned short u; _Float16 h; } c;
        c.u = u;
        return (float)c.h;
    }
    static __device__ __forceinline__ store down(float f) {
        union { _Float16 h; unsigned short u; } c;
        c.h = (_Float16)f;
        return c.u;
    }
};
struct C8Fp32 {
    typedef float store;
    static __device__ __forceinline__ float up(store f) { return f; }
    static __device__ __forceinline__ store down(float f) { return f; }
};

// largest |v| as bits: for finite values the order of the bits is the order of
// the magnitudes, and infinities and NaN lie above them
__device__ __forceinline__ unsigned int c8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// scale byte of a group from the bits of its largest magnitude
__device__ __forceinline__ unsigned int c8_scale(unsigned int top) {
    unsigned int field = top >> 23;
    return field == 255u ? 255u : (field > 7u ? field - 6u : 1u);
}

// 2^-e of a scale byte; 0 for a group that is not finite
__device__ __forceinline__ float c8_inv(unsigned int s) {
    return s == 255u ? 0.f : __uint_as_float((254u - s) << 23);
}

// 2^e of a scale byte; NaN for 255
__device__ __forceinline__ float c8_step(unsigned int s) {
    return s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s << 23);
}

// The code as a byte. v * inv is exact; added to 1.5 * 2^23 it is rounded to the
// nearest integer, ties to even, and its two's complement is in the low bits. In a
// group that is not finite (inv = 0) a code means nothing.
__device__ __forceinline__ unsigned int c8_code_byte(float v, float inv) {
    const float q = __builtin_amdgcn_fmed3f(fmaf(v, inv, 12582912.f), 12582912.f - 127.f, 12582912.f + 127.f);
    return __float_as_uint(q) & 0xffu;
}

// f(integral_constant 0 .. N-1): for where an instruction wants a constant
template <int N, int I = 0, class F>
__device__ __forceinline__ void c8_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        c8_for<N, I + 1>(f);
    }
}

// max over 4 and over 16 neighbouring lanes (DPP: no LDS pass)
__device__ __forceinline__ unsigned int c8_max4(unsigned int m) {
    unsigned int o;
    o = (unsigned int)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true);   // quad_perm 1,0,3,2
    m = m > o ? m : o;
    o = (unsigned int)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true);   // quad_perm 2,3,0,1
    return m > o ? m : o;
}

__device__ __forceinline__ unsigned int c8_max16(unsigned int m) {
    unsigned int o;
    m = c8_max4(m);
    o = (unsigned int)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, true);  // row_half_mirror
    m = m > o ? m : o;
    o = (unsigned int)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, true);  // row_mirror
    return m > o ? m : o;
}
