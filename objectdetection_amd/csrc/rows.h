// rows.h -- loads, stores and conversions shared by the row operators (rms_norm.hip, f8.hip,
// grad_norm.hip): eight consecutive elements of an fp32, bf16 or fp16 row per lane.
#pragma once
#include "common.h"

typedef _Float16 lcf_h;
typedef __bf16 lcf_b;

// Vector types that promise no more alignment than their elements have.  Rows of an odd width, and
// views into a flat buffer, start anywhere; gfx950 takes 16-byte global accesses at any element's
// address, so one code path serves them all.
typedef float lcf_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short lcf_s8u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned lcf_u2u __attribute__((ext_vector_type(2), aligned(4)));

static inline int lcf_type_size(int code) { return code == LCF_F32 ? 4 : 2; }
static inline bool lcf_is_type(int code) { return code == LCF_F32 || code == LCF_BF16 || code == LCF_F16; }

__device__ __forceinline__ float lcf_to_f32(float v) { return v; }
__device__ __forceinline__ float lcf_to_f32(lcf_b v)
{
    return __uint_as_float((unsigned)__builtin_bit_cast(unsigned short, v) << 16);
}
__device__ __forceinline__ float lcf_to_f32(lcf_h v) { return (float)v; }

// to nearest even, as torch's casts round
template <typename T> __device__ __forceinline__ T lcf_from_f32(float v)
{
    if constexpr (sizeof(T) == 4) return v;
    else return (T)v;
}

template <typename T> __device__ __forceinline__ void lcf_ld8(const T *p, float v[8])
{
    if constexpr (sizeof(T) == 4) {
        const lcf_f4u a = *reinterpret_cast<const lcf_f4u *>(p);
        const lcf_f4u b = *reinterpret_cast<const lcf_f4u *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        const lcf_s8u a = *reinterpret_cast<const lcf_s8u *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned short s = a[i];
            v[i] = lcf_to_f32(__builtin_bit_cast(T, s));
        }
    }
}

template <typename T> __device__ __forceinline__ void lcf_st8(T *p, const float v[8])
{
    if constexpr (sizeof(T) == 4) {
        lcf_f4u a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
        *reinterpret_cast<lcf_f4u *>(p) = a;
        *reinterpret_cast<lcf_f4u *>(p + 4) = b;
    } else {
        lcf_s8u a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = __builtin_bit_cast(unsigned short, lcf_from_f32<T>(v[i]));
        *reinterpret_cast<lcf_s8u *>(p) = a;
    }
}

// columns [col, col + 8) of a row of `width`: zeros behind the end
template <typename T> __device__ __forceinline__ void lcf_ld8_tail(const T *row, int col, int width, float v[8])
{
    if (col + 8 <= width) {
        lcf_ld8(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < width ? lcf_to_f32(row[col + i]) : 0.f;
    }
}

template <typename T> __device__ __forceinline__ void lcf_st8_tail(T *row, int col, int width, const float v[8])
{
    if (col + 8 <= width) {
        lcf_st8(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) row[col + i] = lcf_from_f32<T>(v[i]);
    }
}

// weights of a norm: fp32, bf16 or fp16 by a code that is the same for the whole launch
__device__ __forceinline__ void lcf_ld8_code(const void *p, int code, int col, int width, float v[8])
{
    if (code == LCF_F32) lcf_ld8_tail((const float *)p, col, width, v);
    else if (code == LCF_BF16) lcf_ld8_tail((const lcf_b *)p, col, width, v);
    else lcf_ld8_tail((const lcf_h *)p, col, width, v);
}

// ---- 8-bit form.  A block of 128 values is stored as q = rne(v * 2^-e), with 2^e the smallest
// power of two that brings the block's largest finite magnitude inside the format: its maximum is
// 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2), so with amax = m * 2^x, 1 <= m < 2, e is x - 8 (x - 15),
// and one more when m > 1.75.  e is held in [-126, 127] and stored as the E8M0 byte e + 127: the
// scaled MFMA takes that byte as an operand, so scales cost a product no vector instruction, and
// q * 2^e is exact in fp32 and, from e = -124 (e4m3) or -117 (e5m2) on, in bf16: below, the format's least
// values are no bf16 numbers and round to a multiple of 2^-133, bf16's least step.  (At the other end a
// block whose largest magnitude rounds up to 2^128 stands for a number that neither type holds.)  A block
// of zeros has e = 0.
__device__ __forceinline__ int lcf_f8_exponent(float amax, int fmt)
{
    const unsigned u = __float_as_uint(amax);
    if (u == 0) return 0;
    const int e = (int)(u >> 23) - 127 - (fmt == LCF_E4M3 ? 8 : 15) + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float lcf_exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Largest magnitude of N values of a lane, NaN left out (fmax does that by itself).  Infinities do
// not enter a block's scale either, and e4m3 holds none: only where one is found, anywhere in the
// wave (a uniform branch), they are made NaN in place and the others looked through again.
template <int N> __device__ __forceinline__ float lcf_f8_top(float *v)
{
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, __builtin_fabsf(v[i]));
    if (__builtin_expect(__any(top > 3.402823466e38f), 0)) {
        top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (__builtin_fabsf(v[i]) > 3.402823466e38f) v[i] = __uint_as_float(0x7FC00000u);
            top = fmaxf(top, __builtin_fabsf(v[i]));
        }
    }
    return top;
}

// four values, already scaled (finite ones lie inside the format then), to four bytes; NaN stays NaN
__device__ __forceinline__ unsigned lcf_f8_pack4(float a, float b, float c, float d, int fmt)
{
    int r = 0;
    if (fmt == LCF_E4M3) {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    } else {
        r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
    }
    return (unsigned)r;
}

// the largest of the 16 lanes of a row of lanes, in all of them: four rotations on the vector unit
// (a shuffle would go through LDS)
__device__ __forceinline__ float lcf_max16(float v)
{
#define LCF_ROR(n) \
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + n, 0xF, 0xF, false)))
    LCF_ROR(8);
    LCF_ROR(4);
    LCF_ROR(2);
    LCF_ROR(1);
#undef LCF_ROR
    return v;
}
