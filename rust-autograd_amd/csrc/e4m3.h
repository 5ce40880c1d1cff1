// 8-bit operands: float8 e4m3 values (1 sign, 4 exponent, 3 mantissa bits, no infinities, largest 448) with one
// power-of-two scale per row and block of 128 elements along the contraction.  A scale is held as its biased exponent
// (a byte b stands for 2^(b - 127)), which is what the matrix instructions of gfx950 multiply a block by themselves.
#pragma once
#include "ag_internal.h"

namespace ag {

constexpr int kE4m3Block = 128;

inline size_t e4m3_pitch(int n) { return ((size_t)n + kE4m3Block - 1) / kE4m3Block * kE4m3Block; }
inline size_t e4m3_scale_pitch(int n) { return (e4m3_pitch(n) / kE4m3Block + 3) / 4 * 4; }

#if defined(__HIPCC__)
// A quad of floats that need not start on 16 bytes (global loads and stores of 16 bytes take any multiple of 4).
typedef float quad_t __attribute__((ext_vector_type(4)));
typedef float quad_any_t __attribute__((ext_vector_type(4), aligned(4)));

// Elements i..i+3 of a row of n, zeros behind its end.  STREAM: of an array that no cache will hold until it is read again.
template <bool STREAM = false>
__device__ inline quad_t load_quad(const float *row, long long i, long long n)
{
    quad_t v = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= n) {
        const quad_any_t *at = reinterpret_cast<const quad_any_t *>(row + i);
        v = STREAM ? __builtin_nontemporal_load(at) : *at;
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (i + j < n) v[j] = row[i + j];
    }
    return v;
}
template <bool STREAM = false>
__device__ inline void store_quad(float *row, long long i, long long n, quad_t v)
{
    if (i + 4 <= n) {
        quad_any_t *at = reinterpret_cast<quad_any_t *>(row + i);
        if (STREAM) __builtin_nontemporal_store(v, at);
        else *at = v;
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (i + j < n) row[i + j] = v[j];
    }
}

// The bits of |v| where v is finite, 0 where it is not: their integer maximum is that of the finite magnitudes.
__device__ inline unsigned finite_magnitude(float v)
{
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ inline unsigned finite_magnitude(quad_t v)
{
    return max(max(finite_magnitude(v[0]), finite_magnitude(v[1])), max(finite_magnitude(v[2]), finite_magnitude(v[3])));
}

// Biased exponent of the smallest power of two s >= 2^-117 with amax <= 448 s (448 = 1.75 * 2^8), from the bits of amax;
// 1 for a block of zeros.  Integer arithmetic on the exponent field, so there is no rounding to disagree about.  (From 2^-117
// on the smallest value of a block, 2^-9 of its scale, is a normal bf16 number.)
__device__ inline unsigned scale_byte(unsigned amax)
{
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax == 0 ? 127u : (unsigned)max(e, 10);
}
__device__ inline float scale_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Four values times `inv`, rounded to e4m3 (to nearest, ties to even; |v| * inv <= 448).  e4m3 has no infinities: values
// that are not finite become NaN.
__device__ inline unsigned round_e4m3(quad_t v, float inv)
{
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool finite = (__float_as_uint(v[j]) & 0x7fffffffu) < 0x7f800000u;
        s[j] = finite ? v[j] * inv : __uint_as_float(0x7fc00000u);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
    return (unsigned)w;
}

// Maximum over the 32 lanes of a half wave (every lane gets it).
__device__ inline unsigned half_wave_max(unsigned v)
{
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, d, 64));
    return v;
}
#endif

}  // namespace ag
