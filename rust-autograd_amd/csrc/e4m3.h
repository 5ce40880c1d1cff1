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

// The bits of |v|: their integer order is that of the magnitudes, and from kNotFinite on they are an infinity or a NaN.
constexpr unsigned kNotFinite = 0x7f800000u;
__device__ inline unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ inline unsigned magnitude(quad_t v) { return max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3]))); }
// The same with 0 for what is not finite.
__device__ inline unsigned finite_magnitude(float v) { return magnitude(v) < kNotFinite ? magnitude(v) : 0u; }
__device__ inline unsigned finite_magnitude(quad_t v)
{
    return max(max(finite_magnitude(v[0]), finite_magnitude(v[1])), max(finite_magnitude(v[2]), finite_magnitude(v[3])));
}

// Biased exponent of the smallest power of two s >= 2^-117 with amax <= 448 s (448 = 1.75 * 2^8), from the bits of amax;
// 1 for a block of zeros.  Integer arithmetic on the exponent field, so there is no rounding to disagree about.  (From 2^-117
// on the smallest value of a block, 2^-9 of its scale, is a normal bf16 number.  The largest block of f32 has byte 247; its
// elements from 1.9375 * 2^127 on are rounded to 256 * 2^120, which is an infinity in bf16 and f32.)
__device__ inline unsigned scale_byte(unsigned amax)
{
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax == 0 ? 127u : (unsigned)max(e, 10);
}
__device__ inline float scale_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Four finite values times `inv`, rounded to e4m3 (to nearest, ties to even; |v| * inv <= 448).
__device__ inline unsigned round_finite(quad_t v, float inv)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
    return (unsigned)w;
}
// Any four values: e4m3 has no infinities, what is not finite becomes NaN.
__device__ inline unsigned round_any(quad_t v, float inv)
{
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (magnitude(v[j]) >= kNotFinite) v[j] = __uint_as_float(0x7fc00000u);
    return round_finite(v, inv);
}

// Maximum over the 32 lanes of a half wave (every lane gets it): four rotations within the rows of 16 lanes, which cost an
// instruction each, and one exchange between the two rows.
__device__ inline unsigned half_wave_max(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, false));
    return max(v, (unsigned)__builtin_amdgcn_ds_swizzle((int)v, 0x401f));
}

// A block of 128 that the 32 lanes of a half wave hold, a quad each: its scale byte, and the lane's four values.  (All 32
// lanes come here together.  Blocks with infinities or NaN, which take no part in the scale, are gone over twice.)
__device__ inline unsigned round_block(quad_t v, unsigned *byte)
{
    unsigned top = half_wave_max(magnitude(v));
    if (__builtin_expect(top < kNotFinite, 1)) {
        *byte = scale_byte(top);
        return round_finite(v, scale_inverse(*byte));
    }
    top = half_wave_max(finite_magnitude(v));
    *byte = scale_byte(top);
    return round_any(v, scale_inverse(*byte));
}
#endif

}  // namespace ag
