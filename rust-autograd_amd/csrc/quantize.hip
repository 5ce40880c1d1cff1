// f32 arrays rounded to e4m3 with a power-of-two scale per block of 128, along their rows, along their columns (the
// result is then the transposed array), or both from one pass over the input.
#include "e4m3.h"

namespace ag {

// Along the rows.  32 lanes hold one block of 128 elements, a quad each: its largest magnitude is a maximum over the
// half wave, and the block leaves as 32 x 4 bytes = one 128-byte line.  Blocks are independent, so the kernel is one
// stream, bound by HBM: 4 bytes in, 1 byte and 1/128 out per element; 16384 x 8192 117 us (5.8 TB/s).  Block columns
// nb..scale_pitch are padding: scale 1, no data.
constexpr int kRowsPerThread = 4;

__global__ __launch_bounds__(256) void quantize_rows_kernel(const float *__restrict__ x, long long ldx, int cols, unsigned char *__restrict__ q,
                                                            unsigned char *__restrict__ scales, unsigned nb, unsigned nbp, unsigned items)
{
    const unsigned lane = threadIdx.x & 31u;
    const unsigned first = (blockIdx.x * 8u + (threadIdx.x >> 5)) * kRowsPerThread;
    quad_t v[kRowsPerThread];
    unsigned row[kRowsPerThread], b[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const unsigned item = first + i;
        row[i] = item / nbp;
        b[i] = item - row[i] * nbp;
        v[i] = quad_t{0.f, 0.f, 0.f, 0.f};
        if (item < items && b[i] < nb) v[i] = load_quad(x + row[i] * ldx, (long long)b[i] * kE4m3Block + lane * 4, cols);
    }
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        unsigned sb;
        const unsigned bytes = round_block(v[i], &sb);
        if (first + i >= items) continue;
        if (b[i] < nb) *reinterpret_cast<unsigned *>(q + ((size_t)row[i] * nb + b[i]) * kE4m3Block + lane * 4) = bytes;
        if (lane == 0) scales[(size_t)row[i] * nbp + b[i]] = (unsigned char)sb;
    }
}

// Along the columns, and along the rows too where `q` is given: one 128 x 128 tile per block.  Thread (g, lane) of 8 x 32
// holds the quads of 16 consecutive rows (g * 16 ..) at columns lane * 4: a row's block maximum is one over the half wave,
// a column's one over the thread's rows and then over the 8 groups through LDS.  The 16 values that a thread rounds for a
// column are 16 consecutive bytes of the transposed array; they pass through LDS so that each column leaves as one
// 128-byte line.  (LDS pitch 144 = 128 + 16: the 16-byte pieces of a thread's four columns fall on different banks.)
// 16384 x 8192: 164 us both ways (4.9 TB/s of 6 bytes an element; one way after the other 117 + 140), 8192 x 4096 42 us.
// With the half wave's maxima exchanged through LDS and each value tested for being finite the arithmetic bound it: 199
// and 54 us.
__global__ __launch_bounds__(256) void quantize_tile_kernel(const float *__restrict__ x, long long ldx, int rows, int cols,
                                                            unsigned char *__restrict__ q, unsigned char *__restrict__ scales,
                                                            unsigned char *__restrict__ qt, unsigned char *__restrict__ scales_t, unsigned nb,
                                                            unsigned nbp, unsigned mb, unsigned mbp, unsigned first)
{
    constexpr int kPitch = kE4m3Block + 16;
    __shared__ __attribute__((aligned(16))) unsigned colmax[8][kE4m3Block];
    __shared__ __attribute__((aligned(16))) unsigned char turned[kE4m3Block * kPitch];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const unsigned tile = first + blockIdx.x, tb = tile % nb, tm = tile / nb;  // block column, block row
    const long long m0 = (long long)tm * kE4m3Block + g * 16;
    const long long c0 = (long long)tb * kE4m3Block;
    quad_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        v[i] = quad_t{0.f, 0.f, 0.f, 0.f};
        if (m0 + i < rows) v[i] = load_quad(x + (m0 + i) * ldx, c0 + lane * 4, cols);
    }
    unsigned top[4];  // of this thread's columns
    auto column_maxima = [&](auto magnitude_of) {
        unsigned cm[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) cm[j] = max(cm[j], magnitude_of(v[i][j]));
        *reinterpret_cast<uint4 *>(&colmax[g][lane * 4]) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) top[j] = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint4 c = *reinterpret_cast<const uint4 *>(&colmax[k][lane * 4]);
            top[0] = max(top[0], c.x);
            top[1] = max(top[1], c.y);
            top[2] = max(top[2], c.z);
            top[3] = max(top[3], c.w);
        }
    };
    column_maxima([](float x) { return magnitude(x); });
    // (every thread sees the maxima of its own columns only: the block agrees)
    const bool finite = !__syncthreads_or(max(max(top[0], top[1]), max(top[2], top[3])) >= kNotFinite);
    if (!finite) column_maxima([](float x) { return finite_magnitude(x); });
    float inv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned sb = scale_byte(top[j]);
        inv[j] = scale_inverse(sb);
        const long long c = c0 + lane * 4 + j;
        if (g == 0 && c < cols) {
            scales_t[c * mbp + tm] = (unsigned char)sb;
            if (tm == mb - 1)
                for (unsigned k = mb; k < mbp; ++k) scales_t[c * mbp + k] = 127;
        }
    }
    auto turn = [&](auto round) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 w;
            w.x = round(quad_t{v[0][j], v[1][j], v[2][j], v[3][j]}, inv[j]);
            w.y = round(quad_t{v[4][j], v[5][j], v[6][j], v[7][j]}, inv[j]);
            w.z = round(quad_t{v[8][j], v[9][j], v[10][j], v[11][j]}, inv[j]);
            w.w = round(quad_t{v[12][j], v[13][j], v[14][j], v[15][j]}, inv[j]);
            *reinterpret_cast<uint4 *>(turned + (lane * 4 + j) * kPitch + g * 16) = w;
        }
    };
    if (finite) turn([](quad_t x, float s) { return round_finite(x, s); });
    else turn([](quad_t x, float s) { return round_any(x, s); });
    if (q) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            unsigned sb;
            const unsigned bytes = round_block(v[i], &sb);
            if (m0 + i >= rows) continue;
            *reinterpret_cast<unsigned *>(q + ((size_t)(m0 + i) * nb + tb) * kE4m3Block + lane * 4) = bytes;
            if (lane == 0) {
                scales[(size_t)(m0 + i) * nbp + tb] = (unsigned char)sb;
                if (tb == nb - 1)
                    for (unsigned k = nb; k < nbp; ++k) scales[(size_t)(m0 + i) * nbp + k] = 127;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int piece = i * 256 + threadIdx.x, c = piece >> 3, part = piece & 7;
        if (c0 + c < cols)
            *reinterpret_cast<uint4 *>(qt + ((size_t)(c0 + c) * mb + tm) * kE4m3Block + part * 16) =
                *reinterpret_cast<const uint4 *>(turned + c * kPitch + part * 16);
    }
}

ag_status_t quantize_e4m3(const char *who, hipStream_t st, const float *x, long long ldx, int rows, int cols, unsigned char *q, unsigned char *scales,
                          unsigned char *qt, unsigned char *scales_t)
{
    if (rows == 0 || cols == 0) return AG_OK;
    const unsigned nb = (unsigned)(e4m3_pitch(cols) / kE4m3Block), nbp = (unsigned)e4m3_scale_pitch(cols);
    if (!qt) {
        // 8 threads to an item; rows as many at a time as a launch holds (a row has at most 2^24 items)
        const unsigned per = 8u * kRowsPerThread, most = (unsigned)(kMaxThreadsX / 8 - per) / nbp;
        for (unsigned r = 0; r < (unsigned)rows; r += most) {
            const unsigned items = ((unsigned)rows - r < most ? (unsigned)rows - r : most) * nbp;
            hipLaunchKernelGGL(quantize_rows_kernel, dim3((items + per - 1) / per), dim3(256), 0, st, x + r * ldx, ldx, cols,
                               q + (size_t)r * nb * kE4m3Block, scales + (size_t)r * nbp, nb, nbp, items);
        }
    } else {
        const unsigned mb = (unsigned)(e4m3_pitch(rows) / kE4m3Block), mbp = (unsigned)e4m3_scale_pitch(rows);
        const unsigned long long tiles = (unsigned long long)nb * mb, most = kMaxGridX;
        AG_REQUIRE(tiles < (1ull << 32) - most, AG_ERR_INVALID_DIMS, "%s: too many blocks (%llu)", who, tiles);
        for (unsigned long long t = 0; t < tiles; t += most)
            hipLaunchKernelGGL(quantize_tile_kernel, dim3((unsigned)(tiles - t < most ? tiles - t : most)), dim3(256), 0, st, x, ldx, rows, cols, q,
                               scales, qt, scales_t, nb, nbp, mb, mbp, (unsigned)t);
    }
    return check_launch(who);
}

}  // namespace ag

using namespace ag;

extern "C" size_t ag_e4m3_pitch(int n) { return n > 0 ? e4m3_pitch(n) : 0; }
extern "C" size_t ag_e4m3_scale_pitch(int n) { return n > 0 ? e4m3_scale_pitch(n) : 0; }

extern "C" ag_status_t ag_quantize_e4m3_f32(ag_stream_t stream, const float *x, int ldx, int rows, int cols, uint8_t *q, uint8_t *scales,
                                            uint8_t *qt, uint8_t *scales_t)
{
    AG_REQUIRE(rows >= 0 && cols >= 0, AG_ERR_INVALID_DIMS, "quantize_e4m3: negative extent (%d x %d)", rows, cols);
    AG_REQUIRE(ldx >= cols, AG_ERR_INCOMPATIBLE_SHAPE, "quantize_e4m3: ldx (%d) is less than a row of %d elements", ldx, cols);
    if (rows == 0 || cols == 0) return AG_OK;
    AG_REQUIRE(x, AG_ERR_INVALID_DIMS, "quantize_e4m3: null pointer");
    AG_REQUIRE((q != nullptr) == (scales != nullptr) && (qt != nullptr) == (scales_t != nullptr), AG_ERR_INVALID_DIMS,
               "quantize_e4m3: values and scales of an orientation go together");
    AG_REQUIRE(q || qt, AG_ERR_INVALID_DIMS, "quantize_e4m3: no output");
    AG_REQUIRE(aligned16(q) && aligned16(qt), AG_ERR_INVALID_DIMS, "quantize_e4m3: 8-bit outputs must be 16-byte aligned");
    return quantize_e4m3("quantize_e4m3", as_stream(stream), x, ldx, rows, cols, q, scales, qt, scales_t);
}
