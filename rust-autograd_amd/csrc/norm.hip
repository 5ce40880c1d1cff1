// Root-mean-square norm of a row, with the addition of a residual in front of it and the rounding to e4m3 behind it in
// the same pass, and its gradient.
//
//   h = x + residual           y = h * r * w,   r = 1 / sqrt(mean(h^2) + eps)
//   gx = r (w gy) - h r^3 / n * sum(w gy h) (+ gh)          gw = sum over rows of gy h r
//
// The sum of squares, r and the two products of y are in 64 bits and y is rounded to f32 once, so that the same row gives
// the same f32 value however the sum is ordered, and the rounding to 8 bits behind it -- where neighbouring values are 6 %
// apart -- does not depend on the launch shape.  The passes are bound by HBM; 64-bit arithmetic is free there.
#include "e4m3.h"

namespace ag {

// Sum over the block, the same value in every thread.  `part`: one double per wave.
template <int T>
__device__ inline double block_sum(double v, double *part)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    if (T == 64) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) s += part[i];
    return s;
}

struct NormArgs {
    const float *x, *residual, *weight;
    float *h, *y, *rstd;
    unsigned char *q, *scales;
    double eps;
    long long n;
    unsigned nb, nbp;
};

__device__ inline quad_t norm_quad(quad_t h, quad_t w, double r)
{
    quad_t y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (float)((double)h[j] * r * (double)w[j]);
    return y;
}
__device__ inline double square_sum(quad_t h, double s)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)h[j], (double)h[j], s);
    return s;
}

// Writes what the quad at element i of a row gives: the f32 value, and its share of the 8-bit block, which the 32 lanes
// of the half wave hold between them (all of them call this together: the maximum runs over the half wave).
__device__ inline void norm_write(const NormArgs &a, size_t row, long long i, quad_t y)
{
    if (a.y) store_quad<true>(a.y + row * a.n, i, a.n, y);
    if (a.q) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j >= a.n) y[j] = 0.f;  // (padding stays zero where r is not finite)
        unsigned sb;
        const unsigned bytes = round_block(y, &sb);
        const long long b = i / kE4m3Block;
        if (b < a.nb) *reinterpret_cast<unsigned *>(a.q + (row * a.nb) * kE4m3Block + i) = bytes;
        if ((threadIdx.x & 31) == 0 && b < a.nbp) a.scales[row * a.nbp + b] = (unsigned char)sb;
    }
}

// One row per T threads, held in registers (Q quads a thread: rows of up to 4 * Q * T elements), so every input is read
// once; T = 64 packs four rows into a block of 256.  Behind the row's end quads are zero: they pad the 8-bit output.
// Bound by HBM: 16384 x 8192 with residual and 8-bit output 270 us (6.4 TB/s; a copy of 4 GiB reaches 4.7; 16 us more
// without streaming stores and loads, 15 with the half wave's maxima exchanged through LDS); one row of 4096 4.8 us.
// Stores stream always (1024 x 4096: 9.7 and 12.5 us), loads from kStreamBytes on, beyond what the last-level cache keeps
// between two kernels (4096 x 4096, whose arrays it does keep: 36 us without, 39 with; 16384 x 4096: 151 and 139).  The
// quads of a thread come in small steps of the row's length: 16384 x 5001 to 8 bits 197 us with 5 quads a thread, 232
// with 8; its gradient, three quads a thread and four, 246 and 257.
template <int T, int Q, bool STREAM>
__global__ __launch_bounds__(T == 64 ? 256 : T) void rms_norm_kernel(NormArgs a, unsigned rows)
{
    __shared__ double part[T / 64];
    const unsigned t = T == 64 ? threadIdx.x & 63u : threadIdx.x;
    const size_t row = T == 64 ? (size_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;  // (whole waves, and only where T == 64, which has no barrier)
    const float *x = a.x + row * a.n;
    const float *res = a.residual ? a.residual + row * a.n : nullptr;
    quad_t h[Q], w[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) h[k] = load_quad<STREAM>(x, (long long)(k * T + t) * 4, a.n);
    if (res) {
        quad_t b[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) b[k] = load_quad<STREAM>(res, (long long)(k * T + t) * 4, a.n);
#pragma unroll
        for (int k = 0; k < Q; ++k) h[k] += b[k];
    }
    // The weight stays in cache.  It is read ahead of the sum, so that one row alone does not wait twice (1 x 8192 4.9 us,
    // behind it 5.7), but for the longest rows, of which it would send dozens of registers to scratch (2048 x 32768 192 us,
    // ahead 264; six go there all the same).
    constexpr bool LATE = T == 1024 && Q == 8;
    if (!LATE)
#pragma unroll
        for (int k = 0; k < Q; ++k) w[k] = load_quad(a.weight, (long long)(k * T + t) * 4, a.n);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < Q; ++k) s = square_sum(h[k], s);
    s = block_sum<T>(s, part);  // (its barrier also orders every read of the row before the writes: outputs may be the inputs)
    const double r = 1.0 / sqrt(s / (double)a.n + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = (float)r;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const long long i = (long long)(k * T + t) * 4;
        if (a.h) store_quad<true>(a.h + row * a.n, i, a.n, h[k]);
        if (LATE) w[k] = load_quad(a.weight, i, a.n);
        norm_write(a, row, i, norm_quad(h[k], w[k], r));
    }
}

// Rows beyond what the registers hold: two passes over the row, the second from cache where it fits.  A thread reads in
// the second pass only what it read (or wrote, as h) in the first, so outputs may be the inputs here too.
constexpr int kLongT = 1024;
__global__ __launch_bounds__(kLongT) void rms_norm_long_kernel(NormArgs a)
{
    __shared__ double part[kLongT / 64];
    const size_t row = blockIdx.x;
    const float *x = a.x + row * a.n;
    const float *res = a.residual ? a.residual + row * a.n : nullptr;
    const long long end = (a.n + kE4m3Block * 4 - 1) / (kE4m3Block * 4) * (kE4m3Block * 4);  // whole groups of four blocks: the scales' padding too
    double s = 0.0;
    for (long long i = (long long)threadIdx.x * 4; i < a.n; i += kLongT * 4) {
        quad_t h = load_quad(x, i, a.n);
        if (res) h += load_quad(res, i, a.n);
        s = square_sum(h, s);
        if (a.h) store_quad(a.h + row * a.n, i, a.n, h);
    }
    s = block_sum<kLongT>(s, part);
    const double r = 1.0 / sqrt(s / (double)a.n + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = (float)r;
    for (long long i = (long long)threadIdx.x * 4; i < end; i += kLongT * 4) {
        quad_t h = load_quad(a.h ? a.h + row * a.n : x, i, a.n);
        if (!a.h && res) h += load_quad(res, i, a.n);
        norm_write(a, row, i, norm_quad(h, load_quad(a.weight, i, a.n), r));
    }
}

// Calls launch(arguments, rows) for the rows, `threads` each, as many at a time as a launch holds.
template <typename F>
static void norm_in_launches(const NormArgs &a, unsigned rows, unsigned threads, F launch)
{
    const unsigned most = (unsigned)(kMaxThreadsX / threads) / 4 * 4;  // (whole blocks of four rows)
    for (unsigned first = 0; first < rows; first += most) {
        NormArgs p = a;
        const size_t cells = (size_t)first * (size_t)a.n;
        p.x += cells;
        if (p.residual) p.residual += cells;
        if (p.h) p.h += cells;
        if (p.y) p.y += cells;
        if (p.rstd) p.rstd += first;
        if (p.q) p.q += (size_t)first * a.nb * kE4m3Block, p.scales += (size_t)first * a.nbp;
        launch(p, rows - first < most ? rows - first : most);
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------
constexpr size_t kStreamBytes = (size_t)256 << 20;  // of one array

struct NormGradArgs {
    const float *h, *weight, *rstd, *gy, *gh;
    float *gx, *partial;  // partial: [blocks that share the rows][n] sums of gw, or null
    long long n;
};

__device__ inline double dot3(quad_t g, quad_t w, quad_t h, double s)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)g[j] * (double)w[j], (double)h[j], s);
    return s;
}
// r w gy - h c + gh, c = sum(w gy h) / n * r^3, rounded to f32 once.  In 64 bits: c is about w gy / h^2 and leaves f32's
// range where the gradient does not (h of 1e20 and gy of 1e-3: c = 1e-43), and so may w gy.
__device__ inline quad_t grad_quad(quad_t h, quad_t w, quad_t g, quad_t gh, double r, double c)
{
    quad_t o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (float)fma(-(double)h[j], c, fma((double)g[j] * (double)w[j], r, (double)gh[j]));
    return o;
}

// A group of T threads walks rows in steps of the number of groups, with the row in registers and its share of gw beside
// it: gw costs one [G][n] array of partial sums, folded in a fixed order below, instead of a second pass over gy and h.
// T = 64: four groups share a block of 256 and add their sums through LDS at the end.  Bound by HBM: 16384 x 4096 with gh
// 190 us, the fold included (5.7 TB/s; without streaming stores and loads 200).
template <int T, int Q, bool STREAM>
__global__ __launch_bounds__(T == 64 ? 256 : T) void rms_norm_grad_kernel(NormGradArgs a, unsigned rows)
{
    constexpr unsigned PER = T == 64 ? 4 : 1;
    __shared__ double part[2][T / 64];
    __shared__ quad_t sums[T == 64 ? 4 : 1][T == 64 ? Q * 64 : 1];
    const unsigned t = T == 64 ? threadIdx.x & 63u : threadIdx.x, group = T == 64 ? threadIdx.x >> 6 : 0;
    quad_t w[Q], acc[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        w[k] = load_quad(a.weight, (long long)(k * T + t) * 4, a.n);
        acc[k] = quad_t{0.f, 0.f, 0.f, 0.f};
    }
    int turn = 0;
    for (size_t row = (size_t)blockIdx.x * PER + group; row < rows; row += (size_t)gridDim.x * PER, turn ^= 1) {
        const float *hr = a.h + row * a.n, *gr = a.gy + row * a.n;
        quad_t h[Q], g[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            h[k] = load_quad<STREAM>(hr, (long long)(k * T + t) * 4, a.n);
            g[k] = load_quad<STREAM>(gr, (long long)(k * T + t) * 4, a.n);
        }
        const float r = a.rstd[row];
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < Q; ++k) s = dot3(g[k], w[k], h[k], s);
        s = block_sum<T>(s, part[turn]);  // (two arrays in turn: the next row's sums do not wait for this row's readers)
        const double c = s / (double)a.n * (double)r * (double)r * (double)r;
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const long long i = (long long)(k * T + t) * 4;
            // The row stays in f32 over the sum; left to itself the compiler keeps what dot3 widened, in twice the registers
            // (2048 x 16384 114 us, widened 174).  Short rows have some to spare, for the weight (200000 x 128 57 us, all in
            // f32 61, all widened 79) or the products (65536 x 512 103, all in f32 106).
            if (T == 64 && Q == 1) asm volatile("" : "+v"(h[k]), "+v"(g[k]));
            else if (T == 64 && Q == 2) asm volatile("" : "+v"(h[k]));
            else asm volatile("" : "+v"(h[k]), "+v"(g[k]), "+v"(w[k]));
            if (a.gx) {
                quad_t gh = {0.f, 0.f, 0.f, 0.f};
                if (a.gh) gh = load_quad<STREAM>(a.gh + row * a.n, i, a.n);
                store_quad<true>(a.gx + row * a.n, i, a.n, grad_quad(h[k], w[k], g[k], gh, r, c));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[k][j] = fmaf(g[k][j], h[k][j] * r, acc[k][j]);
        }
    }
    if (!a.partial) return;
    float *p = a.partial + (size_t)blockIdx.x * a.n;
    if (T == 64) {
#pragma unroll
        for (int k = 0; k < Q; ++k) sums[group][k * 64 + t] = acc[k];
        __syncthreads();
        for (unsigned i = threadIdx.x; i < Q * 64; i += 256)
            store_quad(p, (long long)i * 4, a.n, ((sums[0][i] + sums[1][i]) + sums[2][i]) + sums[3][i]);
    } else {
#pragma unroll
        for (int k = 0; k < Q; ++k) store_quad(p, (long long)(k * T + t) * 4, a.n, acc[k]);
    }
}

// Rows beyond the registers: the weight's sums first (gx may be gy or gh), then gx in two passes over each row.
__global__ __launch_bounds__(256) void rms_norm_grad_weight_long_kernel(NormGradArgs a, unsigned rows)
{
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= a.n) return;
    quad_t acc = {0.f, 0.f, 0.f, 0.f};
    for (size_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const quad_t h = load_quad(a.h + row * a.n, i, a.n), g = load_quad(a.gy + row * a.n, i, a.n);
        const float r = a.rstd[row];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(g[j], h[j] * r, acc[j]);
    }
    store_quad(a.partial + (size_t)blockIdx.y * a.n, i, a.n, acc);
}
__global__ __launch_bounds__(kLongT) void rms_norm_grad_long_kernel(NormGradArgs a)
{
    __shared__ double part[kLongT / 64];
    const size_t row = blockIdx.x;
    const float *hr = a.h + row * a.n, *gr = a.gy + row * a.n;
    double s = 0.0;
    for (long long i = (long long)threadIdx.x * 4; i < a.n; i += kLongT * 4)
        s = dot3(load_quad(gr, i, a.n), load_quad(a.weight, i, a.n), load_quad(hr, i, a.n), s);
    s = block_sum<kLongT>(s, part);
    const float r = a.rstd[row];
    const double c = s / (double)a.n * (double)r * (double)r * (double)r;
    for (long long i = (long long)threadIdx.x * 4; i < a.n; i += kLongT * 4) {
        quad_t gh = {0.f, 0.f, 0.f, 0.f};
        if (a.gh) gh = load_quad(a.gh + row * a.n, i, a.n);
        store_quad(a.gx + row * a.n, i, a.n, grad_quad(load_quad(hr, i, a.n), load_quad(a.weight, i, a.n), load_quad(gr, i, a.n), gh, r, c));
    }
}

// gw[c] = sum over the G partial rows, `pitch` elements apart, in 64 bits: a block has 32 columns, 128 groups of 8 threads take every 128th row
// each (a quad of columns per thread), and the groups are added in order, by eights and then the sixteen sums.  (With 128
// columns to a block and 32 groups a short row leaves most of the chip idle: the gradient
// of 20000 x 257 takes 49 us that way and 27 this way, of 2000 x 1023 20 and 15.)
constexpr int kFoldGroups = 128;
__global__ __launch_bounds__(kFoldGroups * 8) void rms_norm_grad_fold_kernel(const float *__restrict__ partial, float *__restrict__ gw, long long n,
                                                                            long long pitch, unsigned G)
{
    __shared__ double sums[kFoldGroups][32], eights[kFoldGroups / 8][32];
    const int lane = threadIdx.x & 7, g = threadIdx.x >> 3;
    const long long i = ((long long)blockIdx.x * 8 + lane) * 4;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (i < n)
#pragma unroll 4
        for (unsigned b = g; b < G; b += kFoldGroups) {
            const quad_t v = load_quad(partial + (size_t)b * pitch, i, n);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += (double)v[j];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[g][lane * 4 + j] = s[j];
    __syncthreads();
    const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
    if (part < kFoldGroups / 8) {
        double t = sums[part * 8][c];
#pragma unroll
        for (int k = 1; k < 8; ++k) t += sums[part * 8 + k][c];
        eights[part][c] = t;
    }
    __syncthreads();
    if (part == 0 && (long long)blockIdx.x * 32 + c < n) {
        double t = eights[0][c];
#pragma unroll
        for (int k = 1; k < kFoldGroups / 8; ++k) t += eights[k][c];
        gw[(long long)blockIdx.x * 32 + c] = (float)t;
    }
}

constexpr int kMaxRegisterRow = 4 * 8 * 1024;

// Rows of up to this many elements have a wave each in the gradient: 65536 x 512 takes 69 us, 200000 x 128 59, with a
// block of 256 each 194 and 672.
constexpr int kWaveRow = 1024;

// Blocks that share the rows of a gradient: two per CU with a row at a time (three: 8192 x 4096 208 us for both directions,
// two: 203), eight per CU with four rows at a time where a wave has a row; no more than the rows fill.
inline unsigned norm_grad_blocks(long long rows, int n)
{
    const long long groups = n <= kWaveRow ? (rows + 3) / 4 : rows, most = (n <= kWaveRow ? 8LL : 2LL) * device_cus();
    return (unsigned)(groups < most ? groups : most);
}

}  // namespace ag

using namespace ag;

extern "C" ag_status_t ag_rms_norm_f32(ag_stream_t stream, const float *x, const float *residual, const float *weight, float eps, float *h,
                                       float *y, uint8_t *q, uint8_t *scales, float *rstd, int rows, int n)
{
    AG_REQUIRE(rows >= 0 && n >= 0, AG_ERR_INVALID_DIMS, "rms_norm: negative extent (%d x %d)", rows, n);
    AG_REQUIRE(eps >= 0.f, AG_ERR_INVALID_DIMS, "rms_norm: eps (%g) must be a number >= 0", (double)eps);
    if (rows == 0 || n == 0) return AG_OK;
    AG_REQUIRE(x && weight, AG_ERR_INVALID_DIMS, "rms_norm: null pointer");
    AG_REQUIRE((q != nullptr) == (scales != nullptr), AG_ERR_INVALID_DIMS, "rms_norm: 8-bit values and their scales go together");
    AG_REQUIRE(h || y || q || rstd, AG_ERR_INVALID_DIMS, "rms_norm: no output");
    AG_REQUIRE(!h || h != y, AG_ERR_INVALID_DIMS, "rms_norm: h and y are the same array");
    AG_REQUIRE(aligned16(q), AG_ERR_INVALID_DIMS, "rms_norm: 8-bit output must be 16-byte aligned");
    NormArgs a = {x, residual, weight, h, y, rstd, q, scales, (double)eps, n, (unsigned)(e4m3_pitch(n) / kE4m3Block), (unsigned)e4m3_scale_pitch(n)};
    hipStream_t st = as_stream(stream);
    // Threads of a row: the padding of the scales (a multiple of 512 elements) has to be covered by the quads.
    const long long cells = (long long)e4m3_scale_pitch(n) * kE4m3Block;
    const bool streams = (size_t)rows * (size_t)n * sizeof(float) >= kStreamBytes;
#define NORM(T, Q)                                                                                                                  \
    norm_in_launches(a, (unsigned)rows, T, [&](const NormArgs &p, unsigned r) {                                                     \
        if (streams) hipLaunchKernelGGL((rms_norm_kernel<T, Q, true>), dim3(T == 64 ? (r + 3) / 4 : r), dim3(T == 64 ? 256 : T), 0, st, p, r); \
        else hipLaunchKernelGGL((rms_norm_kernel<T, Q, false>), dim3(T == 64 ? (r + 3) / 4 : r), dim3(T == 64 ? 256 : T), 0, st, p, r);       \
    })
    if (cells <= 512) NORM(64, 2);
    else if (cells <= 1024) NORM(64, 4);
    else if (cells <= 2048) NORM(256, 2);
    else if (cells <= 2560) NORM(128, 5);
    else if (cells <= 4096) NORM(256, 4);
    else if (cells <= 5120) NORM(256, 5);
    else if (cells <= 6144) NORM(256, 6);
    else if (cells <= 8192) NORM(256, 8);
    else if (cells <= 16384) NORM(1024, 4);
    else if (cells <= 20480) NORM(1024, 5);
    else if (cells <= kMaxRegisterRow) NORM(1024, 8);
    else
        norm_in_launches(a, (unsigned)rows, kLongT,
                         [&](const NormArgs &p, unsigned r) { hipLaunchKernelGGL(rms_norm_long_kernel, dim3(r), dim3(kLongT), 0, st, p); });
#undef NORM
    return check_launch("rms_norm");
}

extern "C" size_t ag_rms_norm_grad_f32_workspace(int rows, int n)
{
    if (rows <= 0 || n <= 0) return 0;
    return (size_t)norm_grad_blocks(rows, n) * (size_t)n * sizeof(float);
}

extern "C" ag_status_t ag_rms_norm_grad_f32(ag_stream_t stream, const float *h, const float *weight, const float *rstd, const float *gy,
                                            const float *gh, float *gx, float *gw, int rows, int n, void *ws, size_t ws_bytes)
{
    AG_REQUIRE(rows >= 0 && n >= 0, AG_ERR_INVALID_DIMS, "rms_norm_grad: negative extent (%d x %d)", rows, n);
    if (n == 0) return AG_OK;
    hipStream_t st = as_stream(stream);
    if (rows == 0) {  // no row contributes
        if (!gw) return AG_OK;
        return ag_fill_f32(stream, gw, 0.f, (size_t)n);
    }
    AG_REQUIRE(h && weight && rstd && gy, AG_ERR_INVALID_DIMS, "rms_norm_grad: null pointer");
    AG_REQUIRE(gx || gw, AG_ERR_INVALID_DIMS, "rms_norm_grad: no output");
    AG_REQUIRE(gx != h || !gx, AG_ERR_INVALID_DIMS, "rms_norm_grad: gx must not be h");
    AG_REQUIRE(!gw || (ws && ws_bytes >= ag_rms_norm_grad_f32_workspace(rows, n)), AG_ERR_INVALID_DIMS,
               "rms_norm_grad: workspace of %zu bytes, %zu needed", ws_bytes, ag_rms_norm_grad_f32_workspace(rows, n));
    AG_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 3u) == 0, AG_ERR_INVALID_DIMS, "rms_norm_grad: misaligned workspace");
    AG_REQUIRE(n <= 16384 || rows <= kMaxThreadsX / kLongT, AG_ERR_INVALID_DIMS, "rms_norm_grad: %d rows of %d elements", rows, n);
    const unsigned R = (unsigned)rows, G = norm_grad_blocks(rows, n);
    NormGradArgs a = {h, weight, rstd, gy, gh, gx, gw ? static_cast<float *>(ws) : nullptr, n};
    const bool streams = (size_t)rows * (size_t)n * sizeof(float) >= kStreamBytes;
#define GRAD(T, Q)                                                                                                            \
    do {                                                                                                                      \
        if (streams) hipLaunchKernelGGL((rms_norm_grad_kernel<T, Q, true>), dim3(G), dim3(T == 64 ? 256 : T), 0, st, a, R);    \
        else hipLaunchKernelGGL((rms_norm_grad_kernel<T, Q, false>), dim3(G), dim3(T == 64 ? 256 : T), 0, st, a, R);          \
    } while (0)
    if (n <= 256) GRAD(64, 1);
    else if (n <= 512) GRAD(64, 2);
    else if (n <= kWaveRow) GRAD(64, 4);
    else if (n <= 2048) GRAD(256, 2);
    else if (n <= 4096) GRAD(256, 4);
    else if (n <= 6144) GRAD(512, 3);
    else if (n <= 8192) GRAD(512, 4);
    else if (n <= 16384) GRAD(1024, 4);
    else {
        if (gw) hipLaunchKernelGGL(rms_norm_grad_weight_long_kernel, dim3((unsigned)(((long long)n + 1023) / 1024), G), dim3(256), 0, st, a, R);
        if (gx) hipLaunchKernelGGL(rms_norm_grad_long_kernel, dim3(R), dim3(kLongT), 0, st, a);
    }
#undef GRAD
    if (gw) {
        constexpr long long most = kMaxThreadsX / (kFoldGroups * 8) * 32;  // columns of a launch
        for (long long c = 0; c < n; c += most) {
            const long long count = n - c < most ? n - c : most;
            hipLaunchKernelGGL(rms_norm_grad_fold_kernel, dim3((unsigned)((count + 31) / 32)), dim3(kFoldGroups * 8), 0, st,
                               static_cast<const float *>(ws) + c, gw + c, count, (long long)n, G);
        }
    }
    return check_launch("rms_norm_grad");
}
