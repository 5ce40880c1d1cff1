// The norm over all elements of many arrays together, and clipping by it:
//
//   norm = sqrt(sum over arrays and elements of g^2)      coefficient = norm <= max_norm ? 1 : max_norm / norm
//
// A NaN anywhere gives a NaN coefficient, an infinity the coefficient 0 (1 if max_norm is infinite).  The squares are added in 64 bits (no gradient
// overflows them), each block over its own range and the blocks' sums in order, so a result does not depend on timing.
#include <algorithm>
#include <new>
#include <vector>

#include "e4m3.h"

namespace ag {

// Bound by HBM: 2^28 elements are read in 186 us (5.8 TB/s; a copy of 4 GiB reaches 4.7) and clipped in another 375; 2 * 10^8
// in 430 together (the ranges taken from the last to the first in the second pass and streaming stores 40 us of 533, one
// launch for 148 arrays instead of three and finer ranges the rest).  Inside the Adam update the second pass is not made.
//
// The arrays of one launch lie end to end in one index space, cut into equal ranges for the blocks: one array of 2^28
// elements and two hundred of a hundred load the chip alike.
constexpr int kClipTable = 160;
struct ClipTable {
    const float *x[kClipTable];
    float *out[kClipTable];
    unsigned long long start[kClipTable + 1];  // first index of each array; the last entry is the end
    unsigned long long chunk;                  // elements of a block
    int count;
};

constexpr unsigned long long kClipChunk = 8192;  // elements of a block at the least: 8 quads per thread

template <typename F>
__device__ inline void clip_walk(const ClipTable &tab, unsigned block, F f)
{
    const unsigned long long begin = block * tab.chunk;
    const unsigned long long end = min(begin + tab.chunk, tab.start[tab.count]);
    int i = 0;
    for (int step = 128; step >= 1; step >>= 1)  // the last array that starts at or before `begin`
        if (i + step < tab.count && tab.start[i + step] <= begin) i += step;
    for (unsigned long long at = begin; at < end; ++i) {
        const unsigned long long stop = min(end, tab.start[i + 1]);
        f(i, (long long)(at - tab.start[i]), (long long)(stop - tab.start[i]));
        at = stop;
    }
}

// Sum over the block's range of the squares, in thread 0.  `part`: one double per wave.
template <int T>
__device__ inline double block_square_sum(const ClipTable &tab, double *part)
{
    double s = 0.0;
    clip_walk(tab, blockIdx.x, [&](int i, long long from, long long to) {
        const float *x = tab.x[i];
        long long e = from + (long long)threadIdx.x * 4;
        for (; e + 3 * T * 4 + 4 <= to; e += 4 * T * 4) {
            quad_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const quad_any_t *>(x + e + k * T * 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) s = fma((double)v[k][j], (double)v[k][j], s);
        }
        for (; e < to; e += T * 4) {
            const quad_t v = load_quad(x, e, to);
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)v[j], (double)v[j], s);
        }
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    double t = part[0];
    for (int i = 1; i < T / 64; ++i) t += part[i];
    return t;
}

__device__ inline void write_clip(double squares, double max_norm, float *clip)
{
    const double norm = sqrt(squares);
    clip[0] = (float)norm;
    clip[1] = norm <= max_norm ? 1.f : (float)(max_norm / norm);
}

__global__ __launch_bounds__(256) void square_sums_kernel(ClipTable tab, double *__restrict__ partial)
{
    __shared__ double part[4];
    const double s = block_square_sum<256>(tab, part);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// Few elements: one block does it all.  The small net's 87722 take 0.6 us longer on the device and 2.6 us less on the host,
// which is what a step of that size waits for; at 131072 elements 7.2 and 5.6 us on the device, at 262144 10.5 and 5.5.
constexpr unsigned long long kOneBlock = 131072;
__global__ __launch_bounds__(1024) void small_norm_kernel(ClipTable tab, double max_norm, float *__restrict__ clip)
{
    __shared__ double part[16];
    const double s = block_square_sum<1024>(tab, part);
    if (threadIdx.x == 0) write_clip(s, max_norm, clip);
}

// clip[0] = norm, clip[1] = coefficient; one block.
__global__ __launch_bounds__(1024) void clip_coefficient_kernel(const double *__restrict__ partial, unsigned count, double max_norm, float *__restrict__ clip)
{
    __shared__ double part[16];
    double s = 0.0;
    for (unsigned i = threadIdx.x; i < count; i += 1024) s += partial[i];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = part[0];
        for (int i = 1; i < 16; ++i) t += part[i];
        write_clip(t, max_norm, clip);
    }
}

__global__ __launch_bounds__(256) void clip_scale_kernel(ClipTable tab, const float *__restrict__ clip)
{
    const float c = clip[1];
    // from the last range to the first: what the norm read last is still in the cache
    clip_walk(tab, gridDim.x - 1 - blockIdx.x, [&](int i, long long from, long long to) {
        const float *x = tab.x[i];
        float *out = tab.out[i];
        long long e = from + (long long)threadIdx.x * 4;
        for (; e + 3 * 1024 + 4 <= to; e += 4 * 1024) {
            quad_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const quad_any_t *>(x + e + k * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k) __builtin_nontemporal_store(v[k] * c, reinterpret_cast<quad_any_t *>(out + e + k * 1024));
        }
        for (; e < to; e += 1024) store_quad(out, e, to, load_quad(x, e, to) * c);
    });
}

// Calls f(table, blocks, first block) for the arrays in groups of kClipTable, cut into ranges of `chunk` elements.
template <typename F>
static ag_status_t clip_groups(int count, const float *const *xs, float *const *outs, const size_t *ns, unsigned long long chunk, F f)
{
    size_t first = 0;
    for (int i = 0; i < count;) {
        ClipTable tab = {};
        tab.chunk = chunk;
        unsigned long long at = 0;
        for (; i < count && tab.count < kClipTable; ++i) {
            if (ns[i] == 0) continue;
            tab.x[tab.count] = xs ? xs[i] : nullptr;
            tab.out[tab.count] = outs ? outs[i] : nullptr;
            tab.start[tab.count++] = at;
            at += ns[i];
        }
        if (tab.count == 0) break;
        tab.start[tab.count] = at;
        const size_t blocks = (size_t)((at + chunk - 1) / chunk);
        const ag_status_t e = f(tab, (unsigned)blocks, first);
        if (e != AG_OK) return e;
        first += blocks;
    }
    return AG_OK;
}

// The range of a block: 32 blocks per CU over all arrays, of whole rounds of 4 x 1024 elements, by the sizes alone.  Norm
// and clipping of 2 * 10^8 elements in 148 arrays: 430 us, with 8 blocks per CU 466, with 16 446, with 64 428.
static unsigned long long clip_chunk(int count, const size_t *ns)
{
    unsigned long long all = 0;
    for (int i = 0; i < count; ++i) all += ns[i];
    const unsigned long long chunk = (all / (32ull * (unsigned)device_cus()) + 4095) / 4096 * 4096;
    return chunk < kClipChunk ? kClipChunk : chunk;
}

static size_t clip_blocks(int count, const size_t *ns)
{
    size_t total = 0;
    clip_groups(count, nullptr, nullptr, ns, clip_chunk(count, ns), [&](const ClipTable &, unsigned blocks, size_t) {
        total += blocks;
        return AG_OK;
    });
    return total;
}

static ag_status_t clip_check(const char *who, int count, const float *const *xs, const size_t *ns, float max_norm, const float *clip, const void *ws,
                              size_t ws_bytes)
{
    AG_REQUIRE(count >= 0, AG_ERR_INVALID_DIMS, "%s: %d arrays", who, count);
    AG_REQUIRE(max_norm >= 0.f, AG_ERR_INVALID_DIMS, "%s: max_norm (%g) must be a number >= 0", who, (double)max_norm);
    AG_REQUIRE(clip, AG_ERR_INVALID_DIMS, "%s: null pointer", who);
    AG_REQUIRE(count == 0 || (xs && ns), AG_ERR_INVALID_DIMS, "%s: null pointer table", who);
    for (int i = 0; i < count; ++i) AG_REQUIRE(ns[i] == 0 || xs[i], AG_ERR_INVALID_DIMS, "%s: null pointer (array %d)", who, i);
    const size_t need = clip_blocks(count, ns) * sizeof(double);
    AG_REQUIRE(need == 0 || (ws && ws_bytes >= need), AG_ERR_INVALID_DIMS, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
    AG_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 7u) == 0, AG_ERR_INVALID_DIMS, "%s: misaligned workspace", who);
    return AG_OK;
}

static ag_status_t launch_norm(hipStream_t st, int count, const float *const *xs, const size_t *ns, float max_norm, float *clip, double *partial)
{
    size_t total = 0;
    unsigned long long all = 0;
    for (int i = 0; i < count; ++i) all += ns[i];
    if (count <= kClipTable && all <= kOneBlock) {
        ClipTable none = {};
        if (all == 0) hipLaunchKernelGGL(small_norm_kernel, dim3(1), dim3(1024), 0, st, none, (double)max_norm, clip);
        else
            clip_groups(count, xs, nullptr, ns, kOneBlock, [&](const ClipTable &tab, unsigned, size_t) {
                hipLaunchKernelGGL(small_norm_kernel, dim3(1), dim3(1024), 0, st, tab, (double)max_norm, clip);
                return AG_OK;
            });
        return check_launch("global_norm");
    }
    clip_groups(count, xs, nullptr, ns, clip_chunk(count, ns), [&](const ClipTable &tab, unsigned blocks, size_t first) {
        hipLaunchKernelGGL(square_sums_kernel, dim3(blocks), dim3(256), 0, st, tab, partial + first);
        total += blocks;
        return AG_OK;
    });
    hipLaunchKernelGGL(clip_coefficient_kernel, dim3(1), dim3(1024), 0, st, partial, (unsigned)total, (double)max_norm, clip);
    return check_launch("global_norm");
}

// Blocks of one launch write what others of it read unless every output is its own input or apart from all of them.
static ag_status_t clip_check_overlap(int count, const float *const *xs, float *const *outs, const size_t *ns, const float *clip)
try {
    struct Range {
        uintptr_t from, to;
        int i;
        bool out;
    };
    std::vector<Range> ranges;
    ranges.reserve(2 * (size_t)count);
    for (int i = 0; i < count; ++i) {
        if (ns[i] == 0) continue;
        AG_REQUIRE(outs[i], AG_ERR_INVALID_DIMS, "clip_by_global_norm: null pointer (array %d)", i);
        const uintptr_t x = reinterpret_cast<uintptr_t>(xs[i]), o = reinterpret_cast<uintptr_t>(outs[i]), c = reinterpret_cast<uintptr_t>(clip);
        const size_t bytes = ns[i] * sizeof(float);
        AG_REQUIRE((c + 8 <= x || c >= x + bytes) && (c + 8 <= o || c >= o + bytes), AG_ERR_INVALID_DIMS,
                   "clip_by_global_norm: array %d overlaps the norm and coefficient", i);
        ranges.push_back({o, o + bytes, i, true});
        if (x != o) ranges.push_back({x, x + bytes, i, false});
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    // in the order of their starts: an output may overlap nothing, an input may overlap inputs
    uintptr_t out_end = 0, any_end = 0;
    int out_at = -1, any_at = -1;
    for (const Range &r : ranges) {
        AG_REQUIRE(r.from >= out_end, AG_ERR_INVALID_DIMS, "clip_by_global_norm: the output of array %d overlaps array %d", out_at, r.i);
        AG_REQUIRE(!r.out || r.from >= any_end, AG_ERR_INVALID_DIMS, "clip_by_global_norm: the output of array %d overlaps array %d", r.i, any_at);
        if (r.out && r.to > out_end) out_end = r.to, out_at = r.i;
        if (r.to > any_end) any_end = r.to, any_at = r.i;
    }
    return AG_OK;
} catch (const std::bad_alloc &) {
    return fail(AG_ERR_NDARRAY, "clip_by_global_norm: out of host memory");
}

}  // namespace ag

using namespace ag;

extern "C" size_t ag_global_norm_f32_workspace(int count, const size_t *ns)
{
    return count > 0 && ns ? clip_blocks(count, ns) * sizeof(double) : 0;
}

extern "C" ag_status_t ag_global_norm_f32(ag_stream_t stream, int count, const float *const *xs, const size_t *ns, float max_norm, float *clip,
                                          void *ws, size_t ws_bytes)
{
    const ag_status_t e = clip_check("global_norm", count, xs, ns, max_norm, clip, ws, ws_bytes);
    if (e != AG_OK) return e;
    return launch_norm(as_stream(stream), count, xs, ns, max_norm, clip, static_cast<double *>(ws));
}

extern "C" ag_status_t ag_clip_by_global_norm_f32(ag_stream_t stream, int count, const float *const *xs, float *const *outs, const size_t *ns,
                                                  float max_norm, float *clip, void *ws, size_t ws_bytes)
{
    ag_status_t e = clip_check("clip_by_global_norm", count, xs, ns, max_norm, clip, ws, ws_bytes);
    if (e != AG_OK) return e;
    AG_REQUIRE(count == 0 || outs, AG_ERR_INVALID_DIMS, "clip_by_global_norm: null pointer table");
    e = clip_check_overlap(count, xs, outs, ns, clip);
    if (e != AG_OK) return e;
    hipStream_t st = as_stream(stream);
    e = launch_norm(st, count, xs, ns, max_norm, clip, static_cast<double *>(ws));
    if (e != AG_OK) return e;
    return clip_groups(count, xs, outs, ns, clip_chunk(count, ns), [&](const ClipTable &tab, unsigned blocks, size_t) {
        hipLaunchKernelGGL(clip_scale_kernel, dim3(blocks), dim3(256), 0, st, tab, clip);
        return check_launch("clip_by_global_norm");
    });
}
