// The norm over all elements of many arrays together, and clipping by it:
//
//   norm = sqrt(sum over arrays and elements of g^2)      coefficient = norm <= max_norm ? 1 : max_norm / norm
//
// A NaN anywhere gives a NaN coefficient, an infinity the coefficient 0.  The squares are added in 64 bits (no gradient
// overflows them), each block over its own range and the blocks' sums in order, so a result does not depend on timing.
#include <algorithm>
#include <new>
#include <vector>

#include "e4m3.h"

namespace ag {

// The arrays of one launch lie end to end in one index space, cut into equal ranges for the blocks: one array of 2^28
// elements and two hundred of a hundred load the chip alike.
constexpr int kClipTable = 64;
struct ClipTable {
    const float *x[kClipTable];
    float *out[kClipTable];
    unsigned long long start[kClipTable + 1];  // first index of each array; the last entry is the end
    unsigned long long chunk;                  // elements of a block
    int count;
};

constexpr unsigned long long kClipChunk = 8192;  // elements of a block at the least: 8 quads per thread

template <typename F>
__device__ inline void clip_walk(const ClipTable &tab, F f)
{
    const unsigned long long begin = blockIdx.x * tab.chunk;
    const unsigned long long end = min(begin + tab.chunk, tab.start[tab.count]);
    int i = 0;
    for (int step = kClipTable / 2; step >= 1; step >>= 1)  // the last array that starts at or before `begin`
        if (i + step < tab.count && tab.start[i + step] <= begin) i += step;
    for (unsigned long long at = begin; at < end; ++i) {
        const unsigned long long stop = min(end, tab.start[i + 1]);
        f(i, (long long)(at - tab.start[i]), (long long)(stop - tab.start[i]));
        at = stop;
    }
}

__global__ __launch_bounds__(256) void square_sums_kernel(ClipTable tab, double *__restrict__ partial)
{
    __shared__ double part[4];
    double s = 0.0;
    clip_walk(tab, [&](int i, long long from, long long to) {
        const float *x = tab.x[i];
        long long e = from + (long long)threadIdx.x * 4;
        for (; e + 3 * 1024 + 4 <= to; e += 4 * 1024) {
            quad_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const quad_any_t *>(x + e + k * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) s = fma((double)v[k][j], (double)v[k][j], s);
        }
        for (; e < to; e += 1024) {
            const quad_t v = load_quad(x, e, to);
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)v[j], (double)v[j], s);
        }
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = ((part[0] + part[1]) + part[2]) + part[3];
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
        const double norm = sqrt(t);
        clip[0] = (float)norm;
        clip[1] = norm <= max_norm ? 1.f : (float)(max_norm / norm);
    }
}

__global__ __launch_bounds__(256) void clip_scale_kernel(ClipTable tab, const float *__restrict__ clip)
{
    const float c = clip[1];
    clip_walk(tab, [&](int i, long long from, long long to) {
        const float *x = tab.x[i];
        float *out = tab.out[i];
        long long e = from + (long long)threadIdx.x * 4;
        for (; e + 3 * 1024 + 4 <= to; e += 4 * 1024) {
            quad_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const quad_any_t *>(x + e + k * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<quad_any_t *>(out + e + k * 1024) = v[k] * c;
        }
        for (; e < to; e += 1024) store_quad(out, e, to, load_quad(x, e, to) * c);
    });
}

// Calls f(table, blocks, first block) for the arrays in groups of kClipTable; the cut depends on the sizes alone.
template <typename F>
static ag_status_t clip_groups(int count, const float *const *xs, float *const *outs, const size_t *ns, F f)
{
    unsigned long long all = 0;
    for (int i = 0; i < count; ++i) all += ns[i];
    // eight blocks per CU over all arrays, of whole rounds of 4 x 1024 elements
    unsigned long long chunk = (all / (8ull * (unsigned)device_cus()) + 4095) / 4096 * 4096;
    if (chunk < kClipChunk) chunk = kClipChunk;
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

static size_t clip_blocks(int count, const size_t *ns)
{
    size_t total = 0;
    clip_groups(count, nullptr, nullptr, ns, [&](const ClipTable &, unsigned blocks, size_t) {
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
    clip_groups(count, xs, nullptr, ns, [&](const ClipTable &tab, unsigned blocks, size_t first) {
        hipLaunchKernelGGL(square_sums_kernel, dim3(blocks), dim3(256), 0, st, tab, partial + first);
        total += blocks;
        return AG_OK;
    });
    hipLaunchKernelGGL(clip_coefficient_kernel, dim3(1), dim3(1024), 0, st, partial, (unsigned)total, (double)max_norm, clip);
    return check_launch("global_norm");
}

// Blocks of one launch write what others of it read unless every output is its own input or apart from all of them.
static ag_status_t clip_check_overlap(int count, const float *const *xs, float *const *outs, const size_t *ns)
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
        const uintptr_t x = reinterpret_cast<uintptr_t>(xs[i]), o = reinterpret_cast<uintptr_t>(outs[i]);
        ranges.push_back({o, o + ns[i] * sizeof(float), i, true});
        if (x != o) ranges.push_back({x, x + ns[i] * sizeof(float), i, false});
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
    e = clip_check_overlap(count, xs, outs, ns);
    if (e != AG_OK) return e;
    hipStream_t st = as_stream(stream);
    e = launch_norm(st, count, xs, ns, max_norm, clip, static_cast<double *>(ws));
    if (e != AG_OK) return e;
    return clip_groups(count, xs, outs, ns, [&](const ClipTable &tab, unsigned blocks, size_t) {
        hipLaunchKernelGGL(clip_scale_kernel, dim3(blocks), dim3(256), 0, st, tab, clip);
        return check_launch("clip_by_global_norm");
    });
}
