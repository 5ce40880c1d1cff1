// Matrix product of two e4m3 operands whose scales stand beside them: C[M,N] = A[M,K] . B[N,K]^T in f32, both operands
// contiguous along the contraction.
//
// Operands stay in 8 bits in HBM and LDS and become bf16 on the way into the matrix unit: one instruction
// (v_cvt_scalef32_pk_bf16_fp8) turns two values into bf16 and multiplies them by the block's power of two, all of it
// exact (4 significant bits, an exponent that bf16 holds).  The 8-bit matrix instruction v_mfma_scale_f32_32x32x64_f8f6f4
// would multiply twice as fast, but it does not keep f32 sums: it aligns each group of 8 products to the largest of them
// and drops what lies 2^-14 below (measured: +2^16 - 2^16 + 2^2 within a group gives 0), 1.4e-5 of the result for
// Gaussian operands and 6e-5 for wider ones, whatever the length; the bf16 instruction gives 8e-8 and 4e-7.
#include <type_traits>

#include "e4m3.h"

namespace ag {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

struct GemmE4m3 {
    const unsigned char *a, *a_scales, *b, *b_scales;
    float *c;
    long long ldc, pitch;
    int M, N, blocks, scale_pitch;  // blocks of 128 along the contraction
    int tiles_m, tiles_n;
    int splits, per_split;  // slices of the contraction and blocks of 128 in each; splits > 1: c is [splits][M][N]
};

// A scale byte as the f32 whose exponent field it is.  The widening instruction reads that field alone: 0 is a factor of
// 2^-127 there, 255 gives NaN.
__device__ inline float scale_factor(unsigned word, int i) { return __uint_as_float(((word >> (8 * i)) & 0xffu) << 23); }

// Eight consecutive e4m3 values times s, in bf16.
__device__ inline v8bf widen(int lo, int hi, float s)
{
    const v2bf r0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), r1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const v2bf r2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), r3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return v8bf{r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}

// ---- tiles ------------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) unsigned char lds_byte_t;

// Loads straight from global memory into LDS: lane l's 16 (or 4) bytes land at lds + 16 l (4 l).  In assembly because the
// compiler would wait for every outstanding load in front of each LDS read; the waits are written out below.
__device__ inline void dma16(const unsigned char *base, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ inline void dma4(const unsigned char *base, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ inline const unsigned char *uniform(const unsigned char *p)
{
    const unsigned long long b = reinterpret_cast<unsigned long long>(p);
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(b >> 32));
    return reinterpret_cast<const unsigned char *>(((unsigned long long)hi << 32) | lo);
}

// BM x BN of C per block, WM x WN per wave, 128 of the contraction per step.  LDS holds STAGES steps of both operands, rows
// of 128 bytes, and a word of scales per row (four blocks, one of which the step uses).  The 16-byte piece c of row r stands
// at place c ^ (r & 7) ^ ((r >> 3) & 1), so that 16 consecutive rows read at one piece fall on all 64 banks.
//
// What bounds it is power first: with Gaussian operands the chip holds the matrix instruction alone, fed from registers, at
// 1830 TFLOP/s (1.75 GHz; 2480 with zeros), and lowers its clock as the rest of the loop gets out of the way; and the rest
// of the loop: the matrix unit is busy for 83 % of the time at 1.70 GHz, in the library's bf16 product for 86 % at 1.78.
// 4096^3 takes 97-104 us from run to run (1320-1415 TFLOP/s; the library's bf16 product, from operands twice the size,
// 91-102), 16384 x 8192 x 8192 1.44-1.51 ms (1455-1530; 1.33).  What brought it there, the best of a run each at 4096^3
// and at 16384 x 8192 x 8192: every load of a step issued behind the barrier and operands widened where they are used 104 us,
// 1.61 ms; the next group's operands widened between the instructions of the current one, LDS read a chunk ahead and the
// barrier in front of a step's last chunk 101 us, 1.48 ms; one basic block per step (no tests around the loads) and the
// loads spread over four groups 97 us, 1.44 ms.  Four waves of 128 x 128 need a third less of LDS and widening but stand
// still together: 99 us, 1.46 ms; loads spread singly between the instructions 100 us, 1.48 ms.
template <int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void gemm_e4m3_tile_kernel(GemmE4m3 p)
{
    constexpr int WAVES_N = BN / WN, NW = BM / WM * WAVES_N, MI = WM / 32, NI = WN / 32;
    constexpr int ROWS = BM + BN, STEP = ROWS * 128;
    constexpr int LOADS = ROWS / 8 / NW;                    // 1 KiB loads (8 rows) of a wave per step
    constexpr int SCALE_LOADS = (ROWS / 64 + NW - 1) / NW;  // 64 words of a wave per step
    static_assert(STAGES >= 2 && STAGES <= 4, "ring of two to four steps");
    static_assert(ROWS % (8 * NW) == 0 && BM % 64 == 0 && BN % 64 == 0, "rows divide over the waves");
    __shared__ __attribute__((aligned(1024))) unsigned char tile[STAGES * STEP];
    __shared__ __attribute__((aligned(256))) unsigned scale_words[STAGES][ROWS];
    const unsigned lds = (unsigned)(size_t)(lds_byte_t *)tile, lds_scales = (unsigned)(size_t)(lds_byte_t *)scale_words;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;

    // Consecutive places go down bands of 8 tile rows: the 32 blocks that an XCD runs at a time form a patch of 8 x 4 tiles.
    const unsigned total = (unsigned)p.tiles_m * p.tiles_n;
    unsigned place = xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int)(place / total);
    place -= (unsigned)split * total;
    const unsigned band = place / (8u * p.tiles_n), rest = place - band * 8u * p.tiles_n;
    const unsigned high = min(8u, (unsigned)p.tiles_m - band * 8u);
    const int m0 = (int)(band * 8u + rest % high) * BM, n0 = (int)(rest / high) * BN;

    // what this lane fetches: rows of 128 bytes, 8 lanes each
    const unsigned char *base[LOADS];
    unsigned offset[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r0 = (i * NW + wave) * 8;  // (a group of 8 rows lies in one operand)
        const bool in_a = r0 < BM;
        const int first = in_a ? m0 + r0 : n0 + r0 - BM, last = (in_a ? p.M : p.N) - 1;
        const int start = min(first, last), row = min(first + (lane >> 3), last);
        base[i] = uniform((in_a ? p.a : p.b) + start * p.pitch);
        // (rows are at most 2^28 bytes long, which the host checks: 8 of them stay within 32 bits)
        offset[i] = (unsigned)((row - start) * p.pitch) + (unsigned)(((lane & 7) ^ (lane >> 3) ^ ((i * NW + wave) & 1)) * 16);
    }
    const unsigned char *scale_base[SCALE_LOADS];
    unsigned scale_offset[SCALE_LOADS];
#pragma unroll
    for (int i = 0; i < SCALE_LOADS; ++i) {
        const int r0 = min((i * NW + wave) * 64, ROWS - 64);  // (where they do not divide over the waves, some fetch the last again)
        const bool in_a = r0 < BM;
        const int first = in_a ? m0 + r0 : n0 + r0 - BM, last = (in_a ? p.M : p.N) - 1;
        const int start = min(first, last), row = min(first + lane, last);
        scale_base[i] = uniform((in_a ? p.a_scales : p.b_scales) + (long long)start * p.scale_pitch);
        scale_offset[i] = (unsigned)((row - start) * p.scale_pitch);
    }

    const int k_begin = split * p.per_split, k_end = min(p.blocks, k_begin + p.per_split);
    auto fetch_one = [&](int i, int k, int buffer) {
        dma16(base[i] + (long long)k * 128, offset[i], lds + (unsigned)(buffer * STEP + (i * NW + wave) * 1024));
    };
    auto fetch_scales = [&](int k, int buffer) {
#pragma unroll
        for (int i = 0; i < SCALE_LOADS; ++i)
            dma4(scale_base[i] + (k & ~3), scale_offset[i], lds_scales + (unsigned)(buffer * ROWS * 4 + min((i * NW + wave) * 256, ROWS * 4 - 256)));
    };

    // Two groups of matrix instructions (16 of the contraction each) per chunk of 32.  While a group runs, the next one's
    // operands are widened between its instructions, and the next chunk's pieces are on their way from LDS.  The barrier
    // between two steps stands in front of a step's last chunk, whose pieces are in registers by then.
    v16f acc[MI][NI] = {};
    v4i qa[2][MI], qb[2][NI];
    v4i fa[2][MI], fb[2][NI];  // bf16
    float sa[MI], sb[NI];
    const int row_a = wm * WM + (lane & 31), row_b = BM + wn * WN + (lane & 31);
    auto read = [&](int to, int buffer, int chunk) {
        const unsigned char *at = tile + buffer * STEP + ((chunk * 2 + (lane >> 5)) ^ (lane & 7) ^ ((lane >> 3) & 1)) * 16;
#pragma unroll
        for (int i = 0; i < MI; ++i) qa[to][i] = *reinterpret_cast<const v4i *>(at + (row_a + i * 32) * 128);
#pragma unroll
        for (int j = 0; j < NI; ++j) qb[to][j] = *reinterpret_cast<const v4i *>(at + (row_b + j * 32) * 128);
    };
    auto read_scales = [&](int k, int buffer) {
#pragma unroll
        for (int i = 0; i < MI; ++i) sa[i] = scale_factor(scale_words[buffer][row_a + i * 32], k & 3);
#pragma unroll
        for (int j = 0; j < NI; ++j) sb[j] = scale_factor(scale_words[buffer][row_b + j * 32], k & 3);
    };
    auto widen_group = [&](int to, int from, int h) {
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[to][j] = __builtin_bit_cast(v4i, widen(qb[from][j][2 * h], qb[from][j][2 * h + 1], sb[j]));
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[to][i] = __builtin_bit_cast(v4i, widen(qa[from][i][2 * h], qa[from][i][2 * h + 1], sa[i]));
    };
    // The loads run AHEAD steps in front of the matrix instructions.  A step's go out in four turns in front of as many
    // groups: the last two of the step whose buffer they fill and the first two of the next.
    constexpr int TURNS = 4, AHEAD = STAGES - 1;
    auto fetch_some = [&](int turn, int k, int buffer) {
        if (turn == 0) fetch_scales(k, buffer);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (i * TURNS / LOADS == turn) fetch_one(i, k, buffer);
    };
    auto wrap = [](int buffer) { return buffer >= STAGES ? buffer - STAGES : buffer; };
    // Waits for the loads of the next step (`later` whole steps have been fetched behind it) and for every wave's reads.
    auto arrive = [&](auto later) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(decltype(later)::value * (LOADS + SCALE_LOADS)) : "memory");
    };
    // `after`: how many steps follow, as far as it matters (AHEAD + 1 stands for more).
    auto step = [&](auto after, int k, int buffer) {
        constexpr int AFTER = decltype(after)::value;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            const int chunk = g >> 1, next = (g + 1) & 1;
            if ((g & 1) == 0) {
                if (chunk < 3) {
                    read((chunk + 1) & 1, buffer, chunk + 1);
                } else if (AFTER >= 1) {
                    arrive(std::integral_constant<int, (AFTER < 1 ? 1 : AFTER < AHEAD ? AFTER : AHEAD) - 1>());
                    read(0, wrap(buffer + 1), 0);
                }
            }
            if (g == 7 && AFTER >= 1) read_scales(k + 1, wrap(buffer + 1));
            if (g < 2 && AFTER >= AHEAD) fetch_some(2 + g, k + AHEAD, wrap(buffer + AHEAD));
            if (g >= 6 && AFTER > AHEAD) fetch_some(g - 6, k + AHEAD + 1, buffer);
            if (g < 7 || AFTER >= 1) widen_group(next, ((g + 1) >> 1) & 1, next);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, fa[g & 1][i]), __builtin_bit_cast(v8bf, fb[g & 1][j]),
                                                                         acc[i][j], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < MI * NI; ++t) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                              // a matrix instruction,
                __builtin_amdgcn_sched_group_barrier(0x002, 4 * (MI + NI) / (MI * NI) + 1, 0);  // its share of the vector ones
            }
            // (the widened operands exist here: left to itself the compiler widens them where they are used)
            if (g < 7 || AFTER >= 1) {
#pragma unroll
                for (int i = 0; i < MI; ++i) asm volatile("" : "+v"(fa[next][i]));
#pragma unroll
                for (int j = 0; j < NI; ++j) asm volatile("" : "+v"(fb[next][j]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (k_begin < k_end) {
        const int steps = k_end - k_begin;
        // steps 0 .. AHEAD - 1 whole, and the first two turns of step AHEAD
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (a < steps)
#pragma unroll
                for (int t = 0; t < TURNS; ++t) fetch_some(t, k_begin + a, a);
        if (steps >= AHEAD) arrive(std::integral_constant<int, AHEAD - 1>());
        else arrive(std::integral_constant<int, 0>());
        if (AHEAD < steps) {
            fetch_some(0, k_begin + AHEAD, AHEAD);
            fetch_some(1, k_begin + AHEAD, AHEAD);
        }
        read(0, 0, 0);
        read_scales(k_begin, 0);
        widen_group(0, 0, 0);
        int k = k_begin, buffer = 0;
        for (; k + AHEAD + 1 < k_end; ++k, buffer = wrap(buffer + 1)) step(std::integral_constant<int, AHEAD + 1>(), k, buffer);
        auto last = [&](auto after) {
            if (k_end - 1 - k == decltype(after)::value) {
                step(after, k, buffer);
                ++k;
                buffer = wrap(buffer + 1);
            }
        };
        if constexpr (AHEAD >= 3) last(std::integral_constant<int, 3>());
        if constexpr (AHEAD >= 2) last(std::integral_constant<int, 2>());
        last(std::integral_constant<int, 1>());
        last(std::integral_constant<int, 0>());
    }
    float *c = p.c + (long long)split * p.M * p.ldc;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int n = n0 + wn * WN + j * 32 + (lane & 31);
            const int m = m0 + wm * WM + i * 32 + 4 * (lane >> 5);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = m + 8 * (e / 4) + e % 4;
                if (r < p.M && n < p.N) c[r * p.ldc + n] = acc[i][j][e];
            }
        }
}

// C = the slices' partial results added in order.
__global__ __launch_bounds__(256) void gemm_e4m3_fold_kernel(const float *__restrict__ partial, float *__restrict__ c, long long ldc, int M, int N, int splits)
{
    const long long i = (long long)blockIdx.x * 1024 + threadIdx.x * 4, cells = (long long)M * N;
    if (i >= cells) return;
    quad_t s = load_quad(partial, i, cells);
    for (int k = 1; k < splits; ++k) s += load_quad(partial + k * cells, i, cells);
    const long long m = i / N, n = i - m * N;
    if (n + 4 <= N) {
        *reinterpret_cast<quad_any_t *>(c + m * ldc + n) = s;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long at = i + j;
            if (at < cells) c[at / N * ldc + at % N] = s[j];
        }
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------------------
// Up to 16 * MT rows of A against 16 rows of B per block, operands straight from global memory into the matrix unit's
// layout: the weight is read once, in whole 512-byte pieces of its rows, and nothing is shared between waves but the
// sums.  The waves take pieces of 512 of the contraction in turn, with every load of a piece in flight at once; their sums
// are added in order through LDS.  Lane l holds row l % 16 and 32 consecutive bytes of each 128: group l / 16 of four.
// XR > 0: A is x itself, at most XR rows of it, rounded on the way as ag_quantize_e4m3_f32 rounds it: a wave rounds its
// pieces of the rows with 32 lanes to a block and hands the bytes to the lanes that multiply them through LDS.  One row
// against 4096 x 4096 takes 7.1 us that way (2.4 TB/s of weight: launch, one round of loads, the sums), against 16384 x
// 4096 17.7 us (3.8 TB/s); as two launches 10.2 and 20.8 us, and with the rows rounded by the 4 lanes of the matrix
// layout that hold them 12.0 and 32 us.  At 4 rows the two ways are even (10.0 and 10.2, 22.8 and 20.8 us).
constexpr int kRoundedRows = 4;

// Between LDS accesses of lanes of one wave: they complete in their order, which the compiler must not change.
__device__ inline void hand_over()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int MT, int NW, int XR>
__global__ __launch_bounds__(NW * 64) void gemm_e4m3_skinny_kernel(GemmE4m3 p, const float *__restrict__ x, long long ldx, int K)
{
    static_assert(XR == 0 || (MT == 1 && XR == 4), "rounded on the way for few rows only");
    constexpr int PIECE = 512 + 16;  // bytes of a row's piece in LDS: 16 more than it has, so that rows fall on other banks
    __shared__ float sums[NW][MT][256];
    __shared__ __attribute__((aligned(16))) unsigned char rounded[XR > 0 ? NW : 1][XR > 0 ? XR : 1][PIECE];
    __shared__ __attribute__((aligned(4))) unsigned char rounded_scales[XR > 0 ? NW : 1][XR > 0 ? XR : 1][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, group = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int words = (p.blocks + 3) / 4;
    const int row_b = min(n0 + r16, p.N - 1);
    v4f acc[MT] = {};
    for (int w = wave; w < words; w += NW) {
        const int count = min(4, p.blocks - w * 4);
        v4i qb[4][2], qa[MT][4][2];
        unsigned word_a[MT];
        const unsigned char *b = p.b + row_b * p.pitch + (long long)w * 512 + group * 32, *a[MT];
        const unsigned word_b = *reinterpret_cast<const unsigned *>(p.b_scales + (long long)row_b * p.scale_pitch + w * 4);
        if (XR == 0)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int row_a = min(t * 16 + r16, p.M - 1);
                a[t] = p.a + row_a * p.pitch + (long long)w * 512 + group * 32;
                word_a[t] = *reinterpret_cast<const unsigned *>(p.a_scales + (long long)row_a * p.scale_pitch + w * 4);
            }
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // (in the order of their use: they arrive in it)
            const int at = min(u, count - 1) * 128;  // (a piece that ends early reads its last block again)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                qb[u][h] = *reinterpret_cast<const v4i *>(b + at + h * 16);
                if (XR == 0)
#pragma unroll
                    for (int t = 0; t < MT; ++t) qa[t][u][h] = *reinterpret_cast<const v4i *>(a[t] + at + h * 16);
            }
        }
        if (XR > 0) {
            const int half = lane >> 5, l31 = lane & 31;
            auto round_rows = [&](auto several) {  // the first rows of x (the last one again where there are fewer), loaded together
                constexpr int ROWS = decltype(several)::value;
                quad_t v[ROWS][2];  // blocks half and half + 2 of the piece
                const long long k0 = (long long)w * 512 + half * 128 + l31 * 4;
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float *row = x + min(r, p.M - 1) * ldx;
                    if ((long long)(w + 1) * 512 <= K) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) v[r][i] = *reinterpret_cast<const quad_any_t *>(row + k0 + i * 256);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) v[r][i] = load_quad(row, k0 + i * 256, K);
                    }
                }
#pragma unroll
                for (int r = 0; r < ROWS; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        unsigned sb;
                        *reinterpret_cast<unsigned *>(&rounded[wave][r][(half + 2 * i) * 128 + l31 * 4]) = round_block(v[r][i], &sb);
                        if (l31 == 0) rounded_scales[wave][r][half + 2 * i] = (unsigned char)sb;
                    }
            };
            if (p.M == 1) round_rows(std::integral_constant<int, 1>());
            else if (p.M == 2) round_rows(std::integral_constant<int, 2>());
            else round_rows(std::integral_constant<int, 4>());
            hand_over();
            const bool here = r16 < p.M;
            word_a[0] = here ? *reinterpret_cast<const unsigned *>(rounded_scales[wave][here ? r16 : 0]) : 0x7f7f7f7fu;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const v4i q = *reinterpret_cast<const v4i *>(&rounded[wave][here ? r16 : 0][u * 128 + group * 32 + h * 16]);
                    qa[0][u][h] = here ? q : v4i{0, 0, 0, 0};
                }
            hand_over();
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (u < count) {
                const float sb = scale_factor(word_b, u);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const v8bf vb = widen(qb[u][h][2 * e], qb[u][h][2 * e + 1], sb);
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(qa[t][u][h][2 * e], qa[t][u][h][2 * e + 1], scale_factor(word_a[t], u)), vb,
                                                                            acc[t], 0, 0, 0);
                    }
            }
    }
    // lane l holds column l % 16 and rows 4 (l / 16) .. + 3
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][t][(group * 4 + e) * 16 + r16] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 256; i += NW * 64) {
        float s = sums[0][i / 256][i % 256];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += sums[w][i / 256][i % 256];
        const int m = i / 16, n = n0 + i % 16;
        if (m < p.M && n < p.N) p.c[m * p.ldc + n] = s;
    }
}

// ---- which form, and its launch ---------------------------------------------------------------------------------------
// The rounding of ag_quantize_e4m3_f32 (quantize.hip).
ag_status_t quantize_e4m3(const char *who, hipStream_t st, const float *x, long long ldx, int rows, int cols, unsigned char *q, unsigned char *scales,
                          unsigned char *qt, unsigned char *scales_t);

// Tiles of the output (0: the kernel for few rows) and slices of the contraction, by the extents alone.  Times in us:
//   up to 16 rows               the kernel for few rows: 8 rows x 16384 x 4096 18.0, with tiles of 64 21.4;
//   up to 32 rows, at most a block per CU with a piece per wave      32 x 4096 x 4096 9.3, with tiles of 64 11.3 (but 32 x
//                               16384 x 4096 32.8 against 21.4, and 40 x 300 x 8192 18.0 against 10.7);
//   at most two tiles of 64 per CU       these, four steps deep, the contraction cut until there is a block per CU, not below
//                               8 steps to a slice: 64 x 1000 x 8192 11.6 in 8 slices, 13.6 in 4 (tiles of 128, 12 slices: 15.7);
//                               256 x 4096 x 4096 19.7 (tiles of 128 22.6); 64 x 8192 x 1024 7.6, in 2 slices 10.1;
//   at most a tile of 128 per CU         these, four steps deep: 1024 x 4096 x 4096 36.0 (two steps deep 44.8);
//   else tiles of 128, two blocks per CU, or of 256, one per CU, whichever needs less time by whole rounds of blocks, a round
//                               of the smaller taking 0.62 of one of the larger (2048 x 4096 x 4096: 62 and 72; 4096^3: 128 and 97).
struct Plan {
    int tile, splits;
    bool deep;
};

static Plan plan_product(int M, int N, int K)
{
    const long long steps = (long long)(e4m3_pitch(K) / kE4m3Block), cus = device_cus();
    auto tiles = [&](long long t) { return (M + t - 1) / t * ((N + t - 1) / t); };
    if (M <= 16 || (M <= 32 && N <= 16 * cus && steps <= 32)) return {0, 1, false};
    if (tiles(64) <= 2 * cus) {
        const long long fill = cus / tiles(64), deep = steps / 8;
        return {64, (int)(fill < deep ? (fill > 1 ? fill : 1) : (deep > 1 ? deep : 1)), true};
    }
    if (tiles(128) <= cus) return {128, 1, true};
    const long long rounds128 = (tiles(128) + 2 * cus - 1) / (2 * cus), rounds256 = (tiles(256) + cus - 1) / cus;
    return {rounds128 * 62 < rounds256 * 100 ? 128 : 256, 1, false};
}

static size_t product_workspace(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const Plan f = plan_product(M, N, K);
    return f.splits > 1 ? (size_t)f.splits * M * N * sizeof(float) : 0;
}

static ag_status_t check_product(const char *who, int M, int N, int K, int ldc, const void *b, const void *bs, const void *c)
{
    AG_REQUIRE(M >= 0 && N >= 0 && K >= 0, AG_ERR_INVALID_DIMS, "%s: negative extent (%d x %d x %d)", who, M, N, K);
    AG_REQUIRE(K <= 1 << 28, AG_ERR_INVALID_DIMS, "%s: a contraction of %d elements (at most 2^28)", who, K);
    AG_REQUIRE(ldc >= N, AG_ERR_INCOMPATIBLE_SHAPE, "%s: ldc (%d) is less than a row of %d elements", who, ldc, N);
    if (M == 0 || N == 0) return AG_OK;
    AG_REQUIRE(c && (K == 0 || (b && bs)), AG_ERR_INVALID_DIMS, "%s: null pointer", who);
    AG_REQUIRE(aligned16(b), AG_ERR_INVALID_DIMS, "%s: 8-bit operands must be 16-byte aligned", who);
    AG_REQUIRE((reinterpret_cast<uintptr_t>(bs) & 3u) == 0, AG_ERR_INVALID_DIMS, "%s: scales must be 4-byte aligned", who);
    const Plan f = plan_product(M, N, K);
    if (f.tile == 0) return AG_OK;
    // (the places of a tile's rows and columns are 32-bit ints, behind the last row too)
    AG_REQUIRE(M <= 0x7fffffff - 512 && N <= 0x7fffffff - 512, AG_ERR_INVALID_DIMS, "%s: operands of %d and %d rows", who, M, N);
    const long long tiles = (long long)((M + f.tile - 1) / f.tile) * ((N + f.tile - 1) / f.tile) * f.splits;
    AG_REQUIRE(tiles <= kMaxThreadsX / (f.tile == 256 ? 512 : 256), AG_ERR_INVALID_DIMS, "%s: too many tiles (%lld)", who, tiles);
    return AG_OK;
}

template <int MT, int NW, int XR>
static void launch_skinny_waves(hipStream_t st, GemmE4m3 p, const float *x, long long ldx, int K)
{
    // columns as many at a time as a launch holds
    constexpr int most = (int)(kMaxThreadsX / (NW * 64) * 16 < 0x7ffffff0LL ? kMaxThreadsX / (NW * 64) * 16 : 0x7ffffff0LL);
    const int N = p.N;
    for (int done = 0;; done += most) {
        p.N = N - done < most ? N - done : most;
        hipLaunchKernelGGL((gemm_e4m3_skinny_kernel<MT, NW, XR>), dim3((unsigned)((p.N + 15) / 16)), dim3(NW * 64), 0, st, p, x, ldx, K);
        if (N - done <= most) return;
        p.b += most * p.pitch;
        p.b_scales += (long long)most * p.scale_pitch;
        p.c += most;
    }
}
template <int MT, int XR>
static void launch_skinny(hipStream_t st, const GemmE4m3 &p, const float *x, long long ldx, int K)
{
    const int words = (p.blocks + 3) / 4;  // a wave each, up to eight
    if (words <= 2) launch_skinny_waves<MT, 2, XR>(st, p, x, ldx, K);
    else if (words <= 4) launch_skinny_waves<MT, 4, XR>(st, p, x, ldx, K);
    else launch_skinny_waves<MT, 8, XR>(st, p, x, ldx, K);
}

static ag_status_t product(const char *who, hipStream_t st, GemmE4m3 p, int K, void *ws)
{
    const Plan f = plan_product(p.M, p.N, K);
    if (f.tile == 0) {
        if (p.M <= 16) launch_skinny<1, 0>(st, p, nullptr, 0, K);
        else launch_skinny<2, 0>(st, p, nullptr, 0, K);
        return check_launch(who);
    }
    p.tiles_m = (p.M + f.tile - 1) / f.tile;
    p.tiles_n = (p.N + f.tile - 1) / f.tile;
    p.splits = f.splits;
    p.per_split = (p.blocks + f.splits - 1) / f.splits;
    const unsigned grid = (unsigned)p.tiles_m * p.tiles_n * f.splits;
    float *c = p.c;
    const long long ldc = p.ldc;
    if (f.splits > 1) p.c = static_cast<float *>(ws), p.ldc = p.N;
    if (f.tile == 256)
        hipLaunchKernelGGL((gemm_e4m3_tile_kernel<256, 256, 128, 64, 2>), dim3(grid), dim3(512), 0, st, p);
    else if (f.tile == 128 && f.deep)
        hipLaunchKernelGGL((gemm_e4m3_tile_kernel<128, 128, 64, 64, 4>), dim3(grid), dim3(256), 0, st, p);
    else if (f.tile == 128)
        hipLaunchKernelGGL((gemm_e4m3_tile_kernel<128, 128, 64, 64, 2>), dim3(grid), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((gemm_e4m3_tile_kernel<64, 64, 32, 32, 4>), dim3(grid), dim3(256), 0, st, p);
    if (f.splits > 1) {
        const long long cells = (long long)p.M * p.N;
        hipLaunchKernelGGL(gemm_e4m3_fold_kernel, dim3((unsigned)((cells + 1023) / 1024)), dim3(256), 0, st, static_cast<const float *>(ws), c, ldc, p.M,
                           p.N, f.splits);
    }
    return check_launch(who);
}

static GemmE4m3 params(int M, int N, int K, const unsigned char *a, const unsigned char *as, const unsigned char *b, const unsigned char *bs, float *c,
                       int ldc)
{
    GemmE4m3 p = {a, as, b, bs, c, ldc, (long long)e4m3_pitch(K), M, N, (int)(e4m3_pitch(K) / kE4m3Block), (int)e4m3_scale_pitch(K), 0, 0, 1, 0};
    return p;
}

// Workspace of the product from f32: the rounded x and its scales, then the product's own.
static size_t rounded_bytes(int M, int K) { return (size_t)M * e4m3_pitch(K) + ((size_t)M * e4m3_scale_pitch(K) + 15) / 16 * 16; }

// Few enough rows of x that each block rounds them for itself.
static bool rounds_in_place(int M) { return M <= kRoundedRows; }

}  // namespace ag

using namespace ag;

extern "C" size_t ag_matmul_e4m3_f32_workspace(int M, int N, int K) { return product_workspace(M, N, K); }

extern "C" ag_status_t ag_matmul_e4m3_f32(ag_stream_t stream, int M, int N, int K, const uint8_t *A, const uint8_t *a_scales, const uint8_t *B,
                                          const uint8_t *b_scales, float *C, int ldc, void *ws, size_t ws_bytes)
{
    const ag_status_t e = check_product("matmul_e4m3", M, N, K, ldc, B, b_scales, C);
    if (e != AG_OK) return e;
    if (M == 0 || N == 0) return AG_OK;
    AG_REQUIRE(K == 0 || (A && a_scales), AG_ERR_INVALID_DIMS, "matmul_e4m3: null pointer");
    AG_REQUIRE(aligned16(A), AG_ERR_INVALID_DIMS, "matmul_e4m3: 8-bit operands must be 16-byte aligned");
    AG_REQUIRE((reinterpret_cast<uintptr_t>(a_scales) & 3u) == 0, AG_ERR_INVALID_DIMS, "matmul_e4m3: scales must be 4-byte aligned");
    const size_t need = product_workspace(M, N, K);
    AG_REQUIRE(need == 0 || (ws && ws_bytes >= need), AG_ERR_INVALID_DIMS, "matmul_e4m3: workspace of %zu bytes, %zu needed", ws_bytes, need);
    AG_REQUIRE(need == 0 || aligned16(ws), AG_ERR_INVALID_DIMS, "matmul_e4m3: misaligned workspace");
    return product("matmul_e4m3", as_stream(stream), params(M, N, K, A, a_scales, B, b_scales, C, ldc), K, ws);
}

extern "C" size_t ag_quantize_matmul_e4m3_f32_workspace(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || rounds_in_place(M)) return 0;
    return rounded_bytes(M, K) + product_workspace(M, N, K);
}

extern "C" ag_status_t ag_quantize_matmul_e4m3_f32(ag_stream_t stream, int M, int N, int K, const float *x, int ldx, const uint8_t *B,
                                                   const uint8_t *b_scales, float *C, int ldc, void *ws, size_t ws_bytes)
{
    ag_status_t e = check_product("quantize_matmul_e4m3", M, N, K, ldc, B, b_scales, C);
    if (e != AG_OK) return e;
    AG_REQUIRE(ldx >= K, AG_ERR_INCOMPATIBLE_SHAPE, "quantize_matmul_e4m3: ldx (%d) is less than a row of %d elements", ldx, K);
    if (M == 0 || N == 0) return AG_OK;
    AG_REQUIRE(K == 0 || x, AG_ERR_INVALID_DIMS, "quantize_matmul_e4m3: null pointer");
    const size_t need = ag_quantize_matmul_e4m3_f32_workspace(M, N, K);
    AG_REQUIRE(need == 0 || (ws && ws_bytes >= need), AG_ERR_INVALID_DIMS, "quantize_matmul_e4m3: workspace of %zu bytes, %zu needed", ws_bytes, need);
    AG_REQUIRE(need == 0 || aligned16(ws), AG_ERR_INVALID_DIMS, "quantize_matmul_e4m3: misaligned workspace");
    hipStream_t st = as_stream(stream);
    if (rounds_in_place(M)) {
        launch_skinny<1, kRoundedRows>(st, params(M, N, K, nullptr, nullptr, B, b_scales, C, ldc), x, ldx, K);
        return check_launch("quantize_matmul_e4m3");
    }
    unsigned char *q = static_cast<unsigned char *>(ws), *scales = q + (size_t)M * e4m3_pitch(K);
    e = quantize_e4m3("quantize_matmul_e4m3", st, x, ldx, M, K, q, scales, nullptr, nullptr);
    if (e != AG_OK) return e;
    return product("quantize_matmul_e4m3", st, params(M, N, K, q, scales, B, b_scales, C, ldc), K, q + rounded_bytes(M, K));
}
