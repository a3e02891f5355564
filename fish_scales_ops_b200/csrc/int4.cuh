// Linear layers over 4-bit weights with one scale (and, where the checkpoint has them, one zero point) for each group of
// consecutive weights of a row:
//
//   y[t, n] = sum over groups j of  scale[n, j] * sum over k in j of (code[n, k] - zero[n, j]) * x[t, k]
//
// The difference code - zero is a whole number of at most 5 bits and enters its product exactly; sums are fp32 and the
// scale is applied to them in fp32. Codes lie in 32-bit words of eight consecutive k, rows of K/2 bytes; inside a word
// the even k take the lower four nibbles in their order and the odd k the upper four, so that one mask yields the pair (k, k + 1)
// in the two halves of a register.
//
// Bound by the bytes of the weights (half a byte and the scales) for the few rows of x that a decode step has.
#pragma once

#include "gated.cuh"

namespace fso {

struct Int4Params {
    const void* bias;      // [out_cols], 16 bit like x, or nullptr
    void* out;             // 16 bit [m, out_cols]
    int scale_type;        // 0 bf16, 1 fp16, 2 fp32
    int has_zero;          // otherwise 8
    int m, k;
    int chunk_rows;        // rows of x of a CTA, at most N
    int group_shift;       // log2 of the group size
    int rows0, rows1;      // rows of the first and of the second half of the weight
    int half_cols;         // columns of scale and zero from one half to the other
    int out_cols;          // rows of the weight, or half of them when gated
    int gated;
    int act;
    int steps;             // 256-wide steps of the contraction
    int whole;             // CTAs at the front of the grid that take the whole contraction of a tile
    int splits;            // CTAs of a cluster, which share a tile of the others
    int steps_per_slice;
};

// Eight codes of a word to the eight 16-bit numbers code - zero (bf16: a 64th of that), exactly, with one shift, four masks and
// four multiply-adds; register i gets k = 2 i and 2 i + 1 of the word.
//
// fp16: a code in the low bits of the mantissa of 1024 is 1024 + code, the next one in the ten bits 1024 + 16 code; the first
// less 1024 + zero, and a sixteenth of the second less 64 + zero, are exact.
// bf16 has seven bits of mantissa, too few for two codes. But the bits of the smallest numbers are linear across the border of
// normal ones: the lower eight bits alone, read as bf16, are that whole number times 2^-133. Times 2^127 (the second code, which
// stands 16 times higher, times 2^123) and less zero / 64 it is (code - zero) / 64; the 64 comes back with the sums.
constexpr float kInt4Unit = 64.f;

template <bool kBf16>
struct Int4Zero {
    uint32_t first, second;      // what is taken away from either, twice

    __device__ __forceinline__ void set(uint32_t z)
    {
        if constexpr (kBf16) {
            uint32_t const bits = z * 0x10001u, scale = 0x7F007F00u;
            __nv_bfloat162 const v = __hmul2(*reinterpret_cast<__nv_bfloat162 const*>(&bits), *reinterpret_cast<__nv_bfloat162 const*>(&scale));
            first = second = *reinterpret_cast<uint32_t const*>(&v);
        } else {
            first = 0x64006400u + z * 0x10001u;        // 1024 + zero
            second = 0x54005400u + z * 0x100010u;      // 64 + zero
        }
    }
};

template <bool kBf16>
__device__ __forceinline__ void int4_unpack(uint32_t w, Int4Zero<kBf16> const& zero, uint32_t* r)
{
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        uint32_t const at = w >> (4 * i);
        if constexpr (kBf16) {
            uint32_t const lo = at & 0x000F000Fu, hi = at & 0x00F000F0u, m0 = 0x7F007F00u, m1 = 0x7D007D00u;      // 2^127, 2^123
            __nv_bfloat162 const z = __hneg2(*reinterpret_cast<__nv_bfloat162 const*>(&zero.first));
            __nv_bfloat162 const d = __hfma2(*reinterpret_cast<__nv_bfloat162 const*>(&lo), *reinterpret_cast<__nv_bfloat162 const*>(&m0), z);
            __nv_bfloat162 const e = __hfma2(*reinterpret_cast<__nv_bfloat162 const*>(&hi), *reinterpret_cast<__nv_bfloat162 const*>(&m1), z);
            r[i] = *reinterpret_cast<uint32_t const*>(&d);
            r[i + 1] = *reinterpret_cast<uint32_t const*>(&e);
        } else {
            uint32_t lo, hi;
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(lo) : "r"(at), "n"(0x000F000F), "n"(0x64006400));      // (a & b) | c
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(hi) : "r"(at), "n"(0x00F000F0), "n"(0x64006400));
            __half2 const d = __hsub2(*reinterpret_cast<__half2 const*>(&lo), *reinterpret_cast<__half2 const*>(&zero.first));
            __half2 const e = __hfma2(*reinterpret_cast<__half2 const*>(&hi), __float2half2_rn(0.0625f),
                __hneg2(*reinterpret_cast<__half2 const*>(&zero.second)));
            r[i] = *reinterpret_cast<uint32_t const*>(&d);
            r[i + 1] = *reinterpret_cast<uint32_t const*>(&e);
        }
    }
}

__device__ __forceinline__ uint32_t lds_u16(uint32_t saddr)
{
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(saddr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t lds_u32(uint32_t saddr)
{
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(saddr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t lds_u8(uint32_t saddr)
{
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(saddr) : "memory");
    return v;
}

__device__ __forceinline__ uint4 lds_v4(uint32_t saddr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(saddr) : "memory");
    return v;
}

// Whole warp: 32 lanes x 32 consecutive 32-bit columns of tensor memory, lane i of the warp to lane (base lane + i).
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, uint32_t const (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t* r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem], kind::f16, one CTA. One thread.
__device__ __forceinline__ void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int N, int U>
struct Int4Cfg {
    static constexpr int kWorkers = 8;                   // warps that unpack and drain
    static constexpr int kThreads = 64 + 32 * kWorkers;  // TMA, MMA, workers
    static constexpr int kStep = 256;                    // of the contraction in a stage
    static constexpr int kCodeBytes = 128 * kStep / 2;
    static constexpr int kXBytes = N * kStep * 2;        // four tiles of N rows x 64 elements
    static constexpr int kScaleOff = kCodeBytes + kXBytes;       // [half][group][64 rows], of at most 4 bytes
    static constexpr int kZeroOff = kScaleOff + 2 * U * 64 * 4;
    static constexpr int kStageBytes = (kZeroOff + 2 * U * 64 + 1023) / 1024 * 1024;
    // up to three: a fourth, where it fits, saves one row 2 % on 28672 x 4096 and costs it 5 % on 4096 x 14336
    static constexpr int kStages = (109 * 1024) / kStageBytes < 3 ? (109 * 1024) / kStageBytes : 3;
    static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 512;
    // tensor memory: the unpacked weights of a step (256 elements, 128 columns), then two buffers of group accumulators
    static constexpr int kDCols = 64;
    static constexpr int kTmemCols = 256;                // two CTAs share an SM's 512
    static constexpr int kRedStride = 132;               // floats between the rows of x in the sums
    static_assert(kStages >= 2, "pipeline depth");
    static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
    static_assert(N * kRedStride * 4 <= kStages * kStageBytes, "the sums fit the stages");
};

// Up to N rows of x (the columns of the MMA) against 128 rows of the weight, 64 of each half, so that the gate row and the up
// row of an output meet in one CTA.
//
// The weight bytes are the bound, so they are streamed by TMA, about 100 KB of an SM's on their way, and what has to be done to
// a weight is kept below the time that its half byte takes: a worker reads 32 codes with one load, turns a word of
// eight into four registers with nine instructions (with eleven, three of them shifts, one row on 28672 x 4096 takes
// 17.8 us instead of 16.0) and stores them to tensor memory, where the MMA (kind::f16) takes its A operand from; with A in
// shared memory the same MMA takes 40 cycles instead of 10 (N = 16), more than the bytes do. Every group has an accumulator of
// its own, which the workers scale in fp32 into their registers. The CTAs of a cluster split the contraction of a tile
// where tiles are few or do not come out even, and each adds up a part of the outputs over distributed shared memory, in
// a fixed order.
//
// What a step costs beside the unpacking (waits, arrivals, scales, addresses: as many instructions as the unpacking itself)
// is paid once for 256 of the contraction, 0.9 us for two CTAs of an SM; one buffer of unpacked weights is enough, since the
// MMAs of a step take less than the unpacking of the next. 28672 x 4096, groups of 128 with zero points: 14.9 us for one
// row (4.1 TB/s), 17.0 for 20 (groups of 64: 16.7 for 16), 24.1 for 48, 37888 x 8192 29.4 (5.5 TB/s).
//
// U: units of a step that have sums of their own: its groups, or two halves of 128 where a group is longer.
template <bool kBf16, int N, int U>
__global__ void __launch_bounds__(Int4Cfg<N, U>::kThreads, 2)
int4_kernel(const __grid_constant__ CUtensorMap tm_lo, const __grid_constant__ CUtensorMap tm_hi,
    const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_scale, const __grid_constant__ CUtensorMap tm_zero,
    const Int4Params p)
{
    using C = Int4Cfg<N, U>;
    constexpr int S = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint32_t const raw = smem_u32(smem_raw);
    uint32_t const base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    uint32_t const bars = base + S * C::kStageBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    uint32_t const afull_bar = bars + 16u * S, aempty_bar = afull_bar + 8;
    auto dfull_bar = [&](int d) { return bars + 16u * S + 16 + 8u * d; };
    auto dempty_bar = [&](int d) { return bars + 16u * S + 32 + 8u * d; };
    uint32_t const misc = S * C::kStageBytes + 16 * S + 48;
    // accumulators of so many units share a buffer, a wait and an arrival
    constexpr int UB = U < C::kDCols / N || (N <= 32 && U * N <= 2 * C::kDCols) ? U : C::kDCols / N;
    static_assert(UB >= 1 && U % UB == 0, "batches of units");
    // More than one batch: the MMAs of a step fill both buffers and go on when the workers have drained one. Where that is not all
    // of the step, the workers drain it before they wait for its weights to be done with; otherwise after they have
    // stored the next ones.
    constexpr bool kDrainFirst = U / UB > 2;
    // One batch a step (up to 32 rows; with more, one buffer for it takes 4 % more time than two batches): its end is the end of
    // the step's MMAs, so that the workers' one wait for it, before they store the next weights, answers for both, and the
    // buffer of two steps ago is drained before they hand these over.
    constexpr bool kOneBatch = U == UB;
    constexpr bool kOneBuffer = UB * N > C::kDCols;      // drained before the next weights are handed over
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + misc);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + misc + 4);

    int const warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    int const lane = threadIdx.x & 31;
    int const bx = blockIdx.x;
    bool const split = bx >= p.whole;
    int const splits = split ? p.splits : 1;
    int const tile = split ? p.whole + (bx - p.whole) / p.splits : bx;
    int const rank = split ? (bx - p.whole) % p.splits : 0;
    int const step0 = split ? rank * p.steps_per_slice : 0;
    int const step1 = split ? min(p.steps, step0 + p.steps_per_slice) : p.steps;
    int const t0 = blockIdx.y * p.chunk_rows;
    int const rows = min(p.chunk_rows, p.m - t0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), kOneBatch ? 1 : C::kWorkers + 1);
        }
        mbar_init(afull_bar, C::kWorkers);
        mbar_init(aempty_bar, 1);
        for (int d = 0; d < 2; ++d) {
            mbar_init(dfull_bar(d), 1);
            mbar_init(dempty_bar(d), C::kWorkers);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t const tmem = *tmem_slot;
    griddep_launch_dependents();

    if (warp == 0) {
        // -------------------------------------------------------------------------------- TMA: the weight (immutable bytes, they
        // are fetched under the preceding kernel) and x
        if (elect_one()) {
            int const row0 = tile * 64;
            int const box_groups = max(1, C::kStep >> p.group_shift);
            uint32_t const scale_bytes = box_groups * 64 * (p.scale_type == 2 ? 4 : 2), zero_bytes = box_groups * 64;
            uint32_t const bytes = C::kCodeBytes + p.chunk_rows * (C::kStep * 2) + 2 * scale_bytes + (p.has_zero ? 2 * zero_bytes : 0);
            auto load_weight = [&](int stage, int st) {
                uint32_t const fb = full_bar(stage), dst = base + stage * C::kStageBytes;
                int const g0 = (st * C::kStep) >> p.group_shift;
                mbar_expect_tx(fb, bytes);
                tma_load_2d(dst, &tm_lo, fb, st * (C::kStep / 2), row0);
                tma_load_2d(dst + 8192, &tm_hi, fb, st * (C::kStep / 2), row0);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tma_load_2d(dst + C::kScaleOff + h * (U * 256), &tm_scale, fb, row0 + h * p.half_cols, g0);
                    if (p.has_zero) tma_load_2d(dst + C::kZeroOff + h * (U * 64), &tm_zero, fb, row0 + h * p.half_cols, g0);
                }
            };
            auto load_x = [&](int stage, int st) {
                uint32_t const dst = base + stage * C::kStageBytes + C::kCodeBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) tma_load_2d(dst + i * (N * 128), &tm_x, full_bar(stage), st * C::kStep + i * 64, t0);
            };
            int const npre = min(S, step1 - step0);      // the first stages are free
            for (int i = 0; i < npre; ++i) load_weight(i, step0 + i);
            griddep_wait();
            for (int i = 0; i < npre; ++i) load_x(i, step0 + i);
            int stage = npre == S ? 0 : npre;
            uint32_t phase = npre == S ? 1u : 0u;
            for (int st = step0 + npre; st < step1; ++st) {
                if (!wait_or_abort(empty_bar(stage), phase ^ 1u, abort_flag)) {
                    record_abort(FSO_DEV_WAIT_PRODUCER, abort_flag);
                    break;
                }
                load_weight(stage, st);
                load_x(stage, st);
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------------------------------------- MMA
        if (elect_one()) {
            constexpr uint32_t idesc = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | ((128u >> 4) << 24);
            int stage = 0, dbuf = 0;
            uint32_t phase = 0, aphase = 0, dphase = 0;
            bool ok = true;
            for (int st = step0; ok && st < step1; ++st) {
                if (!wait_or_abort(full_bar(stage), phase, abort_flag) || !wait_or_abort(afull_bar, aphase, abort_flag)) {
                    record_abort(FSO_DEV_WAIT_MMA_FULL, abort_flag);
                    break;
                }
                uint64_t const bdesc = make_desc_sw128(base + stage * C::kStageBytes + C::kCodeBytes);
#pragma unroll
                for (int j = 0; j < U / UB; ++j) {
                    if (!kOneBatch && !wait_or_abort(dempty_bar(dbuf), dphase ^ 1u, abort_flag)) {
                        record_abort(FSO_DEV_WAIT_MMA_TMEM, abort_flag);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 16 * UB / U; ++i) {
                        int const kk = j * (16 * UB / U) + i;      // 16 elements of the contraction
                        int const unit = i / (16 / U);
                        tc_mma_f16_ta(tmem + 128 + dbuf * C::kDCols + unit * N, tmem + kk * 8,
                            bdesc + static_cast<uint64_t>((kk >> 2) * (N * 128 / 16) + 2 * (kk & 3)), idesc, i % (16 / U) > 0 ? 1u : 0u);
                    }
                    if constexpr (!kOneBatch) tc_commit(dfull_bar(dbuf));
                    dbuf ^= kOneBuffer ? 0 : 1;
                    dphase ^= dbuf ^ 1;
                }
                if (!ok) break;
                tc_commit(aempty_bar);
                tc_commit(empty_bar(stage));
                aphase ^= 1u;
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else {
        // -------------------------------------------------------------------------------- workers: lane = row of the weight; the two
        // warps of a quarter share its codes by halves of a step and its sums by halves of the rows of x
        int const quarter = warp & 3, hh = (warp - 2) >> 2;
        int const row = quarter * 32 + lane, in_half = row & 63, half = row >> 6;
        uint32_t const lanes = static_cast<uint32_t>(quarter * 32) << 16;
        uint32_t const code_row = half * 8192 + in_half * 128;
        uint32_t const scale_width = p.scale_type == 2 ? 4 : 2;
        uint32_t const scale_row = C::kScaleOff + half * (U * 256) + in_half * scale_width, zero_row = C::kZeroOff + half * (U * 64) + in_half;
        int const unit_mask = U == 2 && p.group_shift >= 8 ? 0 : U - 1;      // units that share a longer group
        constexpr int kCols = N / 2;
        float acc[kCols] = {};
        float scale_next[U], scale_now[U];
        int stage = 0, dbuf = 0;
        uint32_t phase = 0, aphase = 0, dphase = 0;

        auto drain = [&]() -> bool {      // the units of the step before, scaled
#pragma unroll
            for (int j = 0; j < U; j += UB) {
                if constexpr (!kOneBatch) {
                    if (!wait_or_abort(dfull_bar(dbuf), dphase, abort_flag)) {
                        if (lane == 0) record_abort(FSO_DEV_WAIT_EPILOGUE, abort_flag);
                        return false;
                    }
                    __syncwarp();
                    tc_fence_after();
                }
                constexpr int kAtOnce = kOneBuffer ? 1 : UB;      // units in registers
#pragma unroll
                for (int v = 0; v < UB; v += kAtOnce) {
                    uint32_t r[kAtOnce * kCols];
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                        for (int c = 0; c < kCols; c += 8)
                            tmem_ld_32x8(tmem + lanes + 128 + dbuf * C::kDCols + (v + u) * N + hh * kCols + c, r + u * kCols + c);
                    tmem_ld_wait();
                    if constexpr (!kOneBatch) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(dempty_bar(dbuf));
                    }
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                        for (int c = 0; c < kCols; ++c) acc[c] = fmaf(scale_now[j + v + u], __uint_as_float(r[u * kCols + c]), acc[c]);
                }
                dbuf ^= kOneBuffer ? 0 : 1;
                dphase ^= dbuf ^ 1;
            }
            return true;
        };

        bool ok = true;
        for (int st = step0; ok && st < step1; ++st) {
            if (!wait_or_abort(full_bar(stage), phase, abort_flag)) {
                if (lane == 0) record_abort(FSO_DEV_WAIT_MMA_FULL, abort_flag);
                ok = false;
                break;
            }
            __syncwarp();
            uint32_t const src = base + stage * C::kStageBytes;
            // By branches that the whole grid takes alike up to 32 rows (one row on 28672 x 4096: 4 % less time); beyond, where
            // registers are short, both halves of an fp32 scale are read always (48 rows: 3 % less time than with branches).
            if constexpr (N > 32) {
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    uint32_t const at = src + scale_row + (j & unit_mask) * 64 * scale_width;
                    uint32_t const upper = lds_u16(at + scale_width - 2), lower = lds_u16(at);
                    scale_next[j] = p.scale_type == 1 ? __half2float(__ushort_as_half(static_cast<uint16_t>(upper)))
                                                      : __uint_as_float(upper << 16 | (p.scale_type == 2 ? lower : 0u));
                }
            } else if (p.scale_type == 2) {
#pragma unroll
                for (int j = 0; j < U; ++j) scale_next[j] = __uint_as_float(lds_u32(src + scale_row + (j & unit_mask) * 256));
            } else {
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    uint32_t const v = lds_u16(src + scale_row + (j & unit_mask) * 128);
                    scale_next[j] = p.scale_type == 1 ? __half2float(__ushort_as_half(static_cast<uint16_t>(v))) : __uint_as_float(v << 16);
                }
            }
            constexpr int kZeros = U / 2;      // groups of this worker's 128
            Int4Zero<kBf16> zero[kZeros];
#pragma unroll
            for (int q = 0; q < kZeros; ++q) {
                uint32_t const at = src + zero_row + ((hh * kZeros + q) & unit_mask) * 64;
                uint32_t z = 8u;
                if constexpr (N > 16) {
                    uint32_t const stored = lds_u8(at);
                    z = p.has_zero ? stored : 8u;
                } else {
                    if (p.has_zero) z = lds_u8(at);
                }
                zero[q].set(z);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {      // 64 of the contraction
                int const part = 2 * hh + b;
                uint4 const c0 = lds_v4(src + code_row + (((2 * part) ^ (in_half & 7)) << 4));
                uint4 const c1 = lds_v4(src + code_row + (((2 * part + 1) ^ (in_half & 7)) << 4));
                uint32_t a[32];
                uint32_t const words[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) int4_unpack<kBf16>(words[j], zero[(8 * b + j) * kZeros >> 4], a + 4 * j);
                if (b == 0) {
                    if constexpr (kDrainFirst) {
                        if (st > step0 && !drain()) {
                            ok = false;
                            break;
                        }
                    }
                    if (!wait_or_abort(aempty_bar, aphase ^ 1u, abort_flag)) {
                        if (lane == 0) record_abort(FSO_DEV_WAIT_MMA_TMEM, abort_flag);
                        ok = false;
                        break;
                    }
                    __syncwarp();
                    tc_fence_after();
                    if constexpr (kOneBuffer) {
                        if (st > step0) drain();
                    }
                }
                tmem_st_32x32(tmem + lanes + part * 32, a);
            }
            if (!ok) break;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(afull_bar);
                if constexpr (!kOneBatch) mbar_arrive(empty_bar(stage));
            }
            aphase ^= 1u;
            if (++stage == S) {
                stage = 0;
                phase ^= 1u;
            }
            if constexpr (!kDrainFirst && !kOneBuffer) {
                if (st > step0) ok = drain();
            }
#pragma unroll
            for (int j = 0; j < U; ++j) scale_now[j] = scale_next[j];
        }
        if (ok && step1 > step0) {
            if (kOneBatch && !wait_or_abort(aempty_bar, aphase ^ 1u, abort_flag)) {
                if (lane == 0) record_abort(FSO_DEV_WAIT_EPILOGUE, abort_flag);
                ok = false;
            }
            __syncwarp();
            tc_fence_after();
            if (ok) ok = drain();
        }
        // every MMA and every copy is done: the sums of this slice go where the stages were
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::kWorkers) : "memory");
        if (ok) {
            float* const red = reinterpret_cast<float*>(gbase);
#pragma unroll
            for (int c = 0; c < kCols; ++c) red[(hh * kCols + c) * C::kRedStride + row] = kBf16 ? kInt4Unit * acc[c] : acc[c];
        }
    }
    __syncthreads();
    bool const failed = *abort_flag != 0;
    if (failed) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);      // copies in flight land before the memory is given up
        __syncthreads();
    }
    if (splits > 1) cluster_sync_all();
    griddep_wait();      // the memory of the outputs may have been in use by the preceding kernel
    if (!failed) {
        float const* const red = reinterpret_cast<float const*>(gbase);
        uint32_t const red_addr = smem_u32(red);
        auto sum_of = [&](int r, int c) {
            if (splits == 1) return red[r * C::kRedStride + c];
            float part[8], v = 0.f;      // all loads first: one trip to the other CTAs' memory instead of one for each
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < splits) part[i] = ld_cluster_f32(map_to_cta(red_addr + 4u * (r * C::kRedStride + c), i));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < splits) v += part[i];
            return v;
        };
        int const cols = p.gated ? 64 : 128;
        for (int i = rank * C::kThreads + static_cast<int>(threadIdx.x); i < rows * cols; i += C::kThreads * splits) {
            int const r = p.gated ? i >> 6 : i >> 7, c = p.gated ? i & 63 : i & 127;
            int const half = c >> 6, in_half = tile * 64 + (c & 63);
            if (in_half >= (half ? p.rows1 : p.rows0)) continue;
            int const to = half * p.rows0 + in_half;
            float v = sum_of(r, c);
            if (p.gated) v = gate_value(v, p.act) * sum_of(r, c + 64);
            else if (p.bias != nullptr) v += load16<kBf16>(p.bias, to);
            store16<kBf16>(p.out, static_cast<int64_t>(t0 + r) * p.out_cols + to, v);
        }
    }
    __syncwarp();
    if (splits > 1) cluster_sync_all();      // no CTA leaves while another may still read its sums
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------ the order of the codes

// Eight nibbles in the order of k -> the order of the kernels.
__device__ __forceinline__ uint32_t int4_word(uint32_t w)
{
    uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
    even = (even | even >> 4) & 0x00FF00FFu;
    odd = (odd | odd >> 4) & 0x00FF00FFu;
    return ((even | even >> 8) & 0xFFFFu) | (odd | odd >> 8) << 16;
}

__global__ void int4_pack_kernel(const uint4* __restrict__ in, uint4* __restrict__ out, int64_t vectors)
{
    int64_t const i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= vectors) return;
    uint4 const v = in[i];
    out[i] = make_uint4(int4_word(v.x), int4_word(v.y), int4_word(v.z), int4_word(v.w));
}

// ------------------------------------------------------------------------------------------------ 16-bit weight -> 4 bits
//
// A group is group / 8 neighbouring lanes of eight weights each. Steps are amax / 7 around code 8, or (hi - lo) / 15 with
// zero inside [lo, hi] and the zero point next to -lo / step; the step is rounded to its stored type first, so that the
// codes are the nearest ones for the scale that will multiply them. A group whose step rounds to zero gets code = zero, one
// with a NaN or an infinity a scale that is not a number, so that its row's products show it.
__device__ __forceinline__ float stored_scale(float v, int type)
{
    if (type == 0) return __bfloat162float(__float2bfloat16_rn(v));
    if (type == 1) return __half2float(__float2half_rn(v));
    return v;
}

template <bool kBf16>
__global__ void int4_quantize_kernel(const uint4* __restrict__ w, uint32_t* __restrict__ codes, void* __restrict__ scale,
    int scale_type, uint8_t* __restrict__ zero, int64_t vectors, int lanes, int64_t rows0, int64_t half_cols, int groups)
{
    int64_t const i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    bool const live = i < vectors;      // groups are whole: all lanes of one are live or none is
    uint4 const q = live ? w[i] : make_uint4(0, 0, 0, 0);
    uint32_t const words[4] = {q.x, q.y, q.z, q.w};
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 const f = unpack16<kBf16>(words[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
    float lo = 0.f, hi = 0.f, nan = 0.f;      // minima and maxima pass over a NaN: 0 * v keeps it
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, v[j]);
        hi = fmaxf(hi, v[j]);
        nan += 0.f * v[j];
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        nan += __shfl_xor_sync(0xffffffffu, nan, o);
    }
    float const step = stored_scale((zero != nullptr ? (hi - lo) / 15.f : fmaxf(-lo, hi) / 7.f) + nan, scale_type);
    int const z = zero == nullptr ? 8 : step > 0.f ? min(15, max(0, __float2int_rn(-lo / step))) : 0;
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int const c = step > 0.f ? min(15, max(0, z + __float2int_rn(v[j] / step))) : z;
        packed |= static_cast<uint32_t>(c) << (4 * j);
    }
    if (!live) return;
    codes[i] = int4_word(packed);
    if (i % lanes == 0) {
        int64_t const row_group = i / lanes, row = row_group / groups;
        int64_t const g = (row_group - row * groups) * 2 * half_cols + (row < rows0 ? row : half_cols + row - rows0);
        if (scale_type == 0) store16<true>(scale, g, step);
        else if (scale_type == 1) store16<false>(scale, g, step);
        else static_cast<float*>(scale)[g] = step;
        if (zero != nullptr) zero[g] = static_cast<uint8_t>(z);
    }
}

// Tensor map of the codes [rows, k / 2] in boxes of 128 bytes x 64 rows with the 128-byte swizzle.
inline int make_codes_map(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t k)
{
    return make_operand_map(map, codes, rows, k / 2, 64);
}

// Tensor map of scale or zero [groups, 2 * half_cols] in boxes of 64 rows of the weight x box_groups.
inline int make_steps_map(CUtensorMap* map, const void* base, int64_t groups, int64_t half_cols, int width, int box_groups)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) {
        set_error("cuTensorMapEncodeTiled is not available from this driver");
        return FSO_ERR_UNSUPPORTED;
    }
    cuuint64_t const dims[2] = {static_cast<cuuint64_t>(2 * half_cols), static_cast<cuuint64_t>(groups)};
    cuuint64_t const strides[1] = {static_cast<cuuint64_t>(2 * half_cols * width)};
    cuuint32_t const box[2] = {64u, static_cast<cuuint32_t>(box_groups)};
    cuuint32_t const estr[2] = {1u, 1u};
    CUtensorMapDataType const type = width == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : width == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                                                          : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    CUresult const r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with CUresult %d (scales, %lld groups)", static_cast<int>(r),
            static_cast<long long>(groups));
        return FSO_ERR_INTERNAL;
    }
    return 0;
}

inline int64_t int4_half_cols(int64_t rows) { return ((rows + 1) / 2 + 15) / 16 * 16; }

// CTAs for `tiles` tiles on SMs that hold two CTAs each. Fewer tiles than SMs: clusters split every tile, as far as all of them
// are resident and a slice keeps two steps (eight is the portable cluster size). 48 tiles of 16 steps take a third
// less time in 48 clusters of four (6.3 us) than in clusters of six, of which 45 fit. From there to two tiles for each SM: pairs split as
// many tiles as fill the places that one CTA for each tile would leave. More: the last tiles are split, so that the
// end of the last round is short.
inline unsigned int4_schedule(int tiles, int sms, int const (&clusters)[9], Int4Params& p)
{
    int const places = 2 * sms;
    p.whole = 0;
    p.splits = 1;
    int best = p.steps;
    if (tiles <= sms) {
        for (int c = 2; c <= 8 && 2 * c <= p.steps; ++c) {
            int const per = (p.steps + c - 1) / c;
            if (tiles <= clusters[c] && per < best) {      // in no more CTAs than that slice needs: none is empty
                best = per;
                p.splits = c;
            }
        }
    } else if (p.steps >= 4) {
        p.splits = 2;
        p.whole = tiles <= places ? 2 * tiles - places : (tiles - std::min(tiles, sms)) & ~1;
    }
    p.steps_per_slice = (p.steps + p.splits - 1) / p.splits;
    return static_cast<unsigned>(p.whole + (tiles - p.whole) * p.splits);
}

template <bool kBf16, int N, int U>
inline int launch_int4_inst(CUtensorMap const (&maps)[5], Int4Params const& p, dim3 grid, cudaStream_t stream)
{
    using C = Int4Cfg<N, U>;
    static std::atomic<uint64_t> done{0};
    auto kernel = int4_kernel<kBf16, N, U>;
    int const rc = ensure_smem_attr(kernel, C::kSmemBytes, done);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(p.splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + pdl_attribute(&attr[1]);
    FSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], maps[4], p));
    return launch_status("int4_kernel");
}

template <bool kBf16, int N>
inline int launch_int4_group(int64_t group, CUtensorMap const (&maps)[5], Int4Params const& p, dim3 grid, cudaStream_t stream)
{
    return group == 32 ? launch_int4_inst<kBf16, N, 8>(maps, p, grid, stream)
        : group == 64 ? launch_int4_inst<kBf16, N, 4>(maps, p, grid, stream)
                      : launch_int4_inst<kBf16, N, 2>(maps, p, grid, stream);
}

template <bool kBf16>
inline int launch_int4_rows(int n, int64_t group, CUtensorMap const (&maps)[5], Int4Params const& p, dim3 grid, cudaStream_t stream)
{
    return n == 16 ? launch_int4_group<kBf16, 16>(group, maps, p, grid, stream)
        : n == 32  ? launch_int4_group<kBf16, 32>(group, maps, p, grid, stream)
        : n == 48  ? launch_int4_group<kBf16, 48>(group, maps, p, grid, stream)
                   : launch_int4_group<kBf16, 64>(group, maps, p, grid, stream);
}

// p: scale_type, bias, out, m, k, out_cols, gated and act; the rest is derived here. More than 64 rows of x go in equal parts.
inline int launch_int4(Int4Params p, const void* x, int64_t ldx, int64_t rows, const void* codes, const void* scale, const void* zero,
    int64_t group, bool bf16, cudaStream_t stream)
{
    p.group_shift = 0;
    while ((1ll << p.group_shift) < group) ++p.group_shift;
    p.has_zero = zero != nullptr;
    p.rows0 = static_cast<int>((rows + 1) / 2);
    p.rows1 = static_cast<int>(rows - p.rows0);
    p.half_cols = static_cast<int>(int4_half_cols(rows));
    p.steps = (p.k + 255) / 256;
    int const chunks = (p.m + 63) / 64;
    p.chunk_rows = (p.m + chunks - 1) / chunks;
    int const n = (p.chunk_rows + 15) / 16 * 16;
    int const box_groups = static_cast<int>(std::max<int64_t>(1, 256 / group));
    int64_t const groups = p.k >> p.group_shift;
    uint8_t const* const c = static_cast<uint8_t const*>(codes);
    CUtensorMap maps[5];
    int rc = make_codes_map(&maps[0], c, p.rows0, p.k);
    maps[1] = maps[0];      // a weight of one row has no second half: what is read in its place goes nowhere
    if (rc == 0 && p.rows1 > 0) rc = make_codes_map(&maps[1], c + static_cast<int64_t>(p.rows0) * (p.k / 2), p.rows1, p.k);
    // x in boxes of as many rows as there are: to fill the rest of a tile with zeros costs TMA time (one row on 28672 x 4096: 15.0
    // us, 16.0 with 15 rows of zeros). What lies in its place goes into sums that nobody reads.
    if (rc == 0) rc = make_map16(&maps[2], x, p.m, p.k, ldx, p.chunk_rows);
    if (rc == 0) rc = make_steps_map(&maps[3], scale, groups, p.half_cols, p.scale_type == 2 ? 4 : 2, box_groups);
    maps[4] = maps[3];
    if (rc == 0 && p.has_zero) rc = make_steps_map(&maps[4], zero, groups, p.half_cols, 1, box_groups);
    if (rc != 0) return rc;
    int clusters[9];
    rc = resident_clusters(2, clusters);
    if (rc != 0) return rc;
    dim3 const grid(int4_schedule((p.rows0 + 63) / 64, sm_count(), clusters, p), static_cast<unsigned>(chunks));
    return bf16 ? launch_int4_rows<true>(n, group, maps, p, grid, stream) : launch_int4_rows<false>(n, group, maps, p, grid, stream);
}

}  // namespace fso
