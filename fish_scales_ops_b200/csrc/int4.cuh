// Linear layers over 4-bit weights with one scale (and, where the checkpoint has them, one zero point) for each group of
// consecutive weights of a row:
//
//   y[t, n] = sum over groups j of  scale[n, j] * sum over k in j of (code[n, k] - zero[n, j]) * x[t, k]
//
// The difference code - zero is a whole number of at most 5 bits and enters its product exactly; sums are fp32 and the
// scale is applied to them in fp32. Codes lie two in a byte, the even k in the lower four bits, rows of K/2 bytes.
//
// Bound by the bytes of the weights (half a byte and the scales) for the few rows of x that a decode step has.
#pragma once

#include "gated.cuh"

namespace fso {

struct Int4Params {
    const void* x;         // 16 bit [m, ldx]
    int64_t ldx;
    int scale_type;        // 0 bf16, 1 fp16, 2 fp32
    int has_zero;          // otherwise 8
    const void* bias;      // [out_cols], 16 bit like x, or nullptr
    void* out;             // 16 bit [m, out_cols]
    int m, k;
    int group_shift;       // log2 of the group size
    int rows0, rows1;      // rows of the first and of the second half of the weight
    int half_cols;         // columns of scale and zero from one half to the other
    int out_cols;          // rows of the weight, or half of them when gated
    int gated;
    int act;
    int steps;             // 512-wide steps of the contraction
    int steps_per_slice;
    int splits;            // slices of the contraction = CTAs of a cluster
};

// Eight codes of a word to the eight 16-bit numbers code - zero, exactly: a code in the low bits of the mantissa of 128
// (bf16) or 1024 (fp16) is 128 + code, and taking away 128 + zero is exact. Register i gets the codes i and i + 4, which
// lie 16 bits apart. `zero2` is that minuend twice.
template <bool kBf16>
__device__ __forceinline__ void int4_unpack(uint32_t w, uint32_t zero2, uint32_t (&r)[4])
{
    constexpr uint32_t kOne = kBf16 ? 0x43004300u : 0x64006400u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "n"(0x000F000F), "n"(kOne));      // (a & b) | c
        if constexpr (kBf16) {
            __nv_bfloat162 const d = __hsub2(*reinterpret_cast<__nv_bfloat162 const*>(&v), *reinterpret_cast<__nv_bfloat162 const*>(&zero2));
            r[i] = *reinterpret_cast<uint32_t const*>(&d);
        } else {
            __half2 const d = __hsub2(*reinterpret_cast<__half2 const*>(&v), *reinterpret_cast<__half2 const*>(&zero2));
            r[i] = *reinterpret_cast<uint32_t const*>(&d);
        }
    }
}

// c += A (16 rows x 16 of the contraction) * B (16 x 8 columns), fp32 sums, one warp.
template <bool kBf16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
    uint32_t b1)
{
    if constexpr (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t saddr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}

__device__ __forceinline__ uint32_t lds_u16(uint32_t saddr)
{
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(saddr) : "memory");
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

template <int NT>
struct Int4Cfg {
    static constexpr int kRT = 2;                // 16-row tiles of a warp
    static constexpr int kRows = 64;             // weight rows of a CTA, 32 of each half of the weight
    static constexpr int kStep = 512;            // of the contraction in a stage, 128 for a warp
    static constexpr int kWarps = 16 / kRT;             // four along the contraction, two along the rows
    static constexpr int kThreads = 32 * kWarps + 32;
    static constexpr int kStages = NT == 1 ? 3 : 2;
    static constexpr int kBlocks = 2;
    static constexpr int kWeightBytes = kRows * kStep / 2;
    static constexpr int kXBytes = 8 * NT * kStep * 2;
    static constexpr int kScaleOff = kWeightBytes + kXBytes;                  // [half][group][32 rows], at most 16 groups
    static constexpr int kZeroOff = kScaleOff + 2 * 16 * 32 * 4;
    static constexpr int kStageBytes = kZeroOff + 2 * 16 * 32;                // 16 KB of codes, x, 4 KB + 1 KB
    static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
    static constexpr int kRedStride = kRows + 4; // floats between the rows of x in the partial sums: lanes hit 32 banks
    static_assert(kBlocks * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

// The few rows of x of a decode step (at most 8 * NT in a CTA) against 64 rows of the weight.
//
// Bound by the weight bytes, so they are streamed by TMA, 48 to 64 KB deep and two CTAs to an SM, and everything else is
// sized to stay below the time of a stage. A warp turns its codes into tensor-core fragments in registers
// (mma.sync: the 16-row side is the weight, eight rows of x are one tile; decode never fills a tcgen05 tile, and the
// codes would have to go through shared memory once more to get there). ldmatrix hands a lane the word that holds
// the eight codes k = 8 t .. 8 t + 7 of its weight row; any order of the contraction will do as long as x follows it, so the
// pairs (i, i + 4) that the masks give are met by permuted registers of x. The sums of a group are scaled in fp32 as
// they leave the tensor cores. Four pairs of warps split a stage along the contraction and add up at the end; the CTAs
// of a cluster split it further where rows are few, and each adds up a part of the outputs over distributed shared
// memory, in a fixed order.
//
// GC: 32-wide chunks of a group inside the 128 of a warp (4 for groups of 128 and more).
template <bool kBf16, int NT, int GC>
__global__ void __launch_bounds__(Int4Cfg<NT>::kThreads, Int4Cfg<NT>::kBlocks)
int4_rows_kernel(const __grid_constant__ CUtensorMap tm_lo, const __grid_constant__ CUtensorMap tm_hi,
    const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_scale,
    const __grid_constant__ CUtensorMap tm_zero, const Int4Params p)
{
    using C = Int4Cfg<NT>;
    constexpr int S = C::kStages;
    constexpr int G = 4 / GC;      // groups of a warp and stage
    extern __shared__ uint8_t smem_raw[];
    uint32_t const raw = smem_u32(smem_raw);
    uint32_t const base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    uint32_t const bars = base + S * C::kStageBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + S * C::kStageBytes + 16 * S);

    int const warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    int const lane = threadIdx.x & 31;
    int const tile = blockIdx.x / p.splits;
    int const rank = blockIdx.x - tile * p.splits;
    int const step0 = rank * p.steps_per_slice;
    int const step1 = min(p.steps, step0 + p.steps_per_slice);
    int const t0 = blockIdx.y * (8 * NT);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), C::kWarps);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    griddep_launch_dependents();

    constexpr int RT = C::kRT;
    int const kq = warp & 3, rh = RT == 4 ? 0 : (warp >> 2) & 1;      // this warp's quarter of a step and half of the rows
    float tot[RT][NT][4] = {};
    if (warp == C::kWarps) {
        // -------------------------------------------------------------------------------- weight stream (immutable bytes:
        // it starts under the preceding kernel)
        if (elect_one()) {
            int const row0 = tile * 32;
            int const box_groups = max(1, C::kStep >> p.group_shift);
            uint32_t const scale_bytes = box_groups * 32 * (p.scale_type == 2 ? 4 : 2), zero_bytes = box_groups * 32;
            uint32_t const bytes = C::kWeightBytes + C::kXBytes + 2 * scale_bytes + (p.has_zero ? 2 * zero_bytes : 0);
            auto load_weight = [&](int stage, int st) {
                uint32_t const fb = full_bar(stage), dst = base + stage * C::kStageBytes;
                int const g0 = (st * C::kStep) >> p.group_shift;
                mbar_expect_tx(fb, bytes);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    tma_load_2d(dst + b * 8192, &tm_lo, fb, st * (C::kStep / 2) + b * 128, row0);
                    tma_load_2d(dst + b * 8192 + 4096, &tm_hi, fb, st * (C::kStep / 2) + b * 128, row0);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tma_load_2d(dst + C::kScaleOff + h * 2048, &tm_scale, fb, row0 + h * p.half_cols, g0);
                    if (p.has_zero) tma_load_2d(dst + C::kZeroOff + h * 512, &tm_zero, fb, row0 + h * p.half_cols, g0);
                }
            };
            auto load_x = [&](int stage, int st) {
                uint32_t const dst = base + stage * C::kStageBytes + C::kWeightBytes;
#pragma unroll
                for (int b = 0; b < 8; ++b)
                    tma_load_2d(dst + b * (1024 * NT), &tm_x, full_bar(stage), st * C::kStep + b * 64, t0);
            };
            // the first stages are free; x may still be in the making
            int const npre = min(S, step1 - step0);
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
    } else {
        int const g = lane >> 2, t = lane & 3;
        // ldmatrix: lanes 8 i .. 8 i + 7 give the rows of matrix i: rows 0-7 and 8-15 of a chunk, then of the next chunk
        uint32_t const mrow = ((lane >> 3) & 1) * 8 + (lane & 7);
        uint32_t const mchunk = (kq & 1) * 4 + (lane >> 4);
        uint32_t const moff = (kq >> 1) * 8192 + rh * 4096 + mrow * 128;
        uint32_t const moff0 = moff + ((mchunk ^ (lane & 7)) << 4), moff2 = moff + (((mchunk + 2) ^ (lane & 7)) << 4);

        // B fragments: lane (g, t) takes row g of x and the elements 8 t .. 8 t + 7 of each chunk
        uint32_t const xoff = C::kWeightBytes + kq * 2048 * NT + g * 128;
        uint32_t const xoff0 = xoff + ((t ^ g) << 4), xoff1 = xoff + (((4 + t) ^ g) << 4);

        // scales and zero points of a row and group: lane (g, t) needs those of rows g and g + 8 of each 16
        uint32_t const scale_width = p.scale_type == 2 ? 4 : 2;
        int const group0 = (kq * 128) >> p.group_shift;      // of this warp inside a stage (0 where a group spans stages)
        // (no branch on the kinds of scale and zero point: a stage stays one block of instructions, whose loads the compiler
        // moves ahead of the products)
        auto scale_of = [&](uint32_t sbase, int row, int j) -> float {      // row 0..63 of the tile
            uint32_t const at = sbase + C::kScaleOff + (row >> 5) * 2048 + ((group0 + j) * 32 + (row & 31)) * scale_width;
            uint32_t const upper = lds_u16(at + scale_width - 2), lower = lds_u16(at);
            return p.scale_type == 1 ? __half2float(__ushort_as_half(static_cast<uint16_t>(upper)))
                                     : __uint_as_float(upper << 16 | (p.scale_type == 2 ? lower : 0u));
        };
        auto zero_of = [&](uint32_t sbase, int row, int j) -> uint32_t {
            uint32_t const z = lds_u8(sbase + C::kZeroOff + (row >> 5) * 512 + (group0 + j) * 32 + (row & 31));
            return ((kBf16 ? 0x4300u : 0x6400u) + (p.has_zero ? z : 8u)) * 0x10001u;
        };
        int stage = 0;
        uint32_t phase = 0;
        for (int st = step0; st < step1; ++st) {
            if (!wait_or_abort(full_bar(stage), phase, abort_flag)) {
                if (lane == 0) record_abort(FSO_DEV_WAIT_MMA_FULL, abort_flag);
                break;
            }
            __syncwarp();
            uint32_t const sbase = base + stage * C::kStageBytes;
            uint32_t w[RT][2][4];      // [row tile][chunks 0, 1 or 2, 3]: row g and row g + 8 of the first, then of the second
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                ldmatrix_x4(sbase + moff0 + rt * 2048, w[rt][0]);
                ldmatrix_x4(sbase + moff2 + rt * 2048, w[rt][1]);
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float acc[RT][NT][4] = {};
                uint32_t zero2[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int q = 0; q < 2; ++q) zero2[rt][q] = zero_of(sbase, rh * 32 + rt * 16 + q * 8 + g, j);
#pragma unroll
                for (int cc = 0; cc < GC; ++cc) {
                    int const c = j * GC + cc;
                    uint32_t bx[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint4 const v = lds_v4(sbase + (c & 1 ? xoff1 : xoff0) + (c >> 1) * 1024 * NT + n * 1024);
                        bx[n][0] = __byte_perm(v.x, v.z, 0x5410);      // elements 0 and 4
                        bx[n][1] = __byte_perm(v.x, v.z, 0x7632);      // 1 and 5
                        bx[n][2] = __byte_perm(v.y, v.w, 0x5410);      // 2 and 6
                        bx[n][3] = __byte_perm(v.y, v.w, 0x7632);      // 3 and 7
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        uint32_t a[4], b[4];      // row g, row g + 8
                        int4_unpack<kBf16>(w[rt][c >> 1][2 * (c & 1)], zero2[rt][0], a);
                        int4_unpack<kBf16>(w[rt][c >> 1][2 * (c & 1) + 1], zero2[rt][1], b);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16x8x16<kBf16>(acc[rt][n], a[0], b[0], a[1], b[1], bx[n][0], bx[n][1]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16x8x16<kBf16>(acc[rt][n], a[2], b[2], a[3], b[3], bx[n][2], bx[n][3]);
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float const s0 = scale_of(sbase, rh * 32 + rt * 16 + g, j), s8 = scale_of(sbase, rh * 32 + rt * 16 + 8 + g, j);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        tot[rt][n][0] = fmaf(s0, acc[rt][n][0], tot[rt][n][0]);
                        tot[rt][n][1] = fmaf(s0, acc[rt][n][1], tot[rt][n][1]);
                        tot[rt][n][2] = fmaf(s8, acc[rt][n][2], tot[rt][n][2]);
                        tot[rt][n][3] = fmaf(s8, acc[rt][n][3], tot[rt][n][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty_bar(stage));
            if (++stage == S) {
                stage = 0;
                phase ^= 1u;
            }
        }
    }

    // ---------------------------------------------------------------------------------------- sums of the warps and slices
    __syncthreads();      // every stage has been read: the ring becomes [quarter][row of x][weight row]
    bool const failed = *abort_flag != 0;
    if (failed) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);      // copies in flight land before the memory is given up
        __syncthreads();
    }
    float* const red = reinterpret_cast<float*>(gbase);
    constexpr int kWarpFloats = 8 * NT * C::kRedStride;
    static_assert(4 * kWarpFloats * 4 <= S * C::kStageBytes, "partial sums fit the ring");
    if (warp < C::kWarps) {
        int const g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    red[kq * kWarpFloats + (8 * n + 2 * t + (q & 1)) * C::kRedStride + rh * 32 + rt * 16 + g + 8 * (q >> 1)] = tot[rt][n][q];
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    griddep_wait();      // the memory of the outputs may have been in use by the preceding kernel
    if (warp < C::kWarps && !failed) {
        int const cols = p.gated ? 32 : 64;
        int const rows = min(8 * NT, p.m - t0);
        uint32_t const red_addr = smem_u32(red);
        auto sum_of = [&](int row, int col) {
            float v = 0.f;
            if (p.splits == 1) {
#pragma unroll
                for (int w = 0; w < 4; ++w) v += red[w * kWarpFloats + row * C::kRedStride + col];
                return v;
            }
            for (int r = 0; r < p.splits; ++r) {
                uint32_t const peer = map_to_cta(red_addr + 4u * (row * C::kRedStride + col), r);
#pragma unroll
                for (int w = 0; w < 4; ++w) v += ld_cluster_f32(peer + 4u * (w * kWarpFloats));
            }
            return v;
        };
        for (int i = rank * 32 * C::kWarps + static_cast<int>(threadIdx.x); i < rows * cols; i += 32 * C::kWarps * p.splits) {
            int const row = i / cols, in_tile = i - row * cols;
            int const half = in_tile >> 5, in_half = tile * 32 + (in_tile & 31);      // row of the half
            if (in_half >= (half ? p.rows1 : p.rows0)) continue;
            int const col = half * p.rows0 + in_half;
            float v = sum_of(row, in_tile);
            if (p.gated) v = gate_value(v, p.act) * sum_of(row, in_tile + 32);
            else if (p.bias != nullptr) v += load16<kBf16>(p.bias, col);
            store16<kBf16>(p.out, static_cast<int64_t>(t0 + row) * p.out_cols + col, v);
        }
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync_all();      // no CTA leaves while another may still read its sums
}

// ------------------------------------------------------------------------------------------------ 16-bit weight -> 4 bits
//
// A group is group / 8 neighbouring lanes of eight weights each. Steps are amax / 7 around code 8, or (hi - lo) / 15 with
// zero inside [lo, hi] and the zero point next to -lo / step; the step is rounded to its stored type first, so that the
// codes are the nearest ones for the scale that will multiply them. A group whose step rounds to zero gets code = zero.
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
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, v[j]);
        hi = fmaxf(hi, v[j]);
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float const step = stored_scale(zero != nullptr ? (hi - lo) / 15.f : fmaxf(-lo, hi) / 7.f, scale_type);
    int const z = zero == nullptr ? 8 : step > 0.f ? min(15, max(0, __float2int_rn(-lo / step))) : 0;
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int const c = step > 0.f ? min(15, max(0, z + __float2int_rn(v[j] / step))) : z;
        packed |= static_cast<uint32_t>(c) << (4 * j);
    }
    if (!live) return;
    codes[i] = packed;
    if (i % lanes == 0) {
        int64_t const row_group = i / lanes, row = row_group / groups;
        int64_t const g = (row_group - row * groups) * 2 * half_cols + (row < rows0 ? row : half_cols + row - rows0);
        if (scale_type == 0) store16<true>(scale, g, step);
        else if (scale_type == 1) store16<false>(scale, g, step);
        else static_cast<float*>(scale)[g] = step;
        if (zero != nullptr) zero[g] = static_cast<uint8_t>(z);
    }
}

// Tensor map of the codes [rows, k / 2] in boxes of 128 bytes x box_rows with the 128-byte swizzle.
inline int make_codes_map(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t k, int box_rows)
{
    return make_operand_map(map, codes, rows, k / 2, box_rows);
}

// Slices of the contraction for `tiles` CTAs' worth of rows: as many as it takes for all SMs to have CTAs (two fit), at
// most eight (the portable cluster size), and no empty one.
inline void int4_slices(int64_t tiles, int sms, Int4Params& p)
{
    int s = 1;
    while (s < 8 && tiles * s * 2 <= 3 * sms && s * 2 <= p.steps) ++s;
    p.steps_per_slice = (p.steps + s - 1) / s;
    p.splits = (p.steps + p.steps_per_slice - 1) / p.steps_per_slice;
}

template <bool kBf16, int NT, int GC>
inline int launch_int4_inst(CUtensorMap const (&maps)[5], Int4Params const& p, dim3 grid, cudaStream_t stream)
{
    static std::atomic<uint64_t> done{0};
    using C = Int4Cfg<NT>;
    auto kernel = int4_rows_kernel<kBf16, NT, GC>;
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
    return launch_status("int4_rows_kernel");
}

template <bool kBf16, int NT>
inline int launch_int4_group(int group, CUtensorMap const (&maps)[5], Int4Params const& p, dim3 grid,
    cudaStream_t stream)
{
    return group == 32 ? launch_int4_inst<kBf16, NT, 1>(maps, p, grid, stream)
        : group == 64 ? launch_int4_inst<kBf16, NT, 2>(maps, p, grid, stream)
                      : launch_int4_inst<kBf16, NT, 4>(maps, p, grid, stream);
}

// Tensor map of scale or zero [groups, 2 * half_cols] in boxes of 32 rows of the weight x box_groups.
inline int make_steps_map(CUtensorMap* map, const void* base, int64_t groups, int64_t half_cols, int width, int box_groups)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) {
        set_error("cuTensorMapEncodeTiled is not available from this driver");
        return FSO_ERR_UNSUPPORTED;
    }
    cuuint64_t const dims[2] = {static_cast<cuuint64_t>(2 * half_cols), static_cast<cuuint64_t>(groups)};
    cuuint64_t const strides[1] = {static_cast<cuuint64_t>(2 * half_cols * width)};
    cuuint32_t const box[2] = {32u, static_cast<cuuint32_t>(box_groups)};
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

// p: x, ldx, scale_type, bias, out, m, k, out_cols, gated and act; the rest is derived here.
inline int launch_int4(Int4Params p, int64_t rows, const uint8_t* codes, const void* scale, const void* zero, int64_t group,
    bool bf16, cudaStream_t stream)
{
    p.group_shift = 0;
    while ((1ll << p.group_shift) < group) ++p.group_shift;
    p.has_zero = zero != nullptr;
    p.rows0 = static_cast<int>((rows + 1) / 2);
    p.rows1 = static_cast<int>(rows - p.rows0);
    p.half_cols = static_cast<int>(int4_half_cols(rows));
    p.steps = (p.k + Int4Cfg<1>::kStep - 1) / Int4Cfg<1>::kStep;
    int const tiles = (p.rows0 + 31) / 32;
    int4_slices(tiles, sm_count(), p);
    int const nt = p.m <= 8 ? 1 : 2;
    int const box_groups = static_cast<int>(std::max<int64_t>(1, Int4Cfg<1>::kStep / group));
    int64_t const groups = p.k >> p.group_shift;
    CUtensorMap maps[5];
    int rc = make_codes_map(&maps[0], codes, p.rows0, p.k, 32);
    maps[1] = maps[0];      // a weight of one row has no second half: what is read in its place goes nowhere
    if (rc == 0 && p.rows1 > 0) rc = make_codes_map(&maps[1], codes + static_cast<int64_t>(p.rows0) * (p.k / 2), p.rows1, p.k, 32);
    if (rc == 0) rc = make_map16(&maps[2], p.x, p.m, p.k, p.ldx, 8 * nt);
    if (rc == 0) rc = make_steps_map(&maps[3], scale, groups, p.half_cols, p.scale_type == 2 ? 4 : 2, box_groups);
    maps[4] = maps[3];
    if (rc == 0 && p.has_zero) rc = make_steps_map(&maps[4], zero, groups, p.half_cols, 1, box_groups);
    if (rc != 0) return rc;
    dim3 const grid(static_cast<unsigned>(tiles * p.splits), static_cast<unsigned>((p.m + 8 * nt - 1) / (8 * nt)));
    int const gi = static_cast<int>(std::min<int64_t>(group, 128));
    if (bf16) return nt == 1 ? launch_int4_group<true, 1>(gi, maps, p, grid, stream) : launch_int4_group<true, 2>(gi, maps, p, grid, stream);
    return nt == 1 ? launch_int4_group<false, 1>(gi, maps, p, grid, stream) : launch_int4_group<false, 2>(gi, maps, p, grid, stream);
}

}  // namespace fso
