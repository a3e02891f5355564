// The gated feed-forward projection in 16 bits, h = act(x G^T) * (x U^T), and its gradients, on CTA pairs:
//
//   forward    g = x G^T, u = x U^T            A = x, B = rows of G and U side by side; act and product in the epilogue
//   dx         dg G + du U                     A = [dg | du], B = [G ; U], the two halves of the contraction in turn
//   dG, dU     dg^T x, du^T x                  A = dg^T or du^T, B = x
//
// with dg = dh * u * act'(g), du = dh * act(g) (gated_slopes_kernel). All are a 256 x 256 tile for each pair of CTAs
// (tcgen05.mma kind::f16, cta_group::2, fp32 accumulators in tensor memory), fed by TMA. The operand whose contraction
// runs down its columns (G, U in dx; all operands of dG, dU) is staged as it lies in memory and read by the tensor
// cores "M/N-major": nothing is transposed in memory. The two products of the backward pass share one launch, so that the
// tiles of one fill the rounds that the other leaves open.
//
// What bounds it: the tensor pipe for T from a few hundred on (an MMA of 256 x 256 x 16 takes 128 cycles), the weight
// bytes below that. T = K = 4096, INTER = 7168 in bf16, in bursts: forward 302 us (1590 TFLOP/s), dx 323, dG and dU 303, the tensor
// pipe 94 to 98 % busy; T = 8192, INTER = 14336 back to back at 1.1 to 1.25 GHz under the power cap: forward 1370 to 1400 us,
// 1500 with saved projections.
#pragma once

#include <cmath>
#include <cuda_fp16.h>

#include "gemm_host.cuh"

namespace fso {

enum : int { G16_FORWARD = 0, G16_BACKWARD = 1 };
enum : int { FSO_ACT_SILU = 0, FSO_ACT_GELU = 1, FSO_ACT_GELU_TANH = 2 };

struct Gated16Cfg {
    static constexpr int kStages = 6;
    static constexpr int kEpiWarps = 8;
    static constexpr int kThreads = 128 + 32 * kEpiWarps;
    static constexpr int kOpBytes = 128 * 128;          // one operand of one CTA and stage: 128 rows x 64 elements
    static constexpr int kStageBytes = 2 * kOpBytes;
    static constexpr int kTurnBytes = 32 * 128;         // of each epilogue warp: 32 rows x 128 bytes on their way out
    static constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * kTurnBytes + 1024 + 512;
    static constexpr int kTmemCols = 512;               // two accumulators of 256 columns
    static_assert(kSmemBytes <= 227 * 1024 && kSmemBytes > 116 * 1024, "one CTA per SM");
};

// One product: its tiles, the slices of its contraction and its output.
struct Gated16Product {
    int rows;            // valid rows of the output (dW: of one half)
    int cols;            // valid columns of the output
    int tiles_m;         // 256-row tiles (dW: of both halves)
    int tiles_n;
    int group_m;         // raster: row tiles walked together before the columns advance
    int kb_total;        // 64-wide blocks of the contraction
    int kb_half;         // dx: blocks of the first half; dW: 256-row tiles of one half
    int splits;
    int kb_per_split;
    int vec;             // rows of `out` start on 16-byte boundaries
    void* out;           // 16 bit [rows, ldo]
    int64_t ldo;
    int64_t out_half;    // dW: elements from the first half's output to the second's
    float* ws;           // splits > 1: fp32 sums [splits, rows, ws_cols] (dW: [splits, 2, rows, ws_cols])
    int64_t ws_cols;
};

struct Gated16Params {
    Gated16Product first, second;      // forward: first alone; backward: in either order, tiles_m = 0 where one is not wanted
    int first_is_dw;
    uint16_t* save_hi;   // forward: upper 16 of the 24 bits kept of g and u, [rows, 2 * half_cols], or nullptr
    uint8_t* save_lo;    // forward: lower 8 bits
    int64_t half_cols;   // columns from g to u in the saved arrays and in split sums
};

// ------------------------------------------------------------------------------------------------ activations
//
// a = act(g) and s = act'(g), from act(g) = g P(g): P is the logistic function of g (silu), the normal distribution
// function (gelu), or the logistic function of 2 z, z = sqrt(2/pi) (g + 0.044715 g^3), which is 0.5 (1 + tanh z).
// The logistic function goes through the exponential and an approximate division (2 ulp; zero past 2^126, where the
// function is below 1e-37), so its relative error stays below 1e-5 in both tails; 16-bit outputs cannot see it. 1 - P
// in the slopes loses digits only where it is added to P next to 1.
__device__ __forceinline__ float logistic(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

constexpr float kGeluC = 0.79788456080286535588f;      // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

template <int ACT>
__device__ __forceinline__ float gate_value_of(float g)
{
    if constexpr (ACT == FSO_ACT_SILU) return g * logistic(g);
    else if constexpr (ACT == FSO_ACT_GELU) return g * normcdff(g);
    else return g * logistic(2.f * kGeluC * (g + kGeluCubic * g * g * g));
}

__device__ __forceinline__ float gate_value(float g, int act)
{
    if (act == FSO_ACT_SILU) return gate_value_of<FSO_ACT_SILU>(g);
    if (act == FSO_ACT_GELU) return gate_value_of<FSO_ACT_GELU>(g);
    return gate_value_of<FSO_ACT_GELU_TANH>(g);
}

template <int ACT>
__device__ __forceinline__ void gate_value_slope(float g, float& a, float& s)
{
    float p, dp;      // dp = g P'(g)
    if constexpr (ACT == FSO_ACT_SILU) {
        p = logistic(g);
        dp = g * p * (1.f - p);
    } else if constexpr (ACT == FSO_ACT_GELU) {
        p = normcdff(g);
        dp = g * 0.39894228040143267794f * __expf(-0.5f * g * g);
    } else {
        p = logistic(2.f * kGeluC * (g + kGeluCubic * g * g * g));
        float const c = fminf(fabsf(g), 30.f);      // p is 0 or 1 long before that, and the square of a large g is infinite
        dp = g * p * (1.f - p) * 2.f * kGeluC * (1.f + 3.f * kGeluCubic * c * c);
    }
    a = g * p;
    s = p + dp;
}

// ------------------------------------------------------------------------------------------------ 16-bit and 24-bit values

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi)
{
    if constexpr (kBf16) {
        __nv_bfloat162 const v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t const*>(&v);
    } else {
        __half2 const v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t const*>(&v);
    }
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack16(uint32_t w)
{
    if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<__half2 const*>(&w));
}

template <bool kBf16>
__device__ __forceinline__ float load16(const void* p, int64_t i)
{
    if constexpr (kBf16) return __bfloat162float(static_cast<__nv_bfloat16 const*>(p)[i]);
    else return __half2float(static_cast<__half const*>(p)[i]);
}

template <bool kBf16>
__device__ __forceinline__ void store16(void* p, int64_t i, float v)
{
    if constexpr (kBf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// g and u are kept for the backward pass in 24 bits (the upper 24 of the fp32 value, rounded): in 16 bits their
// rounding would be as large as the one that dg and du go through on the way to the tensor cores and would raise the
// error of the gradients by a quarter; three bytes instead of four cost the pass less memory and traffic.
// Only finite values are rounded up: an infinity or a NaN keeps its upper bits, and a NaN keeps its quiet bit there.
__device__ __forceinline__ uint32_t to_24(float v)
{
    uint32_t const b = __float_as_uint(v);
    return ((b & 0x7F800000u) == 0x7F800000u ? b : b + 0x80u) >> 8;
}

__device__ __forceinline__ float from_24(uint32_t hi, uint32_t lo) { return __uint_as_float((hi << 16) | (lo << 8)); }

// A tile of 32 rows x 16 * kChunks bytes turns in a warp's shared memory: it is held a row to a lane and leaves with
// neighbouring lanes on neighbouring 16-byte chunks of a row, so that whole sectors are written. Chunks are xor-ed with the row:
// both sides of the turn hit all banks.
template <int kChunks>
__device__ __forceinline__ void turn_put(uint32_t turn, int lane, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(turn + lane * (16 * kChunks) + ((chunk ^ ((lane * kChunks / 8) & (kChunks - 1))) << 4)), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}

// Calls to(row, chunk, value) for every chunk of the first `rows` rows.
template <int kChunks, typename To>
__device__ __forceinline__ void turn_out(uint32_t turn, int lane, int rows, To to)
{
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        int const row = i * (32 / kChunks) + lane / kChunks, chunk = lane % kChunks;
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(turn + row * (16 * kChunks) + ((chunk ^ ((row * kChunks / 8) & (kChunks - 1))) << 4))
                     : "memory");
        if (row < rows) to(row, chunk, v);
    }
    __syncwarp();
}

// Four neighbouring g and u of one row: saved values (rows padded to multiples of 16 columns), act and product. `valid`: how
// many of them lie inside the row of the output.
template <bool kBf16>
__device__ __forceinline__ void finish_four(float (&g)[4], float (&u)[4], int act, uint16_t* hi, uint8_t* lo, int64_t at,
    int64_t half_cols, void* out, int64_t to, int valid, bool vec)
{
    if (hi != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = to_24(h ? u[j] : g[j]);
            *reinterpret_cast<uint2*>(hi + at + h * half_cols) =
                make_uint2((b[0] >> 8) | ((b[1] >> 8) << 16), (b[2] >> 8) | ((b[3] >> 8) << 16));
            *reinterpret_cast<uint32_t*>(lo + at + h * half_cols) =
                (b[0] & 0xFFu) | ((b[1] & 0xFFu) << 8) | ((b[2] & 0xFFu) << 16) | (b[3] << 24);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = gate_value(g[j], act) * u[j];
    if (vec && valid >= 4) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + to) = make_uint2(pack16<kBf16>(g[0], g[1]), pack16<kBf16>(g[2], g[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) store16<kBf16>(out, to + j, g[j]);
    }
}

// ------------------------------------------------------------------------------------------------ tensor-core forms

// Instruction descriptor of kind::f16 over a CTA pair: fp32 accumulator, both operands bf16 or both fp16, M = 256,
// N = 256; `a_mn` / `b_mn`: the operand is stored with its M (N) dimension contiguous.
__host__ __device__ constexpr uint32_t make_idesc_f16_pair(bool bf16, bool a_mn, bool b_mn)
{
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u)
        | ((256u >> 3) << 17) | ((256u >> 4) << 24);
}

// Descriptor of an operand tile stored with its M (or N) dimension contiguous: blocks of 64 elements (128 bytes, the
// 128-byte swizzle) x 64 contraction steps, 8 KB each, one block behind the other. Inside a block eight steps are
// 1024 bytes. Advancing by 16 steps adds 2048 bytes.
__device__ __forceinline__ uint64_t make_desc_mn_sw128(uint32_t saddr)
{
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(8192 >> 4) << 16;           // between 64-element blocks
    d |= static_cast<uint64_t>(1024 >> 4) << 32;           // between groups of eight steps
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__device__ __forceinline__ void tc_mma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
    uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// ------------------------------------------------------------------------------------------------ the kernel
//
// The protocol is that of gemm_mxf8_pair_kernel (gemm2.cuh): both CTAs' producers load their own shared memory and
// count bytes on the leader's barrier, the leader issues the MMAs of the pair, each CTA runs its own epilogue. Without
// scale factors two accumulators of 256 columns fill tensor memory, so a tile's epilogue runs under the next tile's
// MMAs. Forward: CTA 0 stages 128 rows of G, CTA 1 the same 128 rows of U, so a CTA's accumulator holds g in columns
// 0..127 and u in columns 128..255 of its own 128 tokens.
// Maps: forward x, G, U (boxes of 128 rows); backward x, G, U, dg, du (boxes of 64 rows).
// ACT: the activation of the forward pass (kernels of their own: with the three of them in one epilogue its code no longer
// fits the instruction cache beside the main loop; 1500 rows on 1032 x 2744 take 33 us that way).
template <int MODE, bool kBf16, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Gated16Cfg::kThreads, 1)
gated16_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_g,
    const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ CUtensorMap tm_dg, const __grid_constant__ CUtensorMap tm_du,
    const Gated16Params p)
{
    using C = Gated16Cfg;
    constexpr int S = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint32_t const raw = smem_u32(smem_raw);
    uint32_t const base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    uint32_t const sA = base;
    uint32_t const sB = sA + S * C::kOpBytes;
    uint32_t const sTurn = sB + S * C::kOpBytes;
    uint32_t const bars = sTurn + C::kEpiWarps * C::kTurnBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * S + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * S + 2 + a); };
    uint32_t const misc_off = static_cast<uint32_t>(S) * C::kStageBytes + C::kEpiWarps * C::kTurnBytes + 8u * (2 * S + 4);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + misc_off);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + misc_off + 4);

    int const warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    int const lane = threadIdx.x & 31;
    uint32_t const rank = cluster_ctarank();
    bool const leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * C::kEpiWarps);
        }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tensormap(&tm_x);
        prefetch_tensormap(&tm_g);
        prefetch_tensormap(&tm_u);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    uint32_t const tmem_base = *tmem_slot;

    int const pair = blockIdx.x >> 1;
    int const num_pairs = gridDim.x >> 1;
    int const items0 = p.first.tiles_m * p.first.tiles_n * p.first.splits;
    int const items = items0 + (MODE == G16_BACKWARD ? p.second.tiles_m * p.second.tiles_n * p.second.splits : 0);

    struct Item {
        int tile_m, tile_n, split, kb0, kb1, half;
        bool dw;
    };
    auto decode = [&](int t) {
        Item c;
        bool const later = MODE == G16_BACKWARD && t >= items0;
        Gated16Product const& q = later ? p.second : p.first;
        c.dw = MODE == G16_BACKWARD && later == (p.first_is_dw == 0);
        if (later) t -= items0;
        int const tiles = q.tiles_m * q.tiles_n;
        c.split = t / tiles;
        int const r = t - c.split * tiles;
        int const span = q.group_m * q.tiles_n;
        int const g = r / span;
        int const first = g * q.group_m;
        int const gsz = min(q.group_m, q.tiles_m - first);
        int const in_g = r - g * span;
        c.tile_n = in_g / gsz;
        c.tile_m = first + (in_g - c.tile_n * gsz);
        c.half = 0;
        if (c.dw) {
            c.half = c.tile_m >= q.kb_half ? 1 : 0;
            c.tile_m -= c.half * q.kb_half;
        }
        c.kb0 = c.split * q.kb_per_split;
        c.kb1 = min(q.kb_total, c.kb0 + q.kb_per_split);
        return c;
    };
    griddep_launch_dependents();
    griddep_wait();      // operands and outputs may be in use by the preceding kernel

    if (warp == 0) {
        // ------------------------------------------------------------------------------------ TMA producer (both CTAs)
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; ok && t < items; t += num_pairs) {
                Item const c = decode(t);
                int const a0 = c.tile_m * 256 + static_cast<int>(rank) * 128;
                int const b0 = MODE == G16_FORWARD ? c.tile_n * 128 : c.tile_n * 256 + static_cast<int>(rank) * 128;
                int const kb_half = MODE == G16_BACKWARD && !c.dw ? (p.first_is_dw ? p.second.kb_half : p.first.kb_half) : 0;
                for (int kb = c.kb0; kb < c.kb1; ++kb) {
                    if (!wait_or_abort(empty_bar(stage), phase ^ 1u, abort_flag)) {
                        record_abort(FSO_DEV_WAIT_PRODUCER, abort_flag);
                        ok = false;
                        break;
                    }
                    uint32_t const fb = map_to_cta(full_bar(stage), 0);
                    if (leader) mbar_expect_tx(full_bar(stage), 2u * C::kStageBytes);
                    uint32_t const da = sA + stage * C::kOpBytes, db = sB + stage * C::kOpBytes;
                    if constexpr (MODE == G16_FORWARD) {
                        tma_load_2d_pair(da, &tm_x, fb, kb * 64, a0);
                        tma_load_2d_pair(db, rank == 0 ? &tm_g : &tm_u, fb, kb * 64, b0);
                    } else if (!c.dw) {
                        bool const upper = kb >= kb_half;
                        int const kc = (upper ? kb - kb_half : kb) * 64;
                        const CUtensorMap* const ta = upper ? &tm_du : &tm_dg;
                        const CUtensorMap* const tb = upper ? &tm_u : &tm_g;
                        tma_load_2d_pair(da, ta, fb, kc, a0);
                        tma_load_2d_pair(da + 8192, ta, fb, kc, a0 + 64);
                        tma_load_2d_pair(db, tb, fb, b0, kc);
                        tma_load_2d_pair(db + 8192, tb, fb, b0 + 64, kc);
                    } else {
                        const CUtensorMap* const ta = c.half ? &tm_du : &tm_dg;
                        tma_load_2d_pair(da, ta, fb, a0, kb * 64);
                        tma_load_2d_pair(da + 8192, ta, fb, a0 + 64, kb * 64);
                        tma_load_2d_pair(db, &tm_x, fb, b0, kb * 64);
                        tma_load_2d_pair(db + 8192, &tm_x, fb, b0 + 64, kb * 64);
                    }
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------ MMA issuer (leader only)
        if (leader && elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int t = pair; ok && t < items; t += num_pairs) {
                Item const c = decode(t);
                if (!wait_or_abort(tempty_bar(acc), acc_phase ^ 1u, abort_flag)) {
                    record_abort(FSO_DEV_WAIT_MMA_TMEM, abort_flag);
                    break;
                }
                tc_fence_after();
                uint32_t const d_tmem = tmem_base + static_cast<uint32_t>(acc * 256);
                for (int kb = c.kb0; kb < c.kb1; ++kb) {
                    if (!wait_or_abort(full_bar(stage), phase, abort_flag)) {
                        record_abort(FSO_DEV_WAIT_MMA_FULL, abort_flag);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    uint32_t const sa = sA + stage * C::kOpBytes, sb = sB + stage * C::kOpBytes;
                    constexpr bool kBmn = MODE == G16_BACKWARD;
                    uint64_t const adesc = c.dw ? make_desc_mn_sw128(sa) : make_desc_sw128(sa);
                    uint64_t const bdesc = kBmn ? make_desc_mn_sw128(sb) : make_desc_sw128(sb);
                    uint32_t const idesc = make_idesc_f16_pair(kBf16, c.dw, kBmn);
                    uint32_t const astep = c.dw ? 128u : 2u;
#pragma unroll
                    for (int k = 0; k < 4; ++k)      // 16 elements of the contraction: 32 bytes of a row, or 16 rows
                        tc_mma_f16_pair(d_tmem, adesc + astep * k, bdesc + (kBmn ? 128u : 2u) * k, idesc,
                            (kb > c.kb0 || k > 0) ? 1u : 0u);
                    tc_commit_pair_both(empty_bar(stage));
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                tc_commit_pair_both(tfull_bar(acc));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------------------------------ epilogue (both CTAs)
        int const quarter = warp & 3;
        int const half = (warp - 4) >> 2;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = pair; t < items; t += num_pairs) {
            Item const c = decode(t);
            if (!wait_or_abort(tfull_bar(acc), acc_phase, abort_flag)) {
                if (lane == 0) record_abort(FSO_DEV_WAIT_EPILOGUE, abort_flag);
                break;
            }
            __syncwarp();      // the loads from tensor memory below are the whole warp's
            tc_fence_after();
            uint32_t const t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * 256);
            Gated16Product const& q = MODE == G16_BACKWARD && c.dw == (p.first_is_dw == 0) ? p.second : p.first;
            int const row0 = c.tile_m * 256 + static_cast<int>(rank) * 128 + quarter * 32;      // of this warp
            int const rows = min(32, q.rows - row0);
            uint32_t const turn = sTurn + (warp - 4) * C::kTurnBytes;
            if constexpr (MODE == G16_FORWARD) {
#pragma unroll 1
                for (int j = 0; j < 2; ++j) {
                    int const in_tile = half * 64 + 32 * j;
                    int const col = c.tile_n * 128 + in_tile;
                    if (col >= q.cols || rows <= 0) break;
                    float g[32], u[32];
                    tmem_ld_32x32(t_row + in_tile, reinterpret_cast<uint32_t(&)[32]>(g));
                    tmem_ld_32x32(t_row + 128 + in_tile, reinterpret_cast<uint32_t(&)[32]>(u));
                    tmem_ld_wait();
                    // columns that exist from `col` on: of the arrays padded to 16, and of the output
                    int const padded = min(32, static_cast<int>(p.half_cols) - col), valid = min(32, q.cols - col);
                    if (q.ws != nullptr) {
                        float* const w = q.ws + (static_cast<int64_t>(c.split) * q.rows + row0) * q.ws_cols + col;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float const (&v)[32] = h ? u : g;
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                turn_put<8>(turn, lane, i, __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                    __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
                            turn_out<8>(turn, lane, rows, [&](int r, int i, uint4 x) {
                                if (4 * i < padded) *reinterpret_cast<uint4*>(w + r * q.ws_cols + h * p.half_cols + 4 * i) = x;
                            });
                        }
                        continue;
                    }
                    if (p.save_hi != nullptr) {
                        int64_t const at = static_cast<int64_t>(row0) * 2 * p.half_cols + col;
                        uint32_t low[16];      // lower bytes of g, then of u
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float const (&v)[32] = h ? u : g;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t b[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) b[e] = to_24(v[8 * i + e]);
                                turn_put<8>(turn, lane, 4 * h + i, (b[0] >> 8) | ((b[1] >> 8) << 16), (b[2] >> 8) | ((b[3] >> 8) << 16),
                                    (b[4] >> 8) | ((b[5] >> 8) << 16), (b[6] >> 8) | ((b[7] >> 8) << 16));
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    low[8 * h + 2 * i + e] = (b[4 * e] & 0xFFu) | ((b[4 * e + 1] & 0xFFu) << 8)
                                        | ((b[4 * e + 2] & 0xFFu) << 16) | (b[4 * e + 3] << 24);
                            }
                        }
                        turn_out<8>(turn, lane, rows, [&](int r, int i, uint4 x) {
                            if (8 * (i & 3) < padded)
                                *reinterpret_cast<uint4*>(p.save_hi + at + r * 2 * p.half_cols + (i >> 2) * p.half_cols + 8 * (i & 3)) = x;
                        });
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            turn_put<4>(turn, lane, i, low[4 * i], low[4 * i + 1], low[4 * i + 2], low[4 * i + 3]);
                        turn_out<4>(turn, lane, rows, [&](int r, int i, uint4 x) {
                            if (16 * (i & 1) < padded)
                                *reinterpret_cast<uint4*>(p.save_lo + at + r * 2 * p.half_cols + (i >> 1) * p.half_cols + 16 * (i & 1)) = x;
                        });
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) g[i] = gate_value_of<ACT>(g[i]) * u[i];
                    if (q.vec) {
                        uint16_t* const to = static_cast<uint16_t*>(q.out) + static_cast<int64_t>(row0) * q.ldo + col;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            turn_put<4>(turn, lane, i, pack16<kBf16>(g[8 * i], g[8 * i + 1]), pack16<kBf16>(g[8 * i + 2], g[8 * i + 3]),
                                pack16<kBf16>(g[8 * i + 4], g[8 * i + 5]), pack16<kBf16>(g[8 * i + 6], g[8 * i + 7]));
                        turn_out<4>(turn, lane, rows, [&](int r, int i, uint4 x) {
                            if (8 * i < valid) *reinterpret_cast<uint4*>(to + r * q.ldo + 8 * i) = x;
                        });
                    } else if (lane < rows) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < valid) store16<kBf16>(q.out, static_cast<int64_t>(row0 + lane) * q.ldo + col + i, g[i]);
                    }
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    int const in_tile = half * 128 + 32 * j;
                    int const col = c.tile_n * 256 + in_tile;
                    if (col >= q.cols || rows <= 0) break;
                    float v[32];
                    tmem_ld_32x32(t_row + in_tile, reinterpret_cast<uint32_t(&)[32]>(v));
                    tmem_ld_wait();
                    int const valid = min(32, q.cols - col);      // a multiple of 8: so is K
                    if (q.ws != nullptr) {
                        int64_t const slab = c.dw ? 2 * c.split + c.half : c.split;
                        float* const w = q.ws + (slab * q.rows + row0) * q.ws_cols + col;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            turn_put<8>(turn, lane, i, __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
                        turn_out<8>(turn, lane, rows, [&](int r, int i, uint4 x) {
                            if (4 * i < valid) *reinterpret_cast<uint4*>(w + r * q.ws_cols + 4 * i) = x;
                        });
                        continue;
                    }
                    uint16_t* const to = static_cast<uint16_t*>(q.out) + c.half * q.out_half + static_cast<int64_t>(row0) * q.ldo + col;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        turn_put<4>(turn, lane, i, pack16<kBf16>(v[8 * i], v[8 * i + 1]), pack16<kBf16>(v[8 * i + 2], v[8 * i + 3]),
                            pack16<kBf16>(v[8 * i + 4], v[8 * i + 5]), pack16<kBf16>(v[8 * i + 6], v[8 * i + 7]));
                    turn_out<4>(turn, lane, rows, [&](int r, int i, uint4 x) {
                        if (8 * i < valid) *reinterpret_cast<uint4*>(to + r * q.ldo + 8 * i) = x;
                    });
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(tempty_bar(acc), 0));
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        __syncwarp();
    }

    // ---------------------------------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, C::kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------ few rows
//
// The forward pass where 256 x 256 tiles are too coarse: 64 rows of G and the same 64 rows of U on MMA-M, up to 256 rows of x
// (a multiple of 16) on MMA-N, one tile for each CTA. Up to 128 rows the weight bytes are the cost, and a deep ring keeps
// more than a hundred kilobytes of an SM's weights on their way: one CTA with all of its shared memory where there is
// one for each SM, two that share it where there are more. Where the tiles leave SMs without work the CTAs of a cluster
// split the contraction, and each adds up its part of the outputs over distributed shared memory, in a fixed order.
// Nothing is read before the preceding kernel has finished: unlike a prepared weight, gate_up may be its output.
// K = 4096, INTER = 14336: 38.6 us for one row (6.1 TB/s), 45 for 128; K = 7168, INTER = 2048: 12.4 and 15.4.
template <int BN>
struct GatedRowsCfg {
    static constexpr int kThreads = 192;       // TMA, MMA, four warps for the accumulators
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = BN * 128;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kBlocks = BN <= 128 ? 2 : 1;      // CTAs that can share an SM
    // stages of a CTA that has its SM to itself, and of one that shares it
    static constexpr int kStagesAlone = (220 * 1024) / kStageBytes;
    static constexpr int kStagesShared = (110 * 1024) / kStageBytes;
    static constexpr int smem_bytes(int stages) { return stages * kStageBytes + 1024 + 512; }
    static constexpr int kRedStride = 132;     // floats between the rows of x in the sums of a slice
    static constexpr int kTmemCols = BN < 32 ? 32 : BN;
    static_assert(smem_bytes(kStagesAlone) + 1024 <= 228 * 1024 && 2 * (smem_bytes(kStagesShared) + 1024) <= 228 * 1024, "shared memory");
    static_assert(16 * kStagesAlone + 16 <= 512, "barriers");
    static_assert(BN * kRedStride * 4 <= (kBlocks == 2 ? kStagesShared : kStagesAlone) * kStageBytes, "the sums fit the stages");
};

struct GatedRowsParams {
    int t, inter, act;
    int n;               // rows of x in a tile, a multiple of 16 and at most BN
    int kb_total, kb_per_split, splits;
    int stages;
    int vec;             // rows of `out` start on 8-byte boundaries
    void* out;
    uint16_t* save_hi;
    uint8_t* save_lo;
    int64_t half_cols;
};

__device__ __forceinline__ void tc_mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr) : "memory");
    return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

template <int BN, bool kBf16>
__global__ void __launch_bounds__(GatedRowsCfg<BN>::kThreads, GatedRowsCfg<BN>::kBlocks)
gated_rows_kernel(const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_u,
    const __grid_constant__ CUtensorMap tm_x, const GatedRowsParams p)
{
    using C = GatedRowsCfg<BN>;
    int const S = p.stages;
    extern __shared__ uint8_t smem_raw[];
    uint32_t const raw = smem_u32(smem_raw);
    uint32_t const base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    uint32_t const sA = base, sB = base + S * C::kABytes;
    uint32_t const bars = base + S * C::kStageBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    uint32_t const done_bar = bars + 16u * S;
    uint32_t const misc = S * C::kStageBytes + 16 * S + 8;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + misc);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + misc + 4);

    int const warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    int const lane = threadIdx.x & 31;
    int const tile = blockIdx.x / p.splits;
    int const rank = blockIdx.x - tile * p.splits;
    int const row0 = blockIdx.y * p.n;
    int const rows = min(p.n, p.t - row0);
    int const kb0 = rank * p.kb_per_split, kb1 = min(p.kb_total, kb0 + p.kb_per_split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
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
    uint32_t const tmem_base = *tmem_slot;
    griddep_launch_dependents();
    griddep_wait();

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_or_abort(empty_bar(stage), phase ^ 1u, abort_flag)) {
                    record_abort(FSO_DEV_WAIT_PRODUCER, abort_flag);
                    break;
                }
                uint32_t const fb = full_bar(stage);
                mbar_expect_tx(fb, C::kABytes + p.n * 128);
                tma_load_2d(sA + stage * C::kABytes, &tm_g, fb, kb * 64, tile * 64);
                tma_load_2d(sA + stage * C::kABytes + 8192, &tm_u, fb, kb * 64, tile * 64);
                tma_load_2d(sB + stage * C::kBBytes, &tm_x, fb, kb * 64, row0);
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t const idesc = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(p.n >> 3) << 17) | ((128u >> 4) << 24);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_or_abort(full_bar(stage), phase, abort_flag)) {
                    record_abort(FSO_DEV_WAIT_MMA_FULL, abort_flag);
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint64_t const adesc = make_desc_sw128(sA + stage * C::kABytes), bdesc = make_desc_sw128(sB + stage * C::kBBytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16(tmem_base, adesc + 2u * k, bdesc + 2u * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                tc_commit(empty_bar(stage));
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok) tc_commit(done_bar);
        }
        __syncwarp();
    } else {
        // the accumulators of a slice to shared memory: every stage has been read by the time they are complete
        if (wait_or_abort(done_bar, 0, abort_flag)) {
            __syncwarp();
            tc_fence_after();
            int const quarter = warp & 3;
            float* const red = reinterpret_cast<float*>(gbase) + quarter * 32 + lane;
            uint32_t const t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                if (c >= rows) break;
                uint32_t r[16];
                tmem_ld_32x16(t_row + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) red[(c + j) * C::kRedStride] = __uint_as_float(r[j]);
            }
            tc_fence_before();
        } else if (lane == 0) {
            record_abort(FSO_DEV_WAIT_EPILOGUE, abort_flag);
        }
        __syncwarp();
    }
    __syncthreads();
    bool const failed = *abort_flag != 0;
    if (failed) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);      // copies in flight land before the memory is given up
        __syncthreads();
    }
    if (p.splits > 1) cluster_sync_all();
    if (!failed) {
        float const* const red = reinterpret_cast<float const*>(gbase);
        uint32_t const red_addr = smem_u32(red);
        // four columns a thread
        for (int i = rank * C::kThreads + static_cast<int>(threadIdx.x); i < rows * 16; i += C::kThreads * p.splits) {
            int const row = i >> 4, in_tile = (i & 15) * 4;
            int const col = tile * 64 + in_tile;
            if (col >= p.inter) continue;
            int const at = row * C::kRedStride + in_tile;
            float g[4] = {}, u[4] = {};
            if (p.splits == 1) {
                float4 const a = *reinterpret_cast<float4 const*>(red + at), b = *reinterpret_cast<float4 const*>(red + at + 64);
                g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
                u[0] = b.x; u[1] = b.y; u[2] = b.z; u[3] = b.w;
            } else {      // all loads first: one trip to the other CTAs' memory instead of one for each
                float4 a[8], b[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r < p.splits) {
                        uint32_t const peer = map_to_cta(red_addr + 4u * at, r);
                        a[r] = ld_cluster_f32x4(peer);
                        b[r] = ld_cluster_f32x4(peer + 256u);
                    }
                }
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r < p.splits) {
                        g[0] += a[r].x; g[1] += a[r].y; g[2] += a[r].z; g[3] += a[r].w;
                        u[0] += b[r].x; u[1] += b[r].y; u[2] += b[r].z; u[3] += b[r].w;
                    }
                }
            }
            int64_t const out_row = row0 + row;
            finish_four<kBf16>(g, u, p.act, p.save_hi, p.save_lo, out_row * 2 * p.half_cols + col, p.half_cols, p.out,
                out_row * p.inter + col, p.inter - col, p.vec != 0);
        }
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync_all();      // no CTA leaves while another may still read its sums
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------ split sums

// out = the sum of the slices of the contraction, in their order, rounded once. Columns are multiples of 8.
template <bool kBf16>
__global__ void gated16_sum_kernel(float const* __restrict__ ws, int splits, int64_t slab, int64_t rows, int cols,
    int64_t ws_cols, uint16_t* __restrict__ out, int64_t ldo)
{
    griddep_launch_dependents();
    griddep_wait();
    int const per_row = cols / 8;
    int64_t const i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= rows * per_row) return;
    int64_t const row = i / per_row;
    int const col = static_cast<int>(i - row * per_row) * 8;
    float v[8] = {};
    for (int s = 0; s < splits; ++s) {
        float4 const* const w = reinterpret_cast<float4 const*>(ws + s * slab + row * ws_cols + col);
        float4 const a = w[0], b = w[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
    *reinterpret_cast<uint4*>(out + row * ldo + col) = make_uint4(pack16<kBf16>(v[0], v[1]), pack16<kBf16>(v[2], v[3]),
        pack16<kBf16>(v[4], v[5]), pack16<kBf16>(v[6], v[7]));
}

// The epilogue of the forward pass for a split contraction: sums, saved values, act and product. Four columns a thread.
template <bool kBf16>
__global__ void gated16_finish_kernel(float const* __restrict__ ws, int splits, int rows, int cols, int64_t half_cols,
    int act, uint16_t* __restrict__ save_hi, uint8_t* __restrict__ save_lo, void* __restrict__ out, int vec)
{
    griddep_launch_dependents();
    griddep_wait();
    int const per_row = static_cast<int>(half_cols / 4);
    int64_t const i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= static_cast<int64_t>(rows) * per_row) return;
    int64_t const row = i / per_row;
    int const col = static_cast<int>(i - row * per_row) * 4;
    float g[4] = {}, u[4] = {};
    for (int s = 0; s < splits; ++s) {
        float const* const w = ws + (static_cast<int64_t>(s) * rows + row) * 2 * half_cols + col;
        float4 const a = *reinterpret_cast<float4 const*>(w), b = *reinterpret_cast<float4 const*>(w + half_cols);
        g[0] += a.x; g[1] += a.y; g[2] += a.z; g[3] += a.w;
        u[0] += b.x; u[1] += b.y; u[2] += b.z; u[3] += b.w;
    }
    finish_four<kBf16>(g, u, act, save_hi, save_lo, row * 2 * half_cols + col, half_cols, out, row * cols + col, cols - col,
        vec != 0);
}

// ------------------------------------------------------------------------------------------------ dg and du
//
// dg = dh * u * act'(g), du = dh * act(g) from the saved g and u, rounded to the 16 bits in which the tensor cores take
// them (the one rounding of the backward pass before its products). Bound by memory: 2 + 2 * 3 bytes in and 4 out for
// each element, 51 us for 4096 x 7168 (352 MB, some of it still in L2). Eight columns a thread.
template <bool kBf16, int ACT>
__global__ void __launch_bounds__(256) gated_slopes_kernel(const void* __restrict__ dh, int64_t ldh, int dh_vec, uint16_t const* __restrict__ save_hi,
    uint8_t const* __restrict__ save_lo, int rows, int cols, int64_t half_cols, uint16_t* __restrict__ out)
{
    griddep_launch_dependents();
    griddep_wait();
    int const per_row = static_cast<int>(half_cols / 8);
    int64_t const i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= static_cast<int64_t>(rows) * per_row) return;
    int64_t const row = i / per_row;
    int const col = static_cast<int>(i - row * per_row) * 8;
    if (col >= cols) return;
    float d[8];
    if (dh_vec) {
        uint4 const w = *reinterpret_cast<uint4 const*>(static_cast<uint16_t const*>(dh) + row * ldh + col);
        uint32_t const q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 const f = unpack16<kBf16>(q[j]);
            d[2 * j] = f.x;
            d[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = col + j < cols ? load16<kBf16>(dh, row * ldh + col + j) : 0.f;
    }
    int64_t const at = row * 2 * half_cols + col;
    uint4 const gh = *reinterpret_cast<uint4 const*>(save_hi + at), uh = *reinterpret_cast<uint4 const*>(save_hi + at + half_cols);
    uint2 const gl = *reinterpret_cast<uint2 const*>(save_lo + at), ul = *reinterpret_cast<uint2 const*>(save_lo + at + half_cols);
    uint32_t const ghw[4] = {gh.x, gh.y, gh.z, gh.w}, uhw[4] = {uh.x, uh.y, uh.z, uh.w};
    uint32_t const glw[2] = {gl.x, gl.y}, ulw[2] = {ul.x, ul.y};
    float dg[8], du[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float const g = from_24((ghw[j / 2] >> (16 * (j & 1))) & 0xFFFFu, (glw[j / 4] >> (8 * (j & 3))) & 0xFFu);
        float const u = from_24((uhw[j / 2] >> (16 * (j & 1))) & 0xFFFFu, (ulw[j / 4] >> (8 * (j & 3))) & 0xFFu);
        float a, s;
        gate_value_slope<ACT>(g, a, s);
        dg[j] = d[j] * u * s;
        du[j] = d[j] * a;
    }
    *reinterpret_cast<uint4*>(out + at) = make_uint4(pack16<kBf16>(dg[0], dg[1]), pack16<kBf16>(dg[2], dg[3]),
        pack16<kBf16>(dg[4], dg[5]), pack16<kBf16>(dg[6], dg[7]));
    *reinterpret_cast<uint4*>(out + at + half_cols) = make_uint4(pack16<kBf16>(du[0], du[1]), pack16<kBf16>(du[2], du[3]),
        pack16<kBf16>(du[4], du[5]), pack16<kBf16>(du[6], du[7]));
}

// ------------------------------------------------------------------------------------------------ host side

// Tensor map of a 16-bit matrix [rows, cols] with `ld` elements between rows, read in boxes of 64 columns x box_rows
// with the 128-byte swizzle; what a box holds outside the matrix reads as zero.
inline int make_map16(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) {
        set_error("cuTensorMapEncodeTiled is not available from this driver");
        return FSO_ERR_UNSUPPORTED;
    }
    cuuint64_t const dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t const strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    cuuint32_t const box[2] = {64u, static_cast<cuuint32_t>(box_rows)};
    cuuint32_t const estr[2] = {1u, 1u};
    CUresult const r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with CUresult %d (16-bit matrix of %lld x %lld, %lld between rows)",
            static_cast<int>(r), static_cast<long long>(rows), static_cast<long long>(cols), static_cast<long long>(ld));
        return FSO_ERR_INTERNAL;
    }
    return 0;
}

// clusters[c], c in 2..8: how many clusters of c CTAs the current device runs together with `per_sm` (1 or 2) CTAs on an SM. Fewer
// than its SMs would hold, since those of a GPC do not divide by every c: 74, 45, 33 and 15 clusters of 2, 3, 4 and 8 on
// 148 SMs with one, 148, 93, 71 and 33 with two. Asked once, about a stand-in with the shared memory of such CTAs: of kernels
// that use tensor memory the driver answers for one CTA on an SM, whatever they allocate.
__global__ void resident_clusters_kernel() {}

inline int resident_clusters(int per_sm, int (&clusters)[9])
{
    static std::atomic<int> known[2][64][9];      // plus one
    static std::atomic<uint64_t> done{0};
    std::atomic<int>* const of_device = known[per_sm - 1][current_device() & 63];
    for (int c = 2; c <= 8; ++c) {
        int n = of_device[c].load(std::memory_order_relaxed);
        if (n == 0) {
            int const rc = ensure_smem_attr(resident_clusters_kernel, 220 * 1024, done);
            if (rc != 0) return rc;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(static_cast<unsigned>(64 * c));
            cfg.blockDim = dim3(256);
            cfg.dynamicSmemBytes = per_sm == 1 ? 220 * 1024 : 110 * 1024;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = static_cast<unsigned>(c);
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            FSO_CUDA(cudaOccupancyMaxActiveClusters(&n, resident_clusters_kernel, &cfg));
            of_device[c].store(++n, std::memory_order_relaxed);
        }
        clusters[c] = n - 1;
    }
    return 0;
}

inline int64_t gated_half_cols(int64_t inter) { return (inter + 15) / 16 * 16; }

// Tiles and slices of the products. Pure host arithmetic.
struct Gated16Plan {
    int rows_n;          // forward: rows of x in a tile of the few-rows kernel, or 0 for the pair kernel
    int tiles_m, tiles_n, kb, kb_half, splits, kb_per_split;
    int64_t ws_bytes, ws_cols;
};

inline int tiles_of(int64_t n, int64_t w) { return static_cast<int>((n + w - 1) / w); }

// FSO_B200_GATED=pair | rows keeps the forward pass of more than 128 rows on one of its two kernels (measurement; read once).
inline int forced_gated_kernel()
{
    static int const v = [] {
        const char* e = std::getenv("FSO_B200_GATED");
        return e == nullptr ? 0 : std::strcmp(e, "pair") == 0 ? 1 : std::strcmp(e, "rows") == 0 ? 2 : 0;
    }();
    return v;
}

// The forward pass. Both kernels are costed in microseconds of a B200, with constants fitted to sweeps over 129 to 2900 rows
// on five weights with either kernel forced: rounds of the schedule times the blocks of a slice (a 64-wide block is 512 cycles
// at 1.55 GHz for 256 rows of x, in proportion below, 264 cycles at the least), what a tile costs beside them, and for the
// pair kernel the traffic of split sums through L2.
inline int plan_gated16_forward(int64_t t, int64_t k, int64_t inter, int sms, Gated16Plan& p)
{
    p = Gated16Plan{};
    int alone[9], shared[9];
    int rc = resident_clusters(1, alone);
    if (rc == 0) rc = resident_clusters(2, shared);
    if (rc != 0) return rc;
    p.kb = tiles_of(k, 64);
    int const pairs = std::max(1, sms / 2);
    // few rows: token tiles of at most 256, equal, multiples of 16
    int const row_tiles = tiles_of(t, 256), weight_tiles = tiles_of(inter, 64);
    int const n = static_cast<int>((tiles_of(t, row_tiles) + 15) / 16 * 16);
    int64_t const tiles = static_cast<int64_t>(row_tiles) * weight_tiles;
    int const slots = n <= 128 && tiles > sms ? 2 * sms : sms;
    // Slices of at least four blocks: at most four and as many as leave all clusters resident, each CTA with an SM to itself and
    // its whole shared memory as a ring (36 tiles of K = 4096, one row: 9.5 us in clusters of three, 14.3 in clusters of
    // four, of which 33 fit); a handful of tiles in eight slices (the portable cluster size), whose CTAs share SMs,
    // because not all GPCs find eight free SMs twice.
    int const limit = n <= 128 && tiles * 8 <= sms ? 8 : 4;
    int s = 1;
    while (s < limit && tiles * (s + 1) <= sms && tiles <= (s < 4 ? alone : shared)[s + 1] && (s + 1) * 4 <= p.kb) ++s;
    int const per = tiles_of(p.kb, s);
    double const rows_us = std::ceil(static_cast<double>(tiles * s) / slots) * (per * std::max(264, 2 * n) / 1550.0 * (slots > sms ? 2 : 1)
        + 2.0 + 0.035 * n) + 3.0;
    // pairs
    p.tiles_m = tiles_of(t, 256);
    p.tiles_n = tiles_of(inter, 128);
    p.ws_cols = 2 * gated_half_cols(inter);
    double pair_us = 1e30;
    int pair_s = 1;
    for (int q = 1; q <= 16 && (q == 1 || q * 4 <= p.kb); ++q) {
        double const rounds = std::ceil(static_cast<double>(p.tiles_m) * p.tiles_n * q / pairs);
        double const us = rounds * tiles_of(p.kb, q) * (512 / 1550.0) + 9.0
            + (q > 1 ? 3.0 + static_cast<double>(q) * t * p.ws_cols * 8 / 8e6 : 0.0);
        if (us < pair_us) {
            pair_us = us;
            pair_s = q;
        }
    }
    bool const rows = t <= 128 || (row_tiles <= 1024 && (forced_gated_kernel() == 0 ? rows_us < pair_us : forced_gated_kernel() == 2));
    p.rows_n = rows ? n : 0;
    p.kb_per_split = rows ? per : tiles_of(p.kb, pair_s);
    p.splits = tiles_of(p.kb, p.kb_per_split);
    p.ws_bytes = !rows && p.splits > 1 ? p.splits * t * p.ws_cols * 4 : 0;
    return 0;
}

// The backward pass: dx and dW share the SM pairs. Where one of them has fewer tiles than there are pairs its contraction is
// cut into slices of about a pair's part of all the work, of at least 512 elements, at most 16.
inline void plan_gated16_backward(int64_t t, int64_t k, int64_t inter, bool need_x, bool need_w, int sms, Gated16Plan& dx,
    Gated16Plan& dw)
{
    int const pairs = std::max(1, sms / 2);
    dx = Gated16Plan{};
    dw = Gated16Plan{};
    dx.kb_half = tiles_of(inter, 64);
    dx.kb = 2 * dx.kb_half;
    dw.kb_half = tiles_of(inter, 256);
    dw.kb = tiles_of(t, 64);
    dx.tiles_n = dw.tiles_n = tiles_of(k, 256);
    dx.tiles_m = need_x ? tiles_of(t, 256) : 0;
    dw.tiles_m = need_w ? 2 * dw.kb_half : 0;
    dx.ws_cols = dw.ws_cols = (k + 15) / 16 * 16;
    int64_t const work = static_cast<int64_t>(dx.tiles_m) * dx.tiles_n * dx.kb + static_cast<int64_t>(dw.tiles_m) * dw.tiles_n * dw.kb;
    int const share = static_cast<int>(std::max<int64_t>(8, std::min<int64_t>(work / pairs, 1 << 24)));
    for (Gated16Plan* p : {&dx, &dw}) {
        p->splits = 1;
        if (static_cast<int64_t>(p->tiles_m) * p->tiles_n < pairs && p->kb > share)
            p->splits = std::min(16, tiles_of(p->kb, share));
        p->kb_per_split = tiles_of(p->kb, p->splits);
        p->splits = tiles_of(p->kb, p->kb_per_split);
        int64_t const rows = p == &dx ? t : 2 * inter;
        p->ws_bytes = p->splits > 1 && p->tiles_m > 0 ? p->splits * rows * p->ws_cols * 4 : 0;
    }
}

// Launch with programmatic dependent launch: every kernel of this file lets its successor start early and waits for its own
// predecessor before it touches memory.
template <typename... Params, typename... Args>
inline int launch_chained(const char* what, void (*kernel)(Params...), unsigned grid, int threads, int smem, cudaStream_t stream,
    Args const&... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.attrs = attr;
    cfg.numAttrs = pdl_attribute(&attr[0]);
    FSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
    return launch_status(what);
}

template <int MODE, bool kBf16, int ACT>
inline int launch_gated16(CUtensorMap const (&m)[5], Gated16Params const& p, int sms, cudaStream_t stream)
{
    static std::atomic<uint64_t> done{0};
    auto kernel = gated16_pair_kernel<MODE, kBf16, ACT>;
    int const rc = ensure_smem_attr(kernel, Gated16Cfg::kSmemBytes, done);
    if (rc != 0) return rc;
    int64_t const items = static_cast<int64_t>(p.first.tiles_m) * p.first.tiles_n * p.first.splits
        + static_cast<int64_t>(p.second.tiles_m) * p.second.tiles_n * p.second.splits;
    FSO_REQUIRE(items < (1ll << 31), "gated projection: %lld tiles are beyond the kernel's index range", static_cast<long long>(items));
    unsigned const pairs = static_cast<unsigned>(std::min<int64_t>(items, std::max(1, sms / 2)));
    return launch_chained("gated16_pair_kernel", kernel, 2 * pairs, Gated16Cfg::kThreads, Gated16Cfg::kSmemBytes, stream, m[0], m[1],
        m[2], m[3], m[4], p);
}

// group_m: about the square root of the tiles in flight, so that a wave reads few rows of either operand: at 8192 x 4096 x 14336
// under the power cap the forward pass takes 1385, 1365, 1353 and 1472 us with 8, 12, 16 and 32 (1473, 1460, 1471 and 1670
// when it saves its projections), dx 1785, 1827 and 1818 with 8, 6 and 16, dW 1812, 1813, 1835 and 1930 with 8, 12, 16, 32.
inline void fill_product(Gated16Product& q, Gated16Plan const& pl, int group_m)
{
    q.tiles_m = pl.tiles_m;
    q.tiles_n = pl.tiles_n;
    q.group_m = std::max(1, std::min(pl.tiles_m, group_m));
    q.kb_total = pl.kb;
    q.kb_half = pl.kb_half;
    q.splits = pl.splits;
    q.kb_per_split = pl.kb_per_split;
    q.ws_cols = pl.ws_cols;
}

inline unsigned blocks_for(int64_t threads, int per_block) { return static_cast<unsigned>((threads + per_block - 1) / per_block); }

template <int BN, bool kBf16>
inline int launch_gated_rows(const void* x, int64_t ldx, const void* gate_up, int64_t k, GatedRowsParams p, cudaStream_t stream)
{
    using C = GatedRowsCfg<BN>;
    static std::atomic<uint64_t> done{0};
    auto kernel = gated_rows_kernel<BN, kBf16>;
    int rc = ensure_smem_attr(kernel, C::smem_bytes(C::kStagesAlone), done);
    if (rc != 0) return rc;
    uint16_t const* const w = static_cast<uint16_t const*>(gate_up);
    CUtensorMap mg, mu, mx;
    rc = make_map16(&mg, w, p.inter, k, k, 64);
    if (rc == 0) rc = make_map16(&mu, w + p.inter * k, p.inter, k, k, 64);
    if (rc == 0) rc = make_map16(&mx, x, p.t, k, ldx, p.n);
    if (rc != 0) return rc;
    int const tiles = (p.inter + 63) / 64, row_tiles = (p.t + p.n - 1) / p.n;
    bool const alone = C::kBlocks == 1 || (p.splits <= 4 && tiles * row_tiles * p.splits <= sm_count());
    p.stages = alone ? C::kStagesAlone : C::kStagesShared;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.splits), static_cast<unsigned>(row_tiles), 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(C::smem_bytes(p.stages));
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(p.splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + pdl_attribute(&attr[1]);
    FSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, mg, mu, mx, p));
    return launch_status("gated_rows_kernel");
}

template <bool kBf16>
inline int gated_forward(const void* x, int64_t ldx, const void* gate_up, void* h, void* save_hi, void* save_lo, int64_t t,
    int64_t k, int64_t inter, int act, void* ws, cudaStream_t stream)
{
    int const sms = sm_count();
    Gated16Plan pl;
    int rc = plan_gated16_forward(t, k, inter, sms, pl);
    if (rc != 0) return rc;
    if (pl.rows_n > 0) {
        GatedRowsParams r{};
        r.t = static_cast<int>(t);
        r.inter = static_cast<int>(inter);
        r.act = act;
        r.n = pl.rows_n;
        r.kb_total = pl.kb;
        r.kb_per_split = pl.kb_per_split;
        r.splits = pl.splits;
        r.out = h;
        r.vec = inter % 4 == 0 && (reinterpret_cast<uintptr_t>(h) & 7u) == 0;
        r.save_hi = static_cast<uint16_t*>(save_hi);
        r.save_lo = static_cast<uint8_t*>(save_lo);
        r.half_cols = gated_half_cols(inter);
        return r.n <= 16 ? launch_gated_rows<16, kBf16>(x, ldx, gate_up, k, r, stream)
            : r.n <= 32  ? launch_gated_rows<32, kBf16>(x, ldx, gate_up, k, r, stream)
            : r.n <= 64  ? launch_gated_rows<64, kBf16>(x, ldx, gate_up, k, r, stream)
            : r.n <= 128 ? launch_gated_rows<128, kBf16>(x, ldx, gate_up, k, r, stream)
                         : launch_gated_rows<256, kBf16>(x, ldx, gate_up, k, r, stream);
    }
    CUtensorMap m[5];
    uint16_t const* const w = static_cast<uint16_t const*>(gate_up);
    rc = make_map16(&m[0], x, t, k, ldx, 128);
    if (rc == 0) rc = make_map16(&m[1], w, inter, k, k, 128);
    if (rc == 0) rc = make_map16(&m[2], w + inter * k, inter, k, k, 128);
    if (rc != 0) return rc;
    m[3] = m[4] = m[0];
    Gated16Params p{};
    fill_product(p.first, pl, 12);
    p.first.rows = static_cast<int>(t);
    p.first.cols = static_cast<int>(inter);
    p.first.vec = inter % 8 == 0 && aligned16(h);
    p.first.out = h;
    p.first.ldo = inter;
    p.first.ws = pl.splits > 1 ? static_cast<float*>(ws) : nullptr;
    p.save_hi = static_cast<uint16_t*>(save_hi);
    p.save_lo = static_cast<uint8_t*>(save_lo);
    p.half_cols = gated_half_cols(inter);
    rc = act == FSO_ACT_SILU ? launch_gated16<G16_FORWARD, kBf16, FSO_ACT_SILU>(m, p, sms, stream)
        : act == FSO_ACT_GELU ? launch_gated16<G16_FORWARD, kBf16, FSO_ACT_GELU>(m, p, sms, stream)
                              : launch_gated16<G16_FORWARD, kBf16, FSO_ACT_GELU_TANH>(m, p, sms, stream);
    if (rc != 0 || pl.splits == 1) return rc;
    return launch_chained("gated16_finish_kernel", gated16_finish_kernel<kBf16>, blocks_for(t * (p.half_cols / 4), 128), 128, 0,
        stream, p.first.ws, pl.splits, p.first.rows, p.first.cols, p.half_cols, act, p.save_hi, p.save_lo, h, p.first.vec);
}

// Workspace of the backward pass: dg and du (16 bit [T, 2 * half_cols]), then the slices of dx and of dW. Enough for one
// gradient alone as well as for both.
inline int64_t gated_slopes_bytes(int64_t t, int64_t inter) { return (t * 2 * gated_half_cols(inter) * 2 + 255) / 256 * 256; }

inline int64_t gated_backward_ws_bytes(int64_t t, int64_t k, int64_t inter, int sms)
{
    int64_t sums = 0;
    for (int need = 1; need < 4; ++need) {
        Gated16Plan dx, dw;
        plan_gated16_backward(t, k, inter, need & 1, need & 2, sms, dx, dw);
        sums = std::max(sums, (dx.ws_bytes + 255) / 256 * 256 + dw.ws_bytes);
    }
    return gated_slopes_bytes(t, inter) + sums;
}

template <bool kBf16>
inline int gated_backward(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* gate_up, const void* save_hi,
    const void* save_lo, void* dx, void* dgate_up, int64_t t, int64_t k, int64_t inter, int act, void* ws, cudaStream_t stream)
{
    if (dx == nullptr && dgate_up == nullptr) return 0;
    int const sms = sm_count();
    int64_t const hc = gated_half_cols(inter);
    uint16_t* const slopes = static_cast<uint16_t*>(ws);
    int const dh_vec = inter % 8 == 0 && ldh % 8 == 0 && aligned16(dh);
    auto slopes_kernel = act == FSO_ACT_SILU ? gated_slopes_kernel<kBf16, FSO_ACT_SILU>
        : act == FSO_ACT_GELU ? gated_slopes_kernel<kBf16, FSO_ACT_GELU> : gated_slopes_kernel<kBf16, FSO_ACT_GELU_TANH>;
    int rc = launch_chained("gated_slopes_kernel", slopes_kernel, blocks_for(t * (hc / 8), 256), 256, 0, stream, dh, ldh,
        dh_vec, static_cast<uint16_t const*>(save_hi), static_cast<uint8_t const*>(save_lo), static_cast<int>(t),
        static_cast<int>(inter), hc, slopes);
    if (rc != 0) return rc;

    Gated16Plan px, pw;
    plan_gated16_backward(t, k, inter, dx != nullptr, dgate_up != nullptr, sms, px, pw);
    float* const sums_x = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + gated_slopes_bytes(t, inter));
    float* const sums_w = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sums_x) + (px.ws_bytes + 255) / 256 * 256);
    uint16_t const* const w = static_cast<uint16_t const*>(gate_up);
    CUtensorMap m[5];
    rc = make_map16(&m[0], x, t, k, ldx, 64);
    if (rc == 0) rc = make_map16(&m[1], w, inter, k, k, 64);
    if (rc == 0) rc = make_map16(&m[2], w + inter * k, inter, k, k, 64);
    if (rc == 0) rc = make_map16(&m[3], slopes, t, inter, 2 * hc, 64);
    if (rc == 0) rc = make_map16(&m[4], slopes + hc, t, inter, 2 * hc, 64);
    if (rc != 0) return rc;
    Gated16Params p{};
    p.first_is_dw = pw.kb_per_split > px.kb_per_split;      // long tiles first: the short ones even out the last round
    Gated16Product& qx = p.first_is_dw ? p.second : p.first;
    Gated16Product& qw = p.first_is_dw ? p.first : p.second;
    fill_product(qx, px, 8);
    qx.rows = static_cast<int>(t);
    qx.cols = static_cast<int>(k);
    qx.vec = 1;
    qx.out = dx;
    qx.ldo = k;
    qx.ws = px.splits > 1 ? sums_x : nullptr;
    fill_product(qw, pw, 8);
    qw.rows = static_cast<int>(inter);
    qw.cols = static_cast<int>(k);
    qw.vec = 1;
    qw.out = dgate_up;
    qw.ldo = k;
    qw.out_half = inter * k;
    qw.ws = pw.splits > 1 ? sums_w : nullptr;
    rc = launch_gated16<G16_BACKWARD, kBf16, 0>(m, p, sms, stream);
    if (rc == 0 && dx != nullptr && px.splits > 1)
        rc = launch_chained("gated16_sum_kernel", gated16_sum_kernel<kBf16>, blocks_for(t * (k / 8), 256), 256, 0, stream, sums_x,
            px.splits, t * px.ws_cols, t, static_cast<int>(k), px.ws_cols, static_cast<uint16_t*>(dx), k);
    if (rc == 0 && dgate_up != nullptr && pw.splits > 1)
        rc = launch_chained("gated16_sum_kernel", gated16_sum_kernel<kBf16>, blocks_for(2 * inter * (k / 8), 256), 256, 0, stream,
            sums_w, pw.splits, 2 * inter * pw.ws_cols, 2 * inter, static_cast<int>(k), pw.ws_cols, static_cast<uint16_t*>(dgate_up), k);
    return rc;
}

}  // namespace fso
