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
    const uint8_t* codes;  // [rows, k / 2]
    const void* scale;     // [rows, k / group]
    int scale_type;        // 0 bf16, 1 fp16, 2 fp32
    const uint8_t* zero;   // [rows, k / group], or nullptr: 8
    const void* bias;      // [out], 16 bit like x, or nullptr
    void* out;             // 16 bit [m, out_cols]
    int m, k, group;
    int out_cols;          // rows of the weight, or half of them when gated
    int act;
};

__device__ __forceinline__ float int4_scale(Int4Params const& p, int64_t i)
{
    if (p.scale_type == 0) return load16<true>(p.scale, i);
    if (p.scale_type == 1) return load16<false>(p.scale, i);
    return static_cast<float const*>(p.scale)[i];
}

// One warp for each output column and eight rows of x; a lane takes eight consecutive k of every 256.
template <bool kBf16, bool kGated>
__global__ void int4_rows_kernel(Int4Params const p)
{
    int const lane = threadIdx.x & 31;
    int64_t const col = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
    if (col >= p.out_cols) return;
    int const t0 = blockIdx.y * 8;
    int const live = min(8, p.m - t0);
    int const groups = p.k / p.group;
    float sums[kGated ? 2 : 1][8];
#pragma unroll
    for (int half = 0; half < (kGated ? 2 : 1); ++half) {
        int64_t const row = col + static_cast<int64_t>(half) * p.out_cols;
        float acc[8] = {};
        for (int k0 = lane * 8; k0 < p.k; k0 += 256) {
            uint32_t const w = *reinterpret_cast<uint32_t const*>(p.codes + row * (p.k / 2) + k0 / 2);
            int64_t const at = row * groups + k0 / p.group;
            float const s = int4_scale(p, at);
            int const z = p.zero != nullptr ? p.zero[at] : 8;
            float q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - z);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (t < live) {
                    uint4 const v = *reinterpret_cast<uint4 const*>(
                        static_cast<uint16_t const*>(p.x) + static_cast<int64_t>(t0 + t) * p.ldx + k0);
                    uint32_t const words[4] = {v.x, v.y, v.z, v.w};
                    float part = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float2 const f = unpack16<kBf16>(words[j]);
                        part = fmaf(q[2 * j], f.x, part);
                        part = fmaf(q[2 * j + 1], f.y, part);
                    }
                    acc[t] = fmaf(s, part, acc[t]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
            sums[half][t] = acc[t];
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if (lane == t && t < live) {
            float v = sums[0][t];
            if constexpr (kGated) v = gate_value(v, p.act) * sums[1][t];
            else if (p.bias != nullptr) v += load16<kBf16>(p.bias, col);
            store16<kBf16>(p.out, static_cast<int64_t>(t0 + t) * p.out_cols + col, v);
        }
    }
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
    int scale_type, uint8_t* __restrict__ zero, int64_t vectors, int lanes)
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
        int64_t const g = i / lanes;
        if (scale_type == 0) store16<true>(scale, g, step);
        else if (scale_type == 1) store16<false>(scale, g, step);
        else static_cast<float*>(scale)[g] = step;
        if (zero != nullptr) zero[g] = static_cast<uint8_t>(z);
    }
}

inline int launch_int4(Int4Params const& p, bool bf16, bool gated, cudaStream_t stream)
{
    dim3 const grid(static_cast<unsigned>((p.out_cols + 3) / 4), static_cast<unsigned>((p.m + 7) / 8));
    if (bf16 && gated) int4_rows_kernel<true, true><<<grid, 128, 0, stream>>>(p);
    else if (bf16) int4_rows_kernel<true, false><<<grid, 128, 0, stream>>>(p);
    else if (gated) int4_rows_kernel<false, true><<<grid, 128, 0, stream>>>(p);
    else int4_rows_kernel<false, false><<<grid, 128, 0, stream>>>(p);
    return launch_status("int4_rows_kernel");
}

}  // namespace fso
