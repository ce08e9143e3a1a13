// The FP8 (E4M3) KV cache: quantised as it is written, behind the key-side RoPE and optionally the per-head RMSNorm, and
// read back through a row map. One f32 scale per cache row and kv head:
//   scale = max |x| / 448,  code = e4m3(x * (1 / scale))  round to nearest even, x the f32 value the bf16 cache would round
// (a scale per head row costs 4 bytes beside head_dim codes and keeps an outlier head from flattening the others).
// A head row whose maximum is below 2^-100 is stored as zeros with scale 0; one that holds an infinity or a NaN is
// stored as zero codes with scale NaN, so that whatever reads it sees NaN.
//
// Bound by HBM bytes. A head row of head_dim values is a group of G = head_dim / 8 lanes (rounded up to a power of two),
// 8 values each: 16-byte loads (bf16), and the rotation partner is a second load of a line the group has fetched
// anyway, which keeps the kernel free of shared memory and of an exchange before the row maximum.
#pragma once

#include "kernels_generic.cuh"
#include "kernels_hot.cuh"
#include "kernels_fp8.cuh"

#include <cuda_fp16.h>

namespace clef {

constexpr int kKvMaxHeadDim = 256;
constexpr float kKvMinAmax = 7.888609052e-31f;   // 2^-100

struct KvWriteArgs {
    const void* q;        // [tokens, q_heads, head_dim] or NULL
    void* q_out;
    int q_heads;
    const void* k;        // [tokens, kv_heads, head_dim]
    const void* v;
    uint8_t* cache_k;     // [cache_rows, kv_heads, head_dim]
    uint8_t* cache_v;
    float* k_scales;      // [cache_rows, kv_heads]
    float* v_scales;
    const float* weight;  // per-head norm of k, NULL without
    const float* cos_t;   // [positions, rotary_dim]
    const float* sin_t;
    const int* seq_start;
    const int* pos_base;
    const int* pos_map;
    const int* cache_map;
    const int* cache_len;
    int tokens, kv_heads, head_dim, rotary_dim, cache_rows;
    float eps;
    FastDiv heads_div;    // q_heads + 2 kv_heads head rows per token
};

// Eight scaled values -> eight E4M3 bytes, round to nearest even, saturating.
__device__ __forceinline__ uint2 e4m3x8_rn(const float* v, float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* p = v + 4 * h;
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}"
            : "=r"(w[h])
            : "f"(__fmul_rn(p[0], inv)), "f"(__fmul_rn(p[1], inv)), "f"(__fmul_rn(p[2], inv)), "f"(__fmul_rn(p[3], inv)));
    }
    return make_uint2(w[0], w[1]);
}

template <typename T>
__device__ __forceinline__ void store8(typename T::storage* p, const float* v);
template <>
__device__ __forceinline__ void store8<Bf16>(uint16_t* p, const float* v) {
    stg_v4(p, make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
}
template <>
__device__ __forceinline__ void store8<F32>(float* p, const float* v) {
    stg_v4(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
    stg_v4(p + 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
}

// G lanes per head row; a warp holds 32 / G head rows. NORM: k rows are normalised first, in the summation order of
// rms_norm_kernel (kernels/elementwise.cu:4-68: quad i with quad i + 32, then the tree 16, 8, 4, 2, 1 over quads).
template <typename T, int G, bool NORM>
__global__ void __launch_bounds__(kCtaThreads)
kv_write_fp8_kernel(KvWriteArgs a) {
    constexpr int PER_WARP = 32 / G;
    const int lane = threadIdx.x & 31, sub = lane % G;
    const int col = sub * 8, half = a.rotary_dim >> 1;
    const bool mine = col < a.head_dim;
    const uint32_t per_token = a.heads_div.d;
    const uint32_t rows = (uint32_t)a.tokens * per_token;
    const uint32_t step = gridDim.x * (kCtaThreads / 32) * PER_WARP;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    // (the shuffles below need the whole warp: its head rows leave the loop together)
    for (uint32_t base = (blockIdx.x * (kCtaThreads / 32) + (threadIdx.x >> 5)) * PER_WARP; base < rows; base += step) {
        const uint32_t row = base + lane / G;
        const bool live = mine && row < rows;
        const uint32_t token = fast_div(row < rows ? row : 0u, a.heads_div);
        const int slot = row < rows ? (int)(row - token * per_token) : 0;
        const bool is_q = slot < a.q_heads;
        const int kv_slot = slot - a.q_heads;
        const bool is_v = kv_slot >= a.kv_heads;
        const int head = is_q ? slot : (is_v ? kv_slot - a.kv_heads : kv_slot);
        const typename T::storage* x = static_cast<const typename T::storage*>(is_q ? a.q : (is_v ? a.v : a.k)) +
                                       ((size_t)token * (is_q ? a.q_heads : a.kv_heads) + head) * a.head_dim;
        const bool rotates = live && !is_v && col < a.rotary_dim;
        const bool upper = col >= half;
        float v[8], other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other[i] = 0.0f;
        if (live) load8<T>(x + col, v);
        if (rotates) load8<T>(x + (upper ? col - half : col + half), other);
        if (NORM) {
            float s0 = quad_sq(make_float4(v[0], v[1], v[2], v[3])), s1 = quad_sq(make_float4(v[4], v[5], v[6], v[7]));
#pragma unroll
            for (int off = G / 2; off > 0; off >>= 1) {
                s0 = __fadd_rn(s0, __shfl_xor_sync(kFullMask, s0, off));
                s1 = __fadd_rn(s1, __shfl_xor_sync(kFullMask, s1, off));
            }
            if (live && !is_q && !is_v) {
                const float inv = inv_rms(__fadd_rn(s0, s1), a.head_dim, a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * (1.0f + a.weight[col + i]);
                if (rotates) {
                    const float* w = a.weight + (upper ? col - half : col + half);
#pragma unroll
                    for (int i = 0; i < 8; ++i) other[i] = other[i] * inv * (1.0f + w[i]);
                }
            }
        }
        if (rotates) {
            const int pos = rope_position((int)token, a.seq_start, a.pos_base, a.pos_map);
            const size_t at = (size_t)pos * a.rotary_dim + (upper ? col - half : col);
            float c[8], s[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *reinterpret_cast<float4*>(c + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at) + i);
                *reinterpret_cast<float4*>(s + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at) + i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float lo, hi;
                rope_pair(upper ? other[i] : v[i], upper ? v[i] : other[i], c[i], s[i], lo, hi);
                v[i] = upper ? hi : lo;
            }
        }
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf_nan(amax, fabsf(v[i]));
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) amax = fmaxf_nan(amax, __shfl_xor_sync(kFullMask, amax, off));
        if (!live) continue;
        if (is_q) {
            store8<T>(static_cast<typename T::storage*>(a.q_out) + ((size_t)token * a.q_heads + head) * a.head_dim + col, v);
            continue;
        }
        const long long at = a.cache_map ? (long long)a.cache_map[token]
                                         : (long long)token + (a.cache_len ? a.cache_len[0] : 0);
        if (at < 0 || at >= a.cache_rows) continue;   // a padding token
        const size_t head_row = (size_t)at * a.kv_heads + head;
        const bool finite = amax < INFINITY, some = amax >= kKvMinAmax;   // both false for a NaN
        const float scale = finite ? (some ? __fdiv_rn(amax, 448.0f) : 0.0f) : __int_as_float(0x7fc00000);
        uint2 code = make_uint2(0u, 0u);
        if (finite && some) code = e4m3x8_rn(v, __frcp_rn(scale));
        stg_v2((is_v ? a.cache_v : a.cache_k) + head_row * a.head_dim + col, code);
        if (sub == 0) (is_v ? a.v_scales : a.k_scales)[head_row] = scale;
    }
}

// Reading back: out[i] = code * scale of cache row row_map[i] (i without a map), k and v in one launch; rows the map puts
// outside the cache come back as zeros. One lane per 8 values.
template <typename T>
__global__ void __launch_bounds__(kCtaThreads)
kv_read_fp8_kernel(typename T::storage* k_out, typename T::storage* v_out, const uint8_t* __restrict__ cache_k,
                   const uint8_t* __restrict__ cache_v, const float* __restrict__ k_scales,
                   const float* __restrict__ v_scales, const int* __restrict__ row_map, size_t pieces, int cache_rows,
                   int kv_heads, FastDiv piece_div, FastDiv heads_div) {
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const size_t step = (size_t)gridDim.x * kCtaThreads;
    for (size_t i = (size_t)blockIdx.x * kCtaThreads + threadIdx.x; i < 2 * pieces; i += step) {
        const bool is_v = i >= pieces;
        const uint32_t piece = (uint32_t)(is_v ? i - pieces : i);
        const uint32_t head_row = fast_div(piece, piece_div), part = piece - head_row * piece_div.d;
        const uint32_t row = fast_div(head_row, heads_div);
        const int at = row_map ? row_map[row] : (int)row;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if ((unsigned)at < (unsigned)cache_rows) {
            const size_t src = (size_t)at * kv_heads + (head_row - row * heads_div.d);
            const uint2 code = ldg_stream_v2((is_v ? cache_v : cache_k) + (src * piece_div.d + part) * 8);
            const float scale = (is_v ? v_scales : k_scales)[src];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint16_t pair = (uint16_t)((h < 2 ? code.x : code.y) >> (16 * (h & 1)));
                uint32_t f16;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16) : "h"(pair));
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16));
                v[2 * h] = f.x * scale;
                v[2 * h + 1] = f.y * scale;
            }
        }
        store8<T>((is_v ? v_out : k_out) + (size_t)piece * 8, v);
    }
}

}  // namespace clef
