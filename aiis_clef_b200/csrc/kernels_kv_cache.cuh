// The FP8 (E4M3) KV cache: quantised as it is written, behind the key-side RoPE and optionally the per-head RMSNorm, and
// read back through a row map. One f32 scale per cache row and kv head:
//   scale = max |x| / 448,  code = e4m3(x * (1 / scale))  round to nearest even, x the f32 value the bf16 cache would round
// (a scale per head row costs 4 bytes beside head_dim codes and keeps an outlier head from flattening the others).
// A head row whose maximum is below 2^-100 is stored as zeros with scale 0; one that holds an infinity or a NaN is
// stored as zero codes with scale NaN, so that whatever reads it sees NaN.
//
// Bound by HBM bytes, if the instructions per row are few. A lane takes 16 values of a head row: 8 of the rotated half
// and their partners half a rotary span up, or 16 that pass through (G = head_dim / 16 lanes for a head row, rounded up
// to a power of two); nothing is exchanged but the row maximum. A warp takes U groups of 32 / G head rows of ONE token,
// requested together: a lane's columns, and with them its cosines and sines, are the same in all of them, and the chain
// position -> table runs beside the rows' own loads. With the per-head norm (k rows only) a lane takes 8 consecutive
// values instead, the order of the sum. Measured: 8,192 tokens of 16 + 2 heads of 128 (84 MB) 18.7 us a call in a stream of
// calls = 4.5 TB/s, 17.2 us under a profiler, alone (a lane of 8 values with its partner fetched by shuffles: 22.4 us).
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
    FastDiv parts_div;    // warps per token
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

// Eight activations as they are loaded.
template <typename T>
struct Raw8 {
    uint4 w[T::kBytes / 2];
};
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float* v);
template <>
__device__ __forceinline__ void widen8<Bf16>(const Raw8<Bf16>& r, float* v) {
    const uint4 d = r.w[0];
    v[0] = bf16_lo(d.x), v[1] = bf16_hi(d.x), v[2] = bf16_lo(d.y), v[3] = bf16_hi(d.y);
    v[4] = bf16_lo(d.z), v[5] = bf16_hi(d.z), v[6] = bf16_lo(d.w), v[7] = bf16_hi(d.w);
}
template <>
__device__ __forceinline__ void widen8<F32>(const Raw8<F32>& r, float* v) {
    const uint4 a = r.w[0], b = r.w[1];
    v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
}

template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const float* v);
template <>
__device__ __forceinline__ Raw8<Bf16> narrow8<Bf16>(const float* v) {
    return Raw8<Bf16>{{make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]))}};
}
template <>
__device__ __forceinline__ Raw8<F32> narrow8<F32>(const float* v) {
    return Raw8<F32>{{make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])),
                      make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]))}};
}

// Where a token's rows go; false for a padding token.
__device__ __forceinline__ bool kv_place(const KvWriteArgs& a, int token, size_t& row) {
    const long long at = a.cache_map ? (long long)a.cache_map[token] : (long long)token + (a.cache_len ? a.cache_len[0] : 0);
    row = (size_t)at;
    return at >= 0 && at < a.cache_rows;
}
// The row of the tables that a token's lanes read. A padding token's position may be anything where only k and v are
// written (they are not), and counts as 0; beside q, whose rows are rotated all the same, only a negative one does. (A
// position, not a branch around the loads, and with q no look at the place: 4.2 us for the k and v of 8,192 tokens of 64
// dims took 5.6 so.)
__device__ __forceinline__ int kv_position(const KvWriteArgs& a, int token) {
    const int pos = rope_position(token, a.seq_start, a.pos_base, a.pos_map);
    if (a.q_heads > 0) return max(pos, 0);
    size_t row;
    return kv_place(a, token, row) ? pos : 0;
}
// The scale of a head row with maximum `amax` (NaN if it holds one), and the factor its values are multiplied by (0: codes 0).
__device__ __forceinline__ float kv_scale(float amax, float& by) {
    const bool finite = amax < INFINITY, some = amax >= kKvMinAmax;   // both false for a NaN
    const float scale = finite ? (some ? __fdiv_rn(amax, 448.0f) : 0.0f) : __int_as_float(0x7fc00000);
    by = finite && some ? __frcp_rn(scale) : 0.0f;
    return scale;
}

template <typename T, int G, int U>
__global__ void __launch_bounds__(kCtaThreads)
kv_write_fp8_kernel(KvWriteArgs a) {
    constexpr int PER_WARP = 32 / G;
    const int lane = threadIdx.x & 31, sub = lane % G;
    const int half = a.rotary_dim >> 1, turning = half >> 3;   // lanes of a row that rotate
    const bool turns_at = sub < turning;
    const int col = turns_at ? sub * 8 : a.rotary_dim + (sub - turning) * 16, col2 = turns_at ? col + half : col + 8;
    const bool in_row = col < a.head_dim, in_row2 = col2 < a.head_dim;
    const int rows = a.q_heads + 2 * a.kv_heads, parts = (int)a.parts_div.d;
    const uint32_t units = (uint32_t)a.tokens * parts;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    for (uint32_t unit = blockIdx.x * (kCtaThreads / 32) + (threadIdx.x >> 5); unit < units; unit += gridDim.x * (kCtaThreads / 32)) {
        const int token = (int)fast_div(unit, a.parts_div);
        const int first = ((int)unit - token * parts) * (U * PER_WARP) + lane / G;
        Raw8<T> raw[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = first + u * PER_WARP, kv = row - a.q_heads;
            const int head = kv < 0 ? row : (kv < a.kv_heads ? kv : kv - a.kv_heads);
            const typename T::storage* x = static_cast<const typename T::storage*>(kv < 0 ? a.q : (kv < a.kv_heads ? a.k : a.v)) +
                                           ((size_t)token * (kv < 0 ? a.q_heads : a.kv_heads) + head) * a.head_dim;
#pragma unroll
            for (int i = 0; i < T::kBytes / 2; ++i) {
                raw[u][0].w[i] = in_row && row < rows ? ldg_stream_v4(reinterpret_cast<const uint8_t*>(x + col) + 16 * i) : make_uint4(0, 0, 0, 0);
                raw[u][1].w[i] = in_row2 && row < rows ? ldg_stream_v4(reinterpret_cast<const uint8_t*>(x + col2) + 16 * i) : make_uint4(0, 0, 0, 0);
            }
        }
        float c[8], s[8];
        if (turns_at) {
            const int pos = kv_position(a, token);
            const size_t at = (size_t)pos * a.rotary_dim + col;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *reinterpret_cast<float4*>(c + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at) + i);
                *reinterpret_cast<float4*>(s + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at) + i);
            }
        }
        size_t place;
        const bool kept = kv_place(a, token, place);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = first + u * PER_WARP;
            if (row - lane / G >= rows) break;   // (the whole warp)
            const bool is_q = row < a.q_heads, is_v = row >= a.q_heads + a.kv_heads, live = in_row && row < rows;
            if (__all_sync(kFullMask, is_q)) {   // rotated or passed through, in the activation type
                if (turns_at) {
                    float v[8], w[8];
                    widen8<T>(raw[u][0], v);
                    widen8<T>(raw[u][1], w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) rope_pair(v[i], w[i], c[i], s[i], v[i], w[i]);
                    raw[u][0] = narrow8<T>(v);
                    raw[u][1] = narrow8<T>(w);
                }
                uint8_t* dst = reinterpret_cast<uint8_t*>(static_cast<typename T::storage*>(a.q_out) + ((size_t)token * a.q_heads + row) * a.head_dim);
#pragma unroll
                for (int i = 0; i < T::kBytes / 2; ++i) {
                    if (in_row) stg_v4(dst + (size_t)col * T::kBytes + 16 * i, raw[u][0].w[i]);
                    if (in_row2) stg_v4(dst + (size_t)col2 * T::kBytes + 16 * i, raw[u][1].w[i]);
                }
                continue;
            }
            float v[8], w[8];
            widen8<T>(raw[u][0], v);
            widen8<T>(raw[u][1], w);
            if (turns_at && !is_v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) rope_pair(v[i], w[i], c[i], s[i], v[i], w[i]);
            }
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = max3_abs_nan(amax, v[i], w[i]);
#pragma unroll
            for (int off = G / 2; off > 0; off >>= 1) amax = fmaxf_nan(amax, __shfl_xor_sync(kFullMask, amax, off));
            if (!live) continue;
            if (is_q) {   // a group with rows of both kinds
                typename T::storage* dst = static_cast<typename T::storage*>(a.q_out) + ((size_t)token * a.q_heads + row) * a.head_dim;
                store8<T>(dst + col, v);
                if (in_row2) store8<T>(dst + col2, w);
            } else if (kept) {
                const size_t head_row = place * a.kv_heads + (row - a.q_heads - (is_v ? a.kv_heads : 0));
                float by;
                const float scale = kv_scale(amax, by);
                uint8_t* dst = (is_v ? a.cache_v : a.cache_k) + head_row * a.head_dim;
                stg_v2(dst + col, by > 0.0f ? e4m3x8_rn(v, by) : make_uint2(0u, 0u));
                if (in_row2) stg_v2(dst + col2, by > 0.0f ? e4m3x8_rn(w, by) : make_uint2(0u, 0u));
                if (sub == 0) (is_v ? a.v_scales : a.k_scales)[head_row] = scale;
            }
        }
    }
}

// k rows normalised first, in the summation order of rms_norm_kernel (kernels/elementwise.cu:4-68: quad i with quad i + 32,
// then the tree 16, 8, 4, 2, 1 over quads); G = head_dim / 8 lanes per head row, k and v rows of a token.
template <typename T, int G>
__global__ void __launch_bounds__(kCtaThreads)
kv_norm_write_fp8_kernel(KvWriteArgs a) {
    constexpr int PER_WARP = 32 / G;
    const int lane = threadIdx.x & 31, sub = lane % G;
    const int col = sub * 8, half = a.rotary_dim >> 1;
    const bool in_row = col < a.head_dim, rotary = col < a.rotary_dim, upper = col >= half;
    const int partner = rotary ? (upper ? lane - (half >> 3) : lane + (half >> 3)) : lane;
    const int rows = 2 * a.kv_heads, parts = (int)a.parts_div.d;
    const uint32_t units = (uint32_t)a.tokens * parts;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    for (uint32_t unit = blockIdx.x * (kCtaThreads / 32) + (threadIdx.x >> 5); unit < units; unit += gridDim.x * (kCtaThreads / 32)) {
        const int token = (int)fast_div(unit, a.parts_div);
        const int row = ((int)unit - token * parts) * PER_WARP + lane / G;
        const bool is_v = row >= a.kv_heads, live = in_row && row < rows;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (live) {
            load8<T>(static_cast<const typename T::storage*>(is_v ? a.v : a.k) +
                     ((size_t)token * a.kv_heads + (is_v ? row - a.kv_heads : row)) * a.head_dim + col, v);
        }
        float c[8], s[8];
        if (rotary) {
            const int pos = kv_position(a, token);
            const size_t at = (size_t)pos * a.rotary_dim + (upper ? col - half : col);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *reinterpret_cast<float4*>(c + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at) + i);
                *reinterpret_cast<float4*>(s + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at) + i);
            }
        }
        float s0 = quad_sq(make_float4(v[0], v[1], v[2], v[3])), s1 = quad_sq(make_float4(v[4], v[5], v[6], v[7]));
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) {
            s0 = __fadd_rn(s0, __shfl_xor_sync(kFullMask, s0, off));
            s1 = __fadd_rn(s1, __shfl_xor_sync(kFullMask, s1, off));
        }
        if (live && !is_v) {
            const float inv = inv_rms(__fadd_rn(s0, s1), a.head_dim, a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * (1.0f + a.weight[col + i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(kFullMask, v[i], partner);
            float lo, hi;
            if (rotary && !is_v) {
                rope_pair(upper ? other : v[i], upper ? v[i] : other, c[i], s[i], lo, hi);
                v[i] = upper ? hi : lo;
            }
        }
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) amax = max3_abs_nan(amax, v[i], v[i + 1]);
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) amax = fmaxf_nan(amax, __shfl_xor_sync(kFullMask, amax, off));
        size_t place;
        if (kv_place(a, token, place) && live) {
            const size_t head_row = place * a.kv_heads + (is_v ? row - a.kv_heads : row);
            float by;
            const float scale = kv_scale(amax, by);
            stg_v2((is_v ? a.cache_v : a.cache_k) + head_row * a.head_dim + col, by > 0.0f ? e4m3x8_rn(v, by) : make_uint2(0u, 0u));
            if (sub == 0) (is_v ? a.v_scales : a.k_scales)[head_row] = scale;
        }
    }
}

// Reading back: out[i] = code * scale of cache row row_map[i] (i without a map); rows the map puts outside the cache come
// back as zeros. A lane takes CODES of a row's k and the same of its v (16 where head_dim allows: 16-byte loads, 32 bytes
// out), so that the way from the row number to the codes is walked once for both, and each thread has one piece: with
// full occupancy that streamed better than several pieces a thread. Bound by HBM bytes: 130,712 rows of 2 x 128 to bf16
// (204 MB) 33.5 us a call in a stream of calls = 6.1 TB/s (30.1 us under a profiler, alone).
template <typename T, int CODES>
__global__ void __launch_bounds__(kCtaThreads)
kv_read_fp8_kernel(typename T::storage* __restrict__ k_out, typename T::storage* __restrict__ v_out,
                   const uint8_t* __restrict__ cache_k, const uint8_t* __restrict__ cache_v, const float* __restrict__ k_scales,
                   const float* __restrict__ v_scales, const int* __restrict__ row_map, uint32_t pieces, int cache_rows,
                   int kv_heads, FastDiv row_div, FastDiv head_div) {
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const uint32_t piece = blockIdx.x * kCtaThreads + threadIdx.x;
    if (piece >= pieces) return;
    const uint32_t row = fast_div(piece, row_div), part = piece - row * row_div.d;
    const int at = row_map ? row_map[row] : (int)row;
    const bool there = (unsigned)at < (unsigned)cache_rows;
    const size_t src = ((size_t)(there ? at : 0) * row_div.d + part) * CODES;
    const size_t head_row = (size_t)(there ? at : 0) * kv_heads + fast_div(part, head_div);
    uint32_t code[2][CODES / 4];
    float scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint8_t* p = (h == 0 ? cache_k : cache_v) + src;
        if (CODES == 16) {
            const uint4 t = there ? ldg_stream_v4(p) : make_uint4(0, 0, 0, 0);
            code[h][0] = t.x, code[h][1] = t.y, code[h][CODES / 4 - 2] = t.z, code[h][CODES / 4 - 1] = t.w;
        } else {
            const uint2 t = there ? ldg_stream_v2(p) : make_uint2(0, 0);
            code[h][0] = t.x, code[h][1] = t.y;
        }
        scale[h] = there ? (h == 0 ? k_scales : v_scales)[head_row] : 0.0f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[CODES];
#pragma unroll
        for (int w = 0; w < CODES / 2; ++w) {
            const uint16_t pair = (uint16_t)(code[h][w / 2] >> (16 * (w & 1)));
            uint32_t f16;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16) : "h"(pair));
            const f32x2 f = f2_mul(__half22float2(*reinterpret_cast<const __half2*>(&f16)), f2_splat(scale[h]));
            v[2 * w] = f.x, v[2 * w + 1] = f.y;
        }
        typename T::storage* dst = (h == 0 ? k_out : v_out) + (size_t)piece * CODES;
        if (T::kBytes == 2 && CODES == 16) {
            U8x32 o;   // (the outputs are 32-byte aligned then)
#pragma unroll
            for (int w = 0; w < 8; ++w) o.w[w] = pack_bf16x2(v[2 * w], v[2 * w + 1 < CODES ? 2 * w + 1 : 0]);
            stg_v8(dst, o);
        } else {
#pragma unroll
            for (int w = 0; w < CODES; w += 8) store8<T>(dst + w, v + w);
        }
    }
}

}  // namespace clef
