// C-ABI of the FP8 (E4M3) KV cache: written behind RoPE, read back through a row map. Declarations:
// include/clef_fused.h. Same contract as the other entry points: asynchronous on the caller's stream, no allocation, no
// synchronisation, grids that depend on the shape arguments only.

#include "../../include/clef_fused.h"

#include <atomic>

#include "abi_support.cuh"
#include "kernels_kv_cache.cuh"

using namespace clef;
using namespace clef::abi;

namespace {

// Warps of `per_warp` head rows of a token.
template <typename K>
void launch_units(K kernel, std::atomic<int>& occ, int rows, int per_warp, cudaStream_t s, const DeviceInfo& dev, KvWriteArgs a) {
    const int per_sm = ctas_per_sm(kernel, 0, occ);
    a.parts_div = make_fast_div((uint32_t)((rows + per_warp - 1) / per_warp));
    const size_t units = (size_t)a.tokens * a.parts_div.d;
    launch_hot(kernel, balanced_grid((units + kCtaThreads / 32 - 1) / (kCtaThreads / 32), (size_t)dev.sms * per_sm), 0, s, a);
}

// U groups of head rows per warp where that still gives every SM 16 warps, one where it does not (8,192 tokens of 16 + 2
// heads of 128: 17.0 us with two or three groups, 18.1 with one or five).
template <typename T, int G>
void launch_kv_write(cudaStream_t s, const DeviceInfo& dev, const KvWriteArgs& a) {
    constexpr int U = 2;
    static std::atomic<int> occ[2];
    const int rows = a.q_heads + 2 * a.kv_heads;
    if ((size_t)a.tokens * rows / (32 / G) >= (size_t)dev.sms * 16 * U) {
        launch_units(kv_write_fp8_kernel<T, G, U>, occ[0], rows, U * (32 / G), s, dev, a);
    } else {
        launch_units(kv_write_fp8_kernel<T, G, 1>, occ[1], rows, 32 / G, s, dev, a);
    }
}
template <typename T, int G>
void launch_kv_norm_write(cudaStream_t s, const DeviceInfo& dev, const KvWriteArgs& a) {
    static std::atomic<int> occ{0};
    launch_units(kv_norm_write_fp8_kernel<T, G>, occ, 2 * a.kv_heads, 32 / G, s, dev, a);
}

template <typename T>
void launch_kv_write_for(cudaStream_t s, const DeviceInfo& dev, const KvWriteArgs& a, bool norm) {
    if (norm) {
        if (a.head_dim <= 64) launch_kv_norm_write<T, 8>(s, dev, a);
        else if (a.head_dim <= 128) launch_kv_norm_write<T, 16>(s, dev, a);
        else launch_kv_norm_write<T, 32>(s, dev, a);
    } else {
        if (a.head_dim <= 64) launch_kv_write<T, 4>(s, dev, a);
        else if (a.head_dim <= 128) launch_kv_write<T, 8>(s, dev, a);
        else launch_kv_write<T, 16>(s, dev, a);
    }
}

int kv_write_impl(const char* what, clef_stream_t stream, KvWriteArgs a, bool with_q, bool norm, int dtype) {
    if (int r = check_dtype(dtype, what)) return r;
    if (a.tokens < 0 || a.kv_heads <= 0 || (with_q && a.q_heads <= 0) || a.head_dim <= 0 || a.rotary_dim < 0 || a.cache_rows < 0) {
        return fail(CLEF_ERR_INVALID, "%s: tokens %d q_heads %d kv_heads %d head_dim %d rotary_dim %d cache_rows %d", what, a.tokens,
                    a.q_heads, a.kv_heads, a.head_dim, a.rotary_dim, a.cache_rows);
    }
    if (a.head_dim % 8 != 0 || a.rotary_dim % 16 != 0 || a.rotary_dim > a.head_dim) {
        return fail(CLEF_ERR_INVALID, "%s: head_dim %d must be a multiple of 8, rotary_dim %d one of 16 and not above head_dim", what,
                    a.head_dim, a.rotary_dim);
    }
    if (a.head_dim > kKvMaxHeadDim) return fail(CLEF_ERR_TOO_LARGE, "%s: head_dim %d above %d", what, a.head_dim, kKvMaxHeadDim);
    if (a.tokens == 0) return CLEF_OK;
    if (!a.cache_k || !a.cache_v || !a.k_scales || !a.v_scales || !a.k || !a.v || !a.cos_t || !a.sin_t ||
        (with_q && (!a.q || !a.q_out)) || (norm && !a.weight)) {
        return fail(CLEF_ERR_INVALID, "%s: null pointer", what);
    }
    if (with_q && a.q_out == a.q) return fail(CLEF_ERR_INVALID, "%s: q_out must not alias q", what);
    if ((with_q && (!aligned(a.q, 16) || !aligned(a.q_out, 16))) || !aligned(a.k, 16) || !aligned(a.v, 16) ||
        !aligned(a.cos_t, 16) || !aligned(a.sin_t, 16) || !aligned(a.cache_k, 8) || !aligned(a.cache_v, 8) ||
        !aligned(a.k_scales, 4) || !aligned(a.v_scales, 4) || !aligned(a.weight, 4)) {
        return fail(CLEF_ERR_INVALID, "%s: activations and tables must be 16-byte aligned, codes 8-byte", what);
    }
    if (!aligned(a.seq_start, 4) || !aligned(a.pos_base, 4) || !aligned(a.pos_map, 4) || !aligned(a.cache_map, 4) ||
        !aligned(a.cache_len, 4)) {
        return fail(CLEF_ERR_INVALID, "%s: positions and maps must be 4-byte aligned", what);
    }
    const long long per_token = (long long)a.q_heads + 2LL * a.kv_heads;
    // the grid-stride counter advances past the last head row by up to one grid of them
    if (per_token * a.tokens >= 0x40000000LL) return fail(CLEF_ERR_TOO_LARGE, "%s: %d tokens x %lld head rows", what, a.tokens, per_token);
    DeviceInfo dev;
    if (int r = device_info(dev)) return r;
    cudaStream_t s = as_stream(stream);
    if (dtype == CLEF_BF16) launch_kv_write_for<Bf16>(s, dev, a, norm);
    else launch_kv_write_for<F32>(s, dev, a, norm);
    return check_launch(what);
}

}  // namespace

extern "C" {

int clef_rope_kv_write_fp8(clef_stream_t stream, uint8_t* cache_k, uint8_t* cache_v, float* k_scales, float* v_scales,
                           const void* k, const void* v, const float* cos_table, const float* sin_table, int tokens,
                           int kv_heads, int head_dim, int rotary_dim, const int32_t* seq_start, const int32_t* pos_base,
                           const int32_t* pos_map, const int32_t* cache_map, const int32_t* cache_len, int cache_rows,
                           int dtype) {
    return kv_write_impl("clef_rope_kv_write_fp8", stream,
                         KvWriteArgs{nullptr, nullptr, 0, k, v, cache_k, cache_v, k_scales, v_scales, nullptr, cos_table, sin_table,
                                     seq_start, pos_base, pos_map, cache_map, cache_len, tokens, kv_heads, head_dim, rotary_dim,
                                     cache_rows, 0.0f, FastDiv{}}, false, false, dtype);
}

int clef_rope_qkv_write_fp8(clef_stream_t stream, void* q_out, const void* q, int q_heads, uint8_t* cache_k,
                            uint8_t* cache_v, float* k_scales, float* v_scales, const void* k, const void* v, int kv_heads,
                            const float* cos_table, const float* sin_table, int tokens, int head_dim, int rotary_dim,
                            const int32_t* seq_start, const int32_t* pos_base, const int32_t* pos_map,
                            const int32_t* cache_map, const int32_t* cache_len, int cache_rows, int dtype) {
    return kv_write_impl("clef_rope_qkv_write_fp8", stream,
                         KvWriteArgs{q, q_out, q_heads, k, v, cache_k, cache_v, k_scales, v_scales, nullptr, cos_table, sin_table,
                                     seq_start, pos_base, pos_map, cache_map, cache_len, tokens, kv_heads, head_dim, rotary_dim,
                                     cache_rows, 0.0f, FastDiv{}}, true, false, dtype);
}

int clef_qk_norm_rope_kv_write_fp8(clef_stream_t stream, uint8_t* cache_k, uint8_t* cache_v, float* k_scales,
                                   float* v_scales, const void* k_raw, const void* v, const float* weight,
                                   const float* cos_table, const float* sin_table, int tokens, int kv_heads, int head_dim,
                                   int rotary_dim, float eps, const int32_t* seq_start, const int32_t* pos_base,
                                   const int32_t* pos_map, const int32_t* cache_map, const int32_t* cache_len,
                                   int cache_rows, int dtype) {
    return kv_write_impl("clef_qk_norm_rope_kv_write_fp8", stream,
                         KvWriteArgs{nullptr, nullptr, 0, k_raw, v, cache_k, cache_v, k_scales, v_scales, weight, cos_table, sin_table,
                                     seq_start, pos_base, pos_map, cache_map, cache_len, tokens, kv_heads, head_dim, rotary_dim,
                                     cache_rows, eps, FastDiv{}}, false, true, dtype);
}

int clef_kv_read_fp8(clef_stream_t stream, void* k_out, void* v_out, const uint8_t* cache_k, const uint8_t* cache_v,
                     const float* k_scales, const float* v_scales, const int32_t* row_map, int rows, int cache_rows,
                     int kv_heads, int head_dim, int dtype) {
    const char* what = "clef_kv_read_fp8";
    if (int r = check_dtype(dtype, what)) return r;
    if (rows < 0 || cache_rows < 0 || kv_heads <= 0 || head_dim <= 0 || head_dim % 8 != 0) {
        return fail(CLEF_ERR_INVALID, "%s: rows %d cache_rows %d kv_heads %d head_dim %d (a multiple of 8)", what, rows, cache_rows,
                    kv_heads, head_dim);
    }
    if (rows == 0) return CLEF_OK;
    if (!k_out || !v_out || !cache_k || !cache_v || !k_scales || !v_scales) return fail(CLEF_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(cache_k, 8) || !aligned(cache_v, 8) || !aligned(k_scales, 4) ||
        !aligned(v_scales, 4) || !aligned(row_map, 4)) {
        return fail(CLEF_ERR_INVALID, "%s: outputs must be 16-byte aligned, codes 8-byte, scales and the map 4-byte", what);
    }
    const unsigned long long head_rows = (unsigned long long)rows * kv_heads;
    if (head_rows >= 0x7fffffffull || head_rows * (head_dim / 8) >= 0x7fffffffull) {
        return fail(CLEF_ERR_TOO_LARGE, "%s: %d rows of %d x %d", what, rows, kv_heads, head_dim);
    }
    DeviceInfo dev;
    if (int r = device_info(dev)) return r;
    cudaStream_t s = as_stream(stream);
    auto launch = [&](auto kernel, int codes, auto* k, auto* v) {
        const size_t pieces = (size_t)head_rows * (head_dim / codes);
        launch_hot(kernel, (unsigned)((pieces + kCtaThreads - 1) / kCtaThreads), 0, s, k, v, cache_k, cache_v, k_scales, v_scales,
                   (const int*)row_map, (uint32_t)pieces, cache_rows, kv_heads, make_fast_div((uint32_t)(kv_heads * (head_dim / codes))),
                   make_fast_div((uint32_t)(head_dim / codes)));
    };
    const bool wide = head_dim % 16 == 0 && aligned(cache_k, 16) && aligned(cache_v, 16) && aligned(k_out, 32) && aligned(v_out, 32);
    if (dtype == CLEF_BF16) {
        if (wide) launch(kv_read_fp8_kernel<Bf16, 16>, 16, (uint16_t*)k_out, (uint16_t*)v_out);
        else launch(kv_read_fp8_kernel<Bf16, 8>, 8, (uint16_t*)k_out, (uint16_t*)v_out);
    } else {
        if (wide) launch(kv_read_fp8_kernel<F32, 16>, 16, (float*)k_out, (float*)v_out);
        else launch(kv_read_fp8_kernel<F32, 8>, 8, (float*)k_out, (float*)v_out);
    }
    return check_launch(what);
}

}  // extern "C"
