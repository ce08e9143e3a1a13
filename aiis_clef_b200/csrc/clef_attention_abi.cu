// C-ABI of attention over a paged KV cache. Declarations: include/clef_fused.h. Same contract as the other entry
// points: asynchronous on the caller's stream, no allocation (the caller gives the workspace), no synchronisation,
// grids that depend on the shape arguments only.

#include "../../include/clef_fused.h"

#include <atomic>
#include <type_traits>

#include "abi_support.cuh"
#include "kernels_attention.cuh"
#include "kernels_attention_mma.cuh"

using namespace clef;
using namespace clef::abi;

namespace {

constexpr int kAttnMaxCtas = 320;     // two per SM of 160: the workspace does not depend on the device
constexpr int kAttnMaxGroup = 64;

struct AttnPlan {
    int rows;            // R: rows of a row tile
    bool chunk;          // attn_chunk_kernel, else attn_rows_kernel
    size_t items;        // bound on the (sequence, kv head, row tile) triples
    size_t bytes;        // of the workspace
};

// attn_rows_kernel up to an average of `most` rows per (sequence, kv head), attn_chunk_kernel above. At 32 rows of 8,192
// keys, 32 sequences: bf16 57 us in rows of 16, 53 us in chunks; FP8 53 against 70 us. Two groups of 8 rows of 256 bf16
// dims do not fit the registers (16 rows: 143 us, in chunks 84 us). Measured with equal rows in all sequences, the limit for
// FP8 at 128 dims alone: a batch of many single tokens and one chunk goes to one of the two whatever its parts would take.
AttnPlan attn_plan(int n_seqs, int total_q, int q_heads, int kv_heads, int head_dim, bool fp8) {
    AttnPlan p;
    const long long rows = (long long)total_q * (q_heads / kv_heads);
    const int most = fp8 ? 32 : (head_dim == 256 ? 8 : 16);
    p.chunk = rows > (long long)most * n_seqs;
    p.rows = p.chunk ? (head_dim == 256 ? 128 : 256) : (rows > 8LL * n_seqs ? 16 : 8);
    p.items = ((size_t)(rows / p.rows) + n_seqs) * kv_heads;
    const size_t ctas = p.chunk ? kAttnMaxCtas / 2 : kAttnMaxCtas;
    p.bytes = (size_t)kAttnMaxCtas * sizeof(AttnDesc) + ctas * 2 * p.rows * (head_dim + 2) * sizeof(float);
    return p;
}

// Raises a kernel's dynamic shared memory limit, once per device.
template <typename K>
int allow_smem(K kernel, size_t bytes, std::atomic<unsigned long long>& done, const char* what) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return e == cudaSuccess ? CLEF_OK : fail(CLEF_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <typename K, typename... Args>
void launch_pdl(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    (void)cudaLaunchKernelEx(&cfg, kernel, args...);   // errors surface in check_launch
}

// Launches `kernel` on the row tiles, and the joining kernel where one may have been cut. Up to WHOLE key tiles a row tile
// is left to one CTA: a join costs a launch and some 4 us, about what the key tiles cost one after the other (7 of them:
// 16.4 us in one CTA, 14.3 us cut and joined).
template <typename T, int D, int R, bool CHUNK, int WHOLE, typename K>
int launch_units(K kernel, unsigned threads, size_t smem, size_t most, cudaStream_t s, AttnArgs a, const AttnPlan& plan,
                 const char* what) {
    const size_t key_tiles = ((size_t)a.table_width * a.page_size + kAttnKeys - 1) / kAttnKeys;
    a.whole = key_tiles <= WHOLE;
    const unsigned ctas = clamp_grid(a.whole ? plan.items : plan.items * key_tiles, most);
    launch_pdl(kernel, dim3(ctas, 1, 1), threads, smem, s, a);
    if (int r = check_launch(what)) return r;
    if (a.whole || ctas <= 1) return CLEF_OK;
    // a run of 32 possible beginnings at most, fewer where more row tiles may begin
    const unsigned runs = clamp_grid(plan.items > (ctas + 31) / 32 ? plan.items : (ctas + 31) / 32, ctas);
    if constexpr (CHUNK) {
        if (ctas > 8 * plan.items) launch_pdl(attn_combine_rows_kernel<T, D, R, 8>, dim3(runs, R / 4, 1), 256, 0, s, a, (int)ctas);
        else launch_pdl(attn_combine_rows_kernel<T, D, R, 1>, dim3(runs, R / 32, 1), 256, 0, s, a, (int)ctas);
    } else {
        if (ctas > 8 * plan.items) launch_pdl(attn_combine_kernel<T, D, R, 8>, dim3(runs, R, D / 64), 256, 0, s, a, (int)ctas);
        else launch_pdl(attn_combine_kernel<T, D, R, 1>, dim3(runs, R / 8, 1), 256, 0, s, a, (int)ctas);
    }
    return check_launch(what);
}

template <typename T, bool FP8, int D, int NT>
int launch_rows(cudaStream_t s, const DeviceInfo& dev, const AttnArgs& a, const AttnPlan& plan, const char* what) {
    constexpr int R = 8 * NT;
    constexpr size_t smem = (size_t)(kAttnThreads / 32) * R * (D + 4 + 2) * sizeof(float);
    static std::atomic<unsigned long long> allowed{0};
    static std::atomic<int> occ{0};
    auto kernel = attn_rows_kernel<T, FP8, D, NT>;
    if (int r = allow_smem(kernel, smem, allowed, what)) return r;
    size_t most = (size_t)dev.sms * ctas_per_sm(kernel, smem, occ);
    if (most > kAttnMaxCtas) most = kAttnMaxCtas;
    return launch_units<T, D, R, false, 4>(kernel, kAttnThreads, smem, most, s, a, plan, what);
}

template <typename T, bool FP8, int D>
int launch_chunk(cudaStream_t s, const DeviceInfo& dev, const AttnArgs& a, const AttnPlan& plan, const char* what) {
    using Sh = ChunkShape<D, FP8>;
    static std::atomic<unsigned long long> allowed{0};
    auto kernel = attn_chunk_kernel<T, FP8, D>;
    if (int r = allow_smem(kernel, Sh::SMEM, allowed, what)) return r;
    const size_t most = dev.sms < kAttnMaxCtas / 2 ? dev.sms : kAttnMaxCtas / 2;
    return launch_units<T, D, Sh::R, true, 4>(kernel, Sh::THREADS, Sh::SMEM, most, s, a, plan, what);
}

template <typename T, bool FP8, int D>
int launch_for(cudaStream_t s, const DeviceInfo& dev, const AttnArgs& a, const AttnPlan& plan, const char* what) {
    if (plan.chunk) return launch_chunk<T, FP8, D>(s, dev, a, plan, what);
    if constexpr (FP8 || D != 256) {   // (a plan of 16 rows)
        if (plan.rows == 16) return launch_rows<T, FP8, D, 2>(s, dev, a, plan, what);
    }
    return launch_rows<T, FP8, D, 1>(s, dev, a, plan, what);
}

template <typename T, bool FP8>
int launch_attention(cudaStream_t s, const DeviceInfo& dev, const AttnArgs& a, const AttnPlan& plan, int head_dim,
                     const char* what) {
    if (head_dim == 64) return launch_for<T, FP8, 64>(s, dev, a, plan, what);
    if (head_dim == 128) return launch_for<T, FP8, 128>(s, dev, a, plan, what);
    return launch_for<T, FP8, 256>(s, dev, a, plan, what);
}

int check_attention_shape(const char* what, int n_seqs, int total_q, int q_heads, int kv_heads, int head_dim) {
    if (n_seqs < 0 || total_q < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0) {
        return fail(CLEF_ERR_INVALID, "%s: n_seqs %d total_q %d q_heads %d kv_heads %d (q_heads a multiple of kv_heads)", what,
                    n_seqs, total_q, q_heads, kv_heads);
    }
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
        return fail(CLEF_ERR_INVALID, "%s: head_dim %d (64, 128 and 256 are served)", what, head_dim);
    }
    const int group = q_heads / kv_heads;
    if (group > kAttnMaxGroup) return fail(CLEF_ERR_TOO_LARGE, "%s: %d query heads per kv head, above %d", what, group, kAttnMaxGroup);
    if ((long long)total_q * group >= 0x40000000LL || (long long)n_seqs * kv_heads >= 0x40000000LL) {
        return fail(CLEF_ERR_TOO_LARGE, "%s: total_q %d x %d heads, %d sequences", what, total_q, q_heads, n_seqs);
    }
    return CLEF_OK;
}

}  // namespace

extern "C" {

int clef_paged_attention_workspace(int n_seqs, int total_q, int q_heads, int kv_heads, int head_dim, size_t* bytes) {
    const char* what = "clef_paged_attention_workspace";
    if (!bytes) return fail(CLEF_ERR_INVALID, "%s: null pointer", what);
    if (int r = check_attention_shape(what, n_seqs, total_q, q_heads, kv_heads, head_dim)) return r;
    *bytes = 0;
    for (int fp8 = 0; fp8 < 2 && n_seqs > 0 && total_q > 0; ++fp8) {
        const size_t need = attn_plan(n_seqs, total_q, q_heads, kv_heads, head_dim, fp8 != 0).bytes;
        if (need > *bytes) *bytes = need;
    }
    return CLEF_OK;
}

int clef_paged_attention(clef_stream_t stream, void* out, const void* q, const void* cache_k, const void* cache_v,
                         const float* k_scales, const float* v_scales, const int32_t* page_table, const int32_t* q_start,
                         const int32_t* kv_len, int n_seqs, int total_q, int q_heads, int kv_heads, int head_dim,
                         int page_size, int table_width, int cache_pages, float scale, void* workspace,
                         size_t workspace_bytes, int cache_dtype, int dtype) {
    const char* what = "clef_paged_attention";
    if (int r = check_dtype(dtype, what)) return r;
    if (cache_dtype != CLEF_BF16 && cache_dtype != CLEF_E4M3) {
        return fail(CLEF_ERR_INVALID, "%s: cache_dtype %d is neither CLEF_BF16 nor CLEF_E4M3", what, cache_dtype);
    }
    if (int r = check_attention_shape(what, n_seqs, total_q, q_heads, kv_heads, head_dim)) return r;
    const int group = q_heads / kv_heads;
    if (page_size <= 0 || table_width <= 0 || cache_pages < 0) {
        return fail(CLEF_ERR_INVALID, "%s: page_size %d table_width %d cache_pages %d", what, page_size, table_width, cache_pages);
    }
    if ((long long)table_width * page_size * group >= 0x40000000LL || (long long)cache_pages * page_size >= 0x7fffffffLL) {
        return fail(CLEF_ERR_TOO_LARGE, "%s: %d pages of %d tokens per sequence, %d pages in the cache", what, table_width,
                    page_size, cache_pages);
    }
    if (n_seqs == 0 || total_q == 0) return CLEF_OK;
    if (!out || !q || !cache_k || !cache_v || !page_table || !q_start || !kv_len || !workspace ||
        (cache_dtype == CLEF_E4M3 && (!k_scales || !v_scales))) {
        return fail(CLEF_ERR_INVALID, "%s: null pointer", what);
    }
    if (out == q) return fail(CLEF_ERR_INVALID, "%s: out must not alias q", what);
    if (!aligned(out, 16) || !aligned(q, 16) || !aligned(cache_k, 16) || !aligned(cache_v, 16) || !aligned(workspace, 16)) {
        return fail(CLEF_ERR_INVALID, "%s: out, q, caches and workspace must be 16-byte aligned", what);
    }
    if (!aligned(page_table, 4) || !aligned(q_start, 4) || !aligned(kv_len, 4) ||
        (cache_dtype == CLEF_E4M3 && (!aligned(k_scales, 4) || !aligned(v_scales, 4)))) {
        return fail(CLEF_ERR_INVALID, "%s: scales, page table and lengths must be 4-byte aligned", what);
    }
    const AttnPlan plan = attn_plan(n_seqs, total_q, q_heads, kv_heads, head_dim, cache_dtype == CLEF_E4M3);
    if (workspace_bytes < plan.bytes) {
        return fail(CLEF_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, plan.bytes);
    }
    DeviceInfo dev;
    if (int r = device_info(dev)) return r;
    AttnArgs a{};
    a.q = q, a.out = out, a.k = cache_k, a.v = cache_v, a.k_scales = k_scales, a.v_scales = v_scales;
    a.table = page_table, a.q_start = q_start, a.kv_len = kv_len;
    a.n_seqs = n_seqs, a.total_q = total_q, a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = group;
    a.page_size = page_size, a.table_width = table_width, a.cache_pages = cache_pages;
    a.group_div = make_fast_div((uint32_t)group), a.page_div = make_fast_div((uint32_t)page_size);
    a.scale_log2 = scale * 1.44269504088896341f;
    a.desc = static_cast<AttnDesc*>(workspace);
    a.part = reinterpret_cast<float*>(a.desc + kAttnMaxCtas);
    cudaStream_t s = as_stream(stream);
    if (dtype == CLEF_BF16) {
        return cache_dtype == CLEF_BF16 ? launch_attention<Bf16, false>(s, dev, a, plan, head_dim, what)
                                        : launch_attention<Bf16, true>(s, dev, a, plan, head_dim, what);
    }
    return cache_dtype == CLEF_BF16 ? launch_attention<F32, false>(s, dev, a, plan, head_dim, what)
                                    : launch_attention<F32, true>(s, dev, a, plan, head_dim, what);
}

}  // extern "C"
