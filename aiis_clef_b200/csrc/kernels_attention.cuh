// Attention of new tokens over a paged KV cache: single generated tokens, chunks of a prompt, and batches that mix
// the two. For query row i of a sequence with n new tokens and kv cached ones (the new ones included, they are the
// last n), the keys it sees are 0 .. kv - n + i:
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp2(scale log2(e) q_i . k_j - m_i),   m_i = running maximum
// Scores, maxima, sums and outputs are f32; q and p enter the products as bf16 over a bf16 cache, as f16 over an FP8 one.
//
// The q heads that share a kv head are rows of ONE product: row x of a (sequence, kv head) is new token x / group,
// head x % group. Rows are cut into row tiles of R, keys into tiles of kAttnKeys, and the (row tile, key tile) units
// of the whole batch are one flat list that every CTA takes an equal, contiguous share of: a lone long sequence
// fills the machine as well as an uneven batch does, and the grid depends on shapes alone. A row tile whose keys
// were cut over several CTAs leaves (m, l, o) partials in the workspace, and a second kernel joins them in a fixed
// order, so results do not depend on timing.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "f32x2.cuh"
#include "kernels_generic.cuh"
#include "kernels_hot.cuh"

namespace clef {

constexpr int kAttnKeys = 128;      // keys of one unit
constexpr int kAttnThreads = 256;   // attn_rows_kernel: 8 warps, 16 keys each per unit

struct AttnArgs {
    const void* q;              // [total_q, q_heads, head_dim]
    void* out;                  // as q
    const void* k;              // [cache_pages * page_size, kv_heads, head_dim], bf16 or E4M3 codes
    const void* v;
    const float* k_scales;      // [cache_pages * page_size, kv_heads], E4M3 caches only
    const float* v_scales;
    const int* table;           // [n_seqs, table_width] page numbers
    const int* q_start;         // [n_seqs + 1] first q row of each sequence
    const int* kv_len;          // [n_seqs]
    int n_seqs, total_q, q_heads, kv_heads, group;
    int page_size, table_width, cache_pages;
    FastDiv group_div, page_div;
    float scale_log2;           // scale * log2(e): the softmax runs on exp2
    int whole;                  // row tiles are not cut: all cost the same, nothing is left to join
    struct AttnDesc* desc;      // workspace: what is in slot 1 of each CTA
    float* part;                // workspace: per slot R maxima, R sums, R x head_dim outputs (attn_chunk_kernel: [head_dim / 4][R][4])
};

// Slot 1 of a CTA holds the beginning of a row tile that later CTAs go on with, slot 0 its CTA's share of a row tile
// begun by an earlier one. What is in slot 1:
struct AttnDesc {
    int parts;                    // CTAs that share the row tile, this one first; 0: the slot is empty
    int tile, head, q0, rows;     // rows: of the sequence and kv head
    int unused[3];
};

__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The lengths of one sequence, clamped so that no value of the maps leads outside q, out or the page table.
struct AttnSeq {
    int q0, n, kv;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int s) {
    AttnSeq r;
    r.q0 = min(max(a.q_start[s], 0), a.total_q);
    r.n = min(max(a.q_start[s + 1], r.q0), a.total_q) - r.q0;
    r.kv = min(max(a.kv_len[s], 0), a.table_width * a.page_size);
    return r;
}

// Keys visible to the last of the first `rows` rows of a sequence (0 if none).
__device__ __forceinline__ int attn_visible(const AttnArgs& a, const AttnSeq& q, int rows) {
    return max(0, q.kv - q.n + (int)fast_div((uint32_t)(rows - 1), a.group_div) + 1);
}
// Key tiles of row tile `tile`, at least one (a row that sees nothing still has to be written).
template <int R>
__device__ __forceinline__ int attn_key_tiles(const AttnArgs& a, const AttnSeq& q, int tile) {
    const int rows = min((tile + 1) * R, q.n * a.group);
    return max(1, (attn_visible(a, q, rows) + kAttnKeys - 1) / kAttnKeys);
}

// Work is shared out by a cost that is linear in the row tile's number, so that sums over row tiles need no loop and no
// division: a row tile of a sequence with kv - n cached keys before its new ones costs
//   OV * unit + max(0, (kv - n) * group + (tile + 1) R)      with unit = group * kAttnKeys the cost of a key tile,
// which is `group` times the keys its last row sees, and OV key tiles' worth for its beginning and end. (Where sequences
// are short, a.whole: every row tile costs 1 and shares are whole numbers of them.)
template <int R, int OV>
__device__ __forceinline__ long long attn_tile_cost(const AttnArgs& a, const AttnSeq& q, int tile) {
    if (a.whole) return 1;
    return (long long)OV * a.group * kAttnKeys + max(0, (q.kv - q.n) * a.group + (tile + 1) * R);
}
// Cost of all row tiles of one (sequence, kv head).
template <int R, int OV>
__device__ __forceinline__ long long attn_seq_cost(const AttnArgs& a, const AttnSeq& q) {
    const int tiles = (q.n * a.group + R - 1) / R;
    if (a.whole) return tiles;
    const int ahead = (q.kv - q.n) * a.group;
    const int none = ahead >= 0 ? 0 : min(tiles, -ahead / R);   // row tiles whose linear part is 0
    const long long some = tiles - none;
    return (long long)tiles * OV * a.group * kAttnKeys + some * ahead + (long long)R * (some * (none + 1) + some * (some - 1) / 2);
}

// A CTA's place in the list: (sequence, kv head, row tile), the row tile's cost, how much of it lies before the CTA's
// share, and how much of the share is left.
struct AttnCursor {
    int seq, head, tile, keys;   // `keys`: key tiles of the row tile
    AttnSeq span;
    long long cost, at, left, share;
};

// The cursor of CTA `cta` of `ctas`. One warp, all lanes; every lane has the result.
template <int R, int OV>
__device__ inline AttnCursor attn_locate(const AttnArgs& a, int cta, int ctas) {
    const int lane = threadIdx.x & 31;
    AttnCursor c;
    c.seq = c.head = c.tile = c.keys = 0;
    c.span = AttnSeq{0, 0, 0};
    c.cost = c.at = 0;
    long long total = 0;
    for (int s = lane; s < a.n_seqs; s += 32) total += a.kv_heads * attn_seq_cost<R, OV>(a, attn_seq(a, s));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(kFullMask, total, off);
    // equal shares, but of a key tile at least: the CTAs that work are the first ones
    c.share = max((total + ctas - 1) / ctas, a.whole ? 1ll : (long long)a.group * kAttnKeys);
    long long at = cta * c.share;
    c.left = min(c.share, total - at);
    if (c.left <= 0) return c;
    long long per_head = 0;
    for (int base = 0; base < a.n_seqs; base += 32) {   // the sequence: scans of 32
        const int s = base + lane;
        const long long mine = s < a.n_seqs ? attn_seq_cost<R, OV>(a, attn_seq(a, s)) : 0;
        long long upto = mine * a.kv_heads;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long t = __shfl_up_sync(kFullMask, upto, off);
            if (lane >= off) upto += t;
        }
        const unsigned past = __ballot_sync(kFullMask, upto > at);
        if (past) {
            const int hit = __ffs(past) - 1;
            c.seq = base + hit;
            per_head = __shfl_sync(kFullMask, mine, hit);
            at -= __shfl_sync(kFullMask, upto, hit) - per_head * a.kv_heads;
            break;
        }
        at -= __shfl_sync(kFullMask, upto, 31);
    }
    c.span = attn_seq(a, c.seq);
    for (; at >= per_head; at -= per_head) ++c.head;
    const int tiles = (c.span.n * a.group + R - 1) / R;
    for (int base = 0; base < tiles; base += 32) {      // the row tile: scans of 32
        const long long mine = base + lane < tiles ? attn_tile_cost<R, OV>(a, c.span, base + lane) : 0;
        long long upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long t = __shfl_up_sync(kFullMask, upto, off);
            if (lane >= off) upto += t;
        }
        const unsigned past = __ballot_sync(kFullMask, upto > at);
        if (past) {
            const int hit = __ffs(past) - 1;
            c.tile = base + hit;
            c.cost = __shfl_sync(kFullMask, mine, hit);
            c.at = at - (__shfl_sync(kFullMask, upto, hit) - c.cost);
            break;
        }
        at -= __shfl_sync(kFullMask, upto, 31);
    }
    c.keys = attn_key_tiles<R>(a, c.span, c.tile);
    return c;
}

// The key tiles [begin, end) of the cursor's row tile that fall to its CTA: where a share ends at cost x of a row tile, the
// key tiles before it are those of round((x - OV units) / unit); none, if it ends within the OV units (the next CTA then
// begins the row tile), all, if the row tile ends in the share.
template <int OV>
__device__ __forceinline__ int attn_tiles_before(const AttnArgs& a, const AttnCursor& c, long long x) {
    const int unit = a.group * kAttnKeys, y = (int)(x - (long long)OV * unit) + unit / 2;
    return y <= 0 ? 0 : min(c.keys, y / unit);
}
template <int OV>
__device__ __forceinline__ void attn_segment(const AttnArgs& a, const AttnCursor& c, int& begin, int& end) {
    begin = attn_tiles_before<OV>(a, c, c.at);
    end = c.at + c.left >= c.cost ? c.keys : attn_tiles_before<OV>(a, c, c.at + c.left);
}
// The description of a row tile that begins in this CTA's share and goes on after it: the shares that follow, up to the
// row tile's end or the one that finds no key tile left.
template <int OV>
__device__ __forceinline__ AttnDesc attn_describe(const AttnArgs& a, const AttnCursor& c) {
    const long long rest = c.cost - (c.at + c.left);
    int more = (int)((rest + c.share - 1) / c.share);
    while (more > 0 && attn_tiles_before<OV>(a, c, c.at + c.left + (more - 1) * c.share) >= c.keys) --more;
    return AttnDesc{1 + more, c.tile, c.head, c.span.q0, c.span.n * a.group};
}

// On to the next row tile, if some of the share is left.
template <int R, int OV>
__device__ __forceinline__ void attn_advance(const AttnArgs& a, AttnCursor& c) {
    c.left -= c.cost - c.at;
    if (c.left <= 0) return;
    c.at = 0;
    if ((c.tile + 1) * R < c.span.n * a.group) {
        ++c.tile;
    } else {
        c.tile = 0;
        if (++c.head == a.kv_heads) {
            c.head = 0;
            do {
                ++c.seq;
                c.span = attn_seq(a, c.seq);
            } while (c.span.n == 0 && c.seq + 1 < a.n_seqs);
        }
    }
    c.cost = attn_tile_cost<R, OV>(a, c.span, c.tile);
    c.keys = attn_key_tiles<R>(a, c.span, c.tile);
}

__device__ __forceinline__ float* attn_slot(const AttnArgs& a, int cta, int slot, int rows, int head_dim) {
    return a.part + (size_t)(2 * cta + slot) * rows * (head_dim + 2);
}

// Cache row of key `t` of sequence `seq`, or -1 where the table names a page that is not there (such a key reads as zeros).
__device__ __forceinline__ int attn_cache_row(const AttnArgs& a, int seq, int t) {
    const int page = (int)fast_div((uint32_t)t, a.page_div);
    const int at = a.table[(size_t)seq * a.table_width + page];
    return (unsigned)at < (unsigned)a.cache_pages ? at * a.page_size + (t - page * a.page_size) : -1;
}

// Four E4M3 codes -> two f16 pairs, exactly.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <bool F16>
__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (F16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// ---------------------------------------------------------------------------------------------
// Few rows per (sequence, kv head): generated tokens and short chunks, bound by the cache bytes.
//
// The product runs transposed, S^T = K Q^T and O^T = V^T P^T, so the 8-wide side of m16n8k16 holds the query rows
// (8 grouped heads fill it) and the 16-wide sides hold keys and head dims. A fragment's place in the contraction is
// free as long as both operands agree, so K and V go from global memory straight into the fragments with 16-byte
// loads, without shared memory: lane (r, c) = (lane / 4, lane % 4) takes 16 bytes at column 16 c of key r for S^T,
// and 16 bytes at column 16 r of keys 2c, 2c + 1, 2c + 8, 2c + 9 for O^T, where a byte permute pairs two keys. Warps
// take 16 keys each, keep their own softmax statistics, and are joined in shared memory at the end of a row tile.
// The next keys are requested as soon as the registers of the current ones are free.
// Bound by the cache bytes: one token over 130,712 keys of 2 x 256 in bf16 (268 MB) 51.6 us with the join = 5.2 TB/s, 64 tokens
// over up to 8,192 keys of 2 x 128 in FP8 (157 MB) 41.5 us = 3.8 TB/s, where the conversions take their part. (Through shared
// memory with asynchronous copies, three steps deep, the latter took 65 us against 49 then.)
// An FP8 cache is multiplied in f16, which holds every E4M3 code and which one conversion instruction gives for two
// codes (bf16 takes five). What else enters the products is brought into f16's range by powers of two: a q row is
// divided by one so that its largest element is in [1, 2), and weight times value scale by the running maximum of the
// value scales that the ROW sees; both are multiplied back in f32. f16 then rounds finer than bf16 (2^-11), down to 2^-14 of
// the maximum.
// ---------------------------------------------------------------------------------------------
template <typename T, bool FP8, int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, (D == 256 || NT > 1 || !FP8) ? 1 : 2)
attn_rows_kernel(AttnArgs a) {
    constexpr int R = 8 * NT, OV = 1;
    constexpr int WARPS = kAttnThreads / 32;
    constexpr int KSTEP = FP8 ? 64 : 32;             // head dims of one 16-byte load by the four lanes of a key
    constexpr int KL = D / KSTEP;                    // such loads per key
    constexpr int VCH = FP8 && D >= 128 ? 16 : 8;    // head dims of V a lane takes at once
    constexpr int VL = D / (8 * VCH);                // such pieces per key
    constexpr int VW = VCH * (FP8 ? 1 : 2) / 4;      // words of a piece
    constexpr int PAD = 4;
    using CacheT = typename std::conditional<FP8, uint8_t, uint16_t>::type;
    __shared__ AttnCursor s_cursor;
    extern __shared__ float s_o[];                   // [WARPS][R][D + PAD], then [WARPS][R] maxima and sums
    float* s_m = s_o + WARPS * R * (D + PAD);
    float* s_l = s_m + WARPS * R;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, c = lane & 3;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const CacheT* kc = static_cast<const CacheT*>(a.k);
    const CacheT* vc = static_cast<const CacheT*>(a.v);
    if (warp == 0) {
        const AttnCursor at = attn_locate<R, OV>(a, blockIdx.x, gridDim.x);
        if (lane == 0) s_cursor = at;
    }
    if (threadIdx.x == 0) a.desc[blockIdx.x].parts = 0;
    __syncthreads();
    AttnCursor cur = s_cursor;
    for (; cur.left > 0; attn_advance<R, OV>(a, cur)) {
        int begin, end;
        attn_segment<OV>(a, cur, begin, end);
        if (begin == end) continue;
        const AttnSeq span = cur.span;
        const int row0 = cur.tile * R, rows = span.n * a.group;
        const int keys = attn_visible(a, span, min(row0 + R, rows));   // seen by any row of the tile
        uint4 kr[2][KL];
        uint32_t vr[4][VL][VW];
        float ks[2], vs[2];
        auto lookup = [&](int tile) {   // lanes 0-15: the cache row of key `lane` of this warp's 16
            const int t = tile * kAttnKeys + warp * 16 + (lane & 15);
            return tile < end && t < keys ? attn_cache_row(a, cur.seq, t) : -1;
        };
        auto load_k = [&](int row16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = __shfl_sync(kFullMask, row16, r + 8 * h);
                const size_t head_row = (size_t)(row < 0 ? 0 : row) * a.kv_heads + cur.head;
                const uint8_t* p = reinterpret_cast<const uint8_t*>(kc + head_row * D) + 16 * c;
#pragma unroll
                for (int i = 0; i < KL; ++i) kr[h][i] = row < 0 ? make_uint4(0, 0, 0, 0) : ldg_stream_v4(p + 64 * i);
                if (FP8) ks[h] = row < 0 ? 0.0f : a.k_scales[head_row];
                if (FP8) vs[h] = row < 0 ? 0.0f : a.v_scales[head_row];
            }
        };
        auto load_v = [&](int row16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = __shfl_sync(kFullMask, row16, 2 * c + (j & 1) + 8 * (j >> 1));
                const uint8_t* p = reinterpret_cast<const uint8_t*>(vc + ((size_t)(row < 0 ? 0 : row) * a.kv_heads + cur.head) * D) + 4 * VW * r;
#pragma unroll
                for (int b = 0; b < VL; ++b) {
                    if (VW == 4) {
                        const uint4 t = row < 0 ? make_uint4(0, 0, 0, 0) : ldg_stream_v4(p + 32 * VW * b);
                        vr[j][b][0] = t.x, vr[j][b][1] = t.y, vr[j][b][VW - 2] = t.z, vr[j][b][VW - 1] = t.w;
                    } else {
                        const uint2 t = row < 0 ? make_uint2(0, 0) : ldg_stream_v2(p + 32 * VW * b);
                        vr[j][b][0] = t.x, vr[j][b][1] = t.y;
                    }
                }
            }
        };
        // the first keys are asked for before q, whose way is shorter
        int row16 = lookup(begin);
        load_k(row16);
        load_v(row16);
        row16 = lookup(begin + 1);
        // q of this lane's row r (and r + 8): the columns that meet its K columns
        uint32_t qf[NT][D / 16][2];
        int lim[NT][2];     // keys seen by rows 2c and 2c + 1 of each 8
        float back[NT][2];  // FP8: score scale of those rows
        float v_most[NT][2];   // FP8: a power of two no value scale so far that those rows see is above; o is that much too small
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int x = row0 + nt * 8 + r;
            const int token = (int)fast_div((uint32_t)x, a.group_div);
            const size_t at = ((size_t)(span.q0 + token) * a.q_heads + cur.head * a.group + (x - token * a.group)) * D;
            const typename T::storage* qr = static_cast<const typename T::storage*>(a.q) + at;
            float4 f[FP8 ? D / 16 : 1];
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < (FP8 ? D / 16 : 0); ++i) {
                // 16 columns (four steps) at 64 (i / 4) + 16 c
                f[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x < rows) f[i] = load_quad<T>(qr + 64 * (i >> 2) + 16 * c + 4 * (i & 3), 0);
                most = fmaxf(fmaxf(fmaxf(most, fabsf(f[i].x)), fmaxf(fabsf(f[i].y), fabsf(f[i].z))), fabsf(f[i].w));
            }
            if (FP8) {
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
                most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
                // the power of two below it, kept where it and its reciprocal are normal numbers
                const int exponent = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 100);
                const float down = __uint_as_float((uint32_t)(127 - exponent) << 23), up = __uint_as_float((uint32_t)(127 + exponent) << 23);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    qf[nt][i][0] = pack_f16x2(f[i].x * down, f[i].y * down);
                    qf[nt][i][1] = pack_f16x2(f[i].z * down, f[i].w * down);
                }
                // row r's factor to the lanes whose columns of S^T are rows 2c and 2c + 1
                back[nt][0] = a.scale_log2 * __shfl_sync(kFullMask, up, 8 * c);
                back[nt][1] = a.scale_log2 * __shfl_sync(kFullMask, up, 8 * c + 4);
            } else {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {   // 8 columns (two steps) at 32 (i / 2) + 8 c
                    const float4 t = x < rows ? load_quad<T>(qr + 32 * (i >> 1) + 8 * c + 4 * (i & 1), 0) : make_float4(0.f, 0.f, 0.f, 0.f);
                    qf[nt][i][0] = pack_bf16x2(t.x, t.y);
                    qf[nt][i][1] = pack_bf16x2(t.z, t.w);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int y = row0 + nt * 8 + 2 * c + e;
                lim[nt][e] = y < rows ? attn_visible(a, span, y + 1) : 0;
            }
        }
        float o[NT][VL][VCH / 2][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int b = 0; b < VL; ++b) {
#pragma unroll
                for (int i = 0; i < VCH / 2; ++i) o[nt][b][i][0] = o[nt][b][i][1] = o[nt][b][i][2] = o[nt][b][i][3] = 0.0f;
            }
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
            v_most[nt][0] = v_most[nt][1] = 0.0f;
        }
        for (int tile = begin; tile < end; ++tile) {
            const int t0 = tile * kAttnKeys + warp * 16;
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const uint32_t w0[4] = {kr[0][i].x, kr[0][i].y, kr[0][i].z, kr[0][i].w};
                const uint32_t w1[4] = {kr[1][i].x, kr[1][i].y, kr[1][i].z, kr[1][i].w};
                if (FP8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t f[4];
                        e4m3x4_to_f16(w0[e], f[0], f[2]);
                        e4m3x4_to_f16(w1[e], f[1], f[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<FP8>(s[nt], f, qf[nt][4 * i + e][0], qf[nt][4 * i + e][1]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t f[4] = {w0[2 * e], w1[2 * e], w0[2 * e + 1], w1[2 * e + 1]};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<FP8>(s[nt], f, qf[nt][2 * i + e][0], qf[nt][2 * i + e][1]);
                    }
                }
            }
            float ks0 = 0.0f, ks1 = 0.0f, vs0 = 0.0f, vs1 = 0.0f;
            if (FP8) {
                ks0 = ks[0], ks1 = ks[1], vs0 = vs[0], vs1 = vs[1];
                float most[NT][2];
                bool raised = false, apart = false;   // apart: rows that see a part of these keys
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        most[nt][e] = fmaxf(t0 + r < lim[nt][e] ? vs0 : 0.0f, t0 + r + 8 < lim[nt][e] ? vs1 : 0.0f);
                        raised |= most[nt][e] > v_most[nt][e];
                        apart |= t0 + 16 > lim[nt][e] && lim[nt][e] > 0;
                    }
                }
                if (__any_sync(kFullMask, raised)) {
                    const bool one = !__any_sync(kFullMask, apart);   // one maximum for all rows, or one for each
                    float all = fmaxf(fmaxf(vs0, vs1), 0.0f);
                    if (one) all = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(all)));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float fix[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float now = all;
                            if (!one) {
                                now = most[nt][e];
#pragma unroll
                                for (int off = 4; off < 32; off <<= 1) now = fmaxf(now, __shfl_xor_sync(kFullMask, now, off));
                            }
                            // up to a power of two, kept where its reciprocal is a normal number too
                            now = __uint_as_float((__float_as_uint(fmaxf(now, 1e-37f)) + 0x007fffffu) & 0x7f800000u);
                            now = fmaxf(fminf(now, 0x1p126f), v_most[nt][e]);
                            fix[e] = v_most[nt][e] * __uint_as_float(0x7f000000u - __float_as_uint(now));   // 0 at first
                            v_most[nt][e] = now;
                        }
#pragma unroll
                        for (int b = 0; b < VL; ++b) {
#pragma unroll
                            for (int i = 0; i < VCH / 2; ++i) {
                                o[nt][b][i][0] *= fix[0], o[nt][b][i][1] *= fix[1];
                                o[nt][b][i][2] *= fix[0], o[nt][b][i][3] *= fix[1];
                            }
                        }
                    }
                }
            }
            const bool more = tile + 1 < end;
            if (more) load_k(row16);
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float k0 = FP8 ? ks0 * back[nt][e] : a.scale_log2, k1 = FP8 ? ks1 * back[nt][e] : a.scale_log2;
                    s[nt][e] = t0 + r < lim[nt][e] ? s[nt][e] * k0 : -INFINITY;
                    s[nt][2 + e] = t0 + r + 8 < lim[nt][e] ? s[nt][2 + e] * k1 : -INFINITY;
                    top[e] = fmaxf(s[nt][e], s[nt][2 + e]);
                }
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(kFullMask, top[0], off));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(kFullMask, top[1], off));
                }
                if (__any_sync(kFullMask, top[0] > m[nt][0] || top[1] > m[nt][1])) {
                    float fix[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float now = fmaxf(m[nt][e], top[e]);
                        fix[e] = now == m[nt][e] ? 1.0f : fast_exp2(m[nt][e] - now);
                        m[nt][e] = now;
                        l[nt][e] *= fix[e];
                    }
#pragma unroll
                    for (int b = 0; b < VL; ++b) {
#pragma unroll
                        for (int i = 0; i < VCH / 2; ++i) {
                            o[nt][b][i][0] *= fix[0], o[nt][b][i][1] *= fix[1];
                            o[nt][b][i][2] *= fix[0], o[nt][b][i][3] *= fix[1];
                        }
                    }
                }
                float p[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float ref = m[nt][e] == -INFINITY ? 0.0f : m[nt][e];   // nothing seen yet: weights of 0
                    p[e] = fast_exp2(s[nt][e] - ref);
                    p[2 + e] = fast_exp2(s[nt][2 + e] - ref);
                    l[nt][e] += p[e] + p[2 + e];
                }
                // weights rounded to bf16 or f16 for the product (the sum above keeps them in f32); hidden keys stay exactly 0,
                // whatever their scale
                if (FP8) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float inv = __uint_as_float(0x7f000000u - __float_as_uint(v_most[nt][e]));   // 1 / v_most, exactly
                        p[e] = t0 + r < lim[nt][e] ? p[e] * (vs0 * inv) : 0.0f;
                        p[2 + e] = t0 + r + 8 < lim[nt][e] ? p[2 + e] * (vs1 * inv) : 0.0f;
                    }
                }
                pf[nt][0] = transpose8x8(FP8 ? pack_f16x2(p[0], p[1]) : pack_bf16x2(p[0], p[1]));
                pf[nt][1] = transpose8x8(FP8 ? pack_f16x2(p[2], p[3]) : pack_bf16x2(p[2], p[3]));
            }
#pragma unroll
            for (int b = 0; b < VL; ++b) {
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    if (FP8) {   // a word is 4 dims: pair keys (0, 1) and (2, 3) dim by dim, then widen
                        uint32_t f[2][4];
                        e4m3x4_to_f16(__byte_perm(vr[0][b][w], vr[1][b][w], 0x5140), f[0][0], f[0][1]);
                        e4m3x4_to_f16(__byte_perm(vr[2][b][w], vr[3][b][w], 0x5140), f[0][2], f[0][3]);
                        e4m3x4_to_f16(__byte_perm(vr[0][b][w], vr[1][b][w], 0x7362), f[1][0], f[1][1]);
                        e4m3x4_to_f16(__byte_perm(vr[2][b][w], vr[3][b][w], 0x7362), f[1][2], f[1][3]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_16816<FP8>(o[nt][b][2 * w + h], f[h], pf[nt][0], pf[nt][1]);
                        }
                    } else {     // a word is 2 dims
                        const uint32_t f[4] = {__byte_perm(vr[0][b][w], vr[1][b][w], 0x5410), __byte_perm(vr[0][b][w], vr[1][b][w], 0x7632),
                                               __byte_perm(vr[2][b][w], vr[3][b][w], 0x5410), __byte_perm(vr[2][b][w], vr[3][b][w], 0x7632)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<FP8>(o[nt][b][w], f, pf[nt][0], pf[nt][1]);
                    }
                }
            }
            if (more) {
                load_v(row16);
                row16 = lookup(tile + 2);
            }
        }
        // this warp's statistics and outputs, then the join of the eight warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(kFullMask, l[nt][e], off);
                const int x = nt * 8 + 2 * c + e;
                if (r == 0) {
                    s_m[warp * R + x] = m[nt][e];
                    s_l[warp * R + x] = l[nt][e];
                }
                float* dst = s_o + (warp * R + x) * (D + PAD) + r * VCH;
#pragma unroll
                for (int b = 0; b < VL; ++b) {
#pragma unroll
                    for (int i = 0; i < VCH / 2; ++i) {
                        const float by = FP8 ? v_most[nt][e] : 1.0f;
                        *reinterpret_cast<float2*>(dst + 8 * VCH * b + 2 * i) = make_float2(o[nt][b][i][e] * by, o[nt][b][i][2 + e] * by);
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = begin == 0 && end == cur.keys;
        const int slot = begin == 0 ? 1 : 0;
        float* part = attn_slot(a, blockIdx.x, slot, R, D);
        if (!whole && begin == 0 && threadIdx.x == 0) a.desc[blockIdx.x] = attn_describe<OV>(a, cur);
        for (int i = threadIdx.x; i < R * (D / 4); i += kAttnThreads) {
            const int x = i / (D / 4), col = (i % (D / 4)) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w * R + x]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = fast_exp2(s_m[w * R + x] - ref);
                const float4 t = *reinterpret_cast<const float4*>(s_o + (w * R + x) * (D + PAD) + col);
                sum = fmaf(f, s_l[w * R + x], sum);
                acc.x = fmaf(f, t.x, acc.x), acc.y = fmaf(f, t.y, acc.y), acc.z = fmaf(f, t.z, acc.z), acc.w = fmaf(f, t.w, acc.w);
            }
            if (whole) {
                if (row0 + x < rows) {
                    const int token = (int)fast_div((uint32_t)(row0 + x), a.group_div);
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    typename T::storage* dst = static_cast<typename T::storage*>(a.out) +
                        ((size_t)(span.q0 + token) * a.q_heads + cur.head * a.group + (row0 + x - token * a.group)) * D + col;
                    store_quad<T>(dst, 0, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
                }
            } else {
                if (col == 0) {
                    part[x] = top;
                    part[R + x] = sum;
                }
                *reinterpret_cast<float4*>(part + 2 * R + (size_t)x * D + col) = acc;
            }
        }
        __syncthreads();   // s_o is reused by the next segment
    }
}

// ---------------------------------------------------------------------------------------------
// Joins the partials of the row tiles that several CTAs shared: slot 1 of the CTA that began one, slot 0 of the CTAs after
// it. blockIdx.x takes a run of CTAs as possible beginnings, 32 at a time. One pass with a running maximum, the statistics
// and outputs of several partials requested together: the time is a chain of memory latencies.
// attn_combine_kernel (partials of attn_rows_kernel): WARPS = 8, few row tiles with many partials: a block per row and 64
// columns, warp w takes every eighth partial, joined in shared memory in a fixed order; WARPS = 1: a warp per row.
// attn_combine_rows_kernel (of attn_chunk_kernel): four rows at a time, of a warp (WARPS = 1) or a block (8), likewise.
// ---------------------------------------------------------------------------------------------
// The next CTA from `from` on, before `to`, that begins a row tile others go on with; `to` if there is none.
__device__ __forceinline__ int attn_next_first(const AttnArgs& a, int from, int to) {
    for (; from < to; from += 32) {
        const int at = from + (int)(threadIdx.x & 31);
        const unsigned begins = __ballot_sync(kFullMask, at < to && a.desc[at].parts > 0);
        if (begins) return from + __ffs(begins) - 1;
    }
    return to;
}
template <typename T>
__device__ __forceinline__ typename T::storage* attn_out_row(const AttnArgs& a, const AttnDesc& d, int row, int head_dim) {
    const int token = (int)fast_div((uint32_t)row, a.group_div);
    return static_cast<typename T::storage*>(a.out) +
           ((size_t)(d.q0 + token) * a.q_heads + d.head * a.group + (row - token * a.group)) * head_dim;
}

template <typename T, int D, int R, int WARPS>
__global__ void __launch_bounds__(256)
attn_combine_kernel(AttnArgs a, int ctas) {
    constexpr int COLS = WARPS == 1 ? D : 64, V = COLS / 32, AHEAD = 8 / (V / 2 > 2 ? 2 : 1);
    __shared__ float s_acc[WARPS == 1 ? 1 : 8][COLS + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = WARPS == 1 ? 0 : warp;
    const int x = WARPS == 1 ? blockIdx.y * 8 + warp : blockIdx.y, col = blockIdx.z * COLS + lane * V;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int from = (int)((long long)blockIdx.x * ctas / gridDim.x), to = (int)((long long)(blockIdx.x + 1) * ctas / gridDim.x);
    for (int first = attn_next_first(a, from, to); first < to; first = attn_next_first(a, first + 1, to)) {
        const AttnDesc d = a.desc[first];
        const int row = d.tile * R + x;
        if (row >= d.rows) continue;   // (the same for the whole block, or a warp of its own)
        float top = -INFINITY, sum = 0.0f, acc[V];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        for (int i0 = sub; i0 < d.parts; i0 += WARPS * AHEAD) {
            float m[AHEAD], l[AHEAD];
            float2 o[AHEAD][V / 2];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j * WARPS;
                if (i < d.parts) {
                    const float* p = attn_slot(a, first + i, i == 0 ? 1 : 0, R, D);
                    m[j] = p[x], l[j] = p[R + x];
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) o[j][e] = reinterpret_cast<const float2*>(p + 2 * R + (size_t)x * D + col)[e];
                }
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) now = fmaxf(now, i0 + j * WARPS < d.parts ? m[j] : -INFINITY);
            const float ref = now == -INFINITY ? 0.0f : now, g = fast_exp2(top - ref);
            top = now;
            sum *= g;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] *= g;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (i0 + j * WARPS < d.parts) {
                    const float f = fast_exp2(m[j] - ref);
                    sum = fmaf(f, l[j], sum);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        acc[2 * e] = fmaf(f, o[j][e].x, acc[2 * e]);
                        acc[2 * e + 1] = fmaf(f, o[j][e].y, acc[2 * e + 1]);
                    }
                }
            }
        }
        float2 out[V / 2];
        if (WARPS == 1) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) out[e] = make_float2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        } else {
            __syncthreads();   // the last row tile's join is over
#pragma unroll
            for (int e = 0; e < V; ++e) s_acc[warp][lane * V + e] = acc[e];
            if (lane == 0) s_acc[warp][COLS] = sum, s_acc[warp][COLS + 1] = top;
            __syncthreads();
            float most = -INFINITY, total = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) most = fmaxf(most, s_acc[w][COLS + 1]);
            if (most == -INFINITY) most = 0.0f;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) out[e] = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = fast_exp2(s_acc[w][COLS + 1] - most);
                total = fmaf(f, s_acc[w][COLS], total);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    out[e].x = fmaf(f, s_acc[w][lane * V + 2 * e], out[e].x);
                    out[e].y = fmaf(f, s_acc[w][lane * V + 2 * e + 1], out[e].y);
                }
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) out[e] = make_float2(out[e].x * inv, out[e].y * inv);
        }
        if (sub == 0) {
            typename T::storage* dst = attn_out_row<T>(a, d, row, D) + col;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                if (T::kBytes == 2) reinterpret_cast<uint32_t*>(dst)[e] = pack_bf16x2(out[e].x, out[e].y);
                else reinterpret_cast<float2*>(dst)[e] = out[e];
            }
        }
    }
}

template <typename T, int D, int R, int WARPS>
__global__ void __launch_bounds__(256)
attn_combine_rows_kernel(AttnArgs a, int ctas) {
    constexpr int Q = D / 32;   // column quads of a lane: lane / 4, lane / 4 + 8, ... of row lane % 4 of the four
    __shared__ float4 s_acc[WARPS == 1 ? 1 : 8][Q][32];
    __shared__ float s_top[WARPS == 1 ? 1 : 8][4], s_sum[WARPS == 1 ? 1 : 8][4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = WARPS == 1 ? 0 : warp;
    const int x0 = WARPS == 1 ? (blockIdx.y * 8 + warp) * 4 : blockIdx.y * 4, x = x0 + (lane & 3);
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int from = (int)((long long)blockIdx.x * ctas / gridDim.x), to = (int)((long long)(blockIdx.x + 1) * ctas / gridDim.x);
    for (int first = attn_next_first(a, from, to); first < to; first = attn_next_first(a, first + 1, to)) {
        const AttnDesc d = a.desc[first];
        if (d.tile * R + x0 >= d.rows) continue;   // (the same for the whole block, or a warp of its own)
        float top = -INFINITY, sum = 0.0f;
        float4 acc[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float m, float l, const float4* o) {
            const float now = fmaxf(top, m), ref = now == -INFINITY ? 0.0f : now;
            const float f = fast_exp2(m - ref), g = fast_exp2(top - ref);
            top = now;
            sum = fmaf(f, l, sum * g);
#pragma unroll
            for (int e = 0; e < Q; ++e) {
                acc[e].x = fmaf(f, o[e].x, acc[e].x * g), acc[e].y = fmaf(f, o[e].y, acc[e].y * g);
                acc[e].z = fmaf(f, o[e].z, acc[e].z * g), acc[e].w = fmaf(f, o[e].w, acc[e].w * g);
            }
        };
#pragma unroll 2
        for (int i = sub; i < d.parts; i += WARPS) {
            const float* p = attn_slot(a, first + i, i == 0 ? 1 : 0, R, D);
            const float4* src = reinterpret_cast<const float4*>(p + 2 * R) + (lane >> 2) * R + x;
            float4 o[Q];
            const float m = p[x], l = p[R + x];
#pragma unroll
            for (int e = 0; e < Q; ++e) o[e] = src[8 * e * R];
            add(m, l, o);
        }
        if (WARPS > 1) {
            __syncthreads();   // the last row tile's join is over
#pragma unroll
            for (int e = 0; e < Q; ++e) s_acc[warp][e][lane] = acc[e];
            if (lane < 4) s_top[warp][lane] = top, s_sum[warp][lane] = sum;
            __syncthreads();
            if (warp > 0) continue;
#pragma unroll 1
            for (int w = 1; w < WARPS; ++w) {
                float4 o[Q];
#pragma unroll
                for (int e = 0; e < Q; ++e) o[e] = s_acc[w][e][lane];
                add(s_top[w][lane & 3], s_sum[w][lane & 3], o);
            }
        }
        if (d.tile * R + x < d.rows) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            typename T::storage* dst = attn_out_row<T>(a, d, d.tile * R + x, D);
#pragma unroll
            for (int e = 0; e < Q; ++e) {
                store_quad<T>(dst, (lane >> 2) + 8 * e, make_float4(acc[e].x * inv, acc[e].y * inv, acc[e].z * inv, acc[e].w * inv));
            }
        }
    }
}

}  // namespace clef
