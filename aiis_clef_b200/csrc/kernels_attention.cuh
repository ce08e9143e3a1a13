// Attention of new tokens over a paged KV cache: single generated tokens, chunks of a prompt, and batches that mix
// the two. For query row i of a sequence with n new tokens and kv cached ones (the new ones included, they are the
// last n), the keys it sees are 0 .. kv - n + i:
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp2(scale log2(e) q_i . k_j - m_i),   m_i = running maximum
// Scores, maxima, sums and outputs are f32; q, p and the cached values enter the products as bf16.
//
// The q heads that share a kv head are rows of ONE product: row x of a (sequence, kv head) is new token x / group,
// head x % group. Rows are cut into row tiles of R, keys into tiles of kAttnKeys, and the (row tile, key tile) units
// of the whole batch are one flat list that every CTA takes an equal, contiguous share of: a lone long sequence
// fills the machine as well as an uneven batch does, and the grid depends on shapes alone. A row tile whose keys
// were cut over several CTAs leaves (m, l, o) partials in the workspace, and attn_combine_kernel joins them in CTA
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
    struct AttnDesc* desc;      // workspace: what is in the two slots of each CTA
    float* part;                // workspace: per slot R maxima, R sums, R x head_dim outputs (attn_chunk_kernel: [head_dim / 4][R][4])
};

// Slot states. Slot 0 of a CTA holds the end (or the middle) of a row tile begun by an earlier CTA, slot 1 the
// beginning of one that a later CTA ends.
enum AttnSlot { kAttnNone = 0, kAttnFirst = 1, kAttnMiddle = 2, kAttnLast = 3 };
struct AttnDesc {
    int state, tile, head, q0, rows;   // rows: of the sequence and kv head
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
// which is `group` times the keys its last row sees, and OV key tiles' worth for its beginning and end.
template <int R, int OV>
__device__ __forceinline__ long long attn_tile_cost(const AttnArgs& a, const AttnSeq& q, int tile) {
    return (long long)OV * a.group * kAttnKeys + max(0, (q.kv - q.n) * a.group + (tile + 1) * R);
}
// Cost of all row tiles of one (sequence, kv head).
template <int R, int OV>
__device__ __forceinline__ long long attn_seq_cost(const AttnArgs& a, const AttnSeq& q) {
    const int tiles = (q.n * a.group + R - 1) / R;
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
    long long cost, at, left;
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
    const long long share = max((total + ctas - 1) / ctas, (long long)a.group * kAttnKeys);
    long long at = cta * share;
    c.left = min(share, total - at);
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
__device__ __forceinline__ void attn_segment(const AttnArgs& a, const AttnCursor& c, int& begin, int& end) {
    const int unit = a.group * kAttnKeys;
    auto before = [&](long long x) {
        const int y = (int)(x - (long long)OV * unit) + unit / 2;
        return y <= 0 ? 0 : min(c.keys, y / unit);
    };
    begin = before(c.at);
    end = c.at + c.left >= c.cost ? c.keys : before(c.at + c.left);
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

// Four E4M3 codes -> two bf16 pairs, exactly: sign, exponent and mantissa bits moved into a bf16 pattern read 2^120 too
// small (the biases are 7 and 127), and one multiplication by 2^120, which also normalises the subnormal codes.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);
    const uint32_t x = (a & 0x80008000u) | ((a >> 4) & 0x07f007f0u), y = (b & 0x80008000u) | ((b >> 4) & 0x07f007f0u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(0x7b807b80u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(0x7b807b80u));
}

__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
    AttnDesc* desc = a.desc + 2 * blockIdx.x;
    if (threadIdx.x < 2) desc[threadIdx.x].state = kAttnNone;
    __syncthreads();
    AttnCursor cur = s_cursor;
    for (; cur.left > 0; attn_advance<R, OV>(a, cur)) {
        int begin, end;
        attn_segment<OV>(a, cur, begin, end);
        if (begin == end) continue;
        const AttnSeq span = cur.span;
        const int row0 = cur.tile * R, rows = span.n * a.group;
        // q of this lane's row r (and r + 8): the columns that meet its K columns
        uint32_t qf[NT][D / 16][2];
        int lim[NT][2];   // keys seen by rows 2c and 2c + 1 of each 8
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int x = row0 + nt * 8 + r;
            const int token = (int)fast_div((uint32_t)x, a.group_div);
            const size_t at = ((size_t)(span.q0 + token) * a.q_heads + cur.head * a.group + (x - token * a.group)) * D;
            const typename T::storage* qr = static_cast<const typename T::storage*>(a.q) + at;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                // bf16: 8 columns (two steps) at 32 (i / 2) + 8 c; FP8: 16 columns (four steps) at 64 (i / 4) + 16 c
                const int col = FP8 ? 64 * (i >> 2) + 16 * c + 4 * (i & 3) : 32 * (i >> 1) + 8 * c + 4 * (i & 1);
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x < rows) f = load_quad<T>(qr + col, 0);
                qf[nt][i][0] = pack_bf16x2(f.x, f.y);
                qf[nt][i][1] = pack_bf16x2(f.z, f.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int y = row0 + nt * 8 + 2 * c + e;
                lim[nt][e] = y < rows ? attn_visible(a, span, y + 1) : 0;
            }
        }
        const int keys = attn_visible(a, span, min(row0 + R, rows));   // seen by any row of the tile
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
        }
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
        int row16 = lookup(begin);
        load_k(row16);
        load_v(row16);
        row16 = lookup(begin + 1);
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
                        e4m3x4_to_bf16(w0[e], f[0], f[2]);
                        e4m3x4_to_bf16(w1[e], f[1], f[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(s[nt], f, qf[nt][4 * i + e][0], qf[nt][4 * i + e][1]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t f[4] = {w0[2 * e], w1[2 * e], w0[2 * e + 1], w1[2 * e + 1]};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(s[nt], f, qf[nt][2 * i + e][0], qf[nt][2 * i + e][1]);
                    }
                }
            }
            const float ks0 = FP8 ? ks[0] * a.scale_log2 : a.scale_log2, ks1 = FP8 ? ks[1] * a.scale_log2 : a.scale_log2;
            const float vs0 = FP8 ? vs[0] : 1.0f, vs1 = FP8 ? vs[1] : 1.0f;
            const bool more = tile + 1 < end;
            if (more) load_k(row16);
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[nt][e] = t0 + r < lim[nt][e] ? s[nt][e] * ks0 : -INFINITY;
                    s[nt][2 + e] = t0 + r + 8 < lim[nt][e] ? s[nt][2 + e] * ks1 : -INFINITY;
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
                // weights rounded to bf16 for the product (the sum above keeps them in f32); masked keys stay exactly 0
                if (FP8) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        p[e] = p[e] == 0.0f ? 0.0f : p[e] * vs0;
                        p[2 + e] = p[2 + e] == 0.0f ? 0.0f : p[2 + e] * vs1;
                    }
                }
                pf[nt][0] = transpose8x8(pack_bf16x2(p[0], p[1]));
                pf[nt][1] = transpose8x8(pack_bf16x2(p[2], p[3]));
            }
#pragma unroll
            for (int b = 0; b < VL; ++b) {
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    if (FP8) {   // a word is 4 dims: pair keys (0, 1) and (2, 3) dim by dim, then widen
                        uint32_t f[2][4];
                        e4m3x4_to_bf16(__byte_perm(vr[0][b][w], vr[1][b][w], 0x5140), f[0][0], f[0][1]);
                        e4m3x4_to_bf16(__byte_perm(vr[2][b][w], vr[3][b][w], 0x5140), f[0][2], f[0][3]);
                        e4m3x4_to_bf16(__byte_perm(vr[0][b][w], vr[1][b][w], 0x7362), f[1][0], f[1][1]);
                        e4m3x4_to_bf16(__byte_perm(vr[2][b][w], vr[3][b][w], 0x7362), f[1][2], f[1][3]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_bf16(o[nt][b][2 * w + h], f[h], pf[nt][0], pf[nt][1]);
                        }
                    } else {     // a word is 2 dims
                        const uint32_t f[4] = {__byte_perm(vr[0][b][w], vr[1][b][w], 0x5410), __byte_perm(vr[0][b][w], vr[1][b][w], 0x7632),
                                               __byte_perm(vr[2][b][w], vr[3][b][w], 0x5410), __byte_perm(vr[2][b][w], vr[3][b][w], 0x7632)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(o[nt][b][w], f, pf[nt][0], pf[nt][1]);
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
                        *reinterpret_cast<float2*>(dst + 8 * VCH * b + 2 * i) = make_float2(o[nt][b][i][e], o[nt][b][i][2 + e]);
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = begin == 0 && end == cur.keys;
        const int slot = begin == 0 ? 1 : 0;
        float* part = attn_slot(a, blockIdx.x, slot, R, D);
        if (!whole && threadIdx.x == 0) {
            desc[slot] = AttnDesc{begin == 0 ? kAttnFirst : (end == cur.keys ? kAttnLast : kAttnMiddle), cur.tile, cur.head, span.q0, rows};
        }
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
// Joins the partials of the row tiles that several CTAs shared: a tile is begun in slot 1 of one CTA and continued in
// slot 0 of the CTAs after it, up to the one marked last. blockIdx.x takes a run of CTAs as possible beginnings.
// attn_combine_kernel: few rows with many partials (attn_rows_kernel), a block per row; the 8 warps take every eighth
// partial and are joined in shared memory in a fixed order.
// attn_combine_rows_kernel: many rows with few partials (attn_chunk_kernel), four rows per warp.
// ---------------------------------------------------------------------------------------------
// Partials of the row tile that CTA `first` begins; a warp looks at the 32 CTAs after it at a time.
__device__ __forceinline__ int attn_parts(const AttnArgs& a, int first, int ctas) {
    for (int from = first + 1;; from += 32) {
        const int at = from + (int)(threadIdx.x & 31);
        const unsigned ends = __ballot_sync(kFullMask, at >= ctas - 1 || a.desc[2 * at].state == kAttnLast);
        if (ends) return from + __ffs(ends) - first;
    }
}
template <typename T>
__device__ __forceinline__ typename T::storage* attn_out_row(const AttnArgs& a, const AttnDesc& d, int row, int head_dim) {
    const int token = (int)fast_div((uint32_t)row, a.group_div);
    return static_cast<typename T::storage*>(a.out) +
           ((size_t)(d.q0 + token) * a.q_heads + d.head * a.group + (row - token * a.group)) * head_dim;
}

template <typename T, int D, int R>
__global__ void __launch_bounds__(256)
attn_combine_kernel(AttnArgs a, int ctas) {
    constexpr int WARPS = 8;
    __shared__ float s_acc[WARPS][D + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int from = (int)((long long)blockIdx.x * ctas / gridDim.x), to = (int)((long long)(blockIdx.x + 1) * ctas / gridDim.x);
    for (int first = from; first < to; ++first) {
        const AttnDesc d = a.desc[2 * first + 1];
        const int x = blockIdx.y, row = d.tile * R + x;
        if (d.state != kAttnFirst || row >= d.rows) continue;
        const int parts = attn_parts(a, first, ctas);
        auto part_of = [&](int i) { return attn_slot(a, first + i, i == 0 ? 1 : 0, R, D); };
        float top = -INFINITY;
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, part_of(i)[x]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float acc[D / 32];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
#pragma unroll 4
        for (int i = warp; i < parts; i += WARPS) {
            const float* p = part_of(i);
            const float f = fast_exp2(p[x] - ref);
            sum = fmaf(f, p[R + x], sum);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(f, p[2 * R + (size_t)x * D + lane + 32 * e], acc[e]);
        }
#pragma unroll
        for (int e = 0; e < D / 32; ++e) s_acc[warp][lane + 32 * e] = acc[e];
        if (lane == 0) s_acc[warp][D] = sum;
        __syncthreads();
        if (threadIdx.x < D / 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float* p = s_acc[w] + 4 * threadIdx.x;
                v.x += p[0], v.y += p[1], v.z += p[2], v.w += p[3];
                total += s_acc[w][D];
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            store_quad<T>(attn_out_row<T>(a, d, row, D), threadIdx.x, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        __syncthreads();
    }
}

template <typename T, int D, int R>
__global__ void __launch_bounds__(256)
attn_combine_rows_kernel(AttnArgs a, int ctas) {
    constexpr int Q = D / 32;   // column quads of a lane: lane / 4, lane / 4 + 8, ... of row lane % 4 of the warp's four
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int from = (int)((long long)blockIdx.x * ctas / gridDim.x), to = (int)((long long)(blockIdx.x + 1) * ctas / gridDim.x);
    for (int first = from; first < to; ++first) {
        const AttnDesc d = a.desc[2 * first + 1];
        const int x0 = (blockIdx.y * 8 + warp) * 4, x = x0 + (lane & 3);
        if (d.state != kAttnFirst || d.tile * R + x0 >= d.rows) continue;
        const int parts = attn_parts(a, first, ctas);
        // one pass with a running maximum: the statistics and outputs of a partial are requested together
        float top = -INFINITY, sum = 0.0f;
        float4 acc[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int i = 0; i < parts; ++i) {
            const float* p = attn_slot(a, first + i, i == 0 ? 1 : 0, R, D);
            const float4* src = reinterpret_cast<const float4*>(p + 2 * R) + (lane >> 2) * R + x;
            float4 o[Q];
            const float m = p[x], l = p[R + x];
#pragma unroll
            for (int e = 0; e < Q; ++e) o[e] = src[8 * e * R];
            const float now = fmaxf(top, m), ref = now == -INFINITY ? 0.0f : now;
            const float f = fast_exp2(m - ref), g = fast_exp2(top - ref);
            top = now;
            sum = fmaf(f, l, sum * g);
#pragma unroll
            for (int e = 0; e < Q; ++e) {
                acc[e].x = fmaf(f, o[e].x, acc[e].x * g), acc[e].y = fmaf(f, o[e].y, acc[e].y * g);
                acc[e].z = fmaf(f, o[e].z, acc[e].z * g), acc[e].w = fmaf(f, o[e].w, acc[e].w * g);
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
