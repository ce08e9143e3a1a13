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
    int4* desc;                 // workspace: two slots per CTA, {sequence, head, row tile, state}
    float* part;                // workspace: per slot R maxima, R sums, R x head_dim outputs
};

// Slot states. Slot 0 of a CTA holds the end (or the middle) of a row tile begun by an earlier CTA, slot 1 the
// beginning of one that a later CTA ends.
enum AttnSlot { kAttnNone = 0, kAttnFirst = 1, kAttnMiddle = 2, kAttnLast = 3 };

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
// Units of row tile `tile`: its key tiles, at least one (a row that sees nothing still has to be written).
template <int R>
__device__ __forceinline__ int attn_tile_units(const AttnArgs& a, const AttnSeq& q, int tile) {
    const int rows = min((tile + 1) * R, q.n * a.group);
    return max(1, (attn_visible(a, q, rows) + kAttnKeys - 1) / kAttnKeys);
}

// sum over i < n of floor((step i + first) / m), all non-negative, m > 0: reduce step and first modulo m, then count
// the lattice points under the line by columns of the exchanged axes (Euclid's algorithm on (step, m)).
__device__ inline long long floor_sum(long long n, long long m, long long step, long long first) {
    long long total = 0;
    while (n > 0) {
        if (step >= m) {
            total += (n * (n - 1) / 2) * (step / m);
            step %= m;
        }
        if (first >= m) {
            total += n * (first / m);
            first %= m;
        }
        const long long top = step * n + first;
        if (top < m) break;
        n = top / m;
        first = top % m;
        const long long t = m;
        m = step;
        step = t;
    }
    return total;
}

// Units of all row tiles of one (sequence, kv head). A full tile i sees floor((A + i R) / (group keys)) + 1 key tiles
// with A = (kv - n) group + R - 1 (1 where that is below 1), the last tile ceil(kv / keys).
template <int R>
__device__ inline long long attn_seq_units(const AttnArgs& a, const AttnSeq& q) {
    const int tiles = (q.n * a.group + R - 1) / R;
    if (tiles == 0) return 0;
    const long long full = tiles - 1, m = (long long)a.group * kAttnKeys;
    const long long A = (long long)(q.kv - q.n) * a.group + R - 1;
    const long long skip = A >= 0 ? 0 : min(full, (-A + R - 1) / R);
    return full + floor_sum(full - skip, m, R, A + skip * R) + max(1, (q.kv + kAttnKeys - 1) / kAttnKeys);
}

// A CTA's place in the list of units: (sequence, kv head, row tile, key tile), and how many units are left to it.
struct AttnCursor {
    int seq, head, tile, key_tile, units;   // `units` of the row tile
    AttnSeq span;
    long long left;
};

// The cursor of CTA `cta` of `ctas`: unit floor(cta * total / ctas) on. One warp, all lanes; every lane has the result.
template <int R>
__device__ inline AttnCursor attn_locate(const AttnArgs& a, int cta, int ctas) {
    const int lane = threadIdx.x & 31;
    long long total = 0;
    for (int s = lane; s < a.n_seqs; s += 32) total += a.kv_heads * attn_seq_units<R>(a, attn_seq(a, s));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(kFullMask, total, off);
    AttnCursor c;
    if (total < ctas) ctas = (int)total;   // the CTAs that work are the first ones, with a unit each at least
    long long at = cta < ctas ? cta * total / ctas : 0;
    c.left = cta < ctas ? (cta + 1) * total / ctas - at : 0;
    c.seq = c.head = c.tile = c.key_tile = c.units = 0;
    c.span = AttnSeq{0, 0, 0};
    if (c.left == 0) return c;
    long long per_head = 0;
    for (int base = 0; base < a.n_seqs; base += 32) {   // the sequence: scans of 32
        const int s = base + lane;
        const long long mine = s < a.n_seqs ? attn_seq_units<R>(a, attn_seq(a, s)) : 0;
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
    c.head = (int)(at / per_head);
    at -= c.head * per_head;
    const int tiles = (c.span.n * a.group + R - 1) / R;
    for (int base = 0; base < tiles; base += 32) {      // the row tile: scans of 32
        const int mine = base + lane < tiles ? attn_tile_units<R>(a, c.span, base + lane) : 0;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(kFullMask, upto, off);
            if (lane >= off) upto += t;
        }
        const unsigned past = __ballot_sync(kFullMask, (long long)upto > at);
        if (past) {
            const int hit = __ffs(past) - 1;
            c.tile = base + hit;
            c.units = __shfl_sync(kFullMask, mine, hit);
            c.key_tile = (int)at - (__shfl_sync(kFullMask, upto, hit) - c.units);
            break;
        }
        at -= __shfl_sync(kFullMask, upto, 31);
    }
    return c;
}

// On to the next row tile (called with units left: there is one).
template <int R>
__device__ __forceinline__ void attn_advance(const AttnArgs& a, AttnCursor& c) {
    c.key_tile = 0;
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
    c.units = attn_tile_units<R>(a, c.span, c.tile);
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
    constexpr int R = 8 * NT;
    constexpr int WARPS = kAttnThreads / 32;
    constexpr int KSTEP = FP8 ? 64 : 32;             // head dims of one 16-byte load by the four lanes of a key
    constexpr int KL = D / KSTEP;                    // such loads per key
    constexpr int VCH = FP8 && D >= 128 ? 16 : 8;    // head dims of V a lane takes at once
    constexpr int VL = D / (8 * VCH);                // such pieces per key
    constexpr int VW = VCH * (FP8 ? 1 : 2) / 4;      // words of a piece
    constexpr int PAD = 4;
    using CacheT = typename std::conditional<FP8, uint8_t, uint16_t>::type;
    extern __shared__ float s_o[];                   // [WARPS][R][D + PAD], then [WARPS][R] maxima and sums
    float* s_m = s_o + WARPS * R * (D + PAD);
    float* s_l = s_m + WARPS * R;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, c = lane & 3;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const CacheT* kc = static_cast<const CacheT*>(a.k);
    const CacheT* vc = static_cast<const CacheT*>(a.v);
    AttnCursor cur = attn_locate<R>(a, blockIdx.x, gridDim.x);
    int4* desc = a.desc + 2 * blockIdx.x;
    if (threadIdx.x < 2) desc[threadIdx.x].w = kAttnNone;
    while (cur.left > 0) {
        const int begin = cur.key_tile, end = (int)min((long long)cur.units, begin + cur.left);
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
        const bool whole = begin == 0 && end == cur.units;
        const int slot = begin == 0 ? 1 : 0;
        float* part = attn_slot(a, blockIdx.x, slot, R, D);
        if (!whole && threadIdx.x == 0) {
            desc[slot] = make_int4(cur.seq, cur.head, cur.tile, begin == 0 ? kAttnFirst : (end == cur.units ? kAttnLast : kAttnMiddle));
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
        cur.left -= end - begin;
        if (cur.left > 0) attn_advance<R>(a, cur);
    }
}

// ---------------------------------------------------------------------------------------------
// Joins the partials of the row tiles that several CTAs shared: a tile is begun in slot 1 of one CTA and continued in
// slot 0 of the CTAs after it, up to the one marked last. blockIdx.x takes a run of CTAs as possible beginnings. WPR
// warps work on a row, one after the other every WPR-th partial, and are joined in shared memory in a fixed order: a
// whole block per row where few rows have many partials (attn_rows_kernel), a warp where many rows have few.
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int R, int WPR>
__global__ void __launch_bounds__(256)
attn_combine_kernel(AttnArgs a, int ctas) {
    constexpr int ROWS = 8 / WPR;   // of a block
    __shared__ float s_acc[8][D + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int from = (int)((long long)blockIdx.x * ctas / gridDim.x), to = (int)((long long)(blockIdx.x + 1) * ctas / gridDim.x);
    for (int first = from; first < to; ++first) {
        const int4 d = a.desc[2 * first + 1];
        if (d.w != kAttnFirst) continue;
        const AttnSeq span = attn_seq(a, d.x);
        const int x = blockIdx.y * ROWS + warp / WPR;
        if (d.z * R + (int)blockIdx.y * ROWS >= span.n * a.group) continue;   // (the same for the whole block)
        int last = first + 1;
        while (last < ctas - 1 && a.desc[2 * last].w != kAttnLast) ++last;
        const int parts = last - first + 1;
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
        for (int i = sub; i < parts; i += WPR) {
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
        for (int i = threadIdx.x; i < ROWS * (D / 4); i += 256) {
            const int r = i / (D / 4), col = (i % (D / 4)) * 4;
            const int mine = d.z * R + blockIdx.y * ROWS + r;
            if (mine >= span.n * a.group) break;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) {
                const float* p = s_acc[r * WPR + w];
                v.x += p[col], v.y += p[col + 1], v.z += p[col + 2], v.w += p[col + 3];
                total += p[D];
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            const int token = (int)fast_div((uint32_t)mine, a.group_div);
            typename T::storage* dst = static_cast<typename T::storage*>(a.out) +
                ((size_t)(span.q0 + token) * a.q_heads + d.y * a.group + (mine - token * a.group)) * D + col;
            store_quad<T>(dst, 0, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        __syncthreads();
    }
}

}  // namespace clef
