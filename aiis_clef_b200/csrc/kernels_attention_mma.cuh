// Attention of chunks of new tokens, bound by the products: tcgen05 with accumulators in tensor memory.
//
// A CTA has the SM to itself. A row tile is TILES x 128 query rows; per key tile of N keys and per 128 rows
//   S = Q K^T     [128 x N] f32, both operands K-major in shared memory (128-byte swizzle),
//   P = exp2(...) bf16, written over S in tensor memory, one thread per row,
//   O += P V      [128 x D] f32, P read from tensor memory, V [keys][dims] as it lies in the cache (MN-major).
// Warps are specialised: one warpgroup of softmax per 128 rows, one warpgroup (two for 256 dims of FP8) that gathers K and
// V rows from the pages into rings of K and of V tiles, one warp that issues the products. For head_dim 64 and 128 the
// products of one row block run under the softmax of the other; head_dim 256 has tensor memory for one row block only.
// Key tiles are 64 keys and S has two buffers per row block, so that the scores of the next step are there when the
// softmax comes to them.
// An FP8 cache is multiplied in f16: the 16 rows that a producer warp widens are brought under one power of two,
// code * (scale / 2^e) in f16 (2^-11 per value, next to the codes' own 2^-4), which the softmax multiplies back: 2^e of K
// with the score scale of those 16 keys, 2^e of V with the reference of their weights. (With scaled rows
// as bf16 the outputs' error was 0.0048 of their size, 0.0020 so.) In the last steps of a row tile, where the mask hides some
// keys from some row, what is hidden must not decide how finely the rest is held: rows whose scales lie further apart than
// 2^13 (K) or 2^4 (V) are multiplied as bare codes there, and the softmax takes their scales one by one, those of K with the
// scores, those of V, against the largest that its row sees, with the weights.
//
// Measured with the join (16 + 2 heads of 128, pages of 64), in 20 calls behind each other and in a long stream of calls, where
// the card holds a lower clock: 8,192 causal tokens 275 to 282 and 308 us = 1,000 and 893 TFLOP/s; 2,011 tokens after 30,757 in
// FP8 600 and 653 us = 872 and 802 TFLOP/s; head_dim 256, FP8, 2,048 tokens after 6,144: 375 us = 642 TFLOP/s in the former. What
// bounds it: the softmax's chain of latencies. When 8,192 tokens took 299 us a step of 64 keys took 2,150 clocks; its products
// filled the tensor pipe for about 1,280 of them (at 64 keys
// the scores' operands come out of shared memory at less than the pipe's rate) and its exponentials their units for
// 1,060, but a thread's way from scores to weights (barrier, load, maximum, fma, exp2, sum, pack, store) was some 1,800 clocks
// alone, and only two warps on each quarter of the SM share it out. The step compiled apart for steps that hide keys: 282 us
// from 295, for FP8 no change where contexts are long and 2 to 4 us more for prompts of 2,048 (35.7 from 31.7 us with 8 + 8 heads),
// where the larger kernel is fetched and bare codes are looked for. Not kept, prefill in us against 299: 128 keys a step with
// one S buffer 325 (the long FP8 case gained 6 %, FP8 prompts of 2,048 lost 13 %), the row blocks' exponentials in turns 297,
// weights against the last reference with the maximum beside them 305, one arrival per warp on the barriers 313,
// a quarter of the exponentials as polynomials 297.
//
// The output is rescaled only when a row's maximum has grown by more than 2^8 since the last time (weights then stay
// below 2^8, exact enough in f32 sums and bf16 weights alike), so the softmax rarely touches O.
//
// Every wait is bounded: after kWaitLimitNs it gives up, all later waits of the CTA return at once, and the rows the
// CTA owns come out as NaN.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "kernels_attention.cuh"

namespace clef {

constexpr unsigned long long kWaitLimitNs = 2000000000ull;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of `parity`; gives up after kWaitLimitNs and raises *gave_up, which ends every later wait.
__device__ __forceinline__ void mbar_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    if (mbar_try(bar, parity)) return;
    const unsigned long long from = global_ns();
    for (int i = 1; !mbar_try(bar, parity); ++i) {
        if (*gave_up) return;
        if ((i & 63) == 0 && global_ns() - from > kWaitLimitNs) {
            *gave_up = 1;
            return;
        }
    }
}

// The same for a whole warp, which goes on together (the tensor memory instructions want it converged).
__device__ __forceinline__ void mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    mbar_wait(bar, parity, gave_up);
    __syncwarp();
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Products and commits are issued by the one lane whose `leader` is set, as predicated instructions of a converged warp:
// their descriptors then stay in uniform registers. (Issued inside a branch that one thread takes, each product cost
// about 75 cycles to issue, more than most take to execute.)
__device__ __forceinline__ void tc_commit(uint64_t* bar, uint32_t leader) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(leader) : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(kFullMask, x, 0); }
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// D[128 x N] (tensor memory) (+)= A B^T; A from shared memory or from tensor memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t leader) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t leader) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
                 : "memory");
}
// 32 consecutive f32 columns of this thread's row.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                   "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
                   "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
                 "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
                 "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tc_ld8(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle. Low word: address / 16 and leading byte offset / 16 in the upper half;
// high word: stride byte offset / 16 (1,024: eight rows of 128 bytes), version, swizzle mode.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t leading) {
    return (addr >> 4) | ((leading >> 4) << 16);
}
__device__ __forceinline__ uint64_t smem_desc(uint32_t low, uint32_t bytes_on) {
    return ((uint64_t)((1024 >> 4) | (1u << 14) | (2u << 29)) << 32) | (low + (bytes_on >> 4));
}
// Instruction descriptor: f32 accumulators, f16 or bf16 operands, A K-major; B K-major or MN-major.
__host__ __device__ constexpr uint32_t mma_idesc(int n, bool b_mn_major, bool f16) {
    return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile of `rows` rows: 64 columns (128 bytes) side by side, the
// chunks of a row permuted by the row's low three bits (the hardware's 128-byte swizzle).
__device__ __forceinline__ uint32_t tile_offset(int row, int chunk, int rows) {
    return (uint32_t)((chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// Eight q values as they are loaded, as f32, and as operands: bf16, or f16 of the values times `by`.
template <typename T>
struct RawQ {
    uint4 w[T::kBytes / 2];
    __device__ __forceinline__ void load(const typename T::storage* p) {
#pragma unroll
        for (int i = 0; i < T::kBytes / 2; ++i) w[i] = ldg_stream_v4(reinterpret_cast<const uint8_t*>(p) + 16 * i);
    }
    __device__ __forceinline__ void floats(float* f) const {
        const uint4 a = w[0], b = w[T::kBytes / 2 - 1];
        if (T::kBytes == 2) {
            f[0] = bf16_lo(a.x), f[1] = bf16_hi(a.x), f[2] = bf16_lo(a.y), f[3] = bf16_hi(a.y);
            f[4] = bf16_lo(a.z), f[5] = bf16_hi(a.z), f[6] = bf16_lo(a.w), f[7] = bf16_hi(a.w);
        } else {
            f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z), f[3] = __uint_as_float(a.w);
            f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y), f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
        }
    }
    __device__ __forceinline__ uint4 bf16() const {
        if (T::kBytes == 2) return w[0];
        float f[8];
        floats(f);
        return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
    __device__ __forceinline__ uint4 f16(float by) const {
        float f[8];
        floats(f);
        return make_uint4(pack_f16x2(f[0] * by, f[1] * by), pack_f16x2(f[2] * by, f[3] * by), pack_f16x2(f[4] * by, f[5] * by),
                          pack_f16x2(f[6] * by, f[7] * by));
    }
};

template <int REGS, bool UP>
__device__ __forceinline__ void set_registers() {
    if (UP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// The power of two that a scale lies below (NaN and infinity: none, -100), kept where it and its reciprocal are normal numbers.
__device__ __forceinline__ int scale_exponent(float scale) {
    return scale < INFINITY ? min(max((int)(__float_as_uint(scale) >> 23) - 126, -100), 126) : -100;
}
constexpr int kBareCodes = 0x1000;   // in place of the exponent of 16 keys that are multiplied as bare codes

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int D, bool FP8>
struct ChunkShape {
    static constexpr int TILES = D == 256 ? 1 : 2;        // row blocks of 128
    static constexpr int R = 128 * TILES;                 // rows of a row tile
    static constexpr int N = 64;                          // keys of a step
    static constexpr int SBUF = 2;                        // S buffers per row block
    static constexpr int SLOTS = D == 256 ? 2 : 4;        // buffers of K tiles, and as many of V tiles
    static constexpr int OV = 2;                          // a row tile's beginning and end cost about two units
    static constexpr int PRODUCERS = D == 256 && FP8 ? 2 : 1;   // warpgroups of them; two share the columns
    static constexpr int THREADS = 128 * (TILES + PRODUCERS + 1);   // softmax, producers, products (one warp of the last)
    // Registers: 512 threads start with 128 each; the softmax, which keeps a row of S, takes what the others leave.
    static constexpr bool SPLIT = THREADS == 512;
    static constexpr int SOFTMAX_REGS = 184, PRODUCER_REGS = PRODUCERS == 2 ? 104 : 80, MMA_REGS = 64;
    static_assert(!SPLIT || TILES * SOFTMAX_REGS + PRODUCERS * PRODUCER_REGS + MMA_REGS <= 512, "more than the block started with");
    static constexpr int Q_BYTES = 128 * D * 2;
    static constexpr int KV_BYTES = N * D * 2;
    static constexpr int S_COL = 0;                       // tensor memory columns: S buffers, then O
    static constexpr int O_COL = TILES * SBUF * N;
    // FP8: steps whose scales and exponents are kept. Those of step n are asked for when its K tile has a slot, so when the
    // scores of step n - SLOTS are done, which come SBUF steps after weights: no softmax is behind step n - SLOTS - 1 then.
    static constexpr int SCALE_STEPS = 2 * SLOTS;
    static constexpr int SMEM = 1024 + TILES * Q_BYTES + 2 * SLOTS * KV_BYTES + (FP8 ? SCALE_STEPS * (2 * N * PRODUCERS + 8) * 4 + TILES * 512 : 0);
};

// Steps of a segment [begin, end) of key tiles, the same for every role: whole tiles of N keys, none that lies past the
// last key a row of the tile sees, one at least.
template <int D, bool FP8>
__device__ __forceinline__ void chunk_steps(const AttnArgs& a, const AttnCursor& c, int begin, int end, int& keys, int& from, int& to) {
    using Sh = ChunkShape<D, FP8>;
    constexpr int PER = kAttnKeys / Sh::N;
    keys = attn_visible(a, c.span, min((c.tile + 1) * Sh::R, c.span.n * a.group));
    from = begin * PER;
    to = max(from + 1, min(end * PER, (keys + Sh::N - 1) / Sh::N));
}

// The first step of a row tile in which some row does not see every key.
template <int N>
__device__ __forceinline__ int chunk_hides_from(const AttnArgs& a, const AttnSeq& span, int row0) {
    return attn_visible(a, span, row0 + 1) / N;
}

// The 128 threads of row block t.
__device__ __forceinline__ void block_barrier(int t) {
    if (t == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
    else asm volatile("bar.sync 2, 128;" ::: "memory");
}

template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(ChunkShape<D, FP8>::THREADS, 1)
attn_chunk_kernel(AttnArgs a) {
    using Sh = ChunkShape<D, FP8>;
    constexpr int TILES = Sh::TILES, R = Sh::R, N = Sh::N, SBUF = Sh::SBUF, SLOTS = Sh::SLOTS, OV = Sh::OV;
    extern __shared__ uint8_t s_raw[];
    __shared__ uint64_t full[2 * SLOTS], empty[2 * SLOTS], q_ready[TILES], s_ready[TILES * SBUF], p_ready[TILES * SBUF], pv_done[TILES * 2], drained;
    __shared__ uint64_t exponents_ready[Sh::SCALE_STEPS];   // FP8
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ AttnCursor s_cursor;
    uint8_t* s_base = s_raw + ((1024 - (smem_addr(s_raw) & 1023)) & 1023);
    uint8_t* s_q = s_base;
    uint8_t* s_kv = s_q + TILES * Sh::Q_BYTES;
    float* s_scales = reinterpret_cast<float*>(s_kv + 2 * SLOTS * Sh::KV_BYTES);   // FP8: [PRODUCERS][SCALE_STEPS][k, v][N]
    int* s_exponents = reinterpret_cast<int*>(s_scales + Sh::PRODUCERS * Sh::SCALE_STEPS * 2 * N);   // FP8: [SCALE_STEPS][k, v][4]
    float* s_q_scale = reinterpret_cast<float*>(s_exponents + Sh::SCALE_STEPS * 8);   // FP8: [TILES][128]
    volatile int* gave_up = &s_gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kProducerWarp = 4 * TILES, kMmaWarp = kProducerWarp + 4 * Sh::PRODUCERS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * SLOTS; ++i) mbar_init(&full[i], 128 * Sh::PRODUCERS), mbar_init(&empty[i], 1);
        for (int i = 0; i < TILES; ++i) mbar_init(&q_ready[i], 128);
        for (int i = 0; i < TILES * SBUF; ++i) mbar_init(&s_ready[i], 1), mbar_init(&p_ready[i], 128);
        for (int i = 0; i < TILES * 2; ++i) mbar_init(&pv_done[i], 1);
        for (int i = 0; i < Sh::SCALE_STEPS; ++i) mbar_init(&exponents_ready[i], 4);
        mbar_init(&drained, 1);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    if (warp == 0) {
        const AttnCursor c = attn_locate<R, OV>(a, blockIdx.x, gridDim.x);
        if (lane == 0) s_cursor = c;
    }
    if (threadIdx.x == 0) a.desc[blockIdx.x].parts = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp < kProducerWarp) {
        // ---- softmax: thread = row -------------------------------------------------------------------------------
        if (Sh::SPLIT) set_registers<Sh::SOFTMAX_REGS, true>();
        AttnCursor cur = s_cursor;
        const int t = warp >> 2;                                    // row block
        const int x = threadIdx.x & 127;                            // row of the block = tensor memory lane
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;          // (32 (warp % 4)) << 16
        const uint32_t o_addr = tmem + lanes + Sh::O_COL + t * D;
        uint8_t* q_tile = s_q + t * Sh::Q_BYTES;
        const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;   // a negative scale negates q instead
        uint32_t kv_steps = 0;                                      // of the CTA, over all segments
        int steps_done = 0;                                         // of this row block, over all segments
        // The product with P of the nth step. Even and odd steps have a barrier each: a wait may be left out, as that for
        // the step after the next one on the same barrier cannot end before this block's softmax has come that far.
        auto wait_outputs = [&](int nth) {
            mbar_wait_warp(&pv_done[2 * t + (nth & 1)], (nth >> 1) & 1, gave_up);
            tc_fence_after();
        };
        for (; cur.left > 0; attn_advance<R, OV>(a, cur)) {
            int begin, end;
            attn_segment<OV>(a, cur, begin, end);
            const AttnSeq span = cur.span;
            const int rows = span.n * a.group, row0 = cur.tile * R + t * 128;
            if (begin == end) continue;
            int keys, from, to;
            chunk_steps<D, FP8>(a, cur, begin, end, keys, from, to);
            const uint32_t kv_first = kv_steps;
            kv_steps += to - from;
            if (row0 >= rows) continue;
            // q: 16-byte chunks, eight lanes to a 128-byte line, rounded to bf16, into the swizzled tile; eight requests in
            // flight (rows past the last repeat it, and are stored as zeros)
#pragma unroll 1
            for (int i0 = 0; i0 < D / 8; i0 += 8) {
                RawQ<T> raw[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = (i0 + j) * 128 + x, y = min(row0 + i / (D / 8), rows - 1);
                    const int token = (int)fast_div((uint32_t)y, a.group_div);
                    raw[j].load(static_cast<const typename T::storage*>(a.q) +
                                ((size_t)(span.q0 + token) * a.q_heads + cur.head * a.group + (y - token * a.group)) * D + i % (D / 8) * 8);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = (i0 + j) * 128 + x, r = i / (D / 8);
                    uint4 w;
                    if (FP8) {   // f16, of the row divided by the power of two that its largest element has
                        float f[8], most = 0.0f;
                        raw[j].floats(f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]));
#pragma unroll
                        for (int off = 1; off < D / 8; off <<= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, off));
                        const int exponent = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 100);
                        w = raw[j].f16(__uint_as_float((uint32_t)(127 - exponent) << 23));
                        if (i % (D / 8) == 0) s_q_scale[t * 128 + r] = __uint_as_float((uint32_t)(127 + exponent) << 23);
                    } else {
                        w = raw[j].bf16();
                    }
                    w = row0 + r < rows ? make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(q_tile + tile_offset(r, i % (D / 8), 128)) = w;
                }
            }
            async_proxy_fence();
            mbar_arrive(&q_ready[t]);
            float scale = fabsf(a.scale_log2);
            int v_exponent = -100;   // FP8: the value scales seen so far are not above 2^v_exponent
            if (FP8) {
                block_barrier(t);
                scale *= s_q_scale[t * 128 + x];
            }
            // rows past the last one are computed along where their warp has a live row (of zeros, nothing hidden), and what
            // comes of them is not stored; a warp without one only keeps step
            const int lim = row0 + x < rows ? attn_visible(a, span, row0 + x + 1) : 0x7fffffff;
            const bool warp_live = row0 + (x & ~31) < rows;
            float m = -INFINITY, l = 0.0f;
            // One step, all keys of which every live row of the row tile sees, or not (compiled twice: a test per pair of keys
            // would cost more than the pair).
            auto one_step = [&](int step, auto with_hidden) {
                constexpr bool HIDES = decltype(with_hidden)::value;
                const int buf = SBUF == 1 ? 0 : (steps_done & 1);
                const uint32_t s_addr = tmem + lanes + Sh::S_COL + (t * SBUF + buf) * N;
                const uint32_t s_parity = (SBUF == 1 ? steps_done : steps_done >> 1) & 1;
                const uint32_t nth_kv = kv_first + (step - from);
                if (FP8) mbar_wait_warp(&exponents_ready[nth_kv % Sh::SCALE_STEPS], (nth_kv / Sh::SCALE_STEPS) & 1, gave_up);
                // score scale and weight exponent of each 16 keys
                constexpr int GROUPS = FP8 ? N / 16 : 1;
                float by[GROUPS];
                int e_v[GROUPS];
                by[0] = scale, e_v[0] = 0;
                const int base = step * N;
                const int* exponents = s_exponents + nth_kv % Sh::SCALE_STEPS * 8;       // of K, then of V
                const float* scales = s_scales + nth_kv % Sh::SCALE_STEPS * 2 * N;       // likewise
                bool bare = false;
                if (FP8) {
                    const int4 ek = *reinterpret_cast<const int4*>(exponents);
                    const int4 ev = *reinterpret_cast<const int4*>(exponents + 4);
                    const int k[4] = {ek.x, ek.y, ek.z, ek.w}, v[4] = {ev.x, ev.y, ev.z, ev.w};
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        by[g] = scale * __uint_as_float((uint32_t)(127 + k[g]) << 23);   // (2^0 for bare codes)
                        e_v[g] = v[g];
                        // the reference that weights are taken against is raised by the largest exponent of V so far, so that
                        // weight times 2^e stays within f16 (O and the sum are divided by the same); groups that the row does
                        // not see have no part in it
                        if (!HIDES || (base + 16 * g < lim && v[g] != kBareCodes)) v_exponent = max(v_exponent, v[g]);
                    }
                    if (HIDES) {
                        bare = k[0] == kBareCodes || k[1] == kBareCodes || k[2] == kBareCodes || k[3] == kBareCodes ||
                               v[0] == kBareCodes || v[1] == kBareCodes || v[2] == kBareCodes || v[3] == kBareCodes;
                        if (bare) {
#pragma unroll 1
                            for (int i = 0; i < N; ++i) {
                                const bool own = exponents[4 + i / 16] == kBareCodes && base + i < lim;
                                v_exponent = own ? max(v_exponent, scale_exponent(scales[N + i])) : v_exponent;
                            }
                            __syncwarp();
                        }
                    }
                    // Weights of a group so far below the reference are 0 in f16 whatever its exponent; they are taken 2^40 below
                    // it, where f32 still holds them for the sum. (Groups without a value have an exponent of -100.) Those of bare
                    // codes are taken against the reference itself.
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) e_v[g] = HIDES && e_v[g] == kBareCodes ? v_exponent : max(e_v[g], v_exponent - 40);
                }
                mbar_wait_warp(&s_ready[t * SBUF + buf], s_parity, gave_up);
                tc_fence_after();
                if (FP8 && HIDES && bare) {   // the scores of bare codes of K take their scales
#pragma unroll 1
                    for (int g = 0; g < N / 16; ++g) {
                        if (exponents[g] != kBareCodes) continue;
                        uint32_t x[16];
                        tc_ld16(s_addr + 16 * g, x);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * scales[16 * g + i]);
                        tc_st16(s_addr + 16 * g, x);
                    }
                    tc_wait_st();
                }
                f32x2 s[N / 2];
#pragma unroll
                for (int c = 0; c < N; c += 32) tc_ld32(s_addr + c, reinterpret_cast<float*>(s + c / 2));
                tc_wait_ld();
                if (HIDES) {
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        s[i].x = base + 2 * i < lim ? s[i].x : -INFINITY;
                        s[i].y = base + 2 * i + 1 < lim ? s[i].y : -INFINITY;
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    constexpr int PAIRS = N / 2 / GROUPS;
                    float top0 = s[g * PAIRS].x, top1 = s[g * PAIRS].y;
#pragma unroll
                    for (int i = 1; i < PAIRS - 1; i += 2) {
                        top0 = max3(top0, s[g * PAIRS + i].x, s[g * PAIRS + i].y);
                        top1 = max3(top1, s[g * PAIRS + i + 1].x, s[g * PAIRS + i + 1].y);
                    }
                    top0 = fmaxf(max3(top0, top1, s[g * PAIRS + PAIRS - 1].x), s[g * PAIRS + PAIRS - 1].y);
                    top = fmaxf(top, top0 == -INFINITY ? top0 : top0 * by[g]);
                }
                if (FP8) top += (float)v_exponent;
                const bool grown = top > m + 8.0f;   // (m = -inf: any key at all)
                if (__any_sync(kFullMask, grown)) {
                    const float now = grown ? top : m;
                    const float fix = now == m ? 1.0f : fast_exp2(m - now);
                    l *= fix;
                    m = now;
                    if (step > from) {
                        // O may still be in the last step's product (S of this step came after the one before it)
                        wait_outputs(steps_done - 1);
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            tc_ld32(o_addr + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= fix;
                            tc_st32(o_addr + c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : -m;
                f32x2 sums[GROUPS][2];
#pragma unroll
                for (int c = 0; c < N / 2; c += 16) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int g = FP8 ? (c + i) / 8 : 0;
                        f32x2 e = f2_fma(s[c + i], f2_splat(by[g]), f2_splat(FP8 ? ref + (float)e_v[g] : ref));
                        if (HIDES) {   // hidden keys: a weight of exactly 0 (and scale 0 would make NaN of their -inf)
                            e.x = base + 2 * (c + i) < lim ? fast_exp2(e.x) : 0.0f;
                            e.y = base + 2 * (c + i) + 1 < lim ? fast_exp2(e.y) : 0.0f;
                        } else {
                            e = f2_pack(fast_exp2(e.x), fast_exp2(e.y));
                        }
                        const bool opens = FP8 ? (c + i) % 8 < 2 : c + i < 2;
                        sums[g][i % 2] = opens ? e : f2_add(sums[g][i % 2], e);
                        p[i] = FP8 ? pack_f16x2(e.x, e.y) : pack_bf16x2(e.x, e.y);
                    }
                    tc_st16(s_addr + c, p);   // over columns of S that are in registers
                }
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const f32x2 sum = f2_add(sums[g][0], sums[g][1]);
                    l = FP8 ? fmaf(sum.x + sum.y, __int_as_float((127 - e_v[g]) << 23), l) : l + (sum.x + sum.y);
                }
                tc_wait_st();
                if (FP8 && HIDES && bare) {   // the weights of bare codes of V take theirs, against the largest that the row sees
                    const float down = __int_as_float((127 - v_exponent) << 23);
#pragma unroll 1
                    for (int g = 0; g < N / 16; ++g) {
                        if (exponents[4 + g] != kBareCodes) continue;
                        uint32_t p[8];
                        tc_ld8(s_addr + 8 * g, p);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {   // (hidden keys have weights of 0 and may have larger scales)
                            const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
                            const float* v = scales + N + 16 * g + 2 * i;
                            p[i] = pack_f16x2(w.x * fminf(v[0] * down, 1.0f), w.y * fminf(v[1] * down, 1.0f));
                        }
                        tc_st8(s_addr + 8 * g, p);
                    }
                    tc_wait_st();
                }
                tc_fence_before();
                mbar_arrive(&p_ready[t * SBUF + buf]);
                ++steps_done;
            };
            // A row block that had no row in the last row tiles is ahead of the keys: the phase of the exponents that it would wait for
            // could be taken for an older one of the same parity. Once the scores of its first step are there, so are the exponents.
            if (FP8) mbar_wait_warp(&s_ready[t * SBUF + (SBUF == 1 ? 0 : (steps_done & 1))], (SBUF == 1 ? steps_done : steps_done >> 1) & 1, gave_up);
            if (warp_live) {
                const int hides_from = min(to, max(from, chunk_hides_from<N>(a, span, cur.tile * R)));
#pragma unroll 1
                for (int step = from; step < hides_from; ++step) one_step(step, std::false_type{});
#pragma unroll 1
                for (int step = hides_from; step < to; ++step) one_step(step, std::true_type{});
            } else {
#pragma unroll 1
                for (int step = from; step < to; ++step, ++steps_done) {
                    const int at = t * SBUF + (SBUF == 1 ? 0 : (steps_done & 1));
                    mbar_wait_warp(&s_ready[at], (SBUF == 1 ? steps_done : steps_done >> 1) & 1, gave_up);
                    mbar_arrive(&p_ready[at]);
                }
            }
            wait_outputs(steps_done - 1);
            const bool whole = begin == 0 && end == cur.keys;
            const int slot = begin == 0 ? 1 : 0;
            float* part = attn_slot(a, blockIdx.x, slot, R, D);
            if (!whole) {
                if (begin == 0 && threadIdx.x == 0) a.desc[blockIdx.x] = attn_describe<OV>(a, cur);
                part[t * 128 + x] = m;
                part[R + t * 128 + x] = *gave_up ? __int_as_float(0x7fc00000) : l;
            }
            float f = 1.0f;
            if (whole) f = l == 0.0f ? 0.0f : 1.0f / l;
            if (*gave_up) f = __int_as_float(0x7fc00000);
            if (!whole) {
                // partials: [D / 4][R][4], so that the 32 rows of a warp are 512 consecutive bytes
                float4* dst = reinterpret_cast<float4*>(part + 2 * R) + t * 128 + x;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    tc_ld32(o_addr + c, o);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) dst[(c + i) / 4 * R] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
            } else {
                // rows of `whole` columns at a time through the q tile (its products are done), then out in whole lines
                constexpr int COLS = T::kBytes == 2 ? D : D / 2;     // as many as the q tile holds
                constexpr int PIECES = COLS * T::kBytes / 16;        // 16-byte pieces of a row
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += COLS) {
#pragma unroll 1
                    for (int c = 0; c < COLS; c += 32) {
                        float o[32];
                        tc_ld32(o_addr + c0 + c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = f == 0.0f ? 0.0f : o[i] * f;
#pragma unroll
                        for (int i = 0; i < 32; i += 16 / T::kBytes) {
                            const uint4 w = T::kBytes == 2
                                ? make_uint4(pack_bf16x2(o[i], o[i + 1]), pack_bf16x2(o[i + 2], o[i + 3]), pack_bf16x2(o[i + 4 & 31], o[i + 5 & 31]),
                                             pack_bf16x2(o[i + 6 & 31], o[i + 7 & 31]))
                                : make_uint4(__float_as_uint(o[i]), __float_as_uint(o[i + 1]), __float_as_uint(o[i + 2]), __float_as_uint(o[i + 3]));
                            *reinterpret_cast<uint4*>(q_tile + tile_offset(x, (c + i) * T::kBytes / 16, 128)) = w;
                        }
                    }
                    block_barrier(t);
#pragma unroll 4
                    for (int i = x; i < 128 * PIECES; i += 128) {
                        const int r = i / PIECES, y = row0 + r;
                        if (y < rows) {
                            const int token = (int)fast_div((uint32_t)y, a.group_div);
                            typename T::storage* dst = static_cast<typename T::storage*>(a.out) +
                                ((size_t)(span.q0 + token) * a.q_heads + cur.head * a.group + (y - token * a.group)) * D + c0;
                            stg_v4(reinterpret_cast<uint8_t*>(dst) + i % PIECES * 16,
                                   *reinterpret_cast<const uint4*>(q_tile + tile_offset(r, i % PIECES, 128)));
                        }
                    }
                    block_barrier(t);   // the tile is written again, with the next columns or the next q
                }
            }
            tc_fence_before();
        }
    } else if (warp < kMmaWarp) {
        // ---- producers: a warp gathers ROWS rows of each tile, lane l of it knows row l's place -----------------
        constexpr int WARPS = 4, ROWS = N / WARPS;
        if (Sh::SPLIT) set_registers<Sh::PRODUCER_REGS, false>();
        AttnCursor cur = s_cursor;
        const int w = (warp - kProducerWarp) & 3, half = (warp - kProducerWarp) >> 2;   // rows; of their columns, with two warpgroups
        using CacheT = typename std::conditional<FP8, uint8_t, uint16_t>::type;
        constexpr int CPR = D * (FP8 ? 1 : 2) / 16;       // 16-byte pieces of a cache row
        constexpr int RPI = 32 / (CPR < 8 ? CPR : 8);     // rows a warp touches at once
        constexpr int LPR = 32 / RPI;                     // lanes per row
        constexpr int NCH = CPR / LPR / Sh::PRODUCERS;    // pieces of a row that a lane takes
        constexpr int PIECES = ROWS / RPI * NCH;          // of a tile
        constexpr int DEPTH = 3;              // tiles on their way
        if (FP8) s_scales += half * Sh::SCALE_STEPS * 2 * N;
        uint32_t asked[2] = {0, 0};           // K and V tiles so far
        // the slots not handed over yet, four bits each, the oldest on top; the fourth: the step hides keys from some row
        uint32_t pending = 0, in_flight = 0;
        static_assert(2 * SLOTS <= 8, "a slot number takes three bits");
        // place of this thread's nth piece of codes: the upper half of what the warp's own rows are widened into
        auto code_at = [&](uint8_t* tile, int n) {
            const int panel = Sh::PRODUCERS == 2 ? 2 * half + 1 : D / 128 + n / 4;   // (64 columns)
            return tile + (D == 64 ? ROWS * 64 : panel * N * 128) + w * ROWS * 128 + (n % 4 * 32 + lane) * 16;
        };
        // Hands over the oldest tile on its way, or all of them, once they have arrived. bf16 rows are where they belong. E4M3
        // codes are widened: each lane takes up the codes that it copied, and when its warp has, the f16 rows are written over
        // them, or the bare codes. A head row that held no number (its scale is NaN) makes its score NaN, whichever of the two
        // it is, and counts as zeros in V: a row that does not see the key is spared.
        uint32_t widened_k = 0, widened_v = 0;
        auto hand_over = [&](bool all) {
            if (in_flight == 0) return;
            if (all) asm volatile("cp.async.wait_group 0;" ::: "memory");
            else asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
            if (!FP8) async_proxy_fence();
            for (; in_flight > (all ? 0u : DEPTH - 1u); --in_flight) {
                const uint32_t entry = pending >> (4 * (in_flight - 1)), slot = entry & 7;
                if (FP8) {
                    uint8_t* tile = s_kv + slot * Sh::KV_BYTES;
                    uint4 code[PIECES];
#pragma unroll
                    for (int n = 0; n < PIECES; ++n) code[n] = *reinterpret_cast<const uint4*>(code_at(tile, n));
                    const uint32_t which = slot / SLOTS, nth = (which == 0 ? widened_k++ : widened_v++) % Sh::SCALE_STEPS;
                    float* sc = s_scales + nth * 2 * N + w * ROWS + lane % ROWS;   // (as this lane or lane % ROWS copied them)
                    __syncwarp();
                    const float k = sc[0], v = sc[N];
                    // the powers of two that no scale of the warp's rows reaches
                    int ev = __reduce_max_sync(kFullMask, scale_exponent(v)), own_e = ev;
                    float own = v;
                    if (which == 0) own_e = __reduce_max_sync(kFullMask, scale_exponent(k)), own = k;
                    if (__builtin_expect(entry & 8, 0)) {   // the last few steps of a row tile: are they bare codes?
                        const auto apart = [](float scale, int e, float least) {
                            const float unit = scale * __int_as_float((127 - e) << 23);
                            return __any_sync(kFullMask, unit > 0.0f && unit < least);
                        };
                        const bool v_bare = apart(v, ev, 0x1p-4f), bare = which == 0 ? apart(k, own_e, 0x1p-13f) : v_bare;
                        if (v_bare) ev = kBareCodes;
                        if (bare) own_e = kBareCodes, own = own > 0.0f ? 1.0f : 0.0f;
                        if (which == 0 && !(v < INFINITY) && lane < ROWS) sc[0] = __int_as_float(0x7fc00000), sc[N] = 0.0f;   // (as the softmax reads them)
                        __syncwarp();
                    }
                    if (which == 0 && lane == 0 && half == 0) {
                        s_exponents[nth * 8 + w] = own_e, s_exponents[nth * 8 + 4 + w] = ev;
                        mbar_arrive(&exponents_ready[nth]);
                    }
                    float unit = own * __uint_as_float((uint32_t)(127 - own_e) << 23);   // (times 1 for bare codes)
                    if (!(v < INFINITY)) unit = which == 0 ? __int_as_float(0x7fc00000) : 0.0f;
                    const uint32_t by = pack_f16x2(unit, unit);
                    __syncwarp();   // (every lane has its codes)
#pragma unroll
                    for (int n = 0; n < PIECES; ++n) {
                        const int r = w * ROWS + n / NCH * RPI + lane / LPR, ch = 2 * (lane % LPR + (n % NCH + half * NCH) * LPR);
                        uint4 lo, hi;
                        e4m3x4_to_f16(code[n].x, lo.x, lo.y);
                        e4m3x4_to_f16(code[n].y, lo.z, lo.w);
                        e4m3x4_to_f16(code[n].z, hi.x, hi.y);
                        e4m3x4_to_f16(code[n].w, hi.z, hi.w);
                        const uint32_t f = __shfl_sync(kFullMask, by, n / NCH * RPI + lane / LPR);
                        lo = make_uint4(mul_f16x2(lo.x, f), mul_f16x2(lo.y, f), mul_f16x2(lo.z, f), mul_f16x2(lo.w, f));
                        hi = make_uint4(mul_f16x2(hi.x, f), mul_f16x2(hi.y, f), mul_f16x2(hi.z, f), mul_f16x2(hi.w, f));
                        *reinterpret_cast<uint4*>(tile + tile_offset(r, ch, N)) = lo;
                        *reinterpret_cast<uint4*>(tile + tile_offset(r, ch + 1, N)) = hi;
                    }
                    async_proxy_fence();
                }
                mbar_arrive(&full[slot]);
            }
        };
        // tile `which` (0: K, 1: V) of the step whose cache rows are row32, some of which the mask hides from some row, or not
        auto fetch = [&](int which, int row32, bool hides) {
            const uint32_t nth = asked[which]++, slot = which * SLOTS + nth % SLOTS, parity = ((nth / SLOTS) & 1) ^ 1;
            uint8_t* tile = s_kv + slot * Sh::KV_BYTES;
            // While the slot is still being read, what has been asked for is handed over as it arrives.
            if (__any_sync(kFullMask, !mbar_try(&empty[slot], parity))) {
                hand_over(true);
                mbar_wait(&empty[slot], parity, gave_up);
            }
            __syncwarp();
            if (FP8 && which == 0 && lane < ROWS) {   // both scales come with K
                const size_t at = (size_t)(row32 < 0 ? 0 : row32) * a.kv_heads + cur.head;
                const uint32_t to = smem_addr(s_scales + nth % Sh::SCALE_STEPS * 2 * N + w * ROWS + lane);
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(a.k_scales + at), "r"(row32 < 0 ? 0 : 4) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + N * 4), "l"(a.v_scales + at), "r"(row32 < 0 ? 0 : 4) : "memory");
            }
            const CacheT* src = static_cast<const CacheT*>(which == 0 ? a.k : a.v);
#pragma unroll
            for (int i = 0; i < ROWS / RPI; ++i) {
                const int r = i * RPI + lane / LPR;
                const int row = __shfl_sync(kFullMask, row32, r);
                const uint8_t* p = reinterpret_cast<const uint8_t*>(src + ((size_t)(row < 0 ? 0 : row) * a.kv_heads + cur.head) * D);
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const int ch = lane % LPR + (j + half * NCH) * LPR;
                    const uint32_t dst = smem_addr(FP8 ? code_at(tile, i * NCH + j) : tile + tile_offset(w * ROWS + r, ch, N));
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p + 16 * ch), "r"(row < 0 ? 0 : 16) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            pending = pending << 4 | (hides ? 8u : 0u) | slot;
            if (++in_flight == DEPTH) hand_over(false);
        };
        for (; cur.left > 0; attn_advance<R, OV>(a, cur)) {
            int begin, end, keys, from, to;
            attn_segment<OV>(a, cur, begin, end);
            if (begin == end) continue;
            chunk_steps<D, FP8>(a, cur, begin, end, keys, from, to);
            const int hides_from = chunk_hides_from<N>(a, cur.span, cur.tile * R);
            auto lookup = [&](int step) {
                const int key = step * N + w * ROWS + (lane % ROWS);
                return step < to && key < keys ? attn_cache_row(a, cur.seq, key) : -1;
            };
            // in the order the products want them: SBUF tiles of K, then V and the K of SBUF steps later
            int rows_of[SBUF + 1];   // cache rows of steps `step` on
#pragma unroll
            for (int j = 0; j <= SBUF; ++j) rows_of[j] = lookup(from + j);
#pragma unroll
            for (int j = 0; j < SBUF; ++j) {
                if (from + j < to) fetch(0, rows_of[j], from + j >= hides_from);
            }
            for (int step = from; step < to; ++step) {
                const int ahead = lookup(step + SBUF + 1);
                fetch(1, rows_of[0], step >= hides_from);
                if (step + SBUF < to) fetch(0, rows_of[SBUF], step + SBUF >= hides_from);
#pragma unroll
                for (int j = 0; j < SBUF; ++j) rows_of[j] = rows_of[j + 1];
                rows_of[SBUF] = ahead;
            }
        }
        hand_over(true);
    } else {
        if (Sh::SPLIT) set_registers<Sh::MMA_REGS, false>();
        AttnCursor cur = s_cursor;
        if (warp == kMmaWarp) {
        // ---- products: one warp, one lane of which issues ----------------------------------------------------------
        const uint32_t leader = elect_lane();
        const uint32_t q_base = uniform((int)smem_addr(s_q)), kv_base = uniform((int)smem_addr(s_kv)), acc = uniform((int)tmem);
        constexpr uint32_t s_idesc = mma_idesc(N, false, FP8), o_idesc = mma_idesc(D, true, FP8);
        uint32_t used = 0;                // K tiles, and V tiles, consumed so far
        int segments[TILES] = {}, steps_done[TILES] = {};
        auto scores = [&](int t, int nth, uint32_t k_slot) {   // S of the nth step of row block t
            const int buf = SBUF == 1 ? 0 : (nth & 1);
            const uint32_t q_low = desc_low(q_base + t * Sh::Q_BYTES, 16);
            const uint32_t k_low = desc_low(kv_base + k_slot * Sh::KV_BYTES, 16);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint64_t qa = smem_desc(q_low, (k >> 2) * 128 * 128 + (k & 3) * 32);
                const uint64_t kb = smem_desc(k_low, (k >> 2) * N * 128 + (k & 3) * 32);
                tc_mma_ss(acc + Sh::S_COL + (t * SBUF + buf) * N, qa, kb, s_idesc, k > 0, leader);
            }
            tc_commit(&s_ready[t * SBUF + buf], leader);
        };
        auto outputs = [&](int t, int nth, uint32_t v_slot, bool add) {
            const int buf = SBUF == 1 ? 0 : (nth & 1);
            const uint32_t v_low = desc_low(kv_base + v_slot * Sh::KV_BYTES, N * 128);
#pragma unroll
            for (int k = 0; k < N / 16; ++k) {
                const uint64_t vb = smem_desc(v_low, k * 2048);
                tc_mma_ts(acc + Sh::O_COL + t * D, acc + Sh::S_COL + (t * SBUF + buf) * N + 8 * k, vb, o_idesc, add || k > 0, leader);
            }
            tc_commit(&pv_done[2 * t + (nth & 1)], leader);
        };
        for (; uniform(cur.left > 0); attn_advance<R, OV>(a, cur)) {
            int begin, end, keys, from, to;
            attn_segment<OV>(a, cur, begin, end);
            if (uniform(begin == end)) continue;
            chunk_steps<D, FP8>(a, cur, begin, end, keys, from, to);
            const int blocks = uniform(cur.span.n * a.group - cur.tile * R > 128 ? TILES : 1);
            const int count = uniform(to - from);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (t < blocks) mbar_wait_warp(&q_ready[t], segments[t]++ & 1, gave_up);
            }
            // the first SBUF steps' scores, then for each step its output and the scores SBUF steps later
            auto k_slot_of = [&](int j) { return (used + j) % SLOTS; };
            auto tile_parity = [&](int j) { return ((used + j) / SLOTS) & 1; };
            for (int j = 0; j < SBUF && j < count; ++j) {
                mbar_wait_warp(&full[k_slot_of(j)], tile_parity(j), gave_up);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (t < blocks) scores(t, steps_done[t] + j, k_slot_of(j));
                }
                tc_commit(&empty[k_slot_of(j)], leader);
            }
            for (int j = 0; j < count; ++j) {
                const uint32_t v_slot = SLOTS + k_slot_of(j), k_slot = k_slot_of(j + SBUF);
                mbar_wait_warp(&full[v_slot], tile_parity(j), gave_up);
                const bool more = j + SBUF < count;
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (t >= blocks) break;
                    const int nth = steps_done[t] + j;
                    const int buf = SBUF == 1 ? 0 : (nth & 1);
                    mbar_wait_warp(&p_ready[t * SBUF + buf], (SBUF == 1 ? nth : nth >> 1) & 1, gave_up);
                    tc_fence_after();
                    outputs(t, nth, v_slot, j > 0);
                    if (t == blocks - 1) tc_commit(&empty[v_slot], leader);
                    if (more) {
                        if (t == 0) {
                            mbar_wait_warp(&full[k_slot], tile_parity(j + SBUF), gave_up);
                            tc_fence_after();
                        }
                        scores(t, nth + SBUF, k_slot);
                        if (t == blocks - 1) tc_commit(&empty[k_slot], leader);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) steps_done[t] += t < blocks ? count : 0;
            used += count;
        }
        // every product and every arrival it triggers has landed before the CTA goes (also after a wait that gave up)
        tc_commit(&drained, leader);
        for (int i = 0; i < (1 << 20) && !mbar_try(&drained, 0); ++i) {
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace clef
