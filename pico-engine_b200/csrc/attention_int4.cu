// Attention of single tokens over the paged cache of 4-bit keys and values (int4_pages.cuh).
//
// A key is mid + step c per group of 32 channels, c = +-(k + 1/2), so a score is the sum over the groups of step (q . c) + mid (sum of q): products of the queries with codes as they stand, and one
// more product of the groups' sums with their middles.  A value likewise: o = sum_j (w_j step_j) c_j + w_j mid_j.  The codes are bfloat16 numbers of 2^-129 units (subnormal, which mma.sync
// keeps exactly), so queries and weights are taken 2^64 higher and sums 2^65 down; the bits of two codes cost two instructions, a rotation and one with a mask, and no conversion.
// Scores, softmax statistics and results are float32 (running maximum and sum, one pass).  The groups' sums of queries keep float32's 24 bits, in three bfloat16 parts, which the product has
// room for.  A weight is rounded to bfloat16 for its product, and once more behind its multiplication by a value's step: scaling the weights takes a multiplication a group and position, scaling
// the products would take one a channel and position.  Results are off by 0.0021 of their size for it, of which their own rounding is 0.0017; a second product with what the second rounding
// leaves brings 0.0019, one with what both leave 0.0017, and the two long cases below then take 70 and 94 us, or 75 and 97, for 65 and 87: the 16 bits a weight of the first form are kept.
//
// Keys (or channels) are the 16 rows of mma.sync m16n8k16 and a key head's queries its 8 columns: eight heads of a group are few for tcgen05.mma, whose operands would have to be written
// to shared memory in 16 bits first.  A warp takes a page and key head at a time, a block of 80 D bytes that one bulk copy brings into its own ring of two, asked for by a warp
// that does nothing else (with copies by each warp for itself 1.03 us a block and SM partition, 0.82 so; three places a warp leave room for fewer warps, which is slower; keys and values
// in copies of their own wait 0.4 us a page longer).  The warps' sums are joined in shared memory, those of a cluster's CTAs through distributed shared memory.
//
// What bounds it: a block's chain of instructions in few warps.  A block of 64 channels takes 618, 319 of them on the logic units (two a pair of codes), 40 on the tensor cores (a quarter of their time).  The same kernel with the arithmetic
// taken out copies its blocks in 46 us where the whole takes 65.5 (64 rows of 20,000 to 32,700, 14 heads of 64 on 2: 266 MB, 41 us at the copy rate of 6.5 TB/s); 63 of 86 (200 rows of up to 6,000,
// 28 heads of 128 on 4: 385 MB, 59 us).  Fifteen warps (eleven of 128 channels, 168 registers) are what registers allow, and do not hide one another's waits: the schedulers issue in 58 of 100 cycles,
// the logic units are busy for 57 of them, DRAM for 53 to 62.  One row of 4,096 positions takes 4.5 us: a launch, and one chain of positions, table, block, join.
#include "int4_pages.cuh"
#include <atomic>

#define AI_MAX_SPLITS 16
#define AI_WAIT_CYCLES 2000000000ll                            // about a second of SM clock

__device__ __forceinline__ float ai_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned ai_pack(float lo, float hi) { __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ unsigned ai_transpose(unsigned a) { unsigned d; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a)); return d; }
__device__ __forceinline__ unsigned ai_times(unsigned a, unsigned b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void ai_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with sums that start at zero
__device__ __forceinline__ void ai_mma0(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ai_max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ void ai_mma8(float (&c)[4], unsigned a0, unsigned a1, unsigned b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

// 2^n as a float, -126 <= n <= 127
__host__ __device__ constexpr float ai_pow2(int n) { return n >= 0 ? (n == 0 ? 1.f : 2.f * ai_pow2(n - 1)) : 0.5f * ai_pow2(n + 1); }
#define AI_UP 64                                               // queries and weights are taken 2^64 higher, since codes are products' operands in units of 2^-129
#define AI_DOWN (AI_UP - 129)                                  // what sums of products with codes are multiplied by

template <int D>
struct AiQuery {
    unsigned q[D / 16][2];                                     // fragments of 2^64 q, the channels of a group in the order of the keys' words
    unsigned sums[D / 64];                                     // of the groups: 2^-65 (sum of q) in three parts, 24 bits, for the product with the middles
};

template <int D>
struct AiState {
    float acc[D / 16][4];                                      // [m][n * 2 + head]: channel 32 (m / 2) + 4 g + 2 (m % 2) + n, heads 2 t and 2 t + 1
    float mids[4];                                             // [head]: group g (below D / 32)
    float top[2], sum[2];                                      // of heads 2 t and 2 t + 1: largest score (times log2 e); this lane's part of the sum of weights (times 2^64)
};

template <int D>
__device__ __forceinline__ void ai_reset(AiState<D>& s) {
#pragma unroll
    for (int m = 0; m < D / 16; ++m) s.acc[m][0] = s.acc[m][1] = s.acc[m][2] = s.acc[m][3] = 0.f;
    s.mids[0] = s.mids[1] = s.mids[2] = s.mids[3] = 0.f;
    s.top[0] = s.top[1] = -INFINITY;
    s.sum[0] = s.sum[1] = 0.f;
}

template <int D>
__device__ __forceinline__ void ai_query(AiQuery<D>& f, const bf16* q, bool there, int t) {
    constexpr int NB = D / 32;
    float sum[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (there) asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(q + 32 * b + 8 * t) : "memory");
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
        sum[b] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xffff0000u);
            sum[b] += lo + hi;
            f.q[2 * b + (i >> 1)][i & 1] = ai_pack(lo * ai_pow2(AI_UP), hi * ai_pow2(AI_UP));
        }
        sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
        sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
        sum[b] *= ai_pow2(AI_DOWN);
    }
    // as the product's operand, a pair of groups a register: the high parts, behind them what those leave, then what these leave (of 64 channels rows 2 t and 2 t + 1, t the part; of 128
    // t & 1 the pair, t / 2 the part, and the third parts in the second half of the rows)
    const int pair = D == 128 ? (t & 1) : 0, part = D == 128 ? t >> 1 : t;
    float a[3], b[3];
    a[0] = pair ? sum[NB > 2 ? 2 : 0] : sum[0]; b[0] = pair ? sum[NB > 2 ? 3 : 1] : sum[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) { a[i + 1] = a[i] - __bfloat162float(__float2bfloat16_rn(a[i])); b[i + 1] = b[i] - __bfloat162float(__float2bfloat16_rn(b[i])); }
    f.sums[0] = part == 0 ? ai_pack(a[0], b[0]) : part == 1 ? ai_pack(a[1], b[1]) : part == 2 ? ai_pack(a[2], b[2]) : 0u;
    if constexpr (D == 128) f.sums[1] = part == 0 ? ai_pack(a[2], b[2]) : 0u;
}

// Positions of a block that are not seen (below lo, above hi) may hold anything: their values' steps and middles become zero, in the warp's own copy.
template <int D>
__device__ __forceinline__ void ai_clear(unsigned char* block, int lo, int hi, int lane) {
#pragma unroll
    for (int p = lane; p < PE_PAGE; p += 32)
        if (p < lo || p > hi) {
            unsigned short* meta = reinterpret_cast<unsigned short*>(block + q4_value_step<D>(p, 0));
#pragma unroll
            for (int b = 0; b < 2 * Int4Block<D>::groups; ++b) meta[b * 16] = 0;
        }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                          // (the copy that will refill the place comes behind these)
    __syncwarp();
}

// Scores of a block's positions for the warp's eight heads: sc[j][2 r + h] of position 16 j + 8 r + g and head 2 t + h, in units of 2^AI_DOWN.
template <int D>
__device__ __forceinline__ void ai_scores(float (&sc)[4][4], const AiQuery<D>& f, const unsigned char* block, int g, int t) {
    constexpr int NB = Int4Block<D>::groups;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned words[2][NB], steps[2][NB / 2], mid[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int p = 16 * j + 8 * r + g;
            const unsigned char* kw = block + q4_key_word<D>(p, 0, t);
            const unsigned char* km = block + q4_key_step<D>(p, 0);
            if constexpr (D == 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(kw);
                words[r][0] = v.x; words[r][1] = v.y; words[r][2] = v.z; words[r][3] = v.w;
                const uint2 st = *reinterpret_cast<const uint2*>(km);
                steps[r][0] = st.x; steps[r][1] = st.y;
                mid[r] = *reinterpret_cast<const unsigned*>(km + 8 + 4 * (t & 1));
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(kw), st = *reinterpret_cast<const uint2*>(km);
                words[r][0] = v.x; words[r][1] = v.y; steps[r][0] = st.x; mid[r] = st.y;
            }
        }
        if constexpr (D == 128) ai_mma0(sc[j], mid[0], mid[1], mid[0], mid[1], f.sums[0], f.sums[1]);
        else ai_mma8(sc[j], mid[0], mid[1], f.sums[0]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float c[4];
            ai_mma0(c, q4_pair(words[0][b], 0), q4_pair(words[1][b], 0), q4_pair(words[0][b], 1), q4_pair(words[1][b], 1), f.q[2 * b][0], f.q[2 * b][1]);
            ai_mma(c, q4_pair(words[0][b], 2), q4_pair(words[1][b], 2), q4_pair(words[0][b], 3), q4_pair(words[1][b], 3), f.q[2 * b + 1][0], f.q[2 * b + 1][1]);
            const float s0 = __uint_as_float((b & 1) ? steps[0][b >> 1] & 0xffff0000u : steps[0][b >> 1] << 16);
            const float s1 = __uint_as_float((b & 1) ? steps[1][b >> 1] & 0xffff0000u : steps[1][b >> 1] << 16);
            sc[j][0] = fmaf(c[0], s0, sc[j][0]); sc[j][1] = fmaf(c[1], s0, sc[j][1]);
            sc[j][2] = fmaf(c[2], s1, sc[j][2]); sc[j][3] = fmaf(c[3], s1, sc[j][3]);
        }
    }
}

// The weights of the scores as operands (positions 16 j + 8 r + 2 t and the next, head g) in w[j][r]; the state's sums are brought to the new largest scores.
// lo <= position <= hi of the block are seen.
template <int D>
__device__ __forceinline__ void ai_weigh(AiState<D>& s, float (&sc)[4][4], unsigned (&w)[4][2], int lo, int hi, float scale, int g) {
    if (lo > 0 || hi < PE_PAGE - 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int p = 16 * j + 8 * r + g;
                if (p < lo || p > hi) sc[j][2 * r] = sc[j][2 * r + 1] = -INFINITY;
            }
    }
    bool moved = false;
    float ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float top = fmaxf(sc[0][h], sc[0][2 + h]);
#pragma unroll
        for (int j = 1; j < 4; ++j) top = ai_max3(top, sc[j][h], sc[j][2 + h]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top *= scale;
        ref[h] = s.top[h];
        moved |= top > s.top[h];
        s.top[h] = fmaxf(s.top[h], top);
    }
    if (__any_sync(0xffffffffu, moved)) {                      // seldom after the first blocks
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float alpha = s.top[h] == -INFINITY ? 1.f : ai_ex2(ref[h] - s.top[h]);
            s.sum[h] *= alpha;
            s.mids[h] *= alpha;
#pragma unroll
            for (int m = 0; m < D / 16; ++m) { s.acc[m][h] *= alpha; s.acc[m][2 + h] *= alpha; }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) ref[h] = s.top[h] == -INFINITY ? 0.f : AI_UP - s.top[h];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = ai_ex2(fmaf(sc[j][e], scale, ref[e & 1])); s.sum[e & 1] += x[e]; }
        w[j][0] = ai_transpose(ai_pack(x[0], x[1]));
        w[j][1] = ai_transpose(ai_pack(x[2], x[3]));
    }
}

template <int D>
__device__ __forceinline__ void ai_values(AiState<D>& s, const unsigned (&w)[4][2], const unsigned char* block, int g, int t) {
    using B = Int4Block<D>;
    constexpr int NB = B::groups;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned char* vm = block + B::value_meta + j * (4 * NB * 16) + t * 8;
        const uint2 mids = *reinterpret_cast<const uint2*>(vm + (NB + (g & (NB - 1))) * 32);       // (rows from NB on are sums that nobody reads)
        ai_mma(s.mids, mids.x, 0u, mids.y, 0u, w[j][0], w[j][1]);
#pragma unroll
        for (int h = 0; h < B::halves; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(block + q4_value_words<D>(j, h, g, t));
            const unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint2 st = *reinterpret_cast<const uint2*>(vm + (2 * h + b) * 32);
                const unsigned q0 = ai_times(w[j][0], st.x), q1 = ai_times(w[j][1], st.y);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const unsigned x = words[2 * b + m];
                    ai_mma(s.acc[4 * h + 2 * b + m], q4_pair(x, 0), q4_pair(x, 1), q4_pair(x, 2), q4_pair(x, 3), q0, q1);
                }
            }
        }
    }
}

template <int D>
__device__ __forceinline__ void ai_block(AiState<D>& s, const AiQuery<D>& f, unsigned char* block, int lo, int hi, float scale, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float sc[4][4];
    unsigned w[4][2];
    if (lo > 0 || hi < PE_PAGE - 1) ai_clear<D>(block, lo, hi, lane);
    ai_scores<D>(sc, f, block, g, t);
    ai_weigh<D>(s, sc, w, lo, hi, scale, g);
    ai_values<D>(s, w, block, g, t);
}

__device__ __forceinline__ unsigned ai_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ai_bar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void ai_bar_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ai_bulk_copy(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void ai_bar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// true when the phase with this parity has completed; a wait is false when it runs out
__device__ __forceinline__ bool ai_bar_test(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0u;
}
__device__ __forceinline__ bool ai_bar_wait(unsigned bar, unsigned parity) {
    unsigned done;
    if (ai_bar_test(bar, parity)) return true;
    const long long deadline = clock64() + AI_WAIT_CYCLES;
    for (;;) {
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if (clock64() > deadline) return false;
    }
}
__device__ __forceinline__ void ai_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void ai_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ unsigned ai_cluster_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned ai_map(unsigned local, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
template <int D>
__device__ __forceinline__ void ai_fetch(unsigned to, const unsigned char* block, unsigned bar) {
    ai_bar_expect(bar, Int4Block<D>::bytes);
    ai_bulk_copy(to, block, Int4Block<D>::bytes, bar);
}
// numbers into another CTA's shared memory; their bytes are counted on that CTA's barrier
__device__ __forceinline__ void ai_send4(unsigned to, float4 v, unsigned bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(__float_as_uint(v.x)),
                 "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)), "r"(bar) : "memory");
}

// WARPS of a CTA compute and one more fetches.  Blocks that such a warp has places for, CTAs an SM.
template <int D, int WARPS>
struct AiShape {
    static constexpr int warps = WARPS, stages = 2, ctas = D == 64 && WARPS < 8 ? 2 : 1, threads = 32 * (warps + 1);
    static constexpr int row = D + 4;                          // floats of a head's results: D sums, largest score, sum of weights
    static constexpr int blocks = warps * stages * Int4Block<D>::bytes, parts = warps * 8 * row * 4;
    static constexpr int ring = ((blocks > parts ? blocks : parts) + 127) / 128 * 128;    // the warps' results lie in the ring later
    static constexpr int gather = AI_MAX_SPLITS * 8 * 4 * 4 + 8 * D * 4;
    static constexpr int smem = ring + gather;
};

template <int D, int WARPS>
__global__ void __launch_bounds__(AiShape<D, WARPS>::threads, AiShape<D, WARPS>::ctas) attention_int4_kernel(
    const bf16* q, int q_stride, const unsigned char* pool, int n_blocks, const int* block_table, int table_stride, int n_rows, const int* tok_pos, const int* tok_row,
    int n_heads, int n_kv, int window, float scale_log2e, int selected, int n_splits, int early, int* status, bf16* out) {
    using S = AiShape<D, WARPS>;
    using B = Int4Block<D>;
    extern __shared__ __align__(128) unsigned char ai_ring[];   // [warp][stage] blocks; later the warps' results; behind it what the other CTAs send
    __shared__ __align__(8) unsigned long long bars[2 * WARPS * S::stages + 1];           // per warp and stage: a block is there; its place is free
    __shared__ int filled[WARPS * S::stages];                  // whether the stage holds a block (a page may not be there)
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = n_splits > 1 ? (int)ai_cluster_rank() : 0, slice = D / n_splits;
    float* gather = reinterpret_cast<float*>(ai_ring + S::ring);                          // [split][8][slice + 4]
    const unsigned gather0 = ai_smem(gather), full0 = ai_smem(bars), empty0 = full0 + 8u * WARPS * S::stages, gbar = empty0 + 8u * WARPS * S::stages;
    const int G = n_heads / n_kv, head_tiles = (G + 7) / 8, kvh = blockIdx.y / head_tiles, h0 = (blockIdx.y % head_tiles) * 8, heads = min(8, G - h0);
    if (threadIdx.x < 2 * WARPS * S::stages + 1) ai_bar_init(full0 + 8u * threadIdx.x, 1u);
    if (threadIdx.x == 2 * WARPS * S::stages && n_splits > 1) ai_bar_expect(gbar, (unsigned)((n_splits - 1) * heads * (slice + 4) * 4));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!early) pdl_wait();
    const int tok = blockIdx.z, place = selected ? tok * n_kv + kvh : tok, pos = min(tok_pos[place], table_stride * PE_PAGE - 1), row = selected ? place : tok_row[tok];
    __syncthreads();
    if (n_splits > 1) ai_cluster_arrive();                     // waited for before the first number goes to another CTA
    const int lo = window > 0 ? max(0, pos - window + 1) : 0, step = n_splits * WARPS;
    const int last = pos >= 0 && row >= 0 && row < n_rows ? pos / PE_PAGE : -1;
    AiState<D> s;
    ai_reset(s);
    if (warp == WARPS) {
        // ---- the warp that fetches: a lane for each of the others, whose pages are first, first + step, ..
        const int first = lo / PE_PAGE + split * WARPS + lane;
        const int n = lane < WARPS && last >= first ? (last - first) / step + 1 : 0;
        const int n_pages = selected ? n_blocks : n_blocks / n_kv;
        const int* table = block_table + (size_t)max(0, min(row, n_rows - 1)) * table_stride + first;
        // (early: the page of the newest position is written by the kernel before this one)
        const int settled = n - (n > 0 && first + (n - 1) * step == last);
        bool waits = early != 0;
        int page = n > 0 ? table[0] : -1, next = n > 1 ? table[step] : -1, stage = 0, round = 0;
        long long deadline = 0;
        for (int i = 0; __any_sync(0xffffffffu, i < n);) {
            const unsigned at = (unsigned)(lane * S::stages + stage);
            bool ready = i < n && !(waits && i >= settled);
            if (ready && round > 0) ready = ai_bar_test(empty0 + 8u * at, (unsigned)(round - 1) & 1u);
            if (ready) {
                const bool there = page >= 0 && page < n_pages;
                filled[at] = there;
                if (there) ai_fetch<D>(ai_smem(ai_ring) + at * B::bytes, pool + (size_t)(selected ? page : page * n_kv + kvh) * B::bytes, full0 + 8u * at);
                else ai_bar_arrive(full0 + 8u * at);
                page = next;
                if (++i + 1 < n) next = table[(i + 1) * step];
                if (++stage == S::stages) { stage = 0; ++round; }
                deadline = 0;
            }
            if (!__any_sync(0xffffffffu, ready)) {
                if (waits) {
                    pdl_wait();
                    waits = false;
                } else if (!deadline) {
                    deadline = clock64() + AI_WAIT_CYCLES;
                } else if (clock64() > deadline && i < n) {
                    atomicExch(status, 21);
                    i = n;
                }
            }
        }
        if (waits) pdl_wait();
    } else {
        // ---- the warps that compute
        if (early) pdl_wait();
        AiQuery<D> f;
        ai_query<D>(f, q + (size_t)tok * q_stride + (size_t)(kvh * G + h0 + g) * D, h0 + g < G, t);
        const float scale = scale_log2e * ai_pow2(-AI_DOWN);
        const int first = lo / PE_PAGE + split * WARPS + warp;
        int stage = 0;
        unsigned phase = 0;
        for (int j = first; j <= last; j += step) {
            const int at = warp * S::stages + stage;
            if (!__all_sync(0xffffffffu, ai_bar_wait(full0 + 8u * at, phase))) {
                if (lane == 0) atomicExch(status, 22);
                break;
            }
            if (filled[at]) ai_block<D>(s, f, ai_ring + at * B::bytes, lo - j * PE_PAGE, pos - j * PE_PAGE, scale, lane);
            __syncwarp();
            if (lane == 0) ai_bar_arrive(empty0 + 8u * at);
            if (++stage == S::stages) { stage = 0; phase ^= 1u; }
        }
    }

    // ---- the warps' results, joined in shared memory (the ring is free once every warp has left its loop)
    __syncthreads();
    float* part = reinterpret_cast<float*>(ai_ring);           // [warp][8][row]
    if (warp < WARPS) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.sum[h] += __shfl_xor_sync(0xffffffffu, s.sum[h], o);
            float* to = part + (warp * 8 + 2 * t + h) * S::row;
            if (g == 0) { to[D] = s.top[h]; to[D + 1] = s.sum[h]; }
#pragma unroll
            for (int b = 0; b < B::groups; ++b) {
                const float mid = __shfl_sync(0xffffffffu, s.mids[h], b * 4 + t) * ai_pow2(-AI_UP);
                *reinterpret_cast<float4*>(to + 32 * b + 4 * g) =
                    make_float4(fmaf(s.acc[2 * b][h], ai_pow2(-AI_DOWN), mid), fmaf(s.acc[2 * b][2 + h], ai_pow2(-AI_DOWN), mid),
                                fmaf(s.acc[2 * b + 1][h], ai_pow2(-AI_DOWN), mid), fmaf(s.acc[2 * b + 1][2 + h], ai_pow2(-AI_DOWN), mid));
            }
        }
    }
    __syncthreads();
    if (n_splits > 1) ai_cluster_wait();
    for (int i = threadIdx.x; i < heads * (D / 4); i += S::threads) {
        const int h = i / (D / 4), c = (i % (D / 4)) * 4;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part[(w * 8 + h) * S::row + D]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* from = part + (w * 8 + h) * S::row;
            const float x = from[D + 1] == 0.f ? 0.f : ai_ex2(from[D] - m);
            const float4 v = *reinterpret_cast<const float4*>(from + c);
            o.x = fmaf(v.x, x, o.x); o.y = fmaf(v.y, x, o.y); o.z = fmaf(v.z, x, o.z); o.w = fmaf(v.w, x, o.w);
            l = fmaf(from[D + 1], x, l);
        }
        if (n_splits == 1) {
            const float r = l == 0.f ? 0.f : 1.f / (l * ai_pow2(-AI_UP));
            const uint2 v = make_uint2(ai_pack(o.x * r, o.y * r), ai_pack(o.z * r, o.w * r));
            *reinterpret_cast<uint2*>(out + ((size_t)tok * n_heads + kvh * G + h0 + h) * D + c) = v;
            continue;
        }
        // the CTA that owns these columns gets them, and each its part of what weighs them
        const int to = c / slice;
        const unsigned place = gather0 + (unsigned)(((split * 8 + h) * (slice + 4) + c - to * slice) * 4);
        if (to == split) *reinterpret_cast<float4*>(gather + (split * 8 + h) * (slice + 4) + c - to * slice) = o;
        else ai_send4(ai_map(place, to), o, ai_map(gbar, to));
        if (c / 4 < n_splits) {
            const int d = c / 4;
            const float4 ml = make_float4(m, l, 0.f, 0.f);
            if (d == split) *reinterpret_cast<float4*>(gather + (split * 8 + h) * (slice + 4) + slice) = ml;
            else ai_send4(ai_map(gather0 + (unsigned)(((split * 8 + h) * (slice + 4) + slice) * 4), d), ml, ai_map(gbar, d));
        }
    }
    if (n_splits == 1) return;
    __syncthreads();
    if (!ai_bar_wait(gbar, 0u)) {
        if (threadIdx.x == 0) atomicExch(status, 22);
        return;
    }
    for (int i = threadIdx.x; i < heads * (slice / 4); i += S::threads) {
        const int h = i / (slice / 4), c = (i % (slice / 4)) * 4;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < n_splits; ++r) m = fmaxf(m, gather[(r * 8 + h) * (slice + 4) + slice]);
        for (int r = 0; r < n_splits; ++r) {
            const float* from = gather + (r * 8 + h) * (slice + 4);
            const float x = from[slice + 1] == 0.f ? 0.f : ai_ex2(from[slice] - m);
            const float4 v = *reinterpret_cast<const float4*>(from + c);
            o.x = fmaf(v.x, x, o.x); o.y = fmaf(v.y, x, o.y); o.z = fmaf(v.z, x, o.z); o.w = fmaf(v.w, x, o.w);
            l = fmaf(from[slice + 1], x, l);
        }
        const float r = l == 0.f ? 0.f : 1.f / (l * ai_pow2(-AI_UP));
        const uint2 v = make_uint2(ai_pack(o.x * r, o.y * r), ai_pack(o.z * r, o.w * r));
        *reinterpret_cast<uint2*>(out + ((size_t)tok * n_heads + kvh * G + h0 + h) * D + split * slice + c) = v;
    }
}

// ---------------------------------------------------------------------------- many pages: every warp an equal run of them
//
// The blocks of all pairs (a place and a tile of eight heads) stand in one row, and each warp takes an equal run of that row, whatever it cuts: rows of unequal lengths keep all
// SMs busy to the end.  A place is a token with its page table: a token of the step, or, over selected pages, a token's key head.  What a warp finds for a pair that it has alone
// it writes; of the others (the first and the last of its run at most) it leaves the sums in a place of its own, and a second kernel joins them.

#define AI_LEAST 4                                             // blocks a warp takes at least
#define AI_MAX_PLACES 1024

template <int D>
struct AiStream {
    static constexpr int warps = D == 64 ? 15 : 11, stages = 2, threads = 32 * (warps + 1), row = D + 4, ring = warps * stages * Int4Block<D>::bytes;
};

struct AiPlaces {
    const int* tok_pos; const int* tok_row; const int* block_table;
    int n, table_stride, n_rows, n_pages, n_kv, n_heads, head_tiles, window, selected;
    __device__ __forceinline__ int pairs() const { return selected ? head_tiles : n_kv * head_tiles; }      // of a place
    __device__ __forceinline__ int position(int place) const { return min(tok_pos[place], table_stride * PE_PAGE - 1); }
    __device__ __forceinline__ int first_seen(int pos) const { return window > 0 ? max(0, pos - window + 1) : 0; }
    // pages of a place; one that sees nothing has a page that is not there
    __device__ __forceinline__ int pages(int place) const {
        const int pos = position(place);
        return pos < 0 ? 1 : pos / PE_PAGE - first_seen(pos) / PE_PAGE + 1;
    }
    __device__ __forceinline__ void heads_of(int place, int pair, int& tok, int& kvh, int& h0) const {
        tok = selected ? place / n_kv : place;
        kvh = selected ? place % n_kv : pair / head_tiles;
        h0 = pair % head_tiles * 8;
    }
};

// Warps that share so many blocks.
__device__ __forceinline__ int ai_workers(int blocks, int most) { return min(most, max(1, blocks / AI_LEAST)); }
// The block that warp w's run begins with.
__device__ __forceinline__ int ai_begin(int w, int blocks, int workers) { return (int)((long long)w * blocks / workers); }

// The number of pages before every place, prefix[n] that of all, into shared memory.
template <int THREADS>
__device__ __forceinline__ void ai_prefix(const AiPlaces& p, int* prefix, int* warp_sums) {
    const int each = (p.n + THREADS - 1) / THREADS, from = min(p.n, (int)threadIdx.x * each), to = min(p.n, from + each), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = 0;
    for (int i = from; i < to; ++i) { const int n = p.pages(i); prefix[i] = n; sum += n; }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
    if (lane == 31) warp_sums[warp] = before;
    before -= sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) if (w < warp) before += warp_sums[w];
    for (int i = from; i < to; ++i) { const int n = prefix[i]; prefix[i] = before; before += n; }
    if (from < p.n && to == p.n) prefix[p.n] = before;
    __syncthreads();
}

// Where a block of the row lies: the place, the pair of the place, the page among the place's pages.
struct AiAt { int place, pair, page, pages; };
__device__ __forceinline__ AiAt ai_find(int x, int pairs, int n, const int* prefix) {
    const int y = x / pairs;
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (prefix[mid] <= y) lo = mid; else hi = mid; }
    const int pages = prefix[lo + 1] - prefix[lo], rest = x - prefix[lo] * pairs, pair = rest / pages;
    return {lo, pair, rest - pair * pages, pages};
}
// The block behind it (there is one); true where another pair begins.
__device__ __forceinline__ bool ai_next(AiAt& a, int pairs, const int* prefix) {
    if (++a.page < a.pages) return false;
    a.page = 0;
    if (++a.pair == pairs) { a.pair = 0; ++a.place; a.pages = prefix[a.place + 1] - prefix[a.place]; }
    return true;
}

template <int D>
__global__ void __launch_bounds__(AiStream<D>::threads, 1) attention_int4_stream_kernel(const bf16* q, int q_stride, const unsigned char* pool, const AiPlaces p, float scale_log2e,
                                                                                        int early, int most, float* partial, int* prefix_out, int* status, bf16* out) {
    using S = AiStream<D>;
    using B = Int4Block<D>;
    constexpr int WARPS = S::warps;
    extern __shared__ __align__(128) unsigned char ai_ring[];   // [warp][stage] blocks, then the prefix
    __shared__ __align__(8) unsigned long long bars[2 * WARPS * S::stages];
    __shared__ int filled[WARPS * S::stages], warp_sums[S::threads / 32];
    int* prefix = reinterpret_cast<int*>(ai_ring + S::ring);
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const unsigned full0 = ai_smem(bars), empty0 = full0 + 8u * WARPS * S::stages;
    if (threadIdx.x < 2 * WARPS * S::stages) ai_bar_init(full0 + 8u * threadIdx.x, 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!early) pdl_wait();
    ai_prefix<S::threads>(p, prefix, warp_sums);                // (its barriers also make those of the ring known)
    const int pairs = p.pairs(), total = prefix[p.n] * pairs, workers = ai_workers(total, most);     // (warp w of the run: block w % grid, so that few are spread over all SMs)
    if ((int)blockIdx.x >= workers) return;                     // (before anything is written: the kernel in front may still run)
    if (warp == WARPS) {
        // ---- the warp that fetches: a lane for each of the others
        const int w = lane * gridDim.x + blockIdx.x, a = lane < WARPS && w < workers ? ai_begin(w, total, workers) : 0, b = lane < WARPS && w < workers ? ai_begin(w + 1, total, workers) : 0;
        AiAt at = {0, 0, 0, 1};
        if (a < b) at = ai_find(a, pairs, p.n, prefix);
        // the block to fetch, and whether the kernel before this one may still write its page
        bool newest = false;
        const auto look = [&]() {
            const int pos = p.position(at.place), row = p.selected ? at.place : p.tok_row[at.place], j = p.first_seen(pos) / PE_PAGE + at.page;
            newest = pos < 0 || j == pos / PE_PAGE;
            if (pos < 0 || row < 0 || row >= p.n_rows) return -1;
            const int page = p.block_table[(size_t)row * p.table_stride + j];
            if (page < 0 || page >= p.n_pages) return -1;
            return p.selected ? page : page * p.n_kv + at.pair / p.head_tiles;
        };
        int block = a < b ? look() : -1, stage = 0, round = 0;
        bool waits = early != 0;
        long long deadline = 0;
        for (int x = a; __any_sync(0xffffffffu, x < b);) {
            const unsigned slot = (unsigned)(lane * S::stages + stage);
            bool ready = x < b && !(waits && newest);
            if (ready && round > 0) ready = ai_bar_test(empty0 + 8u * slot, (unsigned)(round - 1) & 1u);
            if (ready) {
                filled[slot] = block >= 0;
                if (block >= 0) ai_fetch<D>(ai_smem(ai_ring) + slot * B::bytes, pool + (size_t)block * B::bytes, full0 + 8u * slot);
                else ai_bar_arrive(full0 + 8u * slot);
                if (++x < b) { ai_next(at, pairs, prefix); block = look(); }
                if (++stage == S::stages) { stage = 0; ++round; }
                deadline = 0;
            }
            if (!__any_sync(0xffffffffu, ready)) {
                if (waits) {
                    pdl_wait();
                    waits = false;
                } else if (!deadline) {
                    deadline = clock64() + AI_WAIT_CYCLES;
                } else if (clock64() > deadline && x < b) {
                    atomicExch(status, 23);
                    x = b;
                }
            }
        }
        if (waits) pdl_wait();
        if (blockIdx.x == 0) for (int i = lane; i <= p.n; i += 32) prefix_out[i] = prefix[i];
        return;
    }
    // ---- the warps that compute
    const int w = warp * gridDim.x + blockIdx.x;
    if (w >= workers) return;
    const int a = ai_begin(w, total, workers), b = ai_begin(w + 1, total, workers);
    if (a >= b) return;
    AiAt at = ai_find(a, pairs, p.n, prefix);
    if (early) pdl_wait();
    const float scale = scale_log2e * ai_pow2(-AI_DOWN);
    const int G = p.n_heads / p.n_kv;
    AiState<D> s;
    AiQuery<D> f;
    int tok = 0, kvh = 0, h0 = 0, pos = 0, lo = 0, from = 0, stage = 0;
    unsigned phase = 0;
    bool whole_begin = at.page == 0, first_pair = true;
    const auto enter = [&]() {
        p.heads_of(at.place, at.pair, tok, kvh, h0);
        pos = p.position(at.place);
        lo = p.first_seen(pos);
        from = lo / PE_PAGE;
        ai_reset(s);
        ai_query<D>(f, q + (size_t)tok * q_stride + (size_t)(kvh * G + h0 + g) * D, h0 + g < G, t);
    };
    const auto leave = [&](bool whole) {
        // the pair's sums: to the result where this warp had all of it, else to the warp's first or second place
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.sum[h] += __shfl_xor_sync(0xffffffffu, s.sum[h], o);
            const int head = 2 * t + h;
            float* to = partial + ((size_t)(w * 2 + (first_pair ? 0 : 1)) * 8 + head) * S::row;
            const float r = s.sum[h] == 0.f ? 0.f : 1.f / (s.sum[h] * ai_pow2(-AI_UP));
            if (!whole && g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(s.top[h], s.sum[h]);
#pragma unroll
            for (int gr = 0; gr < B::groups; ++gr) {
                const float mid = __shfl_sync(0xffffffffu, s.mids[h], gr * 4 + t) * ai_pow2(-AI_UP);
                const float4 v = make_float4(fmaf(s.acc[2 * gr][h], ai_pow2(-AI_DOWN), mid), fmaf(s.acc[2 * gr][2 + h], ai_pow2(-AI_DOWN), mid),
                                             fmaf(s.acc[2 * gr + 1][h], ai_pow2(-AI_DOWN), mid), fmaf(s.acc[2 * gr + 1][2 + h], ai_pow2(-AI_DOWN), mid));
                if (!whole) *reinterpret_cast<float4*>(to + 32 * gr + 4 * g) = v;
                else if (h0 + head < G)
                    *reinterpret_cast<uint2*>(out + ((size_t)tok * p.n_heads + kvh * G + h0 + head) * D + 32 * gr + 4 * g) = make_uint2(ai_pack(v.x * r, v.y * r), ai_pack(v.z * r, v.w * r));
            }
        }
        first_pair = false;
    };
    enter();
    for (int x = a;;) {
        const int slot = warp * S::stages + stage;
        if (!__all_sync(0xffffffffu, ai_bar_wait(full0 + 8u * slot, phase))) {
            if (lane == 0) atomicExch(status, 24);
            return;
        }
        const int key0 = (from + at.page) * PE_PAGE;
        if (filled[slot]) ai_block<D>(s, f, ai_ring + slot * B::bytes, lo - key0, pos - key0, scale, lane);
        __syncwarp();
        if (lane == 0) ai_bar_arrive(empty0 + 8u * slot);
        if (++stage == S::stages) { stage = 0; phase ^= 1u; }
        if (++x == b) break;
        if (ai_next(at, pairs, prefix)) {
            leave(whole_begin);
            whole_begin = true;
            enter();
        }
    }
    leave(whole_begin && at.page == at.pages - 1);
}

// 4 COLS columns of a pair's sums, left by the warps that had a part of it.  512 threads: four numbers of a head each, 64 / COLS of the warps' places at a time.  (Few pairs: eight, so that
// more blocks share the work: 64 pairs of heads of 128 on 16,000 positions 48 -> 40 us; many pairs: all columns of a block, 800 pairs 96 -> 86 us.)
template <int D, int COLS>
__global__ void __launch_bounds__(512) attention_int4_join_kernel(const AiPlaces p, const int* prefix, const float* partial, int most, bf16* out) {
    constexpr int row = AiStream<D>::row, cols = COLS, groups = 512 / (8 * cols);
    __shared__ float4 sums[groups][8][cols];
    __shared__ float2 tops[groups][8];
    pdl_launch_dependents();
    pdl_wait();
    const int pairs = p.pairs(), place = blockIdx.x / pairs, pair = blockIdx.x - place * pairs;
    const int before = prefix[place], pages = prefix[place + 1] - before, total = prefix[p.n] * pairs, begin = before * pairs + pair * pages, end = begin + pages;
    const int workers = ai_workers(total, most);
    const auto worker_of = [&](int x) { return (int)(((long long)(x + 1) * workers - 1) / total); };       // the last one that begins at x or before
    const int w0 = worker_of(begin), w1 = worker_of(end - 1);
    if (w0 == w1) return;
    int tok, kvh, h0;
    p.heads_of(place, pair, tok, kvh, h0);
    const int G = p.n_heads / p.n_kv, c0 = blockIdx.y * (4 * cols), c = threadIdx.x % cols, h = threadIdx.x / cols % 8, group = threadIdx.x / (8 * cols);
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = w0 + group; w <= w1; w += groups) {
        const float* src = partial + ((size_t)(w * 2 + (ai_begin(w, total, workers) >= begin ? 0 : 1)) * 8 + h) * row;
        const float2 ml = *reinterpret_cast<const float2*>(src + D);
        const float4 v = *reinterpret_cast<const float4*>(src + c0 + 4 * c);
        const float top = fmaxf(m, ml.x), x = l == 0.f ? 0.f : ai_ex2(m - top), y = ml.y == 0.f ? 0.f : ai_ex2(ml.x - top);
        o.x = fmaf(v.x, y, o.x * x); o.y = fmaf(v.y, y, o.y * x); o.z = fmaf(v.z, y, o.z * x); o.w = fmaf(v.w, y, o.w * x);
        l = fmaf(ml.y, y, l * x);
        m = top;
    }
    sums[group][h][c] = o;
    if (c == 0) tops[group][h] = make_float2(m, l);
    __syncthreads();
    if (group || h0 + h >= G) return;
    m = -INFINITY; l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < groups; ++i) m = fmaxf(m, tops[i][h].x);
#pragma unroll
    for (int i = 0; i < groups; ++i) {
        const float2 ml = tops[i][h];
        const float x = ml.y == 0.f ? 0.f : ai_ex2(ml.x - m);
        const float4 v = sums[i][h][c];
        o.x = fmaf(v.x, x, o.x); o.y = fmaf(v.y, x, o.y); o.z = fmaf(v.z, x, o.z); o.w = fmaf(v.w, x, o.w);
        l = fmaf(ml.y, x, l);
    }
    const float r = l == 0.f ? 0.f : 1.f / (l * ai_pow2(-AI_UP));
    *reinterpret_cast<uint2*>(out + ((size_t)tok * p.n_heads + kvh * G + h0 + h) * D + c0 + 4 * c) = make_uint2(ai_pack(o.x * r, o.y * r), ai_pack(o.z * r, o.w * r));
}

namespace {
// What a kernel needs to be told once a device.
inline int ai_allow(const void* kernel, int smem, bool (&done)[64], bool wide) {
    int dev = 0;
    PE_TRY(cudaGetDevice(&dev));
    if (wide && (dev >= 64 || !done[dev]) && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) cudaGetLastError();
    return pe_allow_smem(kernel, smem, done);
}

template <int D, int WARPS>
struct AiLaunch {
    using S = AiShape<D, WARPS>;
    static int allow() {
        static bool done[64] = {};
        return ai_allow((const void*)attention_int4_kernel<D, WARPS>, S::smem, done, true);
    }
    // clusters of so many CTAs (a power of two) that the GPU holds at once; asked once a device
    static int at_once(int splits) {
        static std::atomic<int> known[64][8];                  // one more than the number, 0: not asked yet
        int dev = 0, power = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return 0;
        while ((1 << power) < splits) ++power;
        if (dev < 64) { const int k = known[dev][power].load(std::memory_order_relaxed); if (k) return k - 1; }
        int n = 0;
        if (allow() == 0) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(splits, 1, 1024);
            cfg.blockDim = dim3(S::threads);
            cfg.dynamicSmemBytes = S::smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, attention_int4_kernel<D, WARPS>, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
        }
        if (dev < 64) known[dev][power].store(n + 1, std::memory_order_relaxed);
        return n;
    }
    // CTAs of a (token, key head, tile of heads): as many as run at once, each warp with a page at least.  (Large clusters find room for fewer than the occupancy says while
    // the next kernel's first CTAs wait on some SMs: 8 rows of 4,096 with 4 CTAs each 6.4 us, with 8 each, just as many as fit, 11.1.)
    static int splits(long long triples, int pages) {
        int n = 1;
        while (n < AI_MAX_SPLITS && n * WARPS < pages && at_once(2 * n) * (n >= 4 ? 4 : 5) >= triples * 5) n *= 2;
        return n;
    }
    static int go(const AiPlaces& p, int T, int pages, const bf16* q, int q_stride, const unsigned char* pool, float scale_log2e, int early, int* status, bf16* out, cudaStream_t stream) {
        { const int e = allow(); if (e) return e; }
        const int tiles = p.n_kv * p.head_tiles, n = splits((long long)tiles * T, pages);
        PE_TRY(pe_launch_cluster(attention_int4_kernel<D, WARPS>, dim3(n, tiles, T), dim3(S::threads), S::smem, stream, n, q, q_stride, pool, p.selected ? p.n_pages : p.n_pages * p.n_kv,
                                 p.block_table, p.table_stride, p.n_rows, p.tok_pos, p.tok_row, p.n_heads, p.n_kv, p.window, scale_log2e, p.selected, n, early, status, out));
        PE_LAUNCH_CHECK();
        return 0;
    }
};

template <int D>
struct AiStreamLaunch {
    using S = AiStream<D>;
    static int workers() { return pe_sm_count() * S::warps; }
    static long long scratch(int places) { return (long long)workers() * 2 * 8 * S::row * 4 + (places + 1) * 4ll; }
    static int go(const AiPlaces& p, const bf16* q, int q_stride, const unsigned char* pool, float scale_log2e, int early, void* scratch, int* status, bf16* out, cudaStream_t stream) {
        static bool done[64] = {};
        { const int e = ai_allow((const void*)attention_int4_stream_kernel<D>, S::ring + (AI_MAX_PLACES + 1) * 4, done, false); if (e) return e; }
        float* partial = (float*)scratch;
        int* prefix = (int*)(partial + (size_t)workers() * 2 * 8 * S::row);
        PE_TRY(pe_launch(attention_int4_stream_kernel<D>, dim3(pe_sm_count()), dim3(S::threads), S::ring + (size_t)(p.n + 1) * 4, stream, q, q_stride, pool, p, scale_log2e, early, workers(),
                         partial, prefix, status, out));
        PE_LAUNCH_CHECK();
        const unsigned pairs = (unsigned)(p.n * (p.selected ? p.head_tiles : p.n_kv * p.head_tiles));
        if (pairs <= 2u * (unsigned)pe_sm_count())
            PE_TRY(pe_launch(attention_int4_join_kernel<D, 8>, dim3(pairs, D / 32), dim3(512), 0, stream, p, prefix, partial, workers(), out));
        else
            PE_TRY(pe_launch(attention_int4_join_kernel<D, D / 4>, dim3(pairs), dim3(512), 0, stream, p, prefix, partial, workers(), out));
        PE_LAUNCH_CHECK();
        return 0;
    }
};
}  // namespace

// Whether a call's blocks are dealt to the warps in equal runs.
// Rows of any lengths: from 35,000 blocks on, the longest sequence's for every row (one CTA or cluster a pair / equal runs, us; 14 heads of 64 on 2: 64 rows of 20,000 to 32,700 72 / 65, 200 of
// up to 6,000 37 / 35, 32 of 4,000 to 8,192 16.6 / 22.7; 28 heads of 128 on 4: 200 of up to 6,000 94 / 86, 64 of 6,000 to 8,000 63.7 / 64.5, 16 of 8,000 to 16,000 37 / 40).
// Selected pages and windows are as many a row as the call says: one CTA a pair takes (16 + pages) units for each wave of as many pairs as SMs, equal runs 50 + 1.25 a block and SM (a unit is
// 0.23 us of 128 channels, 0.14 of 64).  28 heads of 128 on 4, us: 38 rows of 128 pages 65 / 48, 48 of 64 37.5 / 37.1, 64 of 64 39 / 44, 48 of 32 21 / 23; 256 rows of 14 heads of 64 on 2 with a
// window of 1,000 21.1 / 19.7.
static bool ai_streams(int T, int n_heads, int n_kv, int hd, int max_context, int selected, int window) {
    const long long places = selected ? (long long)T * n_kv : T, pairs = (long long)T * n_kv * ((n_heads / n_kv + 7) / 8), pages = (max_context - 1) / PE_PAGE + 1, sms = pe_sm_count();
    if (places > AI_MAX_PLACES || pairs * pages > 0x7fffffffll) return false;
    if (!selected && pairs * pages >= 35000) return true;
    return (selected || window > 0) && pairs > sms && 4 * ((pairs + sms - 1) / sms) * (16 + pages) * sms >= 200 * sms + 5 * pairs * pages;
}

// How a call's blocks are dealt out: 2 equal runs for all warps, 1 and 0 one CTA or cluster a pair.
// Form 1, seven warps, of which two CTAs share an SM, where pairs are few and each is cut over many CTAs (one row of 14 heads on 4,096 positions 4.5 us, with fifteen 5.6), but not where one
// CTA's warps have a page each (500 positions 3.6, with seven 3.9); else as many as the registers allow (64 rows of 1,000 to 2,000 7.3, with seven 8.9).
// The form goes by the bound of the positions that the call states: stated far too high it costs up to twice the time (64 rows of 1,000, 14 heads of 64 on 2, us: stated as 1,000 to 16,384
// 5.4, as 32,768 12.9).
static int ai_form(int T, int n_heads, int n_kv, int hd, int max_context, int selected, int window) {
    if (ai_streams(T, n_heads, n_kv, hd, max_context, selected, window)) return 2;
    return (long long)T * n_kv * ((n_heads / n_kv + 7) / 8) <= 8 && (max_context - 1) / PE_PAGE + 1 > (hd == 64 ? 15 : 11);
}

extern "C" void pe_set_pdl(int on) { pe_pdl_enabled() = on ? 1 : 0; }

// The form of a call; -1: sizes that no call takes.
extern "C" int pe_attention_int4_form(int T, int n_heads, int n_kv, int hd, int max_context, int selected, int window) {
    return T <= 0 || n_kv <= 0 || n_heads % n_kv || (hd != 64 && hd != 128) ? -1 : ai_form(T, n_heads, n_kv, hd, max_context, selected, window);
}

// Bytes of scratch that a call needs (0: none).
extern "C" long long pe_attention_int4_scratch(int T, int n_heads, int n_kv, int hd, int max_context, int selected, int window) {
    if (pe_attention_int4_form(T, n_heads, n_kv, hd, max_context, selected, window) != 2) return 0;
    const int places = selected ? T * n_kv : T;
    return hd == 64 ? AiStreamLaunch<64>::scratch(places) : AiStreamLaunch<128>::scratch(places);
}

extern "C" int pe_attention_int4(const void* q, int q_stride, void* out, const void* pool, long long n_blocks, const int* block_table, int table_stride, int n_rows,
                                 const int* tok_pos, const int* tok_row, int T, int n_heads, int n_kv, int hd, int window, float scale, int max_context, int selected,
                                 int early, void* scratch, int* status, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || max_context <= 0 || q_stride % 8 || table_stride < 1 || !status || T > 65535 || n_blocks > 0x7fffffffll ||
        !(scale > 0.f))
        return PE_ERR_UNSUPPORTED;
    if ((((uintptr_t)q | (uintptr_t)pool | (uintptr_t)scratch) & 15) || ((uintptr_t)out & 7)) return PE_ERR_UNSUPPORTED;
    const int head_tiles = (n_heads / n_kv + 7) / 8, pages = (max_context - 1) / PE_PAGE + 1;
    if ((long long)n_kv * head_tiles > 65535) return PE_ERR_UNSUPPORTED;
    early = early && !selected;
    const AiPlaces p = {tok_pos, tok_row, block_table, selected ? T * n_kv : T, table_stride, n_rows, (int)(selected ? n_blocks : n_blocks / n_kv), n_kv, n_heads, head_tiles, window, selected};
    const float scale_log2e = scale * 1.4426950408889634f;
    const int form = ai_form(T, n_heads, n_kv, hd, max_context, selected, window);
    if (scratch && form == 2 && (long long)T * n_kv * head_tiles * table_stride <= 0x7fffffffll) {
        const auto go = [&](auto v) {
            return decltype(v)::go(p, (const bf16*)q, q_stride, (const unsigned char*)pool, scale_log2e, early, scratch, status, (bf16*)out, (cudaStream_t)stream);
        };
        return hd == 64 ? go(AiStreamLaunch<64>()) : go(AiStreamLaunch<128>());
    }
    const auto go = [&](auto v) {
        return decltype(v)::go(p, T, pages, (const bf16*)q, q_stride, (const unsigned char*)pool, scale_log2e, early, status, (bf16*)out, (cudaStream_t)stream);
    };
    if (hd == 64) return form == 1 ? go(AiLaunch<64, 7>()) : go(AiLaunch<64, 15>());
    return form == 1 ? go(AiLaunch<128, 7>()) : go(AiLaunch<128, 11>());
}
