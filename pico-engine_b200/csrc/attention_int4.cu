// Attention of single tokens over the paged cache of 4-bit keys and values (int4_pages.cuh).
#include "int4_pages.cuh"
#include <map>
#include <mutex>
#include <utility>

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
    unsigned sums;                                             // of the groups: 2^-65 (sum of q) in two parts, for the product with the middles
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
    // as the product's operand: rows 2 t and 2 t + 1, first the high parts of the groups, then the low ones
    const int pair = D == 128 ? (t & 1) : 0;
    const bool low = D == 128 ? t >= 2 : t == 1, none = D == 64 && t >= 2;
    float a = pair ? sum[NB > 2 ? 2 : 0] : sum[0], b = pair ? sum[NB > 2 ? 3 : 1] : sum[1];
    if (low) { a -= __bfloat162float(__float2bfloat16_rn(a)); b -= __bfloat162float(__float2bfloat16_rn(b)); }
    f.sums = none ? 0u : ai_pack(a, b);
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
        ai_mma8(sc[j], mid[0], mid[1], f.sums);
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
        uint2 mids = make_uint2(0u, 0u);
        if (g < NB) mids = *reinterpret_cast<const uint2*>(vm + (NB + g) * 32);
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
// true when the phase with this parity has completed; false when the wait ran out
__device__ __forceinline__ bool ai_bar_wait(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
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

// Warps of a CTA, blocks that a warp has places for, CTAs an SM.
template <int D>
struct AiShape {
    static constexpr int warps = 4, stages = 2, ctas = D == 64 ? 4 : 2;
    static constexpr int row = D + 4;                          // floats of a head's results: D sums, largest score, sum of weights
    static constexpr int blocks = warps * stages * Int4Block<D>::bytes, parts = warps * 8 * row * 4;
    static constexpr int ring = ((blocks > parts ? blocks : parts) + 127) / 128 * 128;    // the warps' results lie in the ring later
    static constexpr int gather = AI_MAX_SPLITS * 8 * 4 * 4 + 8 * D * 4;
    static constexpr int smem = ring + gather;
};

template <int D>
__global__ void __launch_bounds__(32 * AiShape<D>::warps, AiShape<D>::ctas) attention_int4_kernel(
    const bf16* q, int q_stride, const unsigned char* pool, int n_blocks, const int* block_table, int table_stride, int n_rows, const int* tok_pos, const int* tok_row,
    int n_heads, int n_kv, int window, float scale_log2e, int selected, int n_splits, int early, int* status, bf16* out) {
    using S = AiShape<D>;
    using B = Int4Block<D>;
    constexpr int WARPS = S::warps;
    extern __shared__ __align__(128) unsigned char ai_ring[];   // [warp][stage] blocks; later the warps' results; behind it what the other CTAs send
    __shared__ __align__(8) unsigned long long bars[WARPS * S::stages + 1];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = n_splits > 1 ? (int)ai_cluster_rank() : 0, slice = D / n_splits;
    float* gather = reinterpret_cast<float*>(ai_ring + S::ring);                          // [split][8][slice + 4]
    const unsigned gather0 = ai_smem(gather), gbar = ai_smem(&bars[WARPS * S::stages]);
    const int G = n_heads / n_kv, head_tiles = (G + 7) / 8, kvh = blockIdx.y / head_tiles, h0 = (blockIdx.y % head_tiles) * 8, heads = min(8, G - h0);
    const unsigned ring0 = ai_smem(ai_ring) + warp * S::stages * Int4Block<D>::bytes, full0 = ai_smem(&bars[warp * S::stages]);
    if (lane == 0) {
        for (int i = 0; i < S::stages; ++i) ai_bar_init(full0 + 8u * i, 1u);
        if (warp == 0) ai_bar_init(gbar, 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (warp == 0 && n_splits > 1) ai_bar_expect(gbar, (unsigned)((n_splits - 1) * heads * (slice + 4) * 4));
    }
    __syncwarp();
    if (n_splits > 1) ai_cluster_arrive();                     // waited for before the first number goes to another CTA
    if (!early) pdl_wait();
    const int tok = blockIdx.z, place = selected ? tok * n_kv + kvh : tok, pos = min(tok_pos[place], table_stride * PE_PAGE - 1), row = selected ? place : tok_row[tok];
    const int lo = window > 0 ? max(0, pos - window + 1) : 0, first = lo / PE_PAGE + split * WARPS + warp, step = n_splits * WARPS;
    const int last = pos >= 0 && row >= 0 && row < n_rows ? pos / PE_PAGE : -1;
    const int n = last >= first ? (last - first) / step + 1 : 0;                          // pages of this warp: first, first + step, ..
    // the entries of the table for this warp's pages base + lane and base + 32 + lane, as blocks (-1: not there)
    const int n_pages = selected ? n_blocks : n_blocks / n_kv;
    const int* table = block_table + (size_t)max(0, min(row, n_rows - 1)) * table_stride;
    const auto entry = [&](int i) {
        if (i >= n) return -1;
        const int page = table[first + i * step];
        if (page < 0 || page >= n_pages) return -1;
        return selected ? page : page * n_kv + kvh;
    };
    int now = entry(lane), next = entry(32 + lane);
    int base = 0;
    const auto block_of = [&](int i) { return __shfl_sync(0xffffffffu, i - base < 32 ? now : next, (i - base) & 31); };
    const auto fetch = [&](int i, int stage) {
        if (i >= n) return;
        const int at = block_of(i);
        if (at >= 0 && lane == 0) ai_fetch<D>(ring0 + stage * B::bytes, pool + (size_t)at * B::bytes, full0 + 8u * stage);
    };
    // (early: the page of the newest position is written by the kernel before this one)
    const int settled = n - (early && n > 0 && first + (n - 1) * step == last);
    int fetched = 0;
    for (; fetched < min(settled, S::stages); ++fetched) fetch(fetched, fetched);
    if (early) {
        pdl_wait();
        for (; fetched < min(n, S::stages); ++fetched) fetch(fetched, fetched);
    }
    AiState<D> s;
    ai_reset(s);
    AiQuery<D> f;
    ai_query<D>(f, q + (size_t)tok * q_stride + (size_t)(kvh * G + h0 + g) * D, h0 + g < G, t);
    const float scale = scale_log2e * ai_pow2(-AI_DOWN);
    unsigned phases = 0;
    bool dead = false;
    for (int i = 0, stage = 0; i < n; ++i) {
        if (i - base == 32) { base += 32; now = next; next = entry(base + 32 + lane); }
        if (block_of(i) >= 0) {
            if (!dead && !__all_sync(0xffffffffu, ai_bar_wait(full0 + 8u * stage, (phases >> stage) & 1u))) {
                dead = true;
                if (lane == 0) atomicExch(status, 21);
            }
            phases ^= 1u << stage;
            const int at = (first + i * step) * PE_PAGE;
            if (!dead) ai_block<D>(s, f, ai_ring + (warp * S::stages + stage) * B::bytes, lo - at, pos - at, scale, lane);
        }
        __syncwarp();
        if (!dead) fetch(i + S::stages, stage);
        if (++stage == S::stages) stage = 0;
    }

    // ---- the warps' results, joined in shared memory (the ring is free once every warp has left its loop)
    __syncthreads();
    float* part = reinterpret_cast<float*>(ai_ring);           // [warp][8][row]
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
    __syncthreads();
    if (n_splits > 1) ai_cluster_wait();
    for (int i = threadIdx.x; i < heads * (D / 4); i += 32 * WARPS) {
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
    for (int i = threadIdx.x; i < heads * (slice / 4); i += 32 * WARPS) {
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

namespace {
template <int D>
struct AiLaunch {
    using S = AiShape<D>;
    static int allow() {
        static bool done[64] = {};
        int dev = 0;
        PE_TRY(cudaGetDevice(&dev));
        if (dev < 64 && done[dev]) return 0;
        PE_TRY(cudaFuncSetAttribute(attention_int4_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem));
        if (cudaFuncSetAttribute(attention_int4_kernel<D>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) cudaGetLastError();
        if (dev < 64) done[dev] = true;
        return 0;
    }
    // clusters of so many CTAs that the GPU holds at once
    static int at_once(int splits) {
        static std::mutex lock;
        static std::map<std::pair<int, int>, int> known;
        std::lock_guard<std::mutex> hold(lock);
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return 0;
        auto it = known.find({dev, splits});
        if (it != known.end()) return it->second;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(splits, 1, 1024);
        cfg.blockDim = dim3(32 * S::warps);
        cfg.dynamicSmemBytes = S::smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, attention_int4_kernel<D>, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
        known[{dev, splits}] = n;
        return n;
    }
    // CTAs of a (token, key head, tile of heads): as many as run at once, each warp with a page at least
    static int splits(long long triples, int units) {
        int n = 1;
        while (n < AI_MAX_SPLITS && n * S::warps < units && at_once(2 * n) >= triples) n *= 2;
        return n;
    }
    static int go(int n_splits, unsigned tokens, unsigned tiles_y, cudaStream_t stream, const bf16* q, int q_stride, const unsigned char* pool, int n_blocks,
                  const int* block_table, int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int n_heads, int n_kv, int window, float scale, int selected,
                  int early, int* status, bf16* out) {
        { const int e = allow(); if (e) return e; }
        PE_TRY(pe_launch_cluster(attention_int4_kernel<D>, dim3(n_splits, tiles_y, tokens), dim3(32 * S::warps), S::smem, stream, n_splits, q, q_stride, pool,
                                 n_blocks, block_table, table_stride, n_rows, tok_pos, tok_row, n_heads, n_kv, window, scale * 1.4426950408889634f, selected, n_splits, early,
                                 status, out));
        PE_LAUNCH_CHECK();
        return 0;
    }
};
}  // namespace

extern "C" void pe_set_pdl(int on) { pe_pdl_enabled() = on ? 1 : 0; }

extern "C" int pe_attention_int4(const void* q, int q_stride, void* out, const void* pool, long long n_blocks, const int* block_table, int table_stride, int n_rows,
                                 const int* tok_pos, const int* tok_row, int T, int n_heads, int n_kv, int hd, int window, float scale, int max_context, int selected,
                                 int early, int* status, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || max_context <= 0 || q_stride % 8 || table_stride < 1 || !status || T > 65535 || n_blocks > 0x7fffffffll || !(scale > 0.f)) return PE_ERR_UNSUPPORTED;
    if ((((uintptr_t)q | (uintptr_t)pool) & 15) || ((uintptr_t)out & 7)) return PE_ERR_UNSUPPORTED;
    const int head_tiles = (n_heads / n_kv + 7) / 8;
    const long long tiles = (long long)n_kv * head_tiles;
    if (tiles > 65535) return PE_ERR_UNSUPPORTED;
    early = early && !selected;
    const int units = ((max_context - 1) / PE_PAGE + 1);
    const auto go = [&](auto v) {
        using L = decltype(v);
        { const int e = L::allow(); if (e) return e; }
        return L::go(L::splits(tiles * T, units), (unsigned)T, (unsigned)tiles, (cudaStream_t)stream, (const bf16*)q, q_stride, (const unsigned char*)pool, (int)n_blocks, block_table,
                     table_stride, n_rows, tok_pos, tok_row, n_heads, n_kv, window, scale, selected, early, status, (bf16*)out);
    };
    return hd == 64 ? go(AiLaunch<64>()) : go(AiLaunch<128>());
}
