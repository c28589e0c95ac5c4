// Attention of single tokens over the paged cache of 4-bit keys and values (int4_pages.cuh).
#include "int4_pages.cuh"

#define AI_WARPS 4
#define AI_WAIT_CYCLES 2000000000ll                            // about a second of SM clock

__device__ __forceinline__ float ai_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned ai_pack(float lo, float hi) { __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ unsigned ai_transpose(unsigned a) { unsigned d; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a)); return d; }
__device__ __forceinline__ unsigned ai_times(unsigned a, unsigned b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void ai_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ai_mma8(float (&c)[4], unsigned a0, unsigned a1, unsigned b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b0));
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

// One block (64 positions of a head) against the warp's eight heads.  lo <= position <= hi are seen (block positions).
template <int D>
__device__ __forceinline__ void ai_block(AiState<D>& s, const AiQuery<D>& f, const unsigned char* block, int lo, int hi, float scale, int g, int t) {
    using B = Int4Block<D>;
    constexpr int NB = B::groups;
    float sc[4][4];
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
        sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
        ai_mma8(sc[j], mid[0], mid[1], f.sums);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            ai_mma(c, q4_pair(words[0][b], 0), q4_pair(words[1][b], 0), q4_pair(words[0][b], 1), q4_pair(words[1][b], 1), f.q[2 * b][0], f.q[2 * b][1]);
            ai_mma(c, q4_pair(words[0][b], 2), q4_pair(words[1][b], 2), q4_pair(words[0][b], 3), q4_pair(words[1][b], 3), f.q[2 * b + 1][0], f.q[2 * b + 1][1]);
            const float s0 = __uint_as_float((b & 1) ? steps[0][b >> 1] & 0xffff0000u : steps[0][b >> 1] << 16);
            const float s1 = __uint_as_float((b & 1) ? steps[1][b >> 1] & 0xffff0000u : steps[1][b >> 1] << 16);
            sc[j][0] = fmaf(c[0], s0, sc[j][0]); sc[j][1] = fmaf(c[1], s0, sc[j][1]);
            sc[j][2] = fmaf(c[2], s1, sc[j][2]); sc[j][3] = fmaf(c[3], s1, sc[j][3]);
        }
    }
    const bool edge = lo > 0 || hi < PE_PAGE - 1;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = 16 * j + 8 * (e >> 1) + g;
            sc[j][e] *= scale;
            if (edge && (p < lo || p > hi)) sc[j][e] = -INFINITY;
            top[e & 1] = fmaxf(top[e & 1], sc[j][e]);
        }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    float ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float m = fmaxf(s.top[h], top[h]);
        const float alpha = m == -INFINITY ? 1.f : ai_ex2(s.top[h] - m);
        s.top[h] = m;
        ref[h] = m == -INFINITY ? 0.f : AI_UP - m;
        s.sum[h] *= alpha;
#pragma unroll
        for (int m2 = 0; m2 < D / 16; ++m2) { s.acc[m2][h] *= alpha; s.acc[m2][2 + h] *= alpha; }
        s.mids[h] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { w[e] = ai_ex2(sc[j][e] + ref[e & 1]); s.sum[e & 1] += w[e]; }
        const unsigned p0 = ai_transpose(ai_pack(w[0], w[1])), p1 = ai_transpose(ai_pack(w[2], w[3]));     // positions 16 j + 2 t, + 1; 16 j + 8 + 2 t, + 1; head g
        // positions that are not seen may hold anything: their steps and middles are taken as zero
        unsigned m0 = ~0u, m1 = ~0u;
        if (edge) {
            const int p = 16 * j + 2 * t;
            m0 = (p >= lo && p <= hi ? 0xffffu : 0u) | (p + 1 >= lo && p + 1 <= hi ? 0xffff0000u : 0u);
            m1 = (p + 8 >= lo && p + 8 <= hi ? 0xffffu : 0u) | (p + 9 >= lo && p + 9 <= hi ? 0xffff0000u : 0u);
        }
        const unsigned char* vm = block + B::value_meta + j * (4 * NB * 16) + t * 8;
        uint2 mids = make_uint2(0u, 0u);
        if (g < NB) mids = *reinterpret_cast<const uint2*>(vm + (NB + g) * 32);
        ai_mma(s.mids, mids.x & m0, 0u, mids.y & m1, 0u, p0, p1);
#pragma unroll
        for (int h = 0; h < B::halves; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(block + q4_value_words<D>(j, h, g, t));
            const unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint2 st = *reinterpret_cast<const uint2*>(vm + (2 * h + b) * 32);
                const unsigned q0 = ai_times(p0, st.x & m0), q1 = ai_times(p1, st.y & m1);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const unsigned w = words[2 * b + m];
                    ai_mma(s.acc[4 * h + 2 * b + m], q4_pair(w, 0), q4_pair(w, 1), q4_pair(w, 2), q4_pair(w, 3), q0, q1);
                }
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(32 * AI_WARPS) attention_int4_kernel(const bf16* q, int q_stride, const unsigned char* pool, long long n_blocks, const int* block_table,
                                                                       int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int n_heads, int n_kv, int window,
                                                                       float scale_log2e, int selected, const int4* tiles, bf16* out) {
    constexpr int ROW = D + 4;
    __shared__ float part[AI_WARPS][8][ROW];
    __shared__ float tops[AI_WARPS][8], sums[AI_WARPS][8];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int G = n_heads / n_kv, head_tiles = (G + 7) / 8, kvh = blockIdx.y / head_tiles, h0 = (blockIdx.y % head_tiles) * 8;
    int tok = blockIdx.x, pos, row;
    if (tiles) {                                               // a run of tokens: row, first token, tokens, position
        const int4 r = tiles[tok >> 7];
        const int i = tok & 127;
        if (i >= r.z) return;
        tok = r.y + i; pos = r.w + i; row = r.x;
    } else {
        const int place = selected ? tok * n_kv + kvh : tok;
        pos = tok_pos[place]; row = selected ? place : tok_row[tok];
    }
    pos = min(pos, table_stride * PE_PAGE - 1);
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    AiState<D> s;
#pragma unroll
    for (int m = 0; m < D / 16; ++m) s.acc[m][0] = s.acc[m][1] = s.acc[m][2] = s.acc[m][3] = 0.f;
    s.mids[0] = s.mids[1] = s.mids[2] = s.mids[3] = 0.f;
    s.top[0] = s.top[1] = -INFINITY;
    s.sum[0] = s.sum[1] = 0.f;
    AiQuery<D> f;
    ai_query<D>(f, q + (size_t)tok * q_stride + (size_t)(kvh * G + h0 + g) * D, h0 + g < G, t);
    if (pos >= 0 && row >= 0 && row < n_rows) {
        const int* table = block_table + (size_t)row * table_stride;
        for (int j = lo / PE_PAGE + warp; j <= pos / PE_PAGE; j += AI_WARPS) {
            const int page = table[j];
            const long long at = selected ? page : (long long)page * n_kv + kvh;
            if (page < 0 || at >= n_blocks) continue;
            ai_block<D>(s, f, pool + (size_t)at * Int4Block<D>::bytes, lo - j * PE_PAGE, pos - j * PE_PAGE, scale_log2e * ai_pow2(-AI_DOWN), g, t);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) s.sum[h] += __shfl_xor_sync(0xffffffffu, s.sum[h], o);
        if (g == 0) { tops[warp][2 * t + h] = s.top[h]; sums[warp][2 * t + h] = s.sum[h]; }
    }
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float mid = __shfl_sync(0xffffffffu, s.mids[h], (m >> 1) * 4 + t);
            float* to = &part[warp][2 * t + h][32 * (m >> 1) + 4 * g + 2 * (m & 1)];
            to[0] = fmaf(s.acc[m][h], ai_pow2(-AI_DOWN), mid * ai_pow2(-AI_UP));
            to[1] = fmaf(s.acc[m][2 + h], ai_pow2(-AI_DOWN), mid * ai_pow2(-AI_UP));
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * D; i += 32 * AI_WARPS) {
        const int h = i / D, d = i % D;
        if (h0 + h >= G) break;
        float m = -INFINITY, o = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < AI_WARPS; ++w) m = fmaxf(m, tops[w][h]);
#pragma unroll
        for (int w = 0; w < AI_WARPS; ++w) {
            const float x = tops[w][h] == -INFINITY && sums[w][h] == 0.f ? 0.f : ai_ex2(tops[w][h] - m);
            o = fmaf(part[w][h][d], x, o);
            l = fmaf(sums[w][h], x, l);
        }
        out[((size_t)tok * n_heads + kvh * G + h0 + h) * D + d] = __float2bfloat16_rn(l == 0.f ? 0.f : o / (l * ai_pow2(-AI_UP)));
    }
}

extern "C" void pe_set_pdl(int on) { pe_pdl_enabled() = on ? 1 : 0; }

extern "C" int pe_attention_int4(const void* q, int q_stride, void* out, const void* pool, long long n_blocks, const int* block_table, int table_stride, int n_rows,
                                 const int* tok_pos, const int* tok_row, int T, int n_heads, int n_kv, int hd, int window, float scale, int max_context, int selected,
                                 int* status, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || max_context <= 0 || q_stride % 8 || table_stride < 1 || !status) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)pool) & 15) return PE_ERR_UNSUPPORTED;
    const long long tiles = (long long)n_kv * ((n_heads / n_kv + 7) / 8);
    if (tiles > 65535) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? attention_int4_kernel<64> : attention_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)T, (unsigned)tiles), dim3(32 * AI_WARPS), 0, (cudaStream_t)stream, (const bf16*)q, q_stride, (const unsigned char*)pool, n_blocks,
                     block_table, table_stride, n_rows, tok_pos, tok_row, n_heads, n_kv, window, scale * 1.4426950408889634f, selected, (const int4*)nullptr, (bf16*)out));
    PE_LAUNCH_CHECK();
    return 0;
}

extern "C" int pe_attention_int4_prompt(const void* q, int q_stride, void* out, const void* pool, long long n_blocks, const int* block_table, int table_stride, int n_rows,
                                        const int* tiles, int n_tiles, int n_tokens, int n_heads, int n_kv, int hd, int window, float scale, int* status, void* stream) {
    if (n_tiles <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || q_stride % 8 || table_stride < 1 || !status) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)tiles) & 15) return PE_ERR_UNSUPPORTED;
    const long long head_tiles = (long long)n_kv * ((n_heads / n_kv + 7) / 8);
    if (head_tiles > 65535) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? attention_int4_kernel<64> : attention_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)n_tiles * 128u, (unsigned)head_tiles), dim3(32 * AI_WARPS), 0, (cudaStream_t)stream, (const bf16*)q, q_stride,
                     (const unsigned char*)pool, n_blocks, block_table, table_stride, n_rows, (const int*)nullptr, (const int*)nullptr, n_heads, n_kv, window,
                     scale * 1.4426950408889634f, 0, (const int4*)tiles, (bf16*)out));
    PE_LAUNCH_CHECK();
    return 0;
}
