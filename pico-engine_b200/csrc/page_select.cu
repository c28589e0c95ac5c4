// The pages of a long context that a token's heads can score highest.
//
// A page j holds keys between lo_j and hi_j, channel by channel (page_bounds).  No key of it scores more against a query q than sum_d max(q_d lo_jd, q_d hi_jd), which is
// sum_d max(q_d, 0) hi_jd + min(q_d, 0) lo_jd.  The heads that share a key head read the same pages, so their bounds are added up: one vector of the sums of the positive
// parts and one of the negative parts against the page's two rows, 2 D multiply-adds a page whatever the number of heads.  Which pages are
// kept is defined by the sums in float64; a bound that is no number counts as the largest.
//
// One kernel scores in float32, a run of pages of a token and key head a block, and leaves every page's score with a bound of its error.  A second one has a block a token and
// head: it finds the last score that is kept by histograms of eight bits, from the first bit in which the scores differ.  Pages whose scores lie further from that one than
// twice the largest error are decided; the others (as a rule the one page of that score) are scored in float64 and chosen by those, of equal ones the earlier page.
// In float64 throughout, the first kernel took 28 us of 44 (48 tokens of 4 heads of 128 on 410 pages): conversions run at an eighth of the rate of multiply-adds.
#include "common.cuh"

#define PS_THREADS 256
#define PS_WARPS (PS_THREADS / 32)

// a float64 as 64 bits that compare like it; NaN above all
__device__ __forceinline__ unsigned long long ps_key(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);      // (-0 is 0)
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ unsigned ps_key(float v) { const unsigned u = __float_as_uint(v); return u >> 31 ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float ps_score(unsigned key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ float ps_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }       // (what is no number stays)

struct PsArgs {
    const bf16* q; const bf16* bounds; const int* block_table; const int* tok_pos; const int* tok_row;
    int q_stride, n_heads, n_kv, n_pages, table_stride, n_rows, keep, most;
    // a token's position (-1: it sees nothing), its pages, its own the last, and its row of the page table
    __device__ __forceinline__ int position(int tok) const {
        const int row = tok_row[tok];
        return row >= 0 && row < n_rows ? max(-1, min(tok_pos[tok], most * PE_PAGE - 1)) : -1;
    }
    __device__ __forceinline__ int pages(int pos) const { return pos < 0 ? 0 : pos / PE_PAGE + 1; }
    __device__ __forceinline__ const int* table(int tok) const { return block_table + (size_t)tok_row[tok] * table_stride; }
};

template <int D>
struct PsScore {
    static_assert(D == 64 || D == 128, "eight or sixteen lanes a page");
    static constexpr int lanes = D / 8, at_once = 32 / lanes, ahead = 4, pages = PS_WARPS * at_once * ahead;     // lanes a page, pages a warp at a time, and how often; pages a block
};

template <int D>
__global__ void __launch_bounds__(PS_THREADS) score_pages_kernel(const PsArgs p, float2* scores) {
    using S = PsScore<D>;
    __shared__ __align__(16) float sums[2][D];
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.y, tok = blockIdx.z, G = p.n_heads / p.n_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % S::lanes;
    const int pages = p.pages(p.position(tok)), first = 1 + (int)blockIdx.x * S::pages;
    if (pages <= p.keep || first >= pages - 1) return;         // (the first and the last page are kept whatever they score)
    const int* table = p.table(tok);
    uint4 v[S::ahead][2];
    int place[S::ahead];                                       // of the page's score, -1: none of this warp's
#pragma unroll
    for (int u = 0; u < S::ahead; ++u) {
        const int j = first + (u * PS_WARPS + warp) * S::at_once + lane / S::lanes, page = j < pages - 1 ? table[j] : -1;
        place[u] = page >= 0 && page < p.n_pages ? j : -1;
        const uint4* row = reinterpret_cast<const uint4*>(p.bounds + ((size_t)max(place[u] >= 0 ? page : 0, 0) * p.n_kv + kvh) * 2 * D) + l;
        v[u][0] = row[D / 8]; v[u][1] = row[0];
    }
    if (threadIdx.x < D) {
        float up = 0.f, down = 0.f;
        const bf16* q = p.q + (size_t)tok * p.q_stride + (size_t)kvh * G * D + threadIdx.x;
#pragma unroll 8
        for (int h = 0; h < G; ++h) {
            const float x = __bfloat162float(q[h * D]);
            up += x > 0.f || x != x ? x : 0.f;
            down += x < 0.f ? x : 0.f;
        }
        sums[0][threadIdx.x] = up; sums[1][threadIdx.x] = down;
    }
    __syncthreads();
    float by[2][8];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 four = *reinterpret_cast<const float4*>(&sums[side][8 * l + e]);
            by[side][e] = four.x; by[side][e + 1] = four.y; by[side][e + 2] = four.z; by[side][e + 3] = four.w;
        }
    // roundings: a head's sum, a product, the chain of a lane's sixteen and the lanes' tree: less than 24 + heads of 2^-24 of the terms' sizes; twice that
    const float unit = (float)(32 + G) * 1.1920929e-7f;
    float r[2 * S::ahead];                                     // scores, then their terms' sizes
#pragma unroll
    for (int u = 0; u < S::ahead; ++u) {
        float s = 0.f, size = 0.f;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const unsigned w[4] = {v[u][side].x, v[u][side].y, v[u][side].z, v[u][side].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float term = by[side][e] * __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
                s += term;
                size += fabsf(term);
            }
        }
        r[u] = s; r[S::ahead + u] = size;
    }
    // eight sums over the page's lanes: each exchange halves what a lane has, until it has one
#pragma unroll
    for (int n = S::ahead, o = 1; n; n >>= 1, o <<= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float give = l & o ? r[i] : r[n + i], have = l & o ? r[n + i] : r[i];
            r[i] = have + __shfl_xor_sync(0xffffffffu, give, o);
        }
#pragma unroll
    for (int o = 8; o < S::lanes; o <<= 1) r[0] += __shfl_xor_sync(0xffffffffu, r[0], o);
    // lane bits 0, 1, 2 have chosen size or score, then bits 1 and 0 of u
    const int mine = ((l >> 1) & 1) * 2 + ((l >> 2) & 1);
    int to = place[0];
#pragma unroll
    for (int u = 1; u < S::ahead; ++u) to = mine == u ? place[u] : to;
    if (l < 8 && to >= 0) {
        float* at = reinterpret_cast<float*>(scores + ((size_t)tok * p.n_kv + kvh) * p.most + to);
        if (l & 1) at[1] = r[0] * unit; else at[0] = r[0];
    }
}

// The `wanted`-th largest of the keys first .. last - 1 of shared memory (a key an element, `step` words apart): keys from `least` on are kept, of those equal to it the first `equal`
// (-1: all).  The whole block calls; bits: 32 or 64.
template <typename Key>
__device__ __forceinline__ void ps_cut(const Key* keys, int first, int last, int wanted, Key& least, int& equal, unsigned* hist, Key (*ends)[PS_WARPS], int* told) {
    constexpr int bits = 8 * (int)sizeof(Key);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Key low = ~(Key)0, high = 0;
    for (int j = first + threadIdx.x; j < last; j += PS_THREADS) { const Key k = keys[j]; low = min(low, k); high = max(high, k); }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { low = min(low, __shfl_xor_sync(0xffffffffu, low, o)); high = max(high, __shfl_xor_sync(0xffffffffu, high, o)); }
    if (lane == 0) { ends[0][warp] = low; ends[1][warp] = high; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PS_WARPS; ++w) { low = min(low, ends[0][w]); high = max(high, ends[1][w]); }
    least = low; equal = wanted;
    if (low == high) return;
    // keys agree from bit `top` on; the next eight bits at a time
    int top = bits == 64 ? 64 - __clzll((long long)(low ^ high)) : 32 - __clz((int)(low ^ high));
    Key prefix = top >= bits ? (Key)0 : high >> top << top;
    for (;;) {
        const int width = min(top, 8), shift = top - width;
        for (int i = threadIdx.x; i < 256; i += PS_THREADS) hist[i] = 0u;
        __syncthreads();
        for (int j = first + threadIdx.x; j < last; j += PS_THREADS) {
            const Key k = keys[j];
            if (top >= bits || (k ^ prefix) >> top == 0) atomicAdd(&hist[(unsigned)(k >> shift) & ((1u << width) - 1u)], 1u);
        }
        __syncthreads();
        if (warp == 0) {
            // eight bins a lane, the highest first: the bin in which the wanted-th lies
            int n = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) n += (int)hist[255 - 8 * lane - i];
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
            if (upto >= wanted && upto - n < wanted) {
                int above = upto - n, i = 0;
                while (above + (int)hist[255 - 8 * lane - i] < wanted) above += (int)hist[255 - 8 * lane - i++];
                told[0] = 255 - 8 * lane - i; told[1] = above; told[2] = (int)hist[255 - 8 * lane - i];
            }
        }
        __syncthreads();
        prefix |= (Key)told[0] << shift;
        wanted -= told[1];
        least = prefix;
        if (told[2] == wanted) { equal = -1; return; }         // all of the bin
        if (shift == 0) { equal = wanted; return; }
        top = shift;
        __syncthreads();                                       // (told and the histogram have been read)
    }
}

template <int D>
__global__ void __launch_bounds__(PS_THREADS) select_pages_kernel(const PsArgs p, const float2* all_scores, int* out_table, int* out_pos) {
    extern __shared__ unsigned long long ps_exact[];           // [most] keys of float64 scores, where some are needed; [most] keys of the scores; [most] entries of the page table; [most] pages to score again
    unsigned* keys = reinterpret_cast<unsigned*>(ps_exact + p.most);
    int* entries = reinterpret_cast<int*>(keys + p.most);
    __shared__ int parts[2][PS_WARPS], told[3];
    __shared__ unsigned hist[256], ends[2][PS_WARPS];
    __shared__ unsigned long long ends64[2][PS_WARPS];
    __shared__ float errors[PS_WARPS];
    __shared__ double sums[2][D];
    __shared__ int n_listed;
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.x, tok = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_kv = p.n_kv, keep = p.keep;
    const int pos = p.position(tok), pages = p.pages(pos);
    const bool choose = pages > keep && keep > 2;
    const int wanted = keep - 2;                               // besides the first and the last page
    if (pages) {
        const int* table = p.table(tok);
        const float2* scores = all_scores + ((size_t)tok * n_kv + kvh) * p.most;
        float error = 0.f;
        for (int j = threadIdx.x; j < pages; j += PS_THREADS) {
            const int page = table[j];
            entries[j] = page < p.n_pages ? page : -1;
            if (choose && j > 0 && j < pages - 1) {
                const bool there = page >= 0 && page < p.n_pages;
                const float2 s = there ? scores[j] : make_float2(-INFINITY, 0.f);
                keys[j] = there ? (s.x != s.x ? ~0u : ps_key(s.x)) : 0u;
                error = ps_max(error, s.y);
            }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) error = ps_max(error, __shfl_xor_sync(0xffffffffu, error, o));
        if (lane == 0) errors[warp] = error;
    }
    __syncthreads();
    // kept: keys above `over`; of those from `under` on that are not, `left` by their float64 scores
    unsigned over = 0u, under = 0u;
    unsigned long long least = 0ull;
    int equal = -1;
    bool refine = false;
    if (choose) {
        unsigned cut;
        int same;
        ps_cut<unsigned>(keys, 1, pages - 1, wanted, cut, same, hist, ends, told);
        float error = 0.f;
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) error = ps_max(error, errors[w]);
        // the score of the last one kept (the least key from `cut` on)
        unsigned last = ~0u;
        for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) if (keys[j] >= cut) last = min(last, keys[j]);
        last = __reduce_min_sync(0xffffffffu, last);
        __syncthreads();
        if (lane == 0) ends[0][warp] = last;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) last = min(last, ends[0][w]);
        const float score = ps_score(last), reach = 2.1f * error;
        const float high = score + reach, low = score - reach;
        const bool none = last == 0u;                          // pages that are not there are among the kept: in the order of the positions
        over = none ? 0u : high == high ? ps_key(high) : ~0u;
        under = none ? 0u : low == low ? ps_key(low) : 1u;
        int n_over = 0, n_near = 0;
        for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) { n_over += keys[j] > over; n_near += keys[j] >= under && keys[j] <= over; }
        n_over = __reduce_add_sync(0xffffffffu, n_over); n_near = __reduce_add_sync(0xffffffffu, n_near);
        if (lane == 0) { parts[0][warp] = n_over; parts[1][warp] = n_near; }
        __syncthreads();
        n_over = n_near = 0;
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) { n_over += parts[0][w]; n_near += parts[1][w]; }
        refine = n_over + n_near != wanted;
        if (refine) {
            // the pages that are near, and the queries' sums
            unsigned* list = reinterpret_cast<unsigned*>(entries + p.most);
            if (threadIdx.x == 0) n_listed = 0;
            if (threadIdx.x < D) {
                const int G = p.n_heads / n_kv;
                const bf16* q = p.q + (size_t)tok * p.q_stride + (size_t)kvh * G * D + threadIdx.x;
                double up = 0.0, down = 0.0;
#pragma unroll 8
                for (int h = 0; h < G; ++h) {
                    const float x = __bfloat162float(q[h * D]);
                    up += x > 0.f || x != x ? x : 0.f;
                    down += x < 0.f ? x : 0.f;
                }
                sums[0][threadIdx.x] = up; sums[1][threadIdx.x] = down;
            }
            __syncthreads();
            for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) {
                ps_exact[j] = keys[j] > over ? ~0ull : 0ull;   // (decided ones beside the others)
                if (keys[j] >= under && keys[j] <= over && entries[j] >= 0) list[atomicAdd(&n_listed, 1)] = j;
            }
            __syncthreads();
            for (int x = warp; x < n_listed; x += PS_WARPS) {
                const int j = list[x];
                const bf16* lo = p.bounds + ((size_t)entries[j] * n_kv + kvh) * 2 * D;
                double s = 0.0;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    s = fma(sums[0][32 * i + lane], (double)__bfloat162float(lo[D + 32 * i + lane]), s);
                    s = fma(sums[1][32 * i + lane], (double)__bfloat162float(lo[32 * i + lane]), s);
                }
                s = warp_sum_d(s);
                // (below the decided ones and above the pages that are not there)
                if (lane == 0) ps_exact[j] = min(max(ps_key(s), 1ull), ~0ull - 1);
            }
            __syncthreads();
            ps_cut<unsigned long long>(ps_exact, 1, pages - 1, wanted, least, equal, hist, ends64, told);
        }
    }
    // the kept pages in the order of the positions
    int* mine = out_table + ((size_t)tok * n_kv + kvh) * keep;
    int done = 0, ties = 0;
    for (int base = 0; base < pages; base += PS_THREADS) {
        const int j = base + threadIdx.x;
        bool kept = j < pages && (pages <= keep || j == pages - 1 || (j == 0 && keep > 1)), tie = false;
        if (choose && j > 0 && j < pages - 1) {
            if (refine) { kept = ps_exact[j] > least || (equal < 0 && ps_exact[j] == least); tie = equal >= 0 && ps_exact[j] == least; }
            else kept = keys[j] >= under;
        }
        if (refine && equal >= 0) {                            // (the same for the whole block)
            const unsigned set = __ballot_sync(0xffffffffu, tie);
            __syncthreads();
            if (lane == 0) parts[0][warp] = __popc(set);
            __syncthreads();
            int at = ties + __popc(set & ((1u << lane) - 1u));
#pragma unroll
            for (int w = 0; w < PS_WARPS; ++w) { if (w < warp) at += parts[0][w]; ties += parts[0][w]; }
            kept |= tie && at < equal;
        }
        const unsigned set = __ballot_sync(0xffffffffu, kept);
        __syncthreads();
        if (lane == 0) parts[1][warp] = __popc(set);
        __syncthreads();
        int at = done + __popc(set & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) { if (w < warp) at += parts[1][w]; done += parts[1][w]; }
        if (kept) mine[at] = entries[j] >= 0 ? entries[j] * n_kv + kvh : -1;
    }
    for (int i = done + threadIdx.x; i < keep; i += PS_THREADS) mine[i] = -1;
    if (threadIdx.x == 0) out_pos[tok * n_kv + kvh] = done ? (done - 1) * PE_PAGE + pos % PE_PAGE : -1;
}

static int ps_most(int max_context, int table_stride) { const int pages = (max_context - 1) / PE_PAGE + 1; return pages < table_stride ? pages : table_stride; }

// Bytes of scratch: a score and its error a page of every token and head.
extern "C" long long pe_select_pages_scratch(int T, int n_kv, int table_stride, int max_context) { return (long long)T * n_kv * ps_most(max_context, table_stride) * 8; }

extern "C" int pe_select_pages(const void* q, int q_stride, int T, int n_heads, int n_kv, int hd, const void* bounds, long long n_pages, const int* block_table,
                               int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep, int max_context, int* out_table, int* out_pos, void* scratch, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_kv > 65535 || T > 65535 || n_heads % n_kv || keep < 1 || max_context < 1 || n_rows < 1 || table_stride < 1 || n_pages * n_kv > 0x7fffffffll)
        return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)bounds) & 15) return PE_ERR_UNSUPPORTED;
    const int most = ps_most(max_context, table_stride);
    const size_t smem = (size_t)most * 20;
    if (smem > 200 * 1024 || ((uintptr_t)scratch & 7) || !scratch) return PE_ERR_UNSUPPORTED;
    const PsArgs p = {(const bf16*)q, (const bf16*)bounds, block_table, tok_pos, tok_row, q_stride, n_heads, n_kv, (int)n_pages, table_stride, n_rows, keep, most};
    float2* scores = (float2*)scratch;
    auto kernel = hd == 64 ? select_pages_kernel<64> : select_pages_kernel<128>;
    const int per = hd == 64 ? PsScore<64>::pages : PsScore<128>::pages;
    if (most > keep && keep > 2) {                                                                    // (else every token has all of its pages)
        PE_TRY(pe_launch(hd == 64 ? score_pages_kernel<64> : score_pages_kernel<128>, dim3((unsigned)((most + per - 1) / per), (unsigned)n_kv, (unsigned)T),
                         dim3(PS_THREADS), 0, (cudaStream_t)stream, p, scores));
        PE_LAUNCH_CHECK();
    }
    if (smem > 40 * 1024) PE_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    PE_TRY(pe_launch(kernel, dim3((unsigned)n_kv, (unsigned)T), dim3(PS_THREADS), smem, (cudaStream_t)stream, p, (const float2*)scores, out_table, out_pos));
    PE_LAUNCH_CHECK();
    return 0;
}
