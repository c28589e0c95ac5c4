// The pages of a long context that a token's heads can score highest.
//
// A page j holds keys between lo_j and hi_j, channel by channel (page_bounds).  But for their rounding to bfloat16 (2^-9 of them), no key of it scores more against a query q than
// sum_d max(q_d lo_jd, q_d hi_jd), which is
// sum_d max(q_d, 0) hi_jd + min(q_d, 0) lo_jd.  The heads that share a key head read the same pages, so their bounds are added up: one vector of the sums of the positive
// parts and one of the negative parts against the page's two rows, 2 D multiply-adds a page whatever the number of heads.  Which pages are
// kept is defined by the sums in float64; a bound that is no number counts as the largest.
//
// A block a token and head scores its pages in float32, with a bound of the errors: eight or sixteen lanes a page, two batches of pages in flight.  It finds the last score that is kept by a
// histogram of eight bits, from the first bit in which the scores differ, and a list of what that leaves.  Pages whose scores lie further from that one than twice the largest error are
// decided; the others (as a rule the one page of that score) are scored in float64 and chosen by those, of equal ones the earlier page.
//
// Bound by what one SM takes in: 48 tokens of 4 heads of 128 on 410 pages (40 MB) 16.0 us, with two blocks on some SMs; one token of 2 heads of 64 on 510 pages 8.5 us, a chain of a dozen
// waits.  With a kernel of its own that scores, a run of pages a block, 22.1 and 8.5; beyond 1,024 pages that one is used (one token on 2,046 pages 15.7 us, in one kernel 18.5).
// A ring filled by asynchronous copies instead of registers: 20.2.  In float64 throughout: 44, since conversions run at an eighth of the rate of multiply-adds.
#include "common.cuh"

#define PS_THREADS 256
#define PS_WARPS (PS_THREADS / 32)
#define PS_MOST_SMEM (200 * 1024)                              // of a block that selects: twenty bytes a page
#define PS_ONE_PAGES 1024                                      // up to so many pages a block scores those that it selects from

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

// the sums of the positive and of the negative parts of a head's queries, into shared memory (T: float or double)
template <int D, typename T>
__device__ __forceinline__ void ps_queries(const PsArgs& p, int tok, int kvh, T (*sums)[D]) {
    if (threadIdx.x >= D) return;
    const int G = p.n_heads / p.n_kv;
    const bf16* q = p.q + (size_t)tok * p.q_stride + (size_t)kvh * G * D + threadIdx.x;
    T up = 0, down = 0;
#pragma unroll 8
    for (int h = 0; h < G; ++h) {
        const float x = __bfloat162float(q[h * D]);
        up += x > 0.f || x != x ? x : 0.f;
        down += x < 0.f ? x : 0.f;
    }
    sums[0][threadIdx.x] = up; sums[1][threadIdx.x] = down;
}

// a lane's sixteen factors, in pairs: those of eight channels of the greatest keys, then of the least
template <int D>
__device__ __forceinline__ void ps_factors(const float (*sums)[D], int l, unsigned long long (&by)[2][4]) {
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const ulonglong2 four = *reinterpret_cast<const ulonglong2*>(&sums[side][8 * l + 2 * e]);
            by[side][e] = four.x; by[side][e + 1] = four.y;
        }
}

// a lane's part of the rows of `ahead` pages
template <int D>
__device__ __forceinline__ void ps_load(const PsArgs& p, int kvh, int l, const int (&page)[PsScore<D>::ahead], uint4 (&v)[PsScore<D>::ahead][2]) {
#pragma unroll
    for (int u = 0; u < PsScore<D>::ahead; ++u) {
        const uint4* row = reinterpret_cast<const uint4*>(p.bounds + ((size_t)max(page[u], 0) * p.n_kv + kvh) * 2 * D) + l;
        v[u][0] = v[u][1] = make_uint4(0u, 0u, 0u, 0u);
        if (page[u] >= 0) { v[u][0] = row[D / 8]; v[u][1] = row[0]; }
    }
}

// The pages' scores, one a lane (l < 4): of page ps_mine(l).  `sizes` gathers the largest size of each number that the lane has met.
__device__ __forceinline__ int ps_mine(int l) { return (l & 1) * 2 + ((l >> 1) & 1); }
template <int D>
__device__ __forceinline__ float ps_scores(const uint4 (&v)[PsScore<D>::ahead][2], const unsigned long long (&by)[2][4], int l, __nv_bfloat162 (&sizes)[2][4]) {
    using S = PsScore<D>;
    float r[S::ahead];
#pragma unroll
    for (int u = 0; u < S::ahead; ++u) {
        unsigned long long s = 0ull;                           // two float32 sums
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const unsigned w[4] = {v[u][side].x, v[u][side].y, v[u][side].z, v[u][side].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned long long x = (unsigned long long)(w[e] & 0xffff0000u) << 32 | (w[e] << 16);
                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(s) : "l"(x), "l"(by[side][e]));
                sizes[side][e] = __hmax2_nan(sizes[side][e], __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[e])));
            }
        }
        r[u] = __uint_as_float((unsigned)s) + __uint_as_float((unsigned)(s >> 32));
    }
    // four sums over the page's lanes: each exchange halves what a lane has, until it has one
#pragma unroll
    for (int n = S::ahead / 2, o = 1; n; n >>= 1, o <<= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float give = l & o ? r[i] : r[n + i], have = l & o ? r[n + i] : r[i];
            r[i] = have + __shfl_xor_sync(0xffffffffu, give, o);
        }
#pragma unroll
    for (int o = 4; o < S::lanes; o <<= 1) r[0] += __shfl_xor_sync(0xffffffffu, r[0], o);
    return r[0];
}

// A bound of the scores' errors, of all pages whose numbers `sizes` has: roundings of a head's sum, a lane's chain of eight twice and the lanes' tree are less than 24 + heads of 2^-24 of
// the terms' sizes, which are less than their sum with every number at its largest; twice that.
template <int D>
__device__ __forceinline__ float ps_error(const PsArgs& p, const unsigned long long (&by)[2][4], const __nv_bfloat162 (&sizes)[2][4]) {
    float size = 0.f;
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 x = __bfloat1622float2(sizes[side][e]);
            size += fabsf(__uint_as_float((unsigned)by[side][e])) * x.x + fabsf(__uint_as_float((unsigned)(by[side][e] >> 32))) * x.y;
        }
#pragma unroll
    for (int o = 1; o < PsScore<D>::lanes; o <<= 1) size += __shfl_xor_sync(0xffffffffu, size, o);
    return size * ((float)(32 + p.n_heads / p.n_kv) * 1.1920929e-7f);
}

template <int D>
__global__ void __launch_bounds__(PS_THREADS) score_pages_kernel(const PsArgs p, float2* scores) {
    using S = PsScore<D>;
    __shared__ __align__(16) float sums[2][D];
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.y, tok = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % S::lanes;
    const int pages = p.pages(p.position(tok)), first = 1 + (int)blockIdx.x * S::pages;
    if (pages <= p.keep || first >= pages - 1) return;         // (the first and the last page are kept whatever they score)
    const int* table = p.table(tok);
    uint4 v[S::ahead][2];
    int place[S::ahead], page[S::ahead];                       // of the page's score, -1: none of this warp's
#pragma unroll
    for (int u = 0; u < S::ahead; ++u) {
        const int j = first + (u * PS_WARPS + warp) * S::at_once + lane / S::lanes;
        page[u] = j < pages - 1 ? table[j] : -1;
        if (page[u] >= p.n_pages) page[u] = -1;
        place[u] = page[u] >= 0 ? j : -1;
    }
    ps_load<D>(p, kvh, l, page, v);
    ps_queries<D>(p, tok, kvh, sums);
    __syncthreads();
    unsigned long long by[2][4];
    __nv_bfloat162 sizes[2][4] = {};
    ps_factors<D>(sums, l, by);
    const float r = ps_scores<D>(v, by, l, sizes), error = ps_error<D>(p, by, sizes);
    int to = place[0];
#pragma unroll
    for (int u = 1; u < S::ahead; ++u) to = ps_mine(l) == u ? place[u] : to;
    if (l < 4 && to >= 0) scores[((size_t)tok * p.n_kv + kvh) * p.most + to] = make_float2(r, error);
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
        if constexpr (bits == 32) {
            // few are left, as a rule after the first histogram: in a list, of which each thread counts those above its own
            const int n = told[2];
            if (n <= PS_THREADS) {
                __syncthreads();                               // (told has been read)
                if (threadIdx.x == 0) told[1] = 0;
                __syncthreads();
                for (int j = first + threadIdx.x; j < last; j += PS_THREADS) if ((keys[j] ^ prefix) >> shift == 0) hist[atomicAdd(&told[1], 1)] = keys[j];
                __syncthreads();
                if (threadIdx.x < n) {
                    const Key k = hist[threadIdx.x];
                    int above = 0, same = 0;
                    for (int i = 0; i < n; ++i) { above += hist[i] > k; same += hist[i] == k; }
                    if (above < wanted && wanted <= above + same) { told[0] = (int)k; told[2] = wanted == above + same ? -1 : wanted - above; }
                }
                __syncthreads();
                least = (Key)told[0]; equal = told[2];
                return;
            }
        }
        top = shift;
        __syncthreads();                                       // (told and the histogram have been read)
    }
}

// SCORES: the block scores its pages itself (all_scores: none)
template <int D, bool SCORES>
__global__ void __launch_bounds__(PS_THREADS) select_pages_kernel(const PsArgs p, const float2* all_scores, int* out_table, int* out_pos) {
    extern __shared__ unsigned long long ps_exact[];           // [most] keys of float64 scores, where some are needed; [most] keys of the scores; [most] entries of the page table; [most] pages to score again
    unsigned* keys = reinterpret_cast<unsigned*>(ps_exact + p.most);
    int* entries = reinterpret_cast<int*>(keys + p.most);
    __shared__ int parts[2][PS_WARPS], told[3];
    __shared__ unsigned hist[256], ends[2][PS_WARPS];
    __shared__ unsigned long long ends64[2][PS_WARPS];
    __shared__ float errors[PS_WARPS];
    __shared__ double sums[2][D];
    __shared__ __align__(16) float sums32[2][D];
    __shared__ int n_listed;
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.x, tok = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_kv = p.n_kv, keep = p.keep;
    const int pos = p.position(tok), pages = p.pages(pos);
    const bool choose = pages > keep && keep > 2;
    const int wanted = keep - 2;                               // besides the first and the last page
    float error = 0.f;
    if (pages) {
        const int* table = p.table(tok);
        const float2* scores = all_scores + ((size_t)tok * n_kv + kvh) * p.most;
        if constexpr (SCORES) { if (choose) ps_queries<D>(p, tok, kvh, sums32); }
        for (int j = threadIdx.x; j < pages; j += PS_THREADS) {
            const int page = table[j];
            const bool there = page >= 0 && page < p.n_pages;
            entries[j] = there ? page : -1;
            if (choose && j > 0 && j < pages - 1) {
                if (SCORES || !there) { keys[j] = 0u; continue; }
                const float2 s = scores[j];
                keys[j] = s.x != s.x ? ~0u : ps_key(s.x);
                error = ps_max(error, s.y);
            }
        }
        if constexpr (SCORES) {
            using S = PsScore<D>;
            __syncthreads();
            if (choose) {
                const int l = lane % S::lanes, run = S::ahead * S::at_once;
                unsigned long long by[2][4];
                __nv_bfloat162 sizes[2][4] = {};
                ps_factors<D>(sums32, l, by);
                uint4 v[2][S::ahead][2];
                const auto fetch = [&](int base, uint4 (&to)[S::ahead][2]) {
                    int page[S::ahead];
#pragma unroll
                    for (int u = 0; u < S::ahead; ++u) { const int j = base + u * S::at_once + lane / S::lanes; page[u] = j < pages - 1 ? entries[j] : -1; }
                    ps_load<D>(p, kvh, l, page, to);
                };
                const auto score = [&](int base, const uint4 (&from)[S::ahead][2]) {
                    const float r = ps_scores<D>(from, by, l, sizes);
                    const int j = base + ps_mine(l) * S::at_once + lane / S::lanes;
                    if (l < 4 && j < pages - 1 && entries[j] >= 0) keys[j] = r != r ? ~0u : ps_key(r);
                };
                const int step = PS_WARPS * run;
                int base = 1 + warp * run;
                if (base < pages - 1) fetch(base, v[0]);
                for (; base < pages - 1; base += 2 * step) {
                    if (base + step < pages - 1) fetch(base + step, v[1]);
                    score(base, v[0]);
                    if (base + step >= pages - 1) break;
                    if (base + 2 * step < pages - 1) fetch(base + 2 * step, v[0]);
                    score(base + step, v[1]);
                }
                error = ps_error<D>(p, by, sizes);
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
        error = 0.f;
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
        if (n_over + n_near != wanted) {
            // the pages that are near, their scores in float64
            unsigned* list = reinterpret_cast<unsigned*>(entries + p.most);
            refine = none || n_near > PS_THREADS;
            if (threadIdx.x == 0) n_listed = 0;
            ps_queries<D>(p, tok, kvh, sums);
            __syncthreads();
            for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) {
                if (refine) ps_exact[j] = keys[j] > over ? ~0ull : 0ull;                  // (decided ones beside the others)
                if (keys[j] >= under && keys[j] <= over && entries[j] >= 0) list[atomicAdd(&n_listed, 1)] = j;
            }
            __syncthreads();
            const int listed = n_listed;
            for (int x = warp; x < listed; x += PS_WARPS) {
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
                if (lane == 0) ps_exact[refine ? j : x] = min(max(ps_key(s), 1ull), ~0ull - 1);
            }
            __syncthreads();
            if (refine) {
                ps_cut<unsigned long long>(ps_exact, 1, pages - 1, wanted, least, equal, hist, ends64, told);
            } else {
                // few: each thread counts those in front of its page
                if (threadIdx.x < listed) {
                    const unsigned j = list[threadIdx.x];
                    const unsigned long long key = ps_exact[threadIdx.x];
                    int before = n_over;
                    for (int x = 0; x < listed; ++x) before += ps_exact[x] > key || (ps_exact[x] == key && list[x] < j);
                    keys[j] = before < wanted ? ~0u : 0u;
                }
                __syncthreads();
            }
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

// scratch: 8 bytes a page of every token and head, a score and its error, where there are more than PS_ONE_PAGES
extern "C" int pe_select_pages(const void* q, int q_stride, int T, int n_heads, int n_kv, int hd, const void* bounds, long long n_pages, const int* block_table,
                               int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep, int max_context, int* out_table, int* out_pos, void* scratch, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_kv > 65535 || T > 65535 || n_heads % n_kv || keep < 1 || max_context < 1 || n_rows < 1 || table_stride < 1 || n_pages * n_kv > 0x7fffffffll)
        return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)bounds) & 15) return PE_ERR_UNSUPPORTED;
    const int most = ps_most(max_context, table_stride);
    const size_t smem = (size_t)most * 20;
    const bool one = most <= PS_ONE_PAGES;
    if (smem > PS_MOST_SMEM || (!one && (((uintptr_t)scratch & 7) || !scratch))) return PE_ERR_UNSUPPORTED;
    const PsArgs p = {(const bf16*)q, (const bf16*)bounds, block_table, tok_pos, tok_row, q_stride, n_heads, n_kv, (int)n_pages, table_stride, n_rows, keep, most};
    float2* scores = (float2*)scratch;
    auto kernel = one ? (hd == 64 ? select_pages_kernel<64, true> : select_pages_kernel<128, true>) : hd == 64 ? select_pages_kernel<64, false> : select_pages_kernel<128, false>;
    const int per = hd == 64 ? PsScore<64>::pages : PsScore<128>::pages;
    if (!one && most > keep && keep > 2) {                     // (else every token has all of its pages)
        PE_TRY(pe_launch(hd == 64 ? score_pages_kernel<64> : score_pages_kernel<128>, dim3((unsigned)((most + per - 1) / per), (unsigned)n_kv, (unsigned)T),
                         dim3(PS_THREADS), 0, (cudaStream_t)stream, p, scores));
        PE_LAUNCH_CHECK();
    }
    static bool allowed[4][64] = {};
    { const int e = pe_allow_smem((const void*)kernel, PS_MOST_SMEM, allowed[2 * (hd == 128) + one]); if (e) return e; }
    PE_TRY(pe_launch(kernel, dim3((unsigned)n_kv, (unsigned)T), dim3(PS_THREADS), smem, (cudaStream_t)stream, p, (const float2*)scores, out_table, out_pos));
    PE_LAUNCH_CHECK();
    return 0;
}
