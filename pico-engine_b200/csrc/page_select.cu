// The pages of a long context that a token's heads can score highest.
//
// A page j holds keys between lo_j and hi_j, channel by channel (page_bounds).  No key of it scores more against a query q than sum_d max(q_d lo_jd, q_d hi_jd), which is
// sum_d max(q_d, 0) hi_jd + min(q_d, 0) lo_jd.  The heads that share a key head read the same pages, so their bounds are added up: one vector of the sums of the positive
// parts and one of the negative parts against the page's two rows, 2 D multiply-adds a page whatever the number of heads.  Sums are float64: which of two pages
// comes first must not depend on the order of the additions.  A bound that is no number counts as the largest.
//
// A cluster of CTAs has the pages of one token and key head in equal shares; eight lanes take a page, 16 bytes at a time.  The scores go to the first CTA's shared memory as 64-bit
// keys that compare like them.  It finds the least key that is kept bit by bit, from the first bit in which the keys differ until as many are above as are wanted: a count
// a bit, some twenty of them.
#include "common.cuh"

#define PS_THREADS 256
#ifndef PS_FILL
#define PS_FILL 4
#endif
#define PS_WARPS (PS_THREADS / 32)

// a float64 as 64 bits that compare like it; NaN above all
__device__ __forceinline__ unsigned long long ps_key(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);      // (-0 is 0)
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ void ps_to_first(unsigned local, unsigned long long v) {
    unsigned remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(local));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}
// a sum over the block; `parts` are two rows that take turns, so that one barrier a sum is enough
__device__ __forceinline__ int ps_sum(int v, int (*parts)[PS_WARPS], int turn) {
    v = __reduce_add_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) parts[turn & 1][threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < PS_WARPS; ++w) s += parts[turn & 1][w];
    return s;
}

template <int D>
__global__ void __launch_bounds__(PS_THREADS) select_pages_kernel(const bf16* q, int q_stride, int n_heads, int n_kv, const bf16* bounds, int n_pages, const int* block_table,
                                                                  int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep, int most, int ctas,
                                                                  int* out_table, int* out_pos) {
    constexpr int each = D / 8;                                                           // channels of a lane
    extern __shared__ unsigned long long ps_keys[];                                       // [most], then [most] entries of the page table
    int* entries = reinterpret_cast<int*>(ps_keys + most);
    __shared__ double sums[2][D];
    __shared__ int parts[2][PS_WARPS];
    __shared__ unsigned long long ends[2][PS_WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.y, tok = blockIdx.z, G = n_heads / n_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = ctas > 1 ? (int)blockIdx.x : 0;                                     // (a cluster is a row of the grid)
    const int pos = max(tok_pos[tok], 0), row = min(max(tok_row[tok], 0), n_rows - 1);
    const int* table = block_table + (size_t)row * table_stride;
    const int pages = min(min(pos / PE_PAGE + 1, table_stride), most);
    const bool all = pages <= keep;
    const int wanted = keep - 2;                                                          // besides the first and the last page
    for (int j = threadIdx.x; j < pages; j += PS_THREADS) { const int page = table[j]; entries[j] = page < n_pages ? page : -1; }
    if (!all && wanted > 0) {
        for (int d = threadIdx.x; d < D; d += PS_THREADS) {
            double up = 0.0, down = 0.0;
#pragma unroll 8
            for (int h = 0; h < G; ++h) {
                const float x = __bfloat162float(q[(size_t)tok * q_stride + (size_t)(kvh * G + h) * D + d]);
                up += x > 0.f || x != x ? x : 0.f;
                down += x < 0.f ? x : 0.f;
            }
            sums[0][d] = up; sums[1][d] = down;
        }
        __syncthreads();
        const int l8 = lane & 7;
        double up[each], down[each];
#pragma unroll
        for (int i = 0; i < each; ++i) { up[i] = sums[0][l8 * 8 + (i / 8) * 64 + i % 8]; down[i] = sums[1][l8 * 8 + (i / 8) * 64 + i % 8]; }
        const unsigned keys0 = (unsigned)__cvta_generic_to_shared(ps_keys);
        // pages 1 .. pages - 2, four a warp at a time
        for (int j0 = 1 + (share * PS_WARPS + warp) * 4; j0 < pages - 1; j0 += ctas * PS_WARPS * 4) {
            const int j = j0 + (lane >> 3), page = j < pages - 1 ? entries[j] : -1;
            const bool there = page >= 0;
            double s = 0.0;
            if (there) {
                const uint4* lo = reinterpret_cast<const uint4*>(bounds + ((size_t)page * n_kv + kvh) * 2 * D) + l8;
                uint4 v[2][each / 8];
#pragma unroll
                for (int i = 0; i < each / 8; ++i) { v[0][i] = lo[D / 8 + 8 * i]; v[1][i] = lo[8 * i]; }
#pragma unroll
                for (int i = 0; i < each / 8; ++i)
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        const unsigned w[4] = {v[side][i].x, v[side][i].y, v[side][i].z, v[side][i].w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const double b = (double)__uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
                            s = fma(side ? down[8 * i + e] : up[8 * i + e], b, s);
                        }
                    }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (l8 == 0 && j < pages - 1) {
                const unsigned long long key = there ? ps_key(s) : 0ull;
                if (share) ps_to_first(keys0 + 8u * j, key); else ps_keys[j] = key;
            }
        }
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (share) return;
    }
    __syncthreads();
    unsigned long long least = 0ull;                                                      // keys from here on are kept, of those equal to it the first `equal`
    int equal = 0x7fffffff, turn = 0;
    if (!all && wanted > 0 && wanted < pages - 2) {
        unsigned long long low = ~0ull, high = 0ull;
        for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) { const unsigned long long k = ps_keys[j]; low = min(low, k); high = max(high, k); }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { low = min(low, __shfl_xor_sync(0xffffffffu, low, o)); high = max(high, __shfl_xor_sync(0xffffffffu, high, o)); }
        if (lane == 0) { ends[0][warp] = low; ends[1][warp] = high; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) { low = min(low, ends[0][w]); high = max(high, ends[1][w]); }
        if (low == high) {
            least = low; equal = wanted;
        } else {
            // the bits in front of the first difference are common; then bit by bit the largest number that at least `wanted` keys reach
            int bit = 63 - __clzll((long long)(low ^ high));
            least = bit == 63 ? 0ull : high >> (bit + 1) << (bit + 1);
            int reach = pages - 2;                                                        // keys from `least` on
            for (; bit >= 0 && reach != wanted; --bit) {
                const unsigned long long next = least | 1ull << bit;
                int n = 0;
                for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) n += ps_keys[j] >= next;
                n = ps_sum(n, parts, turn++);
                if (n >= wanted) { least = next; reach = n; }
            }
            if (reach != wanted) {                                                        // several keys are equal to the last one kept
                int n = 0;
                for (int j = 1 + threadIdx.x; j < pages - 1; j += PS_THREADS) n += ps_keys[j] > least;
                equal = wanted - ps_sum(n, parts, turn++);
            }
        }
    }
    // the kept pages in the order of the positions
    int* mine = out_table + ((size_t)tok * n_kv + kvh) * keep;
    int done = 0, ties = 0;
    for (int base = 0; base < pages; base += PS_THREADS) {
        const int j = base + threadIdx.x;
        bool kept = j < pages && (all || j == pages - 1 || (j == 0 && keep > 1)), tie = false;
        if (!all && wanted > 0 && j > 0 && j < pages - 1) { kept = ps_keys[j] > least; tie = ps_keys[j] == least; }
        if (equal != 0x7fffffff) {                                                        // (the same for the whole block)
            const unsigned set = __ballot_sync(0xffffffffu, tie);
            __syncthreads();
            if (lane == 0) parts[0][warp] = __popc(set);
            __syncthreads();
            int at = ties + __popc(set & ((1u << lane) - 1u));
#pragma unroll
            for (int w = 0; w < PS_WARPS; ++w) { if (w < warp) at += parts[0][w]; ties += parts[0][w]; }
            kept |= tie && at < equal;
        } else {
            kept |= tie;
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
    if (threadIdx.x == 0) out_pos[tok * n_kv + kvh] = (done - 1) * PE_PAGE + pos % PE_PAGE;
}

extern "C" int pe_select_pages(const void* q, int q_stride, int T, int n_heads, int n_kv, int hd, const void* bounds, long long n_pages, const int* block_table,
                               int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep, int max_context, int* out_table, int* out_pos, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_kv > 65535 || T > 65535 || n_heads % n_kv || keep < 1 || max_context < 1 || n_rows < 1 || table_stride < 1 || n_pages * n_kv > 0x7fffffffll)
        return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)bounds) & 15) return PE_ERR_UNSUPPORTED;
    const int most = (max_context - 1) / PE_PAGE + 1 < table_stride ? (max_context - 1) / PE_PAGE + 1 : table_stride;
    const size_t smem = (size_t)most * 12;
    if (smem > 200 * 1024) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? select_pages_kernel<64> : select_pages_kernel<128>;
    if (smem > 40 * 1024) PE_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    // CTAs of a token and head: PS_FILL an SM in all, and each warp four pages at least
    int ctas = 1;
    while (ctas < 8 && (long long)T * n_kv * ctas * 2 <= PS_FILL * pe_sm_count() && ctas * PS_WARPS * 4 < most) ctas *= 2;
    PE_TRY(pe_launch_cluster(kernel, dim3((unsigned)ctas, (unsigned)n_kv, (unsigned)T), dim3(PS_THREADS), smem, (cudaStream_t)stream, (unsigned)ctas, (const bf16*)q, q_stride, n_heads, n_kv,
                             (const bf16*)bounds, (int)n_pages, block_table, table_stride, n_rows, tok_pos, tok_row, keep, most, ctas, out_table, out_pos));
    PE_LAUNCH_CHECK();
    return 0;
}
