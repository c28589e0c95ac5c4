// The pages of a long context that a token's heads can score highest.
//
// A page j holds keys between lo_j and hi_j, channel by channel (page_bounds).  No key of it scores more against a query q than sum_d max(q_d lo_jd, q_d hi_jd), which is
// sum_d max(q_d, 0) hi_jd + min(q_d, 0) lo_jd.  The heads that share a key head read the same pages, so their bounds are added up: one vector of the sums of the positive
// parts and one of the negative parts against the page's two rows, 2 D multiply-adds a page whatever the number of heads.  Sums are float64: which of two pages
// comes first must not depend on the order of the additions.  A bound that is no number counts as the largest.
#include "common.cuh"

#define PS_THREADS 256

// a float64 as 64 bits that compare like it; NaN above all
__device__ __forceinline__ unsigned long long ps_key(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);      // (-0 is 0)
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

template <int D>
__global__ void __launch_bounds__(PS_THREADS) select_pages_kernel(const bf16* q, int q_stride, int n_heads, int n_kv, const bf16* bounds, long long n_pages,
                                                                  const int* block_table, int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep,
                                                                  int most, int* out_table, int* out_pos) {
    extern __shared__ unsigned long long ps_keys[];                                       // [most]
    __shared__ double sums[2][D];
    __shared__ int warp_count[PS_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int tok = blockIdx.x, kvh = blockIdx.y, G = n_heads / n_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = max(tok_pos[tok], 0), row = min(max(tok_row[tok], 0), n_rows - 1);
    const int* table = block_table + (size_t)row * table_stride;
    const int pages = min(min(pos / PE_PAGE + 1, table_stride), most);
    int* mine = out_table + ((size_t)tok * n_kv + kvh) * keep;
    const bool all = pages <= keep;
    const int wanted = keep - 2;                                                          // besides the first and the last page
    if (!all && wanted > 0) {
        for (int d = threadIdx.x; d < D; d += PS_THREADS) {
            double up = 0.0, down = 0.0;
            for (int h = 0; h < G; ++h) {
                const float x = __bfloat162float(q[(size_t)tok * q_stride + (size_t)(kvh * G + h) * D + d]);
                up += x > 0.f || x != x ? x : 0.f;
                down += x < 0.f ? x : 0.f;
            }
            sums[0][d] = up; sums[1][d] = down;
        }
        __syncthreads();
        for (int j = 1 + warp; j < pages - 1; j += PS_THREADS / 32) {
            const int page = table[j];
            double s = 0.0;
            if (page >= 0 && page < n_pages) {
                const bf16* lo = bounds + ((size_t)page * n_kv + kvh) * 2 * D;
                for (int d = lane; d < D; d += 32) s += sums[0][d] * (double)__bfloat162float(lo[D + d]) + sums[1][d] * (double)__bfloat162float(lo[d]);
                s = warp_sum_d(s);
            }
            if (lane == 0) ps_keys[j] = page >= 0 && page < n_pages ? ps_key(s) : 0ull;
        }
        __syncthreads();
    }
    // a page is kept where fewer than `wanted` pages come before it
    int done = 0;
    for (int base = 0; base < pages; base += PS_THREADS) {
        const int j = base + threadIdx.x;
        bool kept = j < pages && (all || j == pages - 1 || (j == 0 && keep > 1));
        if (!kept && j < pages - 1 && j > 0 && wanted > 0) {
            const unsigned long long k = ps_keys[j];
            int before = 0;
            for (int i = 1; i < pages - 1; ++i) before += ps_keys[i] > k || (ps_keys[i] == k && i < j);
            kept = before < wanted;
        }
        const unsigned set = __ballot_sync(0xffffffffu, kept);
        if (lane == 0) warp_count[warp] = __popc(set);
        __syncthreads();
        int at = done + __popc(set & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < PS_THREADS / 32; ++w) { if (w < warp) at += warp_count[w]; done += warp_count[w]; }
        if (kept) { const int page = table[j]; mine[at] = page >= 0 && page < n_pages ? page * n_kv + kvh : -1; }
        __syncthreads();
    }
    for (int i = done + threadIdx.x; i < keep; i += PS_THREADS) mine[i] = -1;
    if (threadIdx.x == 0) out_pos[tok * n_kv + kvh] = (done - 1) * PE_PAGE + pos % PE_PAGE;
}

extern "C" int pe_select_pages(const void* q, int q_stride, int T, int n_heads, int n_kv, int hd, const void* bounds, long long n_pages, const int* block_table,
                               int table_stride, int n_rows, const int* tok_pos, const int* tok_row, int keep, int max_context, int* out_table, int* out_pos, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_kv > 65535 || n_heads % n_kv || keep < 1 || max_context < 1 || n_rows < 1 || table_stride < 1) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)bounds) & 15) return PE_ERR_UNSUPPORTED;
    const int most = min((max_context - 1) / PE_PAGE + 1, table_stride);
    const size_t smem = (size_t)most * 8;
    if (smem > 200 * 1024) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? select_pages_kernel<64> : select_pages_kernel<128>;
    if (smem > 40 * 1024) PE_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    PE_TRY(pe_launch(kernel, dim3((unsigned)T, (unsigned)n_kv), dim3(PS_THREADS), smem, (cudaStream_t)stream, (const bf16*)q, q_stride, n_heads, n_kv, (const bf16*)bounds,
                     n_pages, block_table, table_stride, n_rows, tok_pos, tok_row, keep, most, out_table, out_pos));
    PE_LAUNCH_CHECK();
    return 0;
}
