// Attention of single tokens of which several share the first part of their sequences: the answers to one prompt.  Their page tables name
// the same pages for the shared positions, each row has pages of its own behind them.
//
//   o = sum_j w_j v_j / (sum_j w_j + e^sink),   w_j = exp(scale q.k_j - slope (pos - j)),   j <= pos, j > pos - window or j < keep_first
//
// A warp a row and query head, a key at a time.
#ifndef PE_HEAD_DIM
#error "compile with -DPE_HEAD_DIM=<head size>"
#endif
#include "common.cuh"

#if PE_HEAD_DIM == 64 || PE_HEAD_DIM == 128

#define AS_HD PE_HEAD_DIM
#define AS_PER (AS_HD / 32)

__global__ void __launch_bounds__(128) attention_shared_kernel(const bf16* q, int q_stride, bf16* out, const bf16* k_pool, const bf16* v_pool,
                                                               const int* block_table, int table_stride, const int* tok_pos, const int* tok_row,
                                                               int T, int nh, int nkv, int window, int keep_first, float scale,
                                                               const float* slopes, const float* sinks) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= T * nh) return;
    const int tok = item / nh, h = item % nh, kvh = h / (nh / nkv), pos = tok_pos[tok];
    const int* table = block_table + (size_t)tok_row[tok] * table_stride;
    float qf[AS_PER], o[AS_PER], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < AS_PER; ++i) { qf[i] = to_f(q[(size_t)tok * q_stride + h * AS_HD + lane * AS_PER + i]) * scale; o[i] = 0.f; }
    const float slope = slopes ? slopes[h] : 0.f;
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    for (int j = 0; j <= pos; ++j) {
        if (j < lo && j >= keep_first) { j = lo - 1; continue; }
        const int page = table[j / PE_PAGE];
        if (page < 0) continue;
        const size_t at = (((size_t)page * nkv + kvh) * PE_PAGE + j % PE_PAGE) * AS_HD + lane * AS_PER;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < AS_PER; ++i) s = fmaf(qf[i], to_f(k_pool[at + i]), s);
        s = warp_sum(s) - slope * (float)(pos - j);
        const float m_new = fmaxf(m, s), a = expf(m - m_new), w = expf(s - m_new);
        l = fmaf(l, a, w);
        m = m_new;
#pragma unroll
        for (int i = 0; i < AS_PER; ++i) o[i] = fmaf(o[i], a, w * to_f(v_pool[at + i]));
    }
    if (sinks) l += expf(sinks[h] - m);
#pragma unroll
    for (int i = 0; i < AS_PER; ++i) out[((size_t)tok * nh + h) * AS_HD + lane * AS_PER + i] = __float2bfloat16_rn(l > 0.f ? o[i] / l : 0.f);
}

extern "C" int pe_attention_shared(const void* q, int q_stride, void* out, const void* k_pool, const void* v_pool, long long pool_pages,
                                   const int* block_table, int table_stride, const int* tok_pos, const int* tok_row, const void* groups, int T,
                                   int nh, int nkv, int hd, int window, int keep_first, float scale, int max_context, const float* slopes,
                                   const float* sinks, int early_pages, void* scratch, int* status, void* stream) {
    if (T <= 0) return 0;
    if (hd != AS_HD || nkv <= 0 || nh % nkv || q_stride % 8 || !(scale > 0.f) || (long long)T * nh > 0x7fffffff) return PE_ERR_UNSUPPORTED;
    PE_TRY(pe_launch(attention_shared_kernel, (T * nh + 3) / 4, 128, 0, (cudaStream_t)stream, (const bf16*)q, q_stride, (bf16*)out, (const bf16*)k_pool,
                     (const bf16*)v_pool, block_table, table_stride, tok_pos, tok_row, T, nh, nkv, window, window > 0 ? keep_first : 0, scale, slopes, sinks));
    PE_LAUNCH_CHECK();
    return 0;
}

#else   // other head sizes: the rows of a group are read one by one (attention_decode.cu)

extern "C" int pe_attention_shared(const void*, int, void*, const void*, const void*, long long, const int*, int, const int*, const int*, const void*,
                                   int, int, int, int, int, int, float, int, const float*, const float*, int, void*, int*, void*) {
    return PE_ERR_UNSUPPORTED;
}

#endif
