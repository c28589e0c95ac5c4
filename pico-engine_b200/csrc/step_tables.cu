// The layout of a step from the lengths of its requests: where every token stands (position, batch row, place in the cache) and the
// page table of every row.  What the host would have to send for this is the whole table (rows x pages of the longest sequence, every
// step); what it sends instead are four numbers a row and the pages that the step takes.
//
//   row b brings lens[b] tokens at positions starts[b] ..; its sequence has the row slots[b] of the resident table, whose first held[b]
//   entries are known already.  It needs ceil((starts[b] + lens[b]) / 64) of them; the missing ones are the next numbers of `pages`,
//   dealt to the rows in their order.  A place is page * 64 + position % 64.
//
// Every block adds up what the rows before its own bring and take (a few thousand cached numbers at most) instead of waiting for
// a scan: one launch, no scratch, no order among blocks.  What is written of the resident table is the row's own entries.
#include "common.cuh"

#define ST_THREADS 256

struct StArgs {
    const int *slots, *starts, *lens, *held, *pages;
    int* resident;
    int *tok_pos, *tok_row, *row_first, *places, *tables;
    int rows, n_slots, res_width, n_pages, n_tokens, width;
};

__device__ __forceinline__ int st_need(int start, int len) { return (int)(((long long)start + len + PE_PAGE - 1) / PE_PAGE); }

__global__ void __launch_bounds__(ST_THREADS) step_tables_kernel(const StArgs p) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ int scratch[2][ST_THREADS / 32];
    const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // tokens and new pages of the rows before this one
    int tokens = 0, taken = 0;
    for (int i = threadIdx.x; i < b; i += ST_THREADS) {
        const int n = max(p.lens[i], 0);
        tokens += n;
        taken += max(st_need(p.starts[i], n) - p.held[i], 0);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
        taken += __shfl_xor_sync(0xffffffffu, taken, o);
    }
    if (lane == 0) { scratch[0][warp] = tokens; scratch[1][warp] = taken; }
    __syncthreads();
    tokens = taken = 0;
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; ++w) { tokens += scratch[0][w]; taken += scratch[1][w]; }

    const int slot = p.slots[b], start = p.starts[b], n = max(p.lens[b], 0), held = max(p.held[b], 0);
    const int need = max(st_need(start, n), held);
    int* row = slot >= 0 && slot < p.n_slots ? p.resident + (size_t)slot * p.res_width : nullptr;
    auto page_of = [&](int w) {                                     // entry w of the row's table
        if (!row || w < 0 || w >= p.res_width || w >= need) return -1;
        if (w < held) return row[w];
        const int at = taken + w - held;
        return at < p.n_pages ? p.pages[at] : -1;
    };
    if (threadIdx.x == 0) {
        p.row_first[b] = tokens;
        if (b == p.rows - 1) p.row_first[p.rows] = tokens + n;
    }
    for (int i = threadIdx.x; i < n && tokens + i < p.n_tokens; i += ST_THREADS) {
        const int at = start + i, page = page_of(at / PE_PAGE);
        p.tok_pos[tokens + i] = at;
        p.tok_row[tokens + i] = b;
        p.places[tokens + i] = page >= 0 ? page * PE_PAGE + at % PE_PAGE : -1;
    }
    for (int w = threadIdx.x; w < p.width; w += ST_THREADS) p.tables[(size_t)b * p.width + w] = page_of(w);
    if (row)
        for (int w = held + threadIdx.x; w < min(need, p.res_width); w += ST_THREADS) row[w] = page_of(w);
}

extern "C" int pe_step_tables(const int* slots, const int* starts, const int* lens, const int* held, const int* pages, int n_pages, int* resident,
                              int n_slots, int res_width, int rows, int* tok_pos, int* tok_row, int* row_first, int* places, int n_tokens,
                              int* tables, int width, void* stream) {
    if (rows <= 0) return 0;
    if (n_slots <= 0 || res_width <= 0 || width <= 0 || n_tokens < 0 || n_pages < 0) return PE_ERR_UNSUPPORTED;
    const StArgs p = {slots, starts, lens, held, pages, resident, tok_pos, tok_row, row_first, places, tables, rows, n_slots, res_width, n_pages, n_tokens, width};
    PE_TRY(pe_launch(step_tables_kernel, rows, ST_THREADS, 0, (cudaStream_t)stream, p));
    PE_LAUNCH_CHECK();
    return 0;
}
