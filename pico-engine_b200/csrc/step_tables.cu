// The layout of a step from the lengths of its requests: where every token stands (position, batch row, place in the cache) and the
// page table of every row.  What the host would have to send for this is the whole table (rows x pages of the longest sequence, every
// step); what it sends instead are four numbers a row and the pages that the step takes.
//
//   row b brings lens[b] tokens at positions starts[b] ..; its sequence has the row slots[b] of the resident table, whose first held[b]
//   entries are known already.  It needs ceil((starts[b] + lens[b]) / 64) of them; the missing ones are the next numbers of `pages`,
//   dealt to the rows in their order.  A place is page * 64 + position % 64.
//
// Every block adds up what the rows before its own bring and take (a few thousand cached numbers at most) instead of waiting for
// a scan: one launch, no scratch, no order among blocks.  What is written of the resident table is the row's own entries.  Where rows bring few
// tokens a block has eight of them, a warp each (2,000 rows of one token: 6.3 us with a block a row), where they bring many, a row has several
// blocks that take its tokens and pages in turn (8,000 tokens: 7.7 us with one block).  What is left is latency: a launch, and three fetches that
// depend on one another (lengths, a page, the store behind it).
#include "common.cuh"

#define ST_THREADS 256

struct StArgs {
    const int *slots, *starts, *lens, *held, *pages;
    int* resident;
    int *tok_pos, *tok_row, *row_first, *places, *tables;
    int rows, n_slots, res_width, n_pages, n_tokens, width;
};

__device__ __forceinline__ int st_need(int start, int len) { return (int)(((long long)start + len + PE_PAGE - 1) / PE_PAGE); }

template <int ROWS>                                                 // of a block
__global__ void __launch_bounds__(ST_THREADS) step_tables_kernel(const StArgs p) {
    constexpr int THREADS = ST_THREADS / ROWS;                      // of a row
    pdl_launch_dependents();
    pdl_wait();
    __shared__ int scratch[2][ST_THREADS / 32];
    const int b0 = blockIdx.x * ROWS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = threadIdx.x / THREADS, b = b0 + mine;
    // this block's rows, and tokens and new pages of those before it
    int n = 0, start = 0, held = 0, slot = -1;
    if (b < p.rows) { n = max(p.lens[b], 0); start = p.starts[b]; held = max(p.held[b], 0); slot = p.slots[b]; }
    int tokens = 0, taken = 0;
    for (int i = threadIdx.x; i < b0 + ROWS - 1 && i < p.rows; i += ST_THREADS) {
        const int len = max(p.lens[i], 0), fresh = max(st_need(p.starts[i], len) - max(p.held[i], 0), 0);
        if (ROWS == 1 || i < b0) { tokens += len; taken += fresh; }
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
    const int need = max(st_need(start, n), held);
    if constexpr (ROWS > 1) {                                       // and of the rows of the block before this one
        static_assert(ROWS == ST_THREADS / 32, "a warp a row");
        __syncthreads();
        if (lane == 0) { scratch[0][warp] = n; scratch[1][warp] = need - held; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ROWS; ++w)
            if (w < mine) { tokens += scratch[0][w]; taken += scratch[1][w]; }
    }
    if (b >= p.rows) return;

    int* row = slot >= 0 && slot < p.n_slots ? p.resident + (size_t)slot * p.res_width : nullptr;
    auto page_of = [&](int w) {                                     // entry w of the row's table
        if (!row || w < 0 || w >= p.res_width || w >= need) return -1;
        if (w < held) return row[w];
        const int at = taken + w - held;
        return at < p.n_pages ? p.pages[at] : -1;
    };
    const int first = threadIdx.x % THREADS + blockIdx.y * THREADS, step = THREADS * gridDim.y;
    if (first == 0) {
        p.row_first[b] = tokens;
        if (b == p.rows - 1) p.row_first[p.rows] = tokens + n;
    }
#pragma unroll 4
    for (int i = first; i < min(n, p.n_tokens - tokens); i += step) {
        const int at = start + i, page = page_of(at / PE_PAGE);
        p.tok_pos[tokens + i] = at;
        p.tok_row[tokens + i] = b;
        p.places[tokens + i] = page >= 0 ? page * PE_PAGE + at % PE_PAGE : -1;
    }
#pragma unroll 4
    for (int w = first; w < p.width; w += step) p.tables[(size_t)b * p.width + w] = page_of(w);
    if (row)
        for (int w = held + first; w < min(need, p.res_width); w += step) row[w] = page_of(w);
}

extern "C" int pe_step_tables(const int* slots, const int* starts, const int* lens, const int* held, const int* pages, int n_pages, int* resident,
                              int n_slots, int res_width, int rows, int* tok_pos, int* tok_row, int* row_first, int* places, int n_tokens,
                              int* tables, int width, void* stream) {
    if (rows <= 0) return 0;
    if (n_slots <= 0 || res_width <= 0 || width <= 0 || n_tokens < 0 || n_pages < 0) return PE_ERR_UNSUPPORTED;
    const StArgs p = {slots, starts, lens, held, pages, resident, tok_pos, tok_row, row_first, places, tables, rows, n_slots, res_width, n_pages, n_tokens, width};
    if (rows >= 256 && n_tokens <= 8 * rows) {
        PE_TRY(pe_launch(step_tables_kernel<ST_THREADS / 32>, (rows + ST_THREADS / 32 - 1) / (ST_THREADS / 32), ST_THREADS, 0, (cudaStream_t)stream, p));
    } else {
        const int most = 592 / rows < 1 ? 1 : 592 / rows, wanted = (n_tokens / rows + ST_THREADS - 1) / ST_THREADS;      // four blocks an SM at most
        PE_TRY(pe_launch(step_tables_kernel<1>, dim3(rows, wanted < 1 ? 1 : wanted < most ? wanted : most), ST_THREADS, 0, (cudaStream_t)stream, p));
    }
    PE_LAUNCH_CHECK();
    return 0;
}
