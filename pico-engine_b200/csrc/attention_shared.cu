// Attention of single tokens of which several share the first part of their sequences: the answers to one prompt.  Their page tables name
// the same pages for the shared positions, each row has pages of its own behind them.
//
//   o = sum_j w_j v_j / (sum_j w_j + e^sink),   w_j = exp(scale q.k_j - slope (pos - j)),   j <= pos, j > pos - window or j < keep_first
//
// The first kernel works through two lines of steps, a step being two pages (128 keys) of a key head.
//   shared   the positions of a group's prompt, once for all its rows: rows (tokens x query heads of a key head) fill the 128 rows of a
//            tensor-core tile (attention_decode.cu has the 16 of one token, and reads the prompt once a row).
//   own      each row's positions behind them.
// The work lies in two lines.  Shared: the steps of the tiles, group after group, in each the key heads, in each the tiles of 128 rows; a CTA takes a chunk of
// one tile, or (more tiles than half the CTAs) a run of several (AsDeal).  Own: the pages of the tiles of 16 heads, token after token, in each the key
// heads; every one of a CTA's AS_WORKERS warps takes a run of them, and runs differ by one page at most, whatever the rows' lengths.  There is a CTA an SM, and
// each works on one line; how many take which goes by what their steps and pages cost (as_split).  (CTAs that took some of both went through two starts
// and two ends: 64 answers of 28 heads of 128 on five prompts took 33 us instead of 29.)  Each CTA and each worker leaves sums, maxima and weights of its tiles' rows in scratch
// (float32).  The second kernel joins them, a block a token and key head: m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m).
//
//   warp 0      loader: a tile's queries as one box [tokens][heads of the key head][64 columns], and two pages of keys and values a step
//   warp 1      issues S = Q.K^T three steps ahead of O += P.V
//   warps 4-11  shared: softmax, two warpgroups that take the steps in turn (as in attention_prefill_tcgen05.cu); at the end of a tile both write
//               their half of O.  Own: every warp goes its own way through its run, a page at a time with mma.sync; it asks for the next page itself when
//               it has read the one before.  (Two warpgroups that shared a page and met at two barriers took 2,000 cycles for it.)
//
// What bounds it (64 answers of 14 heads on 31,744 positions, 25.6 us; cycles of a CTA of shared steps): its share of the work 6,300, the first step's keys 5,100, 16
// steps of 1,365 each (their exponentials alone are 1,024; a polynomial on the multiply-add units in the place of a quarter of them made a step longer, since a
// warp's instructions then are what it waits for), the end 4,000; the join's three fetches that depend on one another 4.3 us.  With few shared positions the own
// pages are fetched at 3.8 TB/s once they have begun.  The computing warps keep a row's 128 scores in registers: with 168 a thread the masked variant spilled 500
// bytes, and answers in a window took 25.2 us instead of 21.2 (40 to 68 bytes are spilled still).
//
// P is bfloat16 on both lines, since that is what the tensor cores multiply at their rate; a rounding is 2^-8 of a probability at most, of either sign, and the sums of weights
// are of the unrounded ones.  With the reference point up to 2^AS_LAZY below the maximum the largest probabilities are rounded as well, where a maximum taken exactly makes them
// 1: 0.0021 to 0.0023 of the outputs' size from the 64-bit result, row by row 0.0018.  How pages are dealt out goes by all rows of the call, so a row's bits depend on its neighbours.
//
// All keys of a shared step are visible to all rows but for windows, pages that are not there and the half step behind an odd number of pages,
// so the masks are a variant of their own (MASKED).  Every wait is bounded; one that runs out sets *status to 7, and the roles leave their loops.
#ifndef PE_HEAD_DIM
#error "compile with -DPE_HEAD_DIM=<head size>"
#endif
#include "tcgen05_attention.cuh"

#if PE_HEAD_DIM == 64 || PE_HEAD_DIM == 128

#define AS_HD PE_HEAD_DIM
#define AS_QTILE 128
#define AS_KTILE (2 * PE_PAGE)                     // keys of a step
#define AS_PANELS (AS_HD / 64)
#define AS_STAGES (AS_HD == 64 ? 5 : 3)
#define AS_AHEAD 3
#define AS_THREADS 384                             // three warpgroups: loader, issuer and two warps without work; two that compute
#define AS_REGS_SERVE 72
#define AS_REGS_COMPUTE 216                        // of a thread: 128 x 72 + 256 x 216 = 384 x 168, what the block is launched with (as_launch looks)
#define AS_WORKERS (AS_HD == 64 ? 8 : 6)           // warps that read own pages: each has half a stage, a page of keys and values
#define AS_OTILE 16                                // rows of an own tile
#define AS_OQ_BYTES (AS_OTILE * AS_HD * 2)         // queries of an own tile
#define AS_PAGE_BYTES (PE_PAGE * AS_HD * 2)        // keys (or values) of a page
#define AS_Q_BYTES (AS_QTILE * AS_HD * 2)
#define AS_OUT_BYTES (8 * 1024)                    // in front of the own tiles' queries: the tokens' places in the two lines
#define AS_QAREA_BYTES (AS_Q_BYTES > AS_OUT_BYTES + AS_WORKERS * AS_OQ_BYTES ? AS_Q_BYTES : AS_OUT_BYTES + AS_WORKERS * AS_OQ_BYTES)
#define AS_HALF_BYTES (AS_KTILE * AS_HD * 2)       // keys (or values) of a step
#define AS_STAGE_BYTES (2 * AS_HALF_BYTES)
#define AS_TILE_BYTES (AS_QAREA_BYTES + AS_STAGES * AS_STAGE_BYTES)
static_assert(AS_QAREA_BYTES % 1024 == 0 && 2 * AS_STAGES >= AS_WORKERS, "own pages use the places of the shared ones");
#define AS_BUFFERS 3
#define AS_BARS ((5 + 3 * AS_BUFFERS + 4 * AS_STAGES + 8 + 3 * AS_WORKERS + 1) / 2 * 2)      // (what follows them lies on 16 bytes)
#define AS_WALKS 11                                // the first tile; a working warp's each
#define AS_SMEM_BYTES (AS_TILE_BYTES + 8 * AS_BARS + 2 * AS_QTILE * 4 + AS_WALKS * (int)sizeof(AsWalk) + AS_WORKERS * (int)sizeof(AsOwnWalk) + 4 * (AS_THREADS / 32) * 4)
#define AS_O_COL (AS_BUFFERS * AS_KTILE)
#define AS_LAZY 8.0f
#define AS_MIN_STEPS 2                             // steps of a chunk or run at least, where there are as many
#define AS_MAX_TOKENS 1024                         // whose places in the two lines fit where results leave otherwise
#define AS_MAX_CTAS 160
static_assert(2 * AS_MAX_TOKENS * 4 <= AS_OUT_BYTES, "the tokens' places");
#define AS_MOST_OWN 256                            // runs that a row's own part may lie with, and two more at its ends
#define AS_JOIN_THREADS 512

struct AsScratch {
    int4* plan;                                     // [T][own tiles of all key heads]: where the join finds a row's parts (AsPart)
    float* sums;                                    // [rows][head size]
    float4* ends;                                   // [rows]: reference point (a maximum, in powers of two) and weight of either warpgroup's steps; sums
                                                    //         are relative to the larger of the two
    float* own_sums; float2* own_ends;              // the same of own tiles: maximum, weight
};
struct AsArgs {
    const int4* groups; const int* block_table; int table_stride; const int* tok_pos; const int* tok_row;
    int T, nh, nkv, window, keep_first; float scale_log2e; const float* slopes; float inv_scale;
    int pool_rows, early, grid, least_own; const bf16* q; int q_stride;
    int R, per_tile, own_tiles;                     // query heads of a key head; tokens of a shared tile; own tiles of a token and key head
    AsScratch scratch;
};

// The positions that token t reads with its group; 0: it reads all by itself (alone in its group, or not a group of this step)
__device__ __forceinline__ int as_shared(const int4& g, int t, int T, int table_stride) {
    if (g.y < 2 || g.x < 0 || t < g.x || g.y > T - g.x || t >= g.x + g.y || g.w < g.x || g.w >= g.x + g.y) return 0;
    return max(0, min(g.z / PE_PAGE, table_stride - 1)) * PE_PAGE;
}
// Pages in the order they are read: page j is j < kept ? j : page_lo + j - kept.
struct AsPages {
    int kept, page_lo, n;
    __device__ __forceinline__ int at(int j) const { return j < kept ? j : page_lo + j - kept; }
    __device__ __forceinline__ int steps() const { return (n + 1) / 2; }
    // of the first `end` pages those that a query at `pos` or behind can see
    __device__ __forceinline__ void set(int end, int pos, int window, int keep_first) {
        kept = page_lo = 0;
        n = end;
        if (window > 0) {
            const int keep_pages = min((keep_first + PE_PAGE - 1) / PE_PAGE, end);
            page_lo = min(max(pos - window + 1, 0) / PE_PAGE, end);
            if (page_lo <= keep_pages) page_lo = 0; else kept = keep_pages;
            n = kept + end - page_lo;
        }
    }
};
// How `steps` steps of `tiles` tiles are dealt to `grid` CTAs.
//   chunks  where there are twice as many CTAs as tiles: every tile is cut into chunks of at most `chunk` steps, a chunk a CTA.  (A run that went on into
//           the next tile cost the CTA 6,000 cycles for queries, the pipeline's start and its end, as much as four steps.)
//   runs    else: the steps in their line, in runs that differ by one at most, so a CTA has several tiles and a tile may lie with several CTAs
struct AsRuns {
    int ctas, each, more;                           // the first `more` runs have each + 1, the others each
    __device__ __forceinline__ AsRuns(int steps, int least, int most) {
        ctas = min((steps + least - 1) / least, most);
        each = ctas > 0 ? steps / ctas : 0;
        more = steps - each * ctas;
    }
    __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int cta_of(int s) const { return s < more * (each + 1) ? s / (each + 1) : more + (s - more * (each + 1)) / each; }
};
struct AsDeal {
    int chunk;                                      // most steps of a chunk; 0: runs
    AsRuns runs;
    __device__ __forceinline__ AsDeal(int steps, int tiles, int grid) : runs(steps, AS_MIN_STEPS, grid) {
        chunk = 2 * tiles <= grid && steps > 0 ? max((steps + grid - tiles - 1) / (grid - tiles), AS_MIN_STEPS) : 0;
    }
    // units (chunks or steps) of a tile of n steps
    __device__ __forceinline__ int units(int n) const { return chunk ? (n + chunk - 1) / chunk : n; }
    // the CTAs [x, y) that have the tile of n steps with `before` units in front of it
    __device__ __forceinline__ int2 ctas_of(int before, int n) const { return chunk ? make_int2(before, before + units(n)) : make_int2(runs.cta_of(before), runs.cta_of(before + n - 1) + 1); }
};

// How many of the CTAs take shared steps.  Measured (cycles of a CTA, on top of what both kinds need): a step 1,490, an own page 440 (its warps together), and a
// CTA of shared steps needs the time of three more; with heads of 128 1,930, 1,270 and five (a fifth less or more of a step's cost takes 2 to 10 % longer).  Both kinds end together where
// step (steps / s + more) = page pages / (grid - s).
__device__ __forceinline__ int as_split(int steps, int tiles, int pages, int grid) {
    constexpr float step = AS_HD == 64 ? 1490.f : 1930.f, page = AS_HD == 64 ? 440.f : 1270.f, more = AS_HD == 64 ? 3.f : 5.f;
    if (steps == 0) return 0;
    const float b = more * step * grid - step * steps - page * pages, a2 = 2.f * more * step;
    const int s = __float2int_rn((b + sqrtf(b * b + 2.f * a2 * step * steps * grid)) / a2);
    return min(max(min(s, steps / AS_MIN_STEPS + tiles), 1), grid - 1);
}

__device__ __forceinline__ int as_tiles(const int4& g, const AsArgs& p) { return (g.y + p.per_tile - 1) / p.per_tile; }

// What a token stands for: the group that starts with it (tiles: 0 where none does), and its own part, which counts from the end of the shared positions
struct AsGroup {
    int4 g; AsPages pages; int t, row, before, tiles;       // row: the batch row whose page table names the shared pages; before: units; tiles: of all key heads
    __device__ __forceinline__ int steps() const { return tiles > 0 ? pages.steps() * tiles : 0; }
    __device__ __forceinline__ int units(const AsDeal& d) const { return tiles > 0 ? d.units(pages.steps()) * tiles : 0; }
    __device__ __forceinline__ void load(const AsArgs& p, int first) {
        t = first;
        g = p.groups[t];
        row = p.tok_row[t];                                  // (without a window every row of the group names all shared pages)
        tiles = 0;
        const int shared = g.x == t ? as_shared(g, t, p.T, p.table_stride) : 0;
        if (shared == 0) return;
        if (p.window > 0) row = p.tok_row[g.w];
        pages.set(shared / PE_PAGE, p.window > 0 ? p.tok_pos[g.w] : 0, p.window, p.keep_first);
        tiles = pages.n > 0 ? as_tiles(g, p) * p.nkv : 0;
    }
};
struct AsOwn {
    int t, row, skip, pos, before, steps; AsPages pages;     // steps: a page of a tile each
    __device__ __forceinline__ void set(const AsArgs& p, int token, const int4& g) {
        t = token;
        row = p.tok_row[t];
        const int at = max(p.tok_pos[t], 0);
        skip = min(as_shared(g, t, p.T, p.table_stride), at / PE_PAGE * PE_PAGE);
        pos = at - skip;
        pages.set(min(pos / PE_PAGE + 1, p.table_stride - skip / PE_PAGE), pos, p.window, max(p.keep_first - skip, 0));      // (no further than the table)
        steps = pages.n * p.nkv * p.own_tiles;
    }
    __device__ __forceinline__ void load(const AsArgs& p, int token) { set(p, token, p.groups[token]); }
};
// A CTA's tiles one after the other.  Every warp walks its own copy, in shared memory: one lane takes the step, all of them read.
struct AsWalk {
    AsGroup now;
    int x, end;                                    // the next unit, and where the CTA's end
    int kvh, tile, first, count;                   // the tile, and its steps here
    const int* table;                              // the page table's row that names the shared pages
    __device__ __forceinline__ void place(const AsArgs& p, const AsDeal& d) {
        table = p.block_table + (size_t)now.row * p.table_stride;
        const int n = now.pages.steps(), units = d.units(n), tiles = as_tiles(now.g, p), o = x - now.before, seg = o / units, j = o - seg * units;
        kvh = seg / tiles; tile = seg - kvh * tiles;
        first = d.chunk ? (int)((unsigned)n * j / units) : j;        // (n: half a table row at most, units: the CTAs)
        count = d.chunk ? (int)((unsigned)n * (j + 1) / units) - first : min(n - first, end - x);
    }
    __device__ __forceinline__ bool step(const AsArgs& p, const AsDeal& d) {
        x += d.chunk ? 1 : count;
        if (x >= end) return false;
        while (x >= now.before + now.units(d)) {
            const int before = now.before + now.units(d);
            now.load(p, now.t + (now.tiles > 0 ? now.g.y : 1));
            now.before = before;
        }
        place(p, d);
        return true;
    }
};
struct AsOwnWalk {
    AsOwn now;
    int x, end, kvh, tile, first, count;
    const int* table;
    __device__ __forceinline__ bool step(const AsArgs& p, const AsDeal&) {
        x += count;
        if (x >= end) return false;
        bool moved = count == 0;
        while (x >= now.before + now.steps) {
            const int before = now.before + now.steps;
            now.load(p, now.t + 1);
            now.before = before;
            moved = true;
        }
        if (moved) table = p.block_table + (size_t)now.row * p.table_stride + now.skip / PE_PAGE;
        const int o = x - now.before, n = now.pages.n, tiles = p.own_tiles, seg = o / n;
        first = o - seg * n;
        kvh = seg / tiles; tile = seg - kvh * tiles;
        count = min(n - first, end - x);
        return true;
    }
};
template <typename W>
__device__ __forceinline__ bool as_next(W& w, const AsArgs& p, const AsDeal& d, int lane) {       // the whole warp
    bool more = false;
    __syncwarp();
    if (lane == 0) more = w.step(p, d);
    __syncwarp();
    return __shfl_sync(0xffffffffu, more, 0);
}
// Where CTA c leaves the rows of a tile (tokens x heads of key head kvh), in rows: blocks of different pairs of CTA and tile do not meet, since from one
// pair to the next the CTA or the tile moves on, and with it 128 (16) rows or those of the tile.
__device__ __forceinline__ size_t as_block(int c, const int4& g, const AsArgs& p, int kvh, int tile) {
    return (size_t)c * AS_QTILE + (size_t)g.x * p.nh + (size_t)kvh * g.y * p.R + tile * (p.per_tile * p.R);
}
// (c: a worker's run)
__device__ __forceinline__ size_t as_own_block(int c, int t, const AsArgs& p, int kvh, int tile) {
    return (size_t)c * AS_OTILE + (size_t)t * p.nh + kvh * p.R + tile * AS_OTILE;
}

__device__ __forceinline__ void as_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void as_matrices(unsigned (&r)[4], unsigned at) {     // four 8 x 8 matrices, a row's address a lane
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void as_matrices_turned(unsigned (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// where 16-byte group `chunk` of a row of an own page's keys or values lies: panels of 64 columns, 128-byte swizzle
__device__ __forceinline__ unsigned as_at(unsigned page, int row, int chunk) {
    return page + (chunk >> 3) * (PE_PAGE * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

template <bool MASKED>
__global__ void __launch_bounds__(AS_THREADS, 1) attention_shared_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AsArgs p, int* status) {
    extern __shared__ __align__(1024) unsigned char as_mem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned q_s = at_smem(as_mem), kv_s = q_s + AS_QAREA_BYTES;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(as_mem + AS_TILE_BYTES);
    unsigned& tmem_base_s = *reinterpret_cast<unsigned*>(bars);
    unsigned long long *q_full = bars + 1, *q_empty = bars + 2, *o_empty = bars + 3, *o_full = bars + 4;
    unsigned long long *s_full = bars + 5, *p_full = s_full + AS_BUFFERS, *pv_done = p_full + AS_BUFFERS;
    unsigned long long *k_full = pv_done + AS_BUFFERS, *v_full = k_full + AS_STAGES, *k_empty = v_full + AS_STAGES, *v_empty = k_empty + AS_STAGES;
    unsigned long long* told = v_empty + AS_STAGES;                 // [warpgroup][32 rows]: a step's reference points are there
    unsigned long long *own_q = told + 8, *own_k = own_q + AS_WORKERS, *own_v = own_k + AS_WORKERS;      // [worker]: what it has asked for is there
    float* refs = reinterpret_cast<float*>(bars + AS_BARS);         // [warpgroup][row]: reference point of the group's last step
    AsWalk* walks = reinterpret_cast<AsWalk*>(refs + 2 * AS_QTILE);
    static_assert((AS_TILE_BYTES + 8 * AS_BARS + 2 * AS_QTILE * 4) % alignof(AsWalk) == 0 && sizeof(AsWalk) % alignof(AsOwnWalk) == 0, "the walks' places");
    AsOwnWalk* own_walk = reinterpret_cast<AsOwnWalk*>(walks + AS_WALKS);        // each worker's first own tile
    int *shared_at = reinterpret_cast<int*>(as_mem), *own_at = shared_at + AS_MAX_TOKENS;       // of a CTA with own pages: units in front of a group, pages in front of a token
    int (*scan)[AS_THREADS / 32] = reinterpret_cast<int (*)[AS_THREADS / 32]>(own_walk + AS_WORKERS);
    if (q_s & 1023u) {                                              // every thread alike: nothing is allocated yet
        if (threadIdx.x == 0) atomicExch(status, 6);
        return;
    }
    // The description of the step was there before the kernels in front began, or (early == 0) they have ended: p.early says which.  So have the
    // shared pages.  Queries, and the scratch that the call before may still be reading, wait.
    if (!p.early) pdl_wait();

    // ---- this CTA's share of the steps: all steps and tiles, then a scan over the groups' units and the tokens' pages (a token a thread; tokens beyond are
    // read again)
    AsGroup group;
    AsOwn own;
    auto load = [&](int t) {
        group.tiles = own.steps = 0;
        if (t < p.T) { group.load(p, t); own.set(p, t, group.g); }
    };
    load(threadIdx.x);
    if (warp == 1) {                                                // (while that travels; behind the shares it cost answers in a window 1.0 of 26.3 us)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at_smem(&tmem_base_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        auto init = [](unsigned long long* bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(at_smem(bar)), "r"(count) : "memory"); };
        init(q_full, 1); init(q_empty, 8); init(o_empty, 8); init(o_full, 1);         // q_empty: the eight warps that write the tile's results
        for (int s = 0; s < AS_STAGES; ++s) { init(&k_full[s], 1); init(&v_full[s], 1); init(&k_empty[s], 1); init(&v_empty[s], 1); }
        for (int b = 0; b < AS_BUFFERS; ++b) { init(&s_full[b], 1); init(&p_full[b], 4); init(&pv_done[b], 1); }
        for (int w = 0; w < 8; ++w) init(&told[w], 1);
        for (int w = 0; w < AS_WORKERS; ++w) { init(&own_q[w], 1); init(&own_k[w], 1); init(&own_v[w], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    const bool few = p.T <= AS_THREADS;
    int total[3] = {0, 0, 0};                                       // steps, tiles, own pages
    for (int base = 0; base < p.T; base += AS_THREADS) {
        if (base > 0) load(base + threadIdx.x);
        total[0] += group.steps(); total[1] += group.tiles; total[2] += own.steps;
    }
    auto sum_to = [&](int v) {                                      // of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += up;
        }
        return v;
    };
    int own_sum = sum_to(total[2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { total[0] += __shfl_xor_sync(0xffffffffu, total[0], o); total[1] += __shfl_xor_sync(0xffffffffu, total[1], o); }
    if (lane == 31) { scan[0][warp] = total[0]; scan[1][warp] = total[1]; scan[2][warp] = own_sum; }
    __syncthreads();
    total[0] = total[1] = total[2] = 0;
    own.before = own_sum - own.steps;                               // (few)
#pragma unroll
    for (int w = 0; w < AS_THREADS / 32; ++w) {
        if (w < warp) own.before += scan[2][w];
        total[0] += scan[0][w]; total[1] += scan[1][w]; total[2] += scan[2][w];
    }
    const int cta = blockIdx.x, split = as_split(total[0], total[1], total[2], p.grid), own_cta = cta - split, own_ctas = p.grid - split;
    const AsDeal deal(total[0], total[1], split);
    const AsRuns own_runs(total[2], p.least_own, AS_WORKERS * own_ctas);
    int begin = cta, end = cta + 1, units = 0, own_units = 0;       // this CTA's units of the first line; all so far
    if (cta >= split) begin = end = 0;
    else if (!deal.chunk) { begin = end = 0; if (cta < deal.runs.ctas) { begin = deal.runs.begin(cta); end = deal.runs.begin(cta + 1); } }
    for (int base = 0; base < p.T; base += AS_THREADS) {
        if (!few) load(base + threadIdx.x);
        const int mine = group.units(deal), sum = sum_to(mine);
        own_sum = few ? 0 : sum_to(own.steps);
        __syncthreads();
        if (lane == 31) { scan[3][warp] = sum; if (!few) scan[2][warp] = own_sum; }
        __syncthreads();
        group.before = units + sum - mine;
        if (!few) own.before = own_units + own_sum - own.steps;
#pragma unroll
        for (int w = 0; w < AS_THREADS / 32; ++w) {
            if (w < warp) group.before += scan[3][w];
            units += scan[3][w];
            if (!few) {
                if (w < warp) own.before += scan[2][w];
                own_units += scan[2][w];
            }
        }
        const int t = base + (int)threadIdx.x;
        if (own_cta >= 0 && t < p.T) { shared_at[t] = group.before; own_at[t] = own.before; }
        if (begin < end && begin >= group.before && begin < group.before + mine) {
            AsWalk& w = walks[0];
            w.now = group; w.x = begin; w.end = end;
            w.place(p, deal);                                       // the first tile
        }
        unsigned mine_too = 0;                                      // the workers whose runs begin with this token
        if (own_cta >= 0) {
#pragma unroll
            for (int w = 0; w < AS_WORKERS; ++w) {
                const int run = own_cta + w * own_ctas, from = own_runs.begin(run);
                if (run < own_runs.ctas && from >= own.before && from < own.before + own.steps) mine_too |= 1u << w;
            }
        }
        for (; mine_too; mine_too &= mine_too - 1) {
            const int w = __ffs(mine_too) - 1, run = own_cta + w * own_ctas;
            AsOwnWalk& z = own_walk[w];
            z.now = own; z.x = own_runs.begin(run); z.end = own_runs.begin(run + 1); z.count = 0;
            z.step(p, deal);
        }
    }
    // (the first worker's run comes first; where no row has an own page, the first of these CTAs is there for the plan)
    const bool has_shared = begin < min(end, units), has_own = own_cta >= 0 && own_cta < max(own_runs.ctas, 1);
    if (!has_shared && warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_s), "r"(512u) : "memory");
    if (!has_shared && !has_own) {                                  // (the whole block)
        pdl_wait();
        pdl_launch_dependents();
        return;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base_s;
    const int R = p.R, per_tile = p.per_tile, pool_pages = p.pool_rows / (p.nkv * PE_PAGE);
    // a page that is not there is read from beyond the pool's end, which gives zeros
    auto rows_of = [&](int page, int kvh) { return (unsigned)page < (unsigned)pool_pages ? (page * p.nkv + kvh) * PE_PAGE : p.pool_rows; };
    // what worker k reads (one lane): a page's keys or values into its half of a stage, a tile's queries (they lie side by side) into its part of theirs
    auto own_page = [&](const CUtensorMap* map, int k, int values, int y, unsigned long long* bar) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(bar)), "r"((unsigned)AS_PAGE_BYTES) : "memory");
#pragma unroll
        for (int c = 0; c < AS_PANELS; ++c) at_tma_2d(kv_s + (2 * k + values) * AS_PAGE_BYTES + c * (PE_PAGE * 128), map, 64 * c, y, at_smem(bar));
    };
    auto own_queries = [&](int k, const AsOwnWalk& z) {
        const unsigned bytes = min(AS_OTILE, R - z.tile * AS_OTILE) * AS_HD * 2;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(&own_q[k])), "r"(bytes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(q_s + AS_OUT_BYTES + k * AS_OQ_BYTES), "l"(p.q + (size_t)z.now.t * p.q_stride + (size_t)(z.kvh * R + z.tile * AS_OTILE) * AS_HD), "r"(bytes), "r"(at_smem(&own_q[k])) : "memory");
    };
    // (the first tile has been found; a warp's own copy goes on from there)
    AsWalk& w = walks[warp < 2 ? warp + 1 : warp < 4 ? 0 : warp - 1];
    if (lane == 0 && has_shared && (warp < 2 || warp >= 4)) w = walks[0];
    __syncwarp();
    auto advance = [&](int seg) { return seg == 0 ? has_shared : as_next(w, p, deal, lane); };
    // the same of own tiles, in the same place when the others are done
    AsOwnWalk& ow = *reinterpret_cast<AsOwnWalk*>(&w);
    static_assert(sizeof(AsOwnWalk) <= sizeof(AsWalk) && alignof(AsWalk) >= alignof(AsOwnWalk), "the own walk takes the other's place");

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AS_REGS_SERVE));
    if (warp == 0 && has_own) {                                     // ---------------- the plan of the join, while the workers read
        pdl_wait();                                                 // (scratch is written)
        const int all = p.T * p.nkv * p.own_tiles, ctas = min(own_ctas, max(own_runs.ctas, 1));
        for (int e = own_cta * 32 + lane; e < all; e += ctas * 32) {
            const int tok = e / (p.nkv * p.own_tiles), of = e - tok * (p.nkv * p.own_tiles), kvh = of / p.own_tiles, tile = of - kvh * p.own_tiles;
            const int4 g = p.groups[tok];
            AsOwn row;
            row.set(p, tok, g);
            int o0 = 0, on = 0;
            if (row.pages.n > 0) {                                  // (none: the window of a position beyond the table has left all of its pages behind)
                const int first = own_at[tok] + of * row.pages.n;
                o0 = own_runs.cta_of(first);
                on = min(own_runs.cta_of(first + row.pages.n - 1) + 1 - o0, AS_MOST_OWN + 2);      // (more only for positions behind max_context)
            }
            int c0 = 0, n = 0, at = 0;
            const int shared = as_shared(g, tok, p.T, p.table_stride);
            AsPages pages = {0, 0, 0};
            if (shared > 0) pages.set(shared / PE_PAGE, p.window > 0 ? p.tok_pos[g.w] : 0, p.window, p.keep_first);
            if (pages.n > 0) {
                const int i = tok - g.x, group_tile = i / per_tile;
                const int2 c = deal.ctas_of(shared_at[g.x] + (kvh * as_tiles(g, p) + group_tile) * deal.units(pages.steps()), pages.steps());
                c0 = c.x;
                n = c.y - c.x;
                at = (int)as_block(c0, g, p, kvh, group_tile) + (i - group_tile * per_tile) * R + tile * AS_OTILE;
            }
            p.scratch.plan[e] = make_int4(n, on, at, (int)as_own_block(o0, tok, p, kvh, tile));
        }
    } else if (warp == 0) {                                                // ---------------- loader: one lane asks, the others wait for the walk
        bool ok = true;
        int it = 0, asked_k = 0, asked_v = 0, asked_q = 0;
                // keys and values of two pages (rows y of the pools) into the stage of step `it`
        auto bring = [&](const int (&y)[2]) {
            const int s = it % AS_STAGES;
            auto is_free = [&](unsigned long long* empty) { return it < AS_STAGES || at_wait(at_smem(empty), (unsigned)(it / AS_STAGES - 1) & 1u); };
            auto load = [&](const CUtensorMap* map, unsigned dst, unsigned long long* bar) {
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(bar)), "r"((unsigned)AS_HALF_BYTES) : "memory");
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int c = 0; c < AS_PANELS; ++c) at_tma_2d(dst + c * (AS_KTILE * 128) + x * (PE_PAGE * 128), map, 64 * c, y[x], at_smem(bar));
            };
            if (!is_free(&k_empty[s])) return false;
            load(&map_k, kv_s + s * AS_STAGE_BYTES, &k_full[s]);
            asked_k = it + 1;
            if (!is_free(&v_empty[s])) return false;
            load(&map_v, kv_s + s * AS_STAGE_BYTES + AS_HALF_BYTES, &v_full[s]);
            asked_v = ++it;
            return true;
        };
        for (int seg = 0; ok && advance(seg); ++seg) {
            if (lane == 0) {
                const int count = w.count, first = w.first, kvh = w.kvh;
                const AsPages pages = w.now.pages;
                const int* table = w.table;
                auto page_of = [&](int j) { return j < pages.n ? table[pages.at(j)] : -1; };
                auto ask_q = [&] {
                    if (seg > 0 && !at_wait(at_smem(q_empty), (unsigned)(seg - 1) & 1u)) return false;
                    pdl_wait();
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(q_full)), "r"((unsigned)(per_tile * R * AS_HD * 2)) : "memory");
#pragma unroll
                    for (int c = 0; c < AS_PANELS; ++c)
                        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                                     ::"r"(q_s + c * (AS_QTILE * 128)), "l"(&map_q), "r"(at_smem(q_full)), "r"(64 * c), "r"(kvh * R), "r"(w.now.g.x + w.tile * per_tile) : "memory");
                    ++asked_q;
                    return true;
                };
                int page[2] = {page_of(2 * first), page_of(2 * first + 1)};
                if (seg > 0) ok = ask_q();                          // (the first tile's behind its first step: keys and values need not wait for the kernel in front)
                for (int i = 0; ok && i < count; ++i) {
                    const int y[2] = {rows_of(page[0], kvh), rows_of(page[1], kvh)};
                    if (i + 1 < count) { page[0] = page_of(2 * (first + i) + 2); page[1] = page_of(2 * (first + i) + 3); }       // travel during the waits
                    ok = bring(y);
                    if (ok && seg == 0 && i == 0) ok = ask_q();
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        if (!ok && lane == 0) {                                     // what has been asked for lands before the block ends
            atomicExch(status, 7);
            if (asked_q > 0) at_wait(at_smem(q_full), (unsigned)(asked_q - 1) & 1u);
            for (int n = max(0, asked_k - AS_STAGES); n < asked_k; ++n) at_wait(at_smem(&k_full[n % AS_STAGES]), (unsigned)(n / AS_STAGES) & 1u);
            for (int n = max(0, asked_v - AS_STAGES); n < asked_v; ++n) at_wait(at_smem(&v_full[n % AS_STAGES]), (unsigned)(n / AS_STAGES) & 1u);
        }
    } else if (warp == 1) {                                         // ---------------- MMA issuer: the warp waits, one thread issues
        // Behind the allocation, and behind the end of the kernel in front: the next kernel counts on both (it reads queries and keys without a wait)
        pdl_wait();
        pdl_launch_dependents();
        const unsigned elected = pe_elect();
        const unsigned idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(AS_KTILE >> 3) << 17) | ((unsigned)(AS_QTILE >> 4) << 24);
        const unsigned idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((unsigned)(AS_HD >> 3) << 17) | ((unsigned)(AS_QTILE >> 4) << 24);
        const unsigned long long dq = at_desc(q_s, 0, 1024), dk = at_desc(kv_s, 0, 1024), dv = at_desc(kv_s + AS_HALF_BYTES, AS_KTILE * 128, 1024);
        bool ok = true;
        auto issue_s = [&](int it) -> bool {
            const int s = it % AS_STAGES, b = it % AS_BUFFERS;
            if (it >= AS_BUFFERS && !at_wait_warp(at_smem(&pv_done[b]), (unsigned)(it / AS_BUFFERS - 1) & 1u)) return false;
            if (!at_wait_warp(at_smem(&k_full[s]), (unsigned)(it / AS_STAGES) & 1u)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned long long dks = dk + (unsigned long long)(s * (AS_STAGE_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < AS_HD / 16; ++kk) {
                const unsigned off_q = ((kk / 4) * (AS_QTILE * 128) + (kk % 4) * 32) >> 4, off_k = ((kk / 4) * (AS_KTILE * 128) + (kk % 4) * 32) >> 4;
                at_mma(elected, tmem + b * AS_KTILE, dq + off_q, dks + off_k, idesc_s, kk > 0 ? 1u : 0u);
            }
            at_commit_by(elected, at_smem(&k_empty[s]));
            at_commit_by(elected, at_smem(&s_full[b]));
            return true;
        };
        int it = 0;
        for (int seg = 0; ok && advance(seg); ++seg) {              // S never runs into the next tile: its queries come when this one's results have left their place
            const int count = w.count;
            ok = at_wait_warp(at_smem(q_full), (unsigned)seg & 1u);
            for (int i = 0; ok && i < min(AS_AHEAD, count); ++i) ok = issue_s(it + i);
            for (int i = 0; ok && i < count; ++i, ++it) {
                const int s = it % AS_STAGES, b = it % AS_BUFFERS;
                if (!at_wait_warp(at_smem(&v_full[s]), (unsigned)(it / AS_STAGES) & 1u)) { ok = false; break; }
                if (!at_wait_warp(at_smem(&p_full[b]), (unsigned)(it / AS_BUFFERS) & 1u)) { ok = false; break; }
                if (i == 0 && seg > 0 && !at_wait_warp(at_smem(o_empty), (unsigned)(seg - 1) & 1u)) { ok = false; break; }     // the tile before has left O
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned long long dvs = dv + (unsigned long long)(s * (AS_STAGE_BYTES >> 4));
#pragma unroll
                for (int kk = 0; kk < AS_KTILE / 16; ++kk)
                    at_mma_ts(elected, tmem + AS_O_COL, tmem + b * AS_KTILE + kk * 8, dvs + ((kk * 16 * 128) >> 4), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
                at_commit_by(elected, at_smem(&v_empty[s]));
                at_commit_by(elected, at_smem(&pv_done[b]));
                if (i + 1 == count) at_commit_by(elected, at_smem(o_full));
                if (i + AS_AHEAD < count && !issue_s(it + AS_AHEAD)) { ok = false; break; }
            }
        }
        if (!ok) atomicExch(status, 7);
    }
    } else {                                                        // ---------------- softmax, warps 4..11
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AS_REGS_COMPUTE));
        const int quarter = warp & 3;                               // the 32 lanes of tensor memory this warp may touch
        const int g = (warp - 4) >> 2;                              // the warpgroup: steps g, g + 2, ..
        const int r = quarter * 32 + lane;                          // this thread's row of the tile
        const unsigned lane_addr = tmem + ((unsigned)(quarter * 32) << 16);
        const unsigned long long scale2 = at_two(p.scale_log2e, p.scale_log2e);
        pdl_wait();                                                 // (scratch is written)
        bool ok = true;
        int it0 = 0;                                                // the CTA's steps before this tile
        for (int seg = 0; ok && advance(seg); ++seg) {
            const int count = w.count, first = w.first;
            const int odd_end = w.now.pages.n & 1 ? w.now.pages.n / 2 - first : -1;       // the step whose second page is not there
            const int rows = min(per_tile, w.now.g.y - w.tile * per_tile) * R;
            const bool live = r < rows;
            int pos = 0;
            float slope = 0.f;
            if (MASKED && live) {
                pos = p.tok_pos[w.now.g.x + w.tile * per_tile + r / R];
                if (p.slopes) slope = p.slopes[w.kvh * R + r % R] * p.inv_scale;
            }
            float m_mine = -INFINITY, l_mine = 0.f;
            const int i0 = (g ^ it0) & 1;                           // the group's first step of this tile
            auto page_of = [&](int j) { return j < w.now.pages.n ? w.table[w.now.pages.at(j)] : -1; };
            int page[2] = {0, 0};                                   // (masked: entries of the page table, asked for a step ahead)
            if (MASKED && i0 < count) { page[0] = page_of(2 * (first + i0)); page[1] = page_of(2 * (first + i0) + 1); }
            for (int i = i0; i < count; i += 2) {
                const int it = it0 + i, b = it % AS_BUFFERS;
                const unsigned s_addr = lane_addr + b * AS_KTILE;
                bool there[2] = {live, live && i != odd_end};
                if (MASKED) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) there[x] = live && (unsigned)page[x] < (unsigned)pool_pages;
                    if (i + 2 < count) { page[0] = page_of(2 * (first + i + 2)); page[1] = page_of(2 * (first + i + 2) + 1); }
                }
                if (!at_wait_warp(at_smem(&s_full[b]), (unsigned)(it / AS_BUFFERS) & 1u)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                unsigned raw[AS_KTILE];
#pragma unroll
                for (int c = 0; c < 4; ++c) at_ld32_start(s_addr + 32 * c, raw + 32 * c);
                at_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; ++c) at_pin32(raw + 32 * c);
                float s[AS_KTILE], base[2] = {0.f, 0.f}, mx[8];
#pragma unroll
                for (int c = 0; c < AS_KTILE; ++c) s[c] = __uint_as_float(raw[c]);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float* sx = s + x * PE_PAGE;
                    if (!there[x]) {
                        at_mask_behind<PE_PAGE>(sx, -1);
                    } else if (MASKED) {
                        const int key0 = w.now.pages.at(2 * (first + i) + x) * PE_PAGE;
                        if (p.window > 0 && key0 <= pos - p.window && key0 + PE_PAGE - 1 >= p.keep_first) {
                            const int lo = pos - p.window + 1 - key0, kept_here = p.keep_first - key0;
#pragma unroll
                            for (int c = 0; c < PE_PAGE; ++c)
                                if (c < lo && c >= kept_here) sx[c] = -INFINITY;
                        }
                        if (p.slopes) {                             // the distance's share: what grows along the page here, the page's own part in `base`
                            base[x] = slope * (float)(key0 - pos);
#pragma unroll
                            for (int c = 0; c < PE_PAGE; ++c) sx[c] = fmaf(slope, (float)c, sx[c]);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) mx[4 * x + c] = fmaxf(fmaxf(sx[c], sx[c + 4]), sx[c + 8]);
#pragma unroll
                    for (int c = 12; c < PE_PAGE - 4; c += 8) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[4 * x + k] = fmaxf(fmaxf(mx[4 * x + k], sx[c + k]), sx[c + 4 + k]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[4 * x + k] = fmaxf(mx[4 * x + k], sx[PE_PAGE - 4 + k]);
                }
                const float m_step = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) + base[0], fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])) + base[1]);
                // the row's reference point up to the step before, from the other warpgroup (asked for at a tile's first step too: a wait by
                // parity has to see every phase)
                float m_run = -INFINITY;
                if (it > 0) {
                    if (!at_wait_warp(at_smem(&told[4 * (g ^ 1) + quarter]), (unsigned)((it - 1) >> 1) & 1u)) { ok = false; break; }
                    if (i > 0) m_run = refs[(g ^ 1) * AS_QTILE + r];
                }
                const float m_tile = m_step * p.scale_log2e;
                const float m_new = (m_run != -INFINITY && m_tile <= m_run + AS_LAZY) ? m_run : fmaxf(m_run, m_tile);
                refs[g * AS_QTILE + r] = m_new;
                __syncwarp();
                if (lane == 0) at_arrive(at_smem(&told[4 * g + quarter]));
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = m_run == -INFINITY ? 1.0f : at_exp2(m_run - m_use);
                l_mine *= m_mine == -INFINITY ? 1.0f : at_exp2(m_mine - m_use);
                m_mine = m_new;
                unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float packed[PE_PAGE / 2];
                    const float off = fmaf(base[x], p.scale_log2e, -m_use);
#pragma unroll
                    for (int c = 0; c < PE_PAGE; c += 2) packed[c >> 1] = __uint_as_float(at_exp2_pair(s[x * PE_PAGE + c], s[x * PE_PAGE + c + 1], scale2, at_two(off, off), sum[(c >> 1) & 1]));
                    at_st32(s_addr + x * (PE_PAGE / 2), packed);
                }
                l_mine += at_sum_four(sum[0], sum[1]);
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    if (!at_wait_warp(at_smem(&pv_done[(it - 1) % AS_BUFFERS]), (unsigned)((it - 1) / AS_BUFFERS) & 1u)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int c = 0; c < AS_HD; c += 32) {
                        float o[32];
                        at_ld32(lane_addr + AS_O_COL + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] *= alpha;
                        at_st32(lane_addr + AS_O_COL + c, o);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) at_arrive(at_smem(&p_full[b]));
            }
            if (!ok) break;
            // ---- the tile's end: both groups write their half of O, and the reference point and sum of their own steps.  (Reference points only grow, and
            // the last step's is what O goes by: the larger of the two.)
            it0 += count;
            // (A barrier of the tile's, of which every warp sees every phase.  pv_done[last % 3] would not do: where values come late, the group that took the step before
            // the last can be here before the products of last - 3 are done, and a wait by parity takes the phase before those for the last one.)
            if (!at_wait_warp(at_smem(o_full), (unsigned)seg & 1u)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const size_t block = as_block(cta, w.now.g, p, w.kvh, w.tile);
            if (live) reinterpret_cast<float2*>(p.scratch.ends + block + r)[g] = make_float2(m_mine, l_mine);
            // through the stages (the tile's products have read them, the next tile's come when this is done), 32 columns of the warp's 32 rows at a time, 16-byte
            // pieces exchanged by the row inside a run of eight: a lane storing its own row would touch 32 lines an instruction
            const unsigned stage = kv_s + (warp - 4) * 4096;
            float* to = p.scratch.sums + block * AS_HD + g * (AS_HD / 2);
#pragma unroll
            for (int c = 0; c < AS_HD / 2; c += 32) {
                float o[32];
                at_ld32(lane_addr + AS_O_COL + g * (AS_HD / 2) + c, o);
                if (c + 32 == AS_HD / 2) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) at_arrive(at_smem(o_empty));
                }
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128 + ((k ^ (lane & 7)) << 4)), "f"(o[4 * k]), "f"(o[4 * k + 1]), "f"(o[4 * k + 2]), "f"(o[4 * k + 3]) : "memory");
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {                       // four rows an instruction
                    const int x = 4 * k + (lane >> 3), row = quarter * 32 + x;
                    float4 v;
                    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(stage + x * 128 + (((lane & 7) ^ (x & 7)) << 4)) : "memory");
                    if (row < rows) *reinterpret_cast<float4*>(to + (size_t)row * AS_HD + c + 4 * (lane & 7)) = v;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (what comes next there comes by another proxy)
            __syncwarp();
            if (lane == 0) at_arrive(at_smem(q_empty));
        }
        // ---------------- own pages (of a CTA that has no shared steps): worker k's run
        const int k = warp - 4, gr = lane >> 2, tq = lane & 3;      // fragment row and column of the lane
        bool more = has_own && k < AS_WORKERS && own_cta + k * own_ctas < own_runs.ctas;
        __syncwarp();
        if (lane == 0 && more) ow = own_walk[k];
        __syncwarp();
        const unsigned oq_s = q_s + AS_OUT_BYTES + k * AS_OQ_BYTES, keys = kv_s + 2 * k * AS_PAGE_BYTES, values = keys + AS_PAGE_BYTES;
        unsigned turn = 0, q_turn = 0, asked_k = 1, asked_v = 1, asked_q = 1;       // pages and tiles so far, and what has been asked for
        const bool mine = more;
        if (lane == 0 && more) {                                    // the first page
            const int y = rows_of(ow.table[ow.now.pages.at(ow.first)], ow.kvh);
            own_queries(k, ow);
            own_page(&map_k, k, 0, y, &own_k[k]);
            own_page(&map_v, k, 1, y, &own_v[k]);
        }
        while (more) {
            const AsOwn row = ow.now;
            const int kvh = ow.kvh, tile = ow.tile, head0 = tile * AS_OTILE, heads = min(AS_OTILE, R - head0), count = ow.count, first = ow.first;
            const int keep = max(p.keep_first - row.skip, 0), lo = p.window > 0 ? max(row.pos - p.window + 1, 0) : 0;
            const int* table = ow.table;
            int entry = table[row.pages.at(first)];
            more = as_next(ow, p, deal, lane);                            // the tile behind this one
            float slope[2] = {0.f, 0.f};
            if (p.slopes) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (gr + 8 * x < heads) slope[x] = p.slopes[kvh * R + head0 + gr + 8 * x] * p.inv_scale;
            }
            unsigned qf[AS_HD / 16][4];
            if (!at_wait_warp(at_smem(&own_q[k]), q_turn++ & 1u)) { ok = false; break; }
#pragma unroll
            for (int c = 0; c < AS_HD / 16; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x) {                       // rows gr, gr + 8; columns 2 tq, 2 tq + 8 of the 16
                    const int j = gr + 8 * (x & 1);
                    qf[c][x] = 0u;
                    if (j < heads) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(qf[c][x]) : "r"(oq_s + (j * AS_HD + c * 16 + 8 * (x >> 1) + 2 * tq) * 2) : "memory");
                }
            float acc[AS_HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < AS_HD / 8; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
            for (int i = 0; i < count; ++i, ++turn) {
                const int key0 = row.pages.at(first + i) * PE_PAGE;
                const bool there = (unsigned)entry < (unsigned)pool_pages;
                int y_next = -1;                                    // the page behind this one, of this tile or of the next
                if (i + 1 < count) { entry = table[row.pages.at(first + i + 1)]; y_next = 0; }
                else if (more) { entry = ow.table[ow.now.pages.at(ow.first)]; y_next = 0; }
                const int kvh_next = i + 1 < count ? kvh : ow.kvh;
                if (!at_wait_warp(at_smem(&own_k[k]), turn & 1u)) { ok = false; break; }
                // S of 16 rows and 64 keys
                float sc[8][4];
#pragma unroll
                for (int x = 0; x < 8; ++x) sc[x][0] = sc[x][1] = sc[x][2] = sc[x][3] = 0.f;
#pragma unroll
                for (int c = 0; c < AS_HD / 16; ++c) {              // four fetches in front of the products that wait for them
                    unsigned kf[4][4];                              // keys 0-7 and 8-15 of 16, columns 0-7 and 8-15
#pragma unroll
                    for (int x = 0; x < 4; ++x) as_matrices(kf[x], as_at(keys, x * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * c + ((lane >> 3) & 1)));
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        as_mma(sc[2 * x], qf[c], kf[x][0], kf[x][1]);
                        as_mma(sc[2 * x + 1], qf[c], kf[x][2], kf[x][3]);
                    }
                }
                __syncwarp();
                if (y_next >= 0) y_next = rows_of(entry, kvh_next);
                if (lane == 0 && y_next >= 0) {                     // the keys have been read: the next ones, and behind the tile's last page the next tile's queries
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    if (i + 1 == count) { own_queries(k, ow); ++asked_q; }
                    own_page(&map_k, k, 0, y_next, &own_k[k]);
                    ++asked_k;
                }
                float top[2] = {-INFINITY, -INFINITY};
                const bool whole = there && key0 + PE_PAGE - 1 <= row.pos && key0 >= lo && !p.slopes;
                if (!whole) {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + x * 8 + 2 * tq + (e & 1);
                            if (p.slopes) sc[x][e] = fmaf(-slope[e >> 1], (float)(row.pos - key), sc[x][e]);
                            if (!there || key > row.pos || (key < lo && key >= keep)) sc[x][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int x = 0; x < 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], sc[x][e]);
                float alpha[2], use[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
                    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
                    const float m_new = fmaxf(m[x], top[x] * p.scale_log2e);
                    use[x] = m_new == -INFINITY ? 0.f : m_new;
                    alpha[x] = m[x] == -INFINITY ? 0.f : at_exp2(m[x] - use[x]);
                    m[x] = m_new;
                    l[x] *= alpha[x];
                }
                unsigned pf[4][4];                                  // P as it is the first operand of P V: 16 keys a fragment
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    float e[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) { e[n] = at_exp2(fmaf(sc[x][n], p.scale_log2e, -use[n >> 1])); l[n >> 1] += e[n]; }
                    pf[x >> 1][2 * (x & 1)] = at_pack(e[0], e[1]);
                    pf[x >> 1][2 * (x & 1) + 1] = at_pack(e[2], e[3]);
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int c = 0; c < AS_HD / 8; ++c) { acc[c][0] *= alpha[0]; acc[c][1] *= alpha[0]; acc[c][2] *= alpha[1]; acc[c][3] *= alpha[1]; }
                }
                if (!at_wait_warp(at_smem(&own_v[k]), turn & 1u)) { ok = false; break; }
                // values behind the newest token become zero: a page is taken as its last owner left it, and a weight of zero would not keep a value that is
                // no number out of the sums
                if (there && key0 + PE_PAGE - 1 > row.pos) {
                    const int clean = row.pos - key0 + 1;
                    for (int x = lane; x < (PE_PAGE - clean) * (AS_HD / 8); x += 32)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(as_at(values, clean + x / (AS_HD / 8), x % (AS_HD / 8))), "r"(0u) : "memory");
                    __syncwarp();
                }
#pragma unroll
                for (int c = 0; c < AS_HD / 8; c += 2) {            // sixteen columns of four times 16 keys
                    unsigned vf[4][4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) as_matrices_turned(vf[x], as_at(values, x * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        as_mma(acc[c], pf[x], vf[x][0], vf[x][1]);
                        as_mma(acc[c + 1], pf[x], vf[x][2], vf[x][3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0 && y_next >= 0) { own_page(&map_v, k, 1, y_next, &own_v[k]); ++asked_v; }
            }
            if (!ok) break;
            // ---- the end of the tile's pages here
            const size_t block = as_own_block(own_cta + k * own_ctas, row.t, p, kvh, tile);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int j = gr + 8 * x;
                if (j >= heads) continue;
                if (tq == 0) p.scratch.own_ends[block + j] = make_float2(m[x], l[x]);
                float* to = p.scratch.own_sums + (block + j) * AS_HD + 2 * tq;
#pragma unroll
                for (int c = 0; c < AS_HD / 8; ++c) *reinterpret_cast<float2*>(to + c * 8) = make_float2(acc[c][2 * x], acc[c][2 * x + 1]);
            }
        }
        if (!ok && mine && lane == 0) {                             // what has been asked for lands before the block ends
            at_wait(at_smem(&own_q[k]), (asked_q - 1) & 1u);
            at_wait(at_smem(&own_k[k]), (asked_k - 1) & 1u);
            at_wait(at_smem(&own_v[k]), (asked_v - 1) & 1u);
        }
        if (!ok) atomicExch(status, 7);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1 && has_shared) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The join: a block a token and (16 heads of a) key head.
__global__ void __launch_bounds__(AS_JOIN_THREADS) attention_join_kernel(const __grid_constant__ AsArgs p, bf16* out, const float* sinks) {
    __shared__ float weights[AS_MAX_CTAS + AS_MOST_OWN + 2][AS_OTILE], weight_of[AS_OTILE];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = blockIdx.y, R = p.R;
    const int kvh = blockIdx.x / p.own_tiles, tile = blockIdx.x - kvh * p.own_tiles, head0 = tile * AS_OTILE, heads = min(AS_OTILE, R - head0);
    pdl_wait();
    const int4 plan = p.scratch.plan[tok * gridDim.x + blockIdx.x];
    const int n = min(max(plan.x, 0), AS_MAX_CTAS), on = min(max(plan.y, 0), AS_MOST_OWN + 2);       // results of shared steps, and of own pages
    const size_t row = plan.z, own_row = plan.w;
    // thread x has output x % AS_HD of head x / AS_HD.  The first results of either kind are asked for at once, beside what the weights are made of: a fetch of what
    // another SM has just written takes 1,200 cycles or more, and rows seldom have more results than these
    constexpr int FIRST = 16, FIRST_OWN = 2;
    const float *from = p.scratch.sums + row * AS_HD, *own_from = p.scratch.own_sums + own_row * AS_HD;
    float v[FIRST], u[FIRST_OWN];
    auto ask = [&](int x) {
#pragma unroll
        for (int e = 0; e < FIRST; ++e) v[e] = e < n && x < heads * AS_HD ? from[x + e * (AS_QTILE * AS_HD)] : 0.f;
#pragma unroll
        for (int e = 0; e < FIRST_OWN; ++e) u[e] = e < on && x < heads * AS_HD ? own_from[x + e * (AS_OTILE * AS_HD)] : 0.f;
    };
    ask(threadIdx.x);
    // ---- weights, a warp a head, a partial result a lane
    for (int h = warp; h < heads; h += AS_JOIN_THREADS / 32) {
        auto end_of = [&](int e) {                                  // reference points and weights; sums go by the larger one
            if (e < n) return p.scratch.ends[row + h + (size_t)e * AS_QTILE];
            const float2 o = p.scratch.own_ends[own_row + h + (size_t)(e - n) * AS_OTILE];
            return make_float4(o.x, o.y, -INFINITY, 0.f);
        };
        float4 mine = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
        if (lane < n + on) mine = end_of(lane);
        float top = fmaxf(mine.x, mine.z), sum = 0.f;
#pragma unroll 1
        for (int e = lane + 32; e < n + on; e += 32) { const float4 at = end_of(e); top = fmaxf(top, fmaxf(at.x, at.z)); }
        top = warp_max(top);
        const auto weight = [&](float at) { return at == -INFINITY ? 0.f : at_exp2(at - top); };
#pragma unroll 1
        for (int e = lane; e < n + on; e += 32) {
            const float4 at = e == lane ? mine : end_of(e);
            sum = fmaf(at.y, weight(at.x), fmaf(at.w, weight(at.z), sum));
            weights[e][h] = weight(fmaxf(at.x, at.z));
        }
        sum = warp_sum(sum);
        if (sinks) sum += exp2f(fmaf(sinks[kvh * R + head0 + h], 1.4426950408889634f, -top));      // (a row that saw no key: 2^inf, and 1 / sum = 0)
        if (lane == 0) weight_of[h] = sum > 0.f ? 1.f / sum : 0.f;
    }
    __syncthreads();
    // ---- sums
#pragma unroll 1
    for (int x = threadIdx.x; x < heads * AS_HD; x += AS_JOIN_THREADS) {
        const int h = x / AS_HD;
        if (x >= AS_JOIN_THREADS) ask(x);
        float o = 0.f;
        auto add = [&](float value, int e) { const float at = weights[e][h]; o = at == 0.f ? o : fmaf(value, at, o); };
#pragma unroll
        for (int e = 0; e < FIRST; ++e) if (e < n) add(v[e], e);
#pragma unroll 4
        for (int e = FIRST; e < n; ++e) add(from[x + (size_t)e * (AS_QTILE * AS_HD)], e);
#pragma unroll
        for (int e = 0; e < FIRST_OWN; ++e) if (e < on) add(u[e], n + e);
#pragma unroll 4
        for (int e = FIRST_OWN; e < on; ++e) add(own_from[x + e * (AS_OTILE * AS_HD)], n + e);
        out[((size_t)tok * p.nh + kvh * R + head0) * AS_HD + x] = __float2bfloat16_rn(o * weight_of[h]);
    }
}

namespace {

// queries of `tokens` rows, `stride` elements apart, as boxes of [box_tokens][box_heads][64 columns]
int as_query_map(CUtensorMap* map, const void* q, long long tokens, int heads, long long stride, int box_heads, int box_tokens) {
    at_encode_fn enc = at_encoder();
    if (!enc) return PE_ERR_UNSUPPORTED;
    const cuuint64_t dims[3] = {(cuuint64_t)AS_HD, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)AS_HD * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, elem[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 20000 + (int)r;
}

static_assert(AS_SMEM_BYTES <= 227 * 1024, "shared memory of a block");

template <bool MASKED>
int as_launch(int grid, cudaStream_t stream, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AsArgs& p, int* status) {
    static bool wide = false;
    if (!wide) {
        PE_TRY(cudaFuncSetAttribute(attention_shared_kernel<MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AS_SMEM_BYTES));
        cudaFuncAttributes made;
        PE_TRY(cudaFuncGetAttributes(&made, attention_shared_kernel<MASKED>));
        if (made.numRegs * AS_THREADS < 128 * AS_REGS_SERVE + 256 * AS_REGS_COMPUTE) return PE_ERR_UNSUPPORTED;      // the computing warps would wait for registers for good
        wide = true;
    }
    PE_TRY(pe_launch(attention_shared_kernel<MASKED>, dim3(grid), AS_THREADS, AS_SMEM_BYTES, stream, mq, mk, mv, p, status));
    PE_LAUNCH_CHECK();
    return 0;
}

long long as_plan_bytes(int T, int nh, int nkv) { return ((long long)T * nkv * ((nh / nkv + AS_OTILE - 1) / AS_OTILE) * 16 + 255) / 256 * 256; }
int as_grid() { return pe_sm_count() < AS_MAX_CTAS ? pe_sm_count() : AS_MAX_CTAS; }
long long as_rows(int T, int nh) { return (long long)as_grid() * AS_QTILE + (long long)T * nh; }
long long as_own_rows(int T, int nh) { return (long long)AS_WORKERS * as_grid() * AS_OTILE + (long long)T * nh; }

}  // namespace

extern "C" long long pe_attention_shared_scratch(int T, int nh, int nkv) {
    return as_plan_bytes(T, nh, nkv) + as_rows(T, nh) * (AS_HD * 4 + 16) + as_own_rows(T, nh) * (AS_HD * 4 + 8);
}

extern "C" int pe_attention_shared(const void* q, int q_stride, void* out, const void* k_pool, const void* v_pool, long long pool_pages,
                                   const int* block_table, int table_stride, const int* tok_pos, const int* tok_row, const void* groups, int T,
                                   int nh, int nkv, int hd, int window, int keep_first, float scale, int max_context, const float* slopes,
                                   const float* sinks, int early_pages, void* scratch, int* status, void* stream) {
    if (T <= 0) return 0;
    if (hd != AS_HD || nkv <= 0 || nh % nkv || nh / nkv > AS_QTILE || q_stride % 8 || !(scale > 0.f) || !status || !scratch || keep_first < 0 || table_stride < 1) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)groups | (uintptr_t)scratch) & 15) return PE_ERR_UNSUPPORTED;
    if (pool_pages * nkv * PE_PAGE > 0x7fffff00ll) return PE_ERR_UNSUPPORTED;       // TMA coordinates are 32-bit
    const int R = nh / nkv;
    if (T > AS_MAX_TOKENS || as_rows(T, nh) > 0x7fffffff || (long long)T * nkv * ((R + AS_OTILE - 1) / AS_OTILE) * (table_stride + 1ll) > 0x7fffffffll) return PE_ERR_UNSUPPORTED;      // steps are counted in 32 bits
    CUtensorMap mq, mk, mv;
    int rc = as_query_map(&mq, q, T, nh, q_stride, R, AS_QTILE / R);
    if (rc) return rc;
    rc = at_make_map(&mk, k_pool, pool_pages * nkv * PE_PAGE, hd, hd, PE_PAGE);
    if (rc) return rc;
    rc = at_make_map(&mv, v_pool, pool_pages * nkv * PE_PAGE, hd, hd, PE_PAGE);
    if (rc) return rc;
    AsArgs p = {};
    p.groups = (const int4*)groups; p.block_table = block_table; p.table_stride = table_stride; p.tok_pos = tok_pos; p.tok_row = tok_row;
    p.T = T; p.nh = nh; p.nkv = nkv; p.window = window; p.keep_first = window > 0 ? keep_first : 0; p.scale_log2e = scale * 1.4426950408889634f;
    p.slopes = slopes; p.inv_scale = 1.0f / scale; p.pool_rows = (int)(pool_pages * nkv * PE_PAGE);
    p.R = R; p.per_tile = AS_QTILE / R; p.own_tiles = (R + AS_OTILE - 1) / AS_OTILE;
    p.early = early_pages != 0; p.grid = as_grid();
    p.least_own = ((max_context + PE_PAGE - 1) / PE_PAGE + AS_MOST_OWN - 1) / AS_MOST_OWN;       // a row's own part lies with AS_MOST_OWN runs at most
    p.q = (const bf16*)q; p.q_stride = q_stride;
    char* at = (char*)scratch;
    p.scratch.plan = (int4*)at; at += as_plan_bytes(T, nh, nkv);
    p.scratch.ends = (float4*)at; at += as_rows(T, nh) * 16;
    p.scratch.sums = (float*)at; at += as_rows(T, nh) * AS_HD * 4;
    p.scratch.own_sums = (float*)at; at += as_own_rows(T, nh) * AS_HD * 4;
    p.scratch.own_ends = (float2*)at;
    rc = window > 0 || slopes ? as_launch<true>(p.grid, (cudaStream_t)stream, mq, mk, mv, p, status) : as_launch<false>(p.grid, (cudaStream_t)stream, mq, mk, mv, p, status);
    if (rc) return rc;
    PE_TRY(pe_launch(attention_join_kernel, dim3(nkv * ((R + AS_OTILE - 1) / AS_OTILE), T), AS_JOIN_THREADS, 0, (cudaStream_t)stream, p, (bf16*)out, sinks));
    PE_LAUNCH_CHECK();
    return 0;
}

#else   // other head sizes: the rows of a group are read one by one (attention_decode.cu)

extern "C" long long pe_attention_shared_scratch(int, int, int) { return 0; }
extern "C" int pe_attention_shared(const void*, int, void*, const void*, const void*, long long, const int*, int, const int*, const int*, const void*,
                                   int, int, int, int, int, int, float, int, const float*, const float*, int, void*, int*, void*) {
    return PE_ERR_UNSUPPORTED;
}

#endif
