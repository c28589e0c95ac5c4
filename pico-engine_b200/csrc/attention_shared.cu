// Attention of single tokens of which several share the first part of their sequences: the answers to one prompt.  Their page tables name
// the same pages for the shared positions, each row has pages of its own behind them.
//
//   o = sum_j w_j v_j / (sum_j w_j + e^sink),   w_j = exp(scale q.k_j - slope (pos - j)),   j <= pos, j > pos - window or j < keep_first
//
// This kernel reads the shared positions, once for all rows of a group: rows (tokens x query heads of a key head) fill the 128 rows of a
// tensor-core tile, where attention_decode.cu has the 16 of one token.  Its partial results (sums, maximum, weight of a row, in float32) go to
// scratch, and the kernel of attention_decode.cu, which follows and reads each row's own positions, joins them:
// m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m).
//
//   a CTA an SM takes an equal share of all steps (attention_shared.cuh)
//   warp 0      loader: the tile's queries as one box [tokens][heads of the key head][64 columns], and two pages of keys and values a step
//   warp 1      issues S = Q.K^T three steps ahead of O += P.V
//   warps 2-9   softmax, two warpgroups that take the steps in turn (as in attention_prefill_tcgen05.cu); at the end of a tile both write their half of O
//
// All keys of a step are visible to all rows but for windows, pages that are not there and the half step behind an odd number of pages, so
// the masks are a variant of their own (MASKED).  Every wait is bounded; one that runs out sets *status to 7 and the roles leave their loops.
#ifndef PE_HEAD_DIM
#error "compile with -DPE_HEAD_DIM=<head size>"
#endif
#include "tcgen05_attention.cuh"
#include "attention_shared.cuh"

#if PE_HEAD_DIM == 64 || PE_HEAD_DIM == 128

#define AS_HD PE_HEAD_DIM
#define AS_KTILE (2 * PE_PAGE)                     // keys of a step
#define AS_PANELS (AS_HD / 64)
#define AS_STAGES (AS_HD == 64 ? 5 : 3)
#define AS_AHEAD 3
#define AS_THREADS AS_COUNTED
#define AS_Q_BYTES (AS_QTILE * AS_HD * 2)
#define AS_HALF_BYTES (AS_KTILE * AS_HD * 2)       // keys (or values) of a step
#define AS_STAGE_BYTES (2 * AS_HALF_BYTES)
#define AS_TILE_BYTES (AS_Q_BYTES + AS_STAGES * AS_STAGE_BYTES)
#define AS_BUFFERS 3
#define AS_BARS ((4 + 3 * AS_BUFFERS + 4 * AS_STAGES + 8 + 1) / 2 * 2)      // (what follows them lies on 16 bytes)
#define AS_WALKS (AS_THREADS / 32 + 1)             // the first tile; a warp's each
#define AS_SMEM_BYTES (AS_TILE_BYTES + 8 * AS_BARS + 2 * AS_QTILE * 4 + AS_WALKS * (int)sizeof(AsWalk) + 2 * (AS_THREADS / 32) * 4)
#define AS_O_COL (AS_BUFFERS * AS_KTILE)
#define AS_LAZY 8.0f

struct AsArgs {
    const int4* groups; const int* block_table; int table_stride; const int* tok_pos; const int* tok_row;
    int T, nh, nkv, window, keep_first; float scale_log2e; const float* slopes; float inv_scale;
    int pool_rows, early; AsScratch scratch;
};

// A CTA's tiles one after the other.  Every warp walks its own copy, in shared memory: one lane takes the step, all of them read.
struct AsWalk {
    AsGroup now;
    int x, end;                                    // the next unit, and where the CTA's end
    int kvh, tile, first, count;                   // the tile, and its steps here
    const int* table;                              // the page table's row that names the shared pages
    __device__ __forceinline__ void load(const AsArgs& p, int t) { now.load(p.groups, p.tok_pos, p.tok_row, t, p.T, p.table_stride, p.nh, p.nkv, p.window, p.keep_first); }
    __device__ __forceinline__ void place(const AsArgs& p, const AsDeal& d) {
        table = p.block_table + (size_t)now.row * p.table_stride;
        const int n = as_tile_steps(now.pages), units = d.units(n), tiles = as_tiles(now.g, p.nh, p.nkv), o = x - now.before, seg = o / units, j = o - seg * units;
        kvh = seg / tiles; tile = seg - kvh * tiles;
        first = d.chunk ? (int)((long long)n * j / units) : j;
        count = d.chunk ? (int)((long long)n * (j + 1) / units) - first : min(n - first, end - x);
    }
    __device__ __forceinline__ bool step(const AsArgs& p, const AsDeal& d) {
        x += d.chunk ? 1 : count;
        if (x >= end) return false;
        while (x >= now.before + now.units(d)) {
            const int before = now.before + now.units(d);
            load(p, now.t + (now.tiles > 0 ? now.g.y : 1));
            now.before = before;
        }
        place(p, d);
        return true;
    }
    __device__ __forceinline__ bool next(const AsArgs& p, const AsDeal& d, int lane) {        // the whole warp
        bool more = false;
        __syncwarp();
        if (lane == 0) more = step(p, d);
        __syncwarp();
        return __shfl_sync(0xffffffffu, more, 0);
    }
};

template <bool MASKED>
__global__ void __launch_bounds__(AS_THREADS, 1) attention_shared_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AsArgs p, int* status) {
    extern __shared__ __align__(1024) unsigned char as_mem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned q_s = at_smem(as_mem), kv_s = q_s + AS_Q_BYTES;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(as_mem + AS_TILE_BYTES);
    unsigned& tmem_base_s = *reinterpret_cast<unsigned*>(bars);
    unsigned long long *q_full = bars + 1, *q_empty = bars + 2, *o_empty = bars + 3;
    unsigned long long *s_full = bars + 4, *p_full = s_full + AS_BUFFERS, *pv_done = p_full + AS_BUFFERS;
    unsigned long long *k_full = pv_done + AS_BUFFERS, *v_full = k_full + AS_STAGES, *k_empty = v_full + AS_STAGES, *v_empty = k_empty + AS_STAGES;
    unsigned long long* told = v_empty + AS_STAGES;                 // [warpgroup][32 rows]: a step's reference points are there
    float* refs = reinterpret_cast<float*>(bars + AS_BARS);         // [warpgroup][row]: reference point of the group's last step
    AsWalk* walks = reinterpret_cast<AsWalk*>(refs + 2 * AS_QTILE);
    static_assert((AS_TILE_BYTES + 8 * AS_BARS + 2 * AS_QTILE * 4) % alignof(AsWalk) == 0, "the walks' place");
    int (*scan)[AS_THREADS / 32] = reinterpret_cast<int (*)[AS_THREADS / 32]>(walks + AS_WALKS);
    if (q_s & 1023u) {                                              // every thread alike: nothing is allocated yet
        if (threadIdx.x == 0) atomicExch(status, 6);
        return;
    }
    // The description of the step was there before the kernels in front began, or (early == 0) they have ended: p.early says which.  So have the
    // shared pages.  Queries, and the scratch that the call before may still be reading, wait.
    if (!p.early) pdl_wait();

    // ---- this CTA's share of the steps: all steps and tiles, then a scan over the groups' units (a token a thread; tokens beyond are read again)
    AsGroup mine;
    auto load = [&](int t) {
        mine.tiles = 0;
        if (t < p.T) mine.load(p.groups, p.tok_pos, p.tok_row, t, p.T, p.table_stride, p.nh, p.nkv, p.window, p.keep_first);
    };
    load(threadIdx.x);
    if (threadIdx.x == 32) {
        auto init = [](unsigned long long* bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(at_smem(bar)), "r"(count) : "memory"); };
        init(q_full, 1); init(q_empty, 8); init(o_empty, 8);         // q_empty: the eight warps that write the tile's results through the queries' place
        for (int s = 0; s < AS_STAGES; ++s) { init(&k_full[s], 1); init(&v_full[s], 1); init(&k_empty[s], 1); init(&v_empty[s], 1); }
        for (int b = 0; b < AS_BUFFERS; ++b) { init(&s_full[b], 1); init(&p_full[b], 4); init(&pv_done[b], 1); }
        for (int w = 0; w < 8; ++w) init(&told[w], 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    int steps = 0, tiles = 0;
    for (int base = AS_THREADS; base < p.T; base += AS_THREADS) { steps += mine.steps(); tiles += mine.tiles; load(base + threadIdx.x); }
    steps += mine.steps(); tiles += mine.tiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { steps += __shfl_xor_sync(0xffffffffu, steps, o); tiles += __shfl_xor_sync(0xffffffffu, tiles, o); }
    if (lane == 0) { scan[0][warp] = steps; scan[1][warp] = tiles; }
    __syncthreads();
    steps = tiles = 0;
#pragma unroll
    for (int w = 0; w < AS_THREADS / 32; ++w) { steps += scan[0][w]; tiles += scan[1][w]; }
    const AsDeal deal(steps, tiles, gridDim.x);
    if (p.T > AS_THREADS) {
        load(threadIdx.x);
        if (blockIdx.x == 0 && threadIdx.x == 0) { pdl_wait(); p.scratch.before[p.T] = steps; p.scratch.before[p.T + 1] = tiles; }
    }
    int begin = 0, end = 0, units = 0;                              // this CTA's units, and all so far
    if (!deal.chunk && (int)blockIdx.x < deal.ctas) { begin = deal.begin(blockIdx.x); end = deal.begin(blockIdx.x + 1); }
    if (deal.chunk) { begin = blockIdx.x; end = begin + 1; }
    for (int base = 0; base < p.T; base += AS_THREADS) {
        if (base > 0) load(base + threadIdx.x);
        const int own = mine.units(deal);
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        __syncthreads();
        if (lane == 31) scan[0][warp] = sum;
        __syncthreads();
        mine.before = units + sum - own;
#pragma unroll
        for (int w = 0; w < AS_THREADS / 32; ++w) {
            if (w < warp) mine.before += scan[0][w];
            units += scan[0][w];
        }
        if (p.T > AS_COUNTED && blockIdx.x == 0 && base + (int)threadIdx.x < p.T) { pdl_wait(); p.scratch.before[base + threadIdx.x] = mine.before; }
        if (begin < end && begin >= mine.before && begin < mine.before + own) {
            AsWalk& w = walks[0];
            w.now = mine; w.x = begin; w.end = end;
            w.place(p, deal);                                       // the first tile
        }
    }
    if (begin >= units) end = begin;
    if (begin >= end) {                                             // (the whole block)
        pdl_wait();
        pdl_launch_dependents();
        return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at_smem(&tmem_base_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base_s;
    const int R = p.nh / p.nkv, per_tile = AS_QTILE / R, pool_pages = p.pool_rows / (p.nkv * PE_PAGE);
    // (the first tile has been found; a warp's own copy goes on from there)
    AsWalk& w = walks[warp + 1];
    if (lane == 0) w = walks[0];
    __syncwarp();
    auto advance = [&](int seg) { return seg == 0 ? true : w.next(p, deal, lane); };

    if (warp == 0) {                                                // ---------------- loader: one lane asks, the others wait for the walk
        bool ok = true;
        int it = 0, seg = 0, asked_k = 0, asked_v = 0, asked_q = 0;
        for (; ok && advance(seg); ++seg) {
            if (lane == 0) {
                const int count = w.count, first = w.first, kvh = w.kvh, n = w.now.pages.n;
                const int* table = w.table;
                const AsPages pages = w.now.pages;
                auto page_of = [&](int j) { return j < n ? table[pages.at(j)] : -1; };
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
                for (int i = 0; ok && i < count; ++i, ++it) {
                    const int s = it % AS_STAGES, j = 2 * (first + i);
                    const unsigned k_dst = kv_s + s * AS_STAGE_BYTES, v_dst = k_dst + AS_HALF_BYTES, round = (unsigned)(it / AS_STAGES - 1) & 1u;
                    // a page that is not there is read from beyond the pool's end, which gives zeros
                    const int y[2] = {(unsigned)page[0] < (unsigned)pool_pages ? (page[0] * p.nkv + kvh) * PE_PAGE : p.pool_rows,
                                      (unsigned)page[1] < (unsigned)pool_pages ? (page[1] * p.nkv + kvh) * PE_PAGE : p.pool_rows};
                    if (i + 1 < count) { page[0] = page_of(j + 2); page[1] = page_of(j + 3); }       // travel during the waits
                    auto bring = [&](const CUtensorMap* map, unsigned dst, unsigned long long* bar) {
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(bar)), "r"((unsigned)AS_HALF_BYTES) : "memory");
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int c = 0; c < AS_PANELS; ++c) at_tma_2d(dst + c * (AS_KTILE * 128) + x * (PE_PAGE * 128), map, 64 * c, y[x], at_smem(bar));
                    };
                    if (it >= AS_STAGES && !at_wait(at_smem(&k_empty[s]), round)) { ok = false; break; }
                    bring(&map_k, k_dst, &k_full[s]);
                    asked_k = it + 1;
                    if (it >= AS_STAGES && !at_wait(at_smem(&v_empty[s]), round)) { ok = false; break; }
                    bring(&map_v, v_dst, &v_full[s]);
                    asked_v = it + 1;
                    if (seg == 0 && i == 0) ok = ask_q();
                }
                if (!ok) {                                          // what has been asked for lands before the block ends
                    atomicExch(status, 7);
                    if (asked_q > 0) at_wait(at_smem(q_full), (unsigned)(asked_q - 1) & 1u);
                    for (int n = max(0, asked_k - AS_STAGES); n < asked_k; ++n) at_wait(at_smem(&k_full[n % AS_STAGES]), (unsigned)(n / AS_STAGES) & 1u);
                    for (int n = max(0, asked_v - AS_STAGES); n < asked_v; ++n) at_wait(at_smem(&v_full[n % AS_STAGES]), (unsigned)(n / AS_STAGES) & 1u);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
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
                if (i + AS_AHEAD < count && !issue_s(it + AS_AHEAD)) { ok = false; break; }
            }
        }
        if (!ok) atomicExch(status, 7);
    } else {                                                        // ---------------- softmax, warps 2..9
        const int quarter = warp & 3;                               // the 32 lanes of tensor memory this warp may touch
        const int g = (warp - 2) >> 2;                              // the warpgroup: steps g, g + 2, ..
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
            const int last = it0 + count - 1;
            it0 += count;
            if (!at_wait_warp(at_smem(&pv_done[last % AS_BUFFERS]), (unsigned)(last / AS_BUFFERS) & 1u)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const size_t block = as_block(blockIdx.x, w.now.g, p.nh, p.nkv, w.kvh, w.tile);
            if (live) reinterpret_cast<float2*>(p.scratch.ends + block + r)[g] = make_float2(m_mine, l_mine);
            // through the queries' place (the last S has read them), 16 columns of the warp's 32 rows at a time, 16-byte pieces exchanged by the row inside
            // a run of four: a lane storing its own row would touch 32 lines an instruction
            const unsigned stage = q_s + (warp - 2) * 2048;
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
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)), "f"(o[16 * half + 4 * k]), "f"(o[16 * half + 4 * k + 1]),
                                     "f"(o[16 * half + 4 * k + 2]), "f"(o[16 * half + 4 * k + 3]) : "memory");
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {                   // eight rows an instruction
                        const int x = 8 * k + (lane >> 2), row = quarter * 32 + x;
                        float4 v;
                        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(stage + x * 64 + (((lane & 3) ^ ((x >> 1) & 3)) << 4)) : "memory");
                        if (row < rows) *reinterpret_cast<float4*>(to + (size_t)row * AS_HD + c + 16 * half + 4 * (lane & 3)) = v;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (the next tile's queries come by another proxy)
            __syncwarp();
            if (lane == 0) at_arrive(at_smem(q_empty));
        }
        if (!ok) atomicExch(status, 7);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
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

template <bool MASKED>
int as_launch(int grid, cudaStream_t stream, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AsArgs& p, int* status) {
    static bool wide = false;
    if (!wide) {
        PE_TRY(cudaFuncSetAttribute(attention_shared_kernel<MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AS_SMEM_BYTES));
        wide = true;
    }
    PE_TRY(pe_launch(attention_shared_kernel<MASKED>, dim3(grid), AS_THREADS, AS_SMEM_BYTES, stream, mq, mk, mv, p, status));
    PE_LAUNCH_CHECK();
    return 0;
}

long long as_before_bytes(int T) { return ((long long)(T + 2) * 4 + 255) / 256 * 256; }
int as_grid() { return pe_sm_count() < AS_MAX_CTAS ? pe_sm_count() : AS_MAX_CTAS; }
long long as_rows(int T, int nh) { return (long long)as_grid() * AS_QTILE + (long long)T * nh; }

}  // namespace

extern "C" long long pe_attention_shared_scratch(int T, int nh) { return as_before_bytes(T) + as_rows(T, nh) * (AS_HD * 4 + 16); }

// the kernel of attention_decode.cu for the rows' own positions
int pe_attention_decode_own(const void* q, int q_stride, void* out, const void* k_pool, const void* v_pool, const int* block_table, int table_stride,
                            const int* tok_pos, const int* tok_row, int T, int nh, int nkv, int window, float scale, int max_context, int early_pages,
                            int* status, void* stream, int keep_first, const float* slopes, const float* sinks, const void* groups, const AsScratch& scratch, int grid);

extern "C" int pe_attention_shared(const void* q, int q_stride, void* out, const void* k_pool, const void* v_pool, long long pool_pages,
                                   const int* block_table, int table_stride, const int* tok_pos, const int* tok_row, const void* groups, int T,
                                   int nh, int nkv, int hd, int window, int keep_first, float scale, int max_context, const float* slopes,
                                   const float* sinks, int early_pages, void* scratch, int* status, void* stream) {
    if (T <= 0) return 0;
    if (hd != AS_HD || nkv <= 0 || nh % nkv || nh / nkv > AS_QTILE || q_stride % 8 || !(scale > 0.f) || !status || !scratch || keep_first < 0) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)groups | (uintptr_t)scratch) & 15) return PE_ERR_UNSUPPORTED;
    if (pool_pages * nkv * PE_PAGE > 0x7fffff00ll) return PE_ERR_UNSUPPORTED;       // TMA coordinates are 32-bit
    if ((long long)T * nkv * (table_stride / 2 + 1) > 0x7fffffffll) return PE_ERR_UNSUPPORTED;      // steps are counted in 32 bits
    const int R = nh / nkv;
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
    p.early = early_pages != 0;
    p.scratch.before = (int*)scratch;
    p.scratch.sums = (float*)((char*)scratch + as_before_bytes(T));
    p.scratch.ends = (float4*)(p.scratch.sums + as_rows(T, nh) * AS_HD);
    rc = window > 0 || slopes ? as_launch<true>(as_grid(), (cudaStream_t)stream, mq, mk, mv, p, status)
                              : as_launch<false>(as_grid(), (cudaStream_t)stream, mq, mk, mv, p, status);
    if (rc) return rc;
    return pe_attention_decode_own(q, q_stride, out, k_pool, v_pool, block_table, table_stride, tok_pos, tok_row, T, nh, nkv, window, scale, max_context,
                                   early_pages, status, stream, p.keep_first, slopes, sinks, groups, p.scratch, as_grid());
}

#else   // other head sizes: the rows of a group are read one by one (attention_decode.cu)

extern "C" long long pe_attention_shared_scratch(int, int) { return 0; }
extern "C" int pe_attention_shared(const void*, int, void*, const void*, const void*, long long, const int*, int, const int*, const int*, const void*,
                                   int, int, int, int, int, int, float, int, const float*, const float*, int, void*, int*, void*) {
    return PE_ERR_UNSUPPORTED;
}

#endif
