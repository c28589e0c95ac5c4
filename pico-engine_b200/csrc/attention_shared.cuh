// What the two kernels of attention over shared pages (attention_shared.cu, then attention_decode.cu) agree on: which positions a row reads with
// its group, how the group's work is cut, and where the partial results lie.
//
// The work is cut into steps (two pages, 128 keys, of one key head against one tile of up to 128 rows).  The steps of a tile lie side by side; tiles lie
// in a line, group after group, in each the key heads, in each the tiles of rows.  Two ways to deal them to CTAs (AsDeal):
//   chunks  where there are twice as many CTAs as tiles: every tile is cut into chunks of at most `chunk` steps, a chunk a CTA.  (A run of steps that
//           went on into the next tile cost the CTA 6,000 cycles for queries, the pipeline's start and its end, as much as four steps.)
//   runs    else: the steps in their line, in runs that differ by one at most, so a CTA has several tiles and a tile may lie with several CTAs.
// Each CTA leaves sums, reference points and weights of its tiles' rows.
#pragma once
#include "common.cuh"

#define AS_QTILE 128
#define AS_MIN_STEPS 2                              // steps of a chunk or run at least, where there are as many
#define AS_MAX_CTAS 160
#define AS_COUNTED 320                              // up to so many tokens both kernels count the steps themselves; with more the second takes them from the first

struct AsScratch {
    int* before;                                    // [T + 2], T > AS_COUNTED: units (chunks or steps) in front of the group that starts with token t;
                                                    //         [T], [T + 1]: steps and tiles of all groups
    float* sums;                                    // [rows][head size]
    float4* ends;                                   // [rows]: reference point (a maximum, in powers of two) and weight of either warpgroup's steps; sums
                                                    //         are relative to the larger of the two
};

// The positions that token t reads with its group; 0: it reads all by itself (alone in its group, or not a group of this step)
__device__ __forceinline__ int as_shared(const int4& g, int t, int T, int table_stride) {
    if (g.y < 2 || g.x < 0 || t < g.x || g.y > T - g.x || t >= g.x + g.y || g.w < g.x || g.w >= g.x + g.y) return 0;
    return max(0, min(g.z / PE_PAGE, table_stride)) * PE_PAGE;
}
// The pages of the shared positions that any row of the group can see, in the order they are read: page j is j < kept ? j : page_lo + j - kept.
// `pos`: the group's least position.
struct AsPages {
    int kept, page_lo, n;
    __device__ __forceinline__ int at(int j) const { return j < kept ? j : page_lo + j - kept; }
};
__device__ __forceinline__ int as_tile_steps(const AsPages& pages) { return (pages.n + 1) / 2; }
__device__ __forceinline__ int as_tiles(const int4& g, int nh, int nkv) { const int per_tile = AS_QTILE / (nh / nkv); return (g.y + per_tile - 1) / per_tile; }
__device__ __forceinline__ AsPages as_pages(int shared, int pos, int window, int keep_first) {
    AsPages r = {0, 0, shared / PE_PAGE};
    if (window > 0) {
        const int end = r.n, keep_pages = min((keep_first + PE_PAGE - 1) / PE_PAGE, end);
        r.page_lo = min(max(pos - window + 1, 0) / PE_PAGE, end);
        if (r.page_lo <= keep_pages) r.page_lo = 0; else r.kept = keep_pages;
        r.n = r.kept + end - r.page_lo;
    }
    return r;
}
// How `steps` steps of `tiles` tiles are dealt to `grid` CTAs.
struct AsDeal {
    int chunk;                                      // most steps of a chunk; 0: runs
    int ctas, each, more;                           // runs: the first `more` CTAs have each + 1, the others each
    __device__ __forceinline__ AsDeal(int steps, int tiles, int grid) {
        chunk = 2 * tiles <= grid && steps > 0 ? max((steps + grid - tiles - 1) / (grid - tiles), AS_MIN_STEPS) : 0;
        ctas = min((steps + AS_MIN_STEPS - 1) / AS_MIN_STEPS, grid);
        each = ctas > 0 ? steps / ctas : 0;
        more = steps - each * ctas;
    }
    // units (chunks or steps) of a tile of n steps
    __device__ __forceinline__ int units(int n) const { return chunk ? (n + chunk - 1) / chunk : n; }
    __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int cta_of(int s) const { return s < more * (each + 1) ? s / (each + 1) : more + (s - more * (each + 1)) / each; }
    // the CTAs [x, y) that have the tile of n steps with `before` units in front of it
    __device__ __forceinline__ int2 ctas_of(int before, int n) const { return chunk ? make_int2(before, before + units(n)) : make_int2(cta_of(before), cta_of(before + n - 1) + 1); }
};
// The group that starts with token t: its tiles, the pages they see, and its steps (0 where no group starts)
struct AsGroup {
    int4 g; AsPages pages; int t, row, before, tiles;       // row: the batch row whose page table names the shared pages; before: units; tiles: of all key heads
    __device__ __forceinline__ void load(const int4* groups, const int* tok_pos, const int* tok_row, int first, int T, int table_stride, int nh, int nkv, int window, int keep_first) {
        t = first;
        g = groups[t];
        row = tok_row[t];                                    // (without a window every row of the group names all shared pages)
        tiles = 0;
        const int shared = g.x == t ? as_shared(g, t, T, table_stride) : 0;
        if (shared == 0) return;
        if (window > 0) row = tok_row[g.w];
        pages = as_pages(shared, window > 0 ? tok_pos[g.w] : 0, window, keep_first);
        tiles = pages.n > 0 ? as_tiles(g, nh, nkv) * nkv : 0;
    }
    __device__ __forceinline__ int steps() const { return tiles > 0 ? as_tile_steps(pages) * tiles : 0; }
    __device__ __forceinline__ int units(const AsDeal& d) const { return tiles > 0 ? d.units(as_tile_steps(pages)) * tiles : 0; }
};
// Where CTA c leaves the rows of a tile (tokens x heads of key head kvh), in rows: blocks of different pairs of CTA and tile do not meet, since from one
// pair to the next the CTA or the tile moves on, and with it 128 rows or those of the tile.
__device__ __forceinline__ size_t as_block(int c, const int4& g, int nh, int nkv, int kvh, int tile) {
    const int R = nh / nkv;
    return (size_t)c * AS_QTILE + (size_t)g.x * nh + (size_t)kvh * g.y * R + tile * (AS_QTILE / R * R);
}
