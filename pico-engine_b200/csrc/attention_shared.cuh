// What the two kernels of attention over shared pages (attention_shared.cu, then attention_decode.cu) agree on: which positions a row reads with
// its group, how the group's work is cut, and where the partial results lie.
//
// The work is a line of steps (two pages, 128 keys, of one key head against one tile of up to 128 rows), group after group, in each the key heads, in
// each the tiles.  The N steps are dealt to C CTAs in runs that differ by one at most, whatever the groups' sizes, so a tile's keys may lie with
// several CTAs.  Each leaves sums, reference points and weights of its tile's rows.
#pragma once
#include "common.cuh"

#define AS_QTILE 128
#define AS_MIN_STEPS 2                              // steps a CTA has at least
#define AS_MAX_CTAS 160
#define AS_COUNTED 320                             // up to so many tokens both kernels count the steps themselves; with more the second takes them from the first

struct AsScratch {
    int* before;                                    // [T + 1], T > AS_COUNTED: steps in front of the group that starts with token t; [T]: all of them, N
    float* sums;                                    // a block for each pair of CTA and tile, [head size][rows of the tile]
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
// How the steps are dealt: the first `more` CTAs have each + 1, the others each.
struct AsDeal {
    int ctas, each, more;
    __device__ __forceinline__ AsDeal(int steps, int grid) {
        ctas = min((steps + AS_MIN_STEPS - 1) / AS_MIN_STEPS, grid);
        each = ctas > 0 ? steps / ctas : 0;
        more = steps - each * ctas;
    }
    __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int cta_of(int s) const { return s < more * (each + 1) ? s / (each + 1) : more + (s - more * (each + 1)) / each; }
};
// The group that starts with token t: its tiles, the pages they see, and its steps (0 where no group starts)
struct AsGroup {
    int4 g; AsPages pages; int t, before, steps;
    __device__ __forceinline__ void load(const int4* groups, const int* tok_pos, int first, int T, int table_stride, int nh, int nkv, int window, int keep_first) {
        t = first;
        g = groups[t];
        steps = 0;
        const int shared = g.x == t ? as_shared(g, t, T, table_stride) : 0;
        if (shared == 0) return;
        pages = as_pages(shared, window > 0 ? tok_pos[g.w] : 0, window, keep_first);
        steps = as_tile_steps(pages) * as_tiles(g, nh, nkv) * nkv;
    }
};
// Where CTA c leaves the rows of a tile (tokens x heads of key head kvh), in rows: blocks of different pairs of CTA and tile do not meet, since from one
// pair to the next the CTA or the tile moves on, and with it 128 rows or those of the tile.
__device__ __forceinline__ size_t as_block(int c, const int4& g, int nh, int nkv, int kvh, int tile) {
    const int R = nh / nkv;
    return (size_t)c * AS_QTILE + (size_t)g.x * nh + (size_t)kvh * g.y * R + tile * (AS_QTILE / R * R);
}
