// What the two kernels of attention over shared pages (attention_shared.cu, then attention_decode.cu) agree on: which positions a row reads with
// its group, how the group's work is cut, and where the partial results lie.
//
// The work is a line of steps (two pages, 128 keys, of one key head against one tile of up to 128 rows), group after group, in each the key heads, in
// each the tiles.  CTA c of C takes the steps [c N / C, (c + 1) N / C): every CTA has the same number, whatever the groups' sizes, and a tile's keys
// may lie with several CTAs.  Each leaves sums, reference points and weights of its tile's rows.
#pragma once
#include "common.cuh"

#define AS_QTILE 128
#define AS_MIN_STEPS 2                              // steps a CTA has at least

struct AsScratch {
    long long* before;                              // [T + 1]: steps in front of the group that starts with token t; [T]: all of them, N
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
__device__ __forceinline__ int as_ctas(long long steps, int grid) {
    const long long c = (steps + AS_MIN_STEPS - 1) / AS_MIN_STEPS;
    return c < grid ? (int)c : grid;
}
// the CTA that has step s
__device__ __forceinline__ int as_cta_of(long long s, long long steps, int ctas) { return (int)(((s + 1) * ctas - 1) / steps); }
// Where CTA c leaves row i (token of the group x heads a key head) of key head kvh: rows of different pairs of CTA and tile do not meet, since
// from one pair to the next the CTA or the tile moves on, and with it 128 rows or those of the tile.
__device__ __forceinline__ size_t as_row(int c, const int4& g, int nh, int nkv, int kvh, int i) {
    return (size_t)c * AS_QTILE + (size_t)g.x * nh + (size_t)kvh * g.y * (nh / nkv) + i;
}
