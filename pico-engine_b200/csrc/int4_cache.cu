// A paged cache of 4-bit keys and values (int4_pages.cuh): rows appended with the position rotation on the way, rows read back, and the
// least and greatest key of a page, channel by channel.
#include "int4_pages.cuh"
#include <cuda_fp16.h>

// ---------------------------------------------------------------------------- queries turned, keys and values appended
//
// A query head is turned as the model's table says, in float32, and rounded once.  A key is turned in float64 and rounded once more to bfloat16, the type in which
// a 16-bit cache would hold it: what is coded next to the border of two codes then does not depend on the order of two roundings in float32.
// A word of the values' codes holds four positions, so one warp writes all tokens of a call that fall into the same 16 positions of a sequence: the first of them is its
// leader, the others have nothing to do.  Positions of the tile that are not in the call keep their bits.

template <int D>
__device__ __forceinline__ void q4_load8(const bf16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

template <int D>
__device__ __forceinline__ void store_queries(const bf16* qkv, int row_width, int n_q, const float* cos_t, const float* sin_t, int angles,
                                              const int* tok_pos, bf16* q_out, long long item) {
    constexpr int half = D / 2, parts = half / 8;
    const int part = (int)(item % parts), head = (int)(item / parts % n_q), t = (int)(item / parts / n_q), j = part * 8;
    const bf16* src = qkv + (size_t)t * row_width + head * D;
    bf16* dst = q_out + ((size_t)t * n_q + head) * D;
    uint4 lo = *reinterpret_cast<const uint4*>(src + j), hi = *reinterpret_cast<const uint4*>(src + j + half);
    if (cos_t) {
        const size_t at = (size_t)min(max(tok_pos[t], 0), angles - 1) * half + j;
        const float4* cp = reinterpret_cast<const float4*>(cos_t + at);
        const float4* sp = reinterpret_cast<const float4*>(sin_t + at);
        const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
        const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
        __nv_bfloat162* l2 = reinterpret_cast<__nv_bfloat162*>(&lo);
        __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 a = __bfloat1622float2(l2[e]), b = __bfloat1622float2(h2[e]);
            l2[e] = __floats2bfloat162_rn(a.x * c[2 * e] - b.x * s[2 * e], a.y * c[2 * e + 1] - b.y * s[2 * e + 1]);
            h2[e] = __floats2bfloat162_rn(a.x * s[2 * e] + b.x * c[2 * e], a.y * s[2 * e + 1] + b.y * c[2 * e + 1]);
        }
    }
    *reinterpret_cast<uint4*>(dst + j) = lo;
    *reinterpret_cast<uint4*>(dst + j + half) = hi;
}

// step and mid of the group that four neighbouring lanes hold eight numbers each of, and the levels of the lane's own
__device__ __forceinline__ void q4_group(const float (&x)[8], int (&level)[8], bf16& step, bf16& mid) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = q4_min(lo, x[i]); hi = q4_max(hi, x[i]); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = q4_min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = q4_max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    q4_scale(lo, hi, step, mid);
    const float s = __bfloat162float(step), m = __bfloat162float(mid);
#pragma unroll
    for (int i = 0; i < 8; ++i) level[i] = q4_quantise(x[i], s, m);
}

#define SI_WARPS 8

template <int D>
__global__ void __launch_bounds__(32 * SI_WARPS) store_int4_kernel(const bf16* qkv, int T, int n_q, int n_kv, const float* cos_t, const float* sin_t, int angles,
                                                                  const int* tok_pos, const int* tok_row, unsigned char* pool, long long n_pages,
                                                                  const int* block_table, int table_stride, int n_rows, bf16* q_out, int q_blocks) {
    using B = Int4Block<D>;
    __shared__ __align__(16) unsigned char fields[SI_WARPS][16][D];    // the values' codes of a warp's tile: sign << 3 | magnitude
    pdl_launch_dependents();
    pdl_wait();
    const int row_width = (n_q + 2 * n_kv) * D;
    if ((int)blockIdx.x < q_blocks) {
        const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
        if (item < (long long)T * n_q * (D / 16)) store_queries<D>(qkv, row_width, n_q, cos_t, sin_t, angles, tok_pos, q_out, item);
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long unit = (long long)(blockIdx.x - q_blocks) * SI_WARPS + warp;
    const int kvh = (int)(unit % n_kv);
    const long long tok = unit / n_kv;
    if (tok >= T) return;
    const int first = (int)tok, pos = tok_pos[first], row = tok_row[first], at = pos & 15;
    if (pos < 0 || row < 0 || row >= n_rows || pos / PE_PAGE >= table_stride) return;
    if (at && first > 0 && tok_row[first - 1] == row && tok_pos[first - 1] == pos - 1) return;      // an earlier token leads this tile
    const bool same = lane < 16 - at && first + lane < T && tok_row[first + lane] == row && tok_pos[first + lane] == pos + lane;
    const int n = __ffs(~__ballot_sync(0xffffffffu, same)) - 1;                                     // tokens of the tile
    const int page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
    if (page < 0 || page >= n_pages) return;
    unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
    const int p0 = pos % PE_PAGE;

    constexpr int lanes = D / 8, per_pass = 32 / lanes, half = D / 2;
    const int w = lane % lanes, b = w >> 2, t = w & 3, ch = w * 8, j = ch % half;
    for (int i0 = 0; i0 < n; i0 += per_pass) {
        const int i = i0 + lane / lanes;
        const bool mine = i < n;
        const bf16* src = qkv + (size_t)(first + (mine ? i : 0)) * row_width + (size_t)(n_q + kvh) * D;
        float x[8];
        q4_load8<D>(src + ch, x);
        if (cos_t) {
            float y[8];
            q4_load8<D>(src + (ch < half ? ch + half : ch - half), y);
            const size_t a = (size_t)min(pos + (mine ? i : 0), angles - 1) * half + j;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double c = cos_t[a + e], s = sin_t[a + e];
                const double r = ch < half ? (double)x[e] * c - (double)y[e] * s : (double)y[e] * s + (double)x[e] * c;
                x[e] = __bfloat162float(__float2bfloat16_rn((float)r));
            }
        }
        int level[8];
        bf16 step, mid;
        q4_group(x, level, step, mid);
        unsigned word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) word |= q4_turn(q4_field(level[2 * e]) | q4_field(level[2 * e + 1]) << 16, e);
        const int p = p0 + i;
        if (mine) {
            *reinterpret_cast<unsigned*>(block + q4_key_word<D>(p, b, t)) = word;
            if (t == 0) {
                bf16* meta = reinterpret_cast<bf16*>(block + q4_key_step<D>(p, b));
                meta[0] = step; meta[B::groups] = mid;
            }
        }
        q4_load8<D>(src + (size_t)n_kv * D + ch, x);
        q4_group(x, level, step, mid);
        if (mine) {
            unsigned f[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e >> 2] |= (unsigned)((level[e] ^ (level[e] >> 31)) | (level[e] < 0 ? 8 : 0)) << (8 * (e & 3));
            *reinterpret_cast<uint2*>(&fields[warp][at + i][ch]) = make_uint2(f[0], f[1]);
            if (t == 0) {
                bf16* meta = reinterpret_cast<bf16*>(block + q4_value_step<D>(p, b));
                meta[0] = step; meta[B::groups * 16] = mid;
            }
        }
    }
    __syncwarp();
    // the tile's words: four positions (those of the call), two channels
    const int g = lane >> 2, tt = lane & 3;
    unsigned own = 0;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * f + 2 * tt + e;
            if (r >= at && r < at + n) own |= q4_position_bits(f, e);
        }
    if (!own) return;
#pragma unroll
    for (int h = 0; h < B::halves; ++h) {
        uint4* dst = reinterpret_cast<uint4*>(block + q4_value_words<D>(p0 >> 4, h, g, tt));
        unsigned out[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            unsigned word = 0;
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const unsigned two = *reinterpret_cast<const unsigned short*>(&fields[warp][8 * f + 2 * tt + e][32 * (2 * h + (m >> 1)) + 4 * g + 2 * (m & 1)]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const unsigned code = two >> (8 * c);
                        word |= q4_turn((((code & 8u) << 12) | ((code & 7u) << 4)) << (16 * e), 2 * f + c);
                    }
                }
            out[m] = word;
        }
        if (own != ~0u) {
            const uint4 old = *dst;
            out[0] = (out[0] & own) | (old.x & ~own); out[1] = (out[1] & own) | (old.y & ~own);
            out[2] = (out[2] & own) | (old.z & ~own); out[3] = (out[3] & own) | (old.w & ~own);
        }
        *dst = make_uint4(out[0], out[1], out[2], out[3]);
    }
}

extern "C" int pe_store_int4(const void* qkv, int T, int n_q, int n_kv, int hd, const float* cos_t, const float* sin_t, int angles, const int* tok_pos, const int* tok_row,
                             void* pool, long long n_pages, const int* block_table, int table_stride, int n_rows, void* q_out, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_q <= 0 || n_kv <= 0 || (((uintptr_t)qkv | (uintptr_t)pool | (uintptr_t)q_out) & 15)) return PE_ERR_UNSUPPORTED;
    if (cos_t && (angles <= 0 || (((uintptr_t)cos_t | (uintptr_t)sin_t) & 15))) return PE_ERR_UNSUPPORTED;
    const long long items = (long long)T * n_q * (hd / 16), units = (long long)T * n_kv, threads = 32 * SI_WARPS;
    const long long q_blocks = (items + threads - 1) / threads, blocks = q_blocks + (units + SI_WARPS - 1) / SI_WARPS;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? store_int4_kernel<64> : store_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 0, (cudaStream_t)stream, (const bf16*)qkv, T, n_q, n_kv, cos_t, sin_t, angles, tok_pos,
                     tok_row, (unsigned char*)pool, n_pages, block_table, table_stride, n_rows, (bf16*)q_out, (int)q_blocks));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- rows read back
// A thread reads eight channels of a key and of a value.  Rows whose page is not there are zeros.

template <int D>
__global__ void __launch_bounds__(256) load_int4_kernel(const unsigned char* pool, long long n_pages, int n_kv, const int* tok_pos, const int* tok_row, int T,
                                                        const int* block_table, int table_stride, int n_rows, float* keys, float* values) {
    using B = Int4Block<D>;
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int w = (int)(item % (D / 8)), kvh = (int)(item / (D / 8) % n_kv);
    const long long tok = item / (D / 8) / n_kv;
    if (tok >= T) return;
    const int pos = tok_pos[tok], row = tok_row[tok], b = w >> 2, t = w & 3;
    int page = -1;
    if (pos >= 0 && row >= 0 && row < n_rows && pos / PE_PAGE < table_stride) page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
    float k[8], v[8];
    if (page < 0 || page >= n_pages) {
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.f;
    } else {
        const unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
        const int p = pos % PE_PAGE, r = p & 15, f = r >> 3, tt = (r & 7) >> 1, e1 = r & 1;
        const unsigned word = *reinterpret_cast<const unsigned*>(block + q4_key_word<D>(p, b, t));
        const bf16* km = reinterpret_cast<const bf16*>(block + q4_key_step<D>(p, b));
        const bf16* vm = reinterpret_cast<const bf16*>(block + q4_value_step<D>(p, b));
        const float ks = to_f(km[0]), kc = to_f(km[B::groups]), vs = to_f(vm[0]), vc = to_f(vm[B::groups * 16]);
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = fmaf(ks, q4_level(word, e >> 1, e & 1), kc);
#pragma unroll
        for (int g2 = 0; g2 < 2; ++g2)
#pragma unroll
            for (int m2 = 0; m2 < 2; ++m2) {
                const int m = 2 * b + m2;
                const unsigned vw = *reinterpret_cast<const unsigned*>(block + q4_value_words<D>(p >> 4, m >> 2, 2 * t + g2, tt) + (m & 3) * 4);
                v[4 * g2 + 2 * m2] = fmaf(vs, q4_level(vw, 2 * f, e1), vc);
                v[4 * g2 + 2 * m2 + 1] = fmaf(vs, q4_level(vw, 2 * f + 1, e1), vc);
            }
    }
    const size_t to = ((size_t)tok * n_kv + kvh) * D + w * 8;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<float4*>(keys + to + e) = make_float4(k[e], k[e + 1], k[e + 2], k[e + 3]);
        *reinterpret_cast<float4*>(values + to + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
}

extern "C" int pe_load_int4(const void* pool, long long n_pages, int n_kv, int hd, const int* tok_pos, const int* tok_row, int T, const int* block_table, int table_stride,
                            int n_rows, float* keys, float* values, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || (((uintptr_t)pool | (uintptr_t)keys | (uintptr_t)values) & 15)) return PE_ERR_UNSUPPORTED;
    const long long blocks = ((long long)T * n_kv * (hd / 8) + 255) / 256;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? load_int4_kernel<64> : load_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, (const unsigned char*)pool, n_pages, n_kv, tok_pos, tok_row, T, block_table,
                     table_stride, n_rows, keys, values));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- the bounds of a page's keys
// A warp a token and head: where the token is the last of its page, the least and the greatest of the page's keys, channel by channel, in float32, rounded to bfloat16.

template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(const unsigned char* pool, long long n_pages, int n_kv, const int* tok_pos, const int* tok_row, int T,
                                                          const int* block_table, int table_stride, int n_rows, bf16* bounds) {
    using B = Int4Block<D>;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int kvh = (int)(unit % n_kv);
    const long long tok = unit / n_kv;
    if (tok >= T) return;
    const int pos = tok_pos[tok], row = tok_row[tok];
    if (pos < 0 || pos % PE_PAGE != PE_PAGE - 1 || row < 0 || row >= n_rows || pos / PE_PAGE >= table_stride) return;
    const int page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
    if (page < 0 || page >= n_pages) return;
    const unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
    constexpr int lanes = D / 8, per_pass = 32 / lanes;
    const int w = lane % lanes, b = w >> 2, t = w & 3;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
#pragma unroll 4
    for (int p = lane / lanes; p < PE_PAGE; p += per_pass) {
        const unsigned word = *reinterpret_cast<const unsigned*>(block + q4_key_word<D>(p, b, t));
        const bf16* km = reinterpret_cast<const bf16*>(block + q4_key_step<D>(p, b));
        const float s = to_f(km[0]), c = to_f(km[B::groups]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fmaf(s, q4_level(word, e >> 1, e & 1), c);
            lo[e] = q4_min(lo[e], x); hi[e] = q4_max(hi[e], x);
        }
    }
#pragma unroll
    for (int o = lanes; o < 32; o <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo[e] = q4_min(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
            hi[e] = q4_max(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
        }
    if (lane < lanes) {
        bf16* to = bounds + ((size_t)page * n_kv + kvh) * 2 * D + w * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) { to[e] = __float2bfloat16_rn(lo[e]); to[D + e] = __float2bfloat16_rn(hi[e]); }
    }
}

extern "C" int pe_page_bounds(const void* pool, long long n_pages, int n_kv, int hd, const int* tok_pos, const int* tok_row, int T, const int* block_table,
                              int table_stride, int n_rows, void* bounds, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || (((uintptr_t)pool | (uintptr_t)bounds) & 15)) return PE_ERR_UNSUPPORTED;
    const long long blocks = ((long long)T * n_kv + 7) / 8;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? page_bounds_kernel<64> : page_bounds_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, (const unsigned char*)pool, n_pages, n_kv, tok_pos, tok_row, T, block_table,
                     table_stride, n_rows, (bf16*)bounds));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- pages in 16 bits, for prompts
// What the runs of a prompt read of a 4-bit cache, as operands of tcgen05.mma: values as bfloat16, keys as float16 times a power of two of their page and head (`factors` takes it
// back), so that a key keeps 11 bits whatever its size: with keys of 8 bits the scores' errors are what the results are off by (0.0055 of their size; 0.0024 so).  Positions behind a
// row's last run are zeros.  Expanded once a page and head, for all heads and runs that read it: 7.4 MB to 24 MB of a layer for prompts of 7,541 tokens.
// A block counts the pages of all rows from the runs, then takes every gridDim.x-th of them.

#define XI_MAX_ROWS 1024
#define XI_THREADS 256

template <int D>
__global__ void __launch_bounds__(XI_THREADS) expand_int4_kernel(const unsigned char* pool, int n_pages, int n_kv, const int4* tiles, int n_tiles, const int* block_table, int table_stride,
                                                                 int n_rows, int window, __half* keys, bf16* values, float* factors) {
    using B = Int4Block<D>;
    __shared__ int low[XI_MAX_ROWS], behind[XI_MAX_ROWS], before[XI_MAX_ROWS + 1];     // a row's first page, the position behind its last run, the pages of the rows before it
    __shared__ float largest[XI_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = threadIdx.x; r < n_rows; r += XI_THREADS) { low[r] = 0x7fffffff; behind[r] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < n_tiles; i += XI_THREADS) {
        const int4 run = tiles[i];                             // row, first token, tokens, position
        if (run.x < 0 || run.x >= n_rows || run.z <= 0 || run.w < 0) continue;
        atomicMin(&low[run.x], (window > 0 ? max(0, run.w - window + 1) : 0) / PE_PAGE);
        atomicMax(&behind[run.x], min(run.w + run.z, table_stride * PE_PAGE));
    }
    __syncthreads();
    if (warp == 0) {
        int sum = 0;
        for (int base = 0; base < n_rows; base += 32) {
            const int r = base + lane, n = r < n_rows ? max(0, (behind[r] + PE_PAGE - 1) / PE_PAGE - low[r]) : 0;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
            if (r < n_rows) before[r] = sum + upto - n;
            sum += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) before[n_rows] = sum;
    }
    __syncthreads();
    const long long items = (long long)before[n_rows] * n_kv;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int kvh = (int)(item % n_kv), x = (int)(item / n_kv);
        int row = 0, top = n_rows;
        while (top - row > 1) { const int mid = (row + top) >> 1; if (before[mid] <= x) row = mid; else top = mid; }
        const int j = low[row] + x - before[row], there = min(PE_PAGE, behind[row] - j * PE_PAGE), page = block_table[(size_t)row * table_stride + j];
        if (page < 0 || page >= n_pages) continue;             // (the same for the whole block)
        const size_t at = (size_t)page * n_kv + kvh;
        const unsigned char* block = pool + at * B::bytes;
        // the largest key that the page's steps and middles allow
        float most = 0.f;
        for (int i = threadIdx.x; i < there * B::groups; i += XI_THREADS) {
            const bf16* meta = reinterpret_cast<const bf16*>(block + q4_key_step<D>(i / B::groups, i % B::groups));
            most = fmaxf(most, fmaf(7.5f, fabsf(to_f(meta[0])), fabsf(to_f(meta[B::groups]))));
        }
        most = warp_max(most);
        __syncthreads();                                       // (the last page's maxima have been read)
        if (lane == 0) largest[warp] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < XI_THREADS / 32; ++w) most = fmaxf(most, largest[w]);
        int exponent = 0;
        if (most > 0.f) frexpf(fminf(most, 3.0e38f), &exponent);                          // most <= 2^exponent
        const float up = ldexpf(1.f, 14 - max(exponent, -30));
        if (threadIdx.x == 0) factors[at] = 1.f / up;
        __half* ko = keys + at * PE_PAGE * D;
        bf16* vo = values + at * PE_PAGE * D;
#pragma unroll
        for (int i = threadIdx.x; i < PE_PAGE * B::key_words; i += XI_THREADS) {
            const int p = i / B::key_words, rest = i % B::key_words, t = rest / B::groups, b = rest % B::groups;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (p < there) {
                const unsigned word = *reinterpret_cast<const unsigned*>(block + i * 4);
                const bf16* meta = reinterpret_cast<const bf16*>(block + q4_key_step<D>(p, b));
                const float s = to_f(meta[0]) * up, m = to_f(meta[B::groups]) * up;
                __half2 two[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) two[e] = __floats2half2_rn(fmaf(s, q4_level(word, e, 0), m), fmaf(s, q4_level(word, e, 1), m));
                v = *reinterpret_cast<uint4*>(two);
            }
            *reinterpret_cast<uint4*>(ko + p * D + 32 * b + 8 * t) = v;
        }
#pragma unroll
        for (int i = threadIdx.x; i < 4 * B::halves * 32; i += XI_THREADS) {
            const int tile = i / (B::halves * 32), h = i / 32 % B::halves, g = (i & 31) >> 2, t = i & 3;
            const uint4 four = *reinterpret_cast<const uint4*>(block + B::values + i * 16);
            const unsigned words[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int p = 16 * tile + 8 * f + 2 * t + e;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        uint2 v = make_uint2(0u, 0u);
                        if (p < there) {
                            const bf16* meta = reinterpret_cast<const bf16*>(block + q4_value_step<D>(p, 2 * h + b));
                            const float s = to_f(meta[0]), m = to_f(meta[B::groups * 16]);
                            __nv_bfloat162 two[2];
#pragma unroll
                            for (int w = 0; w < 2; ++w)
                                two[w] = __floats2bfloat162_rn(fmaf(s, q4_level(words[2 * b + w], 2 * f, e), m), fmaf(s, q4_level(words[2 * b + w], 2 * f + 1, e), m));
                            v = *reinterpret_cast<uint2*>(two);
                        }
                        *reinterpret_cast<uint2*>(vo + p * D + 32 * (2 * h + b) + 4 * g) = v;
                    }
                }
        }
    }
}

extern "C" int pe_expand_int4(const void* pool, long long n_pages, int n_kv, int hd, const int* tiles, int n_tiles, const int* block_table, int table_stride, int n_rows, int window,
                              void* keys, void* values, float* factors, void* stream) {
    if (n_tiles <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_rows < 1 || n_rows > XI_MAX_ROWS || n_pages * n_kv > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)pool | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)tiles) & 15) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? expand_int4_kernel<64> : expand_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3(pe_sm_count() * 6), dim3(XI_THREADS), 0, (cudaStream_t)stream, (const unsigned char*)pool, (int)n_pages, n_kv, (const int4*)tiles, n_tiles,
                     block_table, table_stride, n_rows, window, (__half*)keys, (bf16*)values, factors));
    PE_LAUNCH_CHECK();
    return 0;
}
