// A paged cache of 4-bit keys and values (int4_pages.cuh): rows appended with the position rotation on the way, rows read back, and the
// least and greatest key of a page, channel by channel.
#include "int4_pages.cuh"
#include <cuda_fp16.h>

// ---------------------------------------------------------------------------- queries turned, keys and values appended
//
// A query head is turned as the model's table says, in float32, and rounded once.  A key is turned with twice float32's bits and rounded once more to bfloat16, the type in which
// a 16-bit cache would hold it: what is coded next to the border of two codes then does not depend on the order of two roundings in float32.
// Keys, values and queries have blocks of their own; a thread takes eight channels.  A word of the keys' codes is one token's, so keys need their group's four threads only.  A word of the
// values' codes holds four positions: a block takes the values of sixteen tokens of a head as they stand behind one another, and the first of a word's tokens gathers the others from shared
// memory.  A word of which it has all positions is stored; of another two atomic operations change the bits of those that it has, so whoever has the rest (another block, or tokens behind a gap
// of the same one) changes them at the same time.  (Reading and writing the word where nobody else has a part of it: 6.3 us for 64 single tokens appended and read back, so 5.6.)
// Bound by the latency of a thread's chain of loads (position, angles) with as many threads as an SM holds: 7,541 tokens of 28 + 4 heads x 128 are 73 MB read and 59 MB written in 32.5 us
// (36.9 us with 1,024 threads an SM, two query heads a thread; 42.6 us with a block's keys and values in its two halves, which waited for one another; 45 us with the queries' blocks in
// between).  A call for one token takes 3.6 us, which is a launch and one chain of loads.
template <int D>
__device__ __forceinline__ void q4_load8(const bf16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

template <int D>
__device__ __forceinline__ void store_queries(const bf16* qkv, int row_width, int n_q, const float* cos_t, const float* sin_t, int angles, const int* tok_pos, bf16* q_out, long long item) {
    constexpr int half = D / 2, parts = half / 8;
    const int j = (int)(item % parts) * 8, h = (int)(item / parts % n_q), t = (int)(item / parts / n_q);
    const bf16* src = qkv + (size_t)t * row_width + h * D + j;
    bf16* dst = q_out + ((size_t)t * n_q + h) * D + j;
    uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + half);
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
    *reinterpret_cast<uint4*>(dst) = lo;
    *reinterpret_cast<uint4*>(dst + half) = hi;
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
    const float up = q4_up(__bfloat162float(step)), s = __bfloat162float(step) * up, m = __bfloat162float(mid) * up, by = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) level[i] = q4_quantise(x[i] * up, s, m, by);
}

// a c + b s rounded to bfloat16 by way of a float32 that is as if from twice as many bits: products with their errors, and the error of their sum.  Two products, one with its error, are off by
// two units of float32 at most, which matters next to the middle of two bfloat16 numbers only: a thread in a thousand takes the long way.
__device__ __forceinline__ float q4_turned(float a, float c, float b, float s) {
    const float l = __fmul_rn(b, s), el = __fmaf_rn(b, s, -l);
    float r = __fadd_rn(__fmaf_rn(a, c, l), el);
    if (((__float_as_uint(r) - 0x7ffcu) & 0xffffu) <= 8u) {
        const float h = __fmul_rn(a, c), eh = __fmaf_rn(a, c, -h), d = __fadd_rn(h, l), v = __fsub_rn(d, h);
        const float e = __fadd_rn(__fsub_rn(h, __fsub_rn(d, v)), __fsub_rn(l, v));
        r = __fadd_rn(d, __fadd_rn(e, __fadd_rn(eh, el)));
    }
    return __bfloat162float(__float2bfloat16_rn(r));
}

#define SI_THREADS 256
#define SI_TOKENS 16

template <int D>
__global__ void __launch_bounds__(SI_THREADS, 8) store_int4_kernel(const bf16* qkv, int T, int n_q, int n_kv, const float* cos_t, const float* sin_t, int angles,
                                                                const int* tok_pos, const int* tok_row, unsigned char* pool, long long n_pages,
                                                                const int* block_table, int table_stride, int n_rows, bf16* q_out, int k_blocks, int v_blocks) {
    using B = Int4Block<D>;
    __shared__ __align__(16) unsigned char fields[SI_TOKENS][D];       // the values' codes: sign << 3 | magnitude
    __shared__ int at_pos[SI_TOKENS], at_row[SI_TOKENS], at_page[SI_TOKENS];                // page -1: not stored
    __shared__ int leaders[SI_TOKENS], n_leaders, parts[SI_TOKENS];     // first tokens of words; the tokens of a leader's four positions (2 f + e), a byte each, 255: not here
    __shared__ unsigned owns[SI_TOKENS];                                // the bits of those
    pdl_launch_dependents();
    pdl_wait();
    const int row_width = (n_q + 2 * n_kv) * D;
    constexpr int lanes = D / 8, half = D / 2;
    const int w = threadIdx.x % lanes, b = w >> 2, t = w & 3, ch = w * 8;
    if ((int)blockIdx.x >= k_blocks + v_blocks) {
        const long long item = (long long)(blockIdx.x - k_blocks - v_blocks) * SI_THREADS + threadIdx.x;
        if (item < (long long)T * n_q * (D / 16)) store_queries<D>(qkv, row_width, n_q, cos_t, sin_t, angles, tok_pos, q_out, item);
        return;
    }
    if ((int)blockIdx.x < k_blocks) {
        // ---- keys: eight channels a thread, no thread but its group's needed
        const int i = (int)(blockIdx.x / n_kv) * (SI_THREADS / lanes) + threadIdx.x / lanes, kvh = blockIdx.x % n_kv, j = ch % half;
        const bool mine = i < T;
        int pos = -1, row = -1, page = -1;
        float x[8] = {};
        if (mine) {
            pos = tok_pos[i]; row = tok_row[i];
            const bf16* src = qkv + (size_t)i * row_width + (size_t)(n_q + kvh) * D;
            q4_load8<D>(src + ch, x);
            if (pos >= 0 && row >= 0 && row < n_rows && pos / PE_PAGE < table_stride) page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
            if (cos_t) {
                float y[8];
                q4_load8<D>(src + (ch < half ? ch + half : ch - half), y);
                const size_t a = (size_t)min(max(pos, 0), angles - 1) * half + j;
                const float4* cp = reinterpret_cast<const float4*>(cos_t + a);
                const float4* sp = reinterpret_cast<const float4*>(sin_t + a);
                const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
                const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = q4_turned(x[e], c[e], ch < half ? -y[e] : y[e], s[e]);
            }
        }
        int level[8];
        bf16 step, mid;
        q4_group(x, level, step, mid);
        if (page < 0 || page >= n_pages) return;
        unsigned word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) word |= q4_turn(q4_field(level[2 * e]) | q4_field(level[2 * e + 1]) << 16, e);
        unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
        const int p = pos & (PE_PAGE - 1);
        *reinterpret_cast<unsigned*>(block + q4_key_word<D>(p, b, t)) = word;
        bf16* meta = reinterpret_cast<bf16*>(block + q4_key_step<D>(p, b));
        if (t == 0) meta[0] = step;
        if (t == 1) meta[B::groups] = mid;
        return;
    }
    // ---- values of sixteen tokens
    const int kvh = (blockIdx.x - k_blocks) % n_kv, first = (int)((blockIdx.x - k_blocks) / n_kv) * SI_TOKENS, i = threadIdx.x / lanes;
    if (threadIdx.x < SI_TOKENS) {
        const int n = threadIdx.x, pos = first + n < T ? tok_pos[first + n] : -1, row = first + n < T ? tok_row[first + n] : -1;
        int page = -1;
        if (pos >= 0 && row >= 0 && row < n_rows && pos / PE_PAGE < table_stride) page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
        at_pos[n] = pos; at_row[n] = row; at_page[n] = page < n_pages ? page : -1;
    }
    float x[8];
    const bool mine = i < SI_TOKENS && first + i < T;                  // (of 64 channels half the threads have none: whole warps)
    if (mine) q4_load8<D>(qkv + (size_t)(first + i) * row_width + (size_t)(n_q + n_kv + kvh) * D + ch, x);
    __syncthreads();
    if (threadIdx.x < 32) {
        const int n = threadIdx.x, r = n < SI_TOKENS ? at_pos[n] & 15 : 0;
        bool leads = n < SI_TOKENS && at_page[n] >= 0;
        unsigned own = 0, from = ~0u;
        if (leads)
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int to = 8 * f + (r & 6) + e, o = n + to - r;                             // the token of position `to` of the tile
                    if (o < 0 || o >= SI_TOKENS || at_row[o] != at_row[n] || at_pos[o] != at_pos[n] + to - r || at_page[o] < 0) continue;
                    leads &= to >= r;
                    own |= q4_position_bits(f, e);
                    from &= ~(255u << (8 * (2 * f + e))) | (unsigned)o << (8 * (2 * f + e));
                }
        const unsigned set = __ballot_sync(0xffffffffu, leads);
        if (leads) { leaders[__popc(set & ((1u << n) - 1u))] = n; owns[n] = own; parts[n] = (int)from; }
        if (n == 0) n_leaders = __popc(set);
    }
    if (i < SI_TOKENS) {                                               // (a warp as one: the groups' shuffles)
        const int page = mine ? at_page[i] : -1, p = at_pos[i] & (PE_PAGE - 1);
        int level[8];
        bf16 step, mid;
        q4_group(x, level, step, mid);
        if (page >= 0) {
            unsigned f[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e >> 2] |= (unsigned)((level[e] ^ (level[e] >> 31)) | (level[e] < 0 ? 8 : 0)) << (8 * (e & 3));
            *reinterpret_cast<uint2*>(&fields[i][ch]) = make_uint2(f[0], f[1]);
            bf16* meta = reinterpret_cast<bf16*>(pool + ((size_t)page * n_kv + kvh) * B::bytes + q4_value_step<D>(p, b));
            if (t == 0) meta[0] = step;
            if (t == 1) meta[B::groups * 16] = mid;
        }
    }
    __syncthreads();
    // the words of the leaders' positions: m and g as in the block's layout
    constexpr int words = D / 2;
    for (int x = threadIdx.x; x < n_leaders * words; x += SI_THREADS) {
        const int n = leaders[x / words], rest = x % words, m = rest & (D / 16 - 1), g = rest / (D / 16), from = parts[n];
        unsigned word = 0;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int o = (from >> (8 * (2 * f + e))) & 255;
                if (o == 255) continue;
                const unsigned two = *reinterpret_cast<const unsigned short*>(&fields[o][32 * (m >> 1) + 4 * g + 2 * (m & 1)]);
                word |= q4_turn((((two & 8u) << 12) | ((two & 7u) << 4)) << (16 * e), 2 * f) | q4_turn((((two & 0x800u) << 4) | ((two & 0x700u) >> 4)) << (16 * e), 2 * f + 1);
            }
        const int p = at_pos[n] & (PE_PAGE - 1);
        unsigned* dst = reinterpret_cast<unsigned*>(pool + ((size_t)at_page[n] * n_kv + kvh) * B::bytes + q4_value_words<D>(p >> 4, m >> 2, g, (p & 7) >> 1)) + (m & 3);
        const unsigned own = owns[n];
        if (own == ~0u) *dst = word;
        else { atomicAnd(dst, ~own); atomicOr(dst, word); }
    }
}

extern "C" int pe_store_int4(const void* qkv, int T, int n_q, int n_kv, int hd, const float* cos_t, const float* sin_t, int angles, const int* tok_pos, const int* tok_row,
                             void* pool, long long n_pages, const int* block_table, int table_stride, int n_rows, void* q_out, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_q <= 0 || n_kv <= 0 || (((uintptr_t)qkv | (uintptr_t)pool | (uintptr_t)q_out) & 15)) return PE_ERR_UNSUPPORTED;
    if (cos_t && (angles <= 0 || (((uintptr_t)cos_t | (uintptr_t)sin_t) & 15))) return PE_ERR_UNSUPPORTED;
    const long long items = (long long)T * n_q * (hd / 16), q_blocks = (items + SI_THREADS - 1) / SI_THREADS;
    const long long per_k = SI_THREADS / (hd / 8), k_blocks = (T + per_k - 1) / per_k * n_kv, v_blocks = (long long)((T + SI_TOKENS - 1) / SI_TOKENS) * n_kv;
    const long long blocks = k_blocks + v_blocks + q_blocks, threads = SI_THREADS;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? store_int4_kernel<64> : store_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 0, (cudaStream_t)stream, (const bf16*)qkv, T, n_q, n_kv, cos_t, sin_t, angles, tok_pos,
                     tok_row, (unsigned char*)pool, n_pages, block_table, table_stride, n_rows, (bf16*)q_out, (int)k_blocks, (int)v_blocks));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- rows read back
// A thread reads four channels of a key and of a value.  Rows whose page is not there are zeros.  7,541 tokens of 4 heads of 128, 5 MB read and 31 MB written, take 10.2 us: the codes'
// conversions to float32 and a thread's chain of table, code and step.

template <int D>
__global__ void __launch_bounds__(256) load_int4_kernel(const unsigned char* pool, long long n_pages, int n_kv, const int* tok_pos, const int* tok_row, int T,
                                                        const int* block_table, int table_stride, int n_rows, float* keys, float* values) {
    using B = Int4Block<D>;
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int part = (int)(item % (D / 4)), kvh = (int)(item / (D / 4) % n_kv), b = part >> 3, g = part & 7;
    const long long tok = item / (D / 4) / n_kv;
    if (tok >= T) return;
    const int pos = tok_pos[tok], row = tok_row[tok];
    int page = -1;
    if (pos >= 0 && row >= 0 && row < n_rows && pos / PE_PAGE < table_stride) page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
    if (page >= 0 && page < n_pages) {
        const unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
        const int p = pos % PE_PAGE, r = p & 15, f = r >> 3, e = r & 1, i = (g & 1) * 2;
        const unsigned word = *reinterpret_cast<const unsigned*>(block + q4_key_word<D>(p, b, g >> 1));
        const uint2 two = *reinterpret_cast<const uint2*>(block + q4_value_words<D>(p >> 4, b >> 1, g, (r & 7) >> 1) + (b & 1) * 8);
        const bf16* km = reinterpret_cast<const bf16*>(block + q4_key_step<D>(p, b));
        const bf16* vm = reinterpret_cast<const bf16*>(block + q4_value_step<D>(p, b));
        const float ks = to_f(km[0]), kc = to_f(km[B::groups]), vs = to_f(vm[0]), vc = to_f(vm[B::groups * 16]);
        k = make_float4(fmaf(ks, q4_level(word, i, 0), kc), fmaf(ks, q4_level(word, i, 1), kc), fmaf(ks, q4_level(word, i + 1, 0), kc), fmaf(ks, q4_level(word, i + 1, 1), kc));
        v = make_float4(fmaf(vs, q4_level(two.x, 2 * f, e), vc), fmaf(vs, q4_level(two.x, 2 * f + 1, e), vc), fmaf(vs, q4_level(two.y, 2 * f, e), vc),
                        fmaf(vs, q4_level(two.y, 2 * f + 1, e), vc));
    }
    const size_t to = ((size_t)tok * n_kv + kvh) * D + part * 4;
    *reinterpret_cast<float4*>(keys + to) = k;
    *reinterpret_cast<float4*>(values + to) = v;
}

extern "C" int pe_load_int4(const void* pool, long long n_pages, int n_kv, int hd, const int* tok_pos, const int* tok_row, int T, const int* block_table, int table_stride,
                            int n_rows, float* keys, float* values, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || (((uintptr_t)pool | (uintptr_t)keys | (uintptr_t)values) & 15)) return PE_ERR_UNSUPPORTED;
    const long long blocks = ((long long)T * n_kv * (hd / 4) + 255) / 256;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? load_int4_kernel<64> : load_int4_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, (const unsigned char*)pool, n_pages, n_kv, tok_pos, tok_row, T, block_table,
                     table_stride, n_rows, keys, values));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- the bounds of a page's keys
// A block looks at sixteen tokens of a key head.  Of the page of each that is the last of its page: the least and the greatest key, channel by channel, in float32, rounded to bfloat16
// (which keeps their order).  A step of 64 tokens, a few of which end a page, takes 2.0 us, prompts of 7,541 tokens (116 pages of 4 heads of 128, 2.6 MB) 6.9: a launch, and one chain of
// table, codes and a join of eight warps, in one of each four of 1,888 blocks (the others find no page that ends).

template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(const unsigned char* pool, long long n_pages, int n_kv, const int* tok_pos, const int* tok_row, int T,
                                                          const int* block_table, int table_stride, int n_rows, bf16* bounds) {
    using B = Int4Block<D>;
    __shared__ float ends[2][8][D];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.x % n_kv, first = (int)(blockIdx.x / n_kv) * 16;
    int page = -1;
    if (lane < 16 && first + lane < T) {                       // (every warp for itself)
        const int pos = tok_pos[first + lane], row = tok_row[first + lane];
        if (pos >= 0 && pos % PE_PAGE == PE_PAGE - 1 && row >= 0 && row < n_rows && pos / PE_PAGE < table_stride) page = block_table[(size_t)row * table_stride + pos / PE_PAGE];
        if (page >= n_pages) page = -1;
    }
    constexpr int lanes = D / 8, rows = 256 / lanes;           // threads a key, keys at a time
    const int w = threadIdx.x % lanes, b = w >> 2, t = w & 3;
    for (unsigned left = __ballot_sync(0xffffffffu, page >= 0); left; left &= left - 1) {
        const int its = __shfl_sync(0xffffffffu, page, __ffs(left) - 1);
        const unsigned char* block = pool + ((size_t)its * n_kv + kvh) * B::bytes;
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
#pragma unroll
        for (int k = 0; k < PE_PAGE / rows; ++k) {
            const int p = k * rows + threadIdx.x / lanes;
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
        if (lane < lanes)
#pragma unroll
            for (int e = 0; e < 8; ++e) { ends[0][warp][w * 8 + e] = lo[e]; ends[1][warp][w * 8 + e] = hi[e]; }
        __syncthreads();
        if (threadIdx.x < 2 * D) {
            const int side = threadIdx.x / D, d = threadIdx.x % D;
            float x = ends[side][0][d];
#pragma unroll
            for (int k = 1; k < 8; ++k) x = side ? q4_max(x, ends[1][k][d]) : q4_min(x, ends[0][k][d]);
            bounds[(((size_t)its * n_kv + kvh) * 2 + side) * D + d] = __float2bfloat16_rn(x);
        }
        __syncthreads();
    }
}

extern "C" int pe_page_bounds(const void* pool, long long n_pages, int n_kv, int hd, const int* tok_pos, const int* tok_row, int T, const int* block_table,
                              int table_stride, int n_rows, void* bounds, void* stream) {
    if (T <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || (((uintptr_t)pool | (uintptr_t)bounds) & 15)) return PE_ERR_UNSUPPORTED;
    const long long blocks = (long long)((T + 15) / 16) * n_kv;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? page_bounds_kernel<64> : page_bounds_kernel<128>;
    PE_TRY(pe_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, (const unsigned char*)pool, n_pages, n_kv, tok_pos, tok_row, T, block_table,
                     table_stride, n_rows, (bf16*)bounds));
    PE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------- pages in 16 bits, for prompts
// What the runs of a prompt read of a 4-bit cache, as operands of tcgen05.mma: keys and values as float16 times powers of two of their page and head (`factors`: what takes a key back, and the
// exponent f of values 2^(14 - f) higher), so that a number keeps 11 bits whatever its size.  Positions behind a row's last run are zeros.  A value with a group that is no number is zeros, and
// its key is none: a query that sees it has no result then, and one that does not keeps its own (a weight of zero
// would not keep the value out of its sum).  Expanded once a page and head, for all heads and runs that read it.
// Bound by its writes: 7,541 tokens of 4 heads of 128 (and the 4,071 in front of a run of theirs) 7.5 MB read and 24 MB written, 10 to 11 us.
// A block counts the pages of all rows from the runs, then takes every gridDim.x-th of them.
// A page's numbers lie at its own place of a scratch as large as the pool, or, where rows times `row_pages` are fewer, at place row * row_pages + j of one of so many, which `places` says
// instead of the page table: a prompt on a large cache asks for no more than its rows can see.

#define XI_MAX_ROWS 18000                                     // twelve bytes each of shared memory
#define XI_THREADS 256

template <int D>
__global__ void __launch_bounds__(XI_THREADS) expand_int4_kernel(const unsigned char* pool, int n_pages, int n_kv, const int4* tiles, int n_tiles, const int* block_table, int table_stride,
                                                                 int n_rows, int window, int row_pages, int* places, __half* keys, __half* values, float2* factors) {
    using B = Int4Block<D>;
    extern __shared__ int xi_rows[];                           // a row's first page, the position behind its last run, the pages of the rows before it
    int* const low = xi_rows;
    int* const behind = low + n_rows;
    int* const before = behind + n_rows;
    __shared__ float2 largest[XI_THREADS / 32];
    __shared__ int further[XI_THREADS / 32];
    __shared__ bool none[PE_PAGE];                             // positions whose value has a group that is no number
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = threadIdx.x; r < n_rows; r += XI_THREADS) { low[r] = 0x7fffffff; behind[r] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < n_tiles; i += XI_THREADS) {
        const int4 run = tiles[i];                             // row, first token, tokens, position
        if (run.x < 0 || run.x >= n_rows || run.z <= 0 || run.w < 0) continue;
        atomicMin(&low[run.x], (window > 0 ? max(0, run.w - window + 1) : 0) / PE_PAGE);
        atomicMax(&behind[run.x], min(run.w + run.z, row_pages * PE_PAGE));
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
        const int j = low[row] + x - before[row], page = block_table[(size_t)row * table_stride + j];
        const bool held = page >= 0 && page < n_pages;
        const int place = places ? row * row_pages + j : page;
        if (places && kvh == 0 && threadIdx.x == 0) places[place] = held ? place : -1;
        if (!held) continue;                                   // (the same for the whole block)
        int there = min(PE_PAGE, behind[row] - j * PE_PAGE);
        if (there < PE_PAGE && !places) {
            // another row that has the page may see further into it: its block writes the same
            for (int r = threadIdx.x; r < n_rows; r += XI_THREADS)
                if (low[r] <= j && behind[r] > j * PE_PAGE + there && block_table[(size_t)r * table_stride + j] == page) there = min(PE_PAGE, behind[r] - j * PE_PAGE);
            there = -__reduce_min_sync(0xffffffffu, -there);
            __syncthreads();                                   // (the last page's have been read)
            if (lane == 0) further[warp] = there;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < XI_THREADS / 32; ++w) there = max(there, further[w]);
        }
        const size_t at = (size_t)place * n_kv + kvh;
        const unsigned char* block = pool + ((size_t)page * n_kv + kvh) * B::bytes;
        // the largest key and value that the page's steps and middles allow
        float most = 0.f, most_v = 0.f;
        for (int i = threadIdx.x; i < there * B::groups; i += XI_THREADS) {
            const int q = i / B::groups, g = i % B::groups;
            const bf16* meta = reinterpret_cast<const bf16*>(block + q4_key_step<D>(q, g));
            const bf16* vmeta = reinterpret_cast<const bf16*>(block + q4_value_step<D>(q, g));
            most = fmaxf(most, fmaf(7.5f, fabsf(to_f(meta[0])), fabsf(to_f(meta[B::groups]))));
            most_v = fmaxf(most_v, fmaf(7.5f, fabsf(to_f(vmeta[0])), fabsf(to_f(vmeta[B::groups * 16]))));
        }
        most = warp_max(most);
        most_v = warp_max(most_v);
        __syncthreads();                                       // (the last page's maxima and marks have been read)
        if (threadIdx.x < PE_PAGE) {
            bool any = false;
#pragma unroll
            for (int b = 0; b < B::groups; ++b) { const float m = to_f(*reinterpret_cast<const bf16*>(block + q4_value_step<D>(threadIdx.x, b))); any |= m != m; }
            none[threadIdx.x] = any && threadIdx.x < there;
        }
        if (lane == 0) largest[warp] = make_float2(most, most_v);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < XI_THREADS / 32; ++w) { most = fmaxf(most, largest[w].x); most_v = fmaxf(most_v, largest[w].y); }
        int exponent = 0, f = -30;                             // (a page of zero values asks for no more of the weights' range than one of the smallest)
        if (most > 0.f) frexpf(fminf(most, 3.0e38f), &exponent);                          // most <= 2^exponent
        if (most_v > 0.f) frexpf(fminf(most_v, 3.0e38f), &f);
        f = min(max(f, -30), 115);                             // (2^-f and 2^-f times the weights' power are normal numbers)
        const float up = ldexpf(1.f, 14 - max(exponent, -30)), up_v = ldexpf(1.f, 14 - f);
        if (threadIdx.x == 0) factors[at] = make_float2(1.f / up, (float)f);
        __half* ko = keys + at * PE_PAGE * D;
        __half* vo = values + at * PE_PAGE * D;
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
                if (none[p]) v = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
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
                        if (p < there && !none[p]) {
                            const bf16* meta = reinterpret_cast<const bf16*>(block + q4_value_step<D>(p, 2 * h + b));
                            const float s = to_f(meta[0]) * up_v, m = to_f(meta[B::groups * 16]) * up_v;
                            __half2 two[2];
#pragma unroll
                            for (int w = 0; w < 2; ++w)
                                two[w] = __floats2half2_rn(fmaf(s, q4_level(words[2 * b + w], 2 * f, e), m), fmaf(s, q4_level(words[2 * b + w], 2 * f + 1, e), m));
                            v = *reinterpret_cast<uint2*>(two);
                        }
                        *reinterpret_cast<uint2*>(vo + p * D + 32 * (2 * h + b) + 4 * g) = v;
                    }
                }
        }
    }
}

extern "C" int pe_expand_int4(const void* pool, long long n_pages, int n_kv, int hd, const int* tiles, int n_tiles, const int* block_table, int table_stride, int n_rows, int window,
                              int row_pages, int* places, void* keys, void* values, void* factors, void* stream) {
    if (n_tiles <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_rows < 1 || n_rows > XI_MAX_ROWS || n_pages * n_kv > 0x7fffffffll || row_pages < 1 || row_pages > table_stride ||
        (long long)n_rows * row_pages > 0x7fffffffll)
        return PE_ERR_UNSUPPORTED;
    if (((uintptr_t)pool | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)tiles) & 15 || ((uintptr_t)factors & 7)) return PE_ERR_UNSUPPORTED;
    auto kernel = hd == 64 ? expand_int4_kernel<64> : expand_int4_kernel<128>;
    const size_t smem = (size_t)(3 * n_rows + 1) * 4;
    static bool allowed[2][64] = {};
    { const int e = pe_allow_smem((const void*)kernel, (3 * XI_MAX_ROWS + 1) * 4, allowed[hd == 128]); if (e) return e; }
    PE_TRY(pe_launch(kernel, dim3(pe_sm_count() * 6), dim3(XI_THREADS), smem, (cudaStream_t)stream, (const unsigned char*)pool, (int)n_pages, n_kv, (const int4*)tiles, n_tiles,
                     block_table, table_stride, n_rows, window, row_pages, places, (__half*)keys, (__half*)values, (float2*)factors));
    PE_LAUNCH_CHECK();
    return 0;
}
