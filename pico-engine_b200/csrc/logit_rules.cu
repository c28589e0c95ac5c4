// Rules on what a sequence may go on with, applied to float32 logits before the next token is chosen.
//
// For row b of the batch (sequence slot s = slots[b]) and token v, h = history[s][v] (16 bits: the sign bit says that v stands in the
// prompt, the other 15 how often it has been generated):
//     z = logits[b][v]
//     h != 0:   z = z > 0 ? z / repetition : z * repetition
//     count c:  z -= presence + c * frequency                     (c > 0)
//     z += the row's biases of v (a list of ids and values; those of an id that stands there twice are added up first, in the list's order)
//     v is not in the row's mask: z = -inf                        (whatever z was)
//
// A block takes some thousand tokens of a row, eight a thread, all of a thread's loads under way at once; what the result does not
// hang on is not read: where the mask leaves nothing of a warp's 128 tokens, neither logits nor history (run by run, those of 2 in 100 tokens
// spread at random came to so many single sectors that all of them are read faster), and where the row is changed in place, logits of tokens that have not
// been seen, which are not written either.  Biases are few and lie anywhere: a second kernel adds them to the result, an entry a thread
// (picked out of the list and added up in shared memory by every block of the first one they cost as much as all the rest: 64 rows of 151,936 under
// all rules 33 us, 23.8 this way, its lists read while the first one works; penalties alone 19.2 us, a mask alone 13.4).
//
// What bounds it: not DRAM.  Penalties alone move their 98 MB at 5.1 TB/s, but results stay in L2, and the counters see 57 MB of DRAM traffic in 21.7 us (2.6 TB/s).  A block
// goes through slot, mask row, mask word and logits one behind the other and then ends; 64 rows of 151,936 are 4,800 blocks on 1,184 places, and nothing of a block's
// successor is under way while it waits.
#include "common.cuh"
#include <type_traits>

#define LR_THREADS 256
#define LR_CHUNK (LR_THREADS * 8)                   // tokens of a block: eight a thread (with sixteen, and so fewer blocks an SM, 64 rows with penalties took 23 us instead of 19)
#define LR_LIST 512                                 // entries of a list of biases that a block takes in one turn

struct LrArgs {
    const float* logits; float* out; int rows, vocab;
    const int* slots; const short* history; int n_slots;
    const float* penalties;
    const int2* bias_range; const int* bias_ids; const float* bias_values; int n_bias;
    const unsigned* masks; int n_masks, mask_words; const int* mask_rows; int by_slot;      // by_slot: mask_rows has an entry a slot, not a row
};
// the mask of the row whose entry is number `at`, or -1
__device__ __forceinline__ int lr_mask(const LrArgs& p, int at, int entries) { return p.masks && at >= 0 && at < entries ? p.mask_rows[at] : -1; }

// Four tokens at a time: those that lie on 16 bytes of the row (a vocabulary need not be a multiple of four), and what is left at the row's ends one by one.
// ALIGNED: logits and out start on 16 bytes; else every load and store takes one number.  BY_SLOT: p.by_slot (a choice at run time made the mask of a row
// wait for its slot either way: 200 rows of 50,257 under masks 17.5 us instead of 16.2).
template <bool ALIGNED, bool IN_PLACE, bool BY_SLOT>
__global__ void __launch_bounds__(LR_THREADS, 8) adjust_logits_kernel(const LrArgs p) {
    constexpr int TURNS = LR_CHUNK / 4 / LR_THREADS;                // runs of a thread
    pdl_wait();
    pdl_launch_dependents();                                        // (behind the wait: the second kernel reads its lists before this one has ended)
    const int b = blockIdx.y, V = p.vocab;
    const size_t at0 = (size_t)b * V;
    const float* row = p.logits + at0;
    float* out = p.out + at0;
    const int slot = BY_SLOT || p.history ? p.slots[b] : -1, m = BY_SLOT ? lr_mask(p, slot, p.n_slots) : lr_mask(p, b, p.rows);
    const bool known = p.history && slot >= 0 && slot < p.n_slots;
    const short* seen = p.history + (known ? (size_t)slot * V : 0);
    const unsigned* mask = m >= 0 && m < p.n_masks ? p.masks + (size_t)m * p.mask_words : nullptr;
    float repetition = 1.f, inverse = 1.f, presence = 0.f, frequency = 0.f;
    if (known) { repetition = p.penalties[3 * b]; presence = p.penalties[3 * b + 1]; frequency = p.penalties[3 * b + 2]; inverse = 1.f / repetition; }      // (its rounding joins the product's: a step of float32 where a quotient has half of one)
    // the chunk's tokens begin .. end - 1: runs of four from `base` on, before and behind them (first and last chunk) a few single ones
    const int head = min((int)(-at0 & 3), V), base = head + blockIdx.x * LR_CHUNK, stop = min(base + LR_CHUNK, V), runs = (stop - base) >> 2;
    if (blockIdx.x > 0 && base >= V) return;                        // (the single tokens at the row's start have moved the chunks)
    const bool eight = ((size_t)(known ? seen - p.history : 0) + base) % 4 == 0 && !((uintptr_t)p.history & 7);      // the history's runs lie on 8 bytes
    auto bits_of = [&](int v) {                                     // which of the tokens v .. v + 3 are allowed
        if (!mask) return 15u;
        const int word = v >> 5;
        const unsigned lo = mask[word];
        return ((v & 31) > 28 ? __funnelshift_r(lo, word + 1 < p.mask_words ? mask[word + 1] : 0u, v & 31) : lo >> (v & 31)) & 15u;
    };
    unsigned allowed[TURNS];
    short4 h[TURNS];
    float4 z[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int r = k * LR_THREADS + threadIdx.x;
        allowed[k] = r < runs ? bits_of(base + 4 * r) : 0u;
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int v = base + 4 * (k * LR_THREADS + (int)threadIdx.x);
        h[k] = make_short4(0, 0, 0, 0);
        const bool some = __any_sync(0xffffffffu, allowed[k] != 0u) && k * LR_THREADS + (int)threadIdx.x < runs;
        if (known && some) h[k] = eight ? *reinterpret_cast<const short4*>(seen + v) : make_short4(seen[v], seen[v + 1], seen[v + 2], seen[v + 3]);
        if (!IN_PLACE && some) z[k] = ALIGNED ? *reinterpret_cast<const float4*>(row + v) : make_float4(row[v], row[v + 1], row[v + 2], row[v + 3]);
    }
    auto rule = [&](float x, short h_v) {
        const int count = h_v & 0x7fff;
        if (h_v != 0) x *= x > 0.f ? inverse : repetition;
        return count > 0 ? x - fmaf((float)count, frequency, presence) : x;
    };
    // one token by itself
    auto single = [&](int v, bool is_allowed, short h_v) {
        if (!is_allowed) out[v] = -INFINITY;
        else if (!IN_PLACE || h_v != 0) out[v] = rule(row[v], h_v);
    };
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int r = k * LR_THREADS + (int)threadIdx.x, v = base + 4 * r;
        if (r >= runs) continue;
        const short4 t = h[k];
        if constexpr (IN_PLACE) {                                   // only runs in which something changes are read and written
            if (allowed[k] == 15u && t.x == 0 && t.y == 0 && t.z == 0 && t.w == 0) continue;
            if (allowed[k]) z[k] = ALIGNED ? *reinterpret_cast<const float4*>(row + v) : make_float4(row[v], row[v + 1], row[v + 2], row[v + 3]);
        }
        float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (allowed[k] & 1u) x.x = rule(z[k].x, t.x);
        if (allowed[k] & 2u) x.y = rule(z[k].y, t.y);
        if (allowed[k] & 4u) x.z = rule(z[k].z, t.z);
        if (allowed[k] & 8u) x.w = rule(z[k].w, t.w);
        if constexpr (ALIGNED) *reinterpret_cast<float4*>(out + v) = x;
        else { out[v] = x.x; out[v + 1] = x.y; out[v + 2] = x.z; out[v + 3] = x.w; }
    }
    // what is left: up to three tokens in front of the first run and behind the last
    const int before = blockIdx.x == 0 ? head : 0, left = before + (stop - base - 4 * runs);
    if ((int)threadIdx.x < left) {
        const int v = (int)threadIdx.x < before ? (int)threadIdx.x : base + 4 * runs + (int)threadIdx.x - before;
        single(v, bits_of(v) & 1u, known ? seen[v] : (short)0);
    }
}

// out += the row's biases, where the mask allows the token: a block a row.  Biases of a token that stands in the list several times are added up first: by its
// first entry, in the list's order, so that no sum depends on which thread comes first.  How those are found goes by the length of the row's list:
//   up to LR_LIST entries   a table in shared memory tells which entry is a token's first and whether there are others; only then is the list read through
//                           (by every entry it took 11 us for 64 lists of 300)
//   more                    lr_long_list
// LONG: lists may be longer than LR_LIST (the second way takes more shared memory).
#define LR_BITS (1 << 17)

__device__ __forceinline__ bool lr_allows(const unsigned* mask, int id) { return !mask || ((mask[id >> 5] >> (id & 31)) & 1u); }

// A list of any length.  A bit a token (of LR_BITS at a time) tells which ones come twice.  The others add what they have.  Those go, LR_LIST entries a turn, into a
// table; each turn behind adds to their sums what it has of them, and a token whose sum is complete loses its bit, so that its other entries are passed over.
// 64 lists, of 151,936 tokens: 600 each 16 us, 4,096 each 55 us, 119 us where every token comes twice, half a list apart.  (Turn by turn onto the logit, which lost
// what cancels between turns, 15, 56 and 53 us; inlined, since with a call the kernel took 0.5 us longer for short lists too.)
__device__ __forceinline__ void lr_long_list(const LrArgs& p, int first, int last, const unsigned* mask, float* out, int* table, int* ids, float* values, unsigned* twice) {
    constexpr int PER = LR_LIST / LR_THREADS, PLACES = 2 * LR_LIST;
    static_assert(4 * PLACES == LR_BITS / 32, "the first of a token's two bits lies where the table comes");
    unsigned* once = reinterpret_cast<unsigned*>(table);
    int *token = table, *owner = table + PLACES, *lead = table + 2 * PLACES, *count = table + 3 * PLACES;
    constexpr int NONE = 0x7fffffff;
    for (int id0 = 0; id0 < p.vocab; id0 += LR_BITS) {
        const unsigned here = min(LR_BITS, p.vocab - id0);
        auto entry = [&](int e) {                                   // the token of entry e, or -1
            const int id = e < last ? p.bias_ids[e] : -1;
            return id >= id0 && (unsigned)(id - id0) < here ? id : -1;
        };
        auto comes_twice = [&](int id) { return ((twice[(id - id0) >> 5] >> (id & 31)) & 1u) != 0u; };
        __syncthreads();
        for (int i = threadIdx.x; i < LR_BITS / 32; i += LR_THREADS) once[i] = twice[i] = 0u;
        __syncthreads();
        bool some = false;
#pragma unroll 4
        for (int e = first + (int)threadIdx.x; e < last; e += LR_THREADS) {
            const int id = entry(e);
            if (id < 0) continue;
            const unsigned bit = 1u << (id & 31);
            if (atomicOr(&once[(id - id0) >> 5], bit) & bit) { atomicOr(&twice[(id - id0) >> 5], bit); some = true; }
        }
        some = __syncthreads_or(some);
        if (id0 == 0) pdl_wait();
#pragma unroll 4
        for (int e = first + (int)threadIdx.x; e < last; e += LR_THREADS) {
            const int id = entry(e);
            if (id >= 0 && !comes_twice(id) && lr_allows(mask, id)) out[id] += p.bias_values[e];
        }
        if (!some) continue;
        for (int turn = first; turn < last; turn += LR_LIST) {
            // ---- the turn's tokens that are not done, and what the turn itself has of them: values[i] becomes the sum of the token whose first entry is i
            int id[PER], place[PER];
            bool mine = false, is_first[PER];
            __syncthreads();                                        // (the turn before has taken its tokens' bits)
            for (int i = threadIdx.x; i < PLACES; i += LR_THREADS) { token[i] = -1; owner[i] = lead[i] = NONE; count[i] = 0; }
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int i = k * LR_THREADS + threadIdx.x;
                id[k] = i < last - turn ? entry(turn + i) : -1;
                if (id[k] >= 0 && !(comes_twice(id[k]) && lr_allows(mask, id[k]))) id[k] = -1;
                ids[i] = id[k];
                values[i] = id[k] >= 0 ? p.bias_values[turn + i] : 0.f;
                mine |= id[k] >= 0;
            }
            if (!__syncthreads_or(mine)) continue;
            auto home = [](int x) { return ((unsigned)x * 2654435761u) >> 20 & (PLACES - 1); };
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                if (id[k] < 0) continue;
                unsigned at = home(id[k]);
                for (;;) {
                    const int there = atomicCAS(&token[at], -1, id[k]);
                    if (there == -1 || there == id[k]) break;
                    at = (at + 1) & (PLACES - 1);
                }
                place[k] = at;
                atomicMin(&owner[at], k * LR_THREADS + (int)threadIdx.x);
                atomicAdd(&count[at], 1);
            }
            __syncthreads();
            float sum[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int i = k * LR_THREADS + threadIdx.x;
                is_first[k] = id[k] >= 0 && owner[place[k]] == i;
                if (!is_first[k]) continue;
                sum[k] = values[i];
                for (int j = i + 1, left = count[place[k]] - 1; left > 0; ++j)
                    if (ids[j] == id[k]) { sum[k] += values[j]; --left; }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (is_first[k]) { values[k * LR_THREADS + threadIdx.x] = sum[k]; count[place[k]] = 0; }
            // ---- the turns behind, one after the other
            for (int then = turn + LR_LIST; then < last; then += LR_LIST) {
                int found[PER];
                bool any = false;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const int e = then + k * LR_THREADS + (int)threadIdx.x, x = entry(e);
                    found[k] = -1;
                    if (x < 0 || !comes_twice(x)) continue;
                    for (unsigned at = home(x); token[at] != -1; at = (at + 1) & (PLACES - 1))
                        if (token[at] == x) { found[k] = at; break; }
                    if (found[k] < 0) continue;
                    any = true;
                    atomicMin(&lead[found[k]], e);
                    atomicAdd(&count[found[k]], 1);
                }
                if (!__syncthreads_or(any)) continue;
#pragma unroll
                for (int k = 0; k < PER; ++k) {                     // the token's first entry of this turn adds all of them
                    const int e = then + k * LR_THREADS + (int)threadIdx.x;
                    if (found[k] < 0 || lead[found[k]] != e) { found[k] = -1; continue; }
                    const int x = token[found[k]];
                    float add = values[owner[found[k]]] + p.bias_values[e];
                    for (int j = e + 1, left = count[found[k]] - 1; left > 0; ++j)
                        if (p.bias_ids[j] == x) { add += p.bias_values[j]; --left; }
                    values[owner[found[k]]] = add;
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (found[k] >= 0) { lead[found[k]] = NONE; count[found[k]] = 0; }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                if (!is_first[k]) continue;
                out[id[k]] += values[k * LR_THREADS + threadIdx.x];
                atomicAnd(&twice[(id[k] - id0) >> 5], ~(1u << (id[k] & 31)));
            }
        }
    }
}

template <bool LONG>
__global__ void __launch_bounds__(LR_THREADS) add_biases_kernel(const LrArgs p) {
    constexpr int PER = LR_LIST / LR_THREADS, PLACES = 4 * LR_LIST;      // entries of a thread; places of the table, most of them empty
    __shared__ int ids[LR_LIST], table[3 * PLACES];
    __shared__ float values[LR_LIST];
    int *token = table, *first_of = table + PLACES, *count = table + 2 * PLACES;
    pdl_launch_dependents();
    // Lists and masks were there before the first kernel began to work; the wait is for its results.
    const int b = blockIdx.x, m = p.by_slot ? lr_mask(p, p.slots[b], p.n_slots) : lr_mask(p, b, p.rows);
    const int2 list = p.bias_range[b];
    const int last = max(min(list.y, p.n_bias), 0), first = min(max(list.x, 0), last);
    const unsigned* mask = m >= 0 && m < p.n_masks ? p.masks + (size_t)m * p.mask_words : nullptr;
    float* out = p.out + (size_t)b * p.vocab;
    if constexpr (LONG) {
        __shared__ unsigned twice[LR_BITS / 32];
        if (last - first > LR_LIST) {                               // (the whole block)
            lr_long_list(p, first, last, mask, out, table, ids, values, twice);
            return;
        }
    }
    for (int i = threadIdx.x; i < PLACES; i += LR_THREADS) { token[i] = -1; first_of[i] = LR_LIST; count[i] = 0; }
    int id[PER], place[PER];
    float now[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int e = k * LR_THREADS + threadIdx.x;
        id[k] = e < last - first ? p.bias_ids[first + e] : -1;
        values[e] = e < last - first ? p.bias_values[first + e] : 0.f;
        if (id[k] >= p.vocab) id[k] = -1;
        ids[e] = id[k];
    }
    __syncthreads();                                                // (the table is empty)
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (id[k] < 0) continue;
        if (!lr_allows(mask, id[k])) { id[k] = -1; continue; }
        unsigned at = ((unsigned)id[k] * 2654435761u) >> 20 & (PLACES - 1);
        for (;;) {
            const int there = atomicCAS(&token[at], -1, id[k]);
            if (there == -1 || there == id[k]) break;
            at = (at + 1) & (PLACES - 1);
        }
        place[k] = at;
        atomicMin(&first_of[at], k * LR_THREADS + (int)threadIdx.x);
        atomicAdd(&count[at], 1);
    }
    pdl_wait();                                                     // (also where the list is empty: the kernel behind this one counts on the first one's end)
#pragma unroll
    for (int k = 0; k < PER; ++k) now[k] = id[k] >= 0 ? out[id[k]] : 0.f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int e = k * LR_THREADS + threadIdx.x;
        if (id[k] < 0 || first_of[place[k]] != e) continue;
        float sum = values[e];
        for (int i = e + 1, left = count[place[k]] - 1; left > 0; ++i)
            if (ids[i] == id[k]) { sum += values[i]; --left; }
        out[id[k]] = now[k] + sum;
    }
}

// Tokens into the table of what a sequence has seen.  prompt: their sign bits are set; else their counts go up by one, to 32,767 at most.
// states (or null): the state of each sequence's token automaton follows its token, state = transitions[state][token], -1 stays -1;
// the tokens of one sequence are taken in their order.
__global__ void __launch_bounds__(LR_THREADS) note_tokens_kernel(short* history, int n_slots, int vocab, const int* slots, const int* tokens, int n,
                                                                 int prompt, int* states, const int* transitions, int n_states) {
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x * LR_THREADS + threadIdx.x;
    if (i >= n) return;
    const int slot = slots[i], token = tokens[i];
    if (slot < 0 || slot >= n_slots) return;
    if (history && token >= 0 && token < vocab) {
        unsigned short* at = reinterpret_cast<unsigned short*>(history) + (size_t)slot * vocab + token;
        unsigned short old = *at;
        for (;;) {
            const unsigned short to = prompt ? old | 0x8000u : (old & 0x7fffu) == 0x7fffu ? old : old + 1;
            if (to == old) break;
            const unsigned short found = atomicCAS(at, old, to);
            if (found == old) break;
            old = found;
        }
    }
    if (states) {
        for (int j = 0; j < i; ++j)
            if (slots[j] == slot) return;                           // the sequence's first token here takes all of them
        int s = states[slot];
        for (int j = i; j < n; ++j) {
            if (slots[j] != slot) continue;
            const int t = tokens[j];
            s = s >= 0 && s < n_states && t >= 0 && t < vocab ? transitions[(size_t)s * vocab + t] : -1;
        }
        states[slot] = s;
    }
}

extern "C" void pe_set_pdl(int on) { pe_pdl_enabled() = on ? 1 : 0; }     // (this library's own copy of the switch)

extern "C" int pe_adjust_logits(const float* logits, float* out, int rows, int vocab, const int* slots, const void* history, int n_slots,
                                const float* penalties, const void* bias_range, const int* bias_ids, const float* bias_values, int n_bias,
                                const void* masks, int n_masks, const int* mask_rows, int by_slot, void* stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || rows > 65535 || (history && (!slots || !penalties)) || (bias_ids && (!bias_range || !bias_values)) || (masks && !mask_rows) || (by_slot && !slots) ||
        ((uintptr_t)bias_range & 7))
        return PE_ERR_UNSUPPORTED;
    const LrArgs p = {logits, out, rows, vocab, slots, (const short*)history, n_slots, penalties, (const int2*)bias_range, bias_ids, bias_values, n_bias,
                      (const unsigned*)masks, n_masks, (vocab + 31) / 32, mask_rows, by_slot};
    const bool aligned = !(((uintptr_t)logits | (uintptr_t)out) & 15), in_place = logits == out;
    const auto pick = [&](auto by) {
        constexpr bool BY_SLOT = decltype(by)::value;
        return aligned ? (in_place ? adjust_logits_kernel<true, true, BY_SLOT> : adjust_logits_kernel<true, false, BY_SLOT>)
                       : (in_place ? adjust_logits_kernel<false, true, BY_SLOT> : adjust_logits_kernel<false, false, BY_SLOT>);
    };
    const auto kernel = by_slot ? pick(std::true_type()) : pick(std::false_type());
    PE_TRY(pe_launch(kernel, dim3((vocab + LR_CHUNK - 1) / LR_CHUNK, rows), LR_THREADS, 0, (cudaStream_t)stream, p));
    PE_LAUNCH_CHECK();
    if (bias_ids) {
        PE_TRY(pe_launch(n_bias > LR_LIST ? add_biases_kernel<true> : add_biases_kernel<false>, rows, LR_THREADS, 0, (cudaStream_t)stream, p));
        PE_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int pe_note_tokens(void* history, int n_slots, int vocab, const int* slots, const int* tokens, int n, int prompt, int* states,
                              const int* transitions, int n_states, void* stream) {
    if (n <= 0) return 0;
    if (vocab <= 0 || n_slots <= 0 || (states && (!transitions || n_states <= 0)) || (!history && !states)) return PE_ERR_UNSUPPORTED;
    PE_TRY(pe_launch(note_tokens_kernel, (n + LR_THREADS - 1) / LR_THREADS, LR_THREADS, 0, (cudaStream_t)stream, (short*)history, n_slots, vocab, slots, tokens, n,
                     prompt, states, transitions, n_states));
    PE_LAUNCH_CHECK();
    return 0;
}
