// Rules on what a sequence may go on with, applied to float32 logits before the next token is chosen.
//
// For row b of the batch (sequence slot s = slots[b]) and token v, h = history[s][v] (16 bits: the sign bit says that v stands in the
// prompt, the other 15 how often it has been generated):
//     z = logits[b][v]
//     h != 0:   z = z > 0 ? z / repetition : z * repetition
//     count c:  z -= presence + c * frequency                     (c > 0)
//     z += the row's biases of v (a list of ids and values; an id that stands there twice counts twice, in the list's order)
//     v is not in the row's mask: z = -inf                        (whatever z was)
#include "common.cuh"

#define LR_THREADS 256
#define LR_CHUNK 2048

struct LrArgs {
    const float* logits; float* out; int rows, vocab;
    const int* slots; const short* history; int n_slots;
    const float* penalties;
    const int2* bias_range; const int* bias_ids; const float* bias_values; int n_bias;
    const unsigned* masks; int n_masks, mask_words; const int* mask_rows;
};

__global__ void __launch_bounds__(LR_THREADS) adjust_logits_kernel(const LrArgs p) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, begin = blockIdx.x * LR_CHUNK, end = min(p.vocab, begin + LR_CHUNK);
    const float* row = p.logits + (size_t)b * p.vocab;
    float* out = p.out + (size_t)b * p.vocab;
    const int slot = p.history ? p.slots[b] : -1;
    const short* seen = p.history && slot >= 0 && slot < p.n_slots ? p.history + (size_t)slot * p.vocab : nullptr;
    const float repetition = seen ? p.penalties[3 * b] : 1.f, presence = seen ? p.penalties[3 * b + 1] : 0.f, frequency = seen ? p.penalties[3 * b + 2] : 0.f;
    const int2 list = p.bias_ids ? p.bias_range[b] : make_int2(0, 0);
    const int m = p.masks ? p.mask_rows[b] : -1;
    const unsigned* mask = p.masks && m >= 0 && m < p.n_masks ? p.masks + (size_t)m * p.mask_words : nullptr;
    for (int v = begin + threadIdx.x; v < end; v += LR_THREADS) {
        float z = row[v];
        if (seen) {
            const int h = seen[v], count = h & 0x7fff;
            if (h != 0) z = z > 0.f ? z / repetition : z * repetition;
            if (count > 0) z -= fmaf((float)count, frequency, presence);
        }
        float bias = 0.f;
        for (int e = max(list.x, 0); e < min(list.y, p.n_bias); ++e)
            if (p.bias_ids[e] == v) bias += p.bias_values[e];
        z += bias;
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1u)) z = -INFINITY;
        out[v] = z;
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
                                const void* masks, int n_masks, const int* mask_rows, void* stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || rows > 65535 || (history && (!slots || !penalties)) || (bias_ids && (!bias_range || !bias_values)) || (masks && !mask_rows) ||
        ((uintptr_t)bias_range & 7))
        return PE_ERR_UNSUPPORTED;
    const LrArgs p = {logits, out, rows, vocab, slots, (const short*)history, n_slots, penalties, (const int2*)bias_range, bias_ids, bias_values, n_bias,
                      (const unsigned*)masks, n_masks, (vocab + 31) / 32, mask_rows};
    PE_TRY(pe_launch(adjust_logits_kernel, dim3((vocab + LR_CHUNK - 1) / LR_CHUNK, rows), LR_THREADS, 0, (cudaStream_t)stream, p));
    PE_LAUNCH_CHECK();
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
