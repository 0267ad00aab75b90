// A grammar over a vocabulary: which tokens a byte automaton allows in a state, and the state behind a token.  No counterpart in the
// reference.
//
// Bytes that every state treats alike are one class; the automaton's table is n_states x classes, the vocabulary's entries are kept as strings of
// classes.
//
// A mask is a walk of each entry's bytes from each row's state, one look-up a byte, but most walks need not be made.  Many die at their first
// byte; and inside a text, a number or a name the automaton stays where it is, so an entry all of whose bytes lead from the state back to it is allowed
// as a whole.  Which classes an entry has, and which ones lead a state to itself, are sets of 64 bits (class modulo 64: a state's bit is set
// if all classes of the bit lead back), so that this is one comparison.  What it does not decide goes through a warp's list, so that the walks that
// are left are made by full warps.
#include <algorithm>
#include <cstring>
#include <map>
#include <new>
#include <string>
#include <vector>

#include "ctx.cuh"

namespace b200bpe {

constexpr int GR_THREADS = 256, GR_WARPS = GR_THREADS / 32;
constexpr uint32_t GR_DEAD = 0xFFFFu;
constexpr uint32_t GR_TOKENS = 128;                       // of a warp
constexpr uint32_t GR_ROWS = 16;                          // of a CTA: an entry's data is loaded once for all of them

struct Entry {
    unsigned long long classes;      // of the first eight bytes
    unsigned long long all, rest;    // sets of the classes of all bytes, and of all but the first
    uint32_t at, len;                // in text
};

struct GrammarTables {
    const uint16_t* next;            // [state * classes + class]
    const unsigned long long* stays; // [state]: set of the classes that lead back to it
    const uint8_t* accepting;
    const uint8_t* text;             // the entries' classes
    const Entry* entry;
    uint32_t states, classes, entries, end_token;
};

// The state behind all bytes of e from the `from`th on, or GR_DEAD.
__device__ __forceinline__ uint32_t walk(const GrammarTables& g, uint32_t state, const Entry& e, uint32_t from) {
    unsigned long long c = e.classes >> from * 8;
    for (uint32_t k = from; k < min(e.len, 8u) && state != GR_DEAD; k++, c >>= 8) state = g.next[state * g.classes + (uint32_t)(c & 255u)];
    for (uint32_t k = 8; k < e.len && state != GR_DEAD; k++) state = g.next[state * g.classes + g.text[e.at + k]];
    return state;
}

// A CTA makes the words of GR_WARPS * GR_TOKENS tokens for GR_ROWS rows.
// 256 rows of 64,256 entries, an automaton of 224 states: 74 us with a walk for each token and row, # us like this; the vocabulary's data is 2.6 MB, the masks 2 MB.
__global__ void __launch_bounds__(GR_THREADS)
k_grammar_mask(const __grid_constant__ GrammarTables g, const uint32_t* __restrict__ states, uint32_t n_rows, uint32_t* __restrict__ out, uint64_t stride) {
    constexpr uint32_t EACH = GR_TOKENS / 32, ROOM = 2 * GR_TOKENS;
    __shared__ uint16_t s_next[GR_ROWS][256];
    __shared__ unsigned long long s_stays[GR_ROWS];
    __shared__ uint32_t s_state[GR_ROWS];
    __shared__ uint32_t s_words[GR_WARPS][GR_ROWS][EACH], s_list[GR_WARPS][ROOM];     // list: row << 28 | token of the warp << 16 | state
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row0 = blockIdx.y * GR_ROWS, rows = min(GR_ROWS, n_rows - row0);
    const uint32_t token0 = (blockIdx.x * GR_WARPS + warp) * GR_TOKENS;
    if (threadIdx.x < rows) {
        const uint32_t state = states[row0 + threadIdx.x];
        s_state[threadIdx.x] = state;
        s_stays[threadIdx.x] = state < g.states ? g.stays[state] : 0ull;
    }
    Entry e[EACH];
#pragma unroll
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t t = token0 + k * 32 + lane;
        if (t < g.entries) e[k] = g.entry[t];
        else e[k].len = 0u;
        if (t == g.end_token) e[k].len = 0u;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * g.classes; i += GR_THREADS) {
        const uint32_t r = i / g.classes, c = i % g.classes;
        s_next[r][c] = s_state[r] < g.states ? g.next[s_state[r] * g.classes + c] : GR_DEAD;
    }
    __syncthreads();
    uint32_t* list = s_list[warp];
    uint32_t listed = 0;
    auto work_off = [&](uint32_t from, uint32_t n) {           // n at most 32
        __syncwarp();
        if ((uint32_t)lane < n) {
            const uint32_t w = list[from + lane], row = w >> 28, token = w >> 16 & (GR_TOKENS - 1u);
            if (walk(g, w & 0xFFFFu, g.entry[token0 + token], 1) != GR_DEAD) atomicOr(&s_words[warp][row][token >> 5], 1u << (token & 31u));
        }
        __syncwarp();
    };
    for (uint32_t r = 0; r < rows; r++) {
        const unsigned long long leaves = ~s_stays[r];
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) {
            bool ok = false, open = false;
            uint32_t state = GR_DEAD;
            if (e[k].len) {
                ok = !(e[k].all & leaves);
                if (!ok) {
                    state = s_next[r][e[k].classes & 255u];
                    if (state != GR_DEAD) {
                        ok = e[k].len == 1u || !(e[k].rest & ~g.stays[state]);
                        open = !ok;
                    }
                }
            }
            const uint32_t bits = __ballot_sync(0xFFFFFFFFu, ok), others = __ballot_sync(0xFFFFFFFFu, open);
            if (lane == 0) s_words[warp][r][k] = bits;
            if (open) list[listed + __popc(others & ((1u << lane) - 1u))] = r << 28 | (k * 32 + lane) << 16 | state;
            listed += __popc(others);
        }
        if (listed > ROOM - GR_TOKENS) {
            while (listed >= 32) {
                listed -= 32;
                work_off(listed, 32);
            }
        }
    }
    while (listed) {
        const uint32_t n = min(listed, 32u);
        listed -= n;
        work_off(listed, n);
    }
    __syncwarp();
    const uint32_t words = (g.entries + 31u) / 32u, word0 = token0 / 32u;
    for (uint32_t i = lane; i < rows * EACH; i += 32) {
        const uint32_t r = i / EACH, k = i % EACH, w = word0 + k;
        if (w >= words) continue;
        uint32_t bits = s_words[warp][r][k];
        if (g.end_token < g.entries && g.end_token / 32u == w && s_state[r] < g.states && g.accepting[s_state[r]]) bits |= 1u << (g.end_token & 31u);
        out[(row0 + r) * stride + w] = bits;
    }
}

__global__ void __launch_bounds__(GR_THREADS)
k_grammar_advance(const __grid_constant__ GrammarTables g, const uint32_t* states, const uint32_t* __restrict__ tokens, uint32_t n_rows, uint32_t* states_out,
                  uint32_t* __restrict__ history, uint64_t history_stride, uint32_t history_cap, const uint32_t* lengths, uint32_t* lengths_out) {
    const uint32_t r = blockIdx.x * GR_THREADS + threadIdx.x;
    if (r >= n_rows) return;
    const uint32_t t = tokens[r];
    uint32_t state = states[r];
    if (history) {
        const uint32_t n = lengths[r];
        const bool fits = t != B200BPE_NO_TOKEN && n < history_cap;
        if (fits) history[r * history_stride + n] = t;
        lengths_out[r] = n + (fits ? 1u : 0u);
    }
    if (t != B200BPE_NO_TOKEN) {
        uint32_t to = GR_DEAD;
        if (state < g.states && t == g.end_token) to = g.accepting[state] ? state : GR_DEAD;
        else if (state < g.states && t < g.entries && g.entry[t].len) to = walk(g, state, g.entry[t], 0);
        state = to == GR_DEAD ? B200BPE_NO_STATE : to;
    }
    states_out[r] = state;
}

// Another thread may be capturing a graph, which forbids allocations to all threads but relaxed ones.
struct Relaxed {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

struct Grammar {
    CtxHold hold;
    Ctx* ctx = nullptr;
    void* block = nullptr;
    GrammarTables g{};
    ~Grammar() {
        if (!ctx) return;
        const OnDevice on(ctx->device);
        const Relaxed relaxed;
        cudaFree(block);         // waits for the work that reads it
    }
};

}  // namespace b200bpe

struct b200bpe_grammar { b200bpe::Grammar g; };

using namespace b200bpe;

extern "C" {

b200bpe_status b200bpe_grammar_create(b200bpe_ctx* c, const uint8_t* bytes, const uint64_t* offsets, uint32_t n_entries, const uint32_t* transitions,
                                      const uint8_t* accepting, uint32_t n_states, uint32_t end_token, b200bpe_grammar** out) {
    if (!offsets || !transitions || !accepting || !out) return refused("b200bpe_grammar_create: null pointer");
    if (n_states == 0 || n_states >= GR_DEAD + 1) return refused("b200bpe_grammar_create: 1 to 65,535 states");
    if (n_entries == 0 || n_entries >= 0xFFFFFFE0u) return refused("b200bpe_grammar_create: a vocabulary without entries, or with too many");
    if (offsets[0] != 0) return refused("b200bpe_grammar_create: offsets do not begin at 0");
    for (uint32_t i = 0; i < n_entries; i++) if (offsets[i + 1] < offsets[i]) return refused("b200bpe_grammar_create: offsets fall");
    const uint64_t n = offsets[n_entries];
    if (n >= 0xFFFFFFFFu) return refused("b200bpe_grammar_create: more than 4 GiB of entries");
    if (n && !bytes) return refused("b200bpe_grammar_create: null bytes");
    if (!c) return refused("b200bpe_grammar_create: null context");
    try {
        // classes: bytes with the same column
        std::vector<uint16_t> columns((size_t)n_states * 256);
        for (uint32_t s = 0; s < n_states; s++)
            for (uint32_t b = 0; b < 256; b++) {
                const uint32_t to = transitions[(size_t)s * 256 + b];
                columns[(size_t)b * n_states + s] = (uint16_t)(to < n_states ? to : GR_DEAD);
            }
        std::map<std::string, uint32_t> known;
        uint8_t class_of[256];
        std::vector<uint32_t> member;
        for (uint32_t b = 0; b < 256; b++) {
            const std::string column(reinterpret_cast<const char*>(&columns[(size_t)b * n_states]), (size_t)n_states * 2);
            const auto at = known.emplace(column, (uint32_t)member.size());
            if (at.second) member.push_back(b);
            class_of[b] = (uint8_t)at.first->second;
        }
        const uint32_t classes = (uint32_t)member.size();
        auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
        const size_t at_stays = up((size_t)n_states * classes * 2), at_acc = at_stays + up((size_t)n_states * 8), at_entry = at_acc + up(n_states);
        const size_t at_text = at_entry + up((size_t)n_entries * sizeof(Entry));
        std::vector<uint8_t> host(at_text + up(n + 1), 0);
        uint16_t* next = reinterpret_cast<uint16_t*>(host.data());
        unsigned long long* stays = reinterpret_cast<unsigned long long*>(host.data() + at_stays);
        for (uint32_t s = 0; s < n_states; s++) {
            stays[s] = ~0ull;
            for (uint32_t k = 0; k < classes; k++) {
                const uint16_t to = next[(size_t)s * classes + k] = columns[(size_t)member[k] * n_states + s];
                if (to != s) stays[s] &= ~(1ull << (k & 63u));
            }
        }
        std::memcpy(host.data() + at_acc, accepting, n_states);
        for (uint64_t p = 0; p < n; p++) host[at_text + p] = class_of[bytes[p]];
        Entry* entry = reinterpret_cast<Entry*>(host.data() + at_entry);
        for (uint32_t t = 0; t < n_entries; t++) {
            Entry& e = entry[t];
            e.at = (uint32_t)offsets[t];
            e.len = (uint32_t)(offsets[t + 1] - offsets[t]);
            for (uint32_t k = 0; k < e.len; k++) {
                const uint8_t of = host[at_text + e.at + k];
                if (k < 8) e.classes |= (unsigned long long)of << 8 * k;
                e.all |= 1ull << (of & 63u);
                if (k) e.rest |= 1ull << (of & 63u);
            }
        }

        const OnDevice on(c->c.device);
        B2_CUDA(on.error);
        const Relaxed relaxed;
        cudaFuncAttributes fa;
        B2_CUDA(cudaFuncGetAttributes(&fa, k_grammar_mask));        // loads the kernels, so that no call has to
        B2_CUDA(cudaFuncGetAttributes(&fa, k_grammar_advance));
        b200bpe_grammar* h = new b200bpe_grammar();
        Grammar& g = h->g;
        g.ctx = &c->c;
        g.hold.take(c);
        cudaError_t e = cudaMalloc(&g.block, host.size());
        cudaStream_t st = c->c.decode_stream;
        if (e == cudaSuccess) e = cudaMemcpyAsync(g.block, host.data(), host.size(), cudaMemcpyHostToDevice, st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
        if (e != cudaSuccess) {
            cudaGetLastError();
            delete h;
            set_last_error(std::string("b200bpe_grammar_create: ") + cudaGetErrorString(e));
            return e == cudaErrorMemoryAllocation ? B200BPE_ERR_OOM : B200BPE_ERR_CUDA;
        }
        uint8_t* base = static_cast<uint8_t*>(g.block);
        g.g = {reinterpret_cast<uint16_t*>(base), reinterpret_cast<unsigned long long*>(base + at_stays), base + at_acc, base + at_text,
               reinterpret_cast<Entry*>(base + at_entry), n_states, classes, n_entries, end_token};
        *out = h;
        return B200BPE_OK;
    } catch (const std::exception&) {
        return B200BPE_ERR_OOM;
    }
}

b200bpe_status b200bpe_grammar_mask(b200bpe_grammar* h, const uint32_t* states, uint32_t n_rows, uint32_t* mask_out, uint64_t mask_stride, void* stream) {
    if (!h) return refused("b200bpe_grammar_mask: null handle");
    if (n_rows >= 1u << 28) return refused("b200bpe_grammar_mask: more than 2^28 - 1 rows");
    if (n_rows == 0) return B200BPE_OK;
    const GrammarTables& g = h->g.g;
    const uint32_t words = (g.entries + 31u) / 32u;
    if (!states || !mask_out) return refused("b200bpe_grammar_mask: null pointer");
    if (mask_stride < words && n_rows > 1) return refused("b200bpe_grammar_mask: rows of the mask overlap");
    const OnDevice on(h->g.ctx->device);
    B2_CUDA(on.error);
    // (a grid has at most 65,535 CTAs in its second direction)
    constexpr uint32_t most = 65535u * GR_ROWS;
    for (uint32_t r = 0; r < n_rows; r += most) {
        const uint32_t n = std::min(most, n_rows - r);
        const dim3 grid((g.entries + GR_WARPS * GR_TOKENS - 1) / (GR_WARPS * GR_TOKENS), (n + GR_ROWS - 1) / GR_ROWS);
        k_grammar_mask<<<grid, GR_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(g, states + r, n, mask_out + (uint64_t)r * mask_stride, mask_stride);
    }
    B2_CUDA(cudaGetLastError());
    return B200BPE_OK;
}

b200bpe_status b200bpe_grammar_advance(b200bpe_grammar* h, const uint32_t* states, const uint32_t* tokens, uint32_t n_rows, uint32_t* states_out,
                                       uint32_t* history, uint64_t history_stride, uint32_t history_cap, const uint32_t* lengths,
                                       uint32_t* lengths_out, void* stream) {
    if (!h) return refused("b200bpe_grammar_advance: null handle");
    if (n_rows >= 1u << 28) return refused("b200bpe_grammar_advance: more than 2^28 - 1 rows");
    if (n_rows == 0) return B200BPE_OK;
    if (!states || !tokens || !states_out) return refused("b200bpe_grammar_advance: null pointer");
    if (history && (!lengths || !lengths_out)) return refused("b200bpe_grammar_advance: a history without lengths");
    if (history && history_stride < history_cap && n_rows > 1) return refused("b200bpe_grammar_advance: rows of the history overlap");
    if (!history && (lengths || lengths_out)) return refused("b200bpe_grammar_advance: lengths without a history");
    const OnDevice on(h->g.ctx->device);
    B2_CUDA(on.error);
    const uint64_t grid = ((uint64_t)n_rows + GR_THREADS - 1) / GR_THREADS;
    k_grammar_advance<<<(uint32_t)grid, GR_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(h->g.g, states, tokens, n_rows, states_out, history, history_stride,
                                                                                          history_cap, lengths, lengths_out);
    B2_CUDA(cudaGetLastError());
    return B200BPE_OK;
}

void b200bpe_grammar_destroy(b200bpe_grammar* h) { delete h; }

}  // extern "C"
