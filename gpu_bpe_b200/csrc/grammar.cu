// A grammar over a vocabulary: which tokens a byte automaton allows in a state, and the state behind a token.  No counterpart in the
// reference.
//
// Bytes that every state treats alike are one class; the automaton's table is n_states x classes, the vocabulary's entries are kept as strings of
// classes.
#include <algorithm>
#include <cstring>
#include <map>
#include <new>
#include <string>
#include <vector>

#include "ctx.cuh"

namespace b200bpe {

constexpr int GR_THREADS = 256;
constexpr uint32_t GR_DEAD = 0xFFFFu;

struct GrammarTables {
    const uint16_t* next;        // [state * classes + class]
    const uint8_t* accepting;
    const uint8_t* text;         // the entries' classes
    const uint64_t* off;
    uint32_t states, classes, entries, end_token;
};

// The state behind token t's bytes, or GR_DEAD.
__device__ __forceinline__ uint32_t walk(const GrammarTables& g, uint32_t state, uint32_t t) {
    const uint64_t hi = g.off[t + 1];
    for (uint64_t p = g.off[t]; p < hi && state != GR_DEAD; p++) state = g.next[state * g.classes + g.text[p]];
    return state;
}

// A thread per token and row; a warp makes a word.
__global__ void __launch_bounds__(GR_THREADS)
k_grammar_mask(const GrammarTables g, const uint32_t* __restrict__ states, uint32_t n_rows, uint32_t* __restrict__ out, uint64_t stride) {
    const uint32_t words = (g.entries + 31u) / 32u;
    const uint64_t all = (uint64_t)words * n_rows;
    for (uint64_t i = ((uint64_t)blockIdx.x * GR_THREADS + threadIdx.x) >> 5; i < all; i += (uint64_t)gridDim.x * (GR_THREADS / 32)) {
        const uint32_t row = (uint32_t)(i / words), word = (uint32_t)(i % words), t = word * 32u + (threadIdx.x & 31u);
        const uint32_t state = states[row];
        bool ok = false;
        if (state < g.states && t < g.entries)
            ok = t == g.end_token ? g.accepting[state] != 0 : g.off[t + 1] > g.off[t] && walk(g, state, t) != GR_DEAD;
        const uint32_t bits = __ballot_sync(0xFFFFFFFFu, ok);
        if ((threadIdx.x & 31u) == 0) out[row * stride + word] = bits;
    }
}

__global__ void __launch_bounds__(GR_THREADS)
k_grammar_advance(const GrammarTables g, const uint32_t* states, const uint32_t* __restrict__ tokens, uint32_t n_rows, uint32_t* states_out,
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
        else if (state < g.states && t < g.entries && g.off[t + 1] > g.off[t]) to = walk(g, state, t);
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
        const size_t at_off = up((size_t)n_states * classes * 2), at_acc = at_off + up(((size_t)n_entries + 1) * 8), at_text = at_acc + up(n_states);
        std::vector<uint8_t> host(at_text + up(n + 1), 0);
        uint16_t* next = reinterpret_cast<uint16_t*>(host.data());
        for (uint32_t s = 0; s < n_states; s++)
            for (uint32_t k = 0; k < classes; k++) next[(size_t)s * classes + k] = columns[(size_t)member[k] * n_states + s];
        std::memcpy(host.data() + at_off, offsets, ((size_t)n_entries + 1) * 8);
        std::memcpy(host.data() + at_acc, accepting, n_states);
        for (uint64_t p = 0; p < n; p++) host[at_text + p] = class_of[bytes[p]];

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
        g.g = {reinterpret_cast<uint16_t*>(base), base + at_acc, base + at_text, reinterpret_cast<uint64_t*>(base + at_off), n_states, classes, n_entries, end_token};
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
    const uint64_t ctas = ((uint64_t)words * n_rows + GR_THREADS / 32 - 1) / (GR_THREADS / 32);
    const int grid = (int)std::min<uint64_t>(ctas, (uint64_t)h->g.ctx->sm_count * 64);
    k_grammar_mask<<<grid, GR_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(g, states, n_rows, mask_out, mask_stride);
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
