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
// are left are made by full warps.  Most states of a grammar let few bytes through.  So a CTA's entries lie in the order of their first class, and a warp
// passes over the 32 entries whose first classes a state all refuses.
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
constexpr uint32_t GR_TILE = GR_WARPS * GR_TOKENS;        // of a CTA
constexpr uint32_t GR_ROWS = 16;                          // of a CTA, at most: an entry's data is loaded once for all of them

struct __align__(16) Entry {
    unsigned long long classes;      // of the first eight bytes
    unsigned long long rest;         // set of the classes of all bytes but the first
    uint32_t at, len;                // in text
    unsigned long long pad;
};

struct GrammarTables {
    const uint16_t* next;            // [state * classes + class]
    const unsigned long long* stays; // [state]: set of the classes that lead back to it
    const unsigned long long* lives; // [state]: set of the classes that lead somewhere
    const uint8_t* accepting;
    const uint8_t* text;             // the entries' classes
    const Entry* entry;
    // in the order of a tile's entries (those that cannot be allowed by their bytes, the end token and entries without, are not among them)
    const unsigned long long* all;   // set of an entry's classes; 0 behind a tile's last
    const uint32_t* first;           // classes of its first two bytes, its place in the tile << 16, and 1 << 31 if it has more than one byte
    uint32_t states, classes, entries, end_token;
};

// The state behind all bytes of e from the `from`th on, or GR_DEAD.  (Passing over bytes that lead back to a state without looking them up makes
// the lanes of a warp take turns: 33 us became 44.)
__device__ __forceinline__ uint32_t walk(const GrammarTables& g, uint32_t state, const Entry& e, uint32_t from) {
    unsigned long long c = e.classes >> from * 8;
    for (uint32_t k = from; k < min(e.len, 8u) && state != GR_DEAD; k++, c >>= 8) state = g.next[state * g.classes + (uint32_t)(c & 255u)];
    for (uint32_t k = 8; k < e.len && state != GR_DEAD; k++) state = g.next[state * g.classes + g.text[e.at + k]];
    return state;
}

// A CTA makes the words of GR_TILE tokens for some rows.  256 rows of 64,256 entries, an automaton of 205 states and 36 classes: 26 us, where a walk for
// each token and row took 74; 1,500 rows of 32,256 entries: 57 us, against 200.  Of those 256 rows' pairs 93 % die at their first byte, 3 % stay where they are,
// and 4 % are looked at further.  The memory's part is below a microsecond; what bounds it is instructions (14.5 million of warps, 13 us if none waited)
// and the scattered look-ups of the walks.
__global__ void __launch_bounds__(GR_THREADS, 8)
k_grammar_mask(const __grid_constant__ GrammarTables g, const uint32_t* __restrict__ states, uint32_t n_rows, uint32_t* __restrict__ out, uint64_t stride, uint32_t cta_rows) {
    constexpr uint32_t EACH = GR_TOKENS / 32, ROOM = 2 * GR_TOKENS;
    __shared__ uint16_t s_next[GR_ROWS][256];
    __shared__ unsigned long long s_stays[GR_ROWS], s_lives[GR_ROWS];
    __shared__ uint32_t s_state[GR_ROWS];
    __shared__ uint32_t s_words[GR_ROWS][GR_TILE / 32], s_list[GR_WARPS][ROOM], s_listed[GR_WARPS];       // list: row << 28 | place in the tile << 16 | state
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row0 = blockIdx.y * cta_rows, rows = min(cta_rows, n_rows - row0);
    const uint32_t token0 = blockIdx.x * GR_TILE;
    if (threadIdx.x < rows) {
        const uint32_t state = states[row0 + threadIdx.x];
        s_state[threadIdx.x] = state;
        s_stays[threadIdx.x] = state < g.states ? g.stays[state] : 0ull;
        s_lives[threadIdx.x] = state < g.states ? g.lives[state] : 0ull;
    }
    for (uint32_t i = threadIdx.x; i < GR_ROWS * (GR_TILE / 32); i += GR_THREADS) s_words[i / (GR_TILE / 32)][i % (GR_TILE / 32)] = 0u;
    unsigned long long all[EACH], starts[EACH];        // starts: set of the first classes of a warp's entries
    uint32_t first[EACH];
#pragma unroll
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t t = token0 + (k * GR_WARPS + warp) * 32 + lane;         // (both arrays have whole tiles; neighbours are much alike, so each goes to another warp)
        all[k] = g.all[t];
        first[k] = g.first[t];
        const uint32_t bit = all[k] ? 1u << (first[k] & 31u) : 0u;
        starts[k] = (unsigned long long)__reduce_or_sync(0xFFFFFFFFu, first[k] & 32u ? bit : 0u) << 32 | __reduce_or_sync(0xFFFFFFFFu, first[k] & 32u ? 0u : bit);
    }
    __syncthreads();
    for (uint32_t r = warp; r < rows; r += GR_WARPS)
        for (uint32_t c = lane; c < g.classes; c += 32) s_next[r][c] = s_state[r] < g.states ? g.next[s_state[r] * g.classes + c] : GR_DEAD;
    __syncthreads();
    uint32_t* list = s_list[warp];
    uint32_t listed = 0;
    auto work_off = [&](uint32_t w) {
        const uint32_t row = w >> 28, place = w >> 16 & (GR_TILE - 1u), state = w & 0xFFFFu;
        const Entry e = g.entry[token0 + place];
        if (!(e.rest & ~g.stays[state]) || walk(g, state, e, 1) != GR_DEAD) atomicOr(&s_words[row][place >> 5], 1u << (place & 31u));
    };
    for (uint32_t r = 0; r < rows; r++) {
        const unsigned long long leaves = ~s_stays[r], lives = s_lives[r];
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) {
            if (!(starts[k] & lives)) continue;
            bool ok = !(all[k] & leaves), open = false;
            uint32_t state = GR_DEAD;
            if (!ok) {
                state = s_next[r][first[k] & 255u];
                if (state != GR_DEAD) {
                    // (neighbours have the same first class, so that this is one address for most of them)
                    ok = !(first[k] >> 31);
                    open = !ok && g.lives[state] >> (first[k] >> 8 & 63u) & 1ull;
                }
            }
            if (ok && all[k]) atomicOr(&s_words[r][first[k] >> 21 & 31u], 1u << (first[k] >> 16 & 31u));
            const uint32_t others = __ballot_sync(0xFFFFFFFFu, open);
            if (open) list[listed + __popc(others & ((1u << lane) - 1u))] = r << 28 | (first[k] & 0x03FF0000u) | state;
            listed += __popc(others);
        }
        if (listed > ROOM - GR_TOKENS) {
            __syncwarp();
            for (; listed >= 32; listed -= 32) work_off(list[listed - 32 + lane]);
            __syncwarp();
        }
    }
    if (lane == 0) s_listed[warp] = listed;
    __syncthreads();
    // what is left is every warp's
    uint32_t all_listed = 0;
#pragma unroll
    for (int w = 0; w < GR_WARPS; w++) all_listed += s_listed[w];
    for (uint32_t i = threadIdx.x; i < all_listed; i += GR_THREADS) {
        uint32_t w = 0, at = i;
        while (at >= s_listed[w]) at -= s_listed[w++];
        work_off(s_list[w][at]);
    }
    __syncthreads();
    const uint32_t words = (g.entries + 31u) / 32u, word0 = token0 / 32u;
    for (uint32_t i = threadIdx.x; i < rows * (GR_TILE / 32); i += GR_THREADS) {
        const uint32_t r = i / (GR_TILE / 32), k = i % (GR_TILE / 32), w = word0 + k;
        if (w >= words) continue;
        uint32_t bits = s_words[r][k];
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
        if (state < g.states && t < g.entries && t == g.end_token) to = g.accepting[state] ? state : GR_DEAD;
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
    if (n_entries == 0 || n_entries >= 1u << 28) return refused("b200bpe_grammar_create: a vocabulary without entries, or with too many");
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
        const size_t tiled = ((size_t)n_entries + GR_TILE - 1) / GR_TILE * GR_TILE;
        const size_t at_stays = up((size_t)n_states * classes * 2), at_lives = at_stays + up((size_t)n_states * 8), at_acc = at_lives + up((size_t)n_states * 8);
        const size_t at_entry = at_acc + up(n_states), at_all = at_entry + up((size_t)n_entries * sizeof(Entry)), at_first = at_all + up(tiled * 8);
        const size_t at_text = at_first + up(tiled * 4);
        std::vector<uint8_t> host(at_text + up(n + 1), 0);
        uint16_t* next = reinterpret_cast<uint16_t*>(host.data());
        unsigned long long* stays = reinterpret_cast<unsigned long long*>(host.data() + at_stays);
        unsigned long long* lives = reinterpret_cast<unsigned long long*>(host.data() + at_lives);
        for (uint32_t s = 0; s < n_states; s++) {
            stays[s] = ~0ull;
            lives[s] = 0ull;
            for (uint32_t k = 0; k < classes; k++) {
                const uint16_t to = next[(size_t)s * classes + k] = columns[(size_t)member[k] * n_states + s];
                if (to != s) stays[s] &= ~(1ull << (k & 63u));
                if (to != GR_DEAD) lives[s] |= 1ull << (k & 63u);
            }
        }
        std::memcpy(host.data() + at_acc, accepting, n_states);
        for (uint64_t p = 0; p < n; p++) host[at_text + p] = class_of[bytes[p]];
        Entry* entry = reinterpret_cast<Entry*>(host.data() + at_entry);
        unsigned long long* all = reinterpret_cast<unsigned long long*>(host.data() + at_all);
        uint32_t* first = reinterpret_cast<uint32_t*>(host.data() + at_first);
        for (uint32_t t = 0; t < n_entries; t++) {
            Entry& e = entry[t];
            e.at = (uint32_t)offsets[t];
            e.len = (uint32_t)(offsets[t + 1] - offsets[t]);
            for (uint32_t k = 0; k < e.len; k++) {
                const uint8_t of = host[at_text + e.at + k];
                if (k < 8) e.classes |= (unsigned long long)of << 8 * k;
                if (k) e.rest |= 1ull << (of & 63u);
            }
        }
        for (uint32_t t0 = 0; t0 < n_entries; t0 += GR_TILE) {
            const uint32_t t1 = std::min<uint64_t>((uint64_t)t0 + GR_TILE, n_entries);
            uint32_t start[257] = {};
            auto stands = [&](uint32_t t) { return entry[t].len != 0u && t != end_token; };
            for (uint32_t t = t0; t < t1; t++) if (stands(t)) start[(entry[t].classes & 255u) + 1]++;
            for (uint32_t k = 0; k < 256; k++) start[k + 1] += start[k];
            for (uint32_t t = t0; t < t1; t++)
                if (stands(t)) {
                    const uint32_t of = (uint32_t)(entry[t].classes & 255u);
                    const size_t to = (size_t)t0 + start[of]++;
                    all[to] = entry[t].rest | 1ull << (of & 63u);
                    first[to] = (uint32_t)(entry[t].classes & 0xFFFFu) | (t - t0) << 16 | (entry[t].len > 1u ? 1u << 31 : 0u);
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
        g.g = {reinterpret_cast<uint16_t*>(base), reinterpret_cast<unsigned long long*>(base + at_stays),
               reinterpret_cast<unsigned long long*>(base + at_lives), base + at_acc, base + at_text,
               reinterpret_cast<Entry*>(base + at_entry), reinterpret_cast<unsigned long long*>(base + at_all),
               reinterpret_cast<uint32_t*>(base + at_first), n_states, classes, n_entries, end_token};
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
    if ((reinterpret_cast<uint64_t>(states) | reinterpret_cast<uint64_t>(mask_out)) % 4) return refused("b200bpe_grammar_mask: a misaligned pointer");
    if (mask_stride < words && n_rows > 1) return refused("b200bpe_grammar_mask: rows of the mask overlap");
    const OnDevice on(h->g.ctx->device);
    B2_CUDA(on.error);
    // Rows of a CTA: some states have many times the work of others, so that few rows each share the work out better, and many load the entries less
    // often, which pays once there are CTAs for every place on the GPU (148 SMs with eight) about twice over.  63 tiles and 256 rows: 30.6 us with 4, 38.9 with 8,
    // 38.4 with 16; 512 rows: 45.6, 43.5, 48.1; 1,024: 86.7, 72.1, 65.4.  32 tiles and 512 rows: 26.5, 31.4, 34.1; 1,024: 47.2, 39.8, 38.8.  (Fewer than 4 gain a
    // quarter with few tiles and cost it with many: 4 tiles and 256 rows 7.6 us with 2 and 9.8 with 4, 63 tiles 34.9 and 30.6.)
    const uint32_t tiles = (g.entries + GR_TILE - 1) / GR_TILE;
    uint32_t each = GR_ROWS;
    while (each > 4 && (uint64_t)tiles * ((n_rows + each - 1) / each) < 2560) each /= 2;
    const uint32_t most = 65535u * each;             // (a grid has at most 65,535 CTAs in its second direction)
    for (uint32_t r = 0; r < n_rows; r += most) {
        const uint32_t n = std::min(most, n_rows - r);
        k_grammar_mask<<<dim3(tiles, (n + each - 1) / each), GR_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(g, states + r, n, mask_out + (uint64_t)r * mask_stride,
                                                                                                              mask_stride, each);
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
    for (const void* p : {(const void*)states, (const void*)tokens, (const void*)states_out, (const void*)history, (const void*)lengths, (const void*)lengths_out})
        if (reinterpret_cast<uint64_t>(p) % 4) return refused("b200bpe_grammar_advance: a misaligned pointer");
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
