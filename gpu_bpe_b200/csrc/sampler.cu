// The next token of every request: penalties, biases and masks on a model's logits, and the choice of a token.  No counterpart in the
// reference, whose tokens end in decode.
//
// A row of logits is worked on by one cluster of CTAs.  Each CTA holds a slice of the row's adjusted logits x (32 bits) in its shared memory, so
// the row is read from memory once however many passes the choice takes, and the cluster's barriers and distributed shared memory join the
// slices: no workspace in global memory, so a handle can serve any number of streams and graphs at once.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <new>
#include <string>

#include "ctx.cuh"

namespace cg = cooperative_groups;

namespace b200bpe {

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr uint32_t SM_MAX_CLUSTER = 8;           // portable size
constexpr uint32_t SM_MAX_SLICE = 57344;         // 224 KB of 32-bit values
constexpr uint32_t SM_MAX_VOCAB = SM_MAX_SLICE * SM_MAX_CLUSTER;
constexpr uint32_t SM_MAX_BIAS = 1024;
constexpr float SM_GREEDY_BELOW = 1.0f / 65536;

template <class T>
struct Packed {                                  // 16 bytes of logits
    static constexpr int N = 16 / sizeof(T);
    uint4 v;
    __device__ float get(int i) const;
};
template <>
__device__ float Packed<float>::get(int i) const { return __uint_as_float((&v.x)[i]); }
template <>
__device__ float Packed<__half>::get(int i) const { return __half2float(__ushort_as_half((unsigned short)((&v.x)[i >> 1] >> ((i & 1) * 16)))); }
template <>
__device__ float Packed<__nv_bfloat16>::get(int i) const { return __uint_as_float(((&v.x)[i >> 1] >> ((i & 1) * 16)) << 16); }

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void rounded(float x, float* to) { *to = x; }
__device__ __forceinline__ void rounded(float x, __half* to) { *to = __float2half_rn(x); }
__device__ __forceinline__ void rounded(float x, __nv_bfloat16* to) { *to = __float2bfloat16_rn(x); }

// One row's slice in a CTA: tokens [lo, lo + len) of row `row`; token lo + i lies at x[i].  x starts `lead` elements into the CTA's buffer, so that what is
// 16-byte aligned in the logits is so in the buffer, too; places in front of and behind the slice, up to `padded`, hold -infinity.
struct Slice {
    uint32_t row, lo, len, lead, padded;
    float* buf;
    __device__ float* x() const { return buf + lead; }
};

// Tokens of a CTA's slice (the last ones may have fewer, or none): a multiple of 128, so that all slices of a row are aligned alike.
__host__ __device__ constexpr uint32_t slice_tokens(uint32_t vocab, uint32_t ctas) { return (vocab + ctas * 128u - 1u) / (ctas * 128u) * 128u; }

struct Penalty {
    float repetition, presence, frequency;
    // The places of tokens that occur hold SEEN, plus the number of occurrences behind the prompt.
    static constexpr uint32_t SEEN = 0x80000000u;
    __device__ float on(float x, uint32_t mark) const {
        if (mark == 0u) return x;
        if (repetition != 1.0f) x = x > 0.0f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
        const uint32_t c = mark & ~SEEN;
        if (c != 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)c)), presence);
        return x;
    }
};

// The row's mask: bits of token v and those behind it.
struct MaskRow {
    const uint32_t* words;      // null: all tokens are allowed
    bool none;
    __device__ bool allows(uint32_t v) const { return !none && (!words || ((words[v >> 5] >> (v & 31u)) & 1u)); }
};

__device__ __forceinline__ MaskRow mask_row(const b200bpe_logits& in, uint32_t row) {
    MaskRow m{nullptr, false};
    if (!in.mask) return m;
    const uint32_t r = in.mask_rows ? in.mask_rows[row] : row;
    m.none = r >= in.n_mask_rows;
    m.words = m.none ? nullptr : in.mask + (uint64_t)r * in.mask_stride;
    return m;
}

// Fills the slice with x.  SCRUB: a NaN becomes -infinity, and -0 becomes 0.  Called by all threads of the cluster; ends with a barrier of the CTA.
template <class T, bool SCRUB>
__device__ void load_slice(const b200bpe_logits& in, uint32_t vocab, const Slice& s) {
    const float lowest = -INFINITY;
    const T* row = static_cast<const T*>(in.logits) + (uint64_t)s.row * in.row_stride + s.lo;
    const MaskRow mask = mask_row(in, s.row);
    Penalty pen{1.0f, 0.0f, 0.0f};
    uint32_t n_seen = 0;
    if (in.history) {
        if (in.repetition) pen.repetition = in.repetition[s.row];
        if (in.presence) pen.presence = in.presence[s.row];
        if (in.frequency) pen.frequency = in.frequency[s.row];
        if (pen.repetition != 1.0f || pen.presence != 0.0f || pen.frequency != 0.0f) n_seen = min(in.lengths[s.row], in.history_cap);
    }
    // Every CTA of the cluster sees the same row, so all of them take the same branches round the cluster's barriers.
    if (n_seen) {
        cg::cluster_group cluster = cg::this_cluster();
        uint32_t* marks = reinterpret_cast<uint32_t*>(s.buf);
        for (uint32_t i = threadIdx.x; i < s.padded; i += SM_THREADS) marks[i] = 0u;
        cluster.sync();
        const uint32_t* h = in.history + (uint64_t)s.row * in.history_stride;
        const uint32_t prompt = in.prompt_lengths ? in.prompt_lengths[s.row] : 0u;
        const uint32_t whole = slice_tokens(vocab, cluster.num_blocks());
        for (uint32_t i = cluster.block_rank() * SM_THREADS + threadIdx.x; i < n_seen; i += cluster.num_blocks() * SM_THREADS) {
            const uint32_t t = h[i];
            if (t >= vocab) continue;
            uint32_t* at = cluster.map_shared_rank(marks, t / whole) + s.lead + t % whole;
            if (i < prompt) atomicOr(at, Penalty::SEEN);
            else atomicAdd(at, 1u);
        }
        cluster.sync();
    }
    constexpr int N = Packed<T>::N;
    for (uint32_t p = threadIdx.x * N; p < s.padded; p += SM_THREADS * N) {
        float v[N];
        if (p >= s.lead && p + N <= s.lead + s.len) {
            Packed<T> q;
            q.v = __ldg(reinterpret_cast<const uint4*>(row + (p - s.lead)));
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = q.get(k);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = p + k >= s.lead && p + k < s.lead + s.len ? as_float(row[p + k - s.lead]) : lowest;
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const bool mine = p + k >= s.lead && p + k < s.lead + s.len;
            if (n_seen && mine) v[k] = pen.on(v[k], reinterpret_cast<const uint32_t*>(s.buf)[p + k]);
            if (mine && (mask.none || mask.words) && !mask.allows(s.lo + p + k - s.lead)) v[k] = lowest;
            if (SCRUB) v[k] = v[k] != v[k] ? lowest : v[k] + 0.0f;
            s.buf[p + k] = v[k];
        }
    }
    __syncthreads();
    if (in.n_bias) {
        // Place i takes all biases of its token, unless an earlier place has that token.
        const uint32_t* list = in.bias_tokens + (uint64_t)s.row * in.bias_stride;
        const float* by = in.biases + (uint64_t)s.row * in.bias_stride;
        for (uint32_t i = threadIdx.x; i < in.n_bias; i += SM_THREADS) {
            const uint32_t t = list[i];
            if (t < s.lo || t - s.lo >= s.len || !mask.allows(t)) continue;
            bool first = true;
            for (uint32_t j = 0; j < i; j++) first &= list[j] != t;
            if (!first) continue;
            float v = __fadd_rn(s.x()[t - s.lo], by[i]);
            for (uint32_t j = i + 1; j < in.n_bias; j++)
                if (list[j] == t) v = __fadd_rn(v, by[j]);
            if (SCRUB) v = v != v ? lowest : v + 0.0f;
            s.x()[t - s.lo] = v;
        }
        __syncthreads();
    }
}

template <class T>
__device__ Slice slice_of(const b200bpe_logits& in, uint32_t vocab, float* buf) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks();
    const uint32_t whole = slice_tokens(vocab, C);
    Slice s;
    s.row = blockIdx.x / C;
    s.lo = min(cluster.block_rank() * whole, vocab);
    s.len = min(whole, vocab - s.lo);
    const uint64_t at = reinterpret_cast<uint64_t>(static_cast<const T*>(in.logits) + (uint64_t)s.row * in.row_stride);
    s.lead = (uint32_t)(at & 15u) / (uint32_t)sizeof(T);
    s.padded = (s.lead + s.len + 7u) & ~7u;
    s.buf = buf;
    return s;
}

// ── adjusted logits ──
template <class T>
__global__ void __launch_bounds__(SM_THREADS)
k_adjust(const __grid_constant__ b200bpe_logits in, uint32_t vocab, T* out, uint64_t out_stride) {
    extern __shared__ __align__(16) float buf[];
    const Slice s = slice_of<T>(in, vocab, buf);
    load_slice<T, false>(in, vocab, s);
    T* to = out + (uint64_t)s.row * out_stride + s.lo;
    for (uint32_t i = threadIdx.x; i < s.len; i += SM_THREADS) rounded(s.x()[i], to + i);
}

// ── the choice ──
// The order of x as unsigned integers.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Best { float x; uint32_t at; };
struct Total { double mass; uint32_t count; };

struct Shared {
    Best best_warp[SM_WARPS], best_cta[SM_MAX_CLUSTER];
    double mass_warp[SM_WARPS], mass_cta[2][SM_MAX_CLUSTER];
    uint32_t count_warp[SM_WARPS], count_cta[2][SM_MAX_CLUSTER];
    uint32_t cut[SM_MAX_CLUSTER], found;
};

struct Weights {
    double m, by;       // the largest x, 1 / temperature
    __device__ double of(float x) const { return (double)x == m ? 1.0 : exp(((double)x - m) * by); }
};

// What of the row is kept: x with a larger key, and those with the key up to place `last` (of the row).
struct Kept {
    uint32_t key, last;
    __device__ bool has(uint32_t k, uint32_t v) const { return k > key || (k == key && v <= last); }
};

// Sums of a value and a count over the cluster, and every CTA's part of them in s.*_cta[par].
__device__ Total cluster_total(Shared& s, int& par, double mass, uint32_t count) {
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        mass += __shfl_xor_sync(0xFFFFFFFFu, mass, o);
        count += __shfl_xor_sync(0xFFFFFFFFu, count, o);
    }
    __syncthreads();
    if (lane == 0) { s.mass_warp[warp] = mass; s.count_warp[warp] = count; }
    __syncthreads();
    par ^= 1;
    if (threadIdx.x < cluster.num_blocks()) {
        double a = 0;
        uint32_t b = 0;
        for (int w = 0; w < SM_WARPS; w++) { a += s.mass_warp[w]; b += s.count_warp[w]; }
        Shared* peer = cluster.map_shared_rank(&s, threadIdx.x);
        peer->mass_cta[par][cluster.block_rank()] = a;
        peer->count_cta[par][cluster.block_rank()] = b;
    }
    cluster.sync();
    Total t{0, 0};
    for (uint32_t c = 0; c < cluster.num_blocks(); c++) { t.mass += s.mass_cta[par][c]; t.count += s.count_cta[par][c]; }
    return t;
}

// First place of the slice at which base plus the running sum of f(place) is above target; if there is none, the last place where f is not 0.
// Called by all threads of one CTA.
template <class F>
__device__ uint32_t find_place(Shared& s, uint32_t padded, double base, double target, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t span = (padded + SM_WARPS * 32 - 1) / (SM_WARPS * 32) * 32;
    const uint32_t lo = min(span * warp, padded), hi = min(lo + span, padded);
    double sum = 0;
    for (uint32_t p = lo + lane; p < hi; p += 32) sum += f(p);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    __syncthreads();
    if (lane == 0) s.mass_warp[warp] = sum;
    if (threadIdx.x == 0) s.found = 0u;
    __syncthreads();
    double at = base;
    int owner = -1, filled = 0;
    for (int w = 0; w < SM_WARPS && owner < 0; w++) {
        if (s.mass_warp[w] > 0) filled = w;
        if (at + s.mass_warp[w] > target) owner = w;
        else at += s.mass_warp[w];
    }
    if (owner < 0) { owner = filled; at -= s.mass_warp[filled]; }
    if (warp == owner) {
        uint32_t place = 0;
        for (uint32_t p0 = lo; p0 < hi; p0 += 32) {
            const double v = p0 + lane < hi ? f(p0 + lane) : 0.0;
            double run = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, run, o);
                if (lane >= o) run += y;
            }
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, v > 0), above = __ballot_sync(0xFFFFFFFFu, v > 0 && at + run > target);
            if (some) place = p0 + 31 - __clz(some);
            if (above) { place = p0 + __ffs(above) - 1; break; }
            at += __shfl_sync(0xFFFFFFFFu, run, 31);
        }
        if (lane == 0) s.found = place;
    }
    __syncthreads();
    return s.found;
}

template <class T>
__global__ void __launch_bounds__(SM_THREADS)
k_sample(const __grid_constant__ b200bpe_logits in, const __grid_constant__ b200bpe_choice how, uint32_t vocab) {
    extern __shared__ __align__(16) float buf[];
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Slice sl = slice_of<T>(in, vocab, buf);
    load_slice<T, true>(in, vocab, sl);
    cluster.barrier_arrive();        // (nobody writes into a CTA that has not begun)

    // the largest x, and the lowest token that has it
    Best best{-INFINITY, 0xFFFFFFFFu};
    for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS)
        if (buf[p] > best.x) best = {buf[p], p - sl.lead + sl.lo};
    for (int turn = 0; turn < 2; turn++) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float x = __shfl_xor_sync(0xFFFFFFFFu, best.x, o);
            const uint32_t at = __shfl_xor_sync(0xFFFFFFFFu, best.at, o);
            if (x > best.x || (x == best.x && at < best.at)) best = {x, at};
        }
        if (turn == 0) {
            if (lane == 0) s.best_warp[warp] = best;
            __syncthreads();
            best = s.best_warp[lane % SM_WARPS];
        }
    }
    cluster.barrier_wait();
    if (threadIdx.x < C) cluster.map_shared_rank(&s, threadIdx.x)->best_cta[rank] = best;
    cluster.sync();
    best = s.best_cta[0];
    for (uint32_t c = 1; c < C; c++)
        if (s.best_cta[c].x > best.x) best = s.best_cta[c];
    if (best.x == -INFINITY) {          // (the whole cluster)
        if (rank == 0 && threadIdx.x == 0) {
            how.tokens_out[sl.row] = B200BPE_NO_TOKEN;
            if (how.logprobs_out) how.logprobs_out[sl.row] = -INFINITY;
        }
        return;
    }

    const float temperature = how.temperature ? how.temperature[sl.row] : 1.0f;
    const bool greedy = !how.uniform || !(temperature >= SM_GREEDY_BELOW);
    const Weights weights{best.x, greedy ? 1.0 : 1.0 / fmin((double)temperature, 3.4e38)};
    int par = 0;
    double mass = 0;
    for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS) mass += weights.of(buf[p]);
    const double all = cluster_total(s, par, mass, 0u).mass;
    if (greedy) {
        if (rank == 0 && threadIdx.x == 0) {
            how.tokens_out[sl.row] = best.at;
            if (how.logprobs_out) how.logprobs_out[sl.row] = (float)-log(all);
        }
        return;
    }

    // The kept tokens: first as a key, `key` and the number of its ties that stay.
    const uint32_t top_k = how.top_k ? how.top_k[sl.row] : 0u;
    const float top_p = how.top_p ? how.top_p[sl.row] : 1.0f, min_p = how.min_p ? how.min_p[sl.row] : 0.0f;
    const uint32_t lowest = key_of(-INFINITY);
    uint32_t key = lowest, ties = 0xFFFFFFFFu;
    auto total_from = [&](uint32_t from) {          // of x with at least the key `from`
        double mass = 0;
        uint32_t count = 0;
        for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS)
            if (key_of(buf[p]) >= from) { mass += weights.of(buf[p]); count++; }
        return cluster_total(s, par, mass, count);
    };
    if (top_k != 0u && top_k < vocab) {
        uint32_t found = 0;
        for (int b = 31; b >= 0; b--)
            if (total_from(found | 1u << b).count >= top_k) found |= 1u << b;
        if (found > lowest) {
            key = found;
            ties = top_k - total_from(key + 1u).count;
        }
    }
    if (top_p < 1.0f) {
        const double above_k = key == lowest ? 0.0 : total_from(key + 1u).mass;
        const float at_key = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
        const double enough = (double)top_p * (key == lowest ? all : above_k + ties * weights.of(at_key));
        if (!(enough > 0.0)) { key = key_of(best.x); ties = 1u; }
        // the largest key from which on there is enough; the ties of the top_k's key count as far as they stay
        uint32_t found = 0;
        for (int b = 31; b >= 0 && enough > 0.0; b--) {
            const uint32_t k = found | 1u << b;
            if (k > key && total_from(k).mass >= enough) found = k;
            else if (k <= key) found = k;
        }
        if (enough > 0.0 && found > lowest) {
            const double above = total_from(found + 1u).mass;
            const double each = weights.of(__uint_as_float(found & 0x80000000u ? found & 0x7FFFFFFFu : ~found));
            const uint32_t most = found == key ? ties : 0xFFFFFFFFu;
            uint32_t n = 1u;
            if (each > 0.0) n = (uint32_t)fmin(fmax(ceil((enough - above) / each), 1.0), 4.0e9);
            if (n > 1u && above + (n - 1u) * each >= enough) n--;
            key = found;
            ties = min(n, most);
        }
    }
    if (min_p > 0.0f) {
        const double least = (double)best.x + log((double)fminf(min_p, 1.0f)) / weights.by;
        const uint32_t from = key_of(__double2float_ru(least) + 0.0f);
        if (from > key) { key = from; ties = 0xFFFFFFFFu; }
    }
    // the last tie that stays
    Kept kept{key, 0xFFFFFFFFu};
    if (key == lowest) kept.last = 0u, kept.key = lowest;
    if (ties != 0xFFFFFFFFu) {
        uint32_t mine = 0;
        for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS) mine += key_of(buf[p]) == key;
        const uint32_t total = cluster_total(s, par, 0.0, mine).count;
        if (ties < total) {
            uint32_t before = 0, owner = 0;
            while (owner + 1 < C && before + s.count_cta[par][owner] < ties) before += s.count_cta[par][owner++];
            if (rank == owner) {
                const uint32_t p = find_place(s, sl.padded, (double)before, (double)ties - 0.5, [&](uint32_t p) { return key_of(buf[p]) == key ? 1.0 : 0.0; });
                if (threadIdx.x < C) cluster.map_shared_rank(&s, threadIdx.x)->cut[0] = p - sl.lead + sl.lo;
            }
            cluster.sync();
            kept.last = s.cut[0];
        }
    }

    auto weight_at = [&](uint32_t p) {
        const float x = buf[p];
        return x > -INFINITY && kept.has(key_of(x), p - sl.lead + sl.lo) ? weights.of(x) : 0.0;
    };
    mass = 0;
    for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS) mass += weight_at(p);
    const double stay = cluster_total(s, par, mass, 0u).mass;
    const float u = how.uniform[sl.row];
    const double target = (u > 0.0f ? fmin((double)u, 1.0) : 0.0) * stay;
    double before = 0;
    uint32_t owner = 0xFFFFFFFFu, filled = 0;
    for (uint32_t c = 0; c < C && owner == 0xFFFFFFFFu; c++) {
        if (s.mass_cta[par][c] > 0) filled = c;
        if (before + s.mass_cta[par][c] > target) owner = c;
        else before += s.mass_cta[par][c];
    }
    if (owner == 0xFFFFFFFFu) { owner = filled; before -= s.mass_cta[par][filled]; }
    if (rank != owner) return;
    const uint32_t p = find_place(s, sl.padded, before, target, weight_at);
    if (threadIdx.x == 0) {
        how.tokens_out[sl.row] = p - sl.lead + sl.lo;
        const double y = (double)buf[p] == weights.m ? 0.0 : ((double)buf[p] - weights.m) * weights.by;
        if (how.logprobs_out) how.logprobs_out[sl.row] = (float)(y - log(all));
    }
}

struct Sampler {
    CtxHold hold;
    Ctx* ctx = nullptr;
    uint32_t vocab = 0;
};

static b200bpe_status check_logits(const b200bpe_logits* in) {
    if (!in || in->struct_size != sizeof(b200bpe_logits)) return refused("logits: struct_size is not that of b200bpe_logits");
    if (in->dtype > B200BPE_BF16) return refused("logits: unknown dtype");
    if (in->n_rows >= 1u << 28) return refused("logits: more than 2^28 - 1 rows");
    if (in->n_rows == 0) return B200BPE_OK;
    const uint64_t size = in->dtype == B200BPE_F32 ? 4 : 2;
    if (!in->logits || reinterpret_cast<uint64_t>(in->logits) % size) return refused("logits: null or misaligned pointer");
    if (in->history) {
        if (!in->lengths) return refused("logits: a history without lengths");
    } else if (in->lengths || in->prompt_lengths || in->repetition || in->presence || in->frequency) {
        return refused("logits: penalties without a history");
    }
    if (in->n_bias) {
        if (in->n_bias > SM_MAX_BIAS) return refused("logits: more than 1,024 biases a row");
        if (!in->bias_tokens || !in->biases) return refused("logits: null list of biases");
    }
    if (in->mask) {
        if (!in->mask_rows && in->n_mask_rows < in->n_rows) return refused("logits: fewer rows of the mask than of logits");
    } else if (in->mask_rows) {
        return refused("logits: mask_rows without a mask");
    }
    return B200BPE_OK;
}

static uint32_t cluster_for(uint32_t vocab) {
    uint32_t c = 1;
    while (c < SM_MAX_CLUSTER && vocab > c * 2048u) c *= 2;
    return c;
}

template <class K, class... A>
static b200bpe_status launch(K kernel, uint32_t rows, uint32_t vocab, cudaStream_t stream, A... args) {
    const uint32_t c = cluster_for(vocab), whole = slice_tokens(vocab, c);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * c);
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = (whole + 16) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = c;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    cfg.attrs = &a;
    cfg.numAttrs = 1;
    B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return B200BPE_OK;
}

// Loads the kernels, so that no call has to, and lets them have a CTA's whole shared memory.
static cudaError_t ready() {
    const void* kernels[] = {(const void*)k_adjust<float>, (const void*)k_adjust<__half>, (const void*)k_adjust<__nv_bfloat16>,
                             (const void*)k_sample<float>, (const void*)k_sample<__half>, (const void*)k_sample<__nv_bfloat16>};
    for (const void* k : kernels) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (SM_MAX_SLICE + 16) * 4);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace b200bpe

struct b200bpe_sampler { b200bpe::Sampler s; };

using namespace b200bpe;

extern "C" {

b200bpe_status b200bpe_sampler_create(b200bpe_ctx* c, uint32_t vocab_size, b200bpe_sampler** out) {
    if (vocab_size == 0 || vocab_size > SM_MAX_VOCAB) return refused("b200bpe_sampler_create: 1 to 458,752 tokens");
    if (!c || !out) return refused("b200bpe_sampler_create: null pointer");
    const OnDevice on(c->c.device);
    B2_CUDA(on.error);
    B2_CUDA(ready());
    b200bpe_sampler* h = new (std::nothrow) b200bpe_sampler();
    if (!h) return B200BPE_ERR_OOM;
    h->s.ctx = &c->c;
    h->s.hold.take(c);
    h->s.vocab = vocab_size;
    *out = h;
    return B200BPE_OK;
}

b200bpe_status b200bpe_sampler_adjust(b200bpe_sampler* h, const b200bpe_logits* in, void* logits_out, uint64_t out_stride, void* stream) {
    if (const b200bpe_status r = check_logits(in)) return r;
    if (!h) return refused("b200bpe_sampler_adjust: null handle");
    const uint32_t vocab = h->s.vocab;
    if (in->n_rows == 0) return B200BPE_OK;
    const uint64_t size = in->dtype == B200BPE_F32 ? 4 : 2;
    if (!logits_out || reinterpret_cast<uint64_t>(logits_out) % size) return refused("b200bpe_sampler_adjust: null or misaligned output");
    if (out_stride < vocab && in->n_rows > 1) return refused("b200bpe_sampler_adjust: rows of the output overlap");
    if (logits_out == in->logits && out_stride != in->row_stride && in->n_rows > 1) return refused("b200bpe_sampler_adjust: in place with another stride");
    const OnDevice on(h->s.ctx->device);
    B2_CUDA(on.error);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (in->dtype) {
        case B200BPE_F32: return launch(k_adjust<float>, in->n_rows, vocab, st, *in, vocab, static_cast<float*>(logits_out), out_stride);
        case B200BPE_F16: return launch(k_adjust<__half>, in->n_rows, vocab, st, *in, vocab, static_cast<__half*>(logits_out), out_stride);
        default: return launch(k_adjust<__nv_bfloat16>, in->n_rows, vocab, st, *in, vocab, static_cast<__nv_bfloat16*>(logits_out), out_stride);
    }
}

b200bpe_status b200bpe_sampler_sample(b200bpe_sampler* h, const b200bpe_logits* in, const b200bpe_choice* how, void* stream) {
    if (const b200bpe_status r = check_logits(in)) return r;
    if (!how || how->struct_size != sizeof(b200bpe_choice)) return refused("choice: struct_size is not that of b200bpe_choice");
    if (!how->uniform && (how->temperature || how->top_k || how->top_p || how->min_p)) return refused("choice: settings of a draw without uniform");
    if (!h) return refused("b200bpe_sampler_sample: null handle");
    const uint32_t vocab = h->s.vocab;
    if (in->n_rows == 0) return B200BPE_OK;
    if (!how->tokens_out) return refused("choice: null tokens_out");
    const OnDevice on(h->s.ctx->device);
    B2_CUDA(on.error);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (in->dtype) {
        case B200BPE_F32: return launch(k_sample<float>, in->n_rows, vocab, st, *in, *how, vocab);
        case B200BPE_F16: return launch(k_sample<__half>, in->n_rows, vocab, st, *in, *how, vocab);
        default: return launch(k_sample<__nv_bfloat16>, in->n_rows, vocab, st, *in, *how, vocab);
    }
}

void b200bpe_sampler_destroy(b200bpe_sampler* h) { delete h; }

}  // extern "C"
