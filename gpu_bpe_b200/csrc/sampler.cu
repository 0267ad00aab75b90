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
#include <type_traits>

#include "ctx.cuh"

namespace cg = cooperative_groups;

namespace b200bpe {

constexpr int SM_THREADS = 256;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr uint32_t SM_MAX_CLUSTER = 16;
constexpr uint32_t SM_MAX_SLICE = 20480;         // 80 KB of 32-bit values
constexpr uint32_t SM_MAX_VOCAB = SM_MAX_SLICE * SM_MAX_CLUSTER;
constexpr uint32_t SM_ADJUST_SLICE = 8192;       // most tokens that a CTA adjusts for a caller
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

// One row's slice in a CTA: tokens [lo, lo + len) of row `row`; token lo + i lies `lead` + i elements into the CTA's buffer, so that what is
// 16-byte aligned in the logits is so in the buffer, too; places in front of and behind the slice, up to `padded`, hold -infinity.
struct Slice {
    uint32_t row, lo, len, lead, padded;
    uint32_t inner;         // how many places, from the slice's first on, have all of their 16 bytes in it
    float* buf;
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

// Sixteen bytes of logits from place p of the slice on, as values; places outside the slice give -infinity.
template <class T>
__device__ __forceinline__ uint4 fetch(const T* row, const Slice& s, uint32_t p) {
    constexpr uint32_t N = Packed<T>::N;
    if (p - s.lead < s.inner) return __ldcs(reinterpret_cast<const uint4*>(row + (p - s.lead)));
    T v[N];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        v[k] = T(-INFINITY);
        if (p + k >= s.lead && p + k < s.lead + s.len) v[k] = row[p + k - s.lead];
    }
    uint4 q;
    memcpy(&q, v, 16);
    return q;
}

// A warp's part of the slice: places [lo, hi).
struct Span {
    uint32_t lo, hi;
    __device__ Span(uint32_t padded, uint32_t warp) {
        const uint32_t each = (padded + SM_WARPS * 256 - 1) / (SM_WARPS * 256) * 256;
        lo = min(each * warp, padded);
        hi = min(lo + each, padded);
    }
};

// Which places of a slice are not plain logits: bit p & 31 of word p >> 5 is place p's.
template <uint32_t MOST>
struct Special {
    uint32_t any[MOST / 32 + 1];         // masked, or in the history
    uint32_t seen[MOST / 32 + 1];        // in the history, or with a bias: the buffer has its x (-infinity if it is masked)
    uint32_t todo[MOST / 32 + 1];        // not yet, it has its marks
};

// Makes `special`, and x of the places in the history and of those with a bias: so these cost a scattered load a token, not a test and a division for
// every lane of the row.  Returns whether there are any special places.  Called by all threads of the CTA; ends with a barrier.
// Each CTA reads the whole history of its row, and counts what is its own: a history is short beside a row, and L2 has it.  What a thread reads first
// does not depend on anything else that is read, so that a row's settings and the first of its history are one wait.  Up to 2,048 tokens stay in
// registers; a longer history is passed over three times.  256 rows of 131,072 in 16 bits, adjusted: 27 us without a history, 46 with one of 1,500 tokens, 50
// with 2,048, 70 with 2,049, 122 with 4,000 and 854 with 32,768: where histories are as long as prompts, they are what bounds the call.
template <uint32_t MOST, class T>
__device__ __forceinline__ bool find_special(const b200bpe_logits& in, uint32_t vocab, const T* row, const Slice& s, const MaskRow& mask, Special<MOST>& special) {
    constexpr int EACH = 8;                          // of a history, a thread keeps at hand
    Penalty pen{1.0f, 0.0f, 0.0f};
    uint32_t n_seen = 0, prompt = 0, t[EACH];
    const uint32_t* h = nullptr;
    if (in.history) {
        h = in.history + (uint64_t)s.row * in.history_stride;
        n_seen = min(in.lengths[s.row], in.history_cap);
        if (in.prompt_lengths) prompt = in.prompt_lengths[s.row];
        if (in.repetition) pen.repetition = in.repetition[s.row];
        if (in.presence) pen.presence = in.presence[s.row];
        if (in.frequency) pen.frequency = in.frequency[s.row];
#pragma unroll
        for (int k = 0; k < EACH; k++) t[k] = threadIdx.x + k * SM_THREADS < in.history_cap ? h[threadIdx.x + k * SM_THREADS] : 0u;
        if (pen.repetition == 1.0f && pen.presence == 0.0f && pen.frequency == 0.0f) n_seen = 0;
    }
    if (n_seen == 0 && in.n_bias == 0 && !mask.words && !mask.none) return false;
    const uint32_t words = (s.padded + 31u) / 32u, mask_words = (vocab + 31u) / 32u;
    for (uint32_t i = threadIdx.x; i < words; i += SM_THREADS) {
        uint32_t allowed = mask.none ? 0u : 0xFFFFFFFFu;
        if (mask.words) {
            const int v = (int)(s.lo + i * 32u) - (int)s.lead, w = v >> 5;
            const uint32_t lo = w >= 0 && w < (int)mask_words ? mask.words[w] : 0u, hi = w + 1 < (int)mask_words ? mask.words[w + 1] : 0u;
            allowed = __funnelshift_r(lo, hi, (uint32_t)v & 31u);
        }
        special.any[i] = ~allowed;
        special.seen[i] = special.todo[i] = 0u;
    }
    uint32_t* marks = reinterpret_cast<uint32_t*>(s.buf);
    // (only the places that will be counted in are emptied)
    if (n_seen <= EACH * SM_THREADS) {
#pragma unroll
        for (int k = 0; k < EACH; k++)
            if (threadIdx.x + k * SM_THREADS < n_seen && t[k] - s.lo < s.len) marks[t[k] - s.lo + s.lead] = 0u;
    } else {
        for (uint32_t i = threadIdx.x; i < n_seen; i += SM_THREADS)
            if (h[i] - s.lo < s.len) marks[h[i] - s.lo + s.lead] = 0u;
    }
    __syncthreads();
    if (n_seen) {
        auto count = [&](uint32_t p, bool in_prompt) {           // whether this is the first at its place
            if ((in_prompt ? atomicOr(&marks[p], Penalty::SEEN) : atomicAdd(&marks[p], 1u)) != 0u) return false;
            atomicOr(&special.any[p >> 5], 1u << (p & 31u));
            atomicOr(&special.seen[p >> 5], 1u << (p & 31u));
            return true;
        };
        auto make = [&](uint32_t v, uint32_t p, T x) { s.buf[p] = mask.allows(v) ? pen.on(as_float(x), marks[p]) : -INFINITY; };
        if (n_seen <= EACH * SM_THREADS) {
            // counted; when all are, the first at a place makes its x
            T x[EACH];
            uint32_t firsts = 0;
#pragma unroll
            for (int k = 0; k < EACH; k++) {
                const uint32_t i = threadIdx.x + k * SM_THREADS, at = t[k] - s.lo;
                if (i < n_seen && at < s.len && count(at + s.lead, i < prompt)) {
                    firsts |= 1u << k;
                    x[k] = row[at];
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < EACH; k++)
                if (firsts >> k & 1u) make(t[k], t[k] - s.lo + s.lead, x[k]);
        } else {
            // the same, but who was the first is not remembered: the first to come back to a place makes its x
            for (uint32_t i = threadIdx.x; i < n_seen; i += SM_THREADS) {
                const uint32_t at = h[i] - s.lo, p = at + s.lead;
                if (at < s.len && count(p, i < prompt)) atomicOr(&special.todo[p >> 5], 1u << (p & 31u));
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n_seen; i += SM_THREADS) {
                const uint32_t v = h[i], at = v - s.lo, p = at + s.lead, bit = 1u << (p & 31u);
                if (at < s.len && (special.todo[p >> 5] & bit) && (atomicAnd(&special.todo[p >> 5], ~bit) & bit)) make(v, p, row[at]);
            }
        }
        __syncthreads();
    }
    if (in.n_bias) {
        // Place i of the list takes all biases of its token, unless an earlier place has that token.
        const uint32_t* list = in.bias_tokens + (uint64_t)s.row * in.bias_stride;
        const float* by = in.biases + (uint64_t)s.row * in.bias_stride;
        for (uint32_t i = threadIdx.x; i < in.n_bias; i += SM_THREADS) {
            const uint32_t v = list[i], at = v - s.lo, p = at + s.lead, bit = 1u << (p & 31u);
            if (at >= s.len || !mask.allows(v)) continue;
            bool first = true;
            for (uint32_t j = 0; j < i; j++) first &= list[j] != v;
            if (!first) continue;
            float x = __fadd_rn(special.seen[p >> 5] & bit ? s.buf[p] : as_float(row[at]), by[i]);
            for (uint32_t j = i + 1; j < in.n_bias; j++)
                if (list[j] == v) x = __fadd_rn(x, by[j]);
            s.buf[p] = x;
            atomicOr(&special.any[p >> 5], bit);
            atomicOr(&special.seen[p >> 5], bit);
        }
        __syncthreads();
    }
    return true;
}

// Calls to(place, N adjusted logits) for the slice.  The first loads are the caller's (`ahead`, of first_loads): they are on their
// way while special places are found, and a call with one row waits for little else.
constexpr uint32_t SM_AHEAD = 4;
template <class T>
__device__ __forceinline__ void first_loads(const T* row, const Slice& s, uint4 (&ahead)[SM_AHEAD]) {
    constexpr uint32_t N = Packed<T>::N;
    const Span span(s.padded, threadIdx.x >> 5);
#pragma unroll
    for (uint32_t j = 0; j < SM_AHEAD; j++) {
        const uint32_t p = span.lo + (threadIdx.x & 31) * N + j * 32 * N;
        if (p < span.hi) ahead[j] = fetch(row, s, p);
    }
}
template <class T, uint32_t MOST, class F>
__device__ __forceinline__ void each_adjusted(const T* row, const Slice& s, uint4 (&ahead)[SM_AHEAD], bool any_special, const Special<MOST>& special,
                                              F to) {
    constexpr uint32_t N = Packed<T>::N, STEP = 32 * N;
    const Span span(s.padded, threadIdx.x >> 5);
    for (uint32_t p0 = span.lo + (threadIdx.x & 31) * N; p0 < span.hi; p0 += SM_AHEAD * STEP) {
#pragma unroll
        for (uint32_t j = 0; j < SM_AHEAD; j++) {
            const uint32_t p = p0 + j * STEP;
            if (p >= span.hi) break;
            const Packed<T> now{ahead[j]};
            if (p + SM_AHEAD * STEP < span.hi) ahead[j] = fetch(row, s, p + SM_AHEAD * STEP);
            float v[N];
#pragma unroll
            for (uint32_t k = 0; k < N; k++) v[k] = now.get(k);
            if (any_special) {
                constexpr uint32_t ALL = (1u << N) - 1u;
                if (const uint32_t any = special.any[p >> 5] >> (p & 31u) & ALL) {
                    const uint32_t seen = special.seen[p >> 5] >> (p & 31u) & ALL;
                    // (what is seen has its x in the buffer; the others are masked)
                    if (seen) {
#pragma unroll
                        for (uint32_t k = 0; k < N; k += 4) {
                            const float4 x = *reinterpret_cast<const float4*>(s.buf + p + k);
                            const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (uint32_t i = 0; i < 4; i++) v[k + i] = any & (1u << (k + i)) ? seen & (1u << (k + i)) ? y[i] : -INFINITY : v[k + i];
                        }
                    } else {
#pragma unroll
                        for (uint32_t k = 0; k < N; k++) v[k] = any & (1u << k) ? -INFINITY : v[k];
                    }
                }
            }
            to(p, v);
        }
    }
}
template <int N>
__device__ __forceinline__ void store(float* at, const float (&v)[N]) {
#pragma unroll
    for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(at + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
}

// Slice `part` of row `row`, of `whole` tokens but for the last ones.
template <class T>
__device__ __forceinline__ Slice slice_of(const b200bpe_logits& in, uint32_t vocab, uint32_t row, uint32_t part, uint32_t whole, float* buf) {
    Slice s;
    s.row = row;
    s.lo = min(part * whole, vocab);
    s.len = min(whole, vocab - s.lo);
    const uint64_t at = reinterpret_cast<uint64_t>(static_cast<const T*>(in.logits) + (uint64_t)row * in.row_stride);
    s.lead = (uint32_t)(at & 15u) / (uint32_t)sizeof(T);
    s.padded = (s.lead + s.len + 7u) & ~7u;
    s.inner = s.len >= Packed<T>::N ? s.len - Packed<T>::N + 1u : 0u;
    s.buf = buf;
    return s;
}

// ── adjusted logits ──
template <class T>
__device__ __forceinline__ void write_out(T* to, const Slice& s, bool alike, uint32_t p, const float (&x)[Packed<T>::N]) {
    constexpr uint32_t N = Packed<T>::N;
    T v[N];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) rounded(x[k], v + k);
    if (alike && p - s.lead < s.inner) {
        uint4 q;
        memcpy(&q, v, 16);
        __stcs(reinterpret_cast<uint4*>(to + (p - s.lead)), q);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < N; k++)
            if (p + k >= s.lead && p + k < s.lead + s.len) to[p + k - s.lead] = v[k];
    }
}

// A CTA for each slice of a row.  Bound by memory: a row is read and written once, and its special places are few.  256 rows of 131,072 in 32 bits
// (268 MB: 41 us at the memory's rate): 42 us; with masks and biases 50; with histories of 1,500 tokens 60, all together 65, of which what is above 42 is the
// wait for a history, its count and the scattered logits of its tokens, while half of a CTA's loads are on their way (4,096 of 8,192 values in 32 bits).
template <class T>
__global__ void __launch_bounds__(SM_THREADS, 4)
k_adjust(const __grid_constant__ b200bpe_logits in, uint32_t vocab, uint32_t whole, T* out, uint64_t out_stride) {
    extern __shared__ __align__(16) float buf[];
    __shared__ Special<SM_ADJUST_SLICE + 8> special;
    const uint32_t parts = (vocab + whole - 1u) / whole;
    const Slice s = slice_of<T>(in, vocab, blockIdx.x / parts, blockIdx.x % parts, whole, buf);
    const T* row = static_cast<const T*>(in.logits) + (uint64_t)s.row * in.row_stride + s.lo;
    uint4 ahead[SM_AHEAD];
    first_loads(row, s, ahead);
    const MaskRow mask = mask_row(in, s.row);
    const bool any_special = find_special(in, vocab, row, s, mask, special);
    T* to = out + (uint64_t)s.row * out_stride + s.lo;
    // Places that lie on 16 bytes in the logits do so in the output if its rows are aligned like the logits' (in place, and with equal strides).
    const bool alike = (reinterpret_cast<uint64_t>(to) & 15u) == s.lead * sizeof(T);
    each_adjusted(row, s, ahead, any_special, special, [&](uint32_t p, float (&v)[Packed<T>::N]) { write_out<T>(to, s, alike, p, v); });
}

// ── the choice ──
// A thread's largest x, the place of the first vector that has it, and the sum of 2^(x c - n) over its x, n being a whole number next to the largest
// x c: sums with different n are brought to one another by powers of two, without rounding.  Weights have 32 bits here, since 64 for every x of the row would
// be bound by arithmetic (the first version: 398 us for 128 rows of 262,144, 117 now).  A logprob is made of their sum: it is off by at most 2^-22 + 3 * 2^-24 ln(vocabulary)
// before it is rounded to 32 bits.  What they decide is looked at again where it is near (below).
struct Stats {
    // 2^25: up to there the whole number is within 1 of x c (half of a step between floats; further out a weight of the largest x itself could be 2^256).
    static constexpr float FAR = 33554432.0f;
    float c, m = -INFINITY, n = -FAR;
    uint32_t at = 0;
    double sum = 0;
    static __device__ __forceinline__ float two_to(float y) {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(y));
        return w;
    }
    // 2^e for a whole number e of at most 0.
    static __device__ __forceinline__ double power(float e) { return e < -1000.0f ? 0.0 : __hiloint2double((1023 + (int)e) << 20, 0); }
    __device__ __forceinline__ float base(float largest) const { return fminf(fmaxf(rintf(largest * c), -FAR), FAR); }
    // N x of place p on; a NaN among them becomes -infinity, in the buffer too.
    template <int N>
    __device__ __forceinline__ void add(float (&v)[N], uint32_t p, float* buf) {
        float top = v[0];
#pragma unroll
        for (int k = 1; k < N; k++) top = fmaxf(top, v[k]);
        if (top > m) {
            m = top;
            at = p;
            const float to = base(top);
            if (to > n) {
                sum *= power(n - to);
                n = to;
            }
        }
        float w = weights(v);
        if (w != w) {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = fmaxf(v[k], -INFINITY);       // (of a NaN and a number the number)
            store(buf + p, v);
            w = weights(v);
        }
        sum += (double)w;
    }
    template <int N>
    __device__ __forceinline__ float weights(const float (&v)[N]) const {
        float w[N];
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = two_to(fmaf(v[k], c, -n));
#pragma unroll
        for (int o = 1; o < N; o *= 2)
#pragma unroll
            for (int k = 0; k + o < N; k += 2 * o) w[k] += w[k + o];
        return w[0];
    }
};
// The same of a slice that is there.
__device__ __forceinline__ void slice_stats(const Slice& s, Stats& stats) {
    const Span span(s.padded, threadIdx.x >> 5);
    for (uint32_t p = span.lo + (threadIdx.x & 31) * 4; p < span.hi; p += 128) {
        const float4 x = *reinterpret_cast<const float4*>(s.buf + p);
        float v[4] = {x.x, x.y, x.z, x.w};
        stats.add(v, p, s.buf);
    }
}

// The order of x as unsigned integers, and back.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);        // (-0 is 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

constexpr uint32_t LOWEST_KEY = 0x007FFFFFu;     // of -infinity
constexpr uint32_t SM_BINS = 2048;
constexpr uint32_t SM_CANDIDATES = 1024, SM_EACH = SM_CANDIDATES / SM_THREADS;
constexpr uint32_t SM_QUICK_K = 512;             // top_k up to which a row's candidates are looked for without bins
constexpr uint32_t SM_QUICK_P0 = 64, SM_QUICK_P1 = 256;    // where so few weigh what top_p keeps, they are looked for the same way

// Which token is chosen depends on sums of weights: on the first running sum that is above a border.  Sums are made of weights in 32 bits,
// w = 2^(x c - n) with c = log2 e / temperature, and added in 64 bits.  Against the exact weights, up to a factor that all have in common, the
// exponent is off by the roundings of log2 e, c and the product's difference, together 2.5 * 2^-24 (m - x) c + 2^-24, the exponential by 2^-22 of itself, and up to
// eight weights are added in 32 bits first, three roundings.  The factor that brings such sums to the unit of exact ones is an exp2f, off by 2 of its last places,
// 2^-22, and the rounding of its argument.  So a sum is off by at most
//     E = sum w * 2^-24 * (13 + 2.5 ln 2 (m - x) c).
// The mean of (m - x) c under some tokens' weights is their entropy less log2 r, r = sum w / the row's largest w, so at most log2(tokens / r).
//
// A running sum F is compared with a border that is a share u of the whole S = F + R.
//   Where S was made of the same sums as F, what F is off is also in S: F - u S is off by (1 - u) times what F is off, less u times what R is.  At the
//   border F is u S, so that this is at most (1 - u) E(u S) + u E((1 - u) S).
//   Where a part G of F was added in another order than in S (the places of one warp's part, in find_place), its errors are not the same: they are at
//   most E(G) and u E(G) where (1 - u) E(G) was counted, so 2 u E(G) more, and G's own roundings.
//   Where F is exact, u E(S); where the border is, E(u S).
// Sums in 64 bits are off by some steps of 2^-53 besides, and weights below 2^-126 count for nothing in 32 bits: 2^-44 S has room for both.  Where a
// running sum that decides lies within all that of the border, the row's sums are made again of weights in 64 bits.
// 2^(i / 64), to the nearest.
__device__ const double TWO_TO_64THS[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0, 0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0,
    0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0, 0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0, 0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0,
    0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0, 0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0, 0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0,
    0x1.6247eb03a5585p+0, 0x1.6623882552225p+0, 0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0, 0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0,
    0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0, 0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0, 0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0,
    0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0, 0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

struct Weights {
    float m, c, n;              // the largest x, log2 e / temperature, the exponent that all quick weights are relative to
    double steps;               // 64 log2 e / temperature
    const double* table;        // 2^(i / 64)
    __device__ __forceinline__ float quick(float x) const { return Stats::two_to(fmaf(x, c, -n)); }
    // e^((x - m) / temperature) = 2^(t / 64) with t = k + r, |r| <= 1/2: a table's value, the first five terms of the series for r (the sixth is below
    // 4e-14), and a power of two; 11 operations in 64 bits.  Of m itself it is 1.
    __device__ __forceinline__ double exact(float x) const {
        constexpr double MAGIC = 6755399441055744.0, L = 0.693147180559945309 / 64;
        const double t = ((double)x - (double)m) * steps, u = t + MAGIC, r = t - (u - MAGIC);
        const int k = __double2loint(u);
        const double p = table[k & 63] * fma(r, fma(r, fma(r, fma(r, L * L * L * L / 24, L * L * L / 6), L * L / 2), L), 1.0);
        return fmaf(x, c, -n) > -1000.0f ? __hiloint2double(__double2hiint(p) + (k >> 6) * 1048576, __double2loint(p)) : 0.0;
    }
    __device__ __forceinline__ double power_of_largest() const { return (double)n - (double)m * (double)c; }
    __device__ __forceinline__ double to_largest() const { return (double)exp2f((float)power_of_largest()); }        // quick's unit in exact's
};

// E of quick weights whose sum is r, in parts of 2^-24.
__device__ __forceinline__ float off_by(uint32_t vocab, float r) { return r > 0.0f ? r * (13.0f + 1.75f * (1.0f + log2f((float)vocab / r))) : 0.0f; }
constexpr double SM_OFF = 1.01 / 16777216.0;         // (what `off_by` is off itself, and the difference between F and u S)
// How far a running sum may be off from its border, a share of `sum`.
enum class Border { OF_ITS_SUM, EXACT, OF_EXACT_SUMS };        // quick sums, the one made of the other; quick sums, an exact border; exact sums, a share of a quick one
__device__ __forceinline__ double how_near(uint32_t vocab, double sum, double share, Border border) {
    double off;
    if (border == Border::OF_ITS_SUM) off = (1.0 - share) * off_by(vocab, (float)(share * sum)) + share * off_by(vocab, (float)((1.0 - share) * sum));
    else if (border == Border::EXACT) off = off_by(vocab, (float)(share * sum));
    else off = share * off_by(vocab, (float)sum);
    return off * SM_OFF + sum * 0x1p-44;
}

// What of the row is kept: x with a larger key, and those with the key in front of token `end`.
struct Kept {
    uint32_t key, end;
    __device__ __forceinline__ bool has(float x, uint32_t v) const {
        const float at = value_of(key);
        return x > at || (x == at && v < end);
    }
};

// Where a draw falls: in which CTA's slice, what is in front of that, the sum to be passed, and what is near that.
struct Draw { uint32_t owner; double base, target, near; };      // (owner 0xFFFFFFFF: not known)
struct Best { float m, n; uint32_t at, pad; double sum; float cut[4]; };       // a CTA's part of what the first exchange brings

// What a row's first exchange comes to: the sum of all weights in two units and the second in the first, the weights' exponent, and see there.
struct Row { double quick_all, all, unit, steps; float from; bool quick; };

struct Shared {
    Best best[SM_MAX_CLUSTER];
    double part_warp[2][SM_WARPS], part_cta[2][2][SM_MAX_CLUSTER];      // (the second index: one exchange and the next)
    double scan_warp[SM_WARPS], warp_mass[SM_WARPS], step_mass[32], table[64];
    float m_warp[SM_WARPS], n_warp[SM_WARPS], cut[4];
    uint32_t border[2], again, candidates, quick_candidates, flag, place, at, cut_at[2];
    Kept kept;
    Draw draw;
    Row row;
    union {
        uint32_t bins[SM_BINS];
        unsigned long long __align__(16) list[SM_CANDIDATES];      // candidates: key << 32 | ~token
        uint32_t keys[SM_THREADS];
        Special<SM_MAX_SLICE + 8> special;           // until the slice is there
    };
};

// Over a warp, or over each N lanes of it.
template <int N = 32, class V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
template <int N = 32, class V>
__device__ __forceinline__ V warp_run(V v, int lane) {        // over the lanes up to this one, of the first N
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const V y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// One CTA's view of its cluster.
struct Team {
    Shared& s;
    int par = 0;
    uint32_t C, rank;
    int lane, warp;

    __device__ explicit Team(Shared& sh) : s(sh) {
        cg::cluster_group cluster = cg::this_cluster();
        C = cluster.num_blocks();
        rank = cluster.block_rank();
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
    }
    __device__ Shared* peer(uint32_t r) const { return cg::this_cluster().map_shared_rank(&s, r); }
    __device__ void sync() const { cg::this_cluster().sync(); }

    // Sums of two values over the cluster; every CTA's part of them stays in part(i, cta) until the exchange after the next, every warp's part of
    // the first in s.warp_mass until the next.
    __device__ void total(double& a, double& b) {
        a = warp_sum(a);
        b = warp_sum(b);
        __syncthreads();
        if (lane == 0) { s.part_warp[0][warp] = s.warp_mass[warp] = a; s.part_warp[1][warp] = b; }
        __syncthreads();
        par ^= 1;
        if (warp == 0) {
            a = warp_sum<SM_WARPS>(s.part_warp[0][lane % SM_WARPS]);
            b = warp_sum<SM_WARPS>(s.part_warp[1][lane % SM_WARPS]);
            if (lane < C) {
                Shared* p = peer(lane);
                p->part_cta[0][par][rank] = a;
                p->part_cta[1][par][rank] = b;
            }
        }
        sync();
        a = of_ctas(part(0, lane % SM_MAX_CLUSTER));
        b = of_ctas(part(1, lane % SM_MAX_CLUSTER));
    }
    // Sum of what lanes have for CTA `lane % SM_MAX_CLUSTER`.
    __device__ double of_ctas(double v) const { return warp_sum<SM_MAX_CLUSTER>(lane % SM_MAX_CLUSTER < C ? v : 0.0); }
    __device__ double part(int i, uint32_t cta) const { return s.part_cta[i][par][cta]; }

    // Sum of v over the threads before this one; *all: over all.
    template <class V>
    __device__ V before(V v, V* all) {
        V* part = reinterpret_cast<V*>(s.scan_warp);
        const V run = warp_run(v, lane);
        __syncthreads();
        if (lane == 31) part[warp] = run;
        __syncthreads();
        const V sums = warp_run<SM_WARPS>(part[lane % SM_WARPS], lane % SM_WARPS);
        *all = __shfl_sync(0xFFFFFFFFu, sums, SM_WARPS - 1);
        const V base = __shfl_sync(0xFFFFFFFFu, sums, warp - 1);
        return (warp ? base : V(0)) + run - v;
    }
    // The first of N values (a lane's is v; 0 behind the first N lanes) at which the running sum is above target, and the sum in front of it; if there is none, the last above 0.
    template <int N = 32>
    __device__ int first_above(double v, double from, double target, double* base) const {
        const double run = from + warp_run<N>(v, lane);
        const uint32_t above = __ballot_sync(0xFFFFFFFFu, v > 0 && run > target), some = __ballot_sync(0xFFFFFFFFu, v > 0);
        const int i = above ? __ffs(above) - 1 : some ? 31 - __clz(some) : 0;
        *base = __shfl_sync(0xFFFFFFFFu, run - v, i);
        return i;
    }
};

// f(place, four x) for all of a warp's part, with all lanes (some of them behind the end, with -infinity).
template <class F>
__device__ __forceinline__ void each_four(const Slice& sl, int warp, F f) {
    const Span span(sl.padded, warp);
    for (uint32_t p0 = span.lo; p0 < span.hi; p0 += 128) {
        const uint32_t p = p0 + (threadIdx.x & 31) * 4;
        f(p, p < span.hi ? *reinterpret_cast<const float4*>(sl.buf + p) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY));
    }
}

// Sum of the weights of a row's kept places, as parts of the largest one: of weights in 64 bits or in 32.
template <bool EXACT>
__device__ __forceinline__ double kept_mass(const Slice& sl, int warp, const Weights& w, const Kept& kept) {
    double sum = 0;
    const int shift = (int)sl.lo - (int)sl.lead;
    each_four(sl, warp, [&](uint32_t p, const float4& x) {
        const uint32_t v = p + shift;
        const bool a = kept.has(x.x, v), b = kept.has(x.y, v + 1), c = kept.has(x.z, v + 2), d = kept.has(x.w, v + 3);
        if (a | b | c | d) {
            if (EXACT) sum += ((a ? w.exact(x.x) : 0.0) + (b ? w.exact(x.y) : 0.0)) + ((c ? w.exact(x.z) : 0.0) + (d ? w.exact(x.w) : 0.0));
            else sum += (double)(((a ? w.quick(x.x) : 0.0f) + (b ? w.quick(x.y) : 0.0f)) + ((c ? w.quick(x.z) : 0.0f) + (d ? w.quick(x.w) : 0.0f)));
        }
    });
    return EXACT ? sum : sum * w.to_largest();
}

// The first place of the slice at which base plus the running sum of f(place, x) is above target; if there is none, the last with f above 0.  Every
// warp's sum of f is in s.warp_mass.  *near: whether a sum that decided was within `margin` of target (or the sums of parts and of places round apart);
// for quick weights, whose target is a `share` of all of them, and whose sums up to a warp's part are `margin` off, what that part adds comes to it.
// Called by all threads of one CTA: first the part of a warp, then a step of 128 places of it, then a place.  f gives V.
template <class V, class F>
__device__ uint32_t find_place(Team& t, const Slice& sl, double base, double target, double margin, double share, uint32_t vocab, bool* near, F f) {
    static_assert(SM_MAX_SLICE + 8 <= SM_WARPS * 32 * 128, "more than 32 steps in a warp's part");
    constexpr int EACH = 32 / SM_WARPS;
    Shared& s = t.s;
    const Span span(sl.padded, t.first_above<SM_WARPS>(t.lane < SM_WARPS ? s.warp_mass[t.lane] : 0.0, base, target, &base));
    const double part = base;        // what is in front of the warp's part
    // A warp has EACH of the steps, a lane four neighbouring places of each.
    V v[EACH][4], run[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t at = span.lo + (i * SM_WARPS + t.warp) * 128, p = at + t.lane * 4;
        run[i] = v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0;
        if (at < span.hi) {
            const float4 x = p < span.hi ? *reinterpret_cast<const float4*>(sl.buf + p) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            v[i][0] = f(p, x.x);
            v[i][1] = f(p + 1, x.y);
            v[i][2] = f(p + 2, x.z);
            v[i][3] = f(p + 3, x.w);
            run[i] = warp_run((v[i][0] + v[i][1]) + (v[i][2] + v[i][3]), t.lane);
        }
        if (t.lane == 31) s.step_mass[i * SM_WARPS + t.warp] = (double)run[i];
    }
    if (threadIdx.x == 0) { s.place = 0u; s.flag = 1u; }
    __syncthreads();
    const double mass = s.step_mass[t.lane];
    const int step = t.first_above(mass, base, target, &base);
    if (step % SM_WARPS == t.warp) {
        const double whole = __shfl_sync(0xFFFFFFFFu, mass, step);
        if (sizeof(V) == 4) {
            // (the roundings of the part's own sums: of the unit, a product, two sums of four, five steps of a scan, a difference)
            const double front = base + whole - part;
            margin += (10.0 * front + 2.0 * share * off_by(vocab, (float)front)) * SM_OFF;
        }
        uint32_t hit = 0, last = 0;
        bool edge = false;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            if (i * SM_WARPS + t.warp != step) continue;
            const uint32_t p = span.lo + step * 128 + t.lane * 4;
            double sum = base + (double)(run[i] - ((v[i][0] + v[i][1]) + (v[i][2] + v[i][3])));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const double next = sum + (double)v[i][k];
                if (v[i][k] > 0) {
                    last = p + k + 1;
                    if (hit == 0) {
                        edge = fabs(next - target) <= margin || fabs(sum - target) <= margin;
                        if (next > target) hit = p + k + 1;
                    }
                }
                sum = next;
            }
        }
        const uint32_t above = __ballot_sync(0xFFFFFFFFu, hit != 0), some = __ballot_sync(0xFFFFFFFFu, last != 0);
        if (t.lane == (above ? __ffs(above) - 1 : some ? 31 - __clz(some) : 0)) {
            s.place = (above ? hit : some ? last : 1u) - 1u;
            s.flag = edge || !above;
        }
    }
    __syncthreads();
    *near = s.flag != 0;
    return s.place;
}

// Descending order of E * SM_THREADS numbers, E to a thread (its neighbours in the order): a bitonic network, whose steps run within a thread, by
// shuffles, and between warps through `list`, which has them in the end.
template <int E>
__device__ __forceinline__ void sort_threads(unsigned long long* list) {
    constexpr uint32_t N = E * SM_THREADS;
    const uint32_t i0 = threadIdx.x * E;
    unsigned long long a[E];
#pragma unroll
    for (int k = 0; k < E; k++) a[k] = list[i0 + k];
    auto keep = [](unsigned long long mine, unsigned long long other, bool larger) { return (mine > other) == larger ? mine : other; };
#pragma unroll 1
    for (uint32_t size = 2; size <= N; size <<= 1) {
#pragma unroll 1
        for (uint32_t step = size >> 1; step >= 32 * E; step >>= 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < E; k++) list[i0 + k] = a[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < E; k++) a[k] = keep(a[k], list[(i0 + k) ^ step], ((i0 & step) == 0) == ((i0 & size) == 0));
        }
#pragma unroll 1
        for (uint32_t step = min(size >> 1, 16u * E); step >= E; step >>= 1)
#pragma unroll
            for (int k = 0; k < E; k++) a[k] = keep(a[k], __shfl_xor_sync(0xFFFFFFFFu, a[k], step / E), ((i0 & step) == 0) == ((i0 & size) == 0));
#pragma unroll
        for (int step = E / 2; step >= 1; step >>= 1)
            if (size > (uint32_t)step)
#pragma unroll
                for (int k = 0; k < E; k++)
                    if ((k & step) == 0) {
                        const bool down = ((i0 + k) & size) == 0;
                        const unsigned long long x = a[k], y = a[k + step];
                        if ((x < y) == down) { a[k] = y; a[k + step] = x; }
                    }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < E; k++) list[i0 + k] = a[k];
    __syncthreads();
}
// The same of at most SM_THREADS / 2 numbers, all unlike but for zeros behind them: each is put where as many as are larger lie in front.  (For 128 that is
// a third of the instructions of a network; for 256 it would be more.)
__device__ __forceinline__ void sort_few(unsigned long long* list, uint32_t n) {
    uint32_t size = 32;
    while (size < n) size *= 2;
    const uint32_t shares = SM_THREADS / size, e = threadIdx.x / shares, part = threadIdx.x % shares;
    const unsigned long long mine = list[e];
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t j = part * 2; j < size; j += shares * 2) {
        const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(list + j);
        rank += (other.x > mine) + (other.y > mine);
    }
    for (uint32_t o = 1; o < shares; o *= 2) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, o);
    __syncthreads();
    if (part == 0 && mine) list[rank] = mine;
    const uint32_t full = __syncthreads_count(part == 0 && mine != 0ull);
    if (part == 0 && e >= full) list[e] = 0ull;
    __syncthreads();
}
// Of n numbers (zeros behind them are added); returns how many lie at a thread: thread i has those from i * that on.
__device__ __forceinline__ uint32_t sort_down(unsigned long long* list, uint32_t n) {
    const uint32_t size = n <= SM_THREADS ? SM_THREADS : n <= 2 * SM_THREADS ? 2 * SM_THREADS : 4 * SM_THREADS;
    static_assert(SM_CANDIDATES == 4 * SM_THREADS, "the list's room");
    for (uint32_t i = n + threadIdx.x; i < size; i += SM_THREADS) list[i] = 0ull;
    __syncthreads();
    if (n <= SM_THREADS / 2) sort_few(list, n);
    else if (size == SM_THREADS) sort_threads<1>(list);
    else if (size == 2 * SM_THREADS) sort_threads<2>(list);
    else sort_threads<4>(list);
    return size / SM_THREADS;
}

// Bins of x, from the largest downwards: SM_BINS of them over `range`, each round its middle; the last one takes the rest.
struct Bins {
    float m, scale;
    __device__ Bins(float largest, double range) : m(largest), scale((float)(SM_BINS / fmin(range, 3.4e38))) {}
    static constexpr float MAGIC = 8388608.0f;       // added to 0 to 2^22, it leaves the nearest whole number in the lowest bits
    __device__ __forceinline__ float at(float x) const { return (m - x) * scale; }
    // Puts four x into their bins, as far as they lie in front of `end`: as 1, or as its weight in parts of 2^16 of that of its bin's middle, bins being 1/64
    // wide: e^-r by its first terms.
    template <bool MASS>
    __device__ __forceinline__ void put(uint32_t* bins, const float4& x, float end) const {
        const float v[4] = {x.x, x.y, x.z, x.w};
        float a[4], b[4];
        uint32_t n[4];
#pragma unroll
        for (int k = 0; k < 4; k++) a[k] = at(v[k]);
        if (fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) >= end) return;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            b[k] = fminf(a[k], end) + MAGIC;
            const float r = a[k] - (b[k] - MAGIC);
            n[k] = MASS ? __float_as_uint(fmaf(fmaf(r, 8.0f, -1024.0f), r, MAGIC + 65536.0f)) & 0x7FFFFFu : 1u;
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (a[k] < end) atomicAdd(bins + (__float_as_uint(b[k]) & 0x7FFFFFu), n[k]);
    }
    // A value that is above all x of the bins from `bin` on, or, `under`, below all x of the bins up to it: next to the bin's end, by more than `at` is off.
    __device__ float end_of(uint32_t bin, bool under) const {
        if (under && bin >= SM_BINS - 1) return -3.402823466e38f;
        if (!under && bin == 0) return INFINITY;
        const float x = m - ((float)bin + (under ? 0.5f : -0.5f)) / scale, off = (fabsf(m) + fabsf(x)) * 0x1p-21f;
        return under ? fmaxf(x - off, -3.402823466e38f) : x + off;
    }
};

// Appends a lane's values whose bits are set in `in`, of tokens from v0 on, to a list, as far as there is room.
__device__ __forceinline__ void gather(const Team& t, uint32_t* counter, unsigned long long* list, const float (&v)[4], uint32_t in, uint32_t v0) {
    if (!__any_sync(0xFFFFFFFFu, in != 0u)) return;
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t b = __ballot_sync(0xFFFFFFFFu, in >> k & 1u);
        before += __popc(b & ((1u << t.lane) - 1u));
        all += __popc(b);
    }
    uint32_t base = 0;
    if (t.lane == 0) base = atomicAdd(counter, all);
    base = __shfl_sync(0xFFFFFFFFu, base, 0) + before;
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (in >> k & 1u) {
            if (base < SM_CANDIDATES) list[base] = (unsigned long long)key_of(v[k]) << 32 | (uint32_t)~(v0 + k);
            base++;
        }
}
// The candidates of a CTA other than the first, gathered in its own list, go to the first one's: a CTA waits once for the way there and back.  The
// cluster's next barrier makes them seen.
__device__ __forceinline__ void hand_over(Team& t, uint32_t Shared::*counter) {
    Shared& s = t.s;
    if (t.rank == 0) return;
    __syncthreads();
    const uint32_t n = s.*counter;
    if (n == 0) return;
    Shared* lead = t.peer(0);
    if (threadIdx.x == 0) s.place = atomicAdd(&(lead->*counter), n);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(n, SM_CANDIDATES) && s.place + i < SM_CANDIDATES; i += SM_THREADS) lead->list[s.place + i] = s.list[i];
}

struct Settings {
    bool greedy;
    double warm;            // temperature
    uint32_t top_k;         // 0: all
    float top_p, min_p, uniform;
    __device__ Settings(const b200bpe_choice& how, uint32_t row, uint32_t vocab) {
        const float t = how.temperature ? how.temperature[row] : 1.0f;
        greedy = !how.uniform || !(t >= SM_GREEDY_BELOW);
        warm = greedy ? 1.0 : fmin((double)t, 3.4e38);
        top_k = greedy || !how.top_k ? 0u : how.top_k[row];
        if (top_k >= vocab) top_k = 0u;
        const float p = greedy || !how.top_p ? 1.0f : how.top_p[row], m = greedy || !how.min_p ? 0.0f : how.min_p[row];
        top_p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;
        min_p = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
        const float u = greedy ? 0.0f : how.uniform[row];
        uniform = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    }
    // The smallest x that min_p keeps.
    __device__ uint32_t min_key(float m) const {
        return min_p > 0.0f ? key_of(__double2float_ru((double)m + log((double)min_p) * warm)) : LOWEST_KEY;
    }
};

// The part of the row's order at which a running sum, from the largest x on, reaches `target`: of weights (MASS) or of tokens.
// s.bins are filled in all CTAs (weights: in parts of 2^16 of that of the bin's middle), and a barrier of the cluster is behind that.
// Returns what is kept up to and with the token that reaches it, the same in every CTA.  With `set` (nothing was taken away before) `found` is where the
// draw falls, if that is known by the way; the caller has its owner at 0xFFFFFFFF.
template <bool MASS>
__device__ Kept border(Team& t, const Slice& sl, const Weights& w, const Bins& bins, double target, double share, double margin, const Settings* set,
                       uint32_t vocab, Draw& found) {
    const uint32_t whole = slice_tokens(vocab, t.C);
    Shared& s = t.s;
    const int shift = (int)sl.lo - (int)sl.lead;
    // every CTA adds up a part of the bins for all
    const uint32_t mine = SM_BINS / t.C, per = max(mine / SM_THREADS, 1u), first = t.rank * mine + threadIdx.x * per;
    const bool busy = threadIdx.x * per < mine;
    float here[SM_BINS / SM_THREADS], sum = 0;          // (the borders of bins are known to 2^-15 only)
#pragma unroll
    for (uint32_t k = 0; k < SM_BINS / SM_THREADS; k++) {
        here[k] = 0;
        if (busy && k < per) {
            unsigned long long n = 0;
#pragma unroll 8
            for (uint32_t c = 0; c < t.C; c++) n += t.peer(c)->bins[first + k];
            here[k] = MASS ? (float)n * (__expf(-(float)(first + k) / 64) / 65536.0f) : (float)n;
        }
        sum += here[k];
    }
    if (threadIdx.x < 2) s.border[threadIdx.x] = SM_BINS - 1;
    if (threadIdx.x == 0) s.candidates = 0u;
    float all, before = t.before(sum, &all);
    // (t.total's barriers: the parts of a bin may be read until here)
    double a = threadIdx.x == 0 ? (double)all : 0.0, none = 0;
    t.total(a, none);
    double at = (double)before + warp_sum(t.lane < t.rank ? t.part(0, t.lane) : 0.0);
    const double slack = MASS ? 1.0 / 32768 : 0.0;          // 2^-17 a weight, 2 * 2^-24 * 2048 / 64 its place, the bins' weights, and what the target is off
#pragma unroll
    for (uint32_t k = 0; k < SM_BINS / SM_THREADS; k++) {
        if (k >= per || !busy) break;
        const double next = at + (double)here[k];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const double by = e == 0 ? 1.0 + slack : 1.0 - slack;
            if (at * by < target && next * by >= target)
                for (uint32_t c = 0; c < t.C; c++) t.peer(c)->border[e] = first + k;
        }
        at = next;
    }
    t.sync();
    // sums of what is above the border's bins; what lies in them goes to the first CTA
    const float high = bins.end_of(s.border[0], false), low = bins.end_of(max(s.border[0], s.border[1]), true);
    // A border that is a share of all: `rest`, what lies below the border's bins, makes the whole of the same sums as what lies above.  (9 us of 225 for a
    // top_p of 0.9 and 256 rows of 131,072; against the whole as it was loaded, a border would be four times as far from certain.)
    const double unit = MASS ? w.to_largest() : 1.0;
    double above = 0, rest = 0;
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        const float v[4] = {x.x, x.y, x.z, x.w};
        uint32_t in = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) in |= (uint32_t)(v[k] <= high && v[k] >= low) << k;
        if (x.x > high || x.y > high || x.z > high || x.w > high) {
            float e[4];
#pragma unroll
            for (int k = 0; k < 4; k++) e[k] = v[k] > high ? MASS ? w.quick(v[k]) : 1.0f : 0.0f;
            above += (double)((e[0] + e[1]) + (e[2] + e[3]));
        }
        if (MASS && share >= 0) {
            float e[4];
#pragma unroll
            for (int k = 0; k < 4; k++) e[k] = v[k] < low ? w.quick(v[k]) : 0.0f;
            rest += (double)((e[0] + e[1]) + (e[2] + e[3]));
        }
        gather(t, &s.candidates, s.list, v, in, p + shift);      // (the list lies where the bins were)
    });
    hand_over(t, &Shared::candidates);
    above *= unit;
    rest *= unit;
    t.total(above, rest);
    const uint32_t n = t.peer(0)->candidates;
    if (n <= SM_CANDIDATES) {
        uint32_t each = 1;
        for (int turn = 0; turn < 2; turn++) {
            // turn 1: again with the sums in 64 bits
            if (t.rank == 0) {
                if (turn == 0) each = sort_down(s.list, n);
                // neighbours to a thread; flag 1: a sum was near, 2: the bins were misjudged
                double v[SM_EACH], mine = 0;
#pragma unroll
                for (uint32_t k = 0; k < SM_EACH; k++) {
                    const uint32_t i = threadIdx.x * each + k;
                    v[k] = k < each && i < n ? (MASS ? w.exact(value_of((uint32_t)(s.list[i] >> 32))) : 1.0) : 0.0;
                    mine += v[k];
                }
                if (threadIdx.x == 0) { s.flag = 0u; s.place = n ? n - 1 : 0u; }
                double of_list, sum = above + t.before(mine, &of_list);
                if (MASS && share >= 0 && turn == 0) target = share * (above + of_list + rest);
#pragma unroll
                for (uint32_t k = 0; k < SM_EACH; k++) {
                    const double next = sum + v[k];
                    const uint32_t i = k < each ? threadIdx.x * each + k : n;
                    if (i < n && sum < target && next >= target) s.place = i;
                    if (MASS && turn == 0 && i < n && (fabs(sum - target) <= margin || fabs(next - target) <= margin)) s.flag = 1u;
                    sum = next;
                }
                const double near = turn == 0 ? margin : 0.0;
                if (MASS && threadIdx.x == 0 && above >= target - near) s.flag = 1u + turn;
                if (MASS && threadIdx.x == SM_THREADS - 1 && sum < target + near) s.flag = 1u + turn;
                __syncthreads();
                const unsigned long long e = s.list[s.place];
                const Kept kept = n ? Kept{(uint32_t)(e >> 32), ~(uint32_t)e + 1u} : Kept{LOWEST_KEY, 0u};
                const uint32_t near_some = s.flag;
                Draw draw{0xFFFFFFFFu, 0.0, 0.0, 0.0};
                if (MASS && set && near_some == 0u && turn == 0 && set->min_key(w.m) <= kept.key) {
                    // Nothing else takes tokens away: the kept ones' weights by CTA are known, and so is where the draw falls.  (Quick weights, so that
                    // the sums of CTAs and of their warps are the same ones.)
                    __syncthreads();
#pragma unroll
                    for (uint32_t k = 0; k < SM_EACH; k++) {
                        const uint32_t i = threadIdx.x * each + k;
                        if (k < each) s.list[i] = s.list[i] << 32 | __float_as_uint(i <= s.place ? w.quick(value_of((uint32_t)(s.list[i] >> 32))) : 0.0f);
                    }
                    __syncthreads();
                    for (uint32_t c = t.warp; c < t.C; c += SM_WARPS) {
                        double part = 0;
                        for (uint32_t i = t.lane; i < n; i += 32) {
                            const uint32_t token = ~(uint32_t)(s.list[i] >> 32);
                            if (token - c * whole < whole) part += (double)__uint_as_float((uint32_t)s.list[i]);
                        }
                        part = warp_sum(part);
                        if (t.lane == 0) s.step_mass[c] = part * unit + t.part(0, c);
                    }
                    __syncthreads();
                    const double part = t.lane < t.C ? s.step_mass[t.lane] : 0.0;
                    const double stay = warp_sum(part);
                    draw.target = (double)set->uniform * stay;
                    draw.near = how_near(vocab, stay, set->uniform, Border::OF_ITS_SUM);
                    draw.owner = t.first_above<SM_MAX_CLUSTER>(part, 0.0, draw.target, &draw.base);
                }
                if (threadIdx.x < t.C) {
                    Shared* p = t.peer(threadIdx.x);
                    p->kept = kept;
                    p->draw = draw;
                    p->again = near_some;
                }
            }
            t.sync();
            if (s.again == 0u) {
                found = s.draw;
                return s.kept;
            }
            if (turn == 1) break;
            // weights in 64 bits: of all, for the target, and of what is above
            double total = 0;
            above = 0;
            each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
                const float v[4] = {x.x, x.y, x.z, x.w};
                for (int k = 0; k < 4; k++)
                    if (v[k] > -INFINITY) {
                        const double e = w.exact(v[k]);
                        total += e;
                        if (v[k] > high) above += e;
                    }
            });
            t.total(total, above);
            if (share >= 0) target = share * total;
        }
    }
    // Too many candidates (ties, above all): bit by bit, with weights in 64 bits.
    if (MASS && share >= 0) {
        double total = kept_mass<true>(sl, t.warp, w, Kept{LOWEST_KEY, 0u}), none = 0;
        t.total(total, none);
        target = share * total;
    }
    auto from_key = [&](uint32_t key) {
        double mass = 0, none = 0;
        if (MASS) {
            mass = kept_mass<true>(sl, t.warp, w, Kept{key, 0xFFFFFFFFu});
        } else {
            each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
                mass += (double)((key_of(x.x) >= key) + (key_of(x.y) >= key) + (key_of(x.z) >= key) + (key_of(x.w) >= key));
            });
        }
        t.total(mass, none);
        return mass;
    };
    uint32_t least = LOWEST_KEY + 1u, most = key_of(w.m);      // from_key(least) reaches the target, as far as any does
    while (least < most) {
        const uint32_t mid = least + (most - least + 1u) / 2u;
        if (from_key(mid) >= target) least = mid;
        else most = mid - 1u;
    }
    const double more = from_key(least + 1u), each = MASS ? w.exact(value_of(least)) : 1.0;
    double ties = each > 0 ? fmax(ceil((target - more) / each), 1.0) : 1.0;
    if (ties > 1.0 && more + (ties - 1.0) * each >= target) ties -= 1.0;
    double equal = 0;
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        equal += (double)((key_of(x.x) == least) + (key_of(x.y) == least) + (key_of(x.z) == least) + (key_of(x.w) == least));
    });
    t.total(equal, none);
    if (ties >= equal) return Kept{least, 0xFFFFFFFFu};
    double base;
    const uint32_t owner = t.first_above<SM_MAX_CLUSTER>(t.lane < t.C ? t.part(0, t.lane) : 0.0, 0.0, ties - 0.5, &base);
    if (t.rank == owner) {
        bool near;
        const uint32_t p = find_place<double>(t, sl, base, ties - 0.5, 0.0, 0.0, vocab, &near, [&](uint32_t, float x) { return key_of(x) == least ? 1.0 : 0.0; });
        if (threadIdx.x < t.C) t.peer(threadIdx.x)->cut_at[1] = p + shift + 1u;
    }
    t.sync();
    return Kept{least, s.cut_at[1]};
}

// The choice among the candidates in the first CTA's list, which are the row's largest: everything in 64 bits.  With whole < 0 the list has all of the
// top_k; else top_p is a share of `whole`, known up to `near`, and the answer is whether the list has what it keeps.  Called by that CTA's threads.
__device__ bool choose_from_list(Team& t, const Weights& w, const Settings& set, uint32_t n, double whole, double near, float* x, uint32_t* token) {
    Shared& s = t.s;
    uint32_t each = sort_down(s.list, n);
    if (set.top_k) n = min(n, set.top_k);
    // neighbours to a thread
    uint32_t i0 = threadIdx.x * each;
    const uint32_t min_key = set.min_key(w.m);
    double v[SM_EACH], mine = 0, all;
#pragma unroll
    for (uint32_t k = 0; k < SM_EACH; k++) {
        v[k] = k < each && i0 + k < n ? w.exact(value_of((uint32_t)(s.list[i0 + k] >> 32))) : 0.0;
        mine += v[k];
    }
    if (threadIdx.x == 0) { s.place = 0u; s.flag = 0u; }
    double sum = t.before(mine, &all);
    const double enough = (double)set.top_p * (whole < 0 ? all : whole);
    bool open = whole >= 0 && all < enough + near;
    // what stays, with the token in front, so that the order becomes the tokens'
    unsigned long long e[SM_EACH];
#pragma unroll
    for (uint32_t k = 0; k < SM_EACH; k++) {
        const unsigned long long c = k < each && i0 + k < n ? s.list[i0 + k] : 0ull;
        const bool stays = c && (set.top_p >= 1.0f || sum < enough || i0 + k == 0u) && (uint32_t)(c >> 32) >= min_key;
        e[k] = stays ? c << 32 | c >> 32 : 0ull;
        open |= whole >= 0 && c && (fabs(sum - enough) <= near || fabs(sum + v[k] - enough) <= near);
        sum += v[k];
    }
    if (open) s.flag = 1u;
    __syncthreads();
    if (s.flag) return false;
#pragma unroll
    for (uint32_t k = 0; k < SM_EACH; k++)
        if (k < each) s.list[i0 + k] = e[k];
    __syncthreads();
    each = sort_down(s.list, n);             // (the first n, in the order of x, were looked at)
    i0 = threadIdx.x * each;
    mine = 0;
    uint32_t filled = 0;
#pragma unroll
    for (uint32_t k = 0; k < SM_EACH; k++) {
        const unsigned long long c = k < each ? s.list[i0 + k] : 0ull;
        v[k] = c ? w.exact(value_of((uint32_t)c)) : 0.0;
        if (v[k] > 0) filled = i0 + k;
        mine += v[k];
    }
    if (filled) atomicMax(&s.place, filled);         // (without a sum above the target the last one)
    sum = t.before(mine, &all);
    const double target = (double)set.uniform * all;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < SM_EACH; k++) {
        if (v[k] > 0 && sum <= target && sum + v[k] > target) s.place = i0 + k;
        sum += v[k];
    }
    __syncthreads();
    const unsigned long long c = s.list[s.place];
    *x = value_of((uint32_t)c);
    *token = ~(uint32_t)(c >> 32);
    return true;
}

// The choice of a token, a cluster to a row.  What it does for a row depends on the row's settings:
//   the largest x, or a draw without limits: the sums made while loading, one exchange between the CTAs, and for the draw a search by the CTA it falls to;
//   top_k of up to SM_QUICK_K, and a top_p that few tokens make up: the candidates go to the first CTA, which sorts them and does the rest in 64 bits;
//   otherwise: bins (counts or weights) of the whole row say between which two values the border lies, the candidates between them are sorted, and the
//   draw is made over what is above; should ties leave more than SM_CANDIDATES, a bisection of the values takes over.
// 256 rows of 131,072 in 16 bits (67 MB: 10.2 us at the memory's rate), no penalties: 40 us for the largest x, 78 for a draw, 77 with top_k 50, 111 with top_k 400,
// 225 with a top_p of 0.9 that keeps thousands of tokens and 106 with one that keeps few; histories of 1,500 tokens add some 23.  One row of 32,256:
// 5 us, 9, 13, 19, 26 and 14.  Neither memory nor arithmetic bounds it but the length of a row's way through the cluster's barriers: loading
// takes 9,000 cycles of a CTA (24 warps to an SM; exponentials alone 3,000), the first exchange 4,500, a draw 7,000, bins and border some 40,000.  An SM has three
// CTAs, by registers and shared memory.  Slices of 16,384 tokens are the largest of which three fit; smaller ones (clusters of 12 or 16, four CTAs to an
// SM) gain nothing, since what a warp does once for a row, some 600 instructions, is half of all it does at that size (168 us against 137 for a mixed batch, when both were measured).
template <class T>
__global__ void __launch_bounds__(SM_THREADS, 3)
k_sample(const __grid_constant__ b200bpe_logits in, const __grid_constant__ b200bpe_choice how, uint32_t vocab) {
    extern __shared__ __align__(16) float buf[];
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();        // (nobody writes into a CTA that has not begun)
    Team t(s);
    const Slice sl = slice_of<T>(in, vocab, blockIdx.x / t.C, t.rank, slice_tokens(vocab, t.C), buf);
    const int shift = (int)sl.lo - (int)sl.lead;
    const T* row = static_cast<const T*>(in.logits) + (uint64_t)sl.row * in.row_stride + sl.lo;
    uint4 ahead[SM_AHEAD];
    first_loads(row, sl, ahead);
    const double power_64 = TWO_TO_64THS[threadIdx.x % 64];
    const Settings set(how, sl.row, vocab);
    const bool by_k = set.top_k != 0u, by_p = set.top_p < 1.0f, quick_k = by_k && set.top_k <= SM_QUICK_K;
    const bool quick_p = !by_k && by_p && set.top_p > 0.0f;
    Stats stats;
    stats.c = __fdiv_rn(1.44269504f, (float)set.warm);
    {
        const MaskRow mask = mask_row(in, sl.row);
        const bool any_special = find_special(in, vocab, row, sl, mask, s.special);
        each_adjusted(row, sl, ahead, any_special, s.special, [&](uint32_t p, float (&v)[Packed<T>::N]) {
            store(buf + p, v);
            stats.add(v, p, buf);
        });
    }

    // The first exchange: the largest x and the lowest token that has it, the sum of all weights, and for top_k a value that so many are not below.
    float m, n;
    for (bool again = false;; again = true) {
        m = value_of(__reduce_max_sync(0xFFFFFFFFu, key_of(stats.m)));
        n = stats.base(m);
        double sum = stats.sum * Stats::power(stats.n - n);
        sum = warp_sum(sum);
        __syncthreads();
        if (t.lane == 0) { s.m_warp[t.warp] = m; s.n_warp[t.warp] = n; s.part_warp[0][t.warp] = sum; }
        if (threadIdx.x == 0) { s.at = 0xFFFFFFFFu; s.quick_candidates = 0u; }
        if (threadIdx.x < 4) s.cut[threadIdx.x] = -INFINITY;
        if (threadIdx.x < 64) s.table[threadIdx.x] = power_64;
        if (quick_k || quick_p) s.keys[threadIdx.x] = key_of(stats.m);
        else if (by_k)
            for (uint32_t i = threadIdx.x; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0u;
        __syncthreads();
        m = value_of(__reduce_max_sync(0xFFFFFFFFu, key_of(s.m_warp[t.lane % SM_WARPS])));
        n = stats.base(m);
        if (stats.m == m && m > -INFINITY) {
            uint32_t p = stats.at;
            for (int k = 1; k < Packed<T>::N && buf[p] != m; k++) p++;
            atomicMin(&s.at, p + shift);
        }
        if (t.warp < (quick_k ? 4 : quick_p ? 2 : 0)) {
            // cut[l]: at least top_k / 2^l of this slice are not below it.  The largest keys by their upper half that so many threads' largest x have.
            // For top_p: as many as are this CTA's part of 64 and of 256, and in cut[2 + l] what they weigh (not less); of a slice with fewer tokens
            // that are allowed, all.
            const uint32_t of_row = t.warp ? SM_QUICK_P1 : SM_QUICK_P0;
            const uint32_t wanted = quick_k ? (set.top_k + (1u << t.warp) - 1u) >> t.warp : min((of_row + t.C - 1u) / t.C, (of_row * sl.len + vocab - 1u) / vocab);
            uint32_t k[SM_THREADS / 32], most = 0u, least = 0xFFFFu;
#pragma unroll
            for (int i = 0; i < SM_THREADS / 32; i++) {
                k[i] = s.keys[i * 32 + t.lane] >> 16;
                most = max(most, k[i]);
                least = min(least, k[i]);
            }
            most = __reduce_max_sync(0xFFFFFFFFu, most);
            least = __reduce_min_sync(0xFFFFFFFFu, least);
            // (the bits that all of them have alike need no looking at, if there are enough of them)
            const uint32_t unlike = most == least ? 0u : 31u - __clz(most ^ least);
            uint32_t cut = wanted <= SM_THREADS ? most & ~((2u << unlike) - 1u) : 0u;
            for (uint32_t bit = most == least ? 0u : 1u << unlike; bit; bit >>= 1) {
                uint32_t so_many = 0;
#pragma unroll
                for (int i = 0; i < SM_THREADS / 32; i++) so_many += k[i] >= (cut | bit);
                if (__reduce_add_sync(0xFFFFFFFFu, so_many) >= wanted) cut |= bit;
            }
            if (most == least && wanted <= SM_THREADS) cut = most;
            if (t.lane == 0 && cut > LOWEST_KEY >> 16) s.cut[t.warp] = value_of(cut << 16);
            if (quick_p) {
                // (the upper half of -infinity's key, of a thread without an allowed token, is a NaN's)
                double weight = 0;
                uint32_t lowest = 0xFF80u;           // of infinity, where no token is allowed
#pragma unroll
                for (int i = 0; i < SM_THREADS / 32; i++)
                    if (k[i] > LOWEST_KEY >> 16 && k[i] >= cut) {
                        weight += (double)Stats::two_to(fmaf(value_of(k[i] << 16), stats.c, -n));
                        lowest = min(lowest, k[i]);
                    }
                weight = warp_sum(weight);
                lowest = __reduce_min_sync(0xFFFFFFFFu, lowest);
                if (t.lane == 0) {
                    s.cut[t.warp] = value_of(lowest << 16);
                    s.cut[2 + t.warp] = (float)weight;
                }
            }
        }
        __syncthreads();
        if (!again) cluster.barrier_wait();
        if (t.warp == 0) {
            const Best b{m, n, s.at, 0u, warp_sum<SM_WARPS>(s.part_warp[0][t.lane % SM_WARPS] * Stats::power(s.n_warp[t.lane % SM_WARPS] - n)),
                         {s.cut[0], s.cut[1], s.cut[2], s.cut[3]}};
            if (t.lane < t.C) t.peer(t.lane)->best[t.rank] = b;
        }
        t.sync();
        m = value_of(__reduce_max_sync(0xFFFFFFFFu, t.lane < t.C ? key_of(s.best[t.lane].m) : LOWEST_KEY));
        n = stats.base(m);
        if (again || m == -INFINITY || fabsf(m) * stats.c < Stats::FAR) break;
        // So far out that x c has no whole number in 32 bits next to it: with differences from m.  They are exact from m / 2 to 2 m, and what lies
        // further off weighs nothing.
        for (uint32_t p = threadIdx.x; p < sl.padded; p += SM_THREADS) buf[p] = buf[p] == m ? 0.0f : m == INFINITY ? -INFINITY : buf[p] - m;
        __syncthreads();
        Stats near;
        near.c = stats.c;
        stats = near;
        slice_stats(sl, stats);
        t.sync();            // (what came is read)
    }
    if (m == -INFINITY) {          // (the whole cluster)
        if (t.rank == 0 && threadIdx.x == 0) {
            how.tokens_out[sl.row] = B200BPE_NO_TOKEN;
            if (how.logprobs_out) how.logprobs_out[sl.row] = -INFINITY;
        }
        return;
    }
    if (set.greedy && (t.rank != 0 || t.warp != 0)) return;
    auto falls = [&](double part) {          // where the draw falls; a lane's part: that of a CTA
        Draw d;
        const double stay = warp_sum(part);
        d.target = (double)set.uniform * stay;
        d.near = how_near(vocab, stay, set.uniform, Border::OF_ITS_SUM);
        d.owner = t.first_above<SM_MAX_CLUSTER>(part, 0.0, d.target, &d.base);
        return d;
    };
    const bool limits = by_k || by_p || set.min_p > 0.0f;
    // What all warps need to know of the row; one works it out.
    if (t.warp == 0) {
        Row r;
        const Weights w{m, stats.c, n, 0.0, nullptr};
        r.unit = w.to_largest();
        const double part = t.lane < t.C ? s.best[t.lane].sum * Stats::power(s.best[t.lane].n - n) : 0.0;
        r.quick_all = warp_sum(part);
        r.all = r.quick_all * r.unit;
        if (!set.greedy && !limits) {
            const Draw d = falls(part * r.unit);
            if (t.lane == 0) s.draw = d;
        }
        r.steps = set.greedy ? 0.0 : 64 * 1.4426950408889634 / set.warm;
        // A value that all of the top_k, or all that top_p keeps, are not below, if there is such a one.
        r.from = -INFINITY;
        r.quick = quick_k;
        if (quick_k) {
            // At least top_k x are not below the largest value that 2^l of the CTAs have 1/2^l of top_k for.
            for (uint32_t i = t.lane; i < 4 * SM_MAX_CLUSTER; i += 32) {
                const uint32_t l = i / SM_MAX_CLUSTER, c = i % SM_MAX_CLUSTER;
                if (c < t.C && 1u << l <= t.C) {
                    const float mine = s.best[c].cut[l];
                    uint32_t so_many = 0;
                    for (uint32_t o = 0; o < t.C; o++) so_many += s.best[o].cut[l] >= mine;
                    if (so_many >= 1u << l) r.from = fmaxf(r.from, mine);
                }
            }
            r.from = value_of(__reduce_max_sync(0xFFFFFFFFu, key_of(r.from)));
        } else if (quick_p) {
            // What the CTAs' parts of 64, or of 256, weigh is enough.
            for (int l = 0; l < 2 && !r.quick; l++) {
                const double weight = warp_sum(t.lane < t.C ? (double)s.best[t.lane].cut[2 + l] * Stats::power(s.best[t.lane].n - n) : 0.0) * r.unit;
                r.quick = weight >= (double)set.top_p * r.all;
                r.from = value_of(__reduce_min_sync(0xFFFFFFFFu, t.lane < t.C ? key_of(s.best[t.lane].cut[l]) : 0xFFFFFFFFu));
            }
        }
        if (t.lane == 0) s.row = r;
    }
    if (set.greedy) __syncwarp();
    else __syncthreads();
    const Weights w{m, stats.c, n, s.row.steps, s.table};
    const double unit = s.row.unit, all = s.row.all;
    const bool quick = s.row.quick;
    float from = s.row.from;
    auto answer = [&](uint32_t token, float x) {
        how.tokens_out[sl.row] = token;
        if (how.logprobs_out)
            how.logprobs_out[sl.row] = (float)(((double)x - (double)m) / set.warm - (log(s.row.quick_all) + 0.693147180559945309 * w.power_of_largest()));
    };
    if (set.greedy) {
        if (threadIdx.x == 0) {
            uint32_t token = 0xFFFFFFFFu;
            for (uint32_t c = 0; c < t.C; c++)
                if (s.best[c].m == m) token = min(token, s.best[c].at);
            answer(token, m);
        }
        return;
    }

    // The kept tokens.
    Kept kept{LOWEST_KEY, 0u};
    Draw draw{0xFFFFFFFFu, 0.0, 0.0, 0.0};
    if (quick) {
        from = fmaxf(from, -3.402823466e38f);            // (-infinity is never chosen)
        Shared* lead = t.peer(0);
        // (most groups of 512 places have none)
        const Span span(sl.padded, t.warp);
        for (uint32_t p0 = span.lo + t.lane * 4; p0 < span.hi + t.lane * 4; p0 += 512) {
            float4 x[4];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = p0 + j * 128 < span.hi ? *reinterpret_cast<const float4*>(buf + p0 + j * 128) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                top = fmaxf(top, fmaxf(fmaxf(x[j].x, x[j].y), fmaxf(x[j].z, x[j].w)));
            }
            if (!__any_sync(0xFFFFFFFFu, top >= from)) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                uint32_t in = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) in |= (uint32_t)(v[k] >= from) << k;
                gather(t, &s.quick_candidates, s.list, v, in, p0 + j * 128 + shift);
            }
        }
        hand_over(t, &Shared::quick_candidates);
        t.sync();
        const uint32_t so_many = lead->quick_candidates;
        float x;
        uint32_t token;
        if (quick_k) {
            cluster.barrier_arrive();
            if (so_many <= SM_CANDIDATES) {
                if (t.rank != 0) return;
                choose_from_list(t, w, set, so_many, -1.0, 0.0, &x, &token);
                if (threadIdx.x == 0) answer(token, x);
                cluster.barrier_wait();          // (the others have looked at the number)
                return;
            }
            cluster.barrier_wait();
        } else if (so_many <= SM_CANDIDATES) {
            if (t.rank == 0) {
                const bool done = choose_from_list(t, w, set, so_many, all, how_near(vocab, all, set.top_p, Border::OF_EXACT_SUMS), &x, &token);
                if (threadIdx.x == 0 && done) answer(token, x);
                if (threadIdx.x < t.C) t.peer(threadIdx.x)->again = !done;
            }
            t.sync();
            if (s.again == 0u) return;
        }
    }
    if (quick_k || quick_p) {
        for (uint32_t i = threadIdx.x; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0u;
        __syncthreads();
    }
    if (by_k) {
        // (what weighs less than e^-32 does not matter to top_p; it may to top_k, where a temperature is low)
        const Bins bins(m, fmax(32.0 * set.warm, 24.0));
        each_four(sl, t.warp, [&](uint32_t, const float4& x) {
            bins.put<false>(s.bins, x, SM_BINS - 1.5f);
        });
        t.sync();
        kept = border<false>(t, sl, w, bins, (double)set.top_k, -1.0, 0.0, nullptr, vocab, draw);
    }
    if (by_p) {
        double whole = all, none = 0;
        if (by_k) {
            whole = kept_mass<true>(sl, t.warp, w, kept);
            t.total(whole, none);
            for (uint32_t i = threadIdx.x; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0u;
            __syncthreads();
        }
        Kept k{LOWEST_KEY, 0u};
        if (set.top_p > 0.0f) {
            const Bins bins(m, 32.0 * set.warm);
            // All that lie lower than this weigh less than half of what top_p leaves out.
            float end = SM_BINS - 1.5f;
            if (set.top_p < 0.999f) end = fminf(end, 64.0f * logf((float)((double)vocab / (0.5 * (1.0 - set.top_p) * whole))) + 1.0f);
            each_four(sl, t.warp, [&](uint32_t, const float4& x) {
                bins.put<true>(s.bins, x, end);
            });
            t.sync();
            k = border<true>(t, sl, w, bins, (double)set.top_p * whole, by_k ? -1.0 : (double)set.top_p, how_near(vocab, whole, set.top_p, by_k ? Border::EXACT : Border::OF_ITS_SUM),
                             by_k ? nullptr : &set, vocab, draw);
        } else {
            uint32_t token = 0xFFFFFFFFu;
            for (uint32_t c = 0; c < t.C; c++)
                if (s.best[c].m == m) token = min(token, s.best[c].at);
            k = {key_of(m), token + 1u};
        }
        if (k.key > kept.key || (k.key == kept.key && k.end < kept.end)) kept = k;
    }
    const uint32_t min_key = set.min_key(m);
    if (min_key > kept.key) kept = {min_key, 0xFFFFFFFFu};

    // The draw.
    auto chosen = [&](auto exact, const Draw& draw, uint32_t* place) {         // whether this CTA has the token; every warp's sum is in s.warp_mass
        constexpr bool EXACT = decltype(exact)::value;
        if (t.rank == draw.owner) {
            bool near;
            if (EXACT) *place = find_place<double>(t, sl, draw.base, draw.target, 0.0, 0.0, vocab, &near, [&](uint32_t p, float x) { return kept.has(x, p + shift) ? w.exact(x) : 0.0; });
            else *place = find_place<float>(t, sl, draw.base, draw.target, draw.near, set.uniform, vocab, &near, [&](uint32_t p, float x) { return kept.has(x, p + shift) ? w.quick(x) * (float)unit : 0.0f; });
            if (!EXACT && threadIdx.x < t.C) t.peer(threadIdx.x)->cut_at[0] = near;
        }
        return t.rank == draw.owner;
    };
    if (draw.owner != 0xFFFFFFFFu) {
        if (t.rank == draw.owner) {
            // Every warp's sum of what lies above the border's bins is there; of the candidates those that stay are added.  The CTA's own are still in its
            // list, and the first CTA's has all of them, with their weights.
            const Span span(sl.padded, t.warp);
            double mass = 0;
            for (uint32_t i = t.lane; i < s.candidates; i += 32) {
                const unsigned long long e = s.list[i];
                const uint32_t v = ~(uint32_t)(t.rank ? e : e >> 32), p = v - shift;
                if (p < span.lo || p >= span.hi || v < sl.lo || v - sl.lo >= sl.len) continue;
                if (t.rank == 0) mass += (double)__uint_as_float((uint32_t)e) * unit;
                else if (const float x = value_of((uint32_t)(e >> 32)); kept.has(x, v)) mass += (double)w.quick(x) * unit;
            }
            mass = warp_sum(mass);
            if (t.lane == 0) s.warp_mass[t.warp] += mass;
            __syncthreads();
        }
    } else if (!limits) {
        draw = s.draw;
        if (t.rank == draw.owner) {
            if (threadIdx.x < SM_WARPS) s.warp_mass[threadIdx.x] = s.part_warp[0][threadIdx.x] * Stats::power(s.n_warp[threadIdx.x] - n) * unit;
            __syncthreads();
        }
    } else {
        double mass = kept_mass<false>(sl, t.warp, w, kept), none = 0;
        t.total(mass, none);
        draw = falls(t.lane < t.C ? t.part(0, t.lane) : 0.0);
    }
    uint32_t place = 0;
    bool mine = chosen(std::false_type{}, draw, &place);
    t.sync();
    if (s.cut_at[0]) {
        double mass = kept_mass<true>(sl, t.warp, w, kept), none = 0;
        t.total(mass, none);
        mine = chosen(std::true_type{}, falls(t.lane < t.C ? t.part(0, t.lane) : 0.0), &place);
    }
    if (mine && threadIdx.x == 0) answer(place + shift, buf[place]);
}

struct Sampler {
    CtxHold hold;
    Ctx* ctx = nullptr;
    uint32_t vocab = 0;
};

// Whether these pointers to 32-bit values lie as such values have to.
template <class... P>
static bool words(const P*... p) { return (... && (reinterpret_cast<uint64_t>(p) % 4 == 0)); }

static b200bpe_status check_logits(const b200bpe_logits* in) {
    if (!in || in->struct_size != sizeof(b200bpe_logits)) return refused("logits: struct_size is not that of b200bpe_logits");
    if (in->dtype > B200BPE_BF16) return refused("logits: unknown dtype");
    if (in->n_rows >= 1u << 27) return refused("logits: more than 2^27 - 1 rows");
    if (in->n_rows == 0) return B200BPE_OK;
    if (!words(in->history, in->lengths, in->prompt_lengths, in->repetition, in->presence, in->frequency, in->bias_tokens, in->biases, in->mask, in->mask_rows))
        return refused("logits: a misaligned pointer");
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

// CTAs of a row's cluster: slices of 2,048 tokens where eight CTAs are enough for that, of at most 16,384 otherwise (three CTAs to an SM).
static uint32_t cluster_for(uint32_t vocab) {
    uint32_t c = 1;
    while (c < 8 && vocab > c * 2048u) c *= 2;
    while (c < SM_MAX_CLUSTER && vocab > c * 16384u) c *= 2;
    return c;
}

template <class T>
static b200bpe_status launch_sample(const b200bpe_logits& in, const b200bpe_choice& how, uint32_t vocab, cudaStream_t stream) {
    const uint32_t c = cluster_for(vocab);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(in.n_rows * c);
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = (slice_tokens(vocab, c) + 16) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = c;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    cfg.attrs = &a;
    cfg.numAttrs = 1;
    B2_CUDA(cudaLaunchKernelEx(&cfg, k_sample<T>, in, how, vocab));
    return B200BPE_OK;
}

template <class T>
static b200bpe_status launch_adjust(const b200bpe_logits& in, uint32_t vocab, void* out, uint64_t out_stride, int sm_count, cudaStream_t stream) {
    // Small slices have all their loads on their way at once (256 x 131,072 in 32 bits: 41.5 us against 48.0 with 8,192 tokens), but each of them counts the
    // row's history for itself (with histories of 1,500: 61.9 against 60.3; 61 rows of 50,021: 7.7 against 5.7), which costs nothing while SMs are left over.
    const uint64_t most = (uint64_t)in.n_rows * ((vocab + SM_ADJUST_SLICE / 2 - 1) / (SM_ADJUST_SLICE / 2));
    const uint32_t whole = in.history && most > (uint64_t)sm_count * 4 ? SM_ADJUST_SLICE : SM_ADJUST_SLICE / 2;
    const uint64_t parts = (vocab + whole - 1) / whole;
    if (parts * in.n_rows > 0x7FFFFFFFu) return refused("b200bpe_sampler_adjust: too many rows");
    const size_t bytes = in.history || in.n_bias ? (std::min(vocab, whole) + 16) * 4 : 0;
    k_adjust<T><<<(uint32_t)(parts * in.n_rows), SM_THREADS, bytes, stream>>>(in, vocab, whole, static_cast<T*>(out), out_stride);
    B2_CUDA(cudaGetLastError());
    return B200BPE_OK;
}

// Loads the kernels, so that no call has to, and lets them have a CTA's whole shared memory.
static cudaError_t ready() {
    cudaFuncAttributes fa;
    for (const void* k : {(const void*)k_adjust<float>, (const void*)k_adjust<__half>, (const void*)k_adjust<__nv_bfloat16>})
        if (const cudaError_t e = cudaFuncGetAttributes(&fa, k)) return e;
    for (const void* k : {(const void*)k_sample<float>, (const void*)k_sample<__half>, (const void*)k_sample<__nv_bfloat16>}) {
        if (const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (SM_MAX_SLICE + 16) * 4)) return e;
        if (const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
    }
    return cudaSuccess;
}

}  // namespace b200bpe

struct b200bpe_sampler { b200bpe::Sampler s; };

using namespace b200bpe;

extern "C" {

b200bpe_status b200bpe_sampler_create(b200bpe_ctx* c, uint32_t vocab_size, b200bpe_sampler** out) {
    if (vocab_size == 0 || vocab_size > SM_MAX_VOCAB) return refused("b200bpe_sampler_create: 1 to 327,680 tokens");
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
        case B200BPE_F32: return launch_adjust<float>(*in, vocab, logits_out, out_stride, h->s.ctx->sm_count, st);
        case B200BPE_F16: return launch_adjust<__half>(*in, vocab, logits_out, out_stride, h->s.ctx->sm_count, st);
        default: return launch_adjust<__nv_bfloat16>(*in, vocab, logits_out, out_stride, h->s.ctx->sm_count, st);
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
    if (!words(how->uniform, how->temperature, how->top_k, how->top_p, how->min_p, how->tokens_out, how->logprobs_out)) return refused("choice: a misaligned pointer");
    const OnDevice on(h->s.ctx->device);
    B2_CUDA(on.error);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (in->dtype) {
        case B200BPE_F32: return launch_sample<float>(*in, *how, vocab, st);
        case B200BPE_F16: return launch_sample<__half>(*in, *how, vocab, st);
        default: return launch_sample<__nv_bfloat16>(*in, *how, vocab, st);
    }
}

void b200bpe_sampler_destroy(b200bpe_sampler* h) { delete h; }

}  // extern "C"
