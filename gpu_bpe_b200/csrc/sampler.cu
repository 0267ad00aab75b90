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

constexpr int SM_THREADS = 512;
constexpr int SM_WARPS = SM_THREADS / 32;
constexpr uint32_t SM_MAX_CLUSTER = 8;           // portable size
constexpr uint32_t SM_MAX_SLICE = 53248;         // 208 KB of 32-bit values
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

// Sixteen bytes of logits from place p of the slice on, as values; places outside the slice give -infinity.
template <class T>
__device__ __forceinline__ uint4 fetch(const T* row, const Slice& s, uint32_t p) {
    constexpr uint32_t N = Packed<T>::N;
    if (p >= s.lead && p + N <= s.lead + s.len) return __ldcs(reinterpret_cast<const uint4*>(row + (p - s.lead)));
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

// Bits of the N tokens from `token` on (a negative one: of those before the row) in the lowest bits.
template <int N>
__device__ __forceinline__ uint32_t mask_bits(const MaskRow& mask, int token, uint32_t vocab) {
    if (mask.none) return 0u;
    if (!mask.words) return 0xFFFFFFFFu;
    const int w = token >> 5, words = (int)((vocab + 31u) / 32u);
    const uint32_t lo = w >= 0 && w < words ? __ldg(mask.words + w) : 0u;
    if (((uint32_t)token & 31u) + N <= 32u) return lo >> (token & 31);
    return __funnelshift_r(lo, w + 1 < words ? __ldg(mask.words + w + 1) : 0u, (uint32_t)token & 31u);
}

// Fills the slice with x.  SCRUB: a NaN becomes -infinity, and -0 becomes 0.  Called by all threads of the cluster; ends with a barrier of the CTA.
// The first loads of the row are on their way while the history is counted: a call with one row waits for little else.
template <class T, bool SCRUB>
__device__ void load_slice(const b200bpe_logits& in, uint32_t vocab, const Slice& s) {
    constexpr uint32_t N = Packed<T>::N, AHEAD = 4, STEP = SM_THREADS * N;
    const float lowest = -INFINITY;
    const T* row = static_cast<const T*>(in.logits) + (uint64_t)s.row * in.row_stride + s.lo;
    uint4 q[AHEAD];
#pragma unroll
    for (uint32_t j = 0; j < AHEAD; j++)
        if (threadIdx.x * N + j * STEP < s.padded) q[j] = fetch(row, s, threadIdx.x * N + j * STEP);
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
        for (uint32_t i = threadIdx.x * 4; i < s.padded; i += SM_THREADS * 4) *reinterpret_cast<uint4*>(marks + i) = make_uint4(0u, 0u, 0u, 0u);
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
    for (uint32_t p0 = threadIdx.x * N; p0 < s.padded; p0 += AHEAD * STEP) {
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; j++) {
            const uint32_t p = p0 + j * STEP;
            if (p >= s.padded) break;
            const Packed<T> now{q[j]};
            if (p + AHEAD * STEP < s.padded) q[j] = fetch(row, s, p + AHEAD * STEP);
            const uint32_t allowed = mask_bits<N>(mask, (int)(s.lo + p) - (int)s.lead, vocab);
            float v[N];
#pragma unroll
            for (uint32_t k = 0; k < N; k += 4) {
                uint4 mark = make_uint4(0u, 0u, 0u, 0u);
                if (n_seen) mark = *reinterpret_cast<const uint4*>(s.buf + p + k);
                if (mark.x | mark.y | mark.z | mark.w) {
                    v[k] = pen.on(now.get(k), mark.x);
                    v[k + 1] = pen.on(now.get(k + 1), mark.y);
                    v[k + 2] = pen.on(now.get(k + 2), mark.z);
                    v[k + 3] = pen.on(now.get(k + 3), mark.w);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) v[k + i] = now.get(k + i);
                }
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    if (!(allowed >> (k + i) & 1u)) v[k + i] = lowest;
                    if (SCRUB) v[k + i] = fmaxf(v[k + i] + 0.0f, lowest);        // (of a NaN and a number the number)
                }
                *reinterpret_cast<float4*>(s.buf + p + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            }
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
            if (SCRUB) v = fmaxf(v + 0.0f, lowest);
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
    // Places that lie on 16 bytes in the logits do so in the output if its rows are aligned like the logits' (in place, and with equal strides).
    constexpr uint32_t N = Packed<T>::N;
    T* to = out + (uint64_t)s.row * out_stride + s.lo;
    const bool alike = (reinterpret_cast<uint64_t>(to) & 15u) == s.lead * sizeof(T);
    for (uint32_t p = threadIdx.x * N; p < s.padded; p += SM_THREADS * N) {
        T v[N];
#pragma unroll
        for (uint32_t k = 0; k < N; k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(s.buf + p + k);
            rounded(x.x, v + k);
            rounded(x.y, v + k + 1);
            rounded(x.z, v + k + 2);
            rounded(x.w, v + k + 3);
        }
        if (alike && p >= s.lead && p + N <= s.lead + s.len) {
            uint4 q;
            memcpy(&q, v, 16);
            __stcs(reinterpret_cast<uint4*>(to + (p - s.lead)), q);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < N; k++)
                if (p + k >= s.lead && p + k < s.lead + s.len) to[p + k - s.lead] = v[k];
        }
    }
}

// ── the choice ──
// The order of x as unsigned integers, and back.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

constexpr uint32_t LOWEST_KEY = 0x007FFFFFu;     // of -infinity
constexpr uint32_t SM_BINS = 2048;
constexpr uint32_t SM_CANDIDATES = 1024;

// Which token is chosen depends on sums of weights: on the first running sum that is above a border.  Sums are made of weights in 32 bits,
// w = 2^y with y = (x - m) * (log2 e / temperature), and added in 64 bits: y is off by at most three roundings, 3 * 2^-24 |y|, and the exponential
// by 2^-22 of itself; four weights are added in 32 bits first, two more roundings.  So no sum is further off than
//     E = sum w * (2^-22 + 2^-23 + 3 * 2^-24 * ln 2 * |y|),
// and where a border lies within 2 E (E of the sum, E of the border, which is a share of another one) of a sum that decides, the row's sums are made
// again of weights in 64 bits.  An exponential in 64 bits is some 18 operations at half the rate of those in 32, against 5 and a quarter of a special one.
struct Weights {
    float m, c;         // the largest x, log2 e / temperature
    double by;          // 1 / temperature
    __device__ __forceinline__ float power(float x) const { return fmaxf(fminf((x - m) * c, 0.0f), -150.0f); }   // (inf - inf is 0)
    __device__ __forceinline__ float quick(float x) const { return two_to(power(x)); }
    static __device__ __forceinline__ float two_to(float y) {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(y));
        return w;
    }
    __device__ __forceinline__ double log_of(float x) const { return x == m ? 0.0 : ((double)x - (double)m) * by; }
    __device__ __forceinline__ double exact(float x) const { return x == m ? 1.0 : exp(log_of(x)); }
};

// What of the row is kept: x with a larger key, and those with the key in front of token `end`.
struct Kept {
    uint32_t key, end;
    __device__ __forceinline__ bool has(float x, uint32_t v) const {
        const uint32_t k = key_of(x);
        return k > key || (k == key && v < end);
    }
};

struct Best { float x; uint32_t at; };

struct Shared {
    Best best_warp[SM_WARPS], best_cta[SM_MAX_CLUSTER];
    double part_warp[2][SM_WARPS], part_cta[2][2][SM_MAX_CLUSTER];      // (the second index: one exchange and the next)
    double scan_warp[SM_WARPS], warp_mass[SM_WARPS];
    float cut_cta[2][SM_MAX_CLUSTER];
    uint32_t border[2], candidates, flag, place, cut[2];
    Kept kept;
    union {
        uint32_t bins[SM_BINS];
        unsigned long long list[SM_CANDIDATES];      // candidates: key << 32 | ~token
    };
};

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
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
            b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
        }
        __syncthreads();
        if (lane == 0) { s.part_warp[0][warp] = s.warp_mass[warp] = a; s.part_warp[1][warp] = b; }
        __syncthreads();
        par ^= 1;
        if (warp == 0) {
            a = b = 0;
#pragma unroll
            for (int w = 0; w < SM_WARPS; w++) { a += s.part_warp[0][w]; b += s.part_warp[1][w]; }
            if (threadIdx.x < C) {
                Shared* p = peer(threadIdx.x);
                p->part_cta[0][par][rank] = a;
                p->part_cta[1][par][rank] = b;
            }
        }
        sync();
        a = b = 0;
        for (uint32_t c = 0; c < C; c++) { a += part(0, c); b += part(1, c); }
    }
    __device__ double part(int i, uint32_t cta) const { return s.part_cta[i][par][cta]; }

    // Sum of v over the threads before this one; *all: over all.
    __device__ double before(double v, double* all) {
        double run = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xFFFFFFFFu, run, o);
            if (lane >= o) run += y;
        }
        __syncthreads();
        if (lane == 31) s.scan_warp[warp] = run;
        __syncthreads();
        double base = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < SM_WARPS; w++) {
            if (w == warp) base = sum;
            sum += s.scan_warp[w];
        }
        *all = sum;
        return base + run - v;
    }
};

// A warp's part of the slice: places [lo, hi), in steps of 128, four to a lane.
struct Span {
    uint32_t lo, hi;
    __device__ Span(uint32_t padded, int warp) {
        const uint32_t each = (padded + SM_WARPS * 128 - 1) / (SM_WARPS * 128) * 128;
        lo = min(each * warp, padded);
        hi = min(lo + each, padded);
    }
};

template <class F>
__device__ __forceinline__ void each_four(const Slice& sl, int warp, F f) {
    const Span span(sl.padded, warp);
    for (uint32_t p = span.lo + (threadIdx.x & 31) * 4; p < span.hi; p += 128) f(p, *reinterpret_cast<const float4*>(sl.buf + p));
}

// Sum of f over a row's kept places, with weights in 64 bits or in 32.
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
    return sum;
}

// The first place of the slice at which base plus the running sum of f(place, x) is above target; if there is none, the last with f above 0.  Every
// warp's sum of f is in s.warp_mass.  *near: whether a sum that decided was within `margin` of target.  Called by all threads of one CTA.
template <class F>
__device__ uint32_t find_place(Team& t, const Slice& sl, double base, double target, double margin, bool* near, F f) {
    Shared& s = t.s;
    double at = base;
    int owner = -1, filled = 0;
    for (int w = 0; w < SM_WARPS && owner < 0; w++) {
        if (s.warp_mass[w] > 0) filled = w;
        if (at + s.warp_mass[w] > target) owner = w;
        else at += s.warp_mass[w];
    }
    if (owner < 0) {
        owner = filled;
        at = base;
        for (int w = 0; w < owner; w++) at += s.warp_mass[w];
    }
    if (t.warp == owner) {
        const Span span(sl.padded, t.warp);
        uint32_t place = 0;
        bool close = false, found = false;
        for (uint32_t p0 = span.lo; p0 < span.hi && !found; p0 += 128) {
            const uint32_t p = p0 + t.lane * 4;
            double v[4] = {0, 0, 0, 0};
            if (p < span.hi) {
                const float4 x = *reinterpret_cast<const float4*>(sl.buf + p);
                v[0] = f(p, x.x); v[1] = f(p + 1, x.y); v[2] = f(p + 2, x.z); v[3] = f(p + 3, x.w);
            }
            const double mine = (v[0] + v[1]) + (v[2] + v[3]);
            double run = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, run, o);
                if (t.lane >= o) run += y;
            }
            double sum = at + run - mine;
            uint32_t hit = 0, last = 0;
            bool edge = false;
            for (int k = 3; k >= 0; k--) if (v[k] > 0 && last == 0) last = p + k + 1;
            for (int k = 0; k < 4; k++) {
                const double next = sum + v[k];
                if (v[k] > 0 && hit == 0) {
                    edge = fabs(next - target) <= margin || fabs(sum - target) <= margin;
                    if (next > target) hit = p + k + 1;
                }
                sum = next;
            }
            const uint32_t above = __ballot_sync(0xFFFFFFFFu, hit != 0), some = __ballot_sync(0xFFFFFFFFu, last != 0);
            if (above) {
                const int l = __ffs(above) - 1;
                place = __shfl_sync(0xFFFFFFFFu, hit, l) - 1;
                close = __shfl_sync(0xFFFFFFFFu, edge, l);
                found = true;
            } else {
                if (some) place = __shfl_sync(0xFFFFFFFFu, last, 31 - __clz(some)) - 1;
                at += __shfl_sync(0xFFFFFFFFu, run, 31);
            }
        }
        // (no sum above the target: only where rounding, or a uniform of 1, put the target at the whole sum)
        if (t.lane == 0) { s.place = place; s.flag = close || !found; }
    }
    __syncthreads();
    *near = s.flag != 0;
    return s.place;
}

// Descending order of n numbers (n a power of two, at most SM_CANDIDATES).
__device__ void sort_down(unsigned long long* a, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t step = size >> 1; step; step >>= 1) {
            for (uint32_t i = threadIdx.x; i < n / 2; i += SM_THREADS) {
                const uint32_t lo = (i / step) * step * 2 + i % step, hi = lo + step;
                const unsigned long long x = a[lo], y = a[hi];
                if ((x < y) == ((lo & size) == 0)) { a[lo] = y; a[hi] = x; }
            }
            __syncthreads();
        }
}

// Bins of x, from the largest downwards: SM_BINS of them over `range`; the last one takes the rest.
struct Bins {
    float m, scale;
    __device__ Bins(float largest, double range) : m(largest), scale((float)(SM_BINS / fmin(range, 3.4e38))) {}
    __device__ __forceinline__ uint32_t of(float x) const { return min(__float2uint_rz((m - x) * scale), SM_BINS - 1); }   // (not a number is 0)
    // x's weight in parts of 2^16 of its bin's largest, where a bin is 1/64 wide: e^-r by its first terms, rounded down.
    __device__ __forceinline__ uint32_t weight_of(float x, uint32_t bin) const {
        const float r = fmaxf((m - x) * scale - (float)bin, 0.0f) * (1.0f / 64);
        return __float2uint_rz(65536.0f - 65536.0f * r + 32768.0f * r * r);
    }
};

// The part of the row's order at which a running sum, from the largest x on, reaches `target`: of weights (MASS) or of tokens.
// s.bins are filled in all CTAs (weights: in parts of 2^16 of the bin's largest), and a barrier of the cluster is behind that.
// Returns what is kept up to and with the token that reaches it, the same in every CTA.
template <bool MASS>
__device__ Kept border(Team& t, const Slice& sl, const Weights& w, const Bins& bins, double target, double share, double margin) {
    Shared& s = t.s;
    const int shift = (int)sl.lo - (int)sl.lead;
    // every CTA adds up a part of the bins for all
    const uint32_t mine = SM_BINS / t.C, per = max(mine / SM_THREADS, 1u), first = t.rank * mine + threadIdx.x * per;
    const bool busy = threadIdx.x * per < mine;
    double here[SM_BINS / SM_THREADS], sum = 0;
    for (uint32_t k = 0; k < per; k++) {
        here[k] = 0;
        if (busy) {
            unsigned long long n = 0;
            for (uint32_t c = 0; c < t.C; c++) n += t.peer(c)->bins[first + k];
            here[k] = MASS ? (double)n * exp(-(double)(first + k) / 64) / 65536.0 : (double)n;
        }
        sum += here[k];
    }
    if (threadIdx.x < 2) s.border[threadIdx.x] = SM_BINS - 1;
    if (threadIdx.x == 0) s.candidates = 0u;
    double all, at = t.before(sum, &all);
    // (t.total's barriers: the parts of a bin may be read until here)
    double a = threadIdx.x == 0 ? all : 0.0, none = 0;
    t.total(a, none);
    for (uint32_t c = 0; c < t.rank; c++) at += t.part(0, c);
    const double slack = MASS ? 4.0 / 65536 : 0.0;          // of a bin's parts, and of the weights
    for (uint32_t k = 0; k < per && busy; k++) {
        const double next = at + here[k];
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
    const uint32_t from = s.border[0], to = max(s.border[1], from);
    double above = 0, count = 0;
    Shared* lead = t.peer(0);
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        const float v[4] = {x.x, x.y, x.z, x.w};
        float part = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t b = bins.of(v[k]);
            if (v[k] == -INFINITY || b > to) continue;
            if (b < from) {
                if (MASS) part += w.quick(v[k]);
                else part += 1.0f;
            } else {
                const uint32_t n = atomicAdd(&lead->candidates, 1u);
                // (the list lies where the first CTA's bins were)
                if (n < SM_CANDIDATES) lead->list[n] = (unsigned long long)key_of(v[k]) << 32 | (uint32_t)~(p + k + shift);
            }
        }
        above += (double)part;
    });
    t.total(above, count);
    const uint32_t n = t.peer(0)->candidates;
    if (n <= SM_CANDIDATES) {
        for (int turn = 0; turn < 2; turn++) {
            // turn 1: again with the sums in 64 bits
            if (t.rank == 0) {
                uint32_t size = 2;
                while (size < n) size *= 2;
                if (turn == 0) {
                    for (uint32_t i = n + threadIdx.x; i < size; i += SM_THREADS) s.list[i] = 0ull;
                    __syncthreads();
                    sort_down(s.list, size);
                }
                // two neighbours to a thread; flag 1: a sum was near, 2: the bins were misjudged
                double v[2];
                for (int k = 0; k < 2; k++) {
                    const uint32_t i = threadIdx.x * 2 + k;
                    v[k] = i < n ? (MASS ? w.exact(value_of((uint32_t)(s.list[i] >> 32))) : 1.0) : 0.0;
                }
                if (threadIdx.x == 0) { s.flag = 0u; s.place = n ? n - 1 : 0u; }
                double ignored, sum = above + t.before(v[0] + v[1], &ignored);
                for (int k = 0; k < 2; k++) {
                    const double next = sum + v[k];
                    const uint32_t i = threadIdx.x * 2 + k;
                    if (i < n && sum < target && next >= target) s.place = i;
                    if (MASS && turn == 0 && i < n && (fabs(sum - target) <= margin || fabs(next - target) <= margin)) s.flag = 1u;
                    sum = next;
                }
                const double near = turn == 0 ? margin : 0.0;
                if (MASS && threadIdx.x == 0 && above >= target - near) s.flag = 1u + turn;
                if (MASS && threadIdx.x == SM_THREADS - 1 && sum < target + near) s.flag = 1u + turn;
                __syncthreads();
                if (threadIdx.x < t.C) {
                    Shared* p = t.peer(threadIdx.x);
                    const unsigned long long e = s.list[s.place];
                    p->kept = n ? Kept{(uint32_t)(e >> 32), ~(uint32_t)e + 1u} : Kept{LOWEST_KEY, 0u};
                    p->cut[0] = s.flag;
                }
            }
            t.sync();
            if (s.cut[0] == 0u) return s.kept;
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
                        if (bins.of(v[k]) < from) above += e;
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
            mass = kept_mass<true>(sl, t.warp, w, Kept{key - 1u, 0u});
        } else {
            each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
                mass += (double)((key_of(x.x) >= key) + (key_of(x.y) >= key) + (key_of(x.z) >= key) + (key_of(x.w) >= key));
            });
        }
        t.total(mass, none);
        return mass;
    };
    uint32_t low = LOWEST_KEY + 1u, high = key_of(w.m);      // from_key(low) reaches the target, as far as any does
    while (low < high) {
        const uint32_t mid = low + (high - low + 1u) / 2u;
        if (from_key(mid) >= target) low = mid;
        else high = mid - 1u;
    }
    const double more = from_key(low + 1u), each = MASS ? w.exact(value_of(low)) : 1.0;
    double ties = each > 0 ? fmax(ceil((target - more) / each), 1.0) : 1.0;
    if (ties > 1.0 && more + (ties - 1.0) * each >= target) ties -= 1.0;
    double equal = 0;
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        equal += (double)((key_of(x.x) == low) + (key_of(x.y) == low) + (key_of(x.z) == low) + (key_of(x.w) == low));
    });
    t.total(equal, none);
    if (ties >= equal) return Kept{low, 0xFFFFFFFFu};
    double base = 0;
    uint32_t owner = 0;
    while (owner + 1 < t.C && base + t.part(0, owner) < ties) base += t.part(0, owner++);
    if (t.rank == owner) {
        bool near;
        const uint32_t p = find_place(t, sl, base, ties - 0.5, 0.0, &near, [&](uint32_t, float x) { return key_of(x) == low ? 1.0 : 0.0; });
        if (threadIdx.x < t.C) t.peer(threadIdx.x)->cut[1] = p + shift + 1u;
    }
    t.sync();
    return Kept{low, s.cut[1]};
}

template <class T>
__global__ void __launch_bounds__(SM_THREADS, 2)
k_sample(const __grid_constant__ b200bpe_logits in, const __grid_constant__ b200bpe_choice how, uint32_t vocab) {
    extern __shared__ __align__(16) float buf[];
    __shared__ Shared s;
    Team t(s);
    cg::cluster_group cluster = cg::this_cluster();
    const Slice sl = slice_of<T>(in, vocab, buf);
    const int shift = (int)sl.lo - (int)sl.lead;
    load_slice<T, true>(in, vocab, sl);
    cluster.barrier_arrive();        // (nobody writes into a CTA that has not begun)

    // the largest x, and the lowest token that has it
    Best best{-INFINITY, 0xFFFFFFFFu};
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        if (x.x > best.x) best = {x.x, p + shift};
        if (x.y > best.x) best = {x.y, p + 1 + shift};
        if (x.z > best.x) best = {x.z, p + 2 + shift};
        if (x.w > best.x) best = {x.w, p + 3 + shift};
    });
    for (int turn = 0; turn < 2; turn++) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float x = __shfl_xor_sync(0xFFFFFFFFu, best.x, o);
            const uint32_t at = __shfl_xor_sync(0xFFFFFFFFu, best.at, o);
            if (x > best.x || (x == best.x && at < best.at)) best = {x, at};
        }
        if (turn == 0) {
            if (t.lane == 0) s.best_warp[t.warp] = best;
            __syncthreads();
            best = s.best_warp[t.lane % SM_WARPS];
        }
    }
    cluster.barrier_wait();
    if (threadIdx.x < t.C) t.peer(threadIdx.x)->best_cta[t.rank] = best;
    const float temperature = how.temperature ? how.temperature[sl.row] : 1.0f;
    const bool greedy = !how.uniform || !(temperature >= SM_GREEDY_BELOW);
    const uint32_t top_k = greedy || !how.top_k ? 0u : how.top_k[sl.row];
    const float top_p = greedy || !how.top_p ? 1.0f : how.top_p[sl.row], min_p = greedy || !how.min_p ? 0.0f : how.min_p[sl.row];
    const bool by_k = top_k != 0u && top_k < vocab, by_p = top_p < 1.0f;
    if (by_k || by_p)
        for (uint32_t i = threadIdx.x; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0u;
    t.sync();
    best = s.best_cta[0];
    for (uint32_t c = 1; c < t.C; c++)
        if (s.best_cta[c].x > best.x) best = s.best_cta[c];
    if (best.x == -INFINITY) {          // (the whole cluster)
        if (t.rank == 0 && threadIdx.x == 0) {
            how.tokens_out[sl.row] = B200BPE_NO_TOKEN;
            if (how.logprobs_out) how.logprobs_out[sl.row] = -INFINITY;
        }
        return;
    }
    const double warm = greedy ? 1.0 : fmin((double)temperature, 3.4e38);
    const Weights w{best.x, (float)(1.4426950408889634 / warm), 1.0 / warm};
    // (what weighs less than e^-32 does not matter to top_p; it may to top_k, where a temperature is low)
    const Bins k_bins(best.x, fmax(32.0 * warm, 24.0)), p_bins(best.x, 32.0 * warm);

    // all weights; and the bins: of tokens for top_k, of weights for top_p
    double all = 0, spread = 0;
    each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
        const float v[4] = {x.x, x.y, x.z, x.w};
        float e[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            y[k] = w.power(v[k]);
            e[k] = Weights::two_to(y[k]);
            if (by_k) {
                const uint32_t b = k_bins.of(v[k]);
                if (b < SM_BINS - 1) atomicAdd(&s.bins[b], 1u);
            } else if (by_p) {
                const uint32_t b = p_bins.of(v[k]);
                if (b < SM_BINS - 1) atomicAdd(&s.bins[b], p_bins.weight_of(v[k], b));
            }
        }
        all += (double)((e[0] + e[1]) + (e[2] + e[3]));
        spread -= (double)((e[0] * y[0] + e[1] * y[1]) + (e[2] * y[2] + e[3] * y[3]));
    });
    t.total(all, spread);
    const double margin = 2.0 * (3.6e-7 * all + 1.25e-7 * spread);

    Kept kept{LOWEST_KEY, 0u};
    if (greedy) {
        if (t.rank == 0 && threadIdx.x == 0) {
            how.tokens_out[sl.row] = best.at;
            if (how.logprobs_out) how.logprobs_out[sl.row] = (float)-log(all);
        }
        return;
    }
    if (by_k) kept = border<false>(t, sl, w, k_bins, (double)top_k, -1.0, 0.0);
    if (by_p) {
        double whole = all, none = 0;
        if (by_k) {
            // weights of the top_k alone, in 64 bits; their bins
            whole = kept_mass<true>(sl, t.warp, w, kept);
            for (uint32_t i = threadIdx.x; i < SM_BINS; i += SM_THREADS) s.bins[i] = 0u;
            __syncthreads();
            each_four(sl, t.warp, [&](uint32_t p, const float4& x) {
                const float v[4] = {x.x, x.y, x.z, x.w};
                for (int k = 0; k < 4; k++) {
                    const uint32_t b = p_bins.of(v[k]);
                    if (b < SM_BINS - 1) atomicAdd(&s.bins[b], p_bins.weight_of(v[k], b));
                }
            });
            t.total(whole, none);
        }
        const double share = fmax((double)top_p, 0.0);
        Kept k{key_of(best.x), best.at + 1u};
        if (share > 0.0) k = border<true>(t, sl, w, p_bins, share * whole, by_k ? -1.0 : share, margin);
        if (k.key > kept.key || (k.key == kept.key && k.end < kept.end)) kept = k;
    }
    if (min_p > 0.0f) {
        const double least = (double)best.x + log((double)fminf(min_p, 1.0f)) * warm;
        const uint32_t from = key_of(__double2float_ru(least) + 0.0f);
        if (from > kept.key) kept = {from, 0xFFFFFFFFu};
    }

    // the draw
    const float u = how.uniform[sl.row];
    const double draw = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
    auto chosen = [&](auto exact, uint32_t* place) {         // whether this CTA has the token; -1: some sum was near
        constexpr bool EXACT = decltype(exact)::value;
        double mass = kept_mass<EXACT>(sl, t.warp, w, kept), none = 0;
        t.total(mass, none);
        const double target = draw * mass;
        double base = 0;
        uint32_t owner = 0xFFFFFFFFu, filled = 0;
        for (uint32_t c = 0; c < t.C && owner == 0xFFFFFFFFu; c++) {
            if (t.part(0, c) > 0) filled = c;
            if (base + t.part(0, c) > target) owner = c;
            else base += t.part(0, c);
        }
        if (owner == 0xFFFFFFFFu) {
            owner = filled;
            base = 0;
            for (uint32_t c = 0; c < owner; c++) base += t.part(0, c);
        }
        if (t.rank == owner) {
            bool near;
            *place = find_place(t, sl, base, target, EXACT ? 0.0 : margin, &near, [&](uint32_t p, float x) {
                return kept.has(x, p + shift) ? (EXACT ? w.exact(x) : (double)w.quick(x)) : 0.0;
            });
            if (!EXACT && threadIdx.x < t.C) t.peer(threadIdx.x)->cut[0] = near;
        }
        if (!EXACT) t.sync();
        return t.rank == owner;
    };
    uint32_t place = 0;
    bool mine = chosen(std::false_type{}, &place);
    if (s.cut[0]) mine = chosen(std::true_type{}, &place);
    if (mine && threadIdx.x == 0) {
        how.tokens_out[sl.row] = place + shift;
        if (how.logprobs_out) how.logprobs_out[sl.row] = (float)(w.log_of(buf[place]) - log(all));
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
    if (vocab_size == 0 || vocab_size > SM_MAX_VOCAB) return refused("b200bpe_sampler_create: 1 to 425,984 tokens");
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
