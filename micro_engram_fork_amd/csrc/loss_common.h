// What the kernels of the losses over logits share (losses.hip, loss_rows.hip).
#pragma once

#include "me_common.h"

#include <cmath>
#include <cstring>

namespace me {
namespace loss {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kMaxSplits = 64;      // parts of a row whose (m, s) one wavefront joins, a lane each
constexpr int kMaxSpan = 32768;     // logits of one part
constexpr int kMaxTop = 1024;       // teacher entries of a row

// Reads of memory that no thread of the kernel writes. At an address that all threads share they go through the scalar
// cache and wait for none of the vector loads that are under way (those return in the order of their issue).
template <typename T>
__device__ __forceinline__ T constant(const T *p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) T *>(reinterpret_cast<uint64_t>(p));
}
// element i of an int64 or int32 array
__device__ __forceinline__ int64_t constant_index(const void *p, int is64, int64_t i) {
    return is64 ? constant(static_cast<const int64_t *>(p) + i) : constant(static_cast<const int32_t *>(p) + i);
}
// 1- and 2-byte values by way of the whole 4 bytes that hold them
__device__ __forceinline__ uint32_t constant_bytes(const void *p) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return constant(reinterpret_cast<const uint32_t *>(at & ~uint64_t{3})) >> (8 * (at & 3));
}

// Where the logits are: row r at x + (r / rows_per_batch) * batch_stride + (r % rows_per_batch) * row_stride elements.
struct Logits {
    const void *x;
    int64_t n;                // at most INT32_MAX
    uint32_t rows_per_batch;
    int64_t batch_stride, row_stride;
    int32_t vocab;

    __device__ __forceinline__ int64_t offset(int64_t r) const {
        const uint32_t row = static_cast<uint32_t>(r), b = row / rows_per_batch;
        return b * batch_stride + (row - b * rows_per_batch) * row_stride;
    }
};

// The tokens of the rows, and which rows count: a target in [0, vocab) that is not the ignored one, a mask that is set.
struct Tokens {
    const void *targets;  // [n] int32 / int64, or null
    const uint8_t *mask;  // [n], or null
    int64_t ignore;
    int is64;

    __device__ __forceinline__ int64_t at(int64_t r) const {
        return constant_index(targets, is64, r);
    }
    // the row's token, or -1 where the row does not count
    __device__ __forceinline__ int32_t token(int64_t r, int32_t vocab) const {
        const int64_t t = at(r);
        return t >= 0 && t < vocab && t != ignore ? static_cast<int32_t>(t) : -1;
    }
    __device__ __forceinline__ bool counts(int64_t r, int32_t vocab) const {
        if (mask != nullptr && (constant_bytes(mask + r) & 0xff) == 0) return false;
        return targets == nullptr || token(r, vocab) >= 0;
    }
};

// Sequences of the rows: offsets [n_seqs + 1] (packed), or all of one length (offsets null). Offsets are clamped to
// the rows there are, so that no value of theirs reads or writes outside.
struct Seqs {
    const void *offsets;
    int64_t n_seqs, length, n;
    int is64;

    __device__ __forceinline__ int64_t begin(int64_t s) const {
        if (offsets == nullptr) return s * length;
        const int64_t v = constant_index(offsets, is64, s);
        return v < 0 ? 0 : v > n ? n : v;
    }
    // the sequence that holds row r, -1 if none does
    __device__ __forceinline__ int64_t of(int64_t r) const {
        if (offsets == nullptr) return length > 0 && r / length < n_seqs ? r / length : -1;
        int64_t lo = 0, hi = n_seqs;  // the last s with begin(s) <= r
        if (n_seqs == 0 || begin(0) > r) return -1;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (begin(mid) <= r) lo = mid;
            else hi = mid;
        }
        return r < begin(lo + 1) ? lo : -1;
    }
};

// ------------------------------------------------------------------------------------------ row access
// Rows may start at any element (an odd vocabulary, a view without its padding), so the 16-byte accesses are declared
// to need the element's alignment only; gfx950 takes them at any address.
typedef uint32_t u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));

// A row is worked on in units of 16 bytes, one per thread and load: neighbouring lanes then read neighbouring units.
template <typename T>
constexpr int kVec = 16 / sizeof(T);

template <typename T>
struct Raw;  // a unit as loaded
template <>
struct Raw<uint16_t> {
    u32x4_v w;
};
template <>
struct Raw<float> {
    f32x4_v w;
};

// kStream: past the caches (non-temporal), for rows that are read or written once
template <bool kStream>
__device__ __forceinline__ void load_raw(const uint16_t *p, Raw<uint16_t> &r) {
    const auto q = reinterpret_cast<const __attribute__((address_space(1))) u32x4_e2 *>(as_global(p));
    if constexpr (kStream) r.w = __builtin_nontemporal_load(q);
    else r.w = *q;
}
template <bool kStream>
__device__ __forceinline__ void load_raw(const float *p, Raw<float> &r) {
    const auto q = reinterpret_cast<const __attribute__((address_space(1))) f32x4_e4 *>(as_global(p));
    if constexpr (kStream) r.w = __builtin_nontemporal_load(q);
    else r.w = *q;
}
__device__ __forceinline__ void widen(const Raw<uint16_t> &r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(r.w[e] << 16);
        v[2 * e + 1] = __uint_as_float(r.w[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ void widen(const Raw<float> &r, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r.w[e];
}
// values back into the form of loaded fp32 logits
__device__ __forceinline__ void keep_raw(Raw<float> &r, const float (&v)[4]) { r.w = f32x4_v{v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ float load1(const uint16_t *p) { return bf16_bits_to_float(*as_global(p)); }
__device__ __forceinline__ float load1(const float *p) { return *as_global(p); }

// N logits from element j, minus infinity past the end of the row
template <typename T, int N>
__device__ __forceinline__ void load_tail(const T *row, int32_t j, int32_t vocab, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = j + e < vocab ? load1(row + j + e) : -kInf;
}

__device__ __forceinline__ void store1(uint16_t *p, float f) { *as_global(p) = float_to_bf16_bits_rne(f); }
__device__ __forceinline__ void store1(float *p, float f) { *as_global(p) = f; }
template <bool kStream>
__device__ __forceinline__ void store_unit(uint16_t *p, const float (&v)[8]) {
    u32x4_v w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = static_cast<uint32_t>(float_to_bf16_bits_rne(v[2 * e])) |
               (static_cast<uint32_t>(float_to_bf16_bits_rne(v[2 * e + 1])) << 16);
    const auto q = reinterpret_cast<__attribute__((address_space(1))) u32x4_e2 *>(as_global(p));
    if constexpr (kStream) __builtin_nontemporal_store(u32x4_e2(w), q);
    else *q = w;
}
template <bool kStream>
__device__ __forceinline__ void store_unit(float *p, const float (&v)[4]) {
    const auto q = reinterpret_cast<__attribute__((address_space(1))) f32x4_e4 *>(as_global(p));
    const f32x4_v w = {v[0], v[1], v[2], v[3]};
    if constexpr (kStream) __builtin_nontemporal_store(f32x4_e4(w), q);
    else *q = w;
}

template <int N>
__device__ __forceinline__ float tree_sum(const float (&e)[N]) {
    if constexpr (N == 4) return (e[0] + e[1]) + (e[2] + e[3]);
    else return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
}

// ------------------------------------------------------------------------------------------ (m, s) pairs
// m: the logit that exponents are taken from (the largest one seen, or a guess near it), s: sum of exp2((x - m) k) with
// k = log2(e) / temperature.
struct MaxSum {
    float m, s;
};

// one logit; a NaN is put in s, as m goes through fmaxf, which drops it
__device__ __forceinline__ MaxSum pair_of(float x) { return {x, x == x ? 1.0f : x}; }

// exp2((x - m) k); v_exp_f32 is within one unit in the last place and takes minus infinity to 0
__device__ __forceinline__ float exp2_of(float x, float m, float k) { return __builtin_amdgcn_exp2f((x - m) * k); }

__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float k) {
    const float m = fmaxf(a.m, b.m);
    if (m == -kInf) return {m, a.s + b.s};  // nothing but minus infinity so far (a NaN stays in s)
    return {m, a.s * exp2_of(a.m, m, k) + b.s * exp2_of(b.m, m, k)};
}

// The usual way to the sum: m is a guess (the logit of the row's own token, or of a teacher's entry, which no other
// exceeds by more than e^60 in a model that is any good), so nothing is compared or rescaled and each logit takes one
// multiply-add, one exponential and one addition. What the guess cannot serve shows in the sum (and in m itself), and
// is then added up again by add_values, whose m is the running maximum: sums over 2^100 or NaN, where a wrong guess
// would lose digits also those under 2^-60, and guesses so large that the rounding of m k (2^-5 at 1e6), which
// without_rounding takes out, would come near a factor.
struct Guess {
    float m, mk;
    bool fits;
};

__device__ __forceinline__ Guess guess_of(float m, float k) { return {m, m * k, fabsf(m * k) <= 1e6f}; }

__device__ __forceinline__ float guessed_exp(float x, const Guess &g, float k) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, k, -g.mk));
}

// m k is rounded once; this takes that rounding out of a sum
__device__ __forceinline__ float without_rounding(float s, const Guess &g, float k) {
    return s * __builtin_amdgcn_exp2f(-__builtin_fmaf(g.m, k, -g.mk));
}

template <int N>
__device__ __forceinline__ float guessed_sum(const float (&v)[N], const Guess &g, float k) {
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = guessed_exp(v[i], g, k);
    return tree_sum(e);
}

constexpr float kLargestSum = 0x1p100f, kSmallestSum = 0x1p-60f;

template <int N>
__device__ __forceinline__ void add_values(MaxSum &a, const float (&v)[N], float k) {
    float top = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, v[e]);
    const float m = fmaxf(a.m, top);
    const float ref = m == -kInf ? 0.0f : m;
    float part[N];
#pragma unroll
    for (int e = 0; e < N; ++e) part[e] = exp2_of(v[e], ref, k);
    a.s = a.s * exp2_of(a.m, ref, k) + tree_sum(part);
    a.m = m;
}

__device__ __forceinline__ MaxSum wave_join(MaxSum a, float k) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) a = join(a, {__shfl_xor(a.m, off), __shfl_xor(a.s, off)}, k);
    return a;
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}

// Sum of v over the workgroup's wavefronts, in their order; every thread gets it. `slots`: one per wavefront.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T *slots) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    T sum = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) sum += slots[w];
    return sum;
}

__device__ __forceinline__ int32_t teacher_id(const void *ids, int is64, int64_t at, int32_t vocab) {
    const int64_t v = constant_index(ids, is64, at);
    return v >= 0 && v < vocab ? static_cast<int32_t>(v) : -1;
}

// ------------------------------------------------------------------------------------------ weights of the rows
enum Reduction { kMean = 0, kSum = 1, kSequence = 2 };

struct WeightArgs {
    Tokens tokens;
    Seqs seqs;         // read where use_seqs: rows of no sequence do not count
    const void *ids;   // teacher ids [n, top] or null: a row without one in the vocabulary does not count
    float *weight;     // [n]: 0 where a row does not count; else its share of its sequence (kSequence), or 1
    float *counted;    // [2]: how many rows count, and the factor on weight; null: nothing is weighted
    int64_t n;
    int32_t vocab, top;
    int ids64, use_seqs, reduction;
};

__device__ __forceinline__ bool row_counts(const WeightArgs &a, int64_t r) {
    if (!a.tokens.counts(r, a.vocab)) return false;
    if (a.ids != nullptr) {
        for (int32_t i = 0; i < a.top; ++i)  // the first entry is one almost always
            if (teacher_id(a.ids, a.ids64, r * a.top + i, a.vocab) >= 0) return true;
        return false;
    }
    return true;
}

// The weight of row r once make_weights has run: 0 where it does not count.
__device__ __forceinline__ float row_weight(const WeightArgs &a, int64_t r) {
    return constant(a.weight + r) * constant(a.counted + 1);
}

// ------------------------------------------------------------------------------------------ per-row values
enum Op { kLogps, kPreference, kPolicy, kDistill };

struct RowArgs {
    Logits logits;
    Tokens tokens;
    Seqs seqs;
    const MaxSum *part;    // [n, splits]
    WeightArgs weights;    // policy, distillation
    float4 *stats;         // [n] what the gradient needs: (m, 1 / s, 1 - q of the token, -), for distillation
                           // (m, a, -, -) as of distill_finish
    float *logps;          // [n] (nullable)
    float *coef;           // [n] (nullable): the gradient's factor of the row
    float *gap;            // [n] preference: log-probability above the reference's
    const float *old_logps, *ref_logps, *advantages;
    const void *ids, *teacher;
    const float *teacher_lse;
    float *fix;            // [n, top]: the gradient at the teacher's tokens before the row's factor
    int32_t *entry_id;     // for the one-read kernel: [n, top] the entries' tokens and the logits there, [n] the
    float *entry_x, *near; // largest of these; the tokens' probabilities are in fix until it writes that
    double *sums;          // [gridDim, 3]
    float *loss, *out_stats;
    float k, inv_temp, temp, scale, clip_low, clip_high, kl_coef;
    int32_t splits, top;
    int ids64, teacher_bf16, adv_per_seq;
};

struct RowSums {
    double loss = 0, kl = 0, clipped = 0;
};

__device__ __forceinline__ float row_logit(const Logits &l, int64_t off, int32_t j, bool bf16) {
    return bf16 ? load1(static_cast<const uint16_t *>(l.x) + off + j) : load1(static_cast<const float *>(l.x) + off + j);
}

// exp(d) - 1 - d: for small d, where d is nearly all of exp(d) - 1, by its series (the first term left out is 5e-8 of the
// sum at 0.5); infinite for an infinite d.
__device__ __forceinline__ float exp_excess(float d) {
    if (fabsf(d) < 0.5f) {
        const float tail = 1.0f + d * (1.0f / 3) * (1.0f + d * (1.0f / 4) * (1.0f + d * (1.0f / 5) * (1.0f + d * (1.0f / 6) *
                           (1.0f + d * (1.0f / 7) * (1.0f + d * (1.0f / 8))))));
        return 0.5f * d * d * tail;
    }
    return fabsf(d) == kInf ? kInf : expm1f(d) - d;
}

// A row's token against all others. `others` is the (m, s) of these alone, so that a log-probability near 0 and the
// 1 - q of the gradient there keep their digits: log(1 + u) for the others' weight u over the token's.
struct TokenTerms {
    float logp, rest;  // rest: 1 - q
    MaxSum all;        // (m, s) of the whole row
};

__device__ __forceinline__ TokenTerms token_terms(float xt, MaxSum others, float k, float inv_temp) {
    TokenTerms v;
    const float d = (others.m - xt) * inv_temp;
    if (d > 0.0f) v.logp = -(d + logf(others.s + expf(-d)));
    else v.logp = -log1pf(others.s * expf(d));
    if (xt == kInf) v.logp = __builtin_nanf("");  // infinity over infinity
    v.rest = -expm1f(v.logp);
    v.all = join(others, pair_of(xt), k);
    return v;
}

// What the policy loss takes of a row besides its log-probability.
struct Sampled {
    float old_logp, ref_logp, advantage;
};

__device__ __forceinline__ Sampled sampled_row(const RowArgs &a, int64_t r) {
    Sampled v;
    v.old_logp = constant(a.old_logps + r);
    v.ref_logp = a.ref_logps != nullptr ? constant(a.ref_logps + r) : 0.0f;
    v.advantage = constant(a.advantages + (a.adv_per_seq ? max(a.seqs.of(r), int64_t{0}) : r));
    return v;
}

// The policy loss of one row and its derivative by the log-probability, both before the row's weight.
__device__ __forceinline__ void policy_terms(const RowArgs &a, const Sampled &v, float logp, float &loss, float &slope,
                                             float &kl, bool &clipped) {
    const float ratio = expf(logp - v.old_logp);
    const float held = fminf(fmaxf(ratio, 1.0f - a.clip_low), 1.0f + a.clip_high);
    // an advantage of 0 makes no term of a ratio past fp32 either (a NaN stays one)
    const float free_term = v.advantage == 0.0f && ratio == kInf ? 0.0f : ratio * v.advantage;
    const float held_term = held * v.advantage;
    clipped = free_term > held_term;
    loss = -(clipped ? held_term : free_term);
    slope = clipped ? 0.0f : -free_term;
    kl = 0.0f;
    if (a.ref_logps != nullptr) {
        const float d = v.ref_logp - logp;
        kl = exp_excess(d);
        if (a.kl_coef != 0.0f) {  // a coefficient of 0 makes no term of a value past fp32 either
            loss += a.kl_coef * kl;
            slope -= a.kl_coef * expm1f(d);
        }
    }
}

// Teacher entry i of row r, scaled; minus infinity where its id is no token.
__device__ __forceinline__ float teacher_at(const RowArgs &a, int64_t r, int32_t i) {
    const int64_t at = r * a.top + i;
    return (a.teacher_bf16 ? load1(static_cast<const uint16_t *>(a.teacher) + at)
                           : load1(static_cast<const float *>(a.teacher) + at)) * a.inv_temp;
}

// A row's teacher entries, in LDS. p: the probability of the entry's token, which adds up the entries of one token;
// its sign bit is set on all of these but the first, which stands for the token in sums. Ids that are no token are -1,
// with p = 0.
struct Entries {
    int32_t *id;
    float *x;     // the row's logit at the token
    float *p;
    float *raw;   // scratch; after distill_finish the gradient's value at the token before the row's factor
};

constexpr int kEntryBytes = 16;

// Each array has room for a multiple of 4 entries, so that the ids can be read four at a time.
__host__ __device__ __forceinline__ int32_t entry_room(int32_t top) { return (top + 3) / 4 * 4; }

__device__ __forceinline__ Entries entries_at(void *lds, int32_t top) {
    const int32_t room = entry_room(top);
    Entries e;
    e.id = static_cast<int32_t *>(lds);
    e.x = reinterpret_cast<float *>(e.id + room);
    e.p = e.x + room;
    e.raw = e.p + room;
    return e;
}

// LDS written by some lanes of a wavefront and read by others of it: a wavefront's LDS accesses complete in order, so
// only the compiler has to keep them so.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One wavefront fills the entries of row r (lane i the entries i, i + 64, ...).
static __device__ void distill_entries(const RowArgs &a, int64_t r, int64_t off, bool bf16, const Entries &e) {
    const int lane = threadIdx.x & 63;
    const bool rest = a.teacher_lse != nullptr;
    const float lse = rest ? a.teacher_lse[r] : 0.0f;
    float top = -kInf;
    for (int32_t i = lane; i < a.top; i += 64) {
        const int32_t id = teacher_id(a.ids, a.ids64, r * a.top + i, a.logits.vocab);
        const float t = id >= 0 ? teacher_at(a, r, i) : -kInf;
        e.id[i] = id;
        e.raw[i] = t;
        e.x[i] = id >= 0 ? row_logit(a.logits, off, id, bf16) : -kInf;
        top = fmaxf(top, t);
    }
    top = rest ? lse : wave_max(top);
    float sum = 0.0f;
    for (int32_t i = lane; i < a.top; i += 64) {
        const float w = e.id[i] >= 0 ? expf(e.raw[i] - top) : 0.0f;
        e.raw[i] = w;
        sum += w;
    }
    const float norm = rest ? 1.0f : wave_sum(sum);
    if (lane < entry_room(a.top) - a.top) e.id[a.top + lane] = -1;
    wave_lds_order();
    for (int32_t i = lane; i < a.top; i += 64) {
        const int32_t id = e.id[i];
        float p = e.raw[i];
        bool first = true;
        if (id >= 0) {
            for (int32_t j0 = 0; j0 < a.top; j0 += 4) {  // entries of the same token, which there hardly ever are
                const int4 four = *reinterpret_cast<const int4 *>(e.id + j0);
                if (four.x == id || four.y == id || four.z == id || four.w == id) {
                    for (int32_t j = j0; j < j0 + 4; ++j) {
                        if (j == i || e.id[j] != id) continue;
                        p += e.raw[j];
                        first = first && j > i;
                    }
                }
            }
        }
        p = id >= 0 ? p / norm : 0.0f;
        e.p[i] = first ? fabsf(p) : -fabsf(p);  // a NaN may have come with a sign of its own
    }
    wave_lds_order();
}

// The loss of row r before its weight, by a wavefront. `seen` are the (m, s) of the row: of all its tokens, or
// (teacher_lse given) of those that are no entry. Leaves in stats (m, a) such that the gradient at a token that is no
// entry is  weight T a exp2((x - m) k), and in raw (and where `write`, fix) the gradient at the entries over weight T.
static __device__ float distill_finish(const RowArgs &a, int64_t r, MaxSum seen, const Entries &e, float4 &stats,
                                       bool write) {
    const int lane = threadIdx.x & 63;
    const bool rest = a.teacher_lse != nullptr;
    MaxSum all = seen;  // the row's (m, s) over all tokens
    if (rest) {
        MaxSum mine = {-kInf, 0.0f};
        for (int32_t i = lane; i < a.top; i += 64)
            if (e.id[i] >= 0 && !__builtin_signbitf(e.p[i])) mine = join(mine, pair_of(e.x[i]), a.k);
        all = join(seen, wave_join(mine, a.k), a.k);
    }
    const float log_s = logf(all.s), inv_s = 1.0f / all.s;
    float loss = 0.0f, mass = 0.0f;
    for (int32_t i = lane; i < a.top; i += 64) {
        float fix = 0.0f;
        if (e.id[i] >= 0) {
            const bool first = !__builtin_signbitf(e.p[i]);
            const float p = fabsf(e.p[i]), z = (e.x[i] - all.m) * a.inv_temp;
            fix = expf(z) * inv_s - p;
            if (first) {
                mass += p;
                if (!(p <= 0.0f)) loss += p * (logf(p) - (z - log_s));
            }
        }
        e.raw[i] = fix;
        if (write) a.fix[r * a.top + i] = fix;
    }
    loss = wave_sum(loss);
    stats = {all.m, inv_s, 0.0f, 0.0f};
    if (rest) {
        mass = wave_sum(mass);
        const float left = mass < 1.0f ? 1.0f - mass : mass == mass ? 0.0f : mass;
        // probability of the other tokens, as a logarithm: it does not vanish where the entries hold nearly all
        const float log_other = seen.m == -kInf ? -kInf : (seen.m - all.m) * a.inv_temp + logf(seen.s) - log_s;
        if (!(left <= 0.0f)) loss += left * (logf(left) - log_other);
        stats = seen.m == -kInf ? float4{0.0f, 0.0f, 0.0f, 0.0f}
                                : float4{seen.m, (expf(log_other) - left) / seen.s, 0.0f, 0.0f};
    }
    wave_lds_order();
    return loss * (a.temp * a.temp);
}


// ------------------------------------------------------------------------------------------ host side
#define ME_TRY(call)                     \
    do {                                 \
        const int st_ = (call);          \
        if (st_ != ME_OK) return st_;    \
    } while (0)

}  // namespace loss

// loss_rows.hip: whether rows of this size and number take its one-read kernels, and their launch (stream_rows: past
// the caches)
bool takes_row_pass(int64_t n, int64_t vocab, int dtype, int64_t top, bool with_grad);
void launch_row_pass(loss::Op op, const loss::RowArgs &a, int dtype, void *grad, bool stream_rows, hipStream_t s);
}  // namespace me
