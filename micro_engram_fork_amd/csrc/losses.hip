// Losses over the rows of a decoder's logits and their gradients: log-probabilities of given tokens, distillation
// from a teacher's top logits, a preference loss over paired log ratios and a clipped policy loss with a KL term.
//
// Per row x of `vocab` logits, with z = x / temperature:
//   m = max z, s = sum exp(z - m), q = exp(z - m) / s, log-probability of token t = z_t - m - log s
// and every loss here has a row gradient of the form  dx = c (e_t - q)  or, for distillation,  w T (a' q - p) with
// other values at the teacher's few tokens. So all of them are two sweeps over the row: one for (m, s), one that
// writes the gradient, and a few values per row in between. Everything per row and per batch is held in fp32 (losses
// over rows are added in fp64: terms of both signs cancel there, and there are few); bf16 logits are widened exactly
// and a bf16 gradient is rounded once, when it is stored.
//
// Exponents are taken of (x - max x) / temperature, the difference first: a row that holds the type's lowest value
// everywhere then has probabilities 1 / vocab as it should, where x / temperature alone would be minus infinity.
// Logits of minus infinity have probability 0; a row of nothing but minus infinity, and one that holds plus infinity
// or NaN, gives NaN as its definition does.
//
// Rows that do not count (a target that is ignored or no token, a mask) are not read at all: what they hold cannot
// reach the loss, and their gradient is zeros.
#include "me_common.h"

#include <cmath>
#include <cstring>

namespace me {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kMaxSplits = 64;      // parts of a row whose (m, s) one wavefront joins, a lane each
constexpr int kMaxSpan = 32768;     // logits of one part
constexpr int kMaxTop = 1024;       // teacher entries of a row

// Where the logits are: row r at x + (r / rows_per_batch) * batch_stride + (r % rows_per_batch) * row_stride elements.
struct Logits {
    const void *x;
    int64_t n, rows_per_batch, batch_stride, row_stride;
    int32_t vocab;

    __device__ __forceinline__ int64_t offset(int64_t r) const {
        const int64_t b = r / rows_per_batch;
        return b * batch_stride + (r - b * rows_per_batch) * row_stride;
    }
};

// The tokens of the rows, and which rows count: a target in [0, vocab) that is not the ignored one, a mask that is set.
struct Tokens {
    const void *targets;  // [n] int32 / int64, or null
    const uint8_t *mask;  // [n], or null
    int64_t ignore;
    int is64;

    __device__ __forceinline__ int64_t at(int64_t r) const {
        return is64 ? static_cast<const int64_t *>(targets)[r] : static_cast<const int32_t *>(targets)[r];
    }
    // the row's token, or -1 where the row does not count
    __device__ __forceinline__ int32_t token(int64_t r, int32_t vocab) const {
        const int64_t t = at(r);
        return t >= 0 && t < vocab && t != ignore ? static_cast<int32_t>(t) : -1;
    }
    __device__ __forceinline__ bool counts(int64_t r, int32_t vocab) const {
        if (mask != nullptr && mask[r] == 0) return false;
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
        const int64_t v = is64 ? static_cast<const int64_t *>(offsets)[s] : static_cast<const int32_t *>(offsets)[s];
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

template <typename T>
struct Raw8;  // 8 logits as loaded
template <>
struct Raw8<uint16_t> {
    u32x4_v w;
};
template <>
struct Raw8<float> {
    f32x4_v lo, hi;
};

template <bool kNt>
__device__ __forceinline__ void load_raw(const uint16_t *p, Raw8<uint16_t> &r) {
    const auto q = reinterpret_cast<const __attribute__((address_space(1))) u32x4_e2 *>(as_global(p));
    if constexpr (kNt) r.w = __builtin_nontemporal_load(q);
    else r.w = *q;
}
template <bool kNt>
__device__ __forceinline__ void load_raw(const float *p, Raw8<float> &r) {
    const auto q = reinterpret_cast<const __attribute__((address_space(1))) f32x4_e4 *>(as_global(p));
    const auto h = reinterpret_cast<const __attribute__((address_space(1))) f32x4_e4 *>(as_global(p + 4));
    if constexpr (kNt) {
        r.lo = __builtin_nontemporal_load(q);
        r.hi = __builtin_nontemporal_load(h);
    } else {
        r.lo = *q;
        r.hi = *h;
    }
}
__device__ __forceinline__ void widen(const Raw8<uint16_t> &r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(r.w[e] << 16);
        v[2 * e + 1] = __uint_as_float(r.w[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ void widen(const Raw8<float> &r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = r.lo[e];
        v[4 + e] = r.hi[e];
    }
}
__device__ __forceinline__ float load1(const uint16_t *p) { return bf16_bits_to_float(*as_global(p)); }
__device__ __forceinline__ float load1(const float *p) { return *as_global(p); }

// 8 logits from element j, minus infinity past the end of the row
template <typename T>
__device__ __forceinline__ void load8_tail(const T *row, int32_t j, int32_t vocab, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = j + e < vocab ? load1(row + j + e) : -kInf;
}

__device__ __forceinline__ void store1(uint16_t *p, float f) { *as_global(p) = float_to_bf16_bits_rne(f); }
__device__ __forceinline__ void store1(float *p, float f) { *as_global(p) = f; }
__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    u32x4_v w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = static_cast<uint32_t>(float_to_bf16_bits_rne(v[2 * e])) |
               (static_cast<uint32_t>(float_to_bf16_bits_rne(v[2 * e + 1])) << 16);
    *reinterpret_cast<__attribute__((address_space(1))) u32x4_e2 *>(as_global(p)) = w;
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    *reinterpret_cast<__attribute__((address_space(1))) f32x4_e4 *>(as_global(p)) = f32x4_v{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<__attribute__((address_space(1))) f32x4_e4 *>(as_global(p + 4)) = f32x4_v{v[4], v[5], v[6], v[7]};
}

// ------------------------------------------------------------------------------------------ (m, s) pairs
// m: the logit that exponents are taken from (the largest one seen, or a guess near it), s: sum of exp2((x - m) k) with
// k = log2(e) / temperature.
struct MaxSum {
    float m, s;
};

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
// is then added up again by add_values, whose m is the running maximum: sums over 2^100 or NaN, where a wrong guess would
// lose digits also those under 2^-60, and guesses so large that m k could overflow.
struct Guess {
    float m, mk;
    bool fits;
};

__device__ __forceinline__ Guess guess_of(float m, float k) { return {m, m * k, fabsf(m) <= 1e30f}; }

__device__ __forceinline__ float guessed_exp(float x, const Guess &g, float k) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, k, -g.mk));
}

// m k is rounded once; this takes that rounding out of a sum
__device__ __forceinline__ float without_rounding(float s, const Guess &g, float k) {
    return s * __builtin_amdgcn_exp2f(-__builtin_fmaf(g.m, k, -g.mk));
}

__device__ __forceinline__ float sum8(const float (&v)[8], const Guess &g, float k) {
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = guessed_exp(v[i], g, k);
    return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
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
#pragma unroll
    for (int w = N / 2; w > 0; w /= 2) {
#pragma unroll
        for (int e = 0; e < w; ++e) part[e] += part[e + w];
    }
    a.s = a.s * exp2_of(a.m, ref, k) + part[0];
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
__device__ T block_sum(T v, T *slots) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    T sum = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) sum += slots[w];
    return sum;
}

// ------------------------------------------------------------------------------------------ weights of the rows
enum Reduction { kMean = 0, kSum = 1, kSequence = 2 };

struct WeightArgs {
    Tokens tokens;
    Seqs seqs;         // read where use_seqs: rows of no sequence do not count
    const void *ids;   // teacher ids [n, top] or null: a row without one in the vocabulary does not count
    float *weight;     // [n]; null: this workgroup is not launched
    float *counted;    // [1]: how many rows count
    int64_t n;
    int32_t vocab, top;
    int ids64, use_seqs, reduction;
};

__device__ __forceinline__ int32_t teacher_id(const void *ids, int is64, int64_t at, int32_t vocab) {
    const int64_t v = is64 ? static_cast<const int64_t *>(ids)[at] : static_cast<const int32_t *>(ids)[at];
    return v >= 0 && v < vocab ? static_cast<int32_t>(v) : -1;
}

__device__ __forceinline__ bool row_counts(const WeightArgs &a, int64_t r) {
    if (!a.tokens.counts(r, a.vocab)) return false;
    if (a.ids != nullptr) {
        for (int32_t i = 0; i < a.top; ++i)  // the first entry is one almost always
            if (teacher_id(a.ids, a.ids64, r * a.top + i, a.vocab) >= 0) return true;
        return false;
    }
    return true;
}

// weight [n]: 1 over the rows that count (kMean), 1 (kSum), or 1 over the row's sequence's counting rows and the
// sequences that have any (kSequence); 0 for the others. One workgroup: it runs beside the rows' own ones.
__device__ void make_weights(const WeightArgs &a) {
    __shared__ double slots[16];
    const int tid = threadIdx.x, threads = blockDim.x;
    int64_t total = 0;
    if (!a.use_seqs) {
        for (int64_t r = tid; r < a.n; r += threads) total += row_counts(a, r);
        total = static_cast<int64_t>(block_sum(static_cast<double>(total), slots));
        const float w = a.reduction == kSum ? 1.0f : 1.0f / static_cast<float>(total > 0 ? total : 1);
        for (int64_t r = tid; r < a.n; r += threads) a.weight[r] = row_counts(a, r) ? w : 0.0f;
        if (tid == 0) *a.counted = static_cast<float>(total);
        return;
    }
    for (int64_t r = tid; r < a.n; r += threads) a.weight[r] = 0.0f;
    __syncthreads();
    int64_t filled = 0;  // sequences with a counting row, seen by each wavefront's first lane
    const int lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
    for (int64_t s = wave; s < a.seqs.n_seqs; s += waves) {
        const int64_t from = a.seqs.begin(s), to = a.seqs.begin(s + 1);
        int64_t mine = 0;
        for (int64_t r = from + lane; r < to; r += 64) mine += row_counts(a, r);
        mine = wave_sum(mine);
        if (lane == 0) {
            filled += mine > 0;
            total += mine;
        }
        if (a.reduction == kSequence && mine > 0) {
            for (int64_t r = from + lane; r < to; r += 64)
                if (row_counts(a, r)) a.weight[r] = 1.0f / static_cast<float>(mine);
        } else if (mine > 0) {
            for (int64_t r = from + lane; r < to; r += 64)
                if (row_counts(a, r)) a.weight[r] = 1.0f;
        }
    }
    const double all = block_sum(static_cast<double>(total), slots);
    const double some = block_sum(static_cast<double>(filled), slots);
    if (tid == 0) *a.counted = static_cast<float>(all);
    if (a.reduction == kSum) return;
    const double by = a.reduction == kSequence ? some : all;
    const float scale = 1.0f / static_cast<float>(by > 0 ? by : 1);
    for (int64_t r = tid; r < a.n; r += threads) a.weight[r] *= scale;
}

// ------------------------------------------------------------------------------------------ statistics of row parts
struct StatsArgs {
    Logits logits;
    Tokens tokens;
    const void *ids;  // teacher ids [n, top] to leave out of the sums (null: none)
    MaxSum *part;     // [n, splits]
    WeightArgs weights;
    float k;          // log2(e) / temperature
    int32_t splits, span, top;
    int ids64;
};

// (m, s) of one part of a row per workgroup: bound by the bytes of the logits. Four 16-byte loads per thread are in
// flight before the first is used. The workgroup past the last part makes the rows' weights meanwhile.
template <typename T, int kThreads, bool kLeaveOut>
__global__ __launch_bounds__(kThreads) void stats_kernel(const StatsArgs a) {
    const int64_t parts = a.logits.n * a.splits;
    if (blockIdx.x == parts) {
        make_weights(a.weights);
        return;
    }
    const int64_t row = blockIdx.x / a.splits;
    const int32_t part = static_cast<int32_t>(blockIdx.x - row * a.splits);
    const int32_t vocab = a.logits.vocab, tid = threadIdx.x;
    if (!a.tokens.counts(row, vocab)) return;
    const int32_t from = part * a.span, to = min(vocab, from + a.span);
    __shared__ uint32_t left_out[kLeaveOut ? kMaxSpan / 32 : 1];
    if constexpr (kLeaveOut) {
        for (int32_t i = tid; i < (to - from + 31) / 32; i += kThreads) left_out[i] = 0;
        __syncthreads();
        for (int32_t i = tid; i < a.top; i += kThreads) {
            const int32_t id = teacher_id(a.ids, a.ids64, row * a.top + i, vocab);
            if (id >= from && id < to) atomicOr(&left_out[(id - from) >> 5], 1u << ((id - from) & 31));
        }
        __syncthreads();
    }
    const T *x = static_cast<const T *>(a.logits.x) + a.logits.offset(row);
    float near = kInf;  // no guess
    if (a.tokens.targets != nullptr) {
        near = load1(x + a.tokens.token(row, vocab));
    } else {
        const int32_t id = teacher_id(a.ids, a.ids64, row * a.top, vocab);
        if (id >= 0) near = load1(x + id);
    }
    const Guess guess = guess_of(near, a.k);
    const auto leave_out = [&](float (&v)[8], int32_t j) {
        if constexpr (kLeaveOut) {
            const int32_t at = j - from;
            const uint32_t bits = (left_out[at >> 5] >> (at & 31)) & 0xff;
            if (bits != 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (bits >> e & 1) v[e] = -kInf;
            }
        }
    };
    const int32_t whole = (to - from) / 8;  // spans are multiples of 8: only the row's end has a rest
    const auto sweep = [&](auto take) {
        int32_t c = tid;
        for (; c + 3 * kThreads < whole; c += 4 * kThreads) {
            Raw8<T> raw[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_raw<true>(x + from + 8 * (c + u * kThreads), raw[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float v[8];
                widen(raw[u], v);
                leave_out(v, from + 8 * (c + u * kThreads));
                take(v);
            }
        }
        for (; c < whole; c += kThreads) {
            Raw8<T> raw;
            load_raw<true>(x + from + 8 * c, raw);
            float v[8];
            widen(raw, v);
            leave_out(v, from + 8 * c);
            take(v);
        }
        if (from + 8 * whole < to && tid == whole % kThreads) {
            float v[8];
            load8_tail(x, from + 8 * whole, vocab, v);
            leave_out(v, from + 8 * whole);
            take(v);
        }
    };
    __shared__ float sums[kThreads / 64];
    __shared__ MaxSum joined[kThreads / 64];
    if (guess.fits) {
        float sum = 0.0f;
        sweep([&](float (&v)[8]) { sum += sum8(v, guess, a.k); });
        sum = wave_sum(sum);
        if constexpr (kThreads > 64) {
            if ((tid & 63) == 0) sums[tid >> 6] = sum;
            __syncthreads();
            sum = sums[0];
            for (int w = 1; w < kThreads / 64; ++w) sum += sums[w];
        }
        if (sum < kLargestSum && (!kLeaveOut || sum > kSmallestSum)) {
            if (tid == 0) a.part[blockIdx.x] = {guess.m, without_rounding(sum, guess, a.k)};
            return;
        }
    }
    MaxSum acc = {-kInf, 0.0f};
    sweep([&](float (&v)[8]) { add_values<8>(acc, v, a.k); });
    acc = wave_join(acc, a.k);
    if constexpr (kThreads > 64) {
        if ((tid & 63) == 0) joined[tid >> 6] = acc;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kThreads / 64; ++w) acc = join(acc, joined[w], a.k);
        }
    }
    if (tid == 0) a.part[blockIdx.x] = acc;
}

// ------------------------------------------------------------------------------------------ per-row values
enum Op { kLogps, kPreference, kPolicy, kDistill };

struct RowArgs {
    Logits logits;
    Tokens tokens;
    Seqs seqs;
    const MaxSum *part;    // [n, splits]
    const float *weight;   // [n] (policy, distillation)
    const float *counted;  // [1]
    float2 *stats;         // [n] (m, 1 / s): what the gradient needs (distillation: (m, a), see distill_row)
    float *logps;          // [n] (nullable)
    float *coef;           // [n] (nullable): the gradient's factor of the row
    float *gap;            // [n] preference: log-probability above the reference's
    const float *old_logps, *ref_logps, *advantages;
    const void *ids, *teacher;
    const float *teacher_lse;
    float *fix;            // [n, top]: the gradient at the teacher's tokens before the row's factor
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

// exp(d) - 1 - d without the cancellation of small d
__device__ __forceinline__ float exp_excess(float d) { return expm1f(d) - d; }

// The policy loss of one row and its derivative by the log-probability, both before the row's weight.
__device__ __forceinline__ void policy_terms(const RowArgs &a, int64_t r, float logp, float &loss, float &slope, float &kl,
                                             bool &clipped) {
    const float adv = a.advantages[a.adv_per_seq ? a.seqs.of(r) : r];
    const float ratio = expf(logp - a.old_logps[r]);
    const float held = fminf(fmaxf(ratio, 1.0f - a.clip_low), 1.0f + a.clip_high);
    const float free_term = ratio * adv, held_term = held * adv;
    clipped = free_term > held_term;
    loss = -(clipped ? held_term : free_term);
    slope = clipped ? 0.0f : -free_term;
    kl = 0.0f;
    if (a.ref_logps != nullptr) {
        const float d = a.ref_logps[r] - logp;
        kl = exp_excess(d);
        loss += a.kl_coef * kl;
        slope -= a.kl_coef * expm1f(d);
    }
}

// Teacher entry i of row r, scaled; minus infinity where its id is no token.
__device__ __forceinline__ float teacher_at(const RowArgs &a, int64_t r, int32_t i) {
    const int64_t at = r * a.top + i;
    return (a.teacher_bf16 ? load1(static_cast<const uint16_t *>(a.teacher) + at)
                           : load1(static_cast<const float *>(a.teacher) + at)) * a.inv_temp;
}

// One row of the distillation loss by one wavefront, lane i of it for the teacher's entries i, i + 64, ... `seen` are
// the (m, s) of the row: of all its tokens, or (teacher_lse given) of those that are no entry. Entries with the same id are one token
// whose probabilities add up; the first of them stands for all in the sums. Leaves (m, a) in stats so that the
// gradient at a token that is no entry is  weight T a exp2((x - m) k), and in fix the factors at the entries.
__device__ float distill_row(const RowArgs &a, int64_t r, int64_t off, bool bf16, MaxSum seen, int32_t *id, float *prob) {
    const int lane = threadIdx.x & 63;
    const bool rest = a.teacher_lse != nullptr;
    float top = -kInf;
    for (int32_t i = lane; i < a.top; i += 64) {
        id[i] = teacher_id(a.ids, a.ids64, r * a.top + i, a.logits.vocab);
        prob[i] = id[i] >= 0 ? teacher_at(a, r, i) : -kInf;
        top = fmaxf(top, prob[i]);
    }
    top = wave_max(top);
    float sum = 0.0f, log_norm;  // log of what the entries' exponentials are divided by
    if (rest) {
        log_norm = a.teacher_lse[r];
    } else {
        for (int32_t i = lane; i < a.top; i += 64) sum += id[i] >= 0 ? expf(prob[i] - top) : 0.0f;
        sum = wave_sum(sum);
        log_norm = logf(sum);
    }
    const float ref = rest ? 0.0f : top;
    for (int32_t i = lane; i < a.top; i += 64) {
        if (id[i] < 0) prob[i] = 0.0f;
        else prob[i] = rest ? expf(prob[i] - log_norm) : expf(prob[i] - ref) / sum;
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // the row's (m, s) over all tokens
    MaxSum all = seen;
    if (rest) {
        MaxSum mine = {-kInf, 0.0f};
        for (int32_t i = lane; i < a.top; i += 64) {
            bool first = id[i] >= 0;
            for (int32_t j = 0; j < i && first; ++j) first = id[j] != id[i];
            if (first) mine = join(mine, {row_logit(a.logits, off, id[i], bf16), 1.0f}, a.k);
        }
        all = join(seen, wave_join(mine, a.k), a.k);
    }
    const float log_s = logf(all.s), inv_s = 1.0f / all.s;
    float loss = 0.0f, mass = 0.0f;
    for (int32_t i = lane; i < a.top; i += 64) {
        if (id[i] < 0) {
            a.fix[r * a.top + i] = 0.0f;
            continue;
        }
        float p = 0.0f;
        bool first = true;
        for (int32_t j = 0; j < a.top; ++j) {
            if (id[j] == id[i]) {
                p += prob[j];
                first = first && j >= i;
            }
        }
        const float z = (row_logit(a.logits, off, id[i], bf16) - all.m) * a.inv_temp;
        a.fix[r * a.top + i] = expf(z) * inv_s - p;
        if (first) {
            mass += p;
            if (p > 0.0f || p != p) loss += p * (logf(p) - (z - log_s));
        }
    }
    loss = wave_sum(loss);
    float2 st = {all.m, inv_s};
    if (rest) {
        mass = wave_sum(mass);
        const float left = mass < 1.0f ? 1.0f - mass : mass == mass ? 0.0f : mass;
        // probability of the other tokens, as a logarithm: it does not vanish where the entries hold nearly all
        const float log_other = seen.m == -kInf ? -kInf : (seen.m - all.m) * a.inv_temp + logf(seen.s) - log_s;
        if (left > 0.0f || left != left) loss += left * (logf(left) - log_other);
        st = seen.m == -kInf ? float2{0.0f, 0.0f} : float2{seen.m, (expf(log_other) - left) / seen.s};
    }
    if (lane == 0) a.stats[r] = st;
    return loss * (a.temp * a.temp);
}

// A wavefront per row: joins the parts' (m, s), then the loss's own few values.
template <Op kOp, bool kBf16>
__global__ __launch_bounds__(kOp == kDistill ? 256 : 1024) void row_kernel(const RowArgs a) {
    constexpr int kWaves = kOp == kDistill ? 4 : 16;
    __shared__ int32_t id_all[kOp == kDistill ? kWaves * kMaxTop : 1];
    __shared__ float prob_all[kOp == kDistill ? kWaves * kMaxTop : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    RowSums sums;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWaves + wave; r < a.logits.n; r += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int32_t t = kOp == kDistill ? 0 : a.tokens.token(r, a.logits.vocab);
        const float weight = a.weight != nullptr ? a.weight[r] : 1.0f;
        if (t < 0 || (kOp >= kPolicy && weight == 0.0f)) {
            if (lane == 0) {
                if (a.logps != nullptr) a.logps[r] = 0.0f;
                if (a.coef != nullptr) a.coef[r] = 0.0f;
                if (a.gap != nullptr) a.gap[r] = 0.0f;
                if (a.stats != nullptr) a.stats[r] = {0.0f, 0.0f};
            }
            if (kOp == kDistill && a.fix != nullptr)
                for (int32_t i = lane; i < a.top; i += 64) a.fix[r * a.top + i] = 0.0f;
            continue;
        }
        const int64_t off = a.logits.offset(r);
        MaxSum row = {-kInf, 0.0f};
        if (lane < a.splits) row = a.part[r * a.splits + lane];
        row = wave_join(row, a.k);
        if constexpr (kOp == kDistill) {
            const float loss = distill_row(a, r, off, kBf16, row, id_all + wave * kMaxTop, prob_all + wave * kMaxTop);
            if (lane == 0) {
                a.coef[r] = a.scale * weight * a.temp;
                sums.loss += static_cast<double>(loss) * weight;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else if (lane == 0) {
            const float logp = (row_logit(a.logits, off, t, kBf16) - row.m) * a.inv_temp - logf(row.s);
            if (a.stats != nullptr) a.stats[r] = {row.m, 1.0f / row.s};
            if (a.logps != nullptr) a.logps[r] = logp;
            if constexpr (kOp == kPreference) {
                a.gap[r] = logp - a.ref_logps[r];
                a.coef[r] = 0.0f;
            } else if constexpr (kOp == kPolicy) {
                float loss, slope, kl;
                bool clipped;
                policy_terms(a, r, logp, loss, slope, kl, clipped);
                a.coef[r] = a.scale * weight * slope * a.inv_temp;
                sums.loss += static_cast<double>(loss) * weight;
                sums.kl += kl;
                sums.clipped += clipped;
            }
        }
    }
    if constexpr (kOp >= kPolicy) {
        __shared__ double slots[kWaves];
        const double loss = block_sum(sums.loss, slots), kl = block_sum(sums.kl, slots), clipped = block_sum(sums.clipped, slots);
        if (threadIdx.x == 0) {
            if (gridDim.x > 1) {
                a.sums[3 * blockIdx.x] = loss;
                a.sums[3 * blockIdx.x + 1] = kl;
                a.sums[3 * blockIdx.x + 2] = clipped;
            } else {
                *a.loss = static_cast<float>(loss * a.scale);
                if (a.out_stats != nullptr) {
                    const float n = fmaxf(*a.counted, 1.0f);
                    a.out_stats[0] = static_cast<float>(kl / n);
                    a.out_stats[1] = static_cast<float>(clipped / n);
                }
            }
        }
    }
}

// Adds the workgroups' sums in a fixed order.
__global__ __launch_bounds__(256) void total_kernel(const double *sums, int64_t count, const float *counted, float scale,
                                                    float *loss, float *out_stats) {
    __shared__ double slots[4];
    double v[3] = {0, 0, 0};
    for (int64_t i = threadIdx.x; i < count; i += 256)
        for (int c = 0; c < 3; ++c) v[c] += sums[3 * i + c];
    for (int c = 0; c < 3; ++c) v[c] = block_sum(v[c], slots);
    if (threadIdx.x == 0) {
        *loss = static_cast<float>(v[0] * scale);
        if (out_stats != nullptr) {
            const float n = fmaxf(*counted, 1.0f);
            out_stats[0] = static_cast<float>(v[1] / n);
            out_stats[1] = static_cast<float>(v[2] / n);
        }
    }
}

// ------------------------------------------------------------------------------------------ preference pairs
enum PairLoss { kSigmoid = 0, kIpo = 1, kHinge = 2 };

struct PairArgs {
    Tokens tokens;
    Seqs seqs;             // 2 * pairs sequences: the chosen ones, then the rejected ones
    const float *gap;      // [n]
    float *coef;           // [n]
    float *chosen, *rejected, *loss;
    double *sums;          // [pairs]
    int64_t pairs;
    float beta, smoothing;
    int32_t vocab;
    int kind, normalized;
};

// log(1 + exp(-x)) without overflow
__device__ __forceinline__ float softplus_neg(float x) { return fmaxf(-x, 0.0f) + log1pf(expf(-fabsf(x))); }

// One pair by one wavefront: both sequences' sums, the loss, and the factors of their rows' gradients. Returns the loss.
__device__ double pair_terms(const PairArgs &a, int64_t p) {
    const int lane = threadIdx.x & 63;
    float d[2];
    int64_t from[2], to[2];
    float inv_len[2];
    for (int side = 0; side < 2; ++side) {
        const int64_t s = side == 0 ? p : a.pairs + p;
        from[side] = a.seqs.begin(s);
        to[side] = a.seqs.begin(s + 1);
        double sum = 0;  // up to thousands of terms of either sign
        int64_t count = 0;
        for (int64_t r = from[side] + lane; r < to[side]; r += 64) {
            sum += a.gap[r];
            if (a.normalized) count += a.tokens.token(r, a.vocab) >= 0;
        }
        sum = wave_sum(sum);
        count = wave_sum(count);
        inv_len[side] = a.normalized ? 1.0f / static_cast<float>(count > 0 ? count : 1) : 1.0f;
        d[side] = static_cast<float>(sum * inv_len[side]);
    }
    const float h = d[0] - d[1], x = a.beta * h;
    float loss, slope;
    if (a.kind == kSigmoid) {
        loss = (1.0f - a.smoothing) * softplus_neg(x) + a.smoothing * softplus_neg(-x);
        // 1 / (1 + e^-x) - (1 - smoothing), each side's small part kept: sigma(x) - 1 = -sigma(-x)
        const float up = 1.0f / (1.0f + expf(-x)), down = 1.0f / (1.0f + expf(x));
        slope = a.beta * (a.smoothing * up - (1.0f - a.smoothing) * down);
    } else if (a.kind == kIpo) {
        const float e = h - 0.5f / a.beta;
        loss = e * e;
        slope = 2.0f * e;
    } else {
        loss = fmaxf(1.0f - x, 0.0f);
        if (x != x) loss = x;
        slope = x < 1.0f ? -a.beta : 0.0f;
    }
    slope /= static_cast<float>(a.pairs);
    for (int side = 0; side < 2; ++side) {
        const float c = (side == 0 ? slope : -slope) * inv_len[side];
        for (int64_t r = from[side] + lane; r < to[side]; r += 64)
            if (a.tokens.token(r, a.vocab) >= 0) a.coef[r] = c;
    }
    if (lane == 0) {
        a.chosen[p] = a.beta * d[0];
        a.rejected[p] = a.beta * d[1];
    }
    return loss;
}

// A wavefront per pair; with one workgroup the mean as well, else the pairs' losses for total_kernel.
__global__ __launch_bounds__(1024) void pair_kernel(const PairArgs a) {
    __shared__ double slots[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    double sum = 0;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * waves + wave; p < a.pairs; p += static_cast<int64_t>(gridDim.x) * waves) {
        const double loss = pair_terms(a, p);
        if (lane == 0) sum += loss;
    }
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) {
        if (gridDim.x > 1) {
            a.sums[3 * blockIdx.x] = sum;
            a.sums[3 * blockIdx.x + 1] = a.sums[3 * blockIdx.x + 2] = 0;
        } else {
            *a.loss = static_cast<float>(sum / static_cast<double>(a.pairs > 0 ? a.pairs : 1));
        }
    }
}

// ------------------------------------------------------------------------------------------ gradient
struct GradArgs {
    Logits logits;
    Tokens tokens;          // targets null: distillation
    const float2 *stats;    // [n] (m, a)
    const float *coef;      // [n]
    const float *upstream;  // [1] (nullable: 1)
    const void *ids;
    const float *fix;       // [n, top]
    void *grad;             // [n, vocab]
    float k, extra;         // extra: factor on coef
    int32_t splits, span, top;
    int ids64, done_for_one;
};

// One part of a row per workgroup: streams the logits once more and writes the gradient; a copy's bytes, and bound
// by them. Rows whose factor is 0 are filled without being read.
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void grad_kernel(const GradArgs a) {
    const float up = a.upstream != nullptr ? *a.upstream : 1.0f;
    if (a.done_for_one && up == 1.0f) return;
    const int64_t row = blockIdx.x / a.splits;
    const int32_t part = static_cast<int32_t>(blockIdx.x - row * a.splits);
    const int32_t vocab = a.logits.vocab, tid = threadIdx.x;
    const bool distill = a.tokens.targets == nullptr;
    const int32_t t = distill ? -1 : a.tokens.token(row, vocab);
    const int32_t from = part * a.span, to = min(vocab, from + a.span);
    const int32_t whole = (to - from) / 8;
    T *g = static_cast<T *>(a.grad) + row * vocab;
    const float c = (distill || t >= 0) ? a.coef[row] * up * a.extra : 0.0f;
    if (c == 0.0f) {
        const float zeros[8] = {};
        for (int32_t i = tid; i < whole; i += kThreads) store8(g + from + 8 * i, zeros);
        if (tid < to - from - 8 * whole) store1(g + from + 8 * whole + tid, 0.0f);
        return;
    }
    const float2 st = a.stats[row];
    const float factor = distill ? c * st.y : -c * st.y;
    const T *x = static_cast<const T *>(a.logits.x) + a.logits.offset(row);
    const auto values = [&](const float (&v)[8], int32_t j, float (&d)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = factor * exp2_of(v[e], st.x, a.k);
        if (t >= j && t < j + 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (j + e == t) d[e] += c;
        }
    };
    int32_t i = tid;
    for (; i + 3 * kThreads < whole; i += 4 * kThreads) {
        Raw8<T> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_raw<false>(x + from + 8 * (i + u * kThreads), raw[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int32_t j = from + 8 * (i + u * kThreads);
            float v[8], d[8];
            widen(raw[u], v);
            values(v, j, d);
            store8(g + j, d);
        }
    }
    for (; i < whole; i += kThreads) {
        const int32_t j = from + 8 * i;
        Raw8<T> raw;
        load_raw<false>(x + j, raw);
        float v[8], d[8];
        widen(raw, v);
        values(v, j, d);
        store8(g + j, d);
    }
    if (tid < to - from - 8 * whole) {
        const int32_t j = from + 8 * whole + tid;
        store1(g + j, factor * exp2_of(load1(x + j), st.x, a.k) + (j == t ? c : 0.0f));
    }
    if (distill) {  // the teacher's tokens of this part, over what the sweep has stored there
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        for (int32_t e = tid; e < a.top; e += kThreads) {
            const int32_t id = teacher_id(a.ids, a.ids64, row * a.top + e, vocab);
            if (id >= from && id < to) store1(g + id, c * a.fix[row * a.top + e]);
        }
    }
}

// ------------------------------------------------------------------------------------------ host side
// Parts of a row: enough workgroups to fill the part (2048 of 256 threads are resident) for few rows, parts of
// at most kMaxSpan logits for many.
struct Split {
    int32_t splits, span;
};

Split split_of(int64_t n, int64_t vocab) {
    int64_t want = ceil_div(2048, n > 0 ? n : 1);
    if (want > kMaxSplits) want = kMaxSplits;
    int64_t span = ceil_div(ceil_div(vocab, want), 2048) * 2048;
    if (span > kMaxSpan) span = kMaxSpan;
    return {static_cast<int32_t>(ceil_div(vocab, span)), static_cast<int32_t>(span)};
}

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

int64_t row_blocks(Op op, int64_t n) {
    const int64_t per = op == kDistill ? 4 : 16;
    const int64_t blocks = ceil_div(n, per);
    return blocks <= 2 ? 1 : blocks < 2048 ? blocks : 2048;
}

// Workspace: parts, weights, row sums, counted.
struct Space {
    MaxSum *part;
    float *weight, *counted, *gap;
    double *sums;
    size_t bytes;
};

Space carve(void *base, int64_t n, int64_t vocab, int64_t pairs) {
    const Split s = split_of(n, vocab);
    uint8_t *p = static_cast<uint8_t *>(base);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        uint8_t *q = p + at;
        at += align_up(bytes);
        return q;
    };
    Space w;
    w.part = reinterpret_cast<MaxSum *>(take(static_cast<size_t>(n) * s.splits * sizeof(MaxSum)));
    w.weight = reinterpret_cast<float *>(take(static_cast<size_t>(n) * sizeof(float)));
    w.gap = reinterpret_cast<float *>(take(static_cast<size_t>(n) * sizeof(float)));
    const int64_t most = pairs > 2048 ? pairs : 2048;
    w.sums = reinterpret_cast<double *>(take(static_cast<size_t>(most) * 3 * sizeof(double)));
    w.counted = reinterpret_cast<float *>(take(sizeof(float)));
    w.bytes = at;
    return w;
}

int check_logits(const char *what, const Logits &l, int dtype) {
    ME_CHECK_ARG(dtype == ME_BF16 || dtype == ME_F32, "%s: logits must be bf16 or fp32", what);
    ME_CHECK_ARG(l.n >= 0 && l.n <= INT32_MAX, "%s: n out of range", what);
    ME_CHECK_ARG(l.vocab >= 1 && l.vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    ME_CHECK_ARG(l.n == 0 || l.x != nullptr, "%s: logits are null", what);
    ME_CHECK_ARG(l.rows_per_batch >= 1, "%s: rows_per_batch must be positive", what);
    ME_CHECK_ARG(l.row_stride >= 0 && l.batch_stride >= 0, "%s: negative strides", what);
    const Split s = split_of(l.n, l.vocab);
    ME_CHECK_ARG(l.n * s.splits < INT32_MAX, "%s: too many rows", what);
    return ME_OK;
}

int check_temperature(const char *what, double t) {
    ME_CHECK_ARG(t >= 1e-6 && t <= 1e6, "%s: temperature must be in 1e-6..1e6", what);
    return ME_OK;
}

int check_tokens(const char *what, const void *targets, int dtype, int64_t n) {
    ME_CHECK_ARG(n == 0 || targets != nullptr, "%s: targets are null", what);
    ME_CHECK_ARG(dtype == ME_I32 || dtype == ME_I64, "%s: targets must be int32 or int64", what);
    return ME_OK;
}

int check_seqs(const char *what, const void *offsets, int dtype, int64_t n_seqs, int64_t length, int64_t n) {
    ME_CHECK_ARG(n_seqs >= 0 && n_seqs <= INT32_MAX, "%s: n_seqs out of range", what);
    if (offsets != nullptr) {
        ME_CHECK_ARG(dtype == ME_I32 || dtype == ME_I64, "%s: sequence offsets must be int32 or int64", what);
    } else {
        ME_CHECK_ARG(length >= 0 && n_seqs * length == n, "%s: the sequences do not hold the rows", what);
    }
    return ME_OK;
}

template <typename T, int kThreads>
void launch_stats_of(const StatsArgs &a, bool left_out, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(a.logits.n * a.splits + (a.weights.weight != nullptr ? 1 : 0));
    if (blocks == 0) return;
    if (left_out) stats_kernel<T, kThreads, true><<<blocks, kThreads, 0, s>>>(a);
    else stats_kernel<T, kThreads, false><<<blocks, kThreads, 0, s>>>(a);
}

void launch_stats(const StatsArgs &a, int dtype, bool left_out, hipStream_t s) {
    const bool small = a.logits.vocab <= 2048;
    if (dtype == ME_BF16) {
        if (small) launch_stats_of<uint16_t, 64>(a, left_out, s);
        else launch_stats_of<uint16_t, 256>(a, left_out, s);
    } else {
        if (small) launch_stats_of<float, 64>(a, left_out, s);
        else launch_stats_of<float, 256>(a, left_out, s);
    }
}

template <Op kOp>
void launch_rows(const RowArgs &a, int dtype, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(row_blocks(kOp, a.logits.n));
    const int threads = kOp == kDistill ? 256 : 1024;
    if (dtype == ME_BF16) row_kernel<kOp, true><<<blocks, threads, 0, s>>>(a);
    else row_kernel<kOp, false><<<blocks, threads, 0, s>>>(a);
    if (kOp >= kPolicy && blocks > 1)
        total_kernel<<<1, 256, 0, s>>>(a.sums, blocks, a.counted, a.scale, a.loss, a.out_stats);
}

void launch_grad(const GradArgs &a, int dtype, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(a.logits.n * a.splits);
    if (blocks == 0) return;
    const bool small = a.logits.vocab <= 2048;
    if (dtype == ME_BF16) {
        if (small) grad_kernel<uint16_t, 64><<<blocks, 64, 0, s>>>(a);
        else grad_kernel<uint16_t, 256><<<blocks, 256, 0, s>>>(a);
    } else {
        if (small) grad_kernel<float, 64><<<blocks, 64, 0, s>>>(a);
        else grad_kernel<float, 256><<<blocks, 256, 0, s>>>(a);
    }
}

#define ME_TRY(call)                     \
    do {                                 \
        const int st_ = (call);          \
        if (st_ != ME_OK) return st_;    \
    } while (0)

int check_space(const char *what, const Space &w, const void *workspace, size_t bytes) {
    if (workspace == nullptr || bytes < w.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace == nullptr ? size_t{0} : bytes, w.bytes);
        return ME_ERR_WORKSPACE;
    }
    return ME_OK;
}

}  // namespace
}  // namespace me

using namespace me;

extern "C" int me_loss_workspace_size(int64_t n, int64_t vocab, int64_t pairs, size_t *bytes) {
    ME_CHECK_ARG(bytes != nullptr, "me_loss_workspace_size: bytes is null");
    ME_CHECK_ARG(n >= 0 && n <= INT32_MAX && pairs >= 0 && pairs <= INT32_MAX, "me_loss_workspace_size: size out of range");
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "me_loss_workspace_size: vocab must be in 1..%d", kMaxSpan * kMaxSplits);
    *bytes = carve(nullptr, n, vocab, pairs).bytes;
    return ME_OK;
}

extern "C" int me_token_logps(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                              int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                              int64_t ignore_index, double temperature, float *logps, float *row_stats,
                              void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "me_token_logps";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(n == 0 || logps != nullptr, "%s: logps is null", what);
    if (n == 0) return ME_OK;
    const Space w = carve(workspace, n, vocab, 0);
    ME_TRY(check_space(what, w, workspace, workspace_bytes));
    const hipStream_t s = as_stream(stream);
    const Split sp = split_of(n, vocab);
    StatsArgs st = {};
    st.logits = l;
    st.tokens = {targets, nullptr, ignore_index, targets_dtype == ME_I64};
    st.part = w.part;
    st.k = static_cast<float>(1.4426950408889634 / temperature);
    st.splits = sp.splits;
    st.span = sp.span;
    launch_stats(st, dtype, false, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.part = w.part;
    r.stats = reinterpret_cast<float2 *>(row_stats);
    r.logps = logps;
    r.k = st.k;
    r.inv_temp = static_cast<float>(1.0 / temperature);
    r.splits = sp.splits;
    launch_rows<kLogps>(r, dtype, s);
    return check_launch(what);
}

extern "C" int me_token_logps_backward(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                                       int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                                       int64_t ignore_index, double temperature, const float *row_stats,
                                       const float *coef, double coef_scale, const float *upstream, int done_for_one,
                                       void *grad, void *stream) {
    const char *what = "me_token_logps_backward";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(n == 0 || (row_stats != nullptr && coef != nullptr && grad != nullptr), "%s: null pointer", what);
    ME_CHECK_ARG(!done_for_one || upstream != nullptr, "%s: done_for_one needs upstream", what);
    const Split sp = split_of(n, vocab);
    GradArgs g = {};
    g.logits = l;
    g.tokens = {targets, nullptr, ignore_index, targets_dtype == ME_I64};
    g.stats = reinterpret_cast<const float2 *>(row_stats);
    g.coef = coef;
    g.upstream = upstream;
    g.grad = grad;
    g.k = static_cast<float>(1.4426950408889634 / temperature);
    g.extra = static_cast<float>(coef_scale);
    g.splits = sp.splits;
    g.span = sp.span;
    g.done_for_one = done_for_one;
    launch_grad(g, dtype, as_stream(stream));
    return check_launch(what);
}

extern "C" int me_preference(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                             int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                             int64_t ignore_index, const float *ref_logps, const void *seq_offsets, int offsets_dtype,
                             int64_t pairs, int64_t seq_len, int kind, double beta, double smoothing, int normalized,
                             float *loss, float *chosen, float *rejected, float *row_stats, float *coef,
                             void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "me_preference";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(pairs >= 0 && pairs < INT32_MAX / 2, "%s: pairs out of range", what);
    ME_TRY(check_seqs(what, seq_offsets, offsets_dtype, 2 * pairs, seq_len, n));
    ME_CHECK_ARG(kind >= kSigmoid && kind <= kHinge, "%s: unknown loss kind", what);
    ME_CHECK_ARG(beta > 0 && beta <= 1e6, "%s: beta must be positive", what);
    ME_CHECK_ARG(smoothing >= 0 && smoothing <= 1, "%s: smoothing must be in 0..1", what);
    ME_CHECK_ARG(loss != nullptr && (pairs == 0 || (chosen != nullptr && rejected != nullptr)), "%s: null output", what);
    ME_CHECK_ARG(n == 0 || (ref_logps != nullptr && coef != nullptr), "%s: null pointer", what);
    const Space w = carve(workspace, n, vocab, pairs);
    ME_TRY(check_space(what, w, workspace, workspace_bytes));
    const hipStream_t s = as_stream(stream);
    const Split sp = split_of(n, vocab);
    const Tokens tokens = {targets, nullptr, ignore_index, targets_dtype == ME_I64};
    const Seqs seqs = {seq_offsets, 2 * pairs, seq_len, n, offsets_dtype == ME_I64};
    if (n > 0) {
        StatsArgs st = {};
        st.logits = l;
        st.tokens = tokens;
        st.part = w.part;
        st.k = kLog2e;
        st.splits = sp.splits;
        st.span = sp.span;
        launch_stats(st, dtype, false, s);
        RowArgs r = {};
        r.logits = l;
        r.tokens = tokens;
        r.part = w.part;
        r.stats = reinterpret_cast<float2 *>(row_stats);
        r.coef = coef;
        r.gap = w.gap;
        r.ref_logps = ref_logps;
        r.k = kLog2e;
        r.inv_temp = 1.0f;
        r.splits = sp.splits;
        launch_rows<kPreference>(r, dtype, s);
    }
    PairArgs p = {};
    p.tokens = tokens;
    p.seqs = seqs;
    p.gap = w.gap;
    p.coef = coef;
    p.chosen = chosen;
    p.rejected = rejected;
    p.loss = loss;
    p.sums = w.sums;
    p.pairs = pairs;
    p.beta = static_cast<float>(beta);
    p.smoothing = static_cast<float>(smoothing);
    p.vocab = l.vocab;
    p.kind = kind;
    p.normalized = normalized;
    if (pairs <= 16) {
        pair_kernel<<<1, 1024, 0, s>>>(p);
    } else {
        const int64_t blocks = ceil_div(pairs, 4) < 2048 ? ceil_div(pairs, 4) : 2048;
        pair_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
        total_kernel<<<1, 256, 0, s>>>(w.sums, blocks, nullptr, 1.0f / static_cast<float>(pairs), loss, nullptr);
    }
    return check_launch(what);
}

extern "C" int me_policy(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                         int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                         int64_t ignore_index, const float *old_logps, const float *advantages, int adv_per_seq,
                         const float *ref_logps, const void *seq_offsets, int offsets_dtype, int64_t n_seqs,
                         int64_t seq_len, double clip_low, double clip_high, double kl_coef, double temperature,
                         double scale, int reduction, float *loss, float *logps, float *out_stats, float *row_stats,
                         float *coef, void *grad, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "me_policy";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_TRY(check_seqs(what, seq_offsets, offsets_dtype, n_seqs, seq_len, n));
    ME_CHECK_ARG(clip_low >= 0 && clip_high >= 0, "%s: clip bounds must not be negative", what);
    ME_CHECK_ARG(reduction >= kMean && reduction <= kSequence, "%s: unknown reduction", what);
    ME_CHECK_ARG(loss != nullptr && out_stats != nullptr, "%s: null output", what);
    ME_CHECK_ARG(n == 0 || (old_logps != nullptr && advantages != nullptr && logps != nullptr && coef != nullptr),
                 "%s: null pointer", what);
    ME_CHECK_ARG(grad == nullptr || n == 0 || row_stats != nullptr, "%s: grad needs row_stats", what);
    const Space w = carve(workspace, n, vocab, 0);
    ME_TRY(check_space(what, w, workspace, workspace_bytes));
    const hipStream_t s = as_stream(stream);
    const Split sp = split_of(n, vocab);
    StatsArgs st = {};
    st.logits = l;
    st.tokens = {targets, nullptr, ignore_index, targets_dtype == ME_I64};
    st.part = w.part;
    st.k = static_cast<float>(1.4426950408889634 / temperature);
    st.splits = sp.splits;
    st.span = sp.span;
    const Seqs seqs = {seq_offsets, n_seqs, seq_len, n, offsets_dtype == ME_I64};
    st.weights.tokens = st.tokens;
    st.weights.seqs = seqs;
    st.weights.weight = w.weight;
    st.weights.counted = w.counted;
    st.weights.n = n;
    st.weights.vocab = l.vocab;
    st.weights.use_seqs = seq_offsets != nullptr || reduction == kSequence;
    st.weights.reduction = reduction;
    launch_stats(st, dtype, false, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.seqs = seqs;
    r.part = w.part;
    r.weight = w.weight;
    r.counted = w.counted;
    r.stats = reinterpret_cast<float2 *>(row_stats);
    r.logps = logps;
    r.coef = coef;
    r.old_logps = old_logps;
    r.ref_logps = ref_logps;
    r.advantages = advantages;
    r.sums = w.sums;
    r.loss = loss;
    r.out_stats = out_stats;
    r.k = st.k;
    r.inv_temp = static_cast<float>(1.0 / temperature);
    r.scale = static_cast<float>(scale);
    r.clip_low = static_cast<float>(clip_low);
    r.clip_high = static_cast<float>(clip_high);
    r.kl_coef = static_cast<float>(kl_coef);
    r.splits = sp.splits;
    r.adv_per_seq = adv_per_seq;
    launch_rows<kPolicy>(r, dtype, s);
    if (grad != nullptr) {
        GradArgs g = {};
        g.logits = l;
        g.tokens = st.tokens;
        g.stats = r.stats;
        g.coef = coef;
        g.grad = grad;
        g.k = st.k;
        g.extra = 1.0f;
        g.splits = sp.splits;
        g.span = sp.span;
        launch_grad(g, dtype, s);
    }
    return check_launch(what);
}

extern "C" int me_distill(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                          int64_t batch_stride, int64_t row_stride, const void *teacher_ids, int ids_dtype,
                          const void *teacher, int teacher_dtype, int64_t top, const float *teacher_lse,
                          const uint8_t *mask, double temperature, double scale, int reduction, float *loss,
                          float *row_stats, float *coef, float *fix, void *grad, void *workspace,
                          size_t workspace_bytes, void *stream) {
    const char *what = "me_distill";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_temperature(what, temperature));
    ME_CHECK_ARG(ids_dtype == ME_I32 || ids_dtype == ME_I64, "%s: teacher ids must be int32 or int64", what);
    ME_CHECK_ARG(teacher_dtype == ME_BF16 || teacher_dtype == ME_F32, "%s: teacher logits must be bf16 or fp32", what);
    ME_CHECK_ARG(top >= 1 && top <= kMaxTop, "%s: top must be in 1..%d", what, kMaxTop);
    ME_CHECK_ARG(teacher_lse == nullptr || top < vocab, "%s: entries for every token leave no rest", what);
    ME_CHECK_ARG(reduction == kMean || reduction == kSum, "%s: unknown reduction", what);
    ME_CHECK_ARG(loss != nullptr, "%s: null output", what);
    ME_CHECK_ARG(n == 0 || (teacher_ids != nullptr && teacher != nullptr && row_stats != nullptr && coef != nullptr &&
                            fix != nullptr), "%s: null pointer", what);
    const Space w = carve(workspace, n, vocab, 0);
    ME_TRY(check_space(what, w, workspace, workspace_bytes));
    const hipStream_t s = as_stream(stream);
    const Split sp = split_of(n, vocab);
    StatsArgs st = {};
    st.logits = l;
    st.tokens = {nullptr, mask, 0, 0};
    st.ids = teacher_ids;
    st.ids64 = ids_dtype == ME_I64;
    st.top = static_cast<int32_t>(top);
    st.part = w.part;
    st.k = static_cast<float>(1.4426950408889634 / temperature);
    st.splits = sp.splits;
    st.span = sp.span;
    st.weights.tokens = st.tokens;
    st.weights.ids = teacher_ids;
    st.weights.ids64 = st.ids64;
    st.weights.top = st.top;
    st.weights.weight = w.weight;
    st.weights.counted = w.counted;
    st.weights.n = n;
    st.weights.vocab = l.vocab;
    st.weights.reduction = reduction;
    launch_stats(st, dtype, teacher_lse != nullptr, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.part = w.part;
    r.weight = w.weight;
    r.counted = w.counted;
    r.stats = reinterpret_cast<float2 *>(row_stats);
    r.coef = coef;
    r.ids = teacher_ids;
    r.ids64 = st.ids64;
    r.teacher = teacher;
    r.teacher_bf16 = teacher_dtype == ME_BF16;
    r.teacher_lse = teacher_lse;
    r.top = st.top;
    r.fix = fix;
    r.sums = w.sums;
    r.loss = loss;
    r.k = st.k;
    r.inv_temp = static_cast<float>(1.0 / temperature);
    r.temp = static_cast<float>(temperature);
    r.scale = static_cast<float>(scale);
    r.splits = sp.splits;
    launch_rows<kDistill>(r, dtype, s);
    if (grad != nullptr) {
        GradArgs g = {};
        g.logits = l;
        g.stats = r.stats;
        g.coef = coef;
        g.ids = teacher_ids;
        g.ids64 = st.ids64;
        g.fix = fix;
        g.top = st.top;
        g.grad = grad;
        g.k = st.k;
        g.extra = 1.0f;
        g.splits = sp.splits;
        g.span = sp.span;
        launch_grad(g, dtype, s);
    }
    return check_launch(what);
}

extern "C" int me_distill_backward(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                                   int64_t batch_stride, int64_t row_stride, const void *teacher_ids, int ids_dtype,
                                   int64_t top, double temperature, const float *row_stats, const float *coef,
                                   const float *fix, const float *upstream, int done_for_one, void *grad, void *stream) {
    const char *what = "me_distill_backward";
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMaxSpan * kMaxSplits, "%s: vocab must be in 1..%d", what, kMaxSpan * kMaxSplits);
    const Logits l = {logits, n, rows_per_batch, batch_stride, row_stride, static_cast<int32_t>(vocab)};
    ME_TRY(check_logits(what, l, dtype));
    ME_TRY(check_temperature(what, temperature));
    ME_CHECK_ARG(ids_dtype == ME_I32 || ids_dtype == ME_I64, "%s: teacher ids must be int32 or int64", what);
    ME_CHECK_ARG(top >= 1 && top <= kMaxTop, "%s: top must be in 1..%d", what, kMaxTop);
    ME_CHECK_ARG(n == 0 || (teacher_ids != nullptr && row_stats != nullptr && coef != nullptr && fix != nullptr &&
                            grad != nullptr), "%s: null pointer", what);
    ME_CHECK_ARG(!done_for_one || upstream != nullptr, "%s: done_for_one needs upstream", what);
    const Split sp = split_of(n, vocab);
    GradArgs g = {};
    g.logits = l;
    g.stats = reinterpret_cast<const float2 *>(row_stats);
    g.coef = coef;
    g.upstream = upstream;
    g.ids = teacher_ids;
    g.ids64 = ids_dtype == ME_I64;
    g.fix = fix;
    g.top = static_cast<int32_t>(top);
    g.grad = grad;
    g.k = static_cast<float>(1.4426950408889634 / temperature);
    g.extra = 1.0f;
    g.splits = sp.splits;
    g.span = sp.span;
    g.done_for_one = done_for_one;
    launch_grad(g, dtype, as_stream(stream));
    return check_launch(what);
}
