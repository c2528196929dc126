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
#include "loss_common.h"

namespace me {

using namespace loss;

namespace {

// The weight of a row: 1 over the rows that count (kMean), 1 (kSum), or 1 over the row's sequence's counting rows
// and the sequences that have any (kSequence); 0 for a row that does not count. Made by one workgroup, bound by the
// latency of its loads, hence eight of them in flight per thread: 5.7-6.1 us alone for 8192 rows, 7.6-8.7 for 3885
// in 5 sequences, a wavefront each.
template <typename I>
__device__ int64_t count_rows(const WeightArgs &a) {
    const bool of_ids = a.ids != nullptr;
    const I *key = static_cast<const I *>(of_ids ? a.ids : a.tokens.targets);
    const int64_t stride = of_ids ? a.top : 1, ignore = of_ids ? -1 : a.tokens.ignore;
    int64_t total = 0;
    for (int64_t r0 = threadIdx.x; r0 < a.n; r0 += 8 * static_cast<int64_t>(blockDim.x)) {
        I v[8];
        uint8_t in[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {  // eight loads in flight
            const int64_t r = r0 + u * static_cast<int64_t>(blockDim.x), at = r < a.n ? r : a.n - 1;
            v[u] = key[at * stride];
            in[u] = a.tokens.mask != nullptr ? a.tokens.mask[at] : 1;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t r = r0 + u * static_cast<int64_t>(blockDim.x);
            bool counts = r < a.n && in[u] != 0;
            if (counts && !(v[u] >= 0 && v[u] < a.vocab && v[u] != ignore)) counts = of_ids && row_counts(a, r);
            total += counts;
            if (r < a.n) a.weight[r] = counts ? 1.0f : 0.0f;
        }
    }
    return total;
}

__device__ void make_weights(const WeightArgs &a) {
    __shared__ double slots[16];
    const int tid = threadIdx.x, threads = blockDim.x;
    int64_t total = 0;
    if (!a.use_seqs) {
        total = (a.ids != nullptr ? a.ids64 : a.tokens.is64) ? count_rows<int64_t>(a) : count_rows<int32_t>(a);
        total = static_cast<int64_t>(block_sum(static_cast<double>(total), slots));
        if (tid == 0) {
            a.counted[0] = static_cast<float>(total);
            a.counted[1] = a.reduction == kSum ? 1.0f : 1.0f / static_cast<float>(total > 0 ? total : 1);
        }
        return;
    }
    if (a.seqs.offsets != nullptr) {  // rows of no sequence
        for (int64_t r = tid; r < a.n; r += threads) a.weight[r] = 0.0f;
        __syncthreads();
    }
    int64_t filled = 0;  // sequences with a counting row, seen by each wavefront's first lane
    const int lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
    constexpr int kFlight = 8;
    for (int64_t s = wave; s < a.seqs.n_seqs; s += waves) {
        const int64_t from = a.seqs.begin(s), to = a.seqs.begin(s + 1);
        int64_t mine = 0;
        for (int64_t r0 = from + lane; r0 < to; r0 += 64 * kFlight) {
            int32_t t[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) t[u] = a.tokens.token(min(r0 + 64 * u, to - 1), a.vocab);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) mine += r0 + 64 * u < to && t[u] >= 0;
        }
        mine = wave_sum(mine);
        if (lane == 0) {
            filled += mine > 0;
            total += mine;
        }
        const float w = a.reduction == kSequence && mine > 0 ? 1.0f / static_cast<float>(mine) : 1.0f;
        for (int64_t r0 = from + lane; r0 < to; r0 += 64 * kFlight) {
            int32_t t[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) t[u] = a.tokens.token(min(r0 + 64 * u, to - 1), a.vocab);
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (r0 + 64 * u < to) a.weight[r0 + 64 * u] = t[u] >= 0 ? w : 0.0f;
        }
    }
    const double all = block_sum(static_cast<double>(total), slots);
    const double some = block_sum(static_cast<double>(filled), slots);
    if (tid == 0) {
        const double by = a.reduction == kSequence ? some : all;
        a.counted[0] = static_cast<float>(all);
        a.counted[1] = a.reduction == kSum ? 1.0f : 1.0f / static_cast<float>(by > 0 ? by : 1);
    }
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

// (m, s) of one part of a row per workgroup, of all its tokens but the row's own (or but the teacher's entries). Bound
// by the bytes of the logits: the rows of 8 x 511 with a target, 1.6 GB of bf16 logits, take 231 us, 7.0 TB/s (a device
// copy of 4 GB moves 4.9, a fill 6.8). For that the loads go past the caches (262 us otherwise), four 16-byte ones
// (fp32: eight) per thread are in flight, and a logit costs one multiply-add, one exponential and one addition (Guess).
// The workgroup past the last part makes the rows' weights: beside the others where all are resident at one time (2048
// of 256 threads), behind them in larger grids.
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
    int32_t t = -1;
    if (a.tokens.targets != nullptr) {
        t = a.tokens.token(row, vocab);
        near = load1(x + t);
    } else {
        const int32_t id = teacher_id(a.ids, a.ids64, row * a.top, vocab);
        if (id >= 0) near = load1(x + id);
    }
    const Guess guess = guess_of(near, a.k);
    constexpr int N = kVec<T>;
    // v: unit `first` + lane of this part, whose logits the sum leaves out where they are entries' or the row's own
    // token's (which token_terms adds). Only the wavefront that holds the token looks at single lanes for it (every
    // lane at every unit: 380 us instead of 231).
    const int32_t lane = tid & 63;
    const auto leave_out = [&](float (&v)[N], int32_t first) {
        if constexpr (kLeaveOut) {
            const int32_t at = N * (first + lane);
            const uint32_t bits = (left_out[at >> 5] >> (at & 31)) & ((1u << N) - 1);
            if (bits != 0) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (bits >> e & 1) v[e] = -kInf;
            }
        } else {
            const uint32_t ahead = static_cast<uint32_t>(t - from - N * first);
            if (ahead < 64 * N) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (static_cast<uint32_t>(N * lane + e) == ahead) v[e] = -kInf;
            }
        }
    };
    const int32_t whole = (to - from) / N;  // spans are whole units: only the row's end has a rest
    constexpr int kUnroll = sizeof(T) == 2 ? 4 : 8;  // loads in flight per thread
    const auto sweep = [&](auto take) {
        int32_t first = __builtin_amdgcn_readfirstlane(tid & ~63);  // unit of this wavefront's first lane
        for (; first + 63 + (kUnroll - 1) * kThreads < whole; first += kUnroll * kThreads) {
            Raw<T> raw[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) load_raw<true>(x + from + N * (first + lane + u * kThreads), raw[u]);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float v[N];
                widen(raw[u], v);
                leave_out(v, first + u * kThreads);
                take(v);
            }
        }
        for (; first < whole; first += kThreads) {
            if (first + lane < whole) {
                Raw<T> raw;
                load_raw<true>(x + from + N * (first + lane), raw);
                float v[N];
                widen(raw, v);
                leave_out(v, first);
                take(v);
            }
        }
        if (from + N * whole < to && tid == whole % kThreads) {
            float v[N];
            load_tail(x, from + N * whole, vocab, v);
            leave_out(v, whole - lane);
            take(v);
        }
    };
    __shared__ float sums[kThreads / 64];
    __shared__ MaxSum joined[kThreads / 64];
    if (guess.fits) {
        float sum = 0.0f;
        sweep([&](float (&v)[N]) { sum += guessed_sum(v, guess, a.k); });
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
    sweep([&](float (&v)[N]) { add_values(acc, v, a.k); });
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

// A wavefront per row: joins the parts' (m, s), then the loss's own few values. A chain of a few dependent loads per
// row, whatever its length: 3.1 us for one row, 5.4-5.6 for 4088, 8.2-8.6 for 8286.
template <Op kOp, bool kBf16>
__global__ __launch_bounds__(kOp == kDistill ? 256 : 1024) void row_kernel(const RowArgs a) {
    constexpr int kWaves = kOp == kDistill ? 4 : 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t entry_space[];  // distillation: its entries per wavefront
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWaves;
    RowSums sums;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWaves + wave; r < a.logits.n; r += step) {
        const int32_t t = kOp == kDistill ? 0 : a.tokens.token(r, a.logits.vocab);
        const float weight = kOp >= kPolicy ? row_weight(a.weights, r) : 1.0f;
        if (t < 0 || (kOp >= kPolicy && weight == 0.0f)) {
            if (lane == 0) {
                if (a.logps != nullptr) a.logps[r] = 0.0f;
                if (a.coef != nullptr) a.coef[r] = 0.0f;
                if (a.gap != nullptr) a.gap[r] = 0.0f;
                if (a.stats != nullptr) a.stats[r] = {0.0f, 0.0f, 0.0f, 0.0f};
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
            const Entries e = entries_at(entry_space + wave * kEntryBytes * entry_room(a.top), a.top);
            distill_entries(a, r, off, kBf16, e);
            float4 stats;
            const float loss = distill_finish(a, r, row, e, stats, true);
            if (lane == 0) {
                a.stats[r] = stats;
                a.coef[r] = a.scale * weight * a.temp;
                sums.loss += static_cast<double>(loss) * weight;
            }
            wave_lds_order();
        } else if (lane == 0) {
            const TokenTerms token = token_terms(row_logit(a.logits, off, t, kBf16), row, a.k, a.inv_temp);
            const float logp = token.logp;
            if (a.stats != nullptr) a.stats[r] = {token.all.m, 1.0f / token.all.s, token.rest, 0.0f};
            if (a.logps != nullptr) a.logps[r] = logp;
            if constexpr (kOp == kPreference) {
                a.gap[r] = logp - a.ref_logps[r];
                if (a.coef != nullptr) a.coef[r] = 0.0f;
            } else if constexpr (kOp == kPolicy) {
                float loss, slope, kl;
                bool clipped;
                policy_terms(a, sampled_row(a, r), logp, loss, slope, kl, clipped);
                a.coef[r] = a.scale * weight * slope * a.inv_temp;
                sums.loss += static_cast<double>(loss) * weight;
                sums.kl += kl;
                sums.clipped += clipped;
            }
        }
    }
    if constexpr (kOp >= kPolicy) {
        __shared__ double slots[kWaves];
        const double loss = block_sum(sums.loss, slots), kl = block_sum(sums.kl, slots);
        const double clipped = block_sum(sums.clipped, slots);
        if (threadIdx.x == 0) {
            if (gridDim.x > 1) {
                a.sums[3 * blockIdx.x] = loss;
                a.sums[3 * blockIdx.x + 1] = kl;
                a.sums[3 * blockIdx.x + 2] = clipped;
            } else {
                *a.loss = static_cast<float>(loss * a.scale);
                if (a.out_stats != nullptr) {
                    const float n = fmaxf(*a.weights.counted, 1.0f);
                    a.out_stats[0] = static_cast<float>(kl / n);
                    a.out_stats[1] = static_cast<float>(clipped / n);
                }
            }
        }
    }
}

// The weights alone, before a kernel that needs them.
__global__ __launch_bounds__(1024) void weights_kernel(const WeightArgs a) { make_weights(a); }

// The teacher's entries of every row for the one-read kernel, a wavefront per row; the last workgroup makes the
// weights. Apart from that kernel because there a row's chain of ids, logits at them and their sums would be waited
// for by a whole CU (about 17 us of a row's 75 there; all of 4096 rows of 64 entries take 19 us here).
template <bool kBf16>
__global__ __launch_bounds__(256) void entries_kernel(const RowArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t entry_space[];
    if (blockIdx.x == gridDim.x - 1) {
        make_weights(a.weights);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (r >= a.logits.n || !row_counts(a.weights, r)) return;
    const Entries e = entries_at(entry_space + wave * kEntryBytes * entry_room(a.top), a.top);
    distill_entries(a, r, a.logits.offset(r), kBf16, e);
    float near = -kInf;
    for (int32_t i = lane; i < a.top; i += 64) {
        near = fmaxf(near, e.x[i]);
        a.fix[r * a.top + i] = e.p[i];
        a.entry_x[r * a.top + i] = e.x[i];
        a.entry_id[r * a.top + i] = e.id[i];
    }
    near = wave_max(near);
    if (lane == 0) a.near[r] = near;
}

// Adds the workgroups' or rows' sums in a fixed order. One workgroup, bound by the latency of its loads: with four rows
// in flight per thread three sums of 8192 rows take 6.7-7.0 us, one after the other 12.2.
template <int kParts>
__global__ __launch_bounds__(1024) void total_kernel(const double *sums, int64_t count, const float *counted, float scale,
                                                    float *loss, float *out_stats) {
    constexpr int kFlight = 4;
    __shared__ double slots[16];
    double v[3] = {0, 0, 0};
    for (int64_t i0 = threadIdx.x; i0 < count; i0 += 1024 * kFlight) {
        double d[kFlight][kParts];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int64_t i = min(i0 + 1024 * u, count - 1);
#pragma unroll
            for (int c = 0; c < kParts; ++c) d[u][c] = sums[3 * i + c];
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
#pragma unroll
            for (int c = 0; c < kParts; ++c) v[c] += i0 + 1024 * u < count ? d[u][c] : 0.0;
    }
#pragma unroll
    for (int c = 0; c < kParts; ++c) v[c] = block_sum(v[c], slots);
    if (threadIdx.x == 0) {
        *loss = static_cast<float>(v[0] * scale);
        if constexpr (kParts == 3) {
            const float n = fmaxf(*counted, 1.0f);
            out_stats[0] = static_cast<float>(v[1] / n);
            out_stats[1] = static_cast<float>(v[2] / n);
        }
    }
}

void total(const double *sums, int64_t count, const float *counted, float scale, float *loss, float *out_stats,
           hipStream_t s) {
    if (out_stats != nullptr) total_kernel<3><<<1, 1024, 0, s>>>(sums, count, counted, scale, loss, out_stats);
    else total_kernel<1><<<1, 1024, 0, s>>>(sums, count, counted, scale, loss, nullptr);
}

// ------------------------------------------------------------------------------------------ preference pairs
enum PairLoss { kSigmoid = 0, kIpo = 1, kHinge = 2 };

struct PairArgs {
    Tokens tokens;
    Seqs seqs;             // 2 * pairs sequences: the chosen ones, then the rejected ones
    const float *gap;      // [n]
    float *coef;           // [n] (nullable)
    float *chosen, *rejected, *loss;
    double *sums;          // [pairs]
    int64_t pairs;
    double beta;
    float smoothing;
    int32_t vocab;
    int kind, normalized;
};

// log(1 + exp(-x)) without overflow
__device__ __forceinline__ float softplus_neg(float x) { return fmaxf(-x, 0.0f) + log1pf(expf(-fabsf(x))); }

// One pair by one wavefront: both sequences' sums, the loss, and the factors of their rows' gradients. Returns the loss.
// Eight rows per lane are requested at a time: the sums are bound by the loads' latency. The sums and their difference,
// where two large values nearly cancel, are in fp64; what is rounded to fp32 is the difference.
__device__ double pair_terms(const PairArgs &a, int64_t p) {
    constexpr int kFlight = 8;
    const int lane = threadIdx.x & 63;
    double d[2];
    int64_t from[2], to[2];
    float inv_len[2];
    for (int side = 0; side < 2; ++side) {
        const int64_t s = side == 0 ? p : a.pairs + p;
        from[side] = a.seqs.begin(s);
        to[side] = a.seqs.begin(s + 1);
        double sum = 0;  // up to thousands of terms of either sign
        int64_t count = 0;
        for (int64_t r0 = from[side] + lane; r0 < to[side]; r0 += 64 * kFlight) {
            float v[kFlight];
            bool in[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const int64_t r = r0 + 64 * u < to[side] ? r0 + 64 * u : to[side] - 1;
                v[u] = a.gap[r];
                in[u] = a.normalized && a.tokens.token(r, a.vocab) >= 0;
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                if (r0 + 64 * u >= to[side]) break;
                sum += v[u];
                count += in[u];
            }
        }
        sum = wave_sum(sum);
        count = wave_sum(count);
        const double length = a.normalized && count > 0 ? static_cast<double>(count) : 1.0;
        inv_len[side] = static_cast<float>(1.0 / length);
        d[side] = sum / length;
    }
    const double h = d[0] - d[1];
    const float beta = static_cast<float>(a.beta), x = static_cast<float>(a.beta * h);
    float loss, slope;
    if (a.kind == kSigmoid) {
        // a share of 0 makes no term of an infinite value (a sequence with a token that is ruled out)
        loss = a.smoothing < 1.0f ? (1.0f - a.smoothing) * softplus_neg(x) : 0.0f;
        if (a.smoothing > 0.0f) loss += a.smoothing * softplus_neg(-x);
        // 1 / (1 + e^-x) - (1 - smoothing), each side's small part kept: sigma(x) - 1 = -sigma(-x)
        const float up = 1.0f / (1.0f + expf(-x)), down = 1.0f / (1.0f + expf(x));
        slope = beta * (a.smoothing * up - (1.0f - a.smoothing) * down);
    } else if (a.kind == kIpo) {
        const float e = static_cast<float>(h - 0.5 / a.beta);
        loss = e * e;
        slope = 2.0f * e;
    } else {
        loss = fmaxf(1.0f - x, 0.0f);
        if (x != x) loss = x;
        slope = x < 1.0f ? -beta : 0.0f;
    }
    slope /= static_cast<float>(a.pairs);
    for (int side = 0; a.coef != nullptr && side < 2; ++side) {
        const float c = (side == 0 ? slope : -slope) * inv_len[side];
        for (int64_t r0 = from[side] + lane; r0 < to[side]; r0 += 64 * kFlight) {
            int32_t t[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                t[u] = a.tokens.token(r0 + 64 * u < to[side] ? r0 + 64 * u : to[side] - 1, a.vocab);
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (r0 + 64 * u < to[side] && t[u] >= 0) a.coef[r0 + 64 * u] = c;
        }
    }
    if (lane == 0) {
        a.chosen[p] = static_cast<float>(a.beta * d[0]);
        a.rejected[p] = static_cast<float>(a.beta * d[1]);
    }
    return loss;
}

// A wavefront per pair; with one workgroup the mean as well, else the pairs' losses for total_kernel.
__global__ __launch_bounds__(1024) void pair_kernel(const PairArgs a) {
    __shared__ double slots[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    double sum = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * waves;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * waves + wave; p < a.pairs; p += step) {
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
    const float4 *stats;    // [n]
    const float *coef;      // [n]
    const float *upstream;  // [1] (nullable: 1)
    const void *ids;
    const float *fix;       // [n, top]
    void *grad;             // [n, vocab]
    float k, extra;         // extra: factor on coef
    int32_t splits, span, top;
    int ids64, done_for_one;
};

// One part of a row: streams the logits once more and writes the gradient. A copy's bytes, and bound by them: 3.5 GB
// read and 4.3 written (8286 rows of 262,144 bf16 logits, 6640 that count) take 1300 us, 6.0 TB/s, where a device
// copy of 4 GB moves 4.9 (grad_split_of has what the parts' size does to it). Rows whose factor is 0 are filled without
// being read.
template <typename T, int kThreads, bool kStream>
__device__ __forceinline__ void grad_part(const GradArgs &a, float up, int64_t row, int32_t part) {
    constexpr int N = kVec<T>;
    const int32_t vocab = a.logits.vocab, tid = threadIdx.x;
    const bool distill = a.tokens.targets == nullptr;
    const int32_t t = distill ? -1 : a.tokens.token(row, vocab);
    const int32_t from = part * a.span, to = min(vocab, from + a.span);
    const int32_t whole = (to - from) / N;
    T *g = static_cast<T *>(a.grad) + row * vocab;
    const float c = (distill || t >= 0) ? a.coef[row] * up * a.extra : 0.0f;
    if (c == 0.0f) {
        const float zeros[N] = {};
        for (int32_t i = tid; i < whole; i += kThreads) store_unit<kStream>(g + from + N * i, zeros);
        if (tid < to - from - N * whole) store1(g + from + N * whole + tid, 0.0f);
        return;
    }
    const float4 st = a.stats[row];
    const float factor = distill ? c * st.y : -c * st.y, at_token = c * st.z;
    const T *x = static_cast<const T *>(a.logits.x) + a.logits.offset(row);
    const auto values = [&](const float (&v)[N], int32_t j, float (&d)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) d[e] = factor * exp2_of(v[e], st.x, a.k);
        if (t >= j && t < j + N) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (j + e == t) d[e] = at_token;
        }
    };
    constexpr int kUnroll = sizeof(T) == 2 ? 4 : 8;  // loads in flight per thread
    int32_t i = tid;
    for (; i + (kUnroll - 1) * kThreads < whole; i += kUnroll * kThreads) {
        Raw<T> raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) load_raw<kStream>(x + from + N * (i + u * kThreads), raw[u]);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int32_t j = from + N * (i + u * kThreads);
            float v[N], d[N];
            widen(raw[u], v);
            values(v, j, d);
            store_unit<kStream>(g + j, d);
        }
    }
    for (; i < whole; i += kThreads) {
        const int32_t j = from + N * i;
        Raw<T> raw;
        load_raw<kStream>(x + j, raw);
        float v[N], d[N];
        widen(raw, v);
        values(v, j, d);
        store_unit<kStream>(g + j, d);
    }
    if (tid < to - from - N * whole) {
        const int32_t j = from + N * whole + tid;
        store1(g + j, j == t ? at_token : factor * exp2_of(load1(x + j), st.x, a.k));
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

template <typename T, int kThreads, bool kStream>
__global__ __launch_bounds__(kThreads) void grad_kernel(const GradArgs a) {
    const float up = a.upstream != nullptr ? *a.upstream : 1.0f;
    if (a.done_for_one && up == 1.0f) return;
    const int64_t parts = a.logits.n * a.splits;
    for (int64_t p = blockIdx.x; p < parts; p += gridDim.x) {
        const int64_t row = p / a.splits;
        grad_part<T, kThreads, kStream>(a, up, row, static_cast<int32_t>(p - row * a.splits));
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

// Parts of a row for the gradient, which nothing has to join: 16 KB, so that the workgroups that run at one time read
// and write within 32 MB (8286 rows of 262,144 bf16 logits: parts of 64 KB 1430 us, 32 KB 1390, 16 KB 1310, 8 KB 1550,
// where starting the workgroups begins to count; for reading alone the parts' size makes no difference).
Split grad_split_of(int64_t n, int64_t vocab, int dtype) {
    const int32_t most = dtype == ME_BF16 ? 8192 : 4096;
    Split s = split_of(n, vocab);
    if (s.span > most) s = {static_cast<int32_t>(ceil_div(vocab, most)), most};
    return s;
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
    float *weight, *counted, *gap, *entry_x;
    int32_t *entry_id;
    double *sums;
    size_t bytes;
};

Space carve(void *base, int64_t n, int64_t vocab, int64_t pairs, int64_t top = 0) {
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
    const int64_t most = pairs > n ? pairs : n > 2048 ? n : 2048;
    w.sums = reinterpret_cast<double *>(take(static_cast<size_t>(most) * 3 * sizeof(double)));
    w.counted = reinterpret_cast<float *>(take(2 * sizeof(float)));
    w.entry_x = reinterpret_cast<float *>(take(static_cast<size_t>(n) * top * sizeof(float)));
    w.entry_id = reinterpret_cast<int32_t *>(take(static_cast<size_t>(n) * top * sizeof(int32_t)));
    w.bytes = at;
    return w;
}

int check_vocab(const char *what, int64_t vocab) {
    constexpr int64_t kMost = int64_t{kMaxSpan} * kMaxSplits;
    ME_CHECK_ARG(vocab >= 1 && vocab <= kMost, "%s: vocab must be in 1..%d", what, static_cast<int>(kMost));
    return ME_OK;
}

// rows_per_batch past the rows there are makes one batch of them; one that is not positive stays 0 for the check.
Logits logits_of(const void *x, int64_t n, int64_t rows_per_batch, int64_t batch_stride, int64_t row_stride,
                 int64_t vocab) {
    const int64_t per = rows_per_batch < 1 ? 0 : rows_per_batch < INT32_MAX ? rows_per_batch : INT32_MAX;
    return {x, n, static_cast<uint32_t>(per), batch_stride, row_stride, static_cast<int32_t>(vocab)};
}

// Rows of up to kShort tokens take workgroups of one wavefront in both sweeps, longer ones of four.
constexpr int64_t kShort = 2048;

// with_grad: the call writes the gradient, or leaves what it is made from.
int check_logits(const char *what, const Logits &l, int dtype, bool with_grad) {
    ME_CHECK_ARG(dtype == ME_BF16 || dtype == ME_F32, "%s: logits must be bf16 or fp32", what);
    ME_CHECK_ARG(l.n >= 0 && l.n <= INT32_MAX, "%s: n out of range", what);
    ME_CHECK_ARG(l.n == 0 || l.x != nullptr, "%s: logits are null", what);
    ME_CHECK_ARG(l.rows_per_batch >= 1, "%s: rows_per_batch must be positive", what);
    ME_CHECK_ARG(l.row_stride >= 0 && l.batch_stride >= 0, "%s: negative strides", what);
    // A launch of 2^32 threads or more is cut to what its count's lower 32 bits say, without an error. The sweeps have
    // the most: the one-read kernels have no more threads for a row than the gradient's parts, nor without a gradient
    // than the sums' parts. (16 workgroups: the one of the weights, the last of the entries.)
    const Split s = with_grad ? grad_split_of(l.n, l.vocab, dtype) : split_of(l.n, l.vocab);
    ME_CHECK_ARG((l.n * s.splits + 16) * (l.vocab <= kShort ? 64 : 256) <= int64_t{UINT32_MAX}, "%s: too many rows", what);
    return ME_OK;
}

int check_temperature(const char *what, double t) {
    ME_CHECK_ARG(t >= 1e-6 && t <= 1e6, "%s: temperature must be in 1e-6..1e6", what);
    return ME_OK;
}

int check_row_stats(const char *what, const float *row_stats) {
    ME_CHECK_ARG(reinterpret_cast<uint64_t>(row_stats) % 16 == 0, "%s: row_stats must be 16-byte aligned", what);
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
        ME_CHECK_ARG(length >= 0 && length <= INT32_MAX && n_seqs * length == n,
                     "%s: the sequences do not hold the rows", what);
    }
    return ME_OK;
}

template <typename T, int kThreads>
void launch_stats_of(const StatsArgs &a, bool left_out, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(a.logits.n * a.splits + (a.weights.counted != nullptr ? 1 : 0));
    if (blocks == 0) return;
    if (left_out) stats_kernel<T, kThreads, true><<<blocks, kThreads, 0, s>>>(a);
    else stats_kernel<T, kThreads, false><<<blocks, kThreads, 0, s>>>(a);
}

void launch_stats(StatsArgs a, int dtype, bool left_out, hipStream_t s) {
    const bool small = a.logits.vocab <= kShort;
    if (small && a.weights.counted != nullptr && a.logits.n > 1024) {  // too many for a workgroup of one wavefront
        weights_kernel<<<1, 1024, 0, s>>>(a.weights);
        a.weights.counted = nullptr;
    }
    if (dtype == ME_BF16) {
        if (small) launch_stats_of<uint16_t, 64>(a, left_out, s);
        else launch_stats_of<uint16_t, 256>(a, left_out, s);
    } else {
        if (small) launch_stats_of<float, 64>(a, left_out, s);
        else launch_stats_of<float, 256>(a, left_out, s);
    }
}

// Logits and gradient go past the caches where every unit of both is 16-byte aligned and they are too large for the
// last-level cache of 256 MB. (Unaligned units share cache lines, which the caches put together.)
bool streams(const Logits &l, const void *grad, int dtype) {
    const int64_t size = static_cast<int64_t>(dtype_size(dtype)), unit = 16 / size;
    const bool aligned = reinterpret_cast<uint64_t>(l.x) % 16 == 0 && reinterpret_cast<uint64_t>(grad) % 16 == 0 &&
                         l.vocab % unit == 0 && l.row_stride % unit == 0 && l.batch_stride % unit == 0;
    return aligned && l.n * l.vocab * size > int64_t{256} << 20;
}

template <Op kOp>
void launch_rows(const RowArgs &a, int dtype, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(row_blocks(kOp, a.logits.n));
    const int threads = kOp == kDistill ? 256 : 1024;
    const size_t lds = kOp == kDistill ? size_t{4} * kEntryBytes * entry_room(a.top) : 0;
    if (dtype == ME_BF16) row_kernel<kOp, true><<<blocks, threads, lds, s>>>(a);
    else row_kernel<kOp, false><<<blocks, threads, lds, s>>>(a);
    if (kOp >= kPolicy && blocks > 1)
        total(a.sums, blocks, a.weights.counted, a.scale, a.loss, a.out_stats, s);
}

template <typename T, int kThreads>
void launch_grad_of(const GradArgs &a, bool stream_out, hipStream_t s) {
    // a workgroup per part; where most likely nothing is left to do, no more than fill the GPU twice (65,536 workgroups
    // that end at once take 15 us, 4096 take 4; where something is, they take 1450 us for 8192 rows of 262,144 of which
    // a fifth do not count)
    const int64_t parts = a.logits.n * a.splits;
    const unsigned blocks = static_cast<unsigned>(a.done_for_one && parts > 4096 ? 4096 : parts);
    if (stream_out) grad_kernel<T, kThreads, true><<<blocks, kThreads, 0, s>>>(a);
    else grad_kernel<T, kThreads, false><<<blocks, kThreads, 0, s>>>(a);
}

void launch_grad(const GradArgs &a, int dtype, hipStream_t s) {
    if (a.logits.n == 0) return;
    const bool small = a.logits.vocab <= kShort, out = streams(a.logits, a.grad, dtype);
    if (dtype == ME_BF16) {
        if (small) launch_grad_of<uint16_t, 64>(a, out, s);
        else launch_grad_of<uint16_t, 256>(a, out, s);
    } else {
        if (small) launch_grad_of<float, 64>(a, out, s);
        else launch_grad_of<float, 256>(a, out, s);
    }
}

int check_space(const char *what, const Space &w, const void *workspace, size_t bytes) {
    if (reinterpret_cast<uint64_t>(workspace) % 16 != 0) {
        set_error("%s: the workspace is not 16-byte aligned", what);
        return ME_ERR_WORKSPACE;
    }
    if (workspace == nullptr || bytes < w.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace == nullptr ? size_t{0} : bytes, w.bytes);
        return ME_ERR_WORKSPACE;
    }
    return ME_OK;
}

}  // namespace
}  // namespace me

using namespace me;

extern "C" int me_loss_workspace_size(int64_t n, int64_t vocab, int64_t pairs, int64_t top, size_t *bytes) {
    ME_CHECK_ARG(bytes != nullptr, "me_loss_workspace_size: bytes is null");
    ME_CHECK_ARG(n >= 0 && n <= INT32_MAX && pairs >= 0 && pairs <= INT32_MAX && top >= 0 && top <= kMaxTop,
                 "me_loss_workspace_size: size out of range");
    ME_TRY(check_vocab("me_loss_workspace_size", vocab));
    *bytes = carve(nullptr, n, vocab, pairs, top).bytes;
    return ME_OK;
}

extern "C" int me_token_logps(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                              int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                              int64_t ignore_index, double temperature, float *logps, float *row_stats,
                              void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "me_token_logps";
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, row_stats != nullptr));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(n == 0 || logps != nullptr, "%s: logps is null", what);
    ME_TRY(check_row_stats(what, row_stats));
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
    const bool pass = takes_row_pass(n, vocab, dtype, 0, false);
    if (!pass) launch_stats(st, dtype, false, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.part = w.part;
    r.stats = reinterpret_cast<float4 *>(row_stats);
    r.logps = logps;
    r.k = st.k;
    r.inv_temp = static_cast<float>(1.0 / temperature);
    r.splits = sp.splits;
    if (pass) launch_row_pass(kLogps, r, dtype, nullptr, false, s);
    else launch_rows<kLogps>(r, dtype, s);
    return check_launch(what);
}

extern "C" int me_token_logps_backward(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                                       int64_t batch_stride, int64_t row_stride, const void *targets, int targets_dtype,
                                       int64_t ignore_index, double temperature, const float *row_stats,
                                       const float *coef, double coef_scale, const float *upstream, int done_for_one,
                                       void *grad, void *stream) {
    const char *what = "me_token_logps_backward";
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, true));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(n == 0 || (row_stats != nullptr && coef != nullptr && grad != nullptr), "%s: null pointer", what);
    ME_CHECK_ARG(!done_for_one || upstream != nullptr, "%s: done_for_one needs upstream", what);
    ME_TRY(check_row_stats(what, row_stats));
    const Split sp = grad_split_of(n, vocab, dtype);
    GradArgs g = {};
    g.logits = l;
    g.tokens = {targets, nullptr, ignore_index, targets_dtype == ME_I64};
    g.stats = reinterpret_cast<const float4 *>(row_stats);
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
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, row_stats != nullptr));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_CHECK_ARG(pairs >= 0 && pairs < INT32_MAX / 2, "%s: pairs out of range", what);
    ME_TRY(check_seqs(what, seq_offsets, offsets_dtype, 2 * pairs, seq_len, n));
    ME_CHECK_ARG(kind >= kSigmoid && kind <= kHinge, "%s: unknown loss kind", what);
    ME_CHECK_ARG(beta > 0 && beta <= 1e6, "%s: beta must be positive", what);
    ME_CHECK_ARG(smoothing >= 0 && smoothing <= 1, "%s: smoothing must be in 0..1", what);
    ME_TRY(check_row_stats(what, row_stats));
    ME_CHECK_ARG(loss != nullptr && (pairs == 0 || (chosen != nullptr && rejected != nullptr)), "%s: null output", what);
    ME_CHECK_ARG(n == 0 || ref_logps != nullptr, "%s: ref_logps is null", what);
    ME_CHECK_ARG((coef != nullptr) == (row_stats != nullptr), "%s: row_stats and coef go together", what);
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
        const bool pass = takes_row_pass(n, vocab, dtype, 0, false);
        if (!pass) launch_stats(st, dtype, false, s);
        RowArgs r = {};
        r.logits = l;
        r.tokens = tokens;
        r.part = w.part;
        r.stats = reinterpret_cast<float4 *>(row_stats);
        r.coef = coef;
        r.gap = w.gap;
        r.ref_logps = ref_logps;
        r.k = kLog2e;
        r.inv_temp = 1.0f;
        r.splits = sp.splits;
        if (pass) launch_row_pass(kPreference, r, dtype, nullptr, false, s);
        else launch_rows<kPreference>(r, dtype, s);
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
    p.beta = beta;
    p.smoothing = static_cast<float>(smoothing);
    p.vocab = l.vocab;
    p.kind = kind;
    p.normalized = normalized;
    if (pairs <= 16) {
        pair_kernel<<<1, 1024, 0, s>>>(p);
    } else {
        const int64_t blocks = ceil_div(pairs, 4) < 2048 ? ceil_div(pairs, 4) : 2048;
        pair_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
        total(w.sums, blocks, nullptr, 1.0f / static_cast<float>(pairs), loss, nullptr, s);
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
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, grad != nullptr));
    ME_TRY(check_temperature(what, temperature));
    ME_TRY(check_tokens(what, targets, targets_dtype, n));
    ME_TRY(check_seqs(what, seq_offsets, offsets_dtype, n_seqs, seq_len, n));
    ME_CHECK_ARG(clip_low >= 0 && clip_high >= 0, "%s: clip bounds must not be negative", what);
    ME_CHECK_ARG(reduction >= kMean && reduction <= kSequence, "%s: unknown reduction", what);
    ME_CHECK_ARG(loss != nullptr && out_stats != nullptr, "%s: null output", what);
    ME_TRY(check_row_stats(what, row_stats));
    const bool none = n == 0 || (adv_per_seq && n_seqs == 0);  // advantages of nothing have no address
    ME_CHECK_ARG(none || advantages != nullptr, "%s: advantages are null", what);
    ME_CHECK_ARG(n == 0 || (old_logps != nullptr && logps != nullptr && coef != nullptr), "%s: null pointer", what);
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
    const bool pass = takes_row_pass(n, vocab, dtype, 0, grad != nullptr);
    if (pass) weights_kernel<<<1, 1024, 0, s>>>(st.weights);
    else launch_stats(st, dtype, false, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.seqs = seqs;
    r.part = w.part;
    r.weights = st.weights;
    r.stats = reinterpret_cast<float4 *>(row_stats);
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
    if (pass) {
        launch_row_pass(kPolicy, r, dtype, grad, streams(l, grad, dtype), s);
        total(w.sums, n, w.counted, r.scale, loss, out_stats, s);
        return check_launch(what);
    }
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
        const Split gs = grad_split_of(n, vocab, dtype);
        g.splits = gs.splits;
        g.span = gs.span;
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
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, grad != nullptr));
    ME_TRY(check_temperature(what, temperature));
    ME_CHECK_ARG(ids_dtype == ME_I32 || ids_dtype == ME_I64, "%s: teacher ids must be int32 or int64", what);
    ME_CHECK_ARG(teacher_dtype == ME_BF16 || teacher_dtype == ME_F32, "%s: teacher logits must be bf16 or fp32", what);
    ME_CHECK_ARG(top >= 1 && top <= kMaxTop, "%s: top must be in 1..%d", what, kMaxTop);
    ME_CHECK_ARG(teacher_lse == nullptr || top < vocab, "%s: entries for every token leave no rest", what);
    ME_CHECK_ARG(reduction == kMean || reduction == kSum, "%s: unknown reduction", what);
    ME_CHECK_ARG(loss != nullptr, "%s: null output", what);
    ME_TRY(check_row_stats(what, row_stats));
    ME_CHECK_ARG(n == 0 || (teacher_ids != nullptr && teacher != nullptr && row_stats != nullptr && coef != nullptr &&
                            fix != nullptr), "%s: null pointer", what);
    const Space w = carve(workspace, n, vocab, 0, top);
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
    const bool pass = takes_row_pass(n, vocab, dtype, top, grad != nullptr);
    if (!pass) launch_stats(st, dtype, teacher_lse != nullptr, s);
    RowArgs r = {};
    r.logits = l;
    r.tokens = st.tokens;
    r.part = w.part;
    r.weights = st.weights;
    r.stats = reinterpret_cast<float4 *>(row_stats);
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
    if (pass) {
        r.near = w.gap;
        r.entry_x = w.entry_x;
        r.entry_id = w.entry_id;
        const unsigned blocks = static_cast<unsigned>(ceil_div(n, 4) + 1);
        const size_t lds = size_t{4} * kEntryBytes * entry_room(r.top);
        if (dtype == ME_BF16) entries_kernel<true><<<blocks, 256, lds, s>>>(r);
        else entries_kernel<false><<<blocks, 256, lds, s>>>(r);
        launch_row_pass(kDistill, r, dtype, grad, streams(l, grad, dtype), s);
        total(w.sums, n, nullptr, r.scale, loss, nullptr, s);
        return check_launch(what);
    }
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
        const Split gs = grad_split_of(n, vocab, dtype);
        g.splits = gs.splits;
        g.span = gs.span;
        launch_grad(g, dtype, s);
    }
    return check_launch(what);
}

extern "C" int me_distill_backward(const void *logits, int dtype, int64_t n, int64_t vocab, int64_t rows_per_batch,
                                   int64_t batch_stride, int64_t row_stride, const void *teacher_ids, int ids_dtype,
                                   int64_t top, double temperature, const float *row_stats, const float *coef,
                                   const float *fix, const float *upstream, int done_for_one, void *grad, void *stream) {
    const char *what = "me_distill_backward";
    ME_TRY(check_vocab(what, vocab));
    const Logits l = logits_of(logits, n, rows_per_batch, batch_stride, row_stride, vocab);
    ME_TRY(check_logits(what, l, dtype, true));
    ME_TRY(check_temperature(what, temperature));
    ME_CHECK_ARG(ids_dtype == ME_I32 || ids_dtype == ME_I64, "%s: teacher ids must be int32 or int64", what);
    ME_CHECK_ARG(top >= 1 && top <= kMaxTop, "%s: top must be in 1..%d", what, kMaxTop);
    ME_CHECK_ARG(n == 0 || (teacher_ids != nullptr && row_stats != nullptr && coef != nullptr && fix != nullptr &&
                            grad != nullptr), "%s: null pointer", what);
    ME_CHECK_ARG(!done_for_one || upstream != nullptr, "%s: done_for_one needs upstream", what);
    ME_TRY(check_row_stats(what, row_stats));
    const Split sp = grad_split_of(n, vocab, dtype);
    GradArgs g = {};
    g.logits = l;
    g.stats = reinterpret_cast<const float4 *>(row_stats);
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
