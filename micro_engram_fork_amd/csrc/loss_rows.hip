// The policy and distillation losses with their gradient from one read of the logits: a workgroup keeps a row on its
// CU, in registers and for the longest rows in LDS too, between adding up its exponentials and writing its gradient.
//
// Bound by HBM: 2 bytes read and 2 written per bf16 logit, where two sweeps (losses.hip) move 6. A CU has 512 KB of
// registers and 160 KB of LDS: a row of 262,144 bf16 logits is 512 KB, of which 1024 threads hold 22 16-byte slots each
// in registers (88 of the 128 that 16 wavefronts leave a thread: all are taken, and up to 4 values are in scratch) and 9
// in LDS; what is beyond is read a second time. A row's slots are all requested before the first is used, so the whole
// row is in flight at once.
//
// Measured (policy, all rows counting): 8192 rows of 262,144 bf16 logits 1690-1920 us (4.5-5.1 TB/s: one row per CU,
// whose read and sum, 28 us, and write follow each other), of 131,072 775 us (5.5), of 32,000 165-205 us (5.1-6.4,
// several rows per CU), 8192 rows of 50,021 fp32 logits 610 us (5.4).
#include "loss_common.h"

namespace me {

using namespace loss;

namespace {

constexpr int64_t kForwardUnits = 4096;
constexpr int kPassTop = 512;  // teacher entries the kernels' LDS has room for

// The logit at an index that all threads share.
__device__ __forceinline__ float scalar_logit(const uint16_t *x, int32_t j) {
    return __uint_as_float(constant_bytes(x + j) << 16);
}
__device__ __forceinline__ float scalar_logit(const float *x, int32_t j) { return constant(x + j); }

template <typename T, int kThreads, int kRegs, int kLds, bool kStream, Op kOp, bool kRest>
__global__ __launch_bounds__(kThreads) void pass_kernel(const RowArgs a, void *grad) {
    constexpr int N = kVec<T>;
    constexpr bool kDist = kOp == kDistill, kWeighted = kOp >= kPolicy;
    constexpr int kWaves = kThreads / 64;
    constexpr bool kKeepExp = sizeof(T) == 4;  // fp32 slots take the exponentials in place: none for the gradient
    __shared__ Raw<T> held[kLds > 0 ? kLds : 1][kThreads];
    __shared__ __attribute__((aligned(16))) uint8_t entry_space[kDist ? kPassTop * kEntryBytes : 16];
    constexpr bool kBits = kRest && kLds == 0;
    __shared__ uint32_t left_out[kBits ? (kThreads * kRegs * N + 8 + 31) / 32 : 1];
    __shared__ float sums[kWaves];
    const int64_t r = blockIdx.x;
    const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t vocab = a.logits.vocab, whole = vocab / N, rest = vocab - N * whole;
    const int32_t slots = (whole + kThreads - 1) / kThreads;
    T *g = static_cast<T *>(grad) + r * vocab;
    if (kWeighted ? constant(a.weights.weight + r) == 0.0f : a.tokens.token(r, vocab) < 0) {
        if (grad != nullptr) {
            const float zeros[N] = {};
            for (int32_t i = tid; i < whole; i += kThreads) store_unit<kStream>(g + N * i, zeros);
            if (tid < rest) store1(g + N * whole + tid, 0.0f);
        }
        if (tid == 0) {
            if (a.stats != nullptr) a.stats[r] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (a.coef != nullptr) a.coef[r] = 0.0f;
            if (a.logps != nullptr) a.logps[r] = 0.0f;
            if (a.gap != nullptr) a.gap[r] = 0.0f;
            if constexpr (kWeighted)
                for (int c = 0; c < 3; ++c) a.sums[3 * r + c] = 0;
        }
        if constexpr (kDist)
            for (int32_t i = tid; i < a.top; i += kThreads) a.fix[r * a.top + i] = 0.0f;
        return;
    }
    const T *x = static_cast<const T *>(a.logits.x) + a.logits.offset(r);

    // All loads of the row are issued before the first is used, and none of them under a condition: a slot past the
    // row's end loads the last unit again. (Loads return in the order of their issue; after one that may or may not
    // have been issued the compiler can only wait for all.) The entries of a row come before its logits for the same
    // reason, and its other few values through the scalar cache.
    constexpr int kPer = kDist ? (kPassTop + kThreads - 1) / kThreads : 1;  // entries of a thread
    const Entries e = entries_at(entry_space, a.top);
    int32_t entry_id[kPer];
    float entry_p[kPer], entry_x[kPer];
    if constexpr (kDist) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            if (u > 0 && u * kThreads >= a.top) break;
            const int32_t i = min(tid + u * kThreads, a.top - 1);
            entry_id[u] = *as_global(a.entry_id + r * a.top + i);
            entry_p[u] = *as_global(a.fix + r * a.top + i);
            entry_x[u] = *as_global(a.entry_x + r * a.top + i);
        }
    }
    const float last = load1(x + min(N * whole + tid, vocab - 1));
    // slot s of a thread: unit s * kThreads + tid
    const auto load_slot = [&](int32_t s, Raw<T> &raw) {
        load_raw<kStream>(x + N * static_cast<int64_t>(min(s * kThreads + tid, whole - 1)), raw);
    };
    Raw<T> q[kRegs];
#pragma unroll
    for (int c = 0; c < kRegs; ++c) load_slot(c, q[c]);

    const float weight = kWeighted ? row_weight(a.weights, r) : 1.0f;
    int32_t t = -1;
    float xt;
    Sampled sampled = {};
    if constexpr (kDist) {
        xt = constant(a.near + r);
    } else {
        t = a.tokens.token(r, vocab);
        xt = scalar_logit(x, t);
        if constexpr (kOp == kPolicy) sampled = sampled_row(a, r);
        else if constexpr (kOp == kPreference) sampled.ref_logp = constant(a.ref_logps + r);
    }
    const Guess guess = guess_of(xt, a.k);
    const int32_t t_slot = kDist || t >= N * whole ? -1 : t / N / kThreads, t_thread = kDist ? -1 : t / N % kThreads;

    // Where entries are to be left out of the sum: a bit for each token, or where the LDS is taken by logits, a mark for
    // each slot of a wavefront that holds one (few do: such rows are long).
    uint64_t marks = 0;
    if constexpr (kBits) {
        for (int32_t i = tid; i < (vocab + 31) / 32; i += kThreads) left_out[i] = 0;
        if constexpr (kWaves > 1) __syncthreads();
        else wave_lds_order();
    }
    if constexpr (kDist) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int32_t i = tid + u * kThreads;
            if (i < a.top) {
                e.id[i] = entry_id[u];
                e.p[i] = entry_p[u];
                e.x[i] = entry_x[u];
                if constexpr (kBits)
                    if (entry_id[u] >= 0) atomicOr(&left_out[entry_id[u] >> 5], 1u << (entry_id[u] & 31));
            }
        }
        if constexpr (kWaves > 1) __syncthreads();
        else wave_lds_order();
    }
    if constexpr (kRest && !kBits) {
        for (int32_t i0 = 0; i0 < a.top; i0 += 64) {
            const int32_t i = i0 + lane, c = i < a.top ? e.id[i] / N : -1, s = c / kThreads;
            uint64_t hits = __ballot(i < a.top && e.id[i] >= 0 && c < whole && (c % kThreads) >> 6 == wave);
            while (hits != 0) {
                const int src = __builtin_ctzll(hits);
                hits &= hits - 1;
                marks |= 1ull << __builtin_amdgcn_readlane(s, src);
            }
        }
    }
    float tail = tid < rest ? last : -kInf;
    const auto leave_out = [&](int32_t s, float (&v)[N]) {
        if constexpr (kBits) {
            const int32_t j = N * min(s * kThreads + tid, whole - 1);
            const uint32_t bits = left_out[j >> 5] >> (j & 31);
            if (__any((bits & ((1u << N) - 1)) != 0)) {
#pragma unroll
                for (int w = 0; w < N; ++w)
                    if (bits >> w & 1) v[w] = -kInf;
            }
        } else if (marks >> s & 1) {
            const int32_t first = s * kThreads + wave * 64;
            for (int32_t i0 = 0; i0 < a.top; i0 += 64) {
                const int32_t i = i0 + lane, id = i < a.top ? e.id[i] : -1, rel = id / N - first;
                uint64_t hits = __ballot(id >= 0 && rel >= 0 && rel < 64);
                while (hits != 0) {
                    const int src = __builtin_ctzll(hits);
                    hits &= hits - 1;
                    const int32_t token = __builtin_amdgcn_readlane(id, src);
#pragma unroll
                    for (int w = 0; w < N; ++w)
                        if (lane == token / N - first && w == token % N) v[w] = -kInf;
                }
            }
        }
    };

    // ---- sum of exponentials
    float sum = 0.0f;
    const auto add_slot = [&](int32_t s, Raw<T> &raw) {
        float v[N];
        widen(raw, v);
        if ((s + 1) * kThreads > whole && s * kThreads + tid >= whole) {
#pragma unroll
            for (int w = 0; w < N; ++w) v[w] = -kInf;
        }
        if constexpr (kRest) leave_out(s, v);
        if constexpr (!kDist) {  // the row's own token is added by token_terms
            if (s == t_slot) {
#pragma unroll
                for (int w = 0; w < N; ++w)
                    if (tid == t_thread && w == t % N) v[w] = -kInf;
            }
        }
#pragma unroll
        for (int w = 0; w < N; ++w) v[w] = guessed_exp(v[w], guess, a.k);
        if constexpr (kKeepExp) keep_raw(raw, v);
        sum += tree_sum(v);
    };
#pragma unroll
    for (int c = 0; c < kLds; ++c) {  // these make room for the slots past the registers' own
        if (c < slots) {
            add_slot(c, q[c]);
            held[c][tid] = q[c];
        }
        load_slot(kRegs + c, q[c]);
    }
#pragma unroll
    for (int c = kLds; c < kRegs; ++c)
        if (c < slots) add_slot(c, q[c]);
#pragma unroll
    for (int c = 0; c < kLds; ++c)
        if (kRegs + c < slots) add_slot(kRegs + c, q[c]);
    for (int32_t s = kRegs + kLds; s < slots; ++s) {
        Raw<T> raw;
        load_slot(s, raw);
        add_slot(s, raw);
    }
    if constexpr (kRest) {
        if (tid < rest)
            for (int32_t i = 0; i < a.top; ++i)
                if (e.id[i] == N * whole + tid) tail = -kInf;
    }
    if (!kDist && N * whole + tid == t) tail = -kInf;
    sum = wave_sum(sum + guessed_exp(tail, guess, a.k));
    if constexpr (kWaves > 1) {
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = sums[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += sums[w];
    }
    MaxSum row = {guess.m, without_rounding(sum, guess, a.k)};
    const bool guessed = guess.fits && sum < kLargestSum && (!kRest || sum > kSmallestSum);
    if (!guessed) {  // again, with the running maximum
        row = {-kInf, 0.0f};
        for (int32_t j = N * tid; j < vocab; j += N * kThreads) {
            float v[N];
            load_tail(x, j, vocab, v);
            if constexpr (kRest) {
                for (int32_t i = 0; i < a.top; ++i) {
                    const int32_t w0 = e.id[i] - j;
                    if (w0 >= 0 && w0 < N) {
#pragma unroll
                        for (int w = 0; w < N; ++w)
                            if (w == w0) v[w] = -kInf;
                    }
                }
            }
            if constexpr (!kDist) {
#pragma unroll
                for (int w = 0; w < N; ++w)
                    if (j + w == t) v[w] = -kInf;
            }
            add_values(row, v, a.k);
        }
        row = wave_join(row, a.k);
        if constexpr (kWaves > 1) {
            __shared__ MaxSum joined[kWaves];
            if (lane == 0) joined[wave] = row;
            __syncthreads();
            row = joined[0];
            for (int w = 1; w < kWaves; ++w) row = join(row, joined[w], a.k);
        }
    }

    // ---- the loss and the gradient's factors
    float coef, factor, ref, at_token = 0.0f;
    if constexpr (kDist) {  // every wavefront the same, so that none waits for another
        float4 stats;
        const float loss = distill_finish(a, r, row, e, stats, wave == 0);
        coef = a.scale * weight * a.temp;
        factor = coef * stats.y;
        ref = stats.x;
        if (tid == 0) {
            a.stats[r] = stats;
            a.coef[r] = coef;
            a.sums[3 * r] = static_cast<double>(loss) * weight;
        }
    } else {
        const TokenTerms token = token_terms(xt, row, a.k, a.inv_temp);
        const float logp = token.logp, inv_s = 1.0f / token.all.s;
        ref = token.all.m;
        if (tid == 0) {
            if (a.stats != nullptr) a.stats[r] = {ref, inv_s, token.rest, 0.0f};
            if (a.logps != nullptr) a.logps[r] = logp;
        }
        if constexpr (kOp == kPolicy) {
            float loss, slope, kl;
            bool clipped;
            policy_terms(a, sampled, logp, loss, slope, kl, clipped);
            coef = a.scale * weight * slope * a.inv_temp;
            factor = -coef * inv_s;
            at_token = coef * token.rest;
            if (tid == 0) {
                a.coef[r] = coef;
                a.sums[3 * r] = static_cast<double>(loss) * weight;
                a.sums[3 * r + 1] = kl;
                a.sums[3 * r + 2] = clipped;
            }
        } else {
            if constexpr (kOp == kPreference) {
                if (tid == 0) {
                    a.gap[r] = logp - sampled.ref_logp;
                    if (a.coef != nullptr) a.coef[r] = 0.0f;
                }
            }
            return;  // the gradient waits for other rows or for the caller
        }
    }

    // ---- gradient
    if (grad == nullptr) return;
    if (!guessed) {
        for (int32_t j = tid; j < vocab; j += kThreads)
            store1(g + j, !kDist && j == t ? at_token : factor * exp2_of(load1(x + j), ref, a.k));
        if constexpr (kDist) {
            __syncthreads();
            for (int32_t i = tid; i < a.top; i += kThreads)
                if (e.id[i] >= 0) store1(g + e.id[i], coef * e.raw[i]);
        }
        return;
    }
    // exponentials are those of `sum`; the rounding of m k that row.s is without goes into the factor
    factor = without_rounding(factor, guess, a.k);
    const auto put_slot = [&](int32_t s, const Raw<T> &raw) {
        float d[N];
        widen(raw, d);
#pragma unroll
        for (int w = 0; w < N; ++w) {
            if constexpr (!kKeepExp) d[w] = guessed_exp(d[w], guess, a.k);
            d[w] *= factor;
        }
        if constexpr (!kDist) {
            if (s == t_slot) {
#pragma unroll
                for (int w = 0; w < N; ++w)
                    if (tid == t_thread && w == t % N) d[w] = at_token;
            }
        }
        const int32_t c = s * kThreads + tid;
        if (c < whole) store_unit<kStream>(g + N * static_cast<int64_t>(c), d);
    };
#pragma unroll
    for (int c = kLds; c < kRegs; ++c)
        if (c < slots) put_slot(c, q[c]);
#pragma unroll
    for (int c = 0; c < kLds; ++c)
        if (kRegs + c < slots) put_slot(kRegs + c, q[c]);
#pragma unroll
    for (int c = 0; c < kLds; ++c)
        if (c < slots) put_slot(c, held[c][tid]);
    for (int32_t s = kRegs + kLds; s < slots; ++s) {
        Raw<T> raw;
        load_slot(s, raw);
        if constexpr (kKeepExp) {
            float v[N];
            widen(raw, v);
#pragma unroll
            for (int w = 0; w < N; ++w) v[w] = guessed_exp(v[w], guess, a.k);
            keep_raw(raw, v);
        }
        put_slot(s, raw);
    }
    if (tid < rest) {
        const int32_t j = N * whole + tid;
        store1(g + j, !kDist && j == t ? at_token : factor * guessed_exp(tail, guess, a.k));
    }
    if constexpr (kDist) {  // the entries over what the sweep has stored there
        __syncthreads();
        for (int32_t i = tid; i < a.top; i += kThreads)
            if (e.id[i] >= 0) store1(g + e.id[i], coef * e.raw[i]);
    }
}

template <typename T, int kThreads, int kRegs, int kLds, bool kStream = false>
void launch_pass_of(Op op, const RowArgs &a, void *grad, hipStream_t s) {
    const unsigned n = static_cast<unsigned>(a.logits.n);
    if constexpr (kThreads <= 256) {  // (kForwardUnits)
        if (op == kLogps)
            return pass_kernel<T, kThreads, kRegs, kLds, kStream, kLogps, false><<<n, kThreads, 0, s>>>(a, nullptr);
        if (op == kPreference)
            return pass_kernel<T, kThreads, kRegs, kLds, kStream, kPreference, false><<<n, kThreads, 0, s>>>(a, nullptr);
    }
    if (op == kPolicy) pass_kernel<T, kThreads, kRegs, kLds, kStream, kPolicy, false><<<n, kThreads, 0, s>>>(a, grad);
    else if constexpr (kRegs <= 16 || kLds > 0) {
        // (with 22 slots in registers alone, leaving entries out spills 32 registers, fp32 54; the variants of 1024
        // threads that are launched spill 4 at most)
        if (a.teacher_lse != nullptr)
            pass_kernel<T, kThreads, kRegs, kLds, kStream, kDistill, true><<<n, kThreads, 0, s>>>(a, grad);
        else pass_kernel<T, kThreads, kRegs, kLds, kStream, kDistill, false><<<n, kThreads, 0, s>>>(a, grad);
    } else pass_kernel<T, kThreads, kRegs, kLds, kStream, kDistill, false><<<n, kThreads, 0, s>>>(a, grad);
}

template <typename T>
void launch_pass(Op op, const RowArgs &a, void *grad, bool stream_rows, hipStream_t s) {
    const int32_t units = a.logits.vocab / kVec<T>;
    if (units <= 64 * 16) launch_pass_of<T, 64, 16, 0>(op, a, grad, s);
    else if (units <= 256 * 16) launch_pass_of<T, 256, 16, 0>(op, a, grad, s);
    else if (units <= 512 * 16) launch_pass_of<T, 512, 16, 0>(op, a, grad, s);
    else if (units <= 1024 * 16) launch_pass_of<T, 1024, 16, 0>(op, a, grad, s);
    else if (units <= 1024 * 22 && a.teacher_lse == nullptr) launch_pass_of<T, 1024, 22, 0>(op, a, grad, s);
    else if (stream_rows) launch_pass_of<T, 1024, 22, 9, true>(op, a, grad, s);
    else launch_pass_of<T, 1024, 22, 9>(op, a, grad, s);
}

}  // namespace

// Rows from which one read wins, measured as kernel times (policy / distillation with 64 entries and the rest class,
// two sweeps over one read): at 32,768 units (262,144 bf16 logits) 64 rows 0.79 / 0.76, 128 rows 1.06 / 0.90, 256 rows
// 1.19 / 1.11; 8192 units 32 rows 1.01 / 0.95, 64 rows 1.18 / 1.02; 4000 units 16 rows 0.85 / 1.01, 32 rows 1.16; 1000
// units 16 rows 1.03 / 1.10; 125 units 8 rows 1.08. Without a gradient there is nothing to read twice, and the parts of
// many workgroups read faster than a CU's one row (8192 rows of 262,144: 500 us against 615); rows of up to 4096 units
// take one read there too, for its fewer launches (4000 units: 256 rows 20.8 us against 14.6, 8192 rows 103 against 109).
bool takes_row_pass(int64_t n, int64_t vocab, int dtype, int64_t top, bool with_grad) {
    if (n == 0 || vocab < 64 || top > kPassTop) return false;
    const int64_t units = vocab / (dtype == ME_BF16 ? 8 : 4);
    return units <= (with_grad ? 1024 * 40 : kForwardUnits) && n * 192 >= units;
}

void launch_row_pass(Op op, const RowArgs &a, int dtype, void *grad, bool stream_rows, hipStream_t s) {
    if (dtype == ME_BF16) launch_pass<uint16_t>(op, a, grad, stream_rows, s);
    else launch_pass<float>(op, a, grad, stream_rows, s);
}

}  // namespace me
