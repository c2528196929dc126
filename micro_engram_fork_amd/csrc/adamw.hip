// AdamW on gfx950 for all dense tensors of a model at once (DenseAdamW.step; the reference trains the
// engram's projections and scales with torch's AdamW, micro_engram/optim.py:47-63 for its state):
//
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   p' = (1 - lr wd) p - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// HBM-bound: every value is read once and written once, 22 bytes a weight (bf16 weights and gradients,
// fp32 moments), 28 (all fp32) or 10 (bf16, 8-bit moments). Measured: 341 million weights in fp32 1750 us, 5.4 TB/s;
// 929 million in bf16 with 8-bit moments 1906 us, 4.9 TB/s; 16.5 million in bf16 with fp32 ones 55 us in the
// kernel, 6.6 TB/s with the 256 MB cache's help. (A 4 GB copy: 4.8 TB/s.) A thread takes eight values that lie together,
// so that each tensor moves in 8- to 16-byte pieces and one Philox call gives the rounding noise of all
// eight; the tensors of a launch stand in the kernel's arguments (no table to upload, graphs replay it), and a
// workgroup finds its tensor with one load and a ballot over their first chunks.
//
// Moments in 8 bits: blocks of 128 values (16 lanes) with a scale each, a power of two, E8M0. First
// moments are e4m3 with the block's largest in the binade of 2^7 (so that rounding it up still has a code),
// second moments e5m2 with it in that of 2^14: values down to 2^-16 and 2^-30 of the block's largest. With
// powers of two a change of the scale moves no value off the grid, so what a step does not change is not rounded
// again. They are rounded stochastically: a step changes v by a thousandth where a code is a quarter
// wide, and rounding to nearest would hold it where it is. A second moment over zero keeps the smallest code,
// so that no quotient outgrows what the first moment's range allows. The step itself uses m' and v' before
// their rounding.
//
// Noise of the eight values from 8 k on of tensor s at step t: the eight 16-bit halves of Philox4x32-10(key
// seed, counter (k low, k high, t, s)). Weights take a half r, first moments r rotated by eight bits, second moments
// 65535 - r: each is uniform, which is all that an unbiased rounding asks for, and three calls would make the
// 8-bit step compute-bound.
#include "me_common.h"
#include "philox.h"

#include <algorithm>
#include <cmath>

namespace me {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;                      // values per thread
constexpr int kChunk = kThreads * kPer;       // values per workgroup; two or four times as many in rounds took 3-8 % longer
constexpr int kTensors = 42;                 // tensors per launch (kernel arguments stay under 4 KiB)
constexpr int kBlock = 128;                  // values per scale of 8-bit moments
constexpr int64_t kMostChunks = int64_t{1} << 23;

struct Tensor {
    uint8_t *p, *m, *v;
    const uint8_t *g;
    uint8_t *m_scale, *v_scale;
    const float *step_at;  // step count on the device, or null: the three values below
    int64_t n;
    float step_size;       // lr / (1 - b1^t)
    float inv_sqrt_bc2;    // 1 / sqrt(1 - b2^t)
    uint32_t step, stream;
};

struct Args {
    int32_t first[kTensors];  // first chunk of each tensor
    int32_t n_tensors;
    Tensor t[kTensors];
    float beta1, beta2, rest1, rest2, eps, decay;
    double lr, log_beta1, log_beta2;
    uint64_t seed;
    int sr;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

// pieces of tensors that may start at any element
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

template <bool BF16>
__device__ __forceinline__ void load8(const uint8_t *base, int64_t i, int left, float (&x)[kPer]) {
    if constexpr (BF16) {
        const auto at = as_global(reinterpret_cast<const uint16_t *>(base) + i);
        if (left >= kPer) {
            const u32x4_any w = *(gmem_ptr<const u32x4_any>)(at);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = __uint_as_float(w[j] << 16);
                x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[j] = j < left ? bf16_bits_to_float(at[j]) : 0.f;
        }
    } else {
        const auto at = as_global(reinterpret_cast<const float *>(base) + i);
        if (left >= kPer) {
            const f32x4_any a = *(gmem_ptr<const f32x4_any>)(at), b = *(gmem_ptr<const f32x4_any>)(at + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[j] = j < left ? at[j] : 0.f;
        }
    }
}

__device__ __forceinline__ void store8_f32(uint8_t *base, int64_t i, int left, const float (&x)[kPer]) {
    const auto at = as_global(reinterpret_cast<float *>(base) + i);
    if (left >= kPer) {
        f32x4_any a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = x[j], b[j] = x[4 + j];
        *(gmem_ptr<f32x4_any>)(at) = a;
        *(gmem_ptr<f32x4_any>)(at + 4) = b;
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < left) at[j] = x[j];
    }
}

__device__ __forceinline__ void store8_bf16(uint8_t *base, int64_t i, int left, const uint32_t (&w)[4]) {
    const auto at = as_global(reinterpret_cast<uint16_t *>(base) + i);
    if (left >= kPer) {
        u32x4_any a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = w[j];
        *(gmem_ptr<u32x4_any>)(at) = a;
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < left) at[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
}

__device__ __forceinline__ u32x2_v load8_codes(const uint8_t *base, int64_t i, int left) {
    const auto at = as_global(base + i);
    u32x2_v w = {0, 0};
    if (left >= kPer) {
        const u32x2_any x = *(gmem_ptr<const u32x2_any>)(at);
        w = {x[0], x[1]};
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < left) w[j >> 2] |= static_cast<uint32_t>(at[j]) << (8 * (j & 3));
    }
    return w;
}

__device__ __forceinline__ void store8_codes(uint8_t *base, int64_t i, int left, const u32x2_v &w) {
    const auto at = as_global(base + i);
    if (left >= kPer) {
        u32x2_any x = {w[0], w[1]};
        *(gmem_ptr<u32x2_any>)(at) = x;
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < left) at[j] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
    }
}

// 2^(b - 127) of an E8M0 byte (b = 0: the subnormal 2^-127)
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b ? b << 23 : 0x00400000u); }

// SECOND: e5m2, else e4m3
template <bool SECOND>
__device__ __forceinline__ void decode8(const u32x2_v &w, float scale, float (&x)[kPer]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int word = static_cast<int>(w[h]);
        if constexpr (SECOND) {
            x[4 * h] = __builtin_amdgcn_cvt_f32_bf8(word, 0) * scale;
            x[4 * h + 1] = __builtin_amdgcn_cvt_f32_bf8(word, 1) * scale;
            x[4 * h + 2] = __builtin_amdgcn_cvt_f32_bf8(word, 2) * scale;
            x[4 * h + 3] = __builtin_amdgcn_cvt_f32_bf8(word, 3) * scale;
        } else {
            x[4 * h] = __builtin_amdgcn_cvt_f32_fp8(word, 0) * scale;
            x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(word, 1) * scale;
            x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(word, 2) * scale;
            x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(word, 3) * scale;
        }
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false)));
}

// largest value over the 16 lanes of a DPP row, in all of them
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = dpp_max<0xb1>(x);   // quad_perm [1, 0, 3, 2]
    x = dpp_max<0x4e>(x);   // quad_perm [2, 3, 0, 1]
    x = dpp_max<0x141>(x);  // row_half_mirror
    return dpp_max<0x140>(x);  // row_mirror
}

// The eight values as codes, and their block's scale byte: the block's exponent less TOP, so that its
// largest finite value is in the binade of 2^TOP. A code is the value's fp32 bits with `noise` added below the
// BITS that are kept; below the smallest normal code (2^LOWEST) codes are a fixed step apart. Values that
// are not finite take the code of NaN and leave the others of their block as they are.
template <bool SECOND>
__device__ __forceinline__ u32x2_v encode8(const float (&x)[kPer], const uint32_t (&noise)[kPer], uint32_t &scale) {
    constexpr int kBits = SECOND ? 2 : 3, kLowest = SECOND ? -14 : -6, kTop = SECOND ? 14 : 7;
    constexpr int kDrop = 23 - kBits;
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t a = __float_as_uint(x[j]) & 0x7fffffffu;
        most = max(most, a < 0x7f800000u ? a : 0u);
    }
    const int exponent = static_cast<int>(row_max(most) >> 23);
    scale = static_cast<uint32_t>(max(exponent - kTop, 0));
    const float inverse = __uint_as_float((254u - scale) << 23);  // 2^(127 - scale); scale <= 247
    u32x2_v w = {0, 0};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t bits = __float_as_uint(x[j]);
        const float y = __uint_as_float(bits & 0x7fffffffu) * inverse;
        const uint32_t add = (noise[j] << (kDrop - 16)) + (1u << (kDrop - 17));
        uint32_t code = ((__float_as_uint(y) + add) >> kDrop) - static_cast<uint32_t>((126 + kLowest) << kBits);
        constexpr float kLow = SECOND ? 6.103515625e-05f : 0.015625f;         // 2^LOWEST
        constexpr float kUnit = SECOND ? 65536.f : 512.f;                      // 2^(BITS - LOWEST)
        constexpr float kFraction = SECOND ? 0x1p-21f : 0x1p-20f;              // 2^-DROP
        if (y < kLow) code = static_cast<uint32_t>(y * kUnit + static_cast<float>(add) * kFraction);
        if constexpr (SECOND) {
            if (code == 0 && x[j] > 0.f) code = 1;
        } else {
            if (x[j] < 0.f) code |= 0x80u;
        }
        if ((bits & 0x7f800000u) == 0x7f800000u) code = 0x7fu;
        w[j >> 2] |= code << (8 * (j & 3));
    }
    return w;
}

template <bool P16, bool G16, bool EIGHT>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Args a) {
    // the last tensor whose first chunk is at or before this one (tensors have a chunk at least)
    const int lane = threadIdx.x & 63;
    const int bid = static_cast<int>(blockIdx.x);
    const bool before = lane < a.n_tensors && a.first[min(lane, kTensors - 1)] <= bid;
    const int k = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
    const Tensor &t = a.t[k];
    const int64_t n = t.n;
    const int64_t base = static_cast<int64_t>(bid - a.first[k]) * kChunk;
    float step_size = t.step_size, inv_sqrt_bc2 = t.inv_sqrt_bc2;
    uint32_t step = t.step;
    if (t.step_at != nullptr) {  // the same for the whole launch: uniform
        const double s = static_cast<double>(*as_global(t.step_at));
        step = static_cast<uint32_t>(s);
        step_size = static_cast<float>(a.lr / -expm1(s * a.log_beta1));
        inv_sqrt_bc2 = static_cast<float>(1.0 / sqrt(-expm1(s * a.log_beta2)));
    }
    float p[kPer], g[kPer], m[kPer], v[kPer];
    u32x2_v mc, vc;
    uint32_t ms, vs;
    const int64_t at = base + static_cast<int64_t>(threadIdx.x) * kPer;
    const int left = static_cast<int>(min(max(n - at, int64_t{0}), int64_t{kPer}));
    load8<P16>(t.p, at, left, p);
    load8<G16>(t.g, at, left, g);
    if constexpr (EIGHT) {
        mc = load8_codes(t.m, at, left);
        vc = load8_codes(t.v, at, left);
        ms = left > 0 ? as_global(t.m_scale)[at / kBlock] : 0;
        vs = left > 0 ? as_global(t.v_scale)[at / kBlock] : 0;
    } else {
        load8<false>(t.m, at, left, m);
        load8<false>(t.v, at, left, v);
    }
    uint32_t noise[kPer];
    const bool draws = EIGHT || (P16 && a.sr);
    if (draws) {
        const uint64_t group = static_cast<uint64_t>(at) / kPer;
        const uint4 w = philox4x32_10(make_uint4(static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32), step, t.stream),
                                      make_uint2(static_cast<uint32_t>(a.seed), static_cast<uint32_t>(a.seed >> 32)));
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < kPer; ++j) noise[j] = (words[j >> 1] >> (16 * (j & 1))) & 0xffffu;
    }
    if constexpr (EIGHT) {
        decode8<false>(mc, scale_of(ms), m);
        decode8<true>(vc, scale_of(vs), v);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        m[j] = a.beta1 * m[j] + a.rest1 * g[j];
        v[j] = a.beta2 * v[j] + a.rest2 * (g[j] * g[j]);
        // 1 ulp each: far below the rounding of p, of which the quotient is at most a few lr
        const float denom = __builtin_amdgcn_sqrtf(v[j]) * inv_sqrt_bc2 + a.eps;
        p[j] = a.decay * p[j] - step_size * (m[j] * __builtin_amdgcn_rcpf(denom));
    }
    if constexpr (P16) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t half[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                half[h] = a.sr ? stochastic_bf16_bits(p[2 * j + h], noise[2 * j + h])
                               : float_to_bf16_bits_rne(p[2 * j + h]);
            w[j] = half[0] | (half[1] << 16);
        }
        store8_bf16(t.p, at, left, w);
    } else {
        store8_f32(t.p, at, left, p);
    }
    if constexpr (EIGHT) {
        uint32_t turned[kPer], opposite[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            turned[j] = ((noise[j] << 8) | (noise[j] >> 8)) & 0xffffu;
            opposite[j] = 0xffffu - noise[j];
        }
        uint32_t scale;
        const bool leads = left > 0 && (threadIdx.x & 15) == 0;
        store8_codes(t.m, at, left, encode8<false>(m, turned, scale));
        if (leads) as_global(t.m_scale)[at / kBlock] = static_cast<uint8_t>(scale);
        store8_codes(t.v, at, left, encode8<true>(v, opposite, scale));
        if (leads) as_global(t.v_scale)[at / kBlock] = static_cast<uint8_t>(scale);
    } else {
        store8_f32(t.m, at, left, m);
        store8_f32(t.v, at, left, v);
    }
}
// step counts kept on the device, one more each
struct CountArgs {
    float *at[256];
    int n;
};

__global__ __launch_bounds__(256) void count_steps_kernel(const CountArgs a) {
    const int i = static_cast<int>(threadIdx.x);
    if (i < a.n) *a.at[i] += 1.f;
}

template <bool P16, bool G16, bool EIGHT>
void launch(const Args &a, int64_t chunks, hipStream_t s) {
    hipLaunchKernelGGL((adamw_kernel<P16, G16, EIGHT>), dim3(static_cast<unsigned>(chunks)), dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace me

using namespace me;

extern "C" int me_adamw(int32_t n_tensors, void *const *params, const void *const *grads, void *const *exp_avgs,
                        void *const *exp_avg_sqs, void *const *exp_avg_scales, void *const *exp_avg_sq_scales,
                        const int64_t *numels, const double *steps, float *const *device_steps,
                        const int32_t *stream_ids, int param_dtype, int grad_dtype, int state_bits, double lr,
                        double beta1, double beta2, double eps, double weight_decay, int stochastic_rounding,
                        uint64_t seed, void *stream) {
    ME_CHECK_ARG(n_tensors >= 0, "n_tensors must be non-negative");
    if (n_tensors == 0) return ME_OK;
    ME_CHECK_ARG(params && grads && exp_avgs && exp_avg_sqs && numels && stream_ids && (steps || device_steps),
                 "null argument array");
    ME_CHECK_ARG(param_dtype == ME_BF16 || param_dtype == ME_F32, "param dtype must be bf16/fp32");
    ME_CHECK_ARG(grad_dtype == ME_BF16 || grad_dtype == ME_F32, "grad dtype must be bf16/fp32");
    ME_CHECK_ARG(state_bits == 32 || state_bits == 8, "state_bits must be 32 or 8");
    ME_CHECK_ARG(state_bits == 32 || (exp_avg_scales && exp_avg_sq_scales), "8-bit moments need their scales");
    ME_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must be in [0, 1)");
    for (int k = 0; k < n_tensors; ++k) {
        ME_CHECK_ARG(numels[k] >= 0, "tensor %d: negative size", k);
        ME_CHECK_ARG(ceil_div(numels[k], kChunk) <= kMostChunks, "tensor %d: more than 2^34 values", k);
        ME_CHECK_ARG(device_steps ? device_steps[k] != nullptr : steps[k] >= 1, "tensor %d: step must be >= 1", k);
        if (numels[k] == 0) continue;
        ME_CHECK_ARG(params[k] && grads[k] && exp_avgs[k] && exp_avg_sqs[k], "tensor %d: null tensor pointer", k);
        ME_CHECK_ARG(state_bits == 32 || (exp_avg_scales[k] && exp_avg_sq_scales[k]), "tensor %d: null scales", k);
        const uintptr_t pa = param_dtype == ME_BF16 ? 2 : 4, ga = grad_dtype == ME_BF16 ? 2 : 4, sa = state_bits == 32 ? 4 : 1;
        ME_CHECK_ARG(reinterpret_cast<uintptr_t>(params[k]) % pa == 0 && reinterpret_cast<uintptr_t>(grads[k]) % ga == 0 &&
                         reinterpret_cast<uintptr_t>(exp_avgs[k]) % sa == 0 && reinterpret_cast<uintptr_t>(exp_avg_sqs[k]) % sa == 0,
                     "tensor %d: not aligned to its elements", k);
    }
    hipStream_t s = as_stream(stream);
    if (device_steps) {
        for (int k0 = 0; k0 < n_tensors; k0 += 256) {
            CountArgs c{};
            c.n = std::min(256, n_tensors - k0);
            for (int i = 0; i < c.n; ++i) c.at[i] = device_steps[k0 + i];
            hipLaunchKernelGGL(count_steps_kernel, dim3(1), dim3(256), 0, s, c);
            const int rc = check_launch("me_adamw");
            if (rc != ME_OK) return rc;
        }
    }
    Args a{};
    a.beta1 = static_cast<float>(beta1);
    a.beta2 = static_cast<float>(beta2);
    a.rest1 = static_cast<float>(1.0 - beta1);
    a.rest2 = static_cast<float>(1.0 - beta2);
    a.eps = static_cast<float>(eps);
    a.decay = static_cast<float>(1.0 - lr * weight_decay);
    a.lr = lr;
    a.log_beta1 = std::log(beta1);
    a.log_beta2 = std::log(beta2);
    a.seed = seed;
    a.sr = stochastic_rounding != 0;
    const bool p16 = param_dtype == ME_BF16, g16 = grad_dtype == ME_BF16, eight = state_bits == 8;
    int64_t chunks = 0;
    auto flush = [&]() {
        if (a.n_tensors == 0) return ME_OK;
        if (eight) {
            if (p16) g16 ? launch<true, true, true>(a, chunks, s) : launch<true, false, true>(a, chunks, s);
            else g16 ? launch<false, true, true>(a, chunks, s) : launch<false, false, true>(a, chunks, s);
        } else {
            if (p16) g16 ? launch<true, true, false>(a, chunks, s) : launch<true, false, false>(a, chunks, s);
            else g16 ? launch<false, true, false>(a, chunks, s) : launch<false, false, false>(a, chunks, s);
        }
        a.n_tensors = 0;
        chunks = 0;
        return check_launch("me_adamw");
    };
    for (int k = 0; k < n_tensors; ++k) {
        if (numels[k] == 0) continue;
        const int64_t own = ceil_div(numels[k], kChunk);
        if (a.n_tensors == kTensors || chunks + own > kMostChunks) {
            const int rc = flush();
            if (rc != ME_OK) return rc;
        }
        Tensor &t = a.t[a.n_tensors];
        t = Tensor{};
        t.p = static_cast<uint8_t *>(params[k]);
        t.g = static_cast<const uint8_t *>(grads[k]);
        t.m = static_cast<uint8_t *>(exp_avgs[k]);
        t.v = static_cast<uint8_t *>(exp_avg_sqs[k]);
        if (eight) {
            t.m_scale = static_cast<uint8_t *>(exp_avg_scales[k]);
            t.v_scale = static_cast<uint8_t *>(exp_avg_sq_scales[k]);
        }
        t.n = numels[k];
        t.stream = static_cast<uint32_t>(stream_ids[k]);
        if (device_steps) {
            t.step_at = device_steps[k];
        } else {
            t.step_size = static_cast<float>(lr / (1.0 - std::pow(beta1, steps[k])));
            t.inv_sqrt_bc2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, steps[k])));
            t.step = static_cast<uint32_t>(steps[k]);
        }
        a.first[a.n_tensors++] = static_cast<int32_t>(chunks);
        chunks += own;
    }
    return flush();
}
