// Losses over a decoder's head without its logits on gfx950: from hidden states h [n, dim] and head
// W [vocab, dim], with z_ij = h_i . w_j / T, q = softmax(z), o_i = 1 - q_it at the row's target t,
//
//   log q_it = -log(1 + sum_{j != t} exp(z_ij - z_it))                                  (me_head_logps)
//   lse_i - (1 - e) z_it - e / V sum_j z_ij + lam lse_i^2, summed or averaged over rows  (me_head_ce)
//   dz_ij = ca_i q_ij - cb_i (j != t), gt_i (j = t);  dh = dz W / T,  dW = dz^T h / T     (me_head_backward)
//
// (the reference trains with a cross-entropy in pieces of its logits, micro_engram/train/head.py:85-165).
// No pass keeps logits: the forward's product reduces each tile of them to a maximum and a sum per row as it leaves the
// matrix cores; the backward's makes the tile again, writes its gradient in bf16 for a piece of the vocabulary,
// and that piece goes through the products with W and with h. Rows that do not count are left out at the
// start (rows of the products are those that count, gathered), so a padded batch costs what its tokens cost, and
// nothing that stands in such a row is read.
//
// A row's target is kept out of the sums, as in the losses over logits: the weight of the others, and with it the
// loss and the gradient at the target, keeps its digits where the target is all but certain.
// Statistics are fp32; the logits' gradient is rounded to bf16 once (fp32 operands: three parts, exact) before its
// products: one rounding of 2^-9 per term where the sum itself is rounded so at its end.
#include "head_gemm.h"

#include <algorithm>
#include <cmath>

namespace me {
namespace {

using namespace head;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr int64_t kFew = 128;                            // rows up to which the 64-row tiles are taken
constexpr int64_t kPieceBytes = int64_t{512} << 20;      // of a piece's gradient, and of a piece of laid-out weights
constexpr int kHeader = 16;                              // ints before the rows in `saved`: the number of them

// What the forward leaves for the backward: counted rows, and by counted row its source, log2-sum and o; by source
// row its place among the counted ones.
struct Saved {
    int32_t *count, *rows, *place;
    float *lse2, *others;
};

Saved saved_of(void *p, int64_t n) {
    int32_t *i = static_cast<int32_t *>(p);
    float *f = static_cast<float *>(p);
    return {i, i + kHeader, i + kHeader + n, f + kHeader + 2 * n, f + kHeader + 3 * n};
}

// ---- rows that count -------------------------------------------------------------------------------------------
// One workgroup: rows[r] = source of the r-th counted row, place[i] = r or -1, tgt[r] its target.
constexpr int kIndexThreads = 1024;

template <typename T>
__global__ __launch_bounds__(kIndexThreads) void index_kernel(const T *targets, int64_t n, int64_t ignore, int64_t vocab,
                                                              Saved s, int32_t *tgt) {
    __shared__ int sums[kIndexThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int at = 0;
    for (int64_t i0 = 0; i0 < n; i0 += kIndexThreads) {
        const int64_t i = i0 + tid;
        const int64_t t = i < n ? static_cast<int64_t>(targets[i]) : -1;
        const bool ok = i < n && t != ignore && t >= 0 && t < vocab;
        const uint64_t mask = __ballot(ok);
        if (lane == 0) sums[wave] = __popcll(mask);
        __syncthreads();
        int before = at, all = 0;
        for (int w = 0; w < kIndexThreads / 64; ++w) {
            before += w < wave ? sums[w] : 0;
            all += sums[w];
        }
        const int r = before + __popcll(mask & ((uint64_t{1} << lane) - 1));
        if (i < n) s.place[i] = ok ? r : -1;
        if (ok) {
            s.rows[r] = static_cast<int32_t>(i);
            tgt[r] = static_cast<int32_t>(t);
        }
        at += all;
        __syncthreads();
    }
    if (tid == 0) *s.count = at;
}

template <typename T>
__global__ __launch_bounds__(256) void targets_kernel(const T *targets, int64_t n, const int32_t *rows, const int32_t *count, int32_t *tgt) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r < n && r < *count) tgt[r] = static_cast<int32_t>(targets[rows[r]]);
}

// ---- operands as the products read them: [rows][ld] bf16, ld a multiple of 64, zeros past dim; fp32 in three parts -----
struct Layout {
    const void *src;
    int64_t per_batch, batch_stride, row_stride;  // row r: (r / per_batch) * batch_stride + (r % per_batch) * row_stride
    const int32_t *rows, *count;                  // sources of the rows and how many there are; null: as they are
    int64_t n, dim, ld, part;                     // part: bytes
    uint8_t *dst;
};

// x as three bf16 that add up to it: each the nearest bf16 of what remains. What is not finite stands in the
// first part alone.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
    p[0] = float_to_bf16_bits_rne(x);
    float rest = x - bf16_bits_to_float(p[0]);
    if (!(__builtin_fabsf(rest) < __builtin_inff())) rest = 0.f;
    p[1] = float_to_bf16_bits_rne(rest);
    p[2] = float_to_bf16_bits_rne(rest - bf16_bits_to_float(p[1]));
}

template <bool F32>
__global__ __launch_bounds__(256) void layout_kernel(const Layout a) {
    const int64_t units = a.ld / 8;
    const int64_t n = a.count ? min(a.n, static_cast<int64_t>(*a.count)) : a.n;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < n * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = u / units, c = (u - r * units) * 8;
        const int64_t from = a.rows ? a.rows[r] : r;
        const int64_t at = from / a.per_batch * a.batch_stride + from % a.per_batch * a.row_stride + c;
        uint32_t w[3][4] = {};
        uint16_t(&h)[3][8] = reinterpret_cast<uint16_t(&)[3][8]>(w);
        if constexpr (F32) {
            const float *src = static_cast<const float *>(a.src) + at;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint16_t p[3];
                split3(c + j < a.dim ? src[j] : 0.f, p);
                h[0][j] = p[0], h[1][j] = p[1], h[2][j] = p[2];
            }
        } else {
            const uint16_t *src = static_cast<const uint16_t *>(a.src) + at;
            if (c + 8 <= a.dim && reinterpret_cast<uintptr_t>(src) % 16 == 0) {
                const u32x4_v x = *as_global(reinterpret_cast<const u32x4_v *>(src));
#pragma unroll
                for (int j = 0; j < 4; ++j) w[0][j] = x[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[0][j] = c + j < a.dim ? src[j] : 0;
            }
        }
#pragma unroll
        for (int p = 0; p < (F32 ? 3 : 1); ++p)
            *as_global(reinterpret_cast<u32x4_v *>(a.dst + p * a.part + (r * a.ld + c) * 2)) = u32x4_v{w[p][0], w[p][1], w[p][2], w[p][3]};
    }
}

// ---- epilogues -----------------------------------------------------------------------------------------------
// acc[x][y][4 g + e] is row row0 + 32 y + (lane & 31), column col0 + 32 x + 8 g + 4 (lane >> 5) + e of the tile.

// Statistics of a tile's rows over a wave's columns, in units of log2: their maximum and sum without the target,
// the target's own value, and where wanted the plain sum of the values.
struct StatsEpilogue {
    const int32_t *tgt;
    float2 *part;            // by (column part, row): part * part_stride + row * row_stride
    float *sum;              // likewise, or null
    float *at_target;        // by row
    int64_t part_stride, row_stride;
    int64_t first, vocab;    // of the piece: first column, columns that there are
    float k;                 // log2(e) / T

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *, int lane) const {
        const int64_t c0 = t.s0 + col0;
        const int there = static_cast<int>(max(min(vocab - c0, int64_t{32 * SX}), int64_t{0}));
        const int64_t part_at = (first + c0) / (32 * SX);
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            const bool ok = row < t.rows;
            const int64_t off = ok ? tgt[row] - (first + c0) : -1;
            const int mine = off >= 0 && off < there ? static_cast<int>(off) : -1;
            // few waves hold a target of their rows, or the vocabulary's end
            if (there < 32 * SX || __any(mine >= 0))
                row_part<AGPR, true, SX, SY>(acc, y, row, ok, mine, there, part_at, lane);
            else
                row_part<AGPR, false, SX, SY>(acc, y, row, ok, mine, there, part_at, lane);
        }
    }

    template <bool AGPR, bool SOME, int SX, int SY>
    __device__ __forceinline__ void row_part(const floatx16 (&acc)[SX][SY], int y, int64_t row, bool ok, int mine, int there, int64_t part_at,
                                             int lane) const {
        const int half4 = 4 * (lane >> 5);
        float m = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = acc_read<AGPR>(acc[x][y], e);
                if constexpr (SOME) {
                    const int col = 32 * x + 8 * (e >> 2) + half4 + (e & 3);
                    total += col < there ? v : 0.f;
                    if (col == mine) at_target[row] = v * k;
                    if (col == mine || col >= there) v = -__builtin_inff();
                } else {
                    total += v;
                }
                m = fmaxf(m, v);
            }
        m = fmaxf(m, __shfl_xor(m, 32)) * k;
        const float shift = m == -__builtin_inff() ? 0.f : m;
        float s = 0.f;
        if constexpr (SOME) asm volatile("" : "+v"(mine), "+s"(there));  // compared anew: 64 lane masks are not kept
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = acc_read<AGPR>(acc[x][y], e);
                if constexpr (SOME) {
                    const int col = 32 * x + 8 * (e >> 2) + half4 + (e & 3);
                    if (col == mine || col >= there) v = -__builtin_inff();
                }
                s += __builtin_amdgcn_exp2f(fmaf(v, k, -shift));
            }
        s += __shfl_xor(s, 32);
        total += __shfl_xor(total, 32);
        if (ok && lane < 32) {
            part[part_at * part_stride + row * row_stride] = make_float2(m, s);
            if (sum != nullptr) sum[part_at * part_stride + row * row_stride] = total * k;
        }
    }
};

struct RowGrad {
    float lse2, ca, cb, gt;
};

// The logits' gradient of a tile, bf16 or in three parts, as rows of a piece
template <int NPARTS>
struct GradEpilogue {
    const int32_t *tgt;
    const RowGrad *grad;
    uint8_t *out;          // [rows][ld] of each part
    int64_t ld, part;      // ld: columns of the piece, a multiple of 64; part: bytes
    int64_t first, vocab;  // first column of the piece, columns that there are
    float k;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        const int64_t c0 = t.s0 + col0;
        const int there = static_cast<int>(max(min(vocab - c0, int64_t{32 * SX}), int64_t{0}));
        constexpr int kPitch = 64 * SX + 16;  // staged row (bytes)
        constexpr int kChunks = 4 * SX;
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            // 32 rows at a time through LDS, where a wave has two places in turn (with three parts one: a wave's
            // LDS accesses keep their order)
            constexpr int kPlaces = NPARTS == 1 ? 2 : 1;
            static_assert(4 * kPlaces * NPARTS * 32 * kPitch <= (SX == 4 ? kRingBytes : 3 * kUnit), "the stage fits the ring");
            uint8_t *stage = lds + ((threadIdx.x >> 6) * kPlaces + (y % kPlaces)) * (NPARTS * 32 * kPitch);
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            const bool ok = row < t.rows;
            const RowGrad g = ok ? grad[row] : RowGrad{0.f, 0.f, 0.f, 0.f};
            const int64_t off = ok ? tgt[row] - (first + c0) : -1;
            const int mine = off >= 0 && off < there ? static_cast<int>(off) : -1;
            if (there < 32 * SX || __any(mine >= 0))
                stage_rows<AGPR, true, SX, SY>(acc, y, g, mine, there, stage, lane);
            else
                stage_rows<AGPR, false, SX, SY>(acc, y, g, mine, there, stage, lane);
#pragma unroll
            for (int p = 0; p < NPARTS; ++p)
#pragma unroll 4
                for (int it = 0; it < 32 * kChunks / 64; ++it) {
                    const int ch = it * 64 + lane, r = ch / kChunks, cc = ch % kChunks;
                    const int64_t rg = t.r0 + row0 + 32 * y + r, cg = c0 + cc * 8;
                    const u32x4_v v = *reinterpret_cast<const u32x4_v *>(stage + (p * 32 + r) * kPitch + cc * 16);
                    if (rg < t.rows && cg < ld) *as_global(reinterpret_cast<u32x4_v *>(out + p * part + (rg * ld + cg) * 2)) = v;
                }
        }
    }

    template <bool AGPR, bool SOME, int SX, int SY>
    __device__ __forceinline__ void stage_rows(const floatx16 (&acc)[SX][SY], int y, const RowGrad &g, int mine, int there, uint8_t *stage,
                                               int lane) const {
        constexpr int kPitch = 64 * SX + 16;
        const int half4 = 4 * (lane >> 5);
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w[NPARTS][2];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = fmaf(__builtin_amdgcn_exp2f(fmaf(acc_read<AGPR>(acc[x][y], 4 * q + e), k, -g.lse2)), g.ca, -g.cb);
                    if constexpr (SOME) {
                        const int col = 32 * x + 8 * q + half4 + e;
                        if (col == mine) v = g.gt;
                        if (col >= there) v = 0.f;  // past the vocabulary: nothing for the products with W and h
                    }
#pragma unroll
                    for (int p = 0; p < NPARTS; ++p) {
                        const uint16_t b = float_to_bf16_bits_rne(v);
                        reinterpret_cast<uint16_t *>(w[p])[e] = b;
                        v -= bf16_bits_to_float(b);
                        if (p == 0 && NPARTS > 1 && !(__builtin_fabsf(v) < __builtin_inff())) v = 0.f;  // not finite: the first part alone
                    }
                }
#pragma unroll
                for (int p = 0; p < NPARTS; ++p)
                    *reinterpret_cast<uint2 *>(stage + (p * 32 + (lane & 31)) * kPitch + (32 * x + 8 * q + half4) * 2) = make_uint2(w[p][0], w[p][1]);
            }
    }
};

// fp32 sums of a tile, added to what earlier pieces left: [split][rows][ld]
struct AccumulateEpilogue {
    float *out;
    int64_t ld, split_stride;  // ld: a multiple of 4
    int add;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *, int lane) const {
        const int half4 = 4 * (lane >> 5);
        float *o = out + t.split * split_stride;
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            if (row >= t.rows) continue;
#pragma unroll
            for (int x = 0; x < SX; ++x) {
                const int64_t col = t.s0 + col0 + 32 * x + half4;
                const auto at = as_global(reinterpret_cast<f32x4_v *>(o + row * ld + col));
                f32x4_v v[4] = {};
                if (add) {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        if (col + 8 * g < ld) v[g] = at[2 * g];
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[g][e] += acc_read<AGPR>(acc[x][y], 4 * g + e);
                    if (col + 8 * g < ld) at[2 * g] = v[g];
                }
            }
        }
    }
};

// The head's gradient: rows of its own type, `dim` long
template <bool F32>
struct WeightEpilogue {
    uint8_t *out;
    int64_t dim;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        const int half4 = 4 * (lane >> 5);
        const bool whole = dim % 8 == 0;  // rows of whole 16-byte chunks
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            if (!F32 && whole) {
                constexpr int kPitch = 64 * SX + 16, kChunks = 4 * SX;
                static_assert(8 * 32 * kPitch <= kRingBytes, "the stage fits the ring");
                uint8_t *stage = lds + ((threadIdx.x >> 6) * 2 + (y & 1)) * (32 * kPitch);
#pragma unroll
                for (int x = 0; x < SX; ++x)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint32_t w[2];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            reinterpret_cast<uint16_t *>(w)[e] = float_to_bf16_bits_rne(acc_read<AGPR>(acc[x][y], 4 * g + e));
                        *reinterpret_cast<uint2 *>(stage + (lane & 31) * kPitch + (32 * x + 8 * g + half4) * 2) = make_uint2(w[0], w[1]);
                    }
#pragma unroll 4
                for (int it = 0; it < 32 * kChunks / 64; ++it) {
                    const int ch = it * 64 + lane, r = ch / kChunks, cc = ch % kChunks;
                    const int64_t rg = t.r0 + row0 + 32 * y + r, cg = t.s0 + col0 + cc * 8;
                    const u32x4_v v = *reinterpret_cast<const u32x4_v *>(stage + r * kPitch + cc * 16);
                    if (rg < t.rows && cg < dim) *as_global(reinterpret_cast<u32x4_v *>(out + (rg * dim + cg) * 2)) = v;
                }
                continue;
            }
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
#pragma unroll
            for (int x = 0; x < SX; ++x)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int64_t col = t.s0 + col0 + 32 * x + 8 * g + half4;
                    f32x4_v v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc_read<AGPR>(acc[x][y], 4 * g + e);
                    if (row >= t.rows) continue;
                    if (F32 && dim % 4 == 0) {
                        if (col < dim) *as_global(reinterpret_cast<f32x4_v *>(reinterpret_cast<float *>(out) + row * dim + col)) = v;
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < dim) {
                            if constexpr (F32)
                                reinterpret_cast<float *>(out)[row * dim + col + e] = v[e];
                            else
                                reinterpret_cast<uint16_t *>(out)[row * dim + col + e] = float_to_bf16_bits_rne(v[e]);
                        }
                }
        }
    }
};

// ---- rows' results ---------------------------------------------------------------------------------------------
struct FinishArgs {
    const float2 *part;
    const float *sum, *at_target;
    int64_t part_stride, row_stride;
    int parts;
    int64_t n, vocab;
    Saved s;
    float *logps;        // by source row, or null
    float *row_loss;     // by counted row, or null
    float smoothing, z_loss;
};

struct Sum2 {
    float m, s;
};

__device__ __forceinline__ Sum2 join(Sum2 a, Sum2 b) {
    const float m = fmaxf(a.m, b.m);
    const float shift = m == -__builtin_inff() ? 0.f : m;
    return {m, a.s * __builtin_amdgcn_exp2f(a.m - shift) + b.s * __builtin_amdgcn_exp2f(b.m - shift)};
}

// A row's parts joined: WIDE 256 threads per row (few rows), else 64 rows by four threads each
template <bool WIDE>
__global__ __launch_bounds__(256) void finish_kernel(const FinishArgs a) {
    constexpr int kSlices = WIDE ? 256 : 4;
    __shared__ Sum2 s_all[WIDE ? 4 : 256];
    __shared__ double s_sum[WIDE ? 4 : 256];
    const int tid = threadIdx.x, slice = WIDE ? tid : tid >> 6;
    const int64_t r = WIDE ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 64 + (tid & 63);
    const int64_t count = *a.s.count;
    if (WIDE ? r >= count : static_cast<int64_t>(blockIdx.x) * 64 >= count) return;
    Sum2 all = {-__builtin_inff(), 0.f};
    double sum = 0.0;
    if (r < count) {
        for (int p = slice; p < a.parts; p += kSlices) {
            const float2 x = a.part[p * a.part_stride + r * a.row_stride];
            all = join(all, {x.x, x.y});
            if (a.sum) sum += a.sum[p * a.part_stride + r * a.row_stride];
        }
    }
    if constexpr (WIDE) {
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            all = join(all, {__shfl_xor(all.m, d), __shfl_xor(all.s, d)});
            sum += __shfl_xor(sum, d);
        }
        if ((tid & 63) == 0) s_all[tid >> 6] = all, s_sum[tid >> 6] = sum;
    } else {
        s_all[tid] = all, s_sum[tid] = sum;
    }
    __syncthreads();
    if (WIDE ? tid != 0 : (tid >= 64 || r >= count)) return;
    constexpr int kStep = WIDE ? 1 : 64;
    all = s_all[tid], sum = s_sum[tid];
#pragma unroll
    for (int i = 1; i < 4; ++i) all = join(all, s_all[tid + i * kStep]), sum += s_sum[tid + i * kStep];
    // d: how far the others' sum is over the target, log2
    const float zt = a.at_target[r], rest = all.m + log2f(all.s);
    const float d = rest - zt;
    const float e = exp2f(-fabsf(d)), more = log1pf(e);
    const float nll = static_cast<float>(kLn2) * fmaxf(d, 0.f) + more;
    const float others = d > 0.f ? 1.f / (1.f + e) : e / (1.f + e);
    const float lse2 = (d > 0.f ? rest : zt) + more * kLog2e;
    a.s.lse2[r] = lse2;
    a.s.others[r] = d != d ? d : others;
    if (a.logps) a.logps[a.s.rows[r]] = -nll;
    if (a.row_loss) {
        const float lse = static_cast<float>(kLn2) * lse2;
        float loss = nll + a.z_loss * lse * lse;
        if (a.smoothing != 0.f) loss += a.smoothing * static_cast<float>(kLn2 * (zt - sum / static_cast<double>(a.vocab)));
        a.row_loss[r] = loss;
    }
}

__global__ __launch_bounds__(256) void uncounted_logps_kernel(const int32_t *place, int64_t n, float *logps) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < n && place[i] < 0) logps[i] = 0.f;
}

__global__ __launch_bounds__(1024) void total_kernel(const float *row_loss, const int32_t *count, double scale, int mean, float *loss) {
    __shared__ double s[16];
    const int n = *count;
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) sum += static_cast<double>(row_loss[i]);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int i = 0; i < 16; ++i) sum += s[i];
        *loss = static_cast<float>(sum * scale / (mean ? max(n, 1) : 1));
    }
}

struct CoefArgs {
    Saved s;
    int64_t n;
    const float *upstream;  // by source row (per_row) or one
    int per_row, mean;
    double scale;           // of the loss, over T
    float smoothing, z_loss;
    double vocab;
    RowGrad *grad;
};

__global__ __launch_bounds__(256) void coef_kernel(const CoefArgs a) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t count = *a.s.count;
    if (r >= a.n || r >= count) return;
    const float lse2 = a.s.lse2[r], o = a.s.others[r];
    RowGrad g;
    g.lse2 = lse2;
    if (a.per_row) {  // log-probabilities: -upstream times the loss -log q
        const float c = static_cast<float>(-static_cast<double>(a.upstream[a.s.rows[r]]) * a.scale);
        g.ca = c, g.cb = 0.f, g.gt = -c * o;
    } else {
        const double c = static_cast<double>(*a.upstream) * a.scale / (a.mean ? static_cast<double>(max(count, int64_t{1})) : 1.0);
        const double more = 2.0 * a.z_loss * kLn2 * lse2, e = a.smoothing;
        g.ca = static_cast<float>(c * (1.0 + more));
        g.cb = static_cast<float>(c * e / a.vocab);
        g.gt = static_cast<float>(c * (more - (1.0 + more) * o + e - e / a.vocab));
    }
    a.grad[r] = g;
}

// Gradient of the hidden states, source rows in their order: the splits' sums, or zeros
template <bool F32>
__global__ __launch_bounds__(256) void hidden_kernel(const float *sums, int64_t ld, int64_t split_stride, int splits, const int32_t *place,
                                                     int64_t n, int64_t dim, void *out) {
    const int64_t units = ceil_div(dim, 4);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < n * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t i = u / units, c = (u - i * units) * 4;
        const int64_t r = place[i];
        f32x4_v v = {0.f, 0.f, 0.f, 0.f};
        if (r >= 0)
            for (int s = 0; s < splits; ++s) v += *as_global(reinterpret_cast<const f32x4_v *>(sums + s * split_stride + r * ld + c));
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < dim) {
                if constexpr (F32)
                    static_cast<float *>(out)[i * dim + c + e] = v[e];
                else
                    static_cast<uint16_t *>(out)[i * dim + c + e] = float_to_bf16_bits_rne(v[e]);
            }
    }
}

// ---- plan: sizes and places in the workspace ---------------------------------------------------------------------
struct Plan {
    int64_t n, vocab, dim, ld;  // ld: dim rounded up to whole slabs
    bool f32, few, copy_w;      // copy_w: the head is laid out piece by piece
    int np;                     // parts of an operand
    int64_t piece;              // columns of the vocabulary at a time
    int splits;                 // of the product with W
    int64_t h, tgt, part, sum, at_target, row_loss, w, g, grad, acc;  // workspace offsets
    int64_t bytes;
};

int64_t round_up(int64_t x, int64_t to) { return ceil_div(x, to) * to; }

// Splits of the reduction over a piece so that the last round of tiles is as full as it gets; each costs a pass over
// the sums.
int splits_of(int64_t tiles, int64_t at_once, int64_t slabs) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 16 && s <= std::max<int64_t>(1, slabs / 8); ++s) {
        const double cost = static_cast<double>(ceil_div(tiles * s, at_once)) / s + 0.01 * s;
        if (cost < least - 1e-9) least = cost, best = s;
    }
    return best;
}

Plan plan_of(int64_t n, int64_t vocab, int64_t dim, int dtype, const void *weight, int64_t w_stride, bool backward) {
    Plan p{};
    p.n = n, p.vocab = vocab, p.dim = dim, p.ld = round_up(dim, kSlabK);
    p.f32 = dtype == ME_F32;
    p.np = p.f32 ? 3 : 1;
    p.few = n <= kFew;
    p.copy_w = p.f32 || w_stride % 8 != 0 || reinterpret_cast<uintptr_t>(weight) % 16 != 0;
    int64_t piece = round_up(vocab, kTile);
    const int64_t rows = round_up(std::max<int64_t>(n, 1), 64);
    if (p.copy_w) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (p.ld * 2 * p.np) / 2048 * 2048, 2048));
    if (backward) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (rows * 2 * p.np) / 2048 * 2048, 2048));
    // a launch holds fewer than 2^32 threads
    p.piece = std::min(piece, std::max<int64_t>((int64_t{1} << 23) / ceil_div(rows, p.few ? 64 : kTile) * kTile / 2048 * 2048, 2048));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    p.h = take(rows * p.ld * 2 * p.np);
    p.tgt = take(n * 4);
    if (p.copy_w) p.w = take(p.piece * p.ld * 2 * p.np);
    if (!backward) {
        const int64_t parts = ceil_div(vocab, p.few ? 64 : 128) + 4;
        p.part = take(parts * rows * 8);
        p.sum = take(parts * rows * 4);
        p.at_target = take(n * 4);
        p.row_loss = take(n * 4);
    } else {
        p.g = take(rows * p.piece * 2 * p.np);
        p.grad = take(n * static_cast<int64_t>(sizeof(RowGrad)));
        p.splits = splits_of(ceil_div(n, p.few ? 64 : kTile) * ceil_div(dim, kTile), p.few ? 512 : 256, p.piece / kSlabK);
        p.acc = take(p.splits * rows * p.ld * 4);
    }
    p.bytes = at;
    return p;
}

struct Call {
    const void *hidden, *weight, *targets;
    int64_t per_batch, batch_stride, row_stride, w_stride, ignore;
    int tdtype;
    uint8_t *ws;
    Saved s;
    hipStream_t stream;
};

unsigned blocks_for(int64_t units) { return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(units, 256), 1), 16384)); }

void lay_out(bool f32, const Layout &l, hipStream_t s) {
    const unsigned blocks = blocks_for(l.n * (l.ld / 8));
    if (f32)
        hipLaunchKernelGGL(layout_kernel<true>, dim3(blocks), dim3(256), 0, s, l);
    else
        hipLaunchKernelGGL(layout_kernel<false>, dim3(blocks), dim3(256), 0, s, l);
}

int64_t h_part(const Plan &p) { return round_up(std::max<int64_t>(p.n, 1), 64) * p.ld * 2; }

void lay_out_hidden(const Plan &p, const Call &c) {
    lay_out(p.f32, Layout{c.hidden, c.per_batch, c.batch_stride, c.row_stride, c.s.rows, c.s.count, p.n, p.dim, p.ld, h_part(p), c.ws + p.h}, c.stream);
}

Operand hidden_operand(const Plan &p, const Call &c) { return {c.ws + p.h, p.ld, h_part(p)}; }

// The head from row v0 on, `width` rows of it
Operand weight_operand(const Plan &p, const Call &c, int64_t v0, int64_t width) {
    const uint8_t *from = static_cast<const uint8_t *>(c.weight) + v0 * c.w_stride * (p.f32 ? 4 : 2);
    if (!p.copy_w) return {from, c.w_stride, 0};
    const int64_t part = p.piece * p.ld * 2;
    lay_out(p.f32, Layout{from, width, 0, c.w_stride, nullptr, nullptr, width, p.dim, p.ld, part, c.ws + p.w}, c.stream);
    return {c.ws + p.w, p.ld, part};
}

template <bool A_KC, bool B_KC, int SEGS, class Epilogue>
void multiply_large(const Gemm &g, const Epilogue &e, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(workgroups(g, kTile, kTile)));
    hipLaunchKernelGGL((large_kernel<A_KC, B_KC, SEGS, Epilogue>), grid, dim3(kThreads), 0, s, g, e);
}

template <bool B_KC, int SEGS, class Epilogue>
void multiply_few(const Gemm &g, const Epilogue &e, hipStream_t s) {
    constexpr int kTS = 256, kRing = 3;
    const dim3 grid(static_cast<unsigned>(workgroups(g, 64, kTS)));
    hipLaunchKernelGGL((few_kernel<B_KC, kTS, kRing, SEGS, Epilogue>), grid, dim3(kThreads), 0, s, g, e);
}

// logits of a piece: hidden [counted rows] x head rows
template <int SEGS, class Epilogue>
void logits_of(const Plan &p, const Call &c, const Operand &w, int64_t width, const Epilogue &e) {
    Gemm g{hidden_operand(p, c), w, p.n, width, p.dim, c.s.count, 0, 8, 1};
    if (p.few)
        multiply_few<true, SEGS>(g, e, c.stream);
    else
        multiply_large<true, true, SEGS>(g, e, c.stream);
}

int forward(const Plan &p, const Call &c, double temperature, float *logps, float *loss, double smoothing, double z_loss, double scale, int mean) {
    int32_t *tgt = reinterpret_cast<int32_t *>(c.ws + p.tgt);
    if (c.tdtype == ME_I64)
        hipLaunchKernelGGL(index_kernel<int64_t>, dim3(1), dim3(kIndexThreads), 0, c.stream, static_cast<const int64_t *>(c.targets), p.n, c.ignore, p.vocab, c.s, tgt);
    else
        hipLaunchKernelGGL(index_kernel<int32_t>, dim3(1), dim3(kIndexThreads), 0, c.stream, static_cast<const int32_t *>(c.targets), p.n, c.ignore, p.vocab, c.s, tgt);
    FinishArgs f{};
    if (p.n > 0) {
        lay_out_hidden(p, c);
        const int cols = p.few ? 64 : 128;
        const int64_t rows = round_up(p.n, 64);
        StatsEpilogue e{};
        e.tgt = tgt;
        e.part = reinterpret_cast<float2 *>(c.ws + p.part);
        e.sum = smoothing != 0.0 ? reinterpret_cast<float *>(c.ws + p.sum) : nullptr;
        e.at_target = reinterpret_cast<float *>(c.ws + p.at_target);
        const int parts = static_cast<int>(ceil_div(p.vocab, cols));
        e.part_stride = p.few ? 1 : rows;
        e.row_stride = p.few ? parts + 4 : 1;
        e.k = static_cast<float>(1.44269504088896340736 / temperature);
        for (int64_t v0 = 0; v0 < p.vocab; v0 += p.piece) {
            const int64_t width = std::min(p.piece, p.vocab - v0);
            e.first = v0, e.vocab = width;
            const Operand w = weight_operand(p, c, v0, width);
            if (p.f32)
                logits_of<6>(p, c, w, width, e);
            else
                logits_of<1>(p, c, w, width, e);
        }
        f.part = e.part, f.sum = e.sum, f.at_target = e.at_target, f.part_stride = e.part_stride, f.row_stride = e.row_stride, f.parts = parts;
        f.n = p.n, f.vocab = p.vocab, f.s = c.s, f.logps = logps;
        f.row_loss = loss ? reinterpret_cast<float *>(c.ws + p.row_loss) : nullptr;
        f.smoothing = static_cast<float>(smoothing), f.z_loss = static_cast<float>(z_loss);
        if (p.few)
            hipLaunchKernelGGL(finish_kernel<true>, dim3(static_cast<unsigned>(p.n)), dim3(256), 0, c.stream, f);
        else
            hipLaunchKernelGGL(finish_kernel<false>, dim3(static_cast<unsigned>(ceil_div(p.n, 64))), dim3(256), 0, c.stream, f);
        if (logps)
            hipLaunchKernelGGL(uncounted_logps_kernel, dim3(static_cast<unsigned>(ceil_div(p.n, 256))), dim3(256), 0, c.stream, c.s.place, p.n, logps);
    }
    if (loss) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, c.stream, reinterpret_cast<const float *>(c.ws + p.row_loss), c.s.count, scale, mean, loss);
    return check_launch("me_head");
}

int check_call(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t per_batch, const void *weight, int64_t vocab, int64_t w_stride,
               const void *targets, int tdtype, double temperature, const void *saved, const void *ws) {
    ME_CHECK_ARG(dtype == ME_BF16 || dtype == ME_F32, "dtype must be bf16/fp32");
    ME_CHECK_ARG(tdtype == ME_I32 || tdtype == ME_I64, "targets must be int32/int64");
    ME_CHECK_ARG(n >= 0 && n <= (int64_t{1} << 24), "n must be in 0..2^24");
    ME_CHECK_ARG(dim >= 1 && dim <= 65536, "dim must be in 1..65536");
    ME_CHECK_ARG(ceil_div(n, 256) * ceil_div(dim, 256) <= (int64_t{1} << 23), "n times dim must be at most 2^39");
    ME_CHECK_ARG(vocab >= 1 && vocab <= (int64_t{1} << 21), "vocab must be in 1..2^21");
    ME_CHECK_ARG(w_stride >= dim && w_stride <= (int64_t{1} << 22), "weight rows must be dim or more elements apart, at most 2^22");
    ME_CHECK_ARG(n == 0 || (hidden && targets && per_batch >= 1), "hidden and targets are needed");
    ME_CHECK_ARG(weight && saved && ws, "weight, saved and workspace are needed");
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(saved) % 16 == 0 && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "saved and workspace must be 16-byte aligned");
    ME_CHECK_ARG(temperature >= 1e-6 && temperature <= 1e6, "temperature is out of range");
    return ME_OK;
}

}  // namespace
}  // namespace me

using namespace me;

extern "C" int me_head_workspace_size(int64_t n, int64_t vocab, int64_t dim, int dtype, const void *weight, int64_t w_stride, int backward,
                                      size_t *bytes) {
    ME_CHECK_ARG(bytes && n >= 0 && vocab >= 1 && dim >= 1, "bad sizes");
    *bytes = static_cast<size_t>(plan_of(n, vocab, dim, dtype, weight, w_stride, backward != 0).bytes);
    return ME_OK;
}

extern "C" int me_head_logps(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                             int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets, int targets_dtype,
                             int64_t ignore_index, double temperature, float *logps, void *saved, void *workspace, size_t workspace_bytes,
                             void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved, workspace);
    if (rc != ME_OK) return rc;
    const Plan p = plan_of(n, vocab, dim, dtype, weight, w_stride, false);
    ME_CHECK_ARG(workspace_bytes >= static_cast<size_t>(p.bytes), "workspace of %zu bytes, %lld are needed", workspace_bytes, static_cast<long long>(p.bytes));
    ME_CHECK_ARG(n == 0 || logps, "logps is needed");
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_of(saved, n), as_stream(stream)};
    return forward(p, c, temperature, logps, nullptr, 0.0, 0.0, 1.0, 0);
}

extern "C" int me_head_ce(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                          int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets, int targets_dtype,
                          int64_t ignore_index, double temperature, double smoothing, double z_loss, double scale, int reduction, float *loss,
                          void *saved, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved, workspace);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(reduction == ME_REDUCE_MEAN || reduction == ME_REDUCE_SUM, "reduction must be mean or sum");
    ME_CHECK_ARG(loss, "loss is needed");
    const Plan p = plan_of(n, vocab, dim, dtype, weight, w_stride, false);
    ME_CHECK_ARG(workspace_bytes >= static_cast<size_t>(p.bytes), "workspace of %zu bytes, %lld are needed", workspace_bytes, static_cast<long long>(p.bytes));
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_of(saved, n), as_stream(stream)};
    return forward(p, c, temperature, nullptr, loss, smoothing, z_loss, scale, reduction == ME_REDUCE_MEAN);
}

extern "C" int me_head_backward(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                                int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets,
                                int targets_dtype, int64_t ignore_index, double temperature, const float *upstream, int upstream_per_row,
                                double smoothing, double z_loss, double scale, int reduction, const void *saved, void *grad_hidden,
                                void *grad_weight, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved, workspace);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(upstream || (n == 0 && upstream_per_row), "upstream is needed");
    const Plan p = plan_of(n, vocab, dim, dtype, weight, w_stride, true);
    ME_CHECK_ARG(workspace_bytes >= static_cast<size_t>(p.bytes), "workspace of %zu bytes, %lld are needed", workspace_bytes, static_cast<long long>(p.bytes));
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(grad_hidden) % 16 == 0 && reinterpret_cast<uintptr_t>(grad_weight) % 16 == 0, "gradients must be 16-byte aligned");
    if (!grad_hidden && !grad_weight) return ME_OK;
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_of(const_cast<void *>(saved), n), as_stream(stream)};
    hipStream_t s = c.stream;
    int32_t *tgt = reinterpret_cast<int32_t *>(c.ws + p.tgt);
    RowGrad *grad = reinterpret_cast<RowGrad *>(c.ws + p.grad);
    const unsigned row_blocks = static_cast<unsigned>(std::max<int64_t>(ceil_div(n, 256), 1));
    if (n > 0) {
        if (targets_dtype == ME_I64)
            hipLaunchKernelGGL(targets_kernel<int64_t>, dim3(row_blocks), dim3(256), 0, s, static_cast<const int64_t *>(targets), n, c.s.rows, c.s.count, tgt);
        else
            hipLaunchKernelGGL(targets_kernel<int32_t>, dim3(row_blocks), dim3(256), 0, s, static_cast<const int32_t *>(targets), n, c.s.rows, c.s.count, tgt);
        CoefArgs k{c.s, n, upstream, upstream_per_row != 0, reduction == ME_REDUCE_MEAN, scale / temperature, static_cast<float>(smoothing),
                   static_cast<float>(z_loss), static_cast<double>(vocab), grad};
        hipLaunchKernelGGL(coef_kernel, dim3(row_blocks), dim3(256), 0, s, k);
        lay_out_hidden(p, c);
    }
    const int64_t rows = round_up(std::max<int64_t>(n, 1), 64);
    const int64_t g_part = rows * p.piece * 2;
    float *acc = reinterpret_cast<float *>(c.ws + p.acc);
    const float k = static_cast<float>(1.44269504088896340736 / temperature);
    for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
        const int64_t width = std::min(p.piece, vocab - v0);
        const Operand dz{c.ws + p.g, p.piece, g_part};
        if (n > 0) {
            const Operand w = weight_operand(p, c, v0, width);
            if (p.f32)
                logits_of<6>(p, c, w, width, GradEpilogue<3>{tgt, grad, c.ws + p.g, p.piece, g_part, v0, width, k});
            else
                logits_of<1>(p, c, w, width, GradEpilogue<1>{tgt, grad, c.ws + p.g, p.piece, g_part, v0, width, k});
            if (grad_hidden) {
                const Gemm g{dz, w, n, dim, width, c.s.count, 0, 8, p.splits};
                const AccumulateEpilogue e{acc, p.ld, rows * p.ld, v0 > 0};
                if (p.few)
                    p.f32 ? multiply_few<false, 6>(g, e, s) : multiply_few<false, 1>(g, e, s);
                else
                    p.f32 ? multiply_large<true, false, 6>(g, e, s) : multiply_large<true, false, 1>(g, e, s);
            }
        }
        if (grad_weight) {
            const Gemm g{dz, hidden_operand(p, c), width, dim, n, c.s.count, 1, 8, 1};
            uint8_t *out = static_cast<uint8_t *>(grad_weight) + v0 * dim * (p.f32 ? 4 : 2);
            if (p.f32)
                multiply_large<false, false, 6>(g, WeightEpilogue<true>{out, dim}, s);
            else
                multiply_large<false, false, 1>(g, WeightEpilogue<false>{out, dim}, s);
        }
    }
    if (grad_hidden && n > 0) {
        const unsigned blocks = blocks_for(n * ceil_div(dim, 4));
        if (p.f32)
            hipLaunchKernelGGL(hidden_kernel<true>, dim3(blocks), dim3(256), 0, s, acc, p.ld, rows * p.ld, p.splits, c.s.place, n, dim, grad_hidden);
        else
            hipLaunchKernelGGL(hidden_kernel<false>, dim3(blocks), dim3(256), 0, s, acc, p.ld, rows * p.ld, p.splits, c.s.place, n, dim, grad_hidden);
    }
    return check_launch("me_head_backward");
}
