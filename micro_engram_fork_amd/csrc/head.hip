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
// products: one rounding per term where the sum itself is rounded so at its end. Many terms average out, but a row's target
// carries as much as all its other tokens together: what the rounding leaves of it is added to the hidden states' gradient
// in fp32 (hidden_kernel), and for few rows, whose product with h is bound by its result, the head's gradient takes
// what the rounding leaves of every value as more rows of the reduction (takes_rest).
#include "head_gemm.h"

#include <algorithm>
#include <cmath>

namespace me {
namespace {

using namespace head;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;
// Rows up to which the tiles of few rows are taken (takes_few)
constexpr int64_t kFew = 128;
constexpr int64_t kPieceBytes = int64_t{1} << 30;        // of a piece's gradient, and of a piece of laid-out weights
constexpr int kSplits = 8;                               // of a product that fills the chip without
// Rows of fp32 up to which logits are kept (takes_kept)
constexpr int64_t kKeptRows = 384, kKeptMost = 1024;
constexpr int kHeader = 16;                              // ints before the rows in `saved`: the number of them

// What the forward leaves for the backward: the number of counted rows, and by counted row its source, target,
// log2-sum and o; by source row its place among the counted ones.
struct Saved {
    int32_t *count, *rows, *place, *tgt;
    float *lse2, *others;
};

Saved saved_of(void *p, int64_t n) {
    int32_t *i = static_cast<int32_t *>(p);
    float *f = static_cast<float *>(p);
    return {i, i + kHeader, i + kHeader + n, i + kHeader + 2 * n, f + kHeader + 3 * n, f + kHeader + 4 * n};
}

// ---- rows that count -------------------------------------------------------------------------------------------
// One workgroup: rows[r] = source of the r-th counted row, tgt[r] its target, place[i] = r or -1.
constexpr int kIndexThreads = 1024;

template <typename T>
__global__ __launch_bounds__(kIndexThreads) void index_kernel(const T *targets, int64_t n, int64_t ignore, int64_t vocab,
                                                              Saved s, uint32_t *clear) {
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
            s.tgt[r] = static_cast<int32_t>(t);
        }
        at += all;
        __syncthreads();
    }
    if (tid == 0) *s.count = at;
    if (tid == 0 && clear != nullptr) *clear = 0;
}

// ---- what the gradient of a row's logits is made of ---------------------------------------------------------------
// dz_j = ca 2^(z_j - lse2) - cb, gt at the target, z in units of log2
struct RowGrad {
    float lse2, ca, cb, gt;
};

struct Coefs {
    Saved s;
    const float *upstream;  // by source row (per_row) or one
    int per_row, mean;
    double scale;           // of the loss, over T
    float smoothing, z_loss;
    double vocab;
    float *factor;          // null, or takes what all rows share: theirs are then for an upstream of 1, loss a plain sum
    RowGrad *grad;          // null: none of this is wanted
    float *bound;           // of each row's values, or null
    uint32_t *largest;      // set to 0, `pieces` of them
    int pieces;

    __device__ __forceinline__ double shared(int64_t count) const {
        return static_cast<double>(*upstream) * scale / (mean ? static_cast<double>(max(count, int64_t{1})) : 1.0);
    }
    __device__ __forceinline__ RowGrad of(int64_t r, int64_t count) const {
        const float lse2 = s.lse2[r], o = s.others[r];
        RowGrad g;
        g.lse2 = lse2;
        if (per_row) {  // log-probabilities: -upstream times the loss -log q
            const float c = static_cast<float>(-static_cast<double>(upstream[s.rows[r]]) * scale);
            g.ca = c, g.cb = 0.f, g.gt = -c * o;
        } else {
            const double c = factor != nullptr ? 1.0 : shared(count);
            const double more = 2.0 * z_loss * kLn2 * lse2, e = smoothing;
            g.ca = static_cast<float>(c * (1.0 + more));
            g.cb = static_cast<float>(c * e / vocab);
            g.gt = static_cast<float>(c * (more - (1.0 + more) * o + e - e / vocab));
        }
        return g;
    }
    __device__ __forceinline__ void row(int64_t r, int64_t count) const {
        const RowGrad g = of(r, count);
        const float o = s.others[r];
        grad[r] = g;
        // a token's probability is at most that of all but the target
        if (bound) bound[r] = fmaxf(fabsf(g.ca) * (1.0001f * o) + fabsf(g.cb), fabsf(g.gt));
    }
    __device__ __forceinline__ void clear(int64_t thread) const {
        if (thread < pieces) largest[thread] = 0;
    }
};

// ---- operands as the products read them: [rows][ld] bf16, ld a multiple of 64, zeros past dim; fp32 in three parts -----
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));        // pieces of rows that may start
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));     // at any element

struct Layout {
    const void *src;
    int64_t per_batch, batch_stride, row_stride;  // row r: (r / per_batch) * batch_stride + (r % per_batch) * row_stride
    const int32_t *rows, *count;                  // sources of the rows and how many there are; null: as they are
    int64_t n, dim, ld, part;                     // part: bytes
    uint8_t *dst;
    int again;                                    // the rows once more behind the last one
    const int32_t *gate;                          // a count; 0: nothing is laid out. Null: none
};

// Eight values of a row of fp32 from c on, zeros from dim on
__device__ __forceinline__ void load8(const float *row, int64_t c, int64_t dim, float (&x)[8]) {
    const auto at = as_global(row + c);
    if (c + 8 <= dim) {
        const f32x4_any a = *(gmem_ptr<const f32x4_any>)(at), b = *(gmem_ptr<const f32x4_any>)(at + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < dim ? at[j] : 0.f;
    }
}

// x as three bf16 that add up to it: each the nearest bf16 of what remains. What is not finite stands in the
// first part alone.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
    p[0] = float_to_bf16_bits_rne(x);
    float rest = x - bf16_bits_to_float(p[0]);
    if (!(__builtin_fabsf(rest) < __builtin_inff())) rest = 0.f;
    p[1] = float_to_bf16_bits_rne(rest);
    p[2] = float_to_bf16_bits_rne(rest - bf16_bits_to_float(p[1]));
}

// k: of the rows' gradients, which the first of a row's threads makes on the way (the row layout of a backward)
template <bool F32>
__global__ __launch_bounds__(256) void layout_kernel(const Layout a, const Coefs k) {
    if (a.gate != nullptr && *a.gate == 0) return;
    const int64_t units = a.ld / 8;
    const int64_t n = a.count ? min(a.n, static_cast<int64_t>(*a.count)) : a.n;
    if (k.factor != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *k.factor = static_cast<float>(k.shared(n));
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < n * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = u / units, c = (u - r * units) * 8;
        if (k.grad != nullptr && c == 0) k.row(r, n);
        const int64_t from = a.rows ? a.rows[r] : r;
        const int64_t at = from / a.per_batch * a.batch_stride + from % a.per_batch * a.row_stride + c;
        uint32_t w[3][4] = {};
        uint16_t(&h)[3][8] = reinterpret_cast<uint16_t(&)[3][8]>(w);
        if constexpr (F32) {
            float x[8];
            load8(static_cast<const float *>(a.src) + (at - c), c, a.dim, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint16_t p[3];
                split3(x[j], p);
                h[0][j] = p[0], h[1][j] = p[1], h[2][j] = p[2];
            }
        } else {
            const uint16_t *src = static_cast<const uint16_t *>(a.src) + at;
            if (c + 8 <= a.dim) {
                const u32x4_any x = *(gmem_ptr<const u32x4_any>)(as_global(src));
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
        if (!F32 && a.again) *as_global(reinterpret_cast<u32x4_v *>(a.dst + ((n + r) * a.ld + c) * 2)) = u32x4_v{w[0][0], w[0][1], w[0][2], w[0][3]};
    }
}

// fp32 rows in two fp16 parts over a power of two by row, which goes to `scale` (what the parts are multiplied by to
// give the value), and the largest of these, where wanted, to `largest`. A wave per row (32,000 x 1024: 77 us for
// 262 MB read and written, 3.4 TB/s). Of what is not finite, the first part alone.
__global__ __launch_bounds__(256) void layout16_kernel(const Layout a, float *scale, uint32_t *largest, const Coefs k) {
    uint32_t widest = 0;
    if (k.grad != nullptr) k.clear(static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x);
    const int lane = threadIdx.x & 63;
    const int64_t n = a.count ? min(a.n, static_cast<int64_t>(*a.count)) : a.n;
    constexpr int kKept = 4;  // pieces of 512 values that stay in registers; further ones are read again
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); r < n; r += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t from = a.rows ? a.rows[r] : r;
        const float *src = static_cast<const float *>(a.src) + (from / a.per_batch * a.batch_stride + from % a.per_batch * a.row_stride);
        float kept[kKept][8];
        uint32_t most = 0;
        auto look = [&](const float (&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
                most = max(most, b < 0x7f800000u ? b : 0u);
            }
        };
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (i * 512 < a.dim) {
                load8(src, i * 512 + lane * 8, a.dim, kept[i]);
                look(kept[i]);
            }
        for (int64_t c = kKept * 512 + lane * 8; c < a.dim; c += 512) {
            float x[8];
            load8(src, c, a.dim, x);
            look(x);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
        // the largest below 2^15; the power and its inverse are normal fp32 numbers
        const int up = min(max(14 - (static_cast<int>(most >> 23) - 127), -112), 126);
        const float times = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        const uint32_t down = static_cast<uint32_t>(127 - up) << 23;
        widest = max(widest, down);
        if (lane == 0) {
            scale[r] = __uint_as_float(down);
            if (k.grad != nullptr) k.row(r, n);
        }
        auto put = [&](const float (&v)[8], int64_t c) {
            if (c >= a.ld) return;
            halfx8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = v[j] * times;
                hi[j] = static_cast<_Float16>(x);
                const float rest = x - static_cast<float>(hi[j]);
                lo[j] = static_cast<_Float16>(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.f);
            }
            *as_global(reinterpret_cast<halfx8 *>(a.dst + (r * a.ld + c) * 2)) = hi;
            *as_global(reinterpret_cast<halfx8 *>(a.dst + a.part + (r * a.ld + c) * 2)) = lo;
        };
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (i * 512 < a.dim) put(kept[i], i * 512 + lane * 8);
        for (int64_t c = kKept * 512 + lane * 8; c < a.ld; c += 512) {
            float x[8];
            load8(src, c, a.dim, x);
            put(x, c);
        }
    }
    if (largest != nullptr && lane == 0) atomicMax(largest, widest);  // a maximum: the same in any order
}

// What rows and columns of a product of fp16 parts are multiplied by; null: nothing
struct Scales {
    const float *row, *col;  // by counted row; by column of the piece, readable up to whole tiles

    __device__ __forceinline__ float of_row(int64_t r, bool ok) const { return row != nullptr && ok ? row[r] : 1.f; }
    template <bool SCALED>
    __device__ __forceinline__ f32x4_v of_cols(int64_t c) const {
        if constexpr (SCALED)
            return *as_global(reinterpret_cast<const f32x4_v *>(col + c));
        else
            return f32x4_v{1.f, 1.f, 1.f, 1.f};
    }
};

// ---- epilogues -----------------------------------------------------------------------------------------------
// acc[x][y][4 g + e] is row row0 + 32 y + (lane & 31), column col0 + 32 x + 8 g + 4 (lane >> 5) + e of the tile.

// Four values of row lane & 31 at column col of a staged block of 32 rows, bf16 or in parts that add up to them
template <int NPARTS, int SX>
__device__ __forceinline__ void stage4(float (&v)[4], uint8_t *stage, int col, int lane) {
    constexpr int kPitch = 64 * SX + 16;
#pragma unroll
    for (int p = 0; p < NPARTS; ++p) {
        uint32_t w[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t b = float_to_bf16_bits_rne(v[e]);
            reinterpret_cast<uint16_t *>(w)[e] = b;
            if (p + 1 < NPARTS) {
                v[e] -= bf16_bits_to_float(b);
                if (p == 0 && !(__builtin_fabsf(v[e]) < __builtin_inff())) v[e] = 0.f;  // not finite: the first part alone
            }
        }
        *reinterpret_cast<uint2 *>(stage + (p * 32 + (lane & 31)) * kPitch + col * 2) = make_uint2(w[0], w[1]);
    }
}

// Likewise in two fp16 parts
template <int SX>
__device__ __forceinline__ void stage4_half(const float (&v)[4], uint8_t *stage, int col, int lane) {
    constexpr int kPitch = 64 * SX + 16;
    typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
    halfx4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = static_cast<_Float16>(v[e]);
        const float rest = v[e] - static_cast<float>(hi[e]);
        lo[e] = static_cast<_Float16>(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.f);
    }
    *reinterpret_cast<halfx4 *>(stage + (lane & 31) * kPitch + col * 2) = hi;
    *reinterpret_cast<halfx4 *>(stage + (32 + (lane & 31)) * kPitch + col * 2) = lo;
}

// A staged block as 16-byte chunks of rows r0 .. of [rows][ld], from column c0 on
template <int NPARTS, int SX>
__device__ __forceinline__ void store_rows(const uint8_t *stage, uint8_t *out, int64_t ld, int64_t part, int64_t r0, int64_t rows, int64_t c0,
                                           int lane) {
    constexpr int kPitch = 64 * SX + 16, kChunks = 4 * SX;
#pragma unroll
    for (int p = 0; p < NPARTS; ++p)
#pragma unroll 4
        for (int it = 0; it < 32 * kChunks / 64; ++it) {
            const int ch = it * 64 + lane, r = ch / kChunks, cc = ch % kChunks;
            const u32x4_v v = *reinterpret_cast<const u32x4_v *>(stage + (p * 32 + r) * kPitch + cc * 16);
            if (r0 + r < rows && c0 + cc * 8 < ld) *as_global(reinterpret_cast<u32x4_v *>(out + p * part + ((r0 + r) * ld + c0 + cc * 8) * 2)) = v;
        }
}

// Statistics of a tile's rows over a wave's columns, in units of log2: their maximum and sum without the target,
// the target's own value, and where wanted the plain sum of the values.
template <bool SCALED>
struct StatsEpilogue {
    const int32_t *tgt;
    Scales scales;
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
            const float kr = k * scales.of_row(row, ok);
            // few waves hold a target of their rows, or the vocabulary's end
            if (there < 32 * SX || __any(mine >= 0))
                row_part<AGPR, true, SX, SY>(acc, y, row, kr, c0, ok, mine, there, part_at, lane);
            else
                row_part<AGPR, false, SX, SY>(acc, y, row, kr, c0, ok, mine, there, part_at, lane);
        }
    }

    template <bool AGPR, bool SOME, int SX, int SY>
    __device__ __forceinline__ void row_part(const floatx16 (&acc)[SX][SY], int y, int64_t row, float kr, int64_t c0, bool ok, int mine,
                                             int there, int64_t part_at, int lane) const {
        const int half4 = 4 * (lane >> 5);
        float m = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_v cs = scales.of_cols<SCALED>(c0 + 32 * x + 8 * q + half4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = acc_read<AGPR>(acc[x][y], 4 * q + e) * cs[e];
                    if constexpr (SOME) {
                        const int col = 32 * x + 8 * q + half4 + e;
                        total += col < there ? v : 0.f;
                        if (col == mine) at_target[row] = v * kr;
                        if (col == mine || col >= there) v = -__builtin_inff();
                    } else {
                        total += v;
                    }
                    m = fmaxf(m, v);
                }
            }
        m = fmaxf(m, __shfl_xor(m, 32)) * kr;
        const float shift = m == -__builtin_inff() ? 0.f : m;
        float s = 0.f;
        if constexpr (SOME) asm volatile("" : "+v"(mine), "+s"(there));  // compared anew: 64 lane masks are not kept
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_v cs = scales.of_cols<SCALED>(c0 + 32 * x + 8 * q + half4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = acc_read<AGPR>(acc[x][y], 4 * q + e) * cs[e];
                    if constexpr (SOME) {
                        const int col = 32 * x + 8 * q + half4 + e;
                        if (col == mine || col >= there) v = -__builtin_inff();
                    }
                    s += __builtin_amdgcn_exp2f(fmaf(v, kr, -shift));
                }
            }
        s += __shfl_xor(s, 32);
        total += __shfl_xor(total, 32);
        if (ok && lane < 32) {
            part[part_at * part_stride + row * row_stride] = make_float2(m, s);
            if (sum != nullptr) sum[part_at * part_stride + row * row_stride] = total * kr;
        }
    }
};

// The exponentials of a tile's logits, 2^(z - ref) by row and zero at the target, in bf16 as rows of a piece, and their
// sums over a wave's columns
struct ExpEpilogue {
    const int32_t *tgt;
    const float *ref;        // by row, log2
    float *part, *sum;       // by (column part, row), as StatsEpilogue
    float *at_target;
    int64_t part_stride, row_stride;
    uint8_t *out;
    int64_t ld;
    int64_t first, vocab;
    float k;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        const int64_t c0 = t.s0 + col0;
        const int there = static_cast<int>(max(min(vocab - c0, int64_t{32 * SX}), int64_t{0}));
        const int64_t part_at = (first + c0) / (32 * SX);
        constexpr int kPitch = 64 * SX + 16;
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            uint8_t *stage = lds + ((threadIdx.x >> 6) * 2 + (y & 1)) * (32 * kPitch);
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            const bool ok = row < t.rows;
            const float shift = ok ? ref[row] : 0.f;
            const int64_t off = ok ? tgt[row] - (first + c0) : -1;
            const int mine = off >= 0 && off < there ? static_cast<int>(off) : -1;
            float s, total = 0.f;
            if (there < 32 * SX || __any(mine >= 0))
                s = stage_rows<AGPR, true, SX, SY>(acc, y, row, shift, mine, there, total, stage, lane);
            else
                s = stage_rows<AGPR, false, SX, SY>(acc, y, row, shift, mine, there, total, stage, lane);
            s += __shfl_xor(s, 32);
            total += __shfl_xor(total, 32);
            if (ok && lane < 32) {
                part[part_at * part_stride + row * row_stride] = s;
                if (sum != nullptr) sum[part_at * part_stride + row * row_stride] = total * k;
            }
            store_rows<1, SX>(stage, out, ld, 0, t.r0 + row0 + 32 * y, t.rows, c0, lane);
        }
    }

    template <bool AGPR, bool SOME, int SX, int SY>
    __device__ __forceinline__ float stage_rows(const floatx16 (&acc)[SX][SY], int y, int64_t row, float shift, int mine, int there, float &total,
                                                uint8_t *stage, int lane) const {
        const int half4 = 4 * (lane >> 5);
        float s = 0.f;
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = acc_read<AGPR>(acc[x][y], 4 * q + e);
                    v[e] = __builtin_amdgcn_exp2f(fmaf(z, k, -shift));
                    if constexpr (SOME) {
                        const int col = 32 * x + 8 * q + half4 + e;
                        if (col == mine) at_target[row] = z * k;
                        if (col == mine || col >= there) v[e] = 0.f;
                        total += col < there ? z : 0.f;
                    } else {
                        total += z;
                    }
                    s += v[e];
                }
                stage4<1, SX>(v, stage, 32 * x + 8 * q + half4, lane);
            }
        return s;
    }
};

// Power of two that puts a row's gradient times the columns' scales into fp16's range: the largest below 2^15. row: a
// bound of the row's values, largest: of the scales (a power of two)
__device__ __forceinline__ int row_power(float row, uint32_t largest) {
    const int e = static_cast<int>(__float_as_uint(row) >> 23) - 127 + static_cast<int>(largest >> 23) - 127;
    return min(max(14 - e, -126), 126);
}

__device__ __forceinline__ float power_of(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// The logits' gradient of a tile as rows of a piece: bf16 for bf16 operands (PARTS 1), with what that leaves of them as
// rows behind the last counted one (2); for fp32 ones three bf16 parts where the head's gradient is wanted, and two
// fp16 parts, times the columns' scales and the row's power, where the hidden states' is (3)
template <int PARTS>
struct GradEpilogue {
    static constexpr bool F32 = PARTS == 3;
    const int32_t *tgt;
    Scales scales;
    const RowGrad *grad;
    const float *bound;       // of each row's values (F32)
    const uint32_t *largest;  // of the columns' scales (F32)
    uint8_t *out, *half;      // [rows][ld] of each part; null: not wanted
    int64_t ld, part;         // ld: columns of the piece, a multiple of 64; part: bytes
    int64_t first, vocab;     // first column of the piece, columns that there are
    float k;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        if constexpr (F32) {
            if (half != nullptr) rows_of<AGPR, true, SX, SY>(acc, t, row0, col0, lds, lane);
            if (out == nullptr) return;
        }
        rows_of<AGPR, false, SX, SY>(acc, t, row0, col0, lds, lane);
    }

    template <bool AGPR, bool HALF, int SX, int SY>
    __device__ __forceinline__ void rows_of(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        const int64_t c0 = t.s0 + col0;
        const int there = static_cast<int>(max(min(vocab - c0, int64_t{32 * SX}), int64_t{0}));
        constexpr int kParts = HALF ? 2 : PARTS;
        // 32 rows at a time through LDS, where a wave has two places in turn (with parts one: a wave's LDS
        // accesses keep their order)
        constexpr int kPitch = 64 * SX + 16, kPlaces = PARTS > 1 ? 1 : 2;
        static_assert(4 * kPlaces * kParts * 32 * kPitch <= (SX == 4 ? kRingBytes : SX == 2 ? 3 * kUnit : 2 * kUnit), "the stage fits the ring");
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            uint8_t *stage = lds + ((threadIdx.x >> 6) * kPlaces + (y % kPlaces)) * (kParts * 32 * kPitch);
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            const bool ok = row < t.rows;
            RowGrad g = ok ? grad[row] : RowGrad{0.f, 0.f, 0.f, 0.f};
            const int64_t off = ok ? tgt[row] - (first + c0) : -1;
            const int mine = off >= 0 && off < there ? static_cast<int>(off) : -1;
            const float kr = k * scales.of_row(row, ok);
            const float up = HALF && ok ? power_of(row_power(bound[row], *largest)) : 1.f;
            if (F32 || there < 32 * SX || __any(mine >= 0))
                stage_rows<AGPR, HALF, true, SX, SY>(acc, y, g, kr, up, c0, mine, there, stage, lane);
            else
                stage_rows<AGPR, HALF, false, SX, SY>(acc, y, g, kr, up, c0, mine, there, stage, lane);
            store_rows<kParts, SX>(stage, HALF ? half : out, ld, PARTS == 2 ? t.rows * ld * 2 : part, t.r0 + row0 + 32 * y, t.rows, c0, lane);
        }
    }

    template <bool AGPR, bool HALF, bool SOME, int SX, int SY>
    __device__ __forceinline__ void stage_rows(const floatx16 (&acc)[SX][SY], int y, const RowGrad &g, float kr, float up, int64_t c0, int mine,
                                               int there, uint8_t *stage, int lane) const {
        const int half4 = 4 * (lane >> 5);
#pragma unroll
        for (int x = 0; x < SX; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
                const f32x4_v cs = scales.of_cols<F32>(c0 + 32 * x + 8 * q + half4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = fmaf(__builtin_amdgcn_exp2f(fmaf(acc_read<AGPR>(acc[x][y], 4 * q + e) * cs[e], kr, -g.lse2)), g.ca, -g.cb);
                    if constexpr (SOME) {
                        const int col = 32 * x + 8 * q + half4 + e;
                        if (col == mine) v[e] = g.gt;
                        if (col >= there) v[e] = 0.f;  // past the vocabulary: nothing for the products with W and h
                    }
                    if constexpr (HALF) v[e] *= up * (!SOME || 32 * x + 8 * q + half4 + e < there ? cs[e] : 0.f);
                }
                if constexpr (HALF)
                    stage4_half<SX>(v, stage, 32 * x + 8 * q + half4, lane);
                else
                    stage4<PARTS, SX>(v, stage, 32 * x + 8 * q + half4, lane);
            }
    }
};

// fp32 sums of a tile, added to what earlier pieces left: [split][rows][ld]
struct AccumulateEpilogue {
    float *out;
    int64_t ld, split_stride;  // ld: a multiple of 4
    int add;
    const float *bound;        // of fp16 parts: what the rows' powers come from, else null
    const uint32_t *largest;

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *, int lane) const {
        const int half4 = 4 * (lane >> 5);
        float *o = out + t.split * split_stride;
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            const int64_t row = t.r0 + row0 + 32 * y + (lane & 31);
            if (row >= t.rows) continue;
            const float down = bound != nullptr ? power_of(-row_power(bound[row], *largest)) : 1.f;
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
                    for (int e = 0; e < 4; ++e) v[g][e] = fmaf(acc_read<AGPR>(acc[x][y], 4 * g + e), down, v[g][e]);
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
    const float *factor;  // of bf16: what all values are multiplied by, or null

    template <bool AGPR, int SX, int SY>
    __device__ __forceinline__ void run(const floatx16 (&acc)[SX][SY], const Tile &t, int row0, int col0, uint8_t *lds, int lane) const {
        const int half4 = 4 * (lane >> 5);
        const bool whole = dim % 8 == 0;  // rows of whole 16-byte chunks
        const float f = !F32 && factor != nullptr ? *as_global(factor) : 1.f;
#pragma unroll
        for (int y = 0; y < SY; ++y) {
            if (!F32 && whole) {
                constexpr int kPitch = 64 * SX + 16;
                static_assert(8 * 32 * kPitch <= kRingBytes, "the stage fits the ring");
                uint8_t *stage = lds + ((threadIdx.x >> 6) * 2 + (y & 1)) * (32 * kPitch);
#pragma unroll
                for (int x = 0; x < SX; ++x)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = acc_read<AGPR>(acc[x][y], 4 * g + e) * f;
                        stage4<1, SX>(v, stage, 32 * x + 8 * g + half4, lane);
                    }
                store_rows<1, SX>(stage, out, dim, 0, t.r0 + row0 + 32 * y, t.rows, t.s0 + col0, lane);
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
                    for (int e = 0; e < 4; ++e) v[e] = acc_read<AGPR>(acc[x][y], 4 * g + e) * f;
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

// A maximum and the sum of 2^(x - maximum)
struct Sum2 {
    float m, s;
};

__device__ __forceinline__ Sum2 join(Sum2 a, Sum2 b) {
    const float m = fmaxf(a.m, b.m);
    const float shift = m == -__builtin_inff() ? 0.f : m;
    return {m, a.s * __builtin_amdgcn_exp2f(a.m - shift) + b.s * __builtin_amdgcn_exp2f(b.m - shift)};
}

// ---- a few rows: one read of the head by plain products ----------------------------------------------------------
// Up to kVectorRows rows: a workgroup holds them in LDS in fp32, its waves take head rows
// two at a time, each lane 16 bytes of a row at a stride of a KiB, and the 64 partial sums are added across the wave.
// Nothing is laid out first (fp32 parts would be read and written three times over) and the rows are found by every
// workgroup for itself: two launches for a sampled token's log-probability. Lane l keeps the logits of
// the wave's l-th head row of each 64, and statistics are taken of 64 at a time. Bound by the head's read: 32,000 x
// 1024 (131 MB), one row 25 us, 5.3 TB/s; 262,144 x 5376, two rows 944 us, 6.0.
constexpr int kVectorRows = 8;
constexpr int kVectorLds = 64 * 1024;
constexpr int kVectorGroups = 2048;

struct VectorArgs {
    Layout h;
    const float *weight;
    int64_t w_stride, vocab;
    const void *targets;
    int t64;
    int64_t ignore;
    Saved s;
    float *logits;  // [rows][ld] for the backward, as of kept_kernel, or null
    int64_t ld;
    float2 *part;   // [rows][workgroups]
    float *sum;     // likewise, or null
    float *at_target;
    float k;
};

struct Chunk {  // 16 bytes of a row
    float v[4];
    __device__ __forceinline__ void load(const float *row, int64_t c, int64_t dim) {
        const auto at = as_global(row + c);
        if (c + 4 <= dim) {
            const f32x4_any x = *(gmem_ptr<const f32x4_any>)(at);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = x[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = c + j < dim ? at[j] : 0.f;
        }
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

__device__ __forceinline__ float wave_sum(float x) {
    x = dpp_add<0xb1>(x);   // quad_perm [1, 0, 3, 2]
    x = dpp_add<0x4e>(x);   // quad_perm [2, 3, 0, 1]
    x = dpp_add<0x141>(x);  // row_half_mirror
    x = dpp_add<0x140>(x);  // row_mirror
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int N>
__global__ __launch_bounds__(256) void vector_kernel(const VectorArgs a) {
    extern __shared__ __attribute__((aligned(16))) float s_h[];  // [N][pitch]
    __shared__ int s_tgt[N], s_from[N], s_count;
    __shared__ float2 s_part[4][N];
    __shared__ float s_sum[4][N];
    constexpr int kValues = 4, kStep = 64 * kValues;
    constexpr int kUnroll = N >= 8 ? 1 : N >= 4 ? 2 : 4;  // loads in flight against registers
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t pitch = ceil_div(a.h.dim, int64_t{kStep}) * kStep;
    if (tid < 64) {
        const int n = static_cast<int>(a.h.n);
        int64_t t = -1;
        if (lane < n) t = a.t64 ? static_cast<const int64_t *>(a.targets)[lane] : static_cast<const int32_t *>(a.targets)[lane];
        const bool ok = lane < n && t != a.ignore && t >= 0 && t < a.vocab;
        const uint64_t mask = __ballot(ok);
        const int r = __popcll(mask & ((uint64_t{1} << lane) - 1));
        if (ok) s_tgt[r] = static_cast<int>(t), s_from[r] = lane;
        if (lane == 0) s_count = __popcll(mask);
        if (blockIdx.x == 0) {  // for the launches that follow
            if (lane < n) a.s.place[lane] = ok ? r : -1;
            if (ok) a.s.rows[r] = lane, a.s.tgt[r] = static_cast<int>(t);
            if (lane == 0) *a.s.count = __popcll(mask);
        }
    }
    __syncthreads();
    const int count = s_count;
    if (count == 0) return;
    for (int64_t u = tid; u < N * pitch; u += 256) {
        const int r = static_cast<int>(u / pitch);
        const int64_t c = u - r * pitch;
        float x = 0.f;
        if (r < count && c < a.h.dim) {
            const int64_t from = s_from[r], at = from / a.h.per_batch * a.h.batch_stride + from % a.h.per_batch * a.h.row_stride + c;
            x = static_cast<const float *>(a.h.src)[at];
        }
        s_h[u] = x;
    }
    __syncthreads();

    float m[N], s[N], sum[N], z[N];
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = -__builtin_inff(), s[i] = 0.f, sum[i] = 0.f, z[i] = -__builtin_inff();
    auto take = [&]() {  // the statistics of this lane's logits so far
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float top = fmaxf(m[i], z[i]);
            const float shift = top == -__builtin_inff() ? 0.f : top;
            s[i] = s[i] * __builtin_amdgcn_exp2f(m[i] - shift) + __builtin_amdgcn_exp2f(z[i] - shift);
            m[i] = top;
            z[i] = -__builtin_inff();
        }
    };
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4;
    int slot = 0;
    for (int64_t j = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * 2; j < a.vocab; j += waves * 2) {
        const int64_t j1 = min(j + 1, a.vocab - 1);
        const float *w0 = a.weight + j * a.w_stride, *w1 = a.weight + j1 * a.w_stride;
        float acc[2][N] = {};
#pragma unroll kUnroll
        for (int64_t c = lane * kValues; c < a.h.dim; c += kStep) {
            Chunk x0, x1;
            x0.load(w0, c, a.h.dim);
            x1.load(w1, c, a.h.dim);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < kValues; ++e) {
                    const float h = s_h[i * pitch + c + e];
                    acc[0][i] = fmaf(x0.v[e], h, acc[0][i]);
                    acc[1][i] = fmaf(x1.v[e], h, acc[1][i]);
                }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t col = j + b;
            if (col < a.vocab) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float raw = wave_sum(acc[b][i]), v = raw * a.k;
                    if (lane == slot) {
                        if (a.logits != nullptr && i < count) a.logits[i * a.ld + col] = raw;
                        sum[i] += v;
                        if (i < count && col == s_tgt[i])
                            a.at_target[i] = v;
                        else
                            z[i] = v;
                    }
                }
                if (++slot == 64) take(), slot = 0;
            }
        }
    }
    take();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        Sum2 all = {m[i], s[i]};
#pragma unroll
        for (int d = 32; d; d >>= 1) all = join(all, {__shfl_xor(all.m, d), __shfl_xor(all.s, d)});
        const float total = wave_sum(sum[i]);
        if (lane == 0) s_part[wave][i] = make_float2(all.m, all.s), s_sum[wave][i] = total;
    }
    __syncthreads();
    if (tid < N && tid < count) {
        Sum2 all = {s_part[0][tid].x, s_part[0][tid].y};
        float total = s_sum[0][tid];
        for (int w = 1; w < 4; ++w) all = join(all, {s_part[w][tid].x, s_part[w][tid].y}), total += s_sum[w][tid];
        a.part[static_cast<int64_t>(tid) * gridDim.x + blockIdx.x] = make_float2(all.m, all.s);
        if (a.sum) a.sum[static_cast<int64_t>(tid) * gridDim.x + blockIdx.x] = total;
    }
}

// ---- few rows of fp32: their logits are kept ----------------------------------------------------------------------
// For few rows (takes_kept) the product with the head takes the head as it lies, once, and what it gives is small beside
// the head: the logits stay, in fp32, for the backward. So a forward and the gradients of both operands read the head
// twice and write its gradient, which nothing can do without. Bound by these up to some 30 rows; 262,144 x 5376 (5.6 GB), us:
//   rows   logits   product with dz   outer product
//     12     1028             1171            1344     5.5, 4.8 and 4.2 TB/s
//     46     1209             1672            1978
//    128     2294             2775            3057     beyond, by matrix and vector instructions that wait for each other
// (laid out in parts instead: 12 rows 11,500 us in all, here 3270)
constexpr int kKeptCols = 2048;  // logits of a workgroup: 8 of a thread

struct KeptArgs {
    const float *partial;    // [split][rows][ld], null: the logits are in place
    float *logits;           // [counted rows][ld], times k not yet
    int64_t ld, split_stride, vocab;
    int tile_rows, col_tiles, most, cost;  // of the splits
    Saved s;
    float2 *part;            // by (row, workgroup of a row)
    float *sum, *at_target;
    float k;
};

// Adds the product's splits and takes the statistics that the tiles of other calls take as they leave the matrix cores
__global__ __launch_bounds__(256) void kept_kernel(const KeptArgs a) {
    __shared__ Sum2 s_all[4];
    __shared__ float s_sum[4];
    const int64_t r = blockIdx.y;
    const int count = *a.s.count;
    if (r >= count) return;
    const int tid = threadIdx.x;
    const int64_t target = a.s.tgt[r];
    const int splits = a.partial == nullptr ? 0 : splits_for(static_cast<int>(ceil_div(count, a.tile_rows)) * a.col_tiles, a.most, a.cost);
    float z[8], m = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int64_t c = static_cast<int64_t>(blockIdx.x) * kKeptCols + b * 1024 + tid * 4;
        f32x4_v v = {0.f, 0.f, 0.f, 0.f};
        if (c < a.ld) {
            const auto at = as_global(reinterpret_cast<f32x4_v *>(a.logits + r * a.ld + c));
            if (splits == 0) v = *at;
            for (int i = 0; i < splits; ++i) v += *as_global(reinterpret_cast<const f32x4_v *>(a.partial + i * a.split_stride + r * a.ld + c));
            if (splits > 0) *at = v;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool there = c + e < a.vocab;
            const float x = v[e] * a.k;
            total += there ? x : 0.f;
            if (there && c + e == target) a.at_target[r] = x;
            z[4 * b + e] = there && c + e != target ? v[e] : -__builtin_inff();
            m = fmaxf(m, z[4 * b + e]);
        }
    }
    m *= a.k;
    const float shift = m == -__builtin_inff() ? 0.f : m;
    Sum2 all = {m, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) all.s += __builtin_amdgcn_exp2f(fmaf(z[i], a.k, -shift));
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        all = join(all, {__shfl_xor(all.m, d), __shfl_xor(all.s, d)});
        total += __shfl_xor(total, d);
    }
    if ((tid & 63) == 0) s_all[tid >> 6] = all, s_sum[tid >> 6] = total;
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < 4; ++w) all = join(all, s_all[w]), total += s_sum[w];
    const int64_t at = r * gridDim.x + blockIdx.x;
    a.part[at] = make_float2(all.m, all.s);
    if (a.sum) a.sum[at] = total;
}

// Sixteen rows' values of a column as the product of the head's gradient reads them: by block of 16 rows and column
// three bf16 parts of 16 values each, 96 bytes
constexpr int kOuterRows = 16, kOuterBytes = 3 * kOuterRows * 2;

__device__ __forceinline__ void store_parts(uint8_t *to, const float (&x)[kOuterRows]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        floatx8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[8 * h + i];
        const Parts parts(v);
#pragma unroll
        for (int p = 0; p < 3; ++p) *as_global(reinterpret_cast<bf16x8 *>(to + p * kOuterRows * 2 + h * 16)) = parts.p[p];
    }
}

// The logits' gradient from them: [counted rows][ld] for the product with the head, zeros past the vocabulary up
// to whole chunks; and in parts for the product with the hidden states, zeros past the rows
struct KeptGradArgs {
    Coefs k;
    const float *logits;
    float *out;       // null: not wanted
    uint8_t *parts;   // [block of rows][vocab], likewise
    int64_t ld, vocab;
    float scale;
};

__global__ __launch_bounds__(256) void kept_grad_kernel(const KeptGradArgs a) {
    __shared__ RowGrad s_grad[kOuterRows];
    __shared__ int s_tgt[kOuterRows];
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kOuterRows;
    const int count = *a.k.s.count;
    const int rows = static_cast<int>(min(count - r0, int64_t{kOuterRows}));
    if (rows <= 0) return;
    const int tid = threadIdx.x;
    if (tid < rows) s_grad[tid] = a.k.of(r0 + tid, count), s_tgt[tid] = a.k.s.tgt[r0 + tid];
    __syncthreads();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + tid;
    if (c >= a.ld) return;
    float v[kOuterRows];
#pragma unroll
    for (int r = 0; r < kOuterRows; ++r) v[r] = r < rows ? a.logits[(r0 + r) * a.ld + c] : 0.f;
#pragma unroll
    for (int r = 0; r < kOuterRows; ++r) {
        if (r >= rows) break;
        const RowGrad g = s_grad[r];
        v[r] = fmaf(__builtin_amdgcn_exp2f(fmaf(v[r], a.scale, -g.lse2)), g.ca, -g.cb);
        if (c == s_tgt[r]) v[r] = g.gt;
        if (c >= a.vocab) v[r] = 0.f;
        if (a.out != nullptr) a.out[(r0 + r) * a.ld + c] = v[r];
    }
    if (a.parts != nullptr && c < a.vocab) store_parts(a.parts + (blockIdx.y * a.vocab + c) * kOuterBytes, v);
}

// The hidden states in the same way: [block of rows][dim]
__global__ __launch_bounds__(256) void hidden_parts_kernel(const Layout h, uint8_t *parts) {
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kOuterRows, c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int count = *h.count;
    if (r0 >= count || c >= h.dim) return;
    float v[kOuterRows];
#pragma unroll
    for (int r = 0; r < kOuterRows; ++r) {
        v[r] = 0.f;
        if (r0 + r < count) {
            const int64_t from = h.rows[r0 + r];
            v[r] = static_cast<const float *>(h.src)[from / h.per_batch * h.batch_stride + from % h.per_batch * h.row_stride + c];
        }
    }
    store_parts(parts + (blockIdx.y * h.dim + c) * kOuterBytes, v);
}

// The head's gradient from few rows: an outer product of short reduction, bound by the write of the result. Tiles of
// 128 x 128, four waves of 64 x 64; a lane's fragment of a k-step is 16 bytes for each part, straight from L2 without
// LDS, the next step's in flight. A lane's results are one column of the gradient: whole lines of 32 columns leave by each
// store, wherever the rows start.
struct OuterArgs {
    const uint8_t *dz, *h;  // as above
    const int32_t *count;
    int64_t vocab, dim;
    float *out;             // [vocab][dim]
    int col_tiles;
};

__global__ __launch_bounds__(256, 2) void outer_kernel(const OuterArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // each XCD takes a run of tiles, whose operands stay in its L2
    const int tile = static_cast<int>(blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds);
    const int64_t v0 = static_cast<int64_t>(tile / a.col_tiles) * 128 + (wave >> 1) * 64;
    const int64_t d0 = static_cast<int64_t>(tile % a.col_tiles) * 128 + (wave & 1) * 64;
    if (v0 >= a.vocab || d0 >= a.dim) return;
    const int blocks = (*a.count + kOuterRows - 1) / kOuterRows;
    uint32_t vo[2], ho[2];  // columns read: past the last one, the last
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint32_t half = static_cast<uint32_t>(lane >> 5) * 16u;
        vo[x] = static_cast<uint32_t>(min(v0 + 32 * x + (lane & 31), a.vocab - 1)) * kOuterBytes + half;
        ho[x] = static_cast<uint32_t>(min(d0 + 32 * x + (lane & 31), a.dim - 1)) * kOuterBytes + half;
    }
    floatx16 acc[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
    struct Step {
        Parts v[2], h[2];
    };
    auto load = [&](int b, Step &s) {
        const uint8_t *dz = a.dz + b * a.vocab * kOuterBytes, *h = a.h + b * a.dim * kOuterBytes;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                s.v[x].p[p] = *as_global(reinterpret_cast<const bf16x8 *>(dz + vo[x] + p * kOuterRows * 2));
                s.h[x].p[p] = *as_global(reinterpret_cast<const bf16x8 *>(h + ho[x] + p * kOuterRows * 2));
            }
    };
    auto step = [&](const Step &s) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) acc[x][y] = multiply(s.v[x], s.h[y], acc[x][y]);
    };
    Step s0, s1;
    if (blocks > 0) load(0, s0);
    for (int b = 0; b < blocks; b += 2) {
        if (b + 1 < blocks) load(b + 1, s1);
        step(s0);
        if (b + 1 >= blocks) break;
        if (b + 2 < blocks) load(b + 2, s0);
        step(s1);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t v = v0 + 32 * x + 8 * g + 4 * (lane >> 5) + e;
                if (v >= a.vocab) continue;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int64_t d = d0 + 32 * y + (lane & 31);
                    if (d < a.dim) as_global(a.out)[v * a.dim + d] = acc[x][y][4 * g + e];
                }
            }
}

// Sums of the products with the head: [split][rows][ld], in as many splits as the product took for the rows
struct Sums {
    float *at;
    int64_t ld, split_stride;
    int tile_rows, col_tiles, most;
    int cost;

    __device__ __forceinline__ int splits(int64_t rows) const {
        return most == 1 || rows == 0 ? 1 : splits_for(static_cast<int>(ceil_div(rows, tile_rows)) * col_tiles, most, cost);
    }
    __device__ __forceinline__ f32x4_v row4(int64_t row, int64_t c, int splits) const {
        f32x4_v v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < splits; ++s) v += *as_global(reinterpret_cast<const f32x4_v *>(at + s * split_stride + row * ld + c));
        return v;
    }
};

// ---- rows' results ---------------------------------------------------------------------------------------------
struct FinishArgs {
    const float2 *part;
    const float *sum, *at_target;
    const float *exps, *ref;  // in place of part: sums of 2^(z - ref), and ref by row
    int64_t part_stride, row_stride;
    int parts;
    int64_t n, vocab;
    Saved s;
    const int32_t *count, *which;  // rows, and the counted rows that they are; null: those themselves
    float *logps;        // by source row, or null
    float *row_loss;     // by counted row, or null
    float smoothing, z_loss;
    RowGrad *grad;       // of z itself, for rows that are made again: a q, nothing at the target; or null
    int uncounted;       // the logps of source rows that do not count are written too: zeros
};

// A row's parts joined: WIDE 256 threads per row (few rows), else 16 rows by 16 threads each
template <bool WIDE>
__global__ __launch_bounds__(256) void finish_kernel(const FinishArgs a) {
    constexpr int kRows = WIDE ? 1 : 16, kSlices = 256 / kRows, kLast = WIDE ? 4 : 16;
    __shared__ Sum2 s_all[WIDE ? 4 : 256];
    __shared__ double s_sum[WIDE ? 4 : 256];
    const int tid = threadIdx.x, slice = tid / kRows;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + tid % kRows;
    const int64_t count = a.count ? *a.count : *a.s.count;
    if (a.uncounted && a.logps && tid < kRows && r < a.n && a.s.place[r] < 0) a.logps[r] = 0.f;
    if (static_cast<int64_t>(blockIdx.x) * kRows >= count) return;
    Sum2 all = {-__builtin_inff(), 0.f};
    double sum = 0.0;
    if (r < count) {
        if (a.exps) {
            all.m = a.ref[r];
            for (int p = slice; p < a.parts; p += kSlices) all.s += a.exps[p * a.part_stride + r * a.row_stride];
        } else {
            for (int p = slice; p < a.parts; p += kSlices) {
                const float2 x = a.part[p * a.part_stride + r * a.row_stride];
                all = join(all, {x.x, x.y});
            }
        }
        if (a.sum)
            for (int p = slice; p < a.parts; p += kSlices) sum += a.sum[p * a.part_stride + r * a.row_stride];
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
    if (tid >= kRows || r >= count) return;
    all = s_all[tid], sum = s_sum[tid];
    for (int i = 1; i < kLast; ++i) all = join(all, s_all[tid + i * kRows]), sum += s_sum[tid + i * kRows];
    // d: how far the others' sum is over the target, log2
    const float zt = a.at_target[r], rest = all.m + log2f(all.s);
    const float d = (all.m - zt) + log2f(all.s);  // the difference of two large values first: nothing is rounded
    const float e = exp2f(-fabsf(d)), more = log1pf(e);
    const float nll = static_cast<float>(kLn2) * fmaxf(d, 0.f) + more;
    const float others = d > 0.f ? 1.f / (1.f + e) : e / (1.f + e);
    const float lse2 = (d > 0.f ? rest : zt) + more * kLog2e;
    const int64_t c = a.which ? a.which[r] : r;
    a.s.lse2[c] = lse2;
    a.s.others[c] = d != d ? d : others;
    if (a.logps) a.logps[a.s.rows[c]] = -nll;
    if (a.grad) a.grad[r] = {lse2, 1.f + 2.f * a.z_loss * static_cast<float>(kLn2) * lse2, 0.f, 0.f};
    if (a.row_loss) {
        const float lse = static_cast<float>(kLn2) * lse2;
        float loss = nll + a.z_loss * lse * lse;
        if (a.smoothing != 0.f) loss += a.smoothing * static_cast<float>(kLn2 * (zt - sum / static_cast<double>(a.vocab)));
        a.row_loss[c] = loss;
    }
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

// Four values of a row of the hidden states' gradient
template <bool F32>
__device__ __forceinline__ void store4(void *out, int64_t at, int64_t c, int64_t dim, const f32x4_v &v) {
    if constexpr (F32) {
        float *o = static_cast<float *>(out) + at + c;
        if (dim % 4 == 0) {
            *as_global(reinterpret_cast<f32x4_v *>(o)) = v;
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < dim) o[e] = v[e];
    } else {
        uint16_t *o = static_cast<uint16_t *>(out) + at + c;
        uint16_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = float_to_bf16_bits_rne(v[e]);
        if (dim % 4 == 0) {
            *as_global(reinterpret_cast<u32x2_v *>(o)) = u32x2_v{b[0] | (static_cast<uint32_t>(b[1]) << 16), b[2] | (static_cast<uint32_t>(b[3]) << 16)};
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < dim) o[e] = b[e];
    }
}

// What bf16 leaves of the logits' gradient at the rows' targets
struct Rest {
    const RowGrad *grad;
    const int32_t *tgt;
    const uint16_t *weight;
    int64_t w_stride;
    const float *factor;  // of the whole, or null
};

// Gradient of the hidden states, source rows in their order: the splits' sums, or zeros
template <bool F32>
__global__ __launch_bounds__(256) void hidden_kernel(const Sums sums, const int32_t *place, const int32_t *count, int64_t n, int64_t dim, const Rest rest, void *out) {
    const int64_t units = ceil_div(dim, 4);
    const int splits = sums.splits(*count);
    const float f = !F32 && rest.factor != nullptr ? *as_global(rest.factor) : 1.f;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < n * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t i = u / units, c = (u - i * units) * 4;
        const int64_t r = place[i];
        f32x4_v v = {0.f, 0.f, 0.f, 0.f};
        if (r >= 0) {
            v = sums.row4(r, c, splits);
            if constexpr (!F32) {
                const float left = rest.grad[r].gt - round_to_bf16(rest.grad[r].gt);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < dim) v[e] = f * fmaf(left, bf16_bits_to_float(rest.weight[rest.tgt[r] * rest.w_stride + c + e]), v[e]);
            }
        }
        store4<F32>(out, i * dim, c, dim, v);
    }
}

// ---- the hidden states' gradient from the forward's exponentials ---------------------------------------------------
// Where the head takes no gradient, the forward's tiles of logits are worth a second use: their exponentials
// 2^(z - ref), with ref the target's logit, go through the product with W as they are, and the row's sum, known when all
// pieces are through, scales the result: D = a sum_{j != t} q_j w_j + (a q_t - 1) w_t, the gradient of a loss of
// upstream 1 before the factors that rows share; the target's term in fp32. The backward only scales D. ref is no
// maximum: a row whose sum passes 2^100 (its loss is over some 69) or is not finite is made again by the plain way
// (statistics, then gradient), in launches that find no row otherwise.
__global__ __launch_bounds__(256) void ref_kernel(const Layout h, const uint16_t *weight, int64_t w_stride, const int32_t *tgt, float k, float *ref) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= *h.count) return;
    const int lane = threadIdx.x & 63;
    const int64_t from = h.rows[r], at = from / h.per_batch * h.batch_stride + from % h.per_batch * h.row_stride;
    const int64_t w = tgt[r] * w_stride;
    float sum = 0.f;
    const auto x = as_global(static_cast<const uint16_t *>(h.src) + at), y = as_global(weight + w);
    for (int64_t c = lane * 8; c < h.dim; c += 512) {
        if (c + 8 <= h.dim) {
            const u32x4_any a = *(gmem_ptr<const u32x4_any>)(x + c), b = *(gmem_ptr<const u32x4_any>)(y + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sum = fmaf(__uint_as_float(a[j] << 16), __uint_as_float(b[j] << 16), sum);
                sum = fmaf(__uint_as_float(a[j] & 0xffff0000u), __uint_as_float(b[j] & 0xffff0000u), sum);
            }
        } else {
            for (int64_t i = c; i < h.dim; ++i) sum += bf16_bits_to_float(x[i]) * bf16_bits_to_float(y[i]);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    sum *= k;
    if (lane == 0) ref[r] = __builtin_fabsf(sum) < __builtin_inff() ? sum : 0.f;
}

// Rows to make again, in order, with their targets. One workgroup.
struct RedoArgs {
    Saved s;
    const float *ref;
    const int32_t *tgt;
    int32_t *count, *rows, *tgt2;
};

__global__ __launch_bounds__(kIndexThreads) void redo_kernel(const RedoArgs a) {
    __shared__ int sums[kIndexThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = *a.s.count;
    int at = 0;
    for (int i0 = 0; i0 < n; i0 += kIndexThreads) {
        const int i = i0 + tid;
        // the row's sum is 2^(lse2 - ref), at least about 1, as the target is one of its terms; NaN is bad too
        const float over = i < n ? a.s.lse2[i] - a.ref[i] : 0.f;
        const bool bad = !(over > -1.f && over < 100.f);
        const uint64_t mask = __ballot(bad);
        if (lane == 0) sums[wave] = __popcll(mask);
        __syncthreads();
        int before = at, all = 0;
        for (int w = 0; w < kIndexThreads / 64; ++w) {
            before += w < wave ? sums[w] : 0;
            all += sums[w];
        }
        if (bad) {
            const int r = before + __popcll(mask & ((uint64_t{1} << lane) - 1));
            a.rows[r] = i;
            a.tgt2[r] = a.tgt[i];
        }
        at += all;
        __syncthreads();
    }
    if (tid == 0) *a.count = at;
}

// Sums of the head's columns, which a smoothed target's gradient takes in: chunks of rows, then over the chunks
constexpr int kColumnRows = 512;

__global__ __launch_bounds__(256) void column_kernel(const uint16_t *weight, int64_t w_stride, int64_t vocab, int64_t dim, float *part) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= dim) return;
    const int64_t v0 = static_cast<int64_t>(blockIdx.y) * kColumnRows, v1 = min(vocab, v0 + kColumnRows);
    float sum = 0.f;
#pragma unroll 8
    for (int64_t v = v0; v < v1; ++v)
        sum += bf16_bits_to_float(weight[v * w_stride + c]);
    part[blockIdx.y * dim + c] = sum;
}

__global__ __launch_bounds__(256) void column_total_kernel(const float *part, int chunks, int64_t dim, float *out) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= dim) return;
    double sum = 0.0;
    for (int i = 0; i < chunks; ++i) sum += static_cast<double>(part[i * dim + c]);
    out[c] = static_cast<float>(sum);
}

struct UnitArgs {
    Sums sums;
    Saved s;
    const int32_t *count, *which;  // as FinishArgs
    const int32_t *tgt;            // by row of sums
    const float *ref;              // null: sums are of a q
    const uint16_t *weight;
    int64_t w_stride, dim, n;
    float z_loss, smoothing;
    const float *columns;          // sums of the head's columns, null without smoothing
    double vocab;
    float *unit;                   // [counted rows][dim rounded up to 4]
};

__global__ __launch_bounds__(256) void unit_kernel(const UnitArgs a) {
    const int64_t units = ceil_div(a.dim, 4);
    const int64_t count = a.count ? *a.count : *a.s.count;
    const int splits = a.sums.splits(count);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < count * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = u / units, c = (u - r * units) * 4;
        const int64_t at = a.which ? a.which[r] : r;
        const float lse2 = a.s.lse2[at];
        const float more = 2.f * a.z_loss * static_cast<float>(kLn2) * lse2;
        const float own = more - (1.f + more) * a.s.others[at] + a.smoothing;
        const float each = a.columns ? static_cast<float>(a.smoothing / a.vocab) : 0.f;
        const float scale = a.ref ? (1.f + more) * __builtin_amdgcn_exp2f(a.ref[r] - lse2) : 1.f;
        f32x4_v v = a.sums.row4(r, c, splits);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float w = 0.f, all = 0.f;
            if (c + e < a.dim) {
                if (a.columns) all = each * a.columns[c + e];
                w = bf16_bits_to_float(a.weight[a.tgt[r] * a.w_stride + c + e]);
            }
            v[e] = fmaf(v[e], scale, fmaf(own, w, -all));
        }
        *as_global(reinterpret_cast<f32x4_v *>(a.unit + at * units * 4 + c)) = v;
    }
}

// The backward where the forward left D
struct ScaleArgs {
    const float *unit;
    const int32_t *count, *place;
    const float *upstream;
    int per_row, mean;
    double scale;  // of the loss, over T
    int64_t n, dim;
    void *out;
};

__global__ __launch_bounds__(256) void scale_kernel(const ScaleArgs a) {
    const int64_t units = ceil_div(a.dim, 4);
    const double all = a.per_row ? -a.scale : static_cast<double>(*a.upstream) * a.scale / (a.mean ? max(*a.count, 1) : 1);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < a.n * units; u += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t i = u / units, c = (u - i * units) * 4;
        const int64_t r = a.place[i];
        f32x4_v v = {0.f, 0.f, 0.f, 0.f};
        if (r >= 0) {
            const float f = static_cast<float>(a.per_row ? all * static_cast<double>(a.upstream[i]) : all);
            v = *as_global(reinterpret_cast<const f32x4_v *>(a.unit + r * units * 4 + c)) * f;
        }
        store4<false>(a.out, i * a.dim, c, a.dim, v);
    }
}

// ---- plan: sizes and places in the workspace ---------------------------------------------------------------------
// the forward alone, the backward, the forward that leaves D or its logits, the backward that has them
enum Pass { kStats, kBackward, kLeavesUnit, kHasUnit };  // (or, of fp32 in parts, the laid-out head)

struct Plan {
    int64_t n, rows, vocab, dim, ld;  // rows: n rounded up, at least 64; ld: dim rounded up to whole slabs
    bool f32, few, copy_w;            // copy_w: the head is laid out piece by piece
    int tile, cols;                   // rows of a tile, and columns of one of logits
    bool keeps;                       // the laid-out head is the forward's for the backward too (keeps_head)
    bool rest;                        // the gradient's rows twice: as bf16, and what that leaves
    int np, nz;                       // parts of an operand: of the head's gradient; of the logits and the hidden states' gradient
    int64_t piece;                    // columns of the vocabulary at a time
    int splits;                       // of the product with W, at most
    int split_cost;
    int64_t h, part, sum, at_target, row_loss, g, grad, acc;  // workspace offsets
    int64_t ref, redo, h2, tgt2, columns, column_part, factor;
    int64_t z, wz, row_scale, col_scale;  // operands of the logits; fp32: fp16 parts, and their scales
    int64_t half, bound, largest;         // fp32: the gradient in fp16 parts, its rows' bounds, the scales' largest by piece
    int64_t bytes;
};

int64_t round_up(int64_t x, int64_t to) { return ceil_div(x, to) * to; }

// Columns of an array whose rows are read a few hundred bytes at a time, many rows together: an odd number of lines, or the
// rows' pieces would share few of the memory's channels (a vocabulary is often a multiple of a power of two)
int64_t odd_lines(int64_t columns) { return (ceil_div(columns, 64) | 1) * 64; }

// Whether the tiles of few rows are taken, and of 64 rows or 128. Up to 128 rows always: the read of the head is what they
// wait for. More where 64-row tiles all find a place at once, so larger ones would leave CUs without work, and up to
// twice as many where 256-row tiles would and a tile's K loop is short. us, few / 256-row tiles, log-probabilities
// alone unless said otherwise:
//   262,144 x 5376   129 rows 898 (64-row tiles) / 646; 128 rows 547 (128-row tiles, 658 with 64)
//   32,000 x 1024    129 rows 37 / 57, 256 rows 38 / 59, 384 rows 59 / 60
//   32,000 x 2048    256 rows 53 / -, 384 rows 88 / 81;  32,000 x 4096, 256 rows, with the hidden states' gradient 262 / 248
//   5,000 x 512      512 rows 27 / 46
// fp32: where 64-row tiles all find a place at once.
bool takes_few(int64_t n, int64_t vocab, int64_t dim, bool f32) {
    return ceil_div(n, 64) * ceil_div(vocab, kTile) <= 256 || (!f32 && (n <= kFew || (n <= 2 * kFew && vocab <= 65536 && dim <= 2048)));
}

// Whether a call goes by kept logits (a forward alone too, in its workspace): few rows, and more of them where 256-row
// tiles of parts would leave CUs without work. Parts / kept logits, us, the gradient of the hidden states:
//   262,144 x 5376   257 rows 15,663 / 11,401, 384 rows 16,503 / 14,612, 512 rows 17,476 / 19,244
//   32,000 x 1024    257 rows 512 / 328, 512 rows 547 / 510 (250 tiles), 768 rows 738 / 781
//   10,113 x 5376    384 rows 862 / 612, 768 rows 1165 / 1116;  3,423 x 4608, 768 rows 557 / 471
bool takes_kept(int64_t n, int64_t vocab, int dtype) {
    return dtype == ME_F32 && n >= 1 && (n <= kKeptRows || (n <= kKeptMost && ceil_div(n, kTile) * ceil_div(vocab, kTile) <= 256));
}

int64_t kept_ld(int64_t vocab) { return odd_lines(vocab); }

// Parts of a reduction over `slabs` slabs that `tiles` tiles take to fill the chip, at least four slabs each
int most_splits(int64_t tiles, int64_t slabs) {
    return static_cast<int>(std::max<int64_t>(std::min<int64_t>({std::max<int64_t>(256 / tiles, kSplits), kMostSplits, slabs / 4}), 1));
}

// What a call by kept logits needs
struct KeptPlan {
    int64_t n, vocab, dim, ld, h_ld, row_tiles;
    int tile, piece;                       // rows of a tile; Loader's PIECE of the head
    int logit_splits, logit_cost, splits, split_cost;
    int64_t h, logits, partial, part, sum, at_target, row_loss, dz, acc, dz_parts, h_parts, bytes;
};

KeptPlan kept_plan_of(int64_t n, int64_t vocab, int64_t dim, const void *weight, int64_t w_stride, Pass pass, bool smoothed) {
    KeptPlan p{};
    p.n = n, p.vocab = vocab, p.dim = dim, p.ld = kept_ld(vocab), p.h_ld = round_up(dim, 32);
    // the logits' tiles: two workgroups to a CU; the others': one
    p.tile = pass != kHasUnit ? (n <= 32 ? 32 : 64) : static_cast<int>(round_up(ceil_div(n, ceil_div(n, 128)), 32));
    p.row_tiles = ceil_div(n, p.tile);
    p.piece = dim % 4 == 0 && w_stride % 4 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0 ? 16 : 4;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    if (pass != kHasUnit) {
        const int64_t tiles = p.row_tiles * ceil_div(vocab, kTile);
        // the sums' bytes against the head's
        p.logit_splits = tiles > 512 ? 1 : most_splits(tiles, ceil_div(dim, 32));
        p.logit_cost = static_cast<int>(std::min<int64_t>(4096 * 2 * n / dim + 1, kMostCost));
        p.h = take(n * p.h_ld * 4);
        if (pass == kStats) p.logits = take(n * p.ld * 4);
        if (p.logit_splits > 1) p.partial = take(p.logit_splits * n * p.ld * 4);
        const int64_t parts = std::max<int64_t>(ceil_div(p.ld, kKeptCols), n <= kVectorRows ? kVectorGroups : 0);
        p.part = take(parts * n * 8);
        if (smoothed) p.sum = take(parts * n * 4);
        p.at_target = take(n * 4);
        p.row_loss = take(n * 4);
    } else {
        p.splits = most_splits(p.row_tiles * ceil_div(dim, kTile), ceil_div(vocab, 32));
        p.split_cost = static_cast<int>(std::min<int64_t>(4096 * 2 * n / vocab + 1, kMostCost));
        p.dz = take(n * p.ld * 4);
        p.acc = take(p.splits * n * p.h_ld * 4);
        p.dz_parts = take(ceil_div(n, kOuterRows) * vocab * kOuterBytes);
        p.h_parts = take(ceil_div(n, kOuterRows) * dim * kOuterBytes);
    }
    p.bytes = at;
    return p;
}

// Whether the head's gradient takes what bf16 leaves of the logits' gradient: few rows, where one value's rounding can
// make most of a result's error (2 rows: up to 2.5 times that of rounding the result alone, 1.0 with it; 128 rows: 1.3 to
// 1.5). The product is bound by the write of its result, and K of 128 or 256 makes no difference to it.
bool takes_rest(int64_t n, bool f32) { return !f32 && n <= kFew; }

int few_rows(int64_t n, int64_t vocab) { return n <= 64 || ceil_div(n, 64) * ceil_div(vocab, kTile) <= 256 ? 64 : 128; }

// Whether a forward in parts leaves the laid-out head for the backward: up to 1 GiB of it (32,000 x 1024: 77 us of a
// step's 1160 with 1023 rows, 2150 with 2048)
bool keeps_head(int64_t n, int64_t vocab, int64_t dim, int dtype) {
    return dtype == ME_F32 && n >= 1 && !takes_kept(n, vocab, dtype) && vocab * round_up(dim, kSlabK) * 4 <= kPieceBytes;
}

// The head in parts, as long as it is, with its scales and the largest of these
struct KeptHead {
    uint8_t *parts;
    float *scale;
    uint32_t *largest;
    int64_t part, elements;  // part: bytes; elements: 4 bytes each, of all of it
};

KeptHead kept_head_of(float *unit, int64_t vocab, int64_t dim) {
    const int64_t ld = round_up(dim, kSlabK), scales = round_up(vocab, 4) + kTile;
    return {reinterpret_cast<uint8_t *>(unit), unit + vocab * ld, reinterpret_cast<uint32_t *>(unit + vocab * ld + scales), vocab * ld * 2, vocab * ld + scales + 4};
}

// Columns of a wave's statistics
int part_cols(const Plan &p) { return p.few ? p.cols / 4 : 128; }

Plan plan_of(int64_t n, int64_t vocab, int64_t dim, int dtype, const void *weight, int64_t w_stride, Pass pass, bool smoothed) {
    Plan p{};
    p.keeps = dtype == ME_F32 && (pass == kLeavesUnit || pass == kHasUnit);
    if (p.keeps) pass = pass == kLeavesUnit ? kStats : kBackward;
    p.n = n, p.vocab = vocab, p.dim = dim, p.ld = round_up(dim, kSlabK);
    p.f32 = dtype == ME_F32;
    p.np = p.f32 ? 3 : 1;
    p.nz = p.f32 ? 2 : 1;
    p.few = takes_few(n, vocab, dim, p.f32);
    p.rest = pass == kBackward && takes_rest(n, p.f32);
    p.copy_w = p.f32 || dim % 8 != 0 || w_stride % 8 != 0 || reinterpret_cast<uintptr_t>(weight) % 16 != 0;
    p.tile = p.few ? few_rows(n, vocab) : kTile;
    // tiles of 256 / 128 columns, us, log-probabilities or loss alone of 48 rows: 5,000 x 5376 68 / 50, 10,000 x 2048 38 / 30,
    // 25,000 x 4096 57 / 45, 32,000 x 1024 29 / 29
    p.cols = p.few && ceil_div(n, p.tile) * ceil_div(vocab, kTile) <= 128 ? 128 : kTile;
    const int64_t rows = p.rows = round_up(std::max<int64_t>(n, 1), 64);
    int64_t piece = round_up(vocab, kTile);
    if (p.copy_w && !p.keeps) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (p.ld * 2 * p.nz) / 2048 * 2048, 2048));
    if (pass != kStats) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (rows * (p.f32 ? 10 : 2)) / 2048 * 2048, 2048));
    // a launch holds fewer than 2^32 threads
    p.piece = std::min(piece, std::max<int64_t>((int64_t{1} << 23) / ceil_div(rows, p.tile) * kTile / 2048 * 2048, 2048));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    p.grad = take(n * static_cast<int64_t>(sizeof(RowGrad)));
    p.factor = take(4);
    p.z = take(rows * p.ld * 2 * (p.rest ? 2 : p.nz));
    p.h = p.z;
    if (p.copy_w && !p.keeps) p.wz = take(p.piece * p.ld * 2 * p.nz);
    if (p.f32) {
        p.row_scale = take(n * 4);
        if (!p.keeps) p.col_scale = take((p.piece + kTile) * 4);
        if (pass == kBackward) {
            p.h = take(rows * p.ld * 2 * p.np);
            p.half = take(rows * p.piece * 2 * p.nz);
            p.bound = take(n * 4);
            if (!p.keeps) p.largest = take(ceil_div(vocab, p.piece) * 4);
        }
    }
    if (pass != kBackward) {
        const int64_t parts = std::max<int64_t>(ceil_div(vocab, part_cols(p)) + 4, n <= kVectorRows ? kVectorGroups : 0);
        p.part = take(parts * rows * 8);
        if (smoothed) p.sum = take(parts * rows * 4);
        p.at_target = take(n * 4);
        p.row_loss = take(n * 4);
    }
    if (pass != kStats) {
        p.g = take(rows * p.piece * 2 * (p.rest ? 2 : p.np));
        // at least eight slabs each; parts of few tiles are as many as fill the chip, those of many up to kSplits as far as
        // their sums take a piece's memory (2049 rows, 262,144 x 5376: 189 tiles in 4 parts are 2.95 rounds, in 3 2.2)
        const int64_t tiles = ceil_div(rows, p.tile) * ceil_div(dim, kTile);
        const int64_t most = std::max<int64_t>(256 / tiles, std::min<int64_t>(kSplits, kPieceBytes / (rows * p.ld * 4)));
        p.splits = static_cast<int>(std::max<int64_t>(std::min<int64_t>({most, kMostSplits, p.piece / kSlabK / 8}), 1));
        // reading and writing the sums at 4.8 TB/s against a piece's products at 1.25 PFLOP/s; twice, as a round that is not full
        // runs at a higher clock (5000 rows, 100,003 x 2048: 3616 us with 3 parts, 3701 with the 8 that once would choose)
        p.split_cost = static_cast<int>(4096 * 2 * (8.0 / 4.8e12) / (2.0 * static_cast<double>(p.piece) * (p.f32 ? 3 : 1) / 1.25e15)) + 1;
        p.acc = take(p.splits * rows * p.ld * 4);
    }
    if (pass == kLeavesUnit) {
        p.ref = take(n * 4);
        p.redo = take((kHeader + n) * 4);
        p.h2 = take(rows * p.ld * 2);
        p.tgt2 = take(n * 4);
        if (smoothed) {
            p.columns = take(dim * 4);
            p.column_part = take(ceil_div(vocab, kColumnRows) * dim * 4);
        }
    }
    p.bytes = at;
    return p;
}

// Whether a forward for the hidden states' gradient alone leaves D: bf16, where it saves the backward one of three
// products (few rows: one of three reads of the head) and that is worth some ten launches more. (fp32: the
// exponentials would need six products with the head, where the gradient, whose size is known, needs three.)
bool leaves_unit(int64_t n, int64_t vocab, int64_t dim, int dtype) {
    const double product = 2.0 * static_cast<double>(n) * vocab * dim / 1.2e15, read = 2.0 * static_cast<double>(vocab) * dim / 5e12;
    return dtype == ME_BF16 && std::max(product, read) > 50e-6;
}

struct Call {
    const void *hidden, *weight, *targets;
    int64_t per_batch, batch_stride, row_stride, w_stride, ignore;
    int tdtype;
    uint8_t *ws;
    Saved s;
    hipStream_t stream;
    float *unit = nullptr;  // the laid-out head
    bool laid_out = false;  // and it is there already
};

unsigned blocks_for(int64_t units) { return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(units, 256), 1), 16384)); }

void lay_out(bool f32, const Layout &l, hipStream_t s, const Coefs &k = Coefs{}) {
    const unsigned blocks = blocks_for(l.n * (l.ld / 8));
    if (f32)
        hipLaunchKernelGGL(layout_kernel<true>, dim3(blocks), dim3(256), 0, s, l, k);
    else
        hipLaunchKernelGGL(layout_kernel<false>, dim3(blocks), dim3(256), 0, s, l, k);
}

int64_t h_part(const Plan &p) { return p.rows * p.ld * 2; }

Layout hidden_layout(const Plan &p, const Call &c, int64_t to) {
    return {c.hidden, c.per_batch, c.batch_stride, c.row_stride, c.s.rows, c.s.count, p.n, p.dim, p.ld, h_part(p), c.ws + to, p.rest};
}

void lay_out16(const Layout &l, float *scale, uint32_t *largest, hipStream_t s, const Coefs &k = Coefs{}) {
    // a thread for each piece's largest scale among them (pieces of 2048 columns or more: at most 1024)
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>({ceil_div(l.n, 4), 1, k.grad ? 4 : 1}), 2048));
    hipLaunchKernelGGL(layout16_kernel, dim3(blocks), dim3(256), 0, s, l, scale, largest, k);
}

// Rows of a product: the hidden states laid out for the logits, with how many there are, their targets and, of
// fp16 parts, their scales
struct Rows {
    uint8_t *h;
    const int32_t *count, *tgt;
    const float *scale;
};

Rows lay_out_rows(const Plan &p, const Call &c, const Coefs &k = Coefs{}) {
    float *scale = p.f32 ? reinterpret_cast<float *>(c.ws + p.row_scale) : nullptr;
    if (p.f32)
        lay_out16(hidden_layout(p, c, p.z), scale, nullptr, c.stream, k);
    else
        lay_out(false, hidden_layout(p, c, p.z), c.stream, k);
    return {c.ws + p.z, c.s.count, c.s.tgt, scale};
}

// The head from row v0 on, `width` rows of it
struct Head {
    Operand w;
    const float *scale;  // of fp16 parts, by row
};

Head head_of(const Plan &p, const Call &c, int64_t v0, int64_t width, uint32_t *largest = nullptr, const int32_t *gate = nullptr) {
    const uint8_t *from = static_cast<const uint8_t *>(c.weight) + v0 * c.w_stride * (p.f32 ? 4 : 2);
    if (!p.copy_w) return {{from, c.w_stride, 0}, nullptr};
    if (p.keeps) {
        const KeptHead k = kept_head_of(c.unit, p.vocab, p.dim);
        uint8_t *to = k.parts + v0 * p.ld * 2;
        const Layout l{from, width, 0, c.w_stride, nullptr, nullptr, width, p.dim, p.ld, k.part, to, 0, nullptr};
        if (!c.laid_out) lay_out16(l, k.scale + v0, k.largest, c.stream);
        return {{to, p.ld, k.part}, k.scale + v0};
    }
    const int64_t part = p.piece * p.ld * 2;
    const Layout l{from, width, 0, c.w_stride, nullptr, nullptr, width, p.dim, p.ld, part, c.ws + p.wz, 0, gate};
    float *scale = p.f32 ? reinterpret_cast<float *>(c.ws + p.col_scale) : nullptr;
    if (p.f32)
        lay_out16(l, scale, largest, c.stream);
    else
        lay_out(false, l, c.stream);
    return {{c.ws + p.wz, p.ld, part}, scale};
}

template <bool A_KC, bool B_KC, int SEGS, class Epilogue>
void multiply_large(const Gemm &g, const Epilogue &e, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(workgroups(g, kTile, kTile)));
    hipLaunchKernelGGL((large_kernel<A_KC, B_KC, SEGS, Epilogue>), grid, dim3(kThreads), 0, s, g, e);
}

template <bool B_KC, int TS, int SEGS, class Epilogue>
void multiply_few(int tile, const Gemm &g, const Epilogue &e, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(workgroups(g, tile, TS)));
    if constexpr (SEGS == 1) {  // parts: 64 rows alone (takes_few)
        if (tile == 128) {
            hipLaunchKernelGGL((few_kernel<B_KC, 4, TS, 1, 16, Epilogue>), grid, dim3(kThreads), 0, s, g, e);
            return;
        }
    }
    hipLaunchKernelGGL((few_kernel<B_KC, 2, TS, SEGS, 16, Epilogue>), grid, dim3(kThreads), 0, s, g, e);
}

// logits of few rows
template <int SEGS, class Epilogue>
void few_logits(const Plan &p, const Gemm &g, const Epilogue &e, hipStream_t s) {
    p.cols == 128 ? multiply_few<true, 128, SEGS>(p.tile, g, e, s) : multiply_few<true, kTile, SEGS>(p.tile, g, e, s);
}

// fp32 as it lies
template <bool B_KC, int PIECE>
void multiply_kept(int tile, const Gemm &g, const AccumulateEpilogue &e, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(workgroups(g, tile, kTile)));
    if (tile == 32)
        hipLaunchKernelGGL((few_kernel<B_KC, 1, kTile, 0, PIECE, AccumulateEpilogue>), grid, dim3(kThreads), 0, s, g, e);
    else if (B_KC || tile == 64)
        hipLaunchKernelGGL((few_kernel<B_KC, 2, kTile, 0, PIECE, AccumulateEpilogue>), grid, dim3(kThreads), 0, s, g, e);
    else if constexpr (!B_KC) {
        if (tile == 96)
            hipLaunchKernelGGL((few_kernel<false, 3, kTile, 0, PIECE, AccumulateEpilogue>), grid, dim3(kThreads), 0, s, g, e);
        else
            hipLaunchKernelGGL((few_kernel<false, 4, kTile, 0, PIECE, AccumulateEpilogue>), grid, dim3(kThreads), 0, s, g, e);
    }
}

template <bool B_KC>
void multiply_kept(const KeptPlan &p, const Gemm &g, const AccumulateEpilogue &e, hipStream_t s) {
    p.piece == 16 ? multiply_kept<B_KC, 16>(p.tile, g, e, s) : multiply_kept<B_KC, 4>(p.tile, g, e, s);
}

// logits of a piece: rows x head rows
template <int SEGS, class Epilogue>
void logits_of(const Plan &p, const Call &c, const Rows &rows, const Head &w, int64_t width, const Epilogue &e) {
    const Gemm g{{rows.h, p.ld, h_part(p)}, w.w, p.n, width, p.dim, rows.count, 0, 8, 1, 0};
    if (p.few)
        few_logits<SEGS>(p, g, e, c.stream);
    else
        multiply_large<true, true, SEGS>(g, e, c.stream);
}

// product of a piece of the logits' gradient (or exponentials) with the head, onto the sums
void times_head(const Plan &p, const Call &c, const Rows &rows, const Head &w, int64_t v0, int64_t width, const uint32_t *largest = nullptr) {
    const Operand dz{c.ws + (p.f32 ? p.half : p.g), p.piece, p.rows * p.piece * 2};
    const Gemm g{dz, w.w, p.n, p.dim, width, rows.count, 0, 8, p.splits, p.split_cost};
    const AccumulateEpilogue e{reinterpret_cast<float *>(c.ws + p.acc), p.ld, p.rows * p.ld, v0 > 0,
                               p.f32 ? reinterpret_cast<const float *>(c.ws + p.bound) : nullptr, largest};
    if (p.few)
        p.f32 ? multiply_few<false, kTile, 3>(p.tile, g, e, c.stream) : multiply_few<false, kTile, 1>(p.tile, g, e, c.stream);
    else
        p.f32 ? multiply_large<true, false, 3>(g, e, c.stream) : multiply_large<true, false, 1>(g, e, c.stream);
}

Sums sums_of(const Plan &p, const Call &c) {
    return {reinterpret_cast<float *>(c.ws + p.acc), p.ld, p.rows * p.ld, p.tile, static_cast<int>(ceil_div(p.dim, kTile)), p.splits, p.split_cost};
}

// gradient of the logits of a piece, for the products that follow
template <int PARTS>
void gradient_of(const Plan &p, const Call &c, const Rows &rows, const Head &w, int64_t v0, int64_t width, const RowGrad *grad, float k,
                 const uint32_t *largest, bool for_hidden, bool for_weight) {
    constexpr bool kF32 = PARTS == 3;
    const GradEpilogue<PARTS> e{rows.tgt, {rows.scale, w.scale}, grad, kF32 ? reinterpret_cast<const float *>(c.ws + p.bound) : nullptr, largest,
                                !kF32 || for_weight ? c.ws + p.g : nullptr, kF32 && for_hidden ? c.ws + p.half : nullptr, p.piece,
                                p.rows * p.piece * 2, v0, width, k};
    if constexpr (PARTS == 2) {  // few rows
        const Gemm g{{rows.h, p.ld, 0}, w.w, p.n, width, p.dim, rows.count, 0, 8, 1, 0};
        few_logits<1>(p, g, e, c.stream);
    } else {
        logits_of<PARTS>(p, c, rows, w, width, e);
    }
}

void finish(const Plan &p, const FinishArgs &f, hipStream_t s) {
    if (p.few)
        hipLaunchKernelGGL(finish_kernel<true>, dim3(static_cast<unsigned>(p.n)), dim3(256), 0, s, f);
    else
        hipLaunchKernelGGL(finish_kernel<false>, dim3(static_cast<unsigned>(ceil_div(p.n, 16))), dim3(256), 0, s, f);
}

struct Loss {
    double temperature, smoothing, z_loss, scale;
    int mean;
    float *logps, *loss;  // one of them
    float *unit;          // D, or null
};

// D from the sums of the products with the head
void unit_of(const Plan &p, const Call &c, const Loss &l, const Rows &rows, const int32_t *which, const float *ref) {
    UnitArgs u{};
    u.sums = sums_of(p, c);
    u.s = c.s, u.count = rows.count, u.which = which, u.tgt = rows.tgt, u.ref = ref;
    u.weight = static_cast<const uint16_t *>(c.weight), u.w_stride = c.w_stride, u.dim = p.dim, u.n = p.n;
    u.z_loss = static_cast<float>(l.z_loss), u.smoothing = static_cast<float>(l.smoothing);
    u.columns = l.smoothing != 0.0 ? reinterpret_cast<const float *>(c.ws + p.columns) : nullptr;
    u.vocab = static_cast<double>(p.vocab);
    u.unit = l.unit;
    hipLaunchKernelGGL(unit_kernel, dim3(blocks_for(p.n * ceil_div(p.dim, 4))), dim3(256), 0, c.stream, u);
}

// Statistics of the rows' logits, piece by piece
template <bool F32>
void stats_of(const Plan &p, const Call &c, const Rows &rows, StatsEpilogue<F32> e, const int32_t *gate = nullptr) {
    e.tgt = rows.tgt;
    for (int64_t v0 = 0; v0 < p.vocab; v0 += p.piece) {
        const int64_t width = std::min(p.piece, p.vocab - v0);
        const Head w = head_of(p, c, v0, width, nullptr, gate);
        e.first = v0, e.vocab = width, e.scales = {rows.scale, w.scale};
        logits_of<F32 ? 3 : 1>(p, c, rows, w, width, e);
    }
}

template <bool F32>
void forward_rows(const Plan &p, const Call &c, const Loss &l) {
    hipStream_t s = c.stream;
    const Rows rows = lay_out_rows(p, c);
    const int cols = part_cols(p);
    const int parts = static_cast<int>(ceil_div(p.vocab, cols));
    const float k = static_cast<float>(1.44269504088896340736 / l.temperature);
    float *at_target = reinterpret_cast<float *>(c.ws + p.at_target);

    StatsEpilogue<F32> e{};
    e.part = reinterpret_cast<float2 *>(c.ws + p.part);
    e.sum = l.smoothing != 0.0 ? reinterpret_cast<float *>(c.ws + p.sum) : nullptr;
    e.at_target = at_target;
    e.part_stride = p.few ? 1 : p.rows;
    e.row_stride = p.few ? parts + 4 : 1;
    e.k = k;
    FinishArgs f{};
    f.part = e.part, f.sum = e.sum, f.at_target = at_target, f.part_stride = e.part_stride, f.row_stride = e.row_stride, f.parts = parts;
    f.n = p.n, f.vocab = p.vocab, f.s = c.s, f.logps = l.logps, f.uncounted = 1;
    f.row_loss = l.loss ? reinterpret_cast<float *>(c.ws + p.row_loss) : nullptr;
    f.smoothing = static_cast<float>(l.smoothing), f.z_loss = static_cast<float>(l.z_loss);
    if (F32 || !l.unit) {
        stats_of<F32>(p, c, rows, e);
        finish(p, f, s);
        return;
    }
    const uint16_t *weight = static_cast<const uint16_t *>(c.weight);
    float *ref = reinterpret_cast<float *>(c.ws + p.ref);
    hipLaunchKernelGGL(ref_kernel, dim3(static_cast<unsigned>(ceil_div(p.n, 4))), dim3(256), 0, s, hidden_layout(p, c, p.z), weight, c.w_stride,
                       rows.tgt, k, ref);
    if (l.smoothing != 0.0) {
        const dim3 grid(static_cast<unsigned>(ceil_div(p.dim, 256)), static_cast<unsigned>(ceil_div(p.vocab, kColumnRows)));
        float *part = reinterpret_cast<float *>(c.ws + p.column_part);
        hipLaunchKernelGGL(column_kernel, grid, dim3(256), 0, s, weight, c.w_stride, p.vocab, p.dim, part);
        hipLaunchKernelGGL(column_total_kernel, dim3(grid.x), dim3(256), 0, s, part, static_cast<int>(grid.y), p.dim, reinterpret_cast<float *>(c.ws + p.columns));
    }
    float *exps = reinterpret_cast<float *>(c.ws + p.part);
    for (int64_t v0 = 0; v0 < p.vocab; v0 += p.piece) {
        const int64_t width = std::min(p.piece, p.vocab - v0);
        const Head w = head_of(p, c, v0, width);
        logits_of<1>(p, c, rows, w, width, ExpEpilogue{rows.tgt, ref, exps, e.sum, at_target, e.part_stride, e.row_stride, c.ws + p.g, p.piece, v0, width, k});
        times_head(p, c, rows, w, v0, width);
    }
    f.exps = exps, f.ref = ref;
    finish(p, f, s);
    unit_of(p, c, l, rows, nullptr, ref);

    // rows that ref was too far from
    int32_t *redo = reinterpret_cast<int32_t *>(c.ws + p.redo);
    int32_t *tgt2 = reinterpret_cast<int32_t *>(c.ws + p.tgt2);
    RowGrad *grad = reinterpret_cast<RowGrad *>(c.ws + p.grad);
    const Rows again{c.ws + p.h2, redo, tgt2, nullptr};
    hipLaunchKernelGGL(redo_kernel, dim3(1), dim3(kIndexThreads), 0, s, RedoArgs{c.s, ref, rows.tgt, redo, redo + kHeader, tgt2});
    lay_out(false, Layout{rows.h, p.n, 0, p.ld, redo + kHeader, redo, p.n, p.ld, p.ld, 0, again.h, 0, nullptr}, s);
    stats_of<F32>(p, c, again, e, redo);
    f.uncounted = 0, f.exps = nullptr, f.ref = nullptr, f.count = redo, f.which = redo + kHeader, f.grad = grad;
    finish(p, f, s);
    for (int64_t v0 = 0; v0 < p.vocab; v0 += p.piece) {
        const int64_t width = std::min(p.piece, p.vocab - v0);
        const Head w = head_of(p, c, v0, width, nullptr, redo);
        gradient_of<1>(p, c, again, w, v0, width, grad, k, nullptr, true, false);
        times_head(p, c, again, w, v0, width);
    }
    unit_of(p, c, l, again, redo + kHeader, nullptr);
}

void vector_rows(const VectorArgs &a, int rows, unsigned groups, size_t lds, hipStream_t s) {
    if (rows == 1)
        hipLaunchKernelGGL(vector_kernel<1>, dim3(groups), dim3(256), lds, s, a);
    else if (rows == 2)
        hipLaunchKernelGGL(vector_kernel<2>, dim3(groups), dim3(256), lds, s, a);
    else if (rows == 4)
        hipLaunchKernelGGL(vector_kernel<4>, dim3(groups), dim3(256), lds, s, a);
    else
        hipLaunchKernelGGL(vector_kernel<8>, dim3(groups), dim3(256), lds, s, a);
}

void forward_kept(const KeptPlan &p, const Call &c, const Loss &l) {
    hipStream_t s = c.stream;
    // rows gathered and padded to whole slabs: copied as pairs of 16-bit values
    const Layout rows{c.hidden, c.per_batch, 2 * c.batch_stride, 2 * c.row_stride, c.s.rows, c.s.count, p.n, 2 * p.dim, 2 * p.h_ld, 0, c.ws + p.h, 0, nullptr};
    lay_out(false, rows, s);
    float *logits = l.unit ? l.unit : reinterpret_cast<float *>(c.ws + p.logits);
    float *partial = p.logit_splits > 1 ? reinterpret_cast<float *>(c.ws + p.partial) : nullptr;
    const Gemm g{{c.ws + p.h, p.h_ld, 0}, {static_cast<const uint8_t *>(c.weight), c.w_stride, 0}, p.n, p.vocab, p.dim, c.s.count, 0, 8, p.logit_splits, p.logit_cost};
    multiply_kept<true>(p, g, AccumulateEpilogue{partial ? partial : logits, p.ld, p.n * p.ld, 0, nullptr, nullptr}, s);
    const int groups = static_cast<int>(ceil_div(p.ld, kKeptCols));
    KeptArgs a{};
    a.partial = partial, a.logits = logits, a.ld = p.ld, a.split_stride = p.n * p.ld, a.vocab = p.vocab;
    a.tile_rows = p.tile, a.col_tiles = static_cast<int>(ceil_div(p.vocab, kTile)), a.most = p.logit_splits, a.cost = p.logit_cost;
    a.s = c.s;
    a.part = reinterpret_cast<float2 *>(c.ws + p.part);
    a.sum = l.smoothing != 0.0 ? reinterpret_cast<float *>(c.ws + p.sum) : nullptr;
    a.at_target = reinterpret_cast<float *>(c.ws + p.at_target);
    a.k = static_cast<float>(1.44269504088896340736 / l.temperature);
    hipLaunchKernelGGL(kept_kernel, dim3(static_cast<unsigned>(groups), static_cast<unsigned>(p.n)), dim3(256), 0, s, a);
    FinishArgs f{};
    f.part = a.part, f.sum = a.sum, f.at_target = a.at_target, f.part_stride = 1, f.row_stride = groups, f.parts = groups;
    f.n = p.n, f.vocab = p.vocab, f.s = c.s, f.logps = l.logps, f.uncounted = 1;
    f.row_loss = l.loss ? reinterpret_cast<float *>(c.ws + p.row_loss) : nullptr;
    f.smoothing = static_cast<float>(l.smoothing), f.z_loss = static_cast<float>(l.z_loss);
    hipLaunchKernelGGL(finish_kernel<true>, dim3(static_cast<unsigned>(p.n)), dim3(256), 0, s, f);
}

void backward_kept(const KeptPlan &p, const Call &c, const Coefs &k, const float *logits, double temperature, void *grad_hidden, void *grad_weight) {
    hipStream_t s = c.stream;
    float *dz = reinterpret_cast<float *>(c.ws + p.dz);
    const unsigned row_blocks = static_cast<unsigned>(ceil_div(p.n, kOuterRows));
    const KeptGradArgs a{k, logits, grad_hidden ? dz : nullptr, grad_weight ? c.ws + p.dz_parts : nullptr, p.ld, p.vocab, static_cast<float>(1.44269504088896340736 / temperature)};
    hipLaunchKernelGGL(kept_grad_kernel, dim3(static_cast<unsigned>(ceil_div(p.ld, 256)), row_blocks), dim3(256), 0, s, a);
    if (grad_hidden) {
        const Gemm g{{c.ws + p.dz, p.ld, 0}, {static_cast<const uint8_t *>(c.weight), c.w_stride, 0}, p.n, p.dim, p.vocab, c.s.count, 0, 8, p.splits, p.split_cost};
        float *acc = reinterpret_cast<float *>(c.ws + p.acc);
        multiply_kept<false>(p, g, AccumulateEpilogue{acc, p.h_ld, p.n * p.h_ld, 0, nullptr, nullptr}, s);
        const Sums sums{acc, p.h_ld, p.n * p.h_ld, p.tile, static_cast<int>(ceil_div(p.dim, kTile)), p.splits, p.split_cost};
        hipLaunchKernelGGL(hidden_kernel<true>, dim3(blocks_for(p.n * ceil_div(p.dim, 4))), dim3(256), 0, s, sums, c.s.place, c.s.count, p.n, p.dim, Rest{}, grad_hidden);
    }
    if (grad_weight) {
        const Layout h{c.hidden, c.per_batch, c.batch_stride, c.row_stride, c.s.rows, c.s.count, p.n, p.dim};
        hipLaunchKernelGGL(hidden_parts_kernel, dim3(static_cast<unsigned>(ceil_div(p.dim, 256)), row_blocks), dim3(256), 0, s, h, c.ws + p.h_parts);
        const OuterArgs o{c.ws + p.dz_parts, c.ws + p.h_parts, c.s.count, p.vocab, p.dim, static_cast<float *>(grad_weight), static_cast<int>(ceil_div(p.dim, 128))};
        hipLaunchKernelGGL(outer_kernel, dim3(static_cast<unsigned>(round_up(o.col_tiles * ceil_div(p.vocab, 128), kXcds))), dim3(256), 0, s, o);
    }
}

// Whether a forward goes the way of few rows by plain products, and the LDS it takes for its rows. fp32 alone: bf16 rows
// read the head once on the matrix cores as well, at 5.9 TB/s (262,144 x 5376, 1 to 16 rows, 480 us; by plain
// products 718 for one row, 810 for two).
bool takes_vectors(int64_t n, int64_t dim, int &rows, size_t &lds) {
    rows = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8;
    lds = static_cast<size_t>(rows) * round_up(dim, 256) * 4;
    return n <= kVectorRows && lds <= kVectorLds;
}

void forward_vectors(const KeptPlan &p, const Call &c, const Loss &l, int rows, size_t lds) {
    const unsigned groups = static_cast<unsigned>(std::min<int64_t>(ceil_div(p.vocab, 8), kVectorGroups));
    VectorArgs a{};
    a.h = {c.hidden, c.per_batch, c.batch_stride, c.row_stride, nullptr, nullptr, p.n, p.dim};
    a.weight = static_cast<const float *>(c.weight), a.w_stride = c.w_stride, a.vocab = p.vocab, a.targets = c.targets, a.t64 = c.tdtype == ME_I64, a.ignore = c.ignore, a.s = c.s;
    a.logits = l.unit, a.ld = p.ld;
    a.part = reinterpret_cast<float2 *>(c.ws + p.part);
    a.sum = l.smoothing != 0.0 ? reinterpret_cast<float *>(c.ws + p.sum) : nullptr;
    a.at_target = reinterpret_cast<float *>(c.ws + p.at_target);
    a.k = static_cast<float>(1.44269504088896340736 / l.temperature);
    vector_rows(a, rows, groups, lds, c.stream);
    FinishArgs f{};
    f.part = a.part, f.sum = a.sum, f.at_target = a.at_target, f.part_stride = 1, f.row_stride = groups, f.parts = static_cast<int>(groups);
    f.n = p.n, f.vocab = p.vocab, f.s = c.s, f.logps = l.logps, f.uncounted = 1;
    f.row_loss = l.loss ? reinterpret_cast<float *>(c.ws + p.row_loss) : nullptr;
    f.smoothing = static_cast<float>(l.smoothing), f.z_loss = static_cast<float>(l.z_loss);
    hipLaunchKernelGGL(finish_kernel<true>, dim3(static_cast<unsigned>(p.n)), dim3(256), 0, c.stream, f);
}

int forward(int64_t n, int64_t vocab, int64_t dim, int dtype, const Call &call, const Loss &l, size_t there) {
    hipStream_t s = call.stream;
    const Pass pass = l.unit ? kLeavesUnit : kStats;
    const bool smoothed = l.smoothing != 0.0, kept = takes_kept(n, vocab, dtype);
    KeptPlan q{};
    Plan p{};
    if (kept)
        q = kept_plan_of(n, vocab, dim, call.weight, call.w_stride, pass, smoothed);
    else
        p = plan_of(n, vocab, dim, dtype, call.weight, call.w_stride, pass, smoothed);
    Call c = call;
    uint32_t *clear = nullptr;
    if (p.keeps) c.unit = l.unit, clear = kept_head_of(l.unit, vocab, dim).largest;
    const int64_t needed = kept ? q.bytes : p.bytes, row_loss = kept ? q.row_loss : p.row_loss;
    ME_CHECK_ARG(there >= static_cast<size_t>(needed), "workspace of %zu bytes, %lld are needed", there, static_cast<long long>(needed));
    int rows;
    size_t lds;
    if (kept && takes_vectors(n, dim, rows, lds)) {
        forward_vectors(q, c, l, rows, lds);
    } else {
        if (c.tdtype == ME_I64)
            hipLaunchKernelGGL(index_kernel<int64_t>, dim3(1), dim3(kIndexThreads), 0, s, static_cast<const int64_t *>(c.targets), n, c.ignore, vocab, c.s, clear);
        else
            hipLaunchKernelGGL(index_kernel<int32_t>, dim3(1), dim3(kIndexThreads), 0, s, static_cast<const int32_t *>(c.targets), n, c.ignore, vocab, c.s, clear);
        if (kept)
            forward_kept(q, c, l);
        else if (n > 0)
            p.f32 ? forward_rows<true>(p, c, l) : forward_rows<false>(p, c, l);
    }
    if (l.loss) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, s, reinterpret_cast<const float *>(c.ws + row_loss), c.s.count, l.scale, l.mean, l.loss);
    return check_launch("me_head");
}

int check_sizes(int64_t n, int64_t vocab, int64_t dim, int64_t w_stride) {
    ME_CHECK_ARG(n >= 0 && n <= (int64_t{1} << 24), "n must be in 0..2^24");
    ME_CHECK_ARG(dim >= 1 && dim <= 65536, "dim must be in 1..65536");
    ME_CHECK_ARG(ceil_div(n, 256) * ceil_div(dim, 256) <= (int64_t{1} << 22), "n times dim must be at most 2^38");
    ME_CHECK_ARG(vocab >= 1 && vocab <= (int64_t{1} << 21), "vocab must be in 1..2^21");
    ME_CHECK_ARG(w_stride >= dim && w_stride <= (int64_t{1} << 22), "weight rows must be dim or more elements apart, at most 2^22");
    return ME_OK;
}

int check_call(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t per_batch, const void *weight, int64_t vocab, int64_t w_stride,
               const void *targets, int tdtype, double temperature, const void *saved, const void *ws) {
    ME_CHECK_ARG(dtype == ME_BF16 || dtype == ME_F32, "dtype must be bf16/fp32");
    ME_CHECK_ARG(tdtype == ME_I32 || tdtype == ME_I64, "targets must be int32/int64");
    const int rc = check_sizes(n, vocab, dim, w_stride);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(n == 0 || (hidden && targets && per_batch >= 1), "hidden and targets are needed");
    ME_CHECK_ARG(weight && saved && ws, "weight, saved and workspace are needed");
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(saved) % 16 == 0 && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "saved and workspace must be 16-byte aligned");
    ME_CHECK_ARG(temperature >= 1e-6 && temperature <= 1e6, "temperature is out of range");
    return ME_OK;
}

}  // namespace
}  // namespace me

using namespace me;

extern "C" int me_head_workspace_size(int64_t n, int64_t vocab, int64_t dim, int dtype, const void *weight, int64_t w_stride, int pass,
                                      int smoothed, size_t *bytes) {
    ME_CHECK_ARG(bytes && pass >= kStats && pass <= kHasUnit, "bad pass");
    const int rc = check_sizes(n, vocab, dim, w_stride);
    if (rc != ME_OK) return rc;
    if (takes_kept(n, vocab, dtype) && pass != kBackward) {
        *bytes = static_cast<size_t>(kept_plan_of(n, vocab, dim, weight, w_stride, static_cast<Pass>(pass), smoothed != 0).bytes);
        return ME_OK;
    }
    *bytes = pass == kHasUnit && dtype != ME_F32 ? 0 : static_cast<size_t>(plan_of(n, vocab, dim, dtype, weight, w_stride, static_cast<Pass>(pass), smoothed != 0).bytes);
    return ME_OK;
}

extern "C" int me_head_unit_size(int64_t n, int64_t vocab, int64_t dim, int dtype, int for_weight, int64_t *elements) {
    ME_CHECK_ARG(elements, "elements is needed");
    const int rc = check_sizes(n, vocab, dim, dim);
    if (rc != ME_OK) return rc;
    if (takes_kept(n, vocab, dtype))
        *elements = n * kept_ld(vocab);
    else if (keeps_head(n, vocab, dim, dtype))
        *elements = kept_head_of(nullptr, vocab, dim).elements;
    else
        *elements = n > 0 && !for_weight && leaves_unit(n, vocab, dim, dtype) ? n * ceil_div(dim, 4) * 4 : 0;
    return ME_OK;
}

extern "C" int me_head_logps(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                             int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets, int targets_dtype,
                             int64_t ignore_index, double temperature, float *logps, void *saved, float *unit, void *workspace,
                             size_t workspace_bytes, void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved, workspace);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(n == 0 || logps, "logps is needed");
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(unit) % 16 == 0 && (!unit || dtype == ME_BF16 || takes_kept(n, vocab, dtype) || keeps_head(n, vocab, dim, dtype)),
                 "unit must be 16-byte aligned, and NULL where its size is 0 in fp32");
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_of(saved, n), as_stream(stream)};
    return forward(n, vocab, dim, dtype, c, Loss{temperature, 0.0, 0.0, 1.0, 0, logps, nullptr, unit}, workspace_bytes);
}

extern "C" int me_head_ce(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                          int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets, int targets_dtype,
                          int64_t ignore_index, double temperature, double smoothing, double z_loss, double scale, int reduction, float *loss,
                          void *saved, float *unit, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved, workspace);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(reduction == ME_REDUCE_MEAN || reduction == ME_REDUCE_SUM, "reduction must be mean or sum");
    ME_CHECK_ARG(loss, "loss is needed");
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(unit) % 16 == 0 && (!unit || dtype == ME_BF16 || takes_kept(n, vocab, dtype) || keeps_head(n, vocab, dim, dtype)),
                 "unit must be 16-byte aligned, and NULL where its size is 0 in fp32");
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_of(saved, n), as_stream(stream)};
    return forward(n, vocab, dim, dtype, c, Loss{temperature, smoothing, z_loss, scale, reduction == ME_REDUCE_MEAN, nullptr, loss, unit}, workspace_bytes);
}

extern "C" int me_head_backward(const void *hidden, int dtype, int64_t n, int64_t dim, int64_t rows_per_batch, int64_t batch_stride,
                                int64_t row_stride, const void *weight, int64_t vocab, int64_t w_stride, const void *targets,
                                int targets_dtype, int64_t ignore_index, double temperature, const float *upstream, int upstream_per_row,
                                double smoothing, double z_loss, double scale, int reduction, const void *saved, const float *unit,
                                void *grad_hidden, void *grad_weight, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = check_call(hidden, dtype, n, dim, rows_per_batch, weight, vocab, w_stride, targets, targets_dtype, temperature, saved,
                              unit && dtype == ME_BF16 ? saved : workspace);
    if (rc != ME_OK) return rc;
    ME_CHECK_ARG(upstream || (n == 0 && upstream_per_row), "upstream is needed");
    ME_CHECK_ARG(reinterpret_cast<uintptr_t>(grad_hidden) % 16 == 0 && reinterpret_cast<uintptr_t>(grad_weight) % 16 == 0, "gradients must be 16-byte aligned");
    ME_CHECK_ARG(!unit || (dtype == ME_BF16 ? !grad_weight : takes_kept(n, vocab, dtype) || keeps_head(n, vocab, dim, dtype)),
                 "unit is for the hidden states' gradient alone in bf16, and NULL where its size is 0 in fp32");
    if (!grad_hidden && !grad_weight) return ME_OK;
    const Saved saved_rows = saved_of(const_cast<void *>(saved), n);
    const bool f32 = dtype == ME_F32;
    if (unit && takes_kept(n, vocab, dtype)) {
        const KeptPlan q = kept_plan_of(n, vocab, dim, weight, w_stride, kHasUnit, false);
        ME_CHECK_ARG(workspace_bytes >= static_cast<size_t>(q.bytes), "workspace of %zu bytes, %lld are needed", workspace_bytes, static_cast<long long>(q.bytes));
        const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                     static_cast<uint8_t *>(workspace), saved_rows, as_stream(stream)};
        const Coefs coefs{saved_rows, upstream, upstream_per_row != 0, reduction == ME_REDUCE_MEAN, scale / temperature, static_cast<float>(smoothing),
                          static_cast<float>(z_loss), static_cast<double>(vocab)};
        backward_kept(q, c, coefs, unit, temperature, grad_hidden, grad_weight);
        return check_launch("me_head_backward");
    }
    if (unit && !f32) {
        if (n == 0) return ME_OK;
        const ScaleArgs a{unit, saved_rows.count, saved_rows.place, upstream, upstream_per_row != 0, reduction == ME_REDUCE_MEAN, scale / temperature, n, dim, grad_hidden};
        hipLaunchKernelGGL(scale_kernel, dim3(blocks_for(n * ceil_div(dim, 4))), dim3(256), 0, as_stream(stream), a);
        return check_launch("me_head_backward");
    }
    const Plan p = plan_of(n, vocab, dim, dtype, weight, w_stride, unit ? kHasUnit : kBackward, false);
    ME_CHECK_ARG(workspace_bytes >= static_cast<size_t>(p.bytes), "workspace of %zu bytes, %lld are needed", workspace_bytes, static_cast<long long>(p.bytes));
    const Call c{hidden, weight, targets, rows_per_batch, batch_stride, row_stride, w_stride, ignore_index, targets_dtype,
                 static_cast<uint8_t *>(workspace), saved_rows, as_stream(stream), const_cast<float *>(unit), true};
    hipStream_t s = c.stream;
    uint32_t *largest = f32 && !p.keeps ? reinterpret_cast<uint32_t *>(c.ws + p.largest) : nullptr;
    RowGrad *grad = reinterpret_cast<RowGrad *>(c.ws + p.grad);
    Rows rows{};
    // bf16: factors that all rows share come in after the products, so that a target of no probability is -1, which
    // bf16 holds, and no small factor takes values out of its range
    float *factor = !f32 && !upstream_per_row && n > 0 ? reinterpret_cast<float *>(c.ws + p.factor) : nullptr;
    if (n > 0) {
        const Coefs coefs{c.s, upstream, upstream_per_row != 0, reduction == ME_REDUCE_MEAN, scale / temperature, static_cast<float>(smoothing),
                          static_cast<float>(z_loss), static_cast<double>(vocab), factor, grad, f32 ? reinterpret_cast<float *>(c.ws + p.bound) : nullptr,
                          largest, largest ? static_cast<int>(ceil_div(vocab, p.piece)) : 0};
        rows = lay_out_rows(p, c, coefs);
        if (f32 && grad_weight) lay_out(true, hidden_layout(p, c, p.h), s);
    }
    const float k = static_cast<float>(1.44269504088896340736 / temperature);
    for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
        const int64_t width = std::min(p.piece, vocab - v0);
        if (n > 0) {
            uint32_t *widest = p.keeps ? kept_head_of(c.unit, vocab, dim).largest : f32 ? largest + v0 / p.piece : nullptr;
            const Head w = head_of(p, c, v0, width, widest);
            const bool for_hidden = grad_hidden != nullptr, for_weight = grad_weight != nullptr;
            if (f32)
                gradient_of<3>(p, c, rows, w, v0, width, grad, k, widest, for_hidden, for_weight);
            else if (p.rest && for_weight)
                gradient_of<2>(p, c, rows, w, v0, width, grad, k, widest, for_hidden, for_weight);
            else
                gradient_of<1>(p, c, rows, w, v0, width, grad, k, widest, for_hidden, for_weight);
            if (grad_hidden) times_head(p, c, rows, w, v0, width, widest);
        }
        if (grad_weight) {
            const int times = p.rest ? 2 : 1;
            const Gemm g{{c.ws + p.g, p.piece, p.rows * p.piece * 2}, {c.ws + p.h, p.ld, h_part(p)}, width, dim, n * times, c.s.count, 1, 8, 1, 0, times};
            uint8_t *out = static_cast<uint8_t *>(grad_weight) + v0 * dim * (f32 ? 4 : 2);
            if (f32)
                multiply_large<false, false, 6>(g, WeightEpilogue<true>{out, dim, nullptr}, s);
            else
                multiply_large<false, false, 1>(g, WeightEpilogue<false>{out, dim, factor}, s);
        }
    }
    if (grad_hidden && n > 0) {
        const unsigned blocks = blocks_for(n * ceil_div(dim, 4));
        const Rest rest{grad, rows.tgt, static_cast<const uint16_t *>(weight), w_stride, factor};
        if (f32)
            hipLaunchKernelGGL(hidden_kernel<true>, dim3(blocks), dim3(256), 0, s, sums_of(p, c), c.s.place, c.s.count, n, dim, Rest{}, grad_hidden);
        else
            hipLaunchKernelGGL(hidden_kernel<false>, dim3(blocks), dim3(256), 0, s, sums_of(p, c), c.s.place, c.s.count, n, dim, rest, grad_hidden);
    }
    return check_launch("me_head_backward");
}
