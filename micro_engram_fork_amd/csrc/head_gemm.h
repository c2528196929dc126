// Matrix products of the losses over a decoder's head (head.hip) on gfx950: C [R, S] = sum over k of
// A(r, k) B(s, k), bf16 operands, fp32 accumulation on v_mfma_f32_32x32x16_bf16, with what becomes of a
// tile of C left to an epilogue.
//
// An operand is k-contiguous ([rows][K]: hidden states and head for the logits, the logits' gradient for that
// of the hidden states) or row-contiguous ([K][columns]: the head for the gradient of the hidden states; the logits'
// gradient and the hidden states for that of the head, whose reduction runs over tokens). Both stream in 64-wide
// k-slabs into LDS by buffer_load ... lds:
//   k-contiguous    a unit is rows x 128 bytes, the eight 16-byte chunks of a row XOR-swizzled by
//                   (row >> 1) & 7; a fragment is one ds_read_b128 per lane
//   row-contiguous  a unit is 64 k-rows of the tile's columns; a fragment is two ds_read_b64_tr_b16,
//                   which transpose 4 x 16 blocks on the way (see rc_lane_off)
// A 32x32x16 MFMA operand holds, in lane l, the 8 k values 16 ks + 8 (l >> 5) .. + 7 of row / column l & 31.
//
// fp32 operands come in parts, whose products are segments of one reduction; A's part stride and B's lead from one
// part to the next:
//   SEGS 6  three bf16 parts that add up to the value exactly; six of their nine products, the others are below
//           2^-26 of the whole. Keeps every value's digits, whatever the values around it.
//   SEGS 3  two fp16 parts of the value over a power of two by row that puts the row's largest below 2^15; three of
//           their four products, the fourth is below 2^-22 of the whole, its root mean square 2^-25. Half the
//           matrix time; a value's parts hold it to 2^-22 of itself, or 2^-40 of its row's largest where that
//           is more. That is as exact as fp32 where errors count against the rest of a row's sum: for logits, and for
//           the gradient of the hidden states. The gradient of the head has rows of its own for tokens of any
//           probability, down to products that fp16 could not tell from zero: six products.
// Few rows of fp32 (SEGS 0) are read as they lie instead, in 32-wide k-slabs, as laying out the other operand would
// read and write what is otherwise read once; fragments are split into three bf16 parts in registers (Parts), the same six
// products. (v_mfma_f32_32x32x2_f32 takes 2.7 times as long and was the bound from 40 rows on: 262,144 x 5376,
// 46 rows 1661 us, 128 rows 2837.)
#pragma once

#include "me_common.h"

#include <type_traits>

namespace me {
namespace head {

constexpr int kThreads = 256;
constexpr int kSlabBytes = 128;                  // of a k-contiguous row
constexpr int kSlabK = 64;                       // k values of a slab of 16-bit operands
template <int SEGS>
constexpr int kElement = SEGS == 0 ? 4 : 2;      // bytes
template <int SEGS>
constexpr int kSlab = kSlabBytes / kElement<SEGS>;
constexpr int kXcds = 8;
constexpr uint32_t kBufferConfig = 0x00020000u;  // raw buffer descriptor word 3 (gfx9 family)
constexpr uint32_t kOff = 0xffffffffu;           // a load offset past every buffer: reads zeros

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int int32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

struct Operand {
    const uint8_t *base;
    int64_t ld;     // elements from one row (k-row) to the next
    int64_t part;   // bytes from one part to the next
};

struct Gemm {
    Operand a, b;
    int64_t R, S, K;       // output rows (device count below takes their place), columns, reduction length
    const int32_t *count;  // null, or rows that there are: of R (reduce_rows 0) or of K (1)
    int count_is_k;
    int group;             // column tiles that follow one another before the next row tile
    int most_splits;       // parts of the reduction, each with an output of its own: up to so many (splits_for)
    int split_cost;        // of splits_for
    int times = 1;         // rows of K for each that `count` counts
};

// Parts of the reduction that tiles of C take so that the last round of workgroups is as full as it gets: the number of
// them, up to `most`, that takes least time, where each costs `cost` / 4096 of the product's own (its sums are read
// and written once more). The rows may be known to the device alone, so this is decided there, by whoever writes the
// parts and whoever adds them: in integers, so that all of them come to the same; lane l tries l + 1 parts, as one after the
// other took 5 us. Called by whole waves.
constexpr int kMostSplits = 64, kMostCost = 1 << 18;
__device__ inline int splits_for(int tiles, int most, int cost) {
    const uint32_t s = static_cast<uint32_t>(threadIdx.x & 63) + 1, all = static_cast<uint32_t>(tiles) * s;
    // rounds of the chip's 256 CUs against the work, times 4096; past 2^19 workgroups they hardly differ
    const uint32_t time = (all < (1u << 19) ? (((all + 255) / 256) << 20) / all : 4096u) + static_cast<uint32_t>(cost) * s;
    uint32_t best = s <= static_cast<uint32_t>(most) ? time * 64 + s - 1 : ~0u;
#pragma unroll
    for (int d = 32; d; d >>= 1) best = min(best, static_cast<uint32_t>(__shfl_xor(static_cast<int>(best), d)));
    return __builtin_amdgcn_readfirstlane(static_cast<int>(best & 63)) + 1;
}

// segment -> parts of A and B: (0,0) (0,1) (1,0) and for SEGS 6 on to (0,2) (1,1) (2,0)
__device__ __forceinline__ int part_a(int seg) { return (0x910 >> (2 * seg)) & 3; }
__device__ __forceinline__ int part_b(int seg) { return (0x184 >> (2 * seg)) & 3; }

// Eight k values of fp32 as three bf16 that add up to them, each the nearest of what remains. What is not finite, or
// rounds to infinity (from 3.39e38 on), makes its products NaN.
struct Parts {
    bf16x8 p[3];

    Parts() = default;
    __device__ __forceinline__ explicit Parts(const floatx8 &x) {
        p[0] = __builtin_convertvector(x, bf16x8);
        const floatx8 r = x - __builtin_convertvector(p[0], floatx8);
        p[1] = __builtin_convertvector(r, bf16x8);
        p[2] = __builtin_convertvector(r - __builtin_convertvector(p[1], floatx8), bf16x8);
    }
};

__device__ __forceinline__ floatx16 multiply(const Parts &x, const Parts &y, floatx16 acc) {
#pragma unroll
    for (int sum = 2; sum >= 0; --sum)  // small products first
#pragma unroll
        for (int i = 0; i <= sum; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.p[i], y.p[sum - i], acc, 0, 0, 0);
    return acc;
}

template <int SEGS>
__device__ __forceinline__ floatx16 multiply(const bf16x8 &x, const bf16x8 &y, const floatx16 &acc) {
    if constexpr (SEGS == 3)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, x), __builtin_bit_cast(halfx8, y), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
}

__device__ __forceinline__ int32x4 buffer_rsrc(uint64_t base, uint32_t bytes) {
    int32x4 r;
    r.x = static_cast<int>(static_cast<uint32_t>(base));
    r.y = static_cast<int>(static_cast<uint32_t>(base >> 32) & 0xffffu);  // stride 0
    r.z = static_cast<int>(bytes);
    r.w = static_cast<int>(kBufferConfig);
    return r;
}

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint8_t *)p));
}

// One wave moves 64 x 16 bytes: lane l's chunk at byte voffset (+ soffset) of the buffer lands at LDS address
// lds_base + 16 l; a voffset at or past the buffer's size reads zeros. Counted by vmcnt; the caller waits.
__device__ __forceinline__ void dma16(const int32x4 &rsrc, uint32_t lds_base, uint32_t voffset, uint32_t soffset) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds_base), "v"(voffset), "s"(rsrc), "s"(soffset)
                 : "memory");
}

// Likewise 64 x 4 bytes, from addresses that are multiples of 4
__device__ __forceinline__ void dma4(const int32x4 &rsrc, uint32_t lds_base, uint32_t voffset, uint32_t soffset) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds_base), "v"(voffset), "s"(rsrc), "s"(soffset)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// XOR swizzle (in 16-byte chunks) of k-row kr of a row-contiguous unit. 16-bit: the 4 k-rows x 4 chunks that the 32
// lanes of one LDS cycle read are on 16 distinct 16-byte bank groups. fp32: the two halves of a wave read k-rows eight
// apart, of 32 columns each, on the two halves of the banks.
template <int ELEMENT>
__device__ __forceinline__ int rc_swizzle(int kr) {
    return ELEMENT == 4 ? 8 * ((kr >> 3) & 1) : 4 * (kr & 3);
}

// Two transpose reads make a fragment: 16-lane group g takes columns 16 (g & 1) .. + 15 of the 32-wide subtile and
// k-rows 16 ks + 8 (g >> 1) + 4 half .. + 3; its lane i addresses k-row (i >> 2) of those four at columns 4 (i & 3)
// .. + 3 and receives column i's four k values. k-step and half are constant byte offsets.
template <int COLS>
__device__ __forceinline__ uint32_t rc_lane_off(int col0, int lane) {
    static_assert(COLS == 128 || COLS == 256, "16 or 32 chunks per k-row");
    const int i = lane & 15, g = lane >> 4;
    const int c = col0 + 16 * (g & 1) + 4 * (i & 3);
    const int kr = 8 * (g >> 1) + (i >> 2);
    return static_cast<uint32_t>(kr * (2 * COLS) + (((c >> 3) ^ rc_swizzle<2>(kr)) << 4) + (c & 7) * 2);
}

template <int COLS>
__device__ __forceinline__ bf16x8 rc_frag(const uint8_t *unit, int ks, uint32_t off) {
    const auto *p = (const __attribute__((address_space(3))) uint8_t *)(unit + off) + ks * 16 * (2 * COLS);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(p));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(p + 4 * (2 * COLS)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ bf16x8 kc_frag(const uint8_t *unit, int ks, int row, int lane) {
    const int c = ((2 * ks + (lane >> 5)) ^ ((row >> 1) & 7)) << 4;
    return *reinterpret_cast<const bf16x8 *>(unit + row * kSlabBytes + c);
}

// fp32: 8 k values 16 ks + 8 (lane >> 5) .. + 7
__device__ __forceinline__ floatx8 kc_frag_f32(const uint8_t *unit, int ks, int row, int lane) {
    const int c = 4 * ks + 2 * (lane >> 5), x = (row >> 1) & 7;
    const floatx4 lo = *reinterpret_cast<const floatx4 *>(unit + row * kSlabBytes + ((c ^ x) << 4));
    const floatx4 hi = *reinterpret_cast<const floatx4 *>(unit + row * kSlabBytes + (((c + 1) ^ x) << 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Accumulator e of a tile. The large tiles' accumulators fill the AGPRs: read one by one, in the order of the
// program, or the compiler copies all of them to VGPRs that it does not have. Reads by inline asm need their own wait
// after the last MFMA (settle).
template <bool AGPR>
__device__ __forceinline__ float acc_read(const floatx16 &t, int e) {
    if constexpr (AGPR) {
        float v;
        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(t[e]));
        return v;
    } else {
        return t[e];
    }
}

__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" : : : "memory"); }

struct Tile {
    int64_t r0, s0;  // first row and column
    int64_t rows;    // rows that there are (R or the device's count)
    int64_t k0, k1;  // this split's reduction, in k
    int rt, st, split;
};

// Workgroup -> tile: each XCD takes a run of logical tiles; these go through `group` column tiles of
// a row tile before the next row tile, so the tiles that an XCD's CUs work on at a time are a block whose rows and
// columns share its L2. False: no tile (the device's count is short of the launch).
__device__ __forceinline__ bool tile_of(const Gemm &a, int tr, int ts, int slab, Tile &t) {
    int64_t rows = a.R, k = a.K;
    if (a.count != nullptr) {
        const int64_t n = *as_global(a.count);
        if (a.count_is_k)
            k = min(k, n * a.times);
        else
            rows = min(rows, n);
    }
    const int n_rt = static_cast<int>(ceil_div(rows, tr)), n_st = static_cast<int>(ceil_div(a.S, ts));
    const int per_split = n_rt * n_st;
    if (per_split == 0) return false;
    const int splits = a.most_splits == 1 ? 1 : splits_for(per_split, a.most_splits, a.split_cost);
    const int total = per_split * splits;
    const int per_xcd = (total + kXcds - 1) / kXcds;
    const int slot = static_cast<int>(blockIdx.x) / kXcds;
    int i = static_cast<int>(blockIdx.x) % kXcds * per_xcd + slot;
    if (slot >= per_xcd || i >= total) return false;
    t.split = i / per_split;
    i -= t.split * per_split;
    const int in_group = n_rt * a.group;
    const int g = i / in_group;
    i -= g * in_group;
    const int width = min(a.group, n_st - g * a.group);
    t.rt = i / width;
    t.st = g * a.group + (i - t.rt * width);
    t.r0 = static_cast<int64_t>(t.rt) * tr;
    t.s0 = static_cast<int64_t>(t.st) * ts;
    t.rows = rows;
    const int64_t slabs = ceil_div(k, static_cast<int64_t>(slab));
    t.k0 = slabs * t.split / splits * slab;
    t.k1 = min(k, slabs * (t.split + 1) / splits * slab);
    return true;
}

// The loads of one operand's slabs by a wave: LOADS of 1 KiB, fixed per-lane offsets, in pieces of 16 bytes a lane or of 4
// (fp32 rows that start or end anywhere: four instructions for each KiB).
// k-contiguous: load i fills rows 8 (LOADS wave + i) + [0, 8), the KiB's chunk c row + c / 8 at physical chunk c % 8;
// the slab's byte offset goes in soffset, and pieces past K in the last slab read zeros.
// row-contiguous: load i fills one or more k-rows; the descriptor's base moves by the slab's k-rows and its size
// holds those that there are, so that k-rows past K read zeros with no per-lane work.
template <bool KC, int DIM, int LOADS, int ELEMENT, int PIECE = 16>
struct Loader {
    static constexpr int kChunk = 16 / ELEMENT;             // values of a 16-byte chunk
    static constexpr int kSlabValues = kSlabBytes / ELEMENT;
    static constexpr int kSteps = 16 / PIECE;               // instructions of a KiB
    static_assert(PIECE == 16 || (PIECE == 4 && ELEMENT == 4), "pieces of whole values");
    uint64_t base;     // of the tile (k-contiguous) or the operand (row-contiguous)
    int64_t pitch;     // bytes from row to row
    int64_t part;
    int64_t K;         // full reduction length of a segment's operand
    uint32_t range;    // k-contiguous: bytes of the tile's rows
    uint32_t off[LOADS * kSteps];
    bool out[2 * kSteps];  // this lane's piece of an even / odd load is past K in the last slab

    // rows / columns from `first` on up to `there`; k values from k0 on up to k
    __device__ __forceinline__ void init(const Operand &o, int64_t first, int64_t there, int64_t k0, int64_t k, int wave, int lane) {
        pitch = o.ld * ELEMENT;
        part = o.part;
        K = k;
        if constexpr (KC) {
            static_assert(LOADS % 2 == 0 || LOADS == 1 || LOADS == 3, "see out");
            base = reinterpret_cast<uint64_t>(o.base) + static_cast<uint64_t>(first * pitch);
            const int64_t rows = min(there - first, static_cast<int64_t>(DIM));
            range = static_cast<uint32_t>((rows - 1) * pitch + ceil_div(k, kChunk) * 16);
            const int valid = k > k0 ? static_cast<int>(k - (k - 1) / kSlabValues * kSlabValues) : 0;  // k values of the last slab
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const int at = (j * 64 + lane) * PIECE, row = (wave * LOADS + i) * 8 + at / kSlabBytes;
                    const int ch = (at / 16 % 8) ^ ((row >> 1) & 7);
                    off[i * kSteps + j] = row < rows ? static_cast<uint32_t>(row * pitch) + static_cast<uint32_t>(ch * 16 + at % 16) : kOff;
                    out[i % 2 * kSteps + j] = ch * kChunk + at % 16 / ELEMENT >= valid;  // alike for all loads of i's parity
                }
        } else {
            base = reinterpret_cast<uint64_t>(o.base);
            constexpr int kRowBytes = DIM * ELEMENT;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const int at = ((wave * LOADS + i) * 64 * kSteps + j * 64 + lane) * PIECE, kr = at / kRowBytes;
                    const int64_t col = first + kChunk * ((at % kRowBytes / 16) ^ rc_swizzle<ELEMENT>(kr)) + at % 16 / ELEMENT;
                    off[i * kSteps + j] = col < there ? static_cast<uint32_t>(kr * pitch + col * ELEMENT) : kOff;
                }
        }
    }

    // load i of the slab at k0 of part p
    __device__ __forceinline__ void issue(int i, int64_t k0, int p, uint32_t lds) const {
        const uint64_t at = base + static_cast<uint64_t>(p * part);
        int32x4 rsrc;
        uint32_t soffset = 0;
        bool last = false;
        if constexpr (KC) {
            last = k0 + kSlabValues > K;
            rsrc = buffer_rsrc(at, range);
            soffset = static_cast<uint32_t>(k0 * ELEMENT);
        } else {
            const int64_t left = max(min(K - k0, int64_t{kSlabValues}), int64_t{0});
            rsrc = buffer_rsrc(at + static_cast<uint64_t>(k0 * pitch), static_cast<uint32_t>(left * pitch));
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const uint32_t from = KC && last && out[i % 2 * kSteps + j] ? kOff : off[i * kSteps + j];
            if constexpr (PIECE == 16)
                dma16(rsrc, lds, from, soffset);
            else
                dma4(rsrc, lds + static_cast<uint32_t>(j) * 256u, from, soffset);
        }
    }
};

// ---- 256 x 256 tiles: one workgroup per CU, four waves of 128 x 128 -------------------------------------------
// Slabs stream through five 32 KiB units, A of slab s in unit 2s % 5, B in (2s + 1) % 5: two slabs of loads fly
// while one is consumed, one workgroup barrier per slab; fragment reads and loads are issued between MFMAs.
// Bound by power: 3066 rows x 262,144 x 5376 in 6.8 ms, 1.27 PFLOP/s, the matrix cores busy in 71 % of cycles at
// 1.67 GHz (library products of this size reach 1.05 to 1.56, by layout); its tiles' columns go eight to a row tile,
// with 4, 16 and 32 it took 1.4, 4 and 12 % longer. Three segments of fp16 parts: 2048 x 32,000 x 1024 in 344 to
// 543 us by epilogue, 390 to 247 TFLOP/s of fp32 where the library's fp32 product has 153; six of bf16 parts 640 us, 210.
constexpr int kUnit = 32768;
constexpr int kUnits = 5;
constexpr int kRingBytes = kUnits * kUnit;  // 160 KiB
constexpr int kTile = 256;
constexpr int kDma = 8;                     // 1 KiB loads per wave per operand per slab

template <bool A_KC, bool B_KC, int SEGS, class Epilogue>
__global__ __launch_bounds__(kThreads, 1) void large_kernel(const Gemm a, const Epilogue epi) {
    constexpr int kSub = 4;                // 32-wide subtiles of a wave in each direction
    constexpr int kParts = 2 * kSub;       // fragments per k-step
    constexpr int kMfma = kSub * kSub;     // MFMAs per k-step (4 k-steps per slab)
    constexpr int kPre = 4;                // last k-step's MFMAs before the slab's barrier
    __shared__ __attribute__((aligned(16))) uint8_t ring[kRingBytes];

    Tile t;
    if (!tile_of(a, kTile, kTile, kSlabK, t)) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 1, ws = wave & 1;
    // slabs per segment; one of zeros where there is nothing to sum
    const int spq = max(static_cast<int>(ceil_div(t.k1 - t.k0, int64_t{kSlabK})), 1);
    const int slabs = spq * SEGS;

    Loader<A_KC, kTile, kDma, 2> la;
    Loader<B_KC, kTile, kDma, 2> lb;
    la.init(a.a, t.r0, A_KC ? t.rows : a.R, t.k0, t.k1, wave, lane);
    lb.init(a.b, t.s0, a.S, t.k0, t.k1, wave, lane);
    const uint32_t w0 = __builtin_amdgcn_readfirstlane(lds_addr(ring) + static_cast<uint32_t>(wave) * (kDma * 1024u));
    auto issue_a = [&](int sl, int i) {
        const int seg = SEGS == 1 ? 0 : sl / spq;
        uint32_t dst = w0 + static_cast<uint32_t>((2 * sl) % kUnits) * kUnit;
        asm volatile("" : "+s"(dst));
        la.issue(i, t.k0 + static_cast<int64_t>(sl - seg * spq) * kSlabK, SEGS == 1 ? 0 : part_a(seg), dst + static_cast<uint32_t>(i) * 1024u);
    };
    auto issue_b = [&](int sl, int i) {
        const int seg = SEGS == 1 ? 0 : sl / spq;
        uint32_t dst = w0 + static_cast<uint32_t>((2 * sl + 1) % kUnits) * kUnit;
        asm volatile("" : "+s"(dst));
        lb.issue(i, t.k0 + static_cast<int64_t>(sl - seg * spq) * kSlabK, SEGS == 1 ? 0 : part_b(seg), dst + static_cast<uint32_t>(i) * 1024u);
    };
    auto unit_a = [&](int sl) { return ring + ((2 * sl) % kUnits) * kUnit; };
    auto unit_b = [&](int sl) { return ring + ((2 * sl + 1) % kUnits) * kUnit; };

    struct Frag {
        bf16x8 s[kSub], r[kSub];
    };
    uint32_t soff[B_KC ? 1 : kSub], roff[A_KC ? 1 : kSub];
    if constexpr (!B_KC) {
#pragma unroll
        for (int x = 0; x < kSub; ++x) soff[x] = rc_lane_off<kTile>(ws * 128 + 32 * x, lane);
    }
    if constexpr (!A_KC) {
#pragma unroll
        for (int y = 0; y < kSub; ++y) roff[y] = rc_lane_off<kTile>(wr * 128 + 32 * y, lane);
    }
    auto load_part = [&](const uint8_t *ua, const uint8_t *ub, int ks, Frag &f, int p) {
        if (p < kSub) {
            if constexpr (B_KC)
                f.s[p] = kc_frag(ub, ks, ws * 128 + 32 * p + (lane & 31), lane);
            else
                f.s[p] = rc_frag<kTile>(ub, ks, soff[p]);
        } else {
            const int y = p - kSub;
            if constexpr (A_KC)
                f.r[y] = kc_frag(ua, ks, wr * 128 + 32 * y + (lane & 31), lane);
            else
                f.r[y] = rc_frag<kTile>(ua, ks, roff[y]);
        }
    };
    // parts in the order the next k-step's MFMAs first use them: s0, r0 .. r3, s1 ..
    auto part_of = [](int q) { return q == 0 ? 0 : (q <= kSub ? kSub + q - 1 : q - kSub); };

    floatx16 acc[kSub][kSub];
#pragma unroll
    for (int x = 0; x < kSub; ++x)
#pragma unroll
        for (int y = 0; y < kSub; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;

#pragma unroll
    for (int i = 0; i < kDma; ++i) issue_a(0, i);
#pragma unroll
    for (int i = 0; i < kDma; ++i) issue_b(0, i);
    if (slabs > 1) {
#pragma unroll
        for (int i = 0; i < kDma; ++i) issue_a(1, i);
#pragma unroll
        for (int i = 0; i < kDma; ++i) issue_b(1, i);
        wait_vmcnt<2 * kDma>();
    } else {
        wait_vmcnt<0>();
    }
    __syncthreads();
    Frag f0, f1;
#pragma unroll
    for (int q = 0; q < kParts; ++q) load_part(unit_a(0), unit_b(0), 0, f0, part_of(q));

    auto mfma = [&](const Frag &f, int i) {
        acc[i / kSub][i % kSub] = multiply<SEGS>(f.s[i / kSub], f.r[i % kSub], acc[i / kSub][i % kSub]);
        __builtin_amdgcn_sched_barrier(0);
    };
    // Slab s, four k-steps: each k-step's MFMAs run while the next one's fragments are read. k-steps 0 and 1
    // issue A_{s+2} (into B_{s-1}'s unit, free since the previous barrier). k-step 3 waits for slab s+1
    // after its first kPre MFMAs, passes the barrier (every wave has read all of slab s), then issues B_{s+2}
    // (into A_s's unit) and reads slab s+1's k-step 0.
    auto slab = [&](int sl, auto wait, auto dma) {
        const uint8_t *ua = unit_a(sl), *ub = unit_b(sl);
#pragma unroll
        for (int ks = 0; ks < 3; ++ks) {
            Frag &cur = ks % 2 == 0 ? f0 : f1;
            Frag &nxt = ks % 2 == 0 ? f1 : f0;
#pragma unroll
            for (int i = 0; i < kMfma; ++i) {
                mfma(cur, i);
                const int dq = ks * kMfma + i;  // A loads: one per four MFMAs of k-steps 0 and 1
                if (decltype(dma)::value && ks < 2 && dq % (2 * kMfma / kDma) == 0) {
                    issue_a(sl + 2, dq / (2 * kMfma / kDma));
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i < kParts) {
                    load_part(ua, ub, ks + 1, nxt, part_of(i));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kPre; ++i) mfma(f1, i);
        if constexpr (decltype(wait)::value == 1) wait_vmcnt<kDma>();  // A_{s+2} may still fly
        if constexpr (decltype(wait)::value == 2) wait_vmcnt<0>();
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *na = unit_a(sl + 1), *nb = unit_b(sl + 1);
#pragma unroll
        for (int i = kPre; i < kMfma; ++i) {
            mfma(f1, i);
            const int q = i - kPre;
            if (decltype(dma)::value && q < kDma) {
                issue_b(sl + 2, q);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (q < kParts) {  // past the last slab these read a stale unit; unused
                load_part(na, nb, 0, f0, part_of(q));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    using WaitA = std::integral_constant<int, 1>;
    using WaitAll = std::integral_constant<int, 2>;
    using NoWait = std::integral_constant<int, 0>;
#pragma unroll 1
    for (int sl = 0; sl + 2 < slabs; ++sl) slab(sl, WaitA{}, std::true_type{});
    if (slabs >= 2) slab(slabs - 2, WaitAll{}, std::false_type{});
    slab(slabs - 1, NoWait{}, std::false_type{});
    __syncthreads();  // every wave is done with the ring, and no load is in flight
    settle();
    epi.template run<true, kSub, kSub>(acc, t, wr * 128, ws * 128, ring, lane);
}

// ---- 32 to 128 x 256 tiles for few rows ---------------------------------------------------------------------
// The product of a few rows is bound by the one read of its other operand. Four waves next to each other over
// the columns, all 32 BR rows each; whole slabs in a ring of three slots, two in flight while one is consumed, one
// barrier per slab; one workgroup per CU, 64 to 96 KB of loads in flight (48 rows, 262,144 x 5376 in bf16: 488 us with
// exponentials, 459 from the head's other side, 5.8 and 6.1 TB/s). SEGS 0: fp32 as it lies, PIECE as of Loader;
// k-contiguous heads then in two slots, for two workgroups per CU whose reads, splits and products take turns (46
// rows, 262,144 x 5376: 1208 us, with three slots and one workgroup 1485; row-contiguous ones 1637 and 1556).
// TS: columns of a tile, 256 or, where that would leave CUs without one, 128.
template <bool B_KC, int BR, int TS, int SEGS, int PIECE, class Epilogue>
__global__ __launch_bounds__(kThreads) void few_kernel(const Gemm a, const Epilogue epi) {
    constexpr int kTR = 32 * BR, kTS = TS, kRing = SEGS == 0 && B_KC ? 2 : 3, kEl = kElement<SEGS>, kStep = kSlab<SEGS>;
    constexpr int kBS = kTS / 128;                         // 32-wide subtiles of a wave's columns
    constexpr int kUnitA = kTR * kSlabBytes;
    constexpr int kSlot = (kTR + kTS) * kSlabBytes;
    constexpr int kDmaA = kTR / 32, kDmaB = kTS / 32;      // 1 KiB loads per wave and slab
    constexpr int kWait = (kRing - 2) * (kDmaA + kDmaB * (16 / PIECE));  // instructions of the slabs that may fly
    static_assert(kWait <= 63, "vmcnt counts up to 63");
    __shared__ __attribute__((aligned(16))) uint8_t ring[kRing * kSlot];

    Tile t;
    if (!tile_of(a, kTR, kTS, kStep, t)) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int spq = max(static_cast<int>(ceil_div(t.k1 - t.k0, static_cast<int64_t>(kStep))), 1);
    const int slabs = spq * (SEGS == 0 ? 1 : SEGS);
    Loader<true, kTR, kDmaA, kEl> la;
    Loader<B_KC, kTS, kDmaB, kEl, PIECE> lb;
    la.init(a.a, t.r0, t.rows, t.k0, t.k1, wave, lane);
    lb.init(a.b, t.s0, a.S, t.k0, t.k1, wave, lane);
    const uint32_t w0 = __builtin_amdgcn_readfirstlane(lds_addr(ring));
    auto issue = [&](int sl) {
        const int seg = SEGS <= 1 ? 0 : sl / spq;
        const int64_t k0 = t.k0 + static_cast<int64_t>(sl - seg * spq) * kStep;
        uint32_t slot = w0 + static_cast<uint32_t>(sl % kRing) * kSlot;
        asm volatile("" : "+s"(slot));
#pragma unroll
        for (int i = 0; i < kDmaA; ++i) la.issue(i, k0, SEGS <= 1 ? 0 : part_a(seg), slot + static_cast<uint32_t>(wave * kDmaA + i) * 1024u);
#pragma unroll
        for (int i = 0; i < kDmaB; ++i) lb.issue(i, k0, SEGS <= 1 ? 0 : part_b(seg), slot + kUnitA + static_cast<uint32_t>(wave * kDmaB + i) * 1024u);
    };
    uint32_t soff[B_KC ? 1 : kBS];
    if constexpr (!B_KC) {
#pragma unroll
        for (int x = 0; x < kBS; ++x) {
            const int col = wave * 32 * kBS + 32 * x;
            if constexpr (SEGS == 0)  // k-row 8 (lane >> 5) of a k-step, a lane's column
                soff[x] = static_cast<uint32_t>(8 * (lane >> 5) * kTS * 4 + (((col >> 2) ^ rc_swizzle<4>(8 * (lane >> 5))) << 4) + (lane & 31) * 4);
            else
                soff[x] = rc_lane_off<kTS>(col, lane);
        }
    }
    floatx16 acc[kBS][BR];
#pragma unroll
    for (int x = 0; x < kBS; ++x)
#pragma unroll
        for (int y = 0; y < BR; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
#pragma unroll
    for (int sl = 0; sl < kRing - 1; ++sl)
        if (sl < slabs) issue(sl);
    for (int sl = 0; sl < slabs; ++sl) {
        // slab sl landed for this wave (later slabs may fly), then for every wave
        if (sl + kRing - 2 < slabs)
            wait_vmcnt<kWait>();
        else
            wait_vmcnt<0>();
        __syncthreads();
        // the slot of slab sl - 1 is free: every wave read it before this barrier
        if (sl + kRing - 1 < slabs) issue(sl + kRing - 1);
        const uint8_t *ua = ring + (sl % kRing) * kSlot, *ub = ua + kUnitA;
#pragma unroll
        for (int ks = 0; ks < kStep / 16; ++ks) {
            if constexpr (SEGS == 0) {
                auto take_b = [&](int x) {
                    if constexpr (B_KC) {
                        return kc_frag_f32(ub, ks, wave * 32 * kBS + 32 * x + (lane & 31), lane);
                    } else {
                        floatx8 f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float *>(ub + soff[x] + (16 * ks + i) * kTS * 4);
                        return f;
                    }
                };
                Parts fs[kBS];
#pragma unroll
                for (int x = 0; x < kBS; ++x) fs[x] = Parts(take_b(x));
#pragma unroll
                for (int y = 0; y < BR; ++y) {
                    const Parts fr(kc_frag_f32(ua, ks, 32 * y + (lane & 31), lane));
#pragma unroll
                    for (int x = 0; x < kBS; ++x) acc[x][y] = multiply(fs[x], fr, acc[x][y]);
                }
            } else {
                bf16x8 fs[kBS], fr[BR];
#pragma unroll
                for (int x = 0; x < kBS; ++x) {
                    if constexpr (B_KC)
                        fs[x] = kc_frag(ub, ks, wave * 32 * kBS + 32 * x + (lane & 31), lane);
                    else
                        fs[x] = rc_frag<kTS>(ub, ks, soff[x]);
                }
#pragma unroll
                for (int y = 0; y < BR; ++y) fr[y] = kc_frag(ua, ks, 32 * y + (lane & 31), lane);
#pragma unroll
                for (int x = 0; x < kBS; ++x)
#pragma unroll
                    for (int y = 0; y < BR; ++y) acc[x][y] = multiply<SEGS>(fs[x], fr[y], acc[x][y]);
            }
        }
    }
    __syncthreads();
    epi.template run<false, kBS, BR>(acc, t, 0, wave * 32 * kBS, ring, lane);
}

// Workgroups that hold every tile at the largest count
inline int64_t workgroups(const Gemm &a, int tr, int ts) {
    return ceil_div(ceil_div(a.R, tr) * ceil_div(a.S, ts) * a.most_splits, kXcds) * kXcds;
}

}  // namespace head
}  // namespace me
