// Rounding noise and stochastic rounding of the optimizers' kernels.
#pragma once

#include "me_common.h"

namespace me {

// ---- Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11) ----------------------------------------
__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
    constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u;
    constexpr uint32_t kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        // one 32 x 32 -> 64-bit product per word gives both halves (v_mad_u64_u32)
        const uint64_t p0 = static_cast<uint64_t>(kM0) * c.x, p1 = static_cast<uint64_t>(kM1) * c.z;
        c = make_uint4(static_cast<uint32_t>(p1 >> 32) ^ c.y ^ k.x, static_cast<uint32_t>(p1),
                       static_cast<uint32_t>(p0 >> 32) ^ c.w ^ k.y, static_cast<uint32_t>(p0));
        k.x += kW0;
        k.y += kW1;
    }
    return c;
}

// fp32 -> bf16 bits, stochastic: noise added below the kept 16 bits, then truncated; inf and NaN
// convert as usual (optim.py:39-44).
__device__ __forceinline__ uint16_t stochastic_bf16_bits(float x, uint32_t noise) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7f800000u) == 0x7f800000u) return float_to_bf16_bits_rne(x);
    return static_cast<uint16_t>((u + noise) >> 16);
}

}  // namespace me
