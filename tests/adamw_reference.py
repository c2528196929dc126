"""AdamW with the rounding of bf16 weights and 8-bit moments, from the definition in float64 on the CPU.

A kernel's value before rounding is off by the roundings of its fp32 arithmetic, counted at each function
below; a rounded one then lies between the roundings of the exact value less and plus that error, with the same noise
(each rounding here is monotone in its value), which is what the tests ask for.
"""
import numpy as np
import torch

BLOCK = 128
E4M3, E5M2 = (3, -6, 7), (2, -14, 14)  # kept bits, exponent of the smallest normal, of the block's largest


def philox(counter, key):
    """Philox4x32-10: counter [n, 4] uint32 values (uint64 array), key (two ints) -> [n, 4]."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    low, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & low, (a >> s) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def noise(n, seed, step, stream):
    """16 bits for each of a tensor's n values (int64)."""
    groups = np.arange(-(-n // 8), dtype=np.uint64)
    counter = np.stack([groups & np.uint64(0xFFFFFFFF), groups >> np.uint64(32), np.full_like(groups, step),
                        np.full_like(groups, stream)], axis=1)
    w = philox(counter, (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=2).reshape(-1)[:n]
    return torch.from_numpy(halves.astype(np.int64))


def step(p, g, m, v, t, lr, betas, eps, decay):
    """((p, m, v) after the step, (error of each in fp32)): float64 of any shape."""
    b1, b2 = betas
    u = 2.0 ** -24
    tiny = 2.0 ** -150  # and each rounding's least error: half of the smallest subnormal
    m2 = b1 * m + (1 - b1) * g
    # both factors rounded, two products and a sum
    em = 3 * u * ((b1 * m).abs() + ((1 - b1) * g).abs()) + 3 * tiny
    v2 = b2 * v + (1 - b2) * g * g
    ev = 4 * u * v2 + 4 * tiny
    size, root = lr / (1 - b1 ** t), (v2 / (1 - b2 ** t)).sqrt() + eps
    update = size * m2 / root
    # sqrt and reciprocal 1 unit in the last place (2 u) each; the square root halves v's error; factors, product,
    # eps' sum: 6 u more; then p's own factor, product and sum
    # (the least errors of v are 2^-74 in its root, which eps of 1e-8 makes less than 2^-47 of the quotient)
    ep = update.abs() * (2 + 2 + 2 + 7) * u + size * em / root + 3 * u * p.abs() + u * update.abs()
    return ((1 - lr * decay) * p - update, m2, v2), (ep, em, ev)


def bf16_stochastic(x, r):
    """The fp32 nearest x with the noise r added below its upper half, truncated: float64."""
    bits = x.float().view(torch.int32).long() & 0xFFFFFFFF
    out = ((bits + r) & 0xFFFF0000)
    return torch.where(out >= 2**31, out - 2**32, out).int().view(torch.float32).double()


def block_exponent(x):
    """E8M0 byte that each block's largest value gives, before the format's own shift: its biased exponent."""
    n = x.numel()
    full = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    full[:n] = x.abs()
    top = full.view(-1, BLOCK).amax(1).float()
    return (top.view(torch.int32) >> 23).long()


def magnitude(x, r, scale, fmt):
    """Codes (int64) of x >= 0 in units of 2^(scale - 127), with 16 bits of noise each."""
    bits, lowest, _ = fmt
    y = x.double() * torch.exp2(127.0 - scale.double())
    # the grid around y: steps of 2^(e - bits), e its exponent, at least the smallest normal's
    e = torch.frexp(y)[1].long() - 1
    e = torch.where(y > 0, e, lowest).clamp(min=lowest)
    ulp = torch.exp2((e - bits).double())
    k = torch.floor(y / ulp + (r.double() + 0.5) / 65536)
    # k in [2^bits, 2^(bits + 1)] at normals: the code counts on over the binades
    return ((e - lowest) << bits) + k.long()


def values(codes, scale, kind):
    """float64 values of 8-bit moments as the optimizer keeps them."""
    n = codes.numel()
    s = torch.exp2(scale.view(torch.uint8).double() - 127).repeat_interleave(BLOCK)[:n]
    return codes.reshape(-1).view(torch.uint8).view(kind).float().double() * s
