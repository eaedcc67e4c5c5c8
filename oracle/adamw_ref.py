"""AdamW's step and its 8-bit states in 64 bits, on the CPU: what the tests compare the kernels with.

A value a of a mean (root) is held with 3 (4) mantissa bits: floor(a / s + u) s, s = 2^-bits of a's power of two, u in [0, 1) from a hash of
its place, the step and a seed (1/2: to nearest). 128 consecutive values share E, the exponent of the largest value held; what is no
larger than 2^(E - 15) is zero, or for a root that is no zero the next value of the grid, (1 + 2^-4) 2^(E - 15).
"""
import numpy as np

BLOCK = 128
WORD = 1 << 32


def dither(places, step, seed):
    """(what is added for the mean, for the root), in [0, 1)"""
    z = (np.asarray(places, np.uint64) * np.uint64(0x9E3779B1) + np.uint64((step * 0x6C8E9CF5 + seed * 0x5851F42D) % WORD)) % np.uint64(WORD)
    for shift, factor in ((15, 0x7FB5D329), (13, 0x4C957F2B)):
        z = (z ^ (z >> np.uint64(shift))) * np.uint64(factor) % np.uint64(WORD)
    z = z ^ (z >> np.uint64(16))
    return (z & np.uint64(0xFFFF)).astype(np.float64) / 65536, (z >> np.uint64(16)).astype(np.float64) / 65536


def held(a, bits, u):
    """The values that the states hold for a [n] (n a multiple of 128)."""
    a = np.asarray(a, np.float64)
    size = np.abs(a)
    _, e = np.frexp(size)
    s = np.ldexp(1.0, np.maximum(e - 1, -126) - bits)       # (fp32's subnormals have the step of its smallest normal number)
    r = np.where(size > 0, np.floor(size / s + u) * s, 0.0).reshape(-1, BLOCK)
    top = r.max(1, keepdims=True)
    _, e = np.frexp(top)
    zero = np.where(top > 0, np.ldexp(1.0, e - 1 - 15), 0.0)
    r = np.where(r > zero, r, 0.0 if bits == 3 else np.where(r > 0, zero * (1 + 2.0 ** -bits), 0.0))
    return np.copysign(r.reshape(-1), a)


def step(p, g, m, v, t, lr, betas=(0.9, 0.999), eps=1e-8, decay=0.01, clip=1.0):
    """(p, m, v) after step t, before any rounding."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * decay) - lr * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + eps), m, v
