"""Microscaled 4-bit layers restated in 64 bits on the CPU, from the format's definition: the checker of the mxfp4 tests."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
EVEN = torch.tensor([True, False, True, False, True, False, True, False])   # whose mantissa bit is 0


def exponents(x):
    """E of each block of 32 values of a row: [M, K / 32] float64; NaN for a block with an infinity or a NaN."""
    b = x.double().reshape(x.shape[0], -1, 32).abs()
    bad = ~torch.isfinite(b).all(-1)
    a = torch.where(bad, 1.0, b.amax(-1))
    e = (torch.frexp(a)[1] - 3).double().clamp_min(-127)      # frexp: a = f 2^p, f in [0.5, 1)
    return torch.where(bad, float("nan"), torch.where(a == 0, -127.0, e))


def _spread(e, K):
    return e.repeat_interleave(32, 1)[:, :K]


def four_bits(x):
    """The 4-bit values of x: the nearest point of the grid, the one with an even mantissa of two that are as near."""
    E = _spread(exponents(x), x.shape[1])
    v = torch.nan_to_num(x.double(), 0.0, 0.0, 0.0).abs() / torch.exp2(E)
    d = (v.unsqueeze(-1) - GRID).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near & EVEN
    pick = torch.where(even.any(-1, keepdim=True), even, near).float().argmax(-1)
    return torch.copysign(GRID[pick], x.double()) * torch.exp2(E)


def eight_bits(x):
    """The values of the checkpoint's 8-bit codes of x."""
    unit = torch.exp2(_spread(exponents(x), x.shape[1]) - 4)
    return (torch.nan_to_num(x.double(), 0.0, 0.0, 0.0) / unit).round().clamp(-127, 127) * unit


def step(x, w, A=None, B=None, bias=None, dy=None):
    """y, and with dy the gradients (dx, dA, dB, dbias), of the layer, unrounded."""
    xh, wh, xd = four_bits(x), four_bits(w), x.double()
    y = xh @ wh.t()
    out = {}
    if A is not None:
        A, B = A.double(), B.double()
        t = xd @ A
        y = y + t @ B
    if bias is not None:
        y = y + bias.double()
    out["y"] = y
    if dy is not None:
        dy = dy.double()
        dx = dy @ wh
        if A is not None:
            dt = dy @ B.t()
            dx = dx + dt @ A.t()
            out["dA"], out["dB"] = eight_bits(x).t() @ dt, t.t() @ dy
        out["dx"], out["dbias"] = dx, dy.sum(0)
    return out
