"""Quantize a feed-forward block to 4 bits, win back what the rounding lost by tuning its low-rank branches, and serve it.

    python examples/tune_mxfp4_lowrank.py [--dim 640] [--tokens 2048] [--rank 32] [--steps 60]

The block is Linear -> GELU -> Linear with random weights. Each Linear becomes an Mxfp4Linear whose low-rank branch starts as
the best rank-r approximation of what the 4-bit weight lost (its singular vectors). The branches and biases are then tuned to
the original block's outputs over frozen 4-bit weights, the backward passes reading 8-bit checkpoints of the activations, and
the layers are frozen and called as a server calls them. Prints the relative error after each part.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pyraquant_amd.int8_exec import LOWRANK_A_ATTR, LOWRANK_B_ATTR  # noqa: E402
from pyraquant_amd.mxfp4 import Mxfp4Linear, convert_linears_to_mxfp4, dequant_mxfp4, quant_mxfp4  # noqa: E402


def attach_residual_branch(lin: nn.Linear, rank: int) -> None:
    """lr_A lr_B = the rank-r part of (w - its 4-bit values)^T"""
    w = lin.weight.detach().float()
    U, S, Vh = torch.linalg.svd((w - dequant_mxfp4(quant_mxfp4(w), torch.float32)).t().cpu(), full_matrices=False)
    root = S[:rank].sqrt()
    setattr(lin, LOWRANK_A_ATTR, (U[:, :rank] * root).to(w.device, lin.weight.dtype))
    setattr(lin, LOWRANK_B_ATTR, (root[:, None] * Vh[:rank]).to(w.device, lin.weight.dtype))


def run(dim=640, tokens=2048, rank=32, steps=60, dtype=torch.bfloat16, seed=0):
    """(error with the 4-bit weights alone, with the branches as they start, tuned, served)"""
    torch.manual_seed(seed)
    dev = torch.device("cuda")
    block = nn.Sequential(nn.Linear(dim, 4 * dim), nn.GELU(), nn.Linear(4 * dim, dim)).to(dev, dtype)
    sample = lambda: torch.randn(tokens, dim, device=dev).to(dtype)   # noqa: E731
    test = sample()
    with torch.no_grad():
        weights = [m.weight.clone() for m in block if isinstance(m, nn.Linear)]
        biases = [m.bias.clone() for m in block if isinstance(m, nn.Linear)]

    def teacher(x):
        with torch.no_grad():
            return nn.functional.linear(nn.functional.gelu(nn.functional.linear(x, weights[0], biases[0])), weights[1], biases[1])

    def error(net):
        with torch.no_grad():
            want = teacher(test).float()
            return float((net(test).float() - want).norm() / want.norm())

    bare = error(nn.Sequential(Mxfp4Linear(block[0]), nn.GELU(), Mxfp4Linear(block[2])))
    for lin in (block[0], block[2]):
        attach_residual_branch(lin, rank)
    convert_linears_to_mxfp4(block, trainable=True)
    started = error(block)
    opt = torch.optim.Adam(block.parameters(), lr=3e-4)
    for _ in range(steps):
        x = sample()
        loss = (block(x).float() - teacher(x).float()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
    tuned = error(block)
    for m in block:
        if isinstance(m, Mxfp4Linear):
            m.freeze()
    return bare, started, tuned, error(block)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("dim", 640), ("tokens", 2048), ("rank", 32), ("steps", 60)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    for what, e in zip(("4-bit weights", "with low-rank branches", "tuned", "served"), run(a.dim, a.tokens, a.rank, a.steps)):
        print(f"{what:24s} relative error {e:.4f}", flush=True)
