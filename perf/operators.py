"""The work that the microscaled 4-bit layers are measured on: weights converted, layers called, low-rank branches tuned.

    listed()             the fixed cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program has in hand before the call: activations, gradients, weights, the converted layer
    run(state)           one pass, as a program makes it (own), or its plain form in 32 bits
    work(case)           bytes and operations a pass cannot do without
    exact(case, seed)    the same outputs in 64 bits

Kinds of case:
    weight  what a 4-bit copy of a weight holds: quant_mxfp4 and back to values
    linear  y = Mxfp4Linear(x): 4-bit activations and weights, with or without a low-rank branch and a bias
    train   one step of tuning a layer's low-rank branch and bias over frozen 4-bit weights: y, and the gradients of x, lr_A,
            lr_B and the bias; what the backward pass keeps of x are 8-bit codes

The format: 32 consecutive values of a row share the power of two 2^E, E = floor(log2(max |x|)) - 2, and are held as the nearest
of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^E (ties to an even last bit, saturated at 6). The 8-bit codes of the backward pass are
rint(x 2^(4 - E)) in [-127, 127], worth 2^(E - 4) each.

Activations are N(0, 1) with 0.5 % of the channels 20 times larger, weights N(0, 0.02), low-rank factors N(0, 0.02), bias
N(0, 0.01), gradients of the output N(0, 0.05).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST = 65536 * 3072 * 12288      # multiply-adds of the largest listed layer call
MOST_TRAIN = 16384 * 3072 * 12288   # of one product of the largest listed training step


def _case(name, kind, M, K, N, dtype="bf16", rank=0, bias=True):
    return {"name": name, "kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "rank": rank, "bias": bias}


def listed():
    return [
        # loading a small projection (SDXL, 640 channels) into 4 bits
        {"name": "weight_small", "kind": "weight", "K": 640, "N": 640, "dtype": "fp16"},
        # loading FLUX's MLP up-projection
        {"name": "weight_flux_mlp", "kind": "weight", "K": 3072, "N": 12288, "dtype": "bf16"},
        # one token: a per-image embedding's projection, where latency is all
        _case("one_token", "linear", 1, 1280, 1280),
        # two prompts of 77 text tokens: SDXL's cross-attention keys and values, no bias
        _case("text_kv", "linear", 154, 2048, 1280, "fp16", bias=False),
        # FLUX's 512 prompt tokens through the MLP down-projection: few rows, a long K
        _case("text_mlp_down", "linear", 512, 12288, 3072, rank=32),
        # SDXL, routed tokens: an odd row count and a short K
        _case("odd_rows_ff", "linear", 8202, 640, 5120, "fp16"),
        # FLUX 1K, attention projection with its low-rank branch
        _case("attn_1k", "linear", 4096, 3072, 3072, rank=32),
        # FLUX 4K, MLP up-projection: the largest call
        _case("mlp_up_4k", "linear", 65536, 3072, 12288, rank=32),
        # tuning on text tokens alone: a step that is mostly launches
        _case("tune_text", "train", 154, 2048, 640, "fp16", rank=16),
        # tuning an SDXL feed-forward up-projection on an odd count of tokens
        _case("tune_ff", "train", 2050, 1280, 5120, "bf16", rank=64),
        # tuning FLUX's 1K attention projection with its text tokens
        _case("tune_attn_1k", "train", 4352, 3072, 3072, rank=32),
        # tuning FLUX's 2K MLP up-projection: the largest step
        _case("tune_mlp_2k", "train", 16384, 3072, 12288, rank=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("weight", "linear", "linear", "train", "train"))
    K = 32 * _log_int(rng, 8, 384)       # 256 to 12288, most of them no multiple of 128
    N = 16 * _log_int(rng, 16, 768)      # 256 to 12288
    dtype = rng.choice(("bf16", "fp16"))
    if kind == "weight":
        return {"kind": kind, "K": K, "N": N, "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    most = min(65536, MOST // (K * N)) if kind == "linear" else min(16384, MOST_TRAIN // (K * N))
    M = _log_int(rng, 1 if kind == "linear" else 64, most)
    rank = rng.choice((0, 16, 32, 64)) if kind == "linear" else rng.choice((16, 32, 64))
    return {"kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "rank": rank, "bias": rng.random() < 0.75}


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    K, N, dtype = case["K"], case["N"], DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    t = {"w": normal(N, K, std=0.02).to(dtype)}
    if case["kind"] == "weight":
        return t
    x = normal(case["M"], K)
    x[:, torch.randperm(K, generator=g, device=dev)[:round(0.005 * K)]] *= 20
    t["x"] = x.to(dtype)
    if case["rank"]:
        t["lr_A"] = normal(K, case["rank"], std=0.02).to(dtype)
        t["lr_B"] = normal(case["rank"], N, std=0.02).to(dtype)
    if case["bias"]:
        t["bias"] = normal(N, std=0.01)
    if case["kind"] == "train":
        t["dy"] = normal(case["M"], N, std=0.05).to(dtype)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    s = {"kind": case["kind"], **t}
    if case["kind"] == "weight":
        return s
    if own:
        from pyraquant_amd.mxfp4 import Mxfp4Linear

        lin = torch.nn.Linear(case["K"], case["N"], bias=case["bias"], device="meta")
        lin.weight = torch.nn.Parameter(s.pop("w"), requires_grad=False)
        if case["bias"]:
            lin.bias = torch.nn.Parameter(s.pop("bias"), requires_grad=False)
        s["layer"] = Mxfp4Linear(lin, lowrank=(s["lr_A"], s["lr_B"]) if case["rank"] else None,
                                 trainable=case["kind"] == "train")
        if case["kind"] == "train":
            s["x"].requires_grad_()
    else:
        s["w"] = _four_bits(s["w"].float())[0]
    return s


# ---- plain forms, in 32 bits ---------------------------------------------------------------------------------------

def _four_bits(x):
    """(x in the 4-bit format, its 2^E per block of 32)"""
    b = x.reshape(x.shape[0], -1, 32)
    a = b.abs().amax(-1, keepdim=True)
    e = torch.where(a > 0, torch.frexp(a)[1] - 3, -127).clamp_min(-127)   # a = f 2^p, f in [0.5, 1): floor(log2 a) = p - 1
    v = torch.ldexp(b, -e)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return torch.ldexp(((v / step).round() * step).clamp(-6, 6), e).reshape(x.shape), e


def _plain_forward(s, x):
    y = _four_bits(x)[0] @ s["w"].t()
    t = x @ s["lr_A"].float() if "lr_A" in s else None
    if t is not None:
        y += t @ s["lr_B"].float()
    if "bias" in s:
        y += s["bias"]
    return y, t


def _plain_train(s):
    x, dy, dtype = s["x"].float(), s["dy"].float(), s["x"].dtype
    y, t = _plain_forward(s, x)
    e = _four_bits(x)[1]
    kept = torch.ldexp(torch.ldexp(x.reshape(x.shape[0], -1, 32), 4 - e).round().clamp(-127, 127), e - 4).reshape(x.shape)
    dt = dy @ s["lr_B"].float().t()
    out = {"y": y.to(dtype), "dx": (dy @ s["w"] + dt @ s["lr_A"].float().t()).to(dtype),
           "dlr_A": (kept.t() @ dt).to(dtype), "dlr_B": (t.t() @ dy).to(dtype)}
    if "bias" in s:
        out["dbias"] = dy.sum(0)
    return out


def run(state):
    kind = state["kind"]
    if not own:
        if kind == "weight":
            return _four_bits(state["w"].float())[0].to(state["w"].dtype)
        if kind == "linear":
            return _plain_forward(state, state["x"].float())[0].to(state["x"].dtype)
        return _plain_train(state)
    if kind == "weight":
        from pyraquant_amd.mxfp4 import dequant_mxfp4, quant_mxfp4

        return dequant_mxfp4(quant_mxfp4(state["w"]), state["w"].dtype)
    layer, x = state["layer"], state["x"]
    if kind == "linear":
        with torch.no_grad():
            return layer(x)
    y = layer(x)
    wanted = [x, layer.lr_A, layer.lr_B] + ([] if layer.bias is None else [layer.bias])
    grads = torch.autograd.grad(y, wanted, state["dy"])
    return dict(zip(("y", "dx", "dlr_A", "dlr_B", "dbias"), (y.detach(), *grads)))


def work(case):
    K, N = case["K"], case["N"]
    held = N * K * (1 / 2 + 1 / 32)      # 4-bit codes and a byte of scale per 32
    if case["kind"] == "weight":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": N * K * 2 * size, "flops": N * K}
    M, R = case["M"], case["rank"]
    small = 2 * R * (K + N) + (4 * N if case["bias"] else 0)
    if case["kind"] == "linear":
        return {"bytes": 2 * M * (K + N) + held + small, "flops": 2 * M * N * K + 2 * M * R * (K + N)}
    return {"bytes": 4 * M * (K + N) + held + 2 * small, "flops": 4 * M * N * K + 6 * M * R * (K + N)}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------

def _nearest(x):
    """Each value of x as the format holds it, and the exponents E, by comparison with the midpoints of the grid."""
    blocks = x.unflatten(1, (-1, 32))
    top = blocks.abs().amax(2)
    low = top == 0
    E = (torch.log2(torch.where(low, 1.0, top)) + 1e-13).floor()
    E = torch.where(torch.exp2(E) > torch.where(low, 1.0, top), E - 1, E)     # (a logarithm that rounded up to a whole one)
    E = torch.where(low, -127.0, (E - 2).clamp_min(-127.0)).unsqueeze(2)
    v = (blocks / torch.exp2(E)).abs()
    # a tie goes to the neighbour whose last bit is even: down to 0, 1, 2, 4, or up to 1, 2, 4
    h = (0.5 * (v > 0.25) + 0.5 * (v >= 0.75) + 0.5 * (v > 1.25) + 0.5 * (v >= 1.75) + 1.0 * (v > 2.5) + 1.0 * (v >= 3.5)
         + 2.0 * (v > 5))
    return (torch.sign(blocks) * h * torch.exp2(E)).flatten(1), E


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    w = _nearest(t["w"])[0]
    if case["kind"] == "weight":
        return w
    x, E = _nearest(t["x"])
    y = torch.mm(x, w.t())
    del x
    if case["rank"]:
        down = torch.mm(t["x"], t["lr_A"])
        y.addmm_(down, t["lr_B"])
    if case["bias"]:
        y += t["bias"]
    if case["kind"] == "linear":
        return y
    dy = t["dy"]
    dt = torch.mm(dy, t["lr_B"].t())
    unit = torch.exp2(E - 4)
    kept = ((t["x"].unflatten(1, (-1, 32)) / unit).round().clamp(-127, 127) * unit).flatten(1)
    out = {"y": y, "dx": torch.mm(dy, w) + torch.mm(dt, t["lr_A"].t()), "dlr_A": torch.mm(kept.t(), dt),
           "dlr_B": torch.mm(down.t(), dy)}
    if case["bias"]:
        out["dbias"] = dy.sum(0)
    return out
