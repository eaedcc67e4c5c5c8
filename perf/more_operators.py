"""The work that low-rank adapters of many requests over one projection, and the optimizer that tunes them, are measured on.

    listed()             the fixed cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program has in hand before the call: activations, adapters, the optimizer with its states
    run(state)           one pass, as a program makes it (own), or its plain form in 32 bits
    work(case)           bytes and operations a pass cannot do without
    exact(case, seed)    the same outputs in 64 bits

Kinds of case:
    serve  y + scale[id] (x lr_A[id]) lr_B[id] for every row, id the adapter of the row's request (none below 0): what is added to
           the output y of a projection that all requests share
    tune   the same with its backward pass: the result, and the gradients of x and of every adapter's factors
    step   one step of AdamW over the tensors of many layers (an lr_A, an lr_B and a bias each), with states in 32 bits or in 8,
           and with the gradients' common norm held to a limit, or not

States in 8 bits: 128 consecutive values share the exponent E of their largest. The mean of the gradients is held as a sign and one
of (1 + i / 8) 2^(E - 15 + j), the root of the mean of their squares as one of (1 + i / 16) 2^(E - 15 + j), j from 0 to 15; the smallest of these
stands for zero. Both are rounded up or down by a hash of the value's place, the step and a seed, so that a mean that moves by less
than a step of its grid moves on average. Values below the grid are zero, but a root that is no zero is the least one above it.

Activations are N(0, 1) with 0.5 % of the channels 20 times larger, factors N(0, 0.02), gradients of the output N(0, 0.05).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST = 65536 * (1280 + 5120)     # values of x and y of the largest listed call
MOST_TUNE = 16384 * (1280 + 5120)
MOST_STEP = 420 * (32 * (1280 + 5120) + 5120)   # parameters of the largest listed step
LR, BETAS, EPS, DECAY, STEPS = 1e-3, (0.9, 0.999), 1e-8, 0.01, 100   # (STEPS: those that came before)
MAX_NORM = 1.0
BLOCK = 128                      # 8-bit values that share an exponent


def _rows(name, kind, M, K, N, slots, rank, dtype="bf16", each=0):
    """each: rows of a request (0: requests of any length, an id for each row)"""
    return {"name": name, "kind": kind, "M": M, "K": K, "N": N, "slots": slots, "rank": rank, "dtype": dtype, "each": each}


def _step(name, layers, K, N, rank, dtype, bits, clip):
    return {"name": name, "kind": "step", "layers": layers, "K": K, "N": N, "rank": rank, "dtype": dtype, "bits": bits, "clip": clip}


def listed():
    return [
        # one request's single row through one projection, where latency is all
        _rows("one_row", "serve", 1, 1280, 1280, 4, 16, each=1),
        # single rows of 64 requests with 32 adapters among them: every adapter read for a row or two
        _rows("rows_of_64", "serve", 64, 4096, 4096, 32, 16, each=1),
        # two prompts of 77 text tokens: SDXL's cross-attention keys and values
        _rows("text_kv", "serve", 154, 2048, 1280, 8, 8, "fp16", each=77),
        # requests of odd lengths end to end, some without an adapter: SDXL's 640-channel feed-forward
        _rows("ragged_ff", "serve", 8202, 640, 5120, 12, 32, "fp16"),
        # sixteen images, each with a style of its own: the largest call
        _rows("images_ff", "serve", 65536, 1280, 5120, 16, 64, each=4096),
        # tuning on text tokens alone: a step that is mostly launches
        _rows("tune_text", "tune", 308, 2048, 640, 4, 16, "fp16", each=77),
        # an odd count of rows, and a rank that is no power of two
        _rows("tune_odd", "tune", 2051, 1280, 5120, 5, 24),
        # eight styles tuned at once on sixteen images: the largest step of tuning
        _rows("tune_images", "tune", 16384, 1280, 5120, 8, 32, each=1024),
        # the tensors of one layer: latency
        _step("step_layer", 1, 640, 5120, 16, "fp32", 32, False),
        # seven layers of odd widths, all of whose gradients share a limit
        _step("step_odd", 7, 1283, 4999, 24, "bf16", 32, True),
        # 32-bit parameters with states in 8 bits
        _step("step_8bit_fp32", 24, 4096, 4096, 64, "fp32", 8, False),
        # every layer of a model: 1260 tensors in one step
        _step("step_8bit_model", 420, 1280, 5120, 32, "bf16", 8, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("serve", "serve", "tune", "step", "step"))
    rank = rng.choice((4, 8, 16, 24, 32, 64))
    if kind == "step":
        K, N = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
        layers = _log_int(rng, 1, max(1, min(420, MOST_STEP // (rank * (K + N) + N))))
        return {"kind": kind, "layers": layers, "K": K, "N": N, "rank": rank, "dtype": rng.choice(("bf16", "fp16", "fp32")),
                "bits": rng.choice((8, 32)), "clip": rng.random() < 0.5}
    K, N = 8 * _log_int(rng, 16, 1536), 8 * _log_int(rng, 16, 1536)       # 128 to 12288, most of them no multiple of 64
    most = min(65536, MOST // (K + N)) if kind == "serve" else min(16384, MOST_TUNE // (K + N))
    M = _log_int(rng, 1 if kind == "serve" else 64, most)
    each = rng.choice((0, 1, 77, 1024))
    if each > 1:
        each = min(each, M)
        M = M // each * each
    if kind == "tune" and each == 1:
        each = 0
    return {"kind": kind, "M": M, "K": K, "N": N, "slots": rng.randint(1, 16), "rank": rank, "dtype": rng.choice(("bf16", "fp16")),
            "each": each}


def _shapes(case):
    return [s for _ in range(case["layers"]) for s in ((case["K"], case["rank"]), (case["rank"], case["N"]), (case["N"],))]


def _offsets(case):
    """Where each tensor begins in a flat buffer, and the buffer's length: multiples of 128 values."""
    at, offsets = 0, []
    for s in _shapes(case):
        offsets.append(at)
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return offsets, at


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    if case["kind"] == "step":
        offsets, n = _offsets(case)
        sizes = torch.tensor([math.prod(s) for s in _shapes(case)])
        held = torch.tensor([b - a for a, b in zip(offsets, offsets[1:] + [n])])
        counts = torch.stack([sizes, held - sizes], 1).flatten().to(dev)       # of a tensor's values, and of those behind its end
        inside = torch.repeat_interleave(torch.tensor([True, False], device=dev).repeat(len(sizes)), counts, output_size=n)
        t = {"p": (normal(n, std=0.02) * inside).to(dtype), "g": (normal(n, std=1e-3) * inside).to(dtype),
             "m": normal(n, std=3e-4) * inside, "root": 1e-3 * torch.exp(0.7 * normal(n)) * inside}
        if case["bits"] == 8:      # values that the states hold
            t["m"], t["root"] = _eight_bits(t["m"], 3, 0.5), _eight_bits(t["root"], 4, 0.5)
        return t
    M, K, N, S, R = case["M"], case["K"], case["N"], case["slots"], case["rank"]
    x = normal(M, K)
    x[:, torch.randperm(K, generator=g, device=dev)[:round(0.005 * K)]] *= 20
    t = {"x": x.to(dtype), "y": normal(M, N).to(dtype), "lr_A": normal(S, K, R, std=0.02).to(dtype),
         "lr_B": normal(S, R, N, std=0.02).to(dtype), "scale": 0.5 + torch.rand(S, generator=g, device=dev)}
    if case["each"]:
        ids = torch.randint(0, S, (M // case["each"],), generator=g, device=dev, dtype=torch.int32)
    else:      # about 20 requests of random lengths; one id of S + 1 is none
        cuts = torch.sort(torch.randint(0, M, (19,), generator=g, device=dev)).values
        request = torch.searchsorted(cuts, torch.arange(M, device=dev), right=True)
        ids = (torch.randint(0, S + 1, (20,), generator=g, device=dev, dtype=torch.int32) - 1)[request]
    t["ids"] = ids
    if case["kind"] == "tune":
        t["dy"] = normal(M, N, std=0.05).to(dtype)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    s = {"case": case, "kind": case["kind"], **t}
    if case["kind"] == "step":
        s["seed"], s["steps"] = seed, STEPS
        s["places"] = None if own or case["bits"] != 8 else torch.arange(t["p"].numel(), device="cuda")
        if case["bits"] == 32 or not own:
            s["v"] = t["root"] * t["root"]
        if own:
            from pyraquant_amd.optim import AdamW

            params = []
            for at, shape in zip(_offsets(case)[0], _shapes(case)):
                view = slice(at, at + math.prod(shape))
                params.append(torch.nn.Parameter(s["p"][view].view(shape)))
                params[-1].grad = s["g"][view].view(shape)
            s["opt"] = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, bits=case["bits"],
                             max_norm=MAX_NORM if case["clip"] else None, seed=seed)
            s["opt"].load_moments(t["m"], t["root"], STEPS)
        return s
    if own:
        from pyraquant_amd.adapters import LowRankAdapters

        bank = LowRankAdapters(case["K"], case["N"], case["slots"], case["rank"], dtype=DTYPES[case["dtype"]], device="cuda",
                               trainable=case["kind"] == "tune")
        for i, scale in enumerate(s.pop("scale").tolist()):
            bank.set(i, t["lr_A"][i], t["lr_B"][i], scale)
        s["bank"] = bank
        if case["kind"] == "tune":
            s["x"].requires_grad_()
    return s


# ---- plain forms, in 32 bits ---------------------------------------------------------------------------------------

def _eight_bits(a, bits, up):
    """a, in blocks of 128, as the 8-bit states hold it: `bits` below the leading one, cut off after `up` of the last is added (a number, or
    one for each value)."""
    sign, a = torch.sign(a), a.abs()
    drop = 23 - bits
    add = int(up * (1 << drop)) if isinstance(up, float) else up << (drop - 16)
    r = (a.view(torch.int32) + add) >> drop
    r = torch.where(a > 0, r, 0).view(-1, BLOCK)
    least = ((r.amax(1, keepdim=True) >> bits) - 15 << bits) + 1        # the first code above the one that stands for zero
    r = torch.where(r >= least, r, 0 if bits == 3 else torch.where(r > 0, least, 0))
    return (r.flatten() << drop).view(torch.float32) * sign


def _hash(places, step, seed):
    """32 bits for each place, in 64"""
    z = (places * 0x9E3779B1 + step * 0x6C8E9CF5 + seed * 0x5851F42D) & 0xFFFFFFFF
    z = ((z ^ (z >> 15)) * 0x7FB5D329) & 0xFFFFFFFF
    z = ((z ^ (z >> 13)) * 0x4C957F2B) & 0xFFFFFFFF
    return z ^ (z >> 16)


def _plain_step(s):
    case, dtype = s["case"], s["p"].dtype
    s["steps"] += 1
    b1, b2 = BETAS
    g, p, m, v = s["g"].float(), s["p"].float(), s["m"], s["v"]
    out = {}
    if case["clip"]:
        norm = s["g"].double().square().sum().sqrt().float()
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
        out["norm"] = norm
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    size = LR / (1 - b1 ** s["steps"])
    p = p * (1 - LR * DECAY) - size * m / (root / math.sqrt(1 - b2 ** s["steps"]) + EPS)
    s["p"] = out["p"] = p.to(dtype)
    if case["bits"] == 32:
        s["m"], s["v"] = out["m"], out["v"] = m, v
        return out
    h = _hash(s["places"], s["steps"], s["seed"])
    m = _eight_bits(m, 3, (h & 0xFFFF).int())
    root = _eight_bits(root, 4, (h >> 16).int())
    s["m"], s["v"] = m, root * root
    return {**out, "m": m.bfloat16(), "root": root.bfloat16()}


def _wide(f):
    """[slots, C, R] as [C, slots R]"""
    return f.permute(1, 0, 2).flatten(1)


def _plain_adapters(s):
    """All adapters side by side, and each row's own kept of what they give."""
    case, dtype = s["case"], s["x"].dtype
    M, S, R = case["M"], case["slots"], case["rank"]
    x, A, B = s["x"].float(), _wide(s["lr_A"].float()), s["lr_B"].float().flatten(0, 1)
    ids = s["ids"].repeat_interleave(case["each"], output_size=M) if case["each"] else s["ids"]
    mine = (ids[:, None] == torch.arange(S, device=ids.device)) * s["scale"]       # [M, S]: the scale, or 0
    keep = mine.repeat_interleave(R, dim=1)
    t = (x @ A) * keep
    y = (s["y"].float() + t @ B).to(dtype)
    if s["kind"] == "serve":
        return y
    dy = s["dy"].float()
    dt = (dy @ B.t()) * keep
    dA = (x.t() @ dt).view(-1, S, R).permute(1, 0, 2)
    return {"y": y, "dx": (dt @ A.t()).to(dtype), "dlr_A": dA.to(dtype).contiguous(), "dlr_B": (t.t() @ dy).view(S, R, -1).to(dtype)}


def run(state):
    if not own:
        return _plain_step(state) if state["kind"] == "step" else _plain_adapters(state)
    if state["kind"] == "step":
        opt = state["opt"]
        opt.step()
        out = {"p": state["p"]}
        if state["case"]["clip"]:
            out["norm"] = opt.grad_norm
        if state["case"]["bits"] == 32:
            out["m"], out["v"] = opt.states()
        else:
            out["m"], out["root"] = opt.moments(torch.bfloat16)
        return out
    bank = state["bank"]
    if state["kind"] == "serve":
        with torch.no_grad():
            return bank(state["x"], state["y"], state["ids"])
    x = state["x"]
    y = bank(x, state["y"], state["ids"])
    grads = torch.autograd.grad(y, [x, bank.lr_A, bank.lr_B], state["dy"])
    return dict(zip(("y", "dx", "dlr_A", "dlr_B"), (y.detach(), *grads)))


def work(case):
    if case["kind"] == "step":
        n = sum(math.prod(s) for s in _shapes(case))
        size = DTYPES[case["dtype"]].itemsize
        states = 16 if case["bits"] == 32 else 2 * (2 + 2 / BLOCK) + 4     # (with 8 bits, the values are written too)
        return {"bytes": n * (3 * size + states), "flops": 20 * n}
    M, K, N, S, R = case["M"], case["K"], case["N"], case["slots"], case["rank"]
    used = min(S, M // case["each"] if case["each"] else S) * 2 * R * (K + N)
    if case["kind"] == "serve":
        return {"bytes": 2 * M * (K + 2 * N) + used, "flops": 2 * M * R * (K + N)}
    return {"bytes": 2 * M * (2 * K + 3 * N) + 2 * used, "flops": 6 * M * R * (K + N)}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------

def _held(a, bits, u):
    """a as the states hold it: floor(a / step + u) steps, a step 2^-bits of a's power of two."""
    size = a.abs()
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(1e-300))) - bits)
    step = torch.where(size < step * 2 ** bits, step / 2, step)
    step = torch.where(size >= step * 2 ** (bits + 1), step * 2, step)        # (a logarithm that rounded across a whole one)
    r = torch.floor(size / step + u) * step
    r = torch.where(size == 0, 0.0, r).unflatten(0, (-1, BLOCK))
    top = r.amax(1, keepdim=True)
    zero = torch.exp2(torch.frexp(top)[1].double() - 1 - 15)                  # (frexp: a mantissa of [0.5, 1))
    least = zero * (1 + 2.0 ** -bits)
    r = torch.where(r > zero, r, torch.zeros_like(r) if bits == 3 else torch.where(r > 0, least, 0.0))
    return r.flatten() * torch.sign(a)


def _mixed(places, step, seed):
    word, z = 1 << 32, places
    z = (z * 0x9E3779B1 + step * 0x6C8E9CF5 + seed * 0x5851F42D) % word
    for shift, factor in ((15, 0x7FB5D329), (13, 0x4C957F2B)):
        z = torch.bitwise_xor(z, z // 2 ** shift)
        z = ((z // 65536 * factor % 65536) * 65536 + z % 65536 * factor) % word      # (no product over 2^63)
    z = torch.bitwise_xor(z, z // 65536)
    return (z % 65536) / 65536.0, (z // 65536) / 65536.0


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "step":
        p, g, m, root = (t[k].double() for k in ("p", "g", "m", "root"))
        v = root.square() if case["bits"] == 8 else (t["root"] * t["root"]).double()
        (b1, b2), n = BETAS, STEPS + 1
        out = {}
        if case["clip"]:
            out["norm"] = torch.linalg.vector_norm(g)
            g = g / torch.clamp((out["norm"] + 1e-6) / MAX_NORM, min=1.0)
        m = torch.lerp(g, m, b1)
        v = b2 * v + (1 - b2) * g.square()
        hat = m / (1 - b1 ** n) / ((v / (1 - b2 ** n)).sqrt() + EPS)
        out["p"] = p - LR * (hat + DECAY * p)
        if case["bits"] == 32:
            return {**out, "m": m, "v": v}
        um, ur = _mixed(torch.arange(p.numel(), device=p.device), n, seed)
        return {**out, "m": _held(m, 3, um), "root": _held(v.sqrt(), 4, ur)}
    x, A, B, y = (t[k].double() for k in ("x", "lr_A", "lr_B", "y"))
    rows = torch.arange(case["M"], device=x.device)
    ids = t["ids"][rows // case["each"]] if case["each"] else t["ids"]
    out = {"y": y}
    if case["kind"] == "tune":
        dy = t["dy"].double()
        out |= {"dx": torch.zeros_like(x), "dlr_A": torch.zeros_like(A), "dlr_B": torch.zeros_like(B)}
    for i, scale in enumerate(t["scale"].double().tolist()):
        mine = rows[ids == i]
        if not mine.numel():
            continue
        down = torch.mm(x[mine], A[i]) * scale
        y[mine] += torch.mm(down, B[i])
        if case["kind"] == "tune":
            back = torch.mm(dy[mine], B[i].t()) * scale
            out["dx"][mine] = torch.mm(back, A[i].t())
            out["dlr_A"][i] = torch.mm(x[mine].t(), back)
            out["dlr_B"][i] = torch.mm(down.t(), dy[mine])
    return y if case["kind"] == "serve" else out
