"""Adapters of many requests against their formulas in 64 bits.

Bounds, with f = 2^-24, u half a step of the type (bf16 2^-8, fp16 2^-11), w what two 16-bit parts lose of a value: the first is within one of
its own steps of it, 2 u, the second rounded to u of that: 2 u^2 (fp16: at least half of its smallest subnormal, 2^-25):
  t   K sums:      K f |x| |A|, and 2 f for the scale and the sums of parts; as an operand w |t| more
  y   t's bound times |B|, R + 2 sums and base: (R + 4) f |t| |B| + 2 f (|base| + |y|), and u |y|
  dA, dB: sums over M rows of products with t or dt: that one's bound times |x| or |dy|, M f of the terms, and u of the result
(u of a result among fp16's subnormals: at least 2^-25.)
"""
import ctypes
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
F = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BOTH = (torch.bfloat16, torch.float16)


def _bank(A, B, scale, trainable=False):
    from pyraquant_amd.adapters import LowRankAdapters

    slots, K, R = A.shape
    bank = LowRankAdapters(K, B.shape[2], slots, R, dtype=A.dtype, device="cuda", trainable=trainable)
    for i, s in enumerate(scale.tolist()):
        bank.set(i, A[i], B[i], s)
    return bank


def _problem(M, K, N, slots, R, dtype, ids, seed=0, wide=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    x, y = r(M, K).to(dtype), r(M, N).to(dtype)
    A, B = (r(slots, K, R) * K ** -0.5).to(dtype), (r(slots, R, N) * R ** -0.5).to(dtype)
    scale = torch.rand(slots, generator=g, device="cuda") + 0.5
    if ids == "one":
        i = torch.full((M,), slots - 1, device="cuda")
    elif ids == "none":
        i = torch.full((M,), -1, device="cuda")
    elif ids == "rows":      # any id for any row, some past either end
        i = torch.randint(-1, slots + 1, (M,), generator=g, device="cuda")
        i[::7] = torch.tensor([-(1 << 31), (1 << 31) - 1, -2, slots], device="cuda").repeat(M)[: len(i[::7])]
    else:                    # runs of any length
        cuts = torch.sort(torch.randint(0, M + 1, (6,), generator=g, device="cuda")).values
        i = torch.randint(-1, slots, (7,), generator=g, device="cuda")[torch.searchsorted(cuts, torch.arange(M, device="cuda"), right=True)]
    return x, y, i.long() if wide else i.int(), A, B, scale


def _want(x, y, ids, A, B, scale, dy=None):
    """(results, bounds) in 64 bits"""
    M, K = x.shape
    (slots, _, R), N = A.shape, B.shape[2]
    u = U[x.dtype]
    w, tiny = 2 * u * u, 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    x64, y64, A64, B64, s64 = (t.detach().double() for t in (x, y, A, B, scale))
    dev = x.device
    out = {"y": y64.clone()}
    off = {"y": torch.zeros_like(y64)}
    if dy is not None:
        dy64 = dy.double()
        for k, like in (("dx", x64), ("dA", A64), ("dB", B64)):
            out[k], off[k] = torch.zeros_like(like), torch.zeros_like(like)
    for i in range(slots):
        rows = torch.arange(M, device=dev)[ids.to(dev) == i]
        if not len(rows):
            continue
        xs, a, b, s = x64[rows], A64[i], B64[i], float(s64[i])
        t = xs @ a * s
        t_off = s * (K + 2) * F * (xs.abs() @ a.abs())
        t_part = w * (t.abs() + t_off) + tiny
        term = t @ b
        out["y"][rows] += term
        mag = (t.abs() + t_off) @ b.abs()
        o = (t_off + t_part) @ b.abs() + (R + 4) * F * mag + 2 * F * (y64[rows].abs() + term.abs())
        off["y"][rows] = o + u * (out["y"][rows].abs() + o) + tiny
        if dy is None:
            continue
        d = dy64[rows]
        dt = d @ b.t() * s
        d_off = s * (N + 2) * F * (d.abs() @ b.abs().t())
        d_part = w * (dt.abs() + d_off) + tiny
        out["dx"][rows] = dt @ a.t()
        o = (d_off + d_part) @ a.abs().t() + (R + 4) * F * ((dt.abs() + d_off) @ a.abs().t())
        off["dx"][rows] = o + u * (out["dx"][rows].abs() + o) + tiny
        m = len(rows)
        out["dA"][i] = xs.t() @ dt
        o = xs.abs().t() @ (d_off + d_part) + (m + 300) * F * (xs.abs().t() @ (dt.abs() + d_off))
        off["dA"][i] = o + u * (out["dA"][i].abs() + o) + tiny
        out["dB"][i] = t.t() @ d
        o = (t_off + t_part).t() @ d.abs() + (m + 300) * F * ((t.abs() + t_off).t() @ d.abs())
        off["dB"][i] = o + u * (out["dB"][i].abs() + o) + tiny
    return out, off


def _near(got, want, off, what):
    over = (got.double() - want).abs() - off
    assert bool((over <= 0).all()), (what, float(over.max()), int((over > 0).sum()), got.numel())


SIZES = [(1, 8, 8, 1, 1), (1, 1280, 1288, 4, 16), (2, 24, 40, 2, 3), (15, 64, 72, 3, 8), (17, 136, 16, 5, 17), (33, 320, 264, 2, 24),
         (63, 128, 520, 40, 32), (64, 256, 64, 3, 33), (65, 1288, 8, 2, 64), (127, 40, 1000, 6, 15), (300, 2048, 136, 4, 48), (1025, 96, 328, 7, 16),
         (2051, 520, 808, 3, 32), (40, 2600, 72, 5, 64), (70, 72, 2600, 4, 64), (1, 10752, 16, 2, 8), (700, 136, 264, 9, 40)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("ids", ("one", "runs", "rows", "none"))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_backward(cuda, size, ids, dtype):
    M, K, N, slots, R = size
    x, y, i, A, B, scale = _problem(*size, dtype, ids, seed=M + R, wide=M % 2 == 0)
    dy = torch.randn(M, N, device=cuda).to(dtype)
    want, off = _want(x, y, i, A, B, scale, dy)
    frozen, tuned = _bank(A, B, scale), _bank(A, B, scale, trainable=True)
    none = (i < 0) | (i >= slots)
    with torch.no_grad():
        got = frozen(x, y, i)
        _near(got, want["y"], off["y"], "y")
        assert torch.equal(got[none], y[none]) and torch.equal(tuned(x, y, i), got)
        room = torch.full((M * N + 64,), 7.0, dtype=dtype, device=cuda)
        into = room[32: 32 + M * N].view(M, N)
        assert frozen(x, y, i, out=into) is into and torch.equal(into, got)
        into.copy_(y)
        frozen(x, into, i, out=into)
        assert torch.equal(into, got) and bool((room[:32] == 7).all()) and bool((room[32 + M * N:] == 7).all())
    x.requires_grad_()
    y.requires_grad_()
    out = tuned(x, y, i)
    assert torch.equal(out, got)
    dx, dy0, dA, dB = torch.autograd.grad(out, (x, y, tuned.lr_A, tuned.lr_B), dy)
    assert torch.equal(dy0, dy)
    for k, v in (("dx", dx), ("dA", dA), ("dB", dB)):
        _near(v, want[k], off[k], k)
    assert not dx[none].any()
    used = torch.zeros(slots, dtype=torch.bool, device=cuda)
    used[i[~none].long()] = True
    assert not dA[~used].any() and not dB[~used].any()
    fx, fy = torch.autograd.grad(frozen(x, y, i), (x, y), dy)
    assert torch.equal(fx, dx) and torch.equal(fy, dy)
    # what is wanted alone is the same
    assert torch.equal(torch.autograd.grad(tuned(x.detach(), y.detach(), i), tuned.lr_B, dy)[0], dB)
    assert torch.equal(torch.autograd.grad(tuned(x.detach(), y.detach(), i), tuned.lr_A, dy)[0], dA)


@pytest.mark.parametrize("dtype", BOTH)
def test_gradients_against_differences(cuda, dtype):
    """The result is linear in x, in lr_A and in lr_B: a step of any size in one of them moves sum(g y) by the gradient times the step, up to
    what the two results are off (their bounds times |g|) and the gradient's own bound times |step|."""
    x, y, i, A, B, scale = _problem(70, 72, 40, 3, 8, dtype, "runs", seed=5)
    y.zero_()
    g = torch.randn(70, 40, device=cuda).to(dtype)
    bank = _bank(A, B, scale, trainable=True)
    x.requires_grad_()
    grads = torch.autograd.grad(bank(x, y, i), (x, bank.lr_A, bank.lr_B), g)
    _, off = _want(x, y, i, A, B, scale, g)

    def loss(x, A, B):
        with torch.no_grad():
            r = _bank(A, B, scale)(x, y, i)
        return float((r.double() * g.double()).sum()), float((_want(x, y, i, A, B, scale)[1]["y"] * g.double().abs()).sum())

    start, start_off = loss(x, A, B)
    for k, (grad, name) in enumerate(zip(grads, ("dx", "dA", "dB"))):
        args = [x.detach(), A, B]
        moved = (args[k] + torch.randn(args[k].shape, device=cuda).to(dtype)).to(dtype)
        step = moved.double() - args[k].double()
        args[k] = moved
        end, end_off = loss(*args)
        expected = float((grad.double() * step).sum())
        assert abs(end - start - expected) <= start_off + end_off + float((off[name] * step.abs()).sum()), name


def test_requests_stay_apart(cuda):
    """NaN and infinities in one request's rows and in one adapter change nothing elsewhere, whatever shares a tile with them."""
    for ids in ("rows", "runs"):
        x, y, i, A, B, scale = _problem(200, 136, 264, 4, 20, torch.bfloat16, ids, seed=1)
        dy = torch.randn(200, 264, device=cuda).bfloat16()
        clean = _bank(A, B, scale, trainable=True)
        A2, B2, x2 = A.clone(), B.clone(), x.clone()
        A2[2, 5] = float("nan")
        B2[2, :, 7] = float("inf")
        x2[i == 2] = float("nan")
        x2[i == -1] = float("inf")
        dirty = _bank(A2, B2, scale, trainable=True)
        good = i != 2
        y1, y2 = clean(x, y, i), dirty(x2, y, i)
        assert torch.equal(y1[good], y2[good])
        g1 = torch.autograd.grad(y1, (clean.lr_A, clean.lr_B), dy)
        g2 = torch.autograd.grad(y2, (dirty.lr_A, dirty.lr_B), dy)
        for a, b in zip(g1, g2):
            assert torch.equal(a[[0, 1, 3]], b[[0, 1, 3]])
        xs = [x.clone().requires_grad_(), x2.clone().requires_grad_()]
        d = [torch.autograd.grad(m(v, y, i), v, dy)[0] for m, v in zip((clean, dirty), xs)]
        assert torch.equal(d[0][good], d[1][good])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("R", (1, 17, 33))
def test_infinities_and_padding(cuda, dtype, R):
    """An infinity in x stays one where its products have one sign: the zeros that pad ranks do not make it NaN. Zero rows times an
    infinite factor are NaN, as in the formula."""
    x, y, i, A, B, scale = _problem(20, 64, 72, 2, R, dtype, "one", seed=2)
    A, B = A.abs() + 0.01, B.abs() + 0.01
    x[3, 5] = float("inf")
    with torch.no_grad():
        got = _bank(A, B, scale)(x, y, i)
        assert bool(torch.isposinf(got[3]).all()) and bool(got[:3].isfinite().all()) and bool(got[4:].isfinite().all())
        x[3, 5], B[1, 0, 9] = 1.0, float("inf")
        x[7] = 0
        got = _bank(A, B, scale)(x, y, i)
        bad = ~got.isfinite()
        assert bool(bad[:, 9].all()) and not bad[:, :9].any() and not bad[:, 10:].any() and bool(got[7, 9].isnan())


def test_values_past_fp16(cuda):
    """t and dt past 65504 where results are not: taken with a power of two, to the same bounds."""
    x, y, i, A, B, scale = _problem(150, 264, 136, 3, 20, torch.float16, "runs", seed=3)
    A = (A.float() * 4000).half()
    B = (B.float() * 2.0 ** -10).half()
    x = (x.float() * 30).half()
    dy = torch.randn(150, 136, device=cuda).half()
    want, off = _want(x, y, i, A, B, scale, dy)
    bank = _bank(A, B, scale, trainable=True)
    assert float((x.double() @ A[1].double()).abs().max()) > 1e5
    x.requires_grad_()
    out = bank(x, y, i)
    _near(out, want["y"], off["y"], "y")
    grads = torch.autograd.grad(out, (x, bank.lr_A, bank.lr_B), dy * 2.0 ** -6)
    dy2 = (dy * 2.0 ** -6)
    want, off = _want(x.detach(), y, i, A, B, scale, dy2)
    for v, k in zip(grads, ("dx", "dA", "dB")):
        fits = want[k].abs() < 60000
        assert bool(((v.double() - want[k]).abs() <= off[k])[fits].all()), k
    # and dt: a large dy over large factors, a small A
    B2, A2 = (B.float() * 2.0 ** 16).half(), (A.float() * 2.0 ** -22).half()
    dy3 = (dy.float() * 2000).half()
    want, off = _want(x.detach(), y, i, A2, B2, scale, dy3)
    bank = _bank(A2, B2, scale, trainable=True)
    assert float((dy3.double() @ B2[1].double().t()).abs().max()) > 1e5
    grads = torch.autograd.grad(bank(x, y, i), (x, bank.lr_A), dy3)
    for v, k in zip(grads, ("dx", "dA")):
        fits = want[k].abs() < 60000
        assert bool(((v.double() - want[k]).abs() <= off[k])[fits].all()), k


def test_shapes_strides_and_ids(cuda):
    """Leading dimensions with an id for some of them, an id for all rows, none at all; rows of larger tensors, at odd places, turned."""
    x, y, i, A, B, scale = _problem(24, 64, 40, 3, 8, torch.bfloat16, "rows", seed=4)
    bank = _bank(A, B, scale)
    with torch.no_grad():
        flat = bank(x, y, i)
        assert torch.equal(bank(x.view(2, 3, 4, 64), y.view(2, 3, 4, 40), i.view(2, 3, 4)).view(24, 40), flat)
        i3 = torch.tensor([2, -1, 0], device=cuda)
        each = bank(x, y, i3.repeat_interleave(8))
        assert torch.equal(bank(x.view(3, 8, 64), y.view(3, 8, 40), i3).view(24, 40), each)
        i6 = torch.tensor([[2, -1], [0, 1], [1, 1]], device=cuda)
        assert torch.equal(bank(x.view(3, 2, 4, 64), y.view(3, 2, 4, 40), i6).view(24, 40), bank(x, y, i6.flatten().repeat_interleave(4)))
        assert torch.equal(bank(x, y, torch.tensor(1, device=cuda)), bank(x, y, torch.ones(24, dtype=torch.int32, device=cuda)))
        assert torch.equal(bank(x[0], y[0], torch.tensor(1, device=cuda)), bank(x[:1], y[:1], torch.tensor([1], device=cuda))[0])
        assert bank(x[:0], y[:0], i[:0]).shape == (0, 40) and bank(x.view(24, 1, 64)[:, :0], y.view(24, 1, 40)[:, :0], i).shape == (24, 0, 40)
        big_x, big_y = torch.zeros(24, 200, dtype=x.dtype, device=cuda), torch.zeros(48, 41, dtype=x.dtype, device=cuda)
        for at in (8, 9, 11):
            big_x[:, at:at + 64], big_y[::2, 1:] = x, y
            assert torch.equal(bank(big_x[:, at:at + 64], big_y[::2, 1:], torch.stack([i, i], 1)[:, 0]), flat)
        assert torch.equal(bank(x.t().contiguous().t(), y.t().contiguous().t(), i), flat)
        assert torch.equal(bank(x[:1].expand(24, 64), y, i), bank(x[:1].repeat(24, 1), y, i))
    tuned = _bank(A, B, scale, trainable=True)
    v = x.clone().requires_grad_()
    tuned(v.view(2, 12, 64), y.view(2, 12, 40), i.view(2, 12)).sum().backward()      # (a gradient without strides)
    ones = torch.ones(24, 40, dtype=x.dtype, device=cuda)
    ref = torch.autograd.grad(tuned(v, y, i), (v, tuned.lr_A, tuned.lr_B), ones)
    assert all(torch.equal(a, b) for a, b in zip((v.grad, tuned.lr_A.grad, tuned.lr_B.grad), ref))
    empty = tuned(v[:0], y[:0], i[:0])
    g = torch.autograd.grad(empty, (v, tuned.lr_A, tuned.lr_B), torch.ones_like(empty))
    assert not any(t.any() for t in g) and g[1].shape == tuned.lr_A.shape


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,each,K,N,slots,R", [(9, 300, 136, 264, 9, 24), (5, 1000, 520, 72, 12, 16), (40, 70, 64, 1032, 30, 64), (3, 2000, 1032, 64, 65, 8),
                                                (128, 128, 8, 136, 6, 32)])
def test_batches_of_long_requests(cuda, n, each, K, N, slots, R, dtype):
    """An id for each request of many rows: the same bits as with an id for each row, forward and back (but for the sums over rows, whose
    chunks are whole requests), whole tiles of one adapter among others with several and with none, and every adapter's gradient written."""
    x, y, _, A, B, scale = _problem(n * each, K, N, slots, R, dtype, "one", seed=n)
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-1, slots + 1, (n,), generator=g, device=cuda)
    dy = torch.randn(n * each, N, device=cuda).to(dtype)
    bank = _bank(A, B, scale, trainable=True)
    x.requires_grad_()
    rows = ids.repeat_interleave(each)
    out = bank(x.view(n, each, K), y.view(n, each, N), ids)
    junk = torch.full((1 << 26,), float("nan"), device=cuda)      # (memory that the workspaces may get)
    del junk
    got = torch.autograd.grad(out, (x, bank.lr_A, bank.lr_B), dy.view(n, each, N))
    flat = bank(x, y, rows)
    want = torch.autograd.grad(flat, (x, bank.lr_A, bank.lr_B), dy)
    assert torch.equal(out.view(flat.shape), flat) and torch.equal(got[0], want[0])
    exact, off = _want(x.detach(), y, rows, A, B, scale, dy)
    _near(flat.detach(), exact["y"], off["y"], "y")
    for k, v, r in zip(("dx", "dA", "dB"), got, want):
        _near(v, exact[k], off[k], k)
        _near(r, exact[k], off[k], k)


def test_factors_of_another_type(cuda):
    """fp32 factors are cast in each call, and get gradients in fp32; a frozen module answers as the tuned one."""
    x, y, i, A, B, scale = _problem(40, 64, 72, 3, 12, torch.bfloat16, "runs")
    bank = _bank(A.float(), B.float(), scale, trainable=True)
    out = bank(x, y, i)
    out.backward(torch.ones_like(out))
    assert bank.lr_A.grad.dtype == torch.float32 and bank.lr_B.grad.any()
    exact = _bank(A, B, scale, trainable=True)
    assert torch.equal(exact(x, y, i), out)
    with torch.no_grad():
        assert torch.equal(bank.freeze()(x, y, i), out) and bank.lr_Af.dtype == torch.float32
        assert torch.equal(exact.freeze()(x, y, i), out) and torch.equal(bank.freeze(torch.bfloat16)(x, y, i), out)


def test_refusals(cuda):
    x, y, i, A, B, scale = _problem(24, 64, 40, 3, 8, torch.bfloat16, "runs")
    bank, tuned = _bank(A, B, scale), _bank(A, B, scale, trainable=True)
    with torch.no_grad():
        for bad in ((x[:, :56], y, i), (x, y[:20], i), (x, y, i[:20]), (x, y, i.view(24, 1)), (x.view(2, 12, 64), y, i.view(2, 12)), (x, y, i.cpu()),
                    (x, y.cpu(), i), (x.view(4, 6, 64), y.view(4, 6, 40), i[:6])):
            with pytest.raises(AssertionError):
                bank(*bad)
        for bad in ((x.float(), y, i), (x, y.half(), i), (x, y, i.float()), (x, y, i.short())):
            with pytest.raises(ValueError):
                bank(*bad)
        for out in (y[:20], y.t().contiguous().t(), torch.cat([y, y])[1:25].view(-1)[4:].view(-1), torch.empty(24, 64, device=cuda, dtype=y.dtype)):
            with pytest.raises(AssertionError):
                bank(x, y, i, out=out)
        both = torch.cat([y, y]).view(-1)
        with pytest.raises(AssertionError, match="shares memory"):
            bank(x, both[:960].view(24, 40), i, out=both[80:1040].view(24, 40))
        with pytest.raises(ValueError):
            bank(x, y, i, out=torch.empty_like(y, dtype=torch.float16))
    with pytest.raises(AssertionError, match="without gradients"):
        tuned(x, y, i, out=torch.empty_like(y))
    with pytest.raises(AssertionError, match="no gradients"):
        from pyraquant_amd.adapters import _load_adapt

        _load_adapt()(x, y, i, bank.lr_Af.requires_grad_(), bank.lr_Bf, bank.scale, 8, True, None)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            tuned(torch.autograd.forward_ad.make_dual(x, x), y, i)
    v = x.clone().requires_grad_()
    out = tuned(v, y, i)
    dx, dA = torch.autograd.grad(out, (v, tuned.lr_A), y, create_graph=True)
    for g, wrt in ((dx, tuned.lr_A), (dx, tuned.lr_B), (dA, v), (dA, tuned.lr_B)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(g.float().square().sum(), wrt, retain_graph=True)
    out = tuned(v, y, i)
    i.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_same_bits_streams_and_graphs(cuda):
    """The same bits every time, on another stream, in replays whose ids, factors and scales are others than the captured ones, and in two
    graphs replayed in turn; a captured backward pass."""
    M, K, N, slots, R = 300, 520, 264, 4, 24
    x, y, i, A, B, scale = _problem(M, K, N, slots, R, torch.bfloat16, "runs", seed=7)
    dy = torch.randn(M, N, device=cuda).bfloat16()
    bank, tuned = _bank(A, B, scale), _bank(A, B, scale, trainable=True)
    v = x.clone().requires_grad_()

    def both(m, ids):
        out = tuned(v, y, ids)
        return (out.detach(), *torch.autograd.grad(out, (v, tuned.lr_A, tuned.lr_B), dy))

    first = both(tuned, i)
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(first, both(tuned, i)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = both(tuned, i)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, there))
    ids = i.clone()
    graphs = []
    for call in (lambda: (bank(x, y, ids),), lambda: both(tuned, ids)):
        with torch.set_grad_enabled(bool(graphs)):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = call()
        graphs.append((graph, outs))
    for k in range(4):
        new = torch.randint(-1, slots, (M,), device=cuda) if k % 2 else torch.sort(torch.randint(-1, slots, (M,), device=cuda)).values
        ids.copy_(new)
        at = (A[k] * 0.5 + k, B[k] - k, 0.25 + k)
        bank.set(k, *at)
        tuned.set(k, *at)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(graphs[0][1][0], bank(x, y, ids.clone()))
        assert all(torch.equal(a, b) for a, b in zip(graphs[1][1], both(tuned, ids.clone())))


def test_captured_training_step(cuda):
    """A backward pass that accumulates, captured: replays add the same gradients; one that would meet an eager graph of the same leaves is
    refused before anything runs, through views and casts of them too."""
    n, each, K, N, slots, R = 3, 50, 136, 72, 4, 8
    x, y, _, A, B, scale = _problem(n * each, K, N, slots, R, torch.bfloat16, "runs", seed=5)
    ids = torch.tensor([2, -1, 0], device=cuda)
    dy = torch.randn(n, each, N, device=cuda).bfloat16()
    for dtype in (torch.bfloat16, torch.float32):
        tuned = _bank(A.to(dtype), B.to(dtype), scale, trainable=True)
        leaves = [x.clone().requires_grad_(), tuned.lr_A, tuned.lr_B]

        def step():
            tuned(leaves[0].view(n, each, K), y.view(n, each, N), ids).backward(dy)

        step()
        want = [v.grad.clone() for v in leaves]
        kept = tuned(leaves[0].view(n, each, K), y.view(n, each, N), ids)
        with pytest.raises(RuntimeError, match="outside the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
        del kept
        for v in leaves:
            v.grad.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for k in range(3):
            for v in leaves:
                v.grad.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(v.grad, w) for v, w in zip(leaves, want))
            _bank(A, B, scale)(x, y, ids.repeat_interleave(each))      # (eager work between)


def test_places_past_32_bits(cuda):
    """Rows beyond 2^31 values of y, then of x: the last rows answer as alone, forward and back, and the others too by their sums."""
    M, slots, R = 270000, 2, 8
    for K, N in ((64, 8192), (8192, 64)):
        g = torch.Generator(device="cuda").manual_seed(K)
        x = torch.randn(M, K, generator=g, device=cuda, dtype=torch.bfloat16).requires_grad_()
        y = torch.zeros(M, N, device=cuda, dtype=torch.bfloat16)
        A = torch.randn(slots, K, R, generator=g, device=cuda).bfloat16()
        B = torch.randn(slots, R, N, generator=g, device=cuda).bfloat16()
        ids = torch.zeros(M, dtype=torch.int32, device=cuda)
        ids[-100:] = 1
        ids[1000:1010] = -1
        scale = torch.ones(slots, device=cuda)
        bank = _bank(A, B, scale, trainable=True)
        out = bank(x, y, ids)
        dy = torch.zeros_like(y)
        dy[-100:] = 1
        dx, dA, dB = torch.autograd.grad(out, (x, bank.lr_A, bank.lr_B), dy)
        want, off = _want(x[-100:].detach(), y[-100:], ids[-100:], A, B, scale, dy[-100:])
        _near(out[-100:].detach(), want["y"], off["y"], "y")
        _near(dx[-100:], want["dx"], off["dx"], "dx")
        _near(dA, want["dA"], off["dA"], "dA")
        _near(dB, want["dB"], off["dB"], "dB")
        assert not out[1000:1010].any() and not dx[: -100].any()
        mid = slice(M // 2, M // 2 + 64)
        want, off = _want(x[mid].detach(), y[mid], ids[mid], A, B, scale)
        _near(out[mid].detach(), want["y"], off["y"], "y")
        del out, dy, dx, y, x


def test_kernels_write_what_they_say(cuda):
    """Through the C ABI, with guards around every output: parts only in rows with an adapter, gradients and orders whole."""
    from pyraquant_amd import _lib
    from pyraquant_amd.adapters import _down_axes, _up_axes

    L = _lib.load()
    for (M, K, N, slots, R), ids in itertools.product(((70, 264, 136, 3, 20), (1, 8, 8, 1, 1), (333, 72, 1032, 2, 64)), ("rows", "runs")):
        x, y, i, A, B, scale = _problem(M, K, N, slots, R, torch.bfloat16, ids, seed=K)
        P = 16 if R <= 16 else 32 if R <= 32 else 64
        p, stream = _lib.ptr, _lib.stream_of(x.device)

        def guarded(n, dtype):
            t = torch.full((n + 256,), 7.0 if dtype.is_floating_point else 7, dtype=dtype, device=cuda)
            return t, t[128:128 + n]

        def whole(*pairs):
            torch.cuda.synchronize()
            for t, _ in pairs:
                assert bool((t[:128] == 7).all()) and bool((t[-128:] == 7).all())

        size = L.pq_adapter_factor_size
        ad, au, bd, bu = (guarded(slots * size(c, P), torch.bfloat16) for c in (K, K, N, N))
        _lib.check(L.pq_adapter_factors(p(A), 0, p(B), 1, slots, K, N, R, P, p(ad[1]), p(au[1]), p(bd[1]), p(bu[1]), stream), "factors")
        whole(ad, au, bd, bu)
        for f, axes, m in ((ad, _down_axes, A), (au, _up_axes, A), (bd, _down_axes, B.transpose(1, 2)), (bu, _up_axes, B.transpose(1, 2))):
            v = f[1].view(slots, -1, P)
            v = axes(v).reshape(v.shape)
            assert torch.equal(v[:, : m.shape[1], :R], m) and not v[:, m.shape[1]:].any() and not v[:, :, R:].any()
        again = [guarded(slots * size(c, P), torch.bfloat16) for c in (K, K, N, N)]      # from these orders, and by the other natural one
        _lib.check(L.pq_adapter_factors(p(ad[1]), 2, p(bu[1]), 3, slots, K, N, P, P, *(p(t[1]) for t in again), stream), "factors")
        whole(*again)
        assert all(torch.equal(x[1], y[1]) for x, y in zip(again, (ad, au, bd, bu)))
        At, Bt = A.transpose(1, 2).contiguous(), B.transpose(1, 2).contiguous()
        _lib.check(L.pq_adapter_factors(p(At), 1, p(Bt), 0, slots, K, N, R, P, *(p(t[1]) for t in again), stream), "factors")
        assert all(torch.equal(x[1], y[1]) for x, y in zip(again, (ad, au, bd, bu)))
        S, Sd = L.pq_adapter_slices(M, K), L.pq_adapter_slices(M, N)
        t, dt = guarded(S * M * P, torch.float32), guarded(Sd * M * P, torch.float32)
        dy = torch.randn(M, N, device=cuda).bfloat16()
        _lib.check(L.pq_adapter_down(p(x), 0, M, K, K, p(ad[1]), slots, P, p(i), 32, 1, p(t[1]), stream), "down")
        _lib.check(L.pq_adapter_down(p(dy), 0, M, N, N, p(bd[1]), slots, P, p(i), 32, 1, p(dt[1]), stream), "down")
        whole(t, dt)
        none = (i < 0) | (i >= slots)
        assert bool((t[1].view(S, M, P)[:, none] == 7).all())
        dx, dA, dB = guarded(M * K, torch.bfloat16), guarded(slots * K * R, torch.bfloat16), guarded(slots * R * N, torch.bfloat16)
        tj, dtj, alone = (guarded(M * P, torch.float32) for _ in range(3))
        up = lambda parts, n, g, C, out, joined: _lib.check(L.pq_adapter_up(   # noqa: E731
            p(parts[1]), n, p(scale), g, slots, C, R, P, p(i), 32, 1, None, 0, out, C, p(joined[1]), 0, M, stream), "up")
        up(t, S, None, N, None, tj)
        up(dt, Sd, p(au[1]), K, p(dx[1]), dtj)
        up(dt, Sd, None, K, None, alone)
        whole(tj, dtj, alone)
        assert torch.equal(alone[1], dtj[1]) and bool((tj[1].view(M, P)[none] == 7).all()) and not tj[1].view(M, P)[~none][:, R:].any()
        # both products in one launch
        y1, dx1, t1, dt1, t2 = guarded(M * N, torch.bfloat16), guarded(M * K, torch.bfloat16), *(guarded(M * P, torch.float32) for _ in range(3))
        one = lambda v, C, f, g, D, base, out, joined: _lib.check(L.pq_adapter_rows(   # noqa: E731
            p(v), 0, M, C, C, p(f[1]), p(scale), p(g[1]), slots, D, R, P, p(i), 32, 1, p(base), D, p(out[1]) if out else None, D, p(joined[1]), stream), "rows")
        one(x, K, ad, bu, N, y, y1, t1)
        one(dy, N, bd, au, K, None, dx1, dt1)
        one(x, K, ad, bu, N, None, None, t2)
        whole(y1, dx1, t1, dt1, t2)
        assert torch.equal(t1[1], t2[1]) and bool((t1[1].view(M, P)[none] == 7).all()) and not t1[1].view(M, P)[~none][:, R:].any()
        want, off = _want(x, y, i, A, B, scale, dy)
        _near(y1[1].view(M, N), want["y"], off["y"], "y")
        _near(dx1[1].view(M, K), want["dx"], off["dx"], "dx")
        assert torch.equal(y1[1].view(M, N)[none], y[none]) and not dx1[1].view(M, K)[none].any()
        room = L.pq_adapter_grads_workspace_size(M, K, N, slots, P, 1)
        ws = torch.full((room + 256,), 255, dtype=torch.uint8, device=cuda)
        _lib.check(L.pq_adapter_grads(p(x), K, p(dy), N, 0, p(tj[1]), p(dtj[1]), p(i), 32, 1, M, K, N, slots, R, P, p(dA[1]), p(dB[1]), p(ws), room,
                                      stream), "grads")
        whole(dx, dA, dB)
        assert bool((ws[room:] == 255).all())
        want, off = _want(x, y, i, A, B, scale, dy)
        for got, k in ((dx, "dx"), (dA, "dA"), (dB, "dB")):
            _near(got[1].view(want[k].shape), want[k], off[k], k)


@pytest.mark.parametrize("kind", ("int8", "mxfp4", "linear", "split"))
def test_layers_with_adapters(cuda, kind):
    """What a layer with adapters answers is the layer's own result with theirs added; nothing chosen, the layer's own; gradients of the input
    through a 4-bit layer and its adapters together."""
    from pyraquant_amd import Mxfp4Linear, add_adapters, convert_linears_to_int8, convert_linears_to_mxfp4
    from pyraquant_amd.weights import SplitInLinear

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(256, 512), torch.nn.GELU(), torch.nn.Linear(512, 256)).to(cuda, torch.bfloat16)
    if kind == "split":
        net[2] = SplitInLinear(net[2], 256)
    if kind in ("int8", "split"):
        convert_linears_to_int8(net, whitelist=lambda n: False)
    if kind == "mxfp4":
        convert_linears_to_mxfp4(net, whitelist=lambda n: False)
    net.requires_grad_(False)
    styles = add_adapters(net, 3, 8, whitelist=lambda n: False)
    assert sorted(styles.layers) == ["0", "2"]
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: (torch.randn(*s, generator=g, device=cuda) * 0.05).bfloat16()   # noqa: E731
    styles.set(0, {"0": (r(256, 8), r(8, 512)), "2": (r(512, 4), r(4, 256))})
    styles.set(2, {"2": (r(512, 8), r(8, 256))}, 0.5)
    x = torch.randn(4, 50, 256, device=cuda).bfloat16()
    ids = torch.tensor([2, -1, 0, 1], device=cuda)
    with torch.no_grad():
        plain = net(x)
        with styles.use(ids):
            got = net(x)
        h = net[0].layer(x)
        h = styles.layers["0"](x, h, ids)
        h = net[1](h)
        want = styles.layers["2"](h, net[2].layer(h), ids)
        assert torch.equal(got, want) and torch.equal(got[1], plain[1]) and torch.equal(got[3], plain[3]) and not torch.equal(got[0], plain[0])
        assert torch.equal(net(x), plain)
        # one request's answer does not depend on the others
        with styles.use(torch.tensor([2, 2, 0, 0], device=cuda)):
            assert torch.equal(net(x)[0], got[0]) and torch.equal(net(x)[2], got[2])
    if kind == "mxfp4":
        v = x.clone().requires_grad_()
        with styles.use(ids):
            out = net[0](v)
        dy = torch.randn_like(out)
        dx, = torch.autograd.grad(out, v, dy)
        w = v.detach().clone().requires_grad_()
        base, = torch.autograd.grad(net[0].layer(w), w, dy)
        own, = torch.autograd.grad(styles.layers["0"](w, torch.zeros_like(dy), ids), w, dy)
        assert torch.equal(dx, base + own) and isinstance(net[0].layer, Mxfp4Linear)


@pytest.mark.parametrize("bits", (32, 8))
def test_tuned_together_and_served_together(cuda, bits):
    """Three adapters tuned at once beside 4-bit layers, each on requests of its own: every step's gradients are those that the adapter gets
    alone, AdamW steps them all, and the frozen ones answer mixed batches as the tuned ones did."""
    from pyraquant_amd import AdamW, add_adapters, convert_linears_to_mxfp4

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(128, 256), torch.nn.GELU(), torch.nn.Linear(256, 128)).to(cuda, torch.bfloat16)
    convert_linears_to_mxfp4(net, whitelist=lambda n: False)
    styles = add_adapters(net, 3, 8, dtype=torch.float32, trainable=True, whitelist=lambda n: False)
    for s in range(3):
        styles.set(s, {n: (torch.randn(b.in_features, 8, device=cuda) * 0.05, torch.randn(8, b.out_features, device=cuda) * 0.05) for n, b in styles.layers.items()})
    assert len(styles.parameters()) == 4 and all(p.requires_grad for p in styles.parameters())
    opt = AdamW(styles.parameters(), lr=1e-3, bits=bits, max_norm=1.0)
    ids = torch.tensor([0, 1, 2, 1], device=cuda)
    start = [p.detach().clone() for p in styles.parameters()]
    for step in range(5):
        x = torch.randn(4, 64, 128, device=cuda).bfloat16()
        target = torch.randn(4, 64, 128, device=cuda).bfloat16()
        with styles.use(ids):
            loss = (net(x).float() - target.float()).square().mean()
        opt.zero_grad()
        loss.backward()
        if step == 0:
            together = [p.grad.clone() for p in styles.parameters()]
            with styles.use(torch.tensor([0, -1, -1, -1], device=cuda)):
                (net(x).float() - target.float()).square()[0].sum().div(target.numel()).backward(inputs=styles.parameters())
            for p, g in zip(styles.parameters(), together):
                alone = p.grad[0] - g[0]
                assert float((alone - g[0]).norm()) <= 0.02 * float(g[0].norm())     # (sums of the same terms, each rounded to bf16 twice)
                p.grad = g
        opt.step()
        assert float(opt.grad_norm) > 0
    assert all(not torch.equal(a, b) for a, b in zip(start, styles.parameters()))
    x = torch.randn(4, 64, 128, device=cuda).bfloat16()
    with torch.no_grad(), styles.use(torch.tensor([2, 0, -1, 1], device=cuda)):
        tuned = net(x)
        styles.freeze(torch.bfloat16)
        assert torch.equal(net(x), tuned)
