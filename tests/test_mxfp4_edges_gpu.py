"""Microscaled 4-bit layers where a wrong or a lost result would go unseen by a comparison at ordinary values: what is held in
between, values at the ends of their types, every choice of operands and of what is wanted.

Bounds as in test_mxfp4_gpu: u is the unit roundoff of the 16-bit type with half a place to spare (2^-8 for bf16, 2^-11 for fp16), a
sum of n products in fp32 is within n 2^-23 of the sum of the magnitudes of its terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BOTH = (torch.bfloat16, torch.float16)
F = 2.0 ** -23


def _layer(K, N, R, dtype, seed, std=0.3, bias=False, weight=0.0, factors=None, trainable=True):
    """A layer whose weight is N(0, weight) (all zeros by default: what it computes is its low-rank branch) and its factors."""
    from pyraquant_amd.mxfp4 import Mxfp4Linear

    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(K, N, bias=bias)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * weight)
        if bias:
            lin.bias.copy_(torch.randn(N, generator=g))
    A, B = ((torch.randn(*s, generator=g) * std).to(factors or dtype).cuda() for s in ((K, R), (R, N))) if R else (None, None)
    return Mxfp4Linear(lin.to(dtype), device="cuda", lowrank=(A, B) if R else None, trainable=trainable), A, B


def _rand(*shape, dtype, seed, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


# ---- what is held in between ----------------------------------------------------------------------------------------

def _through(x, A, B, dtype):
    """(x A) B in 64 bits, and how far from it a result may be whose x A lost no more than u^2 of itself: twice the type's bits
    (in fp16, and 2^-25: its subnormals' half place)."""
    u, small = U[dtype], 2.0 ** -25 if dtype == torch.float16 else 0.0
    x, A, B = x.double(), A.double(), B.double()
    t = x @ A
    lost = x.shape[1] * F * (x.abs() @ A.abs())
    t_off = lost + u * u * (t.abs() + lost) + small
    y = t @ B
    off = t_off @ B.abs() + 2 * (A.shape[1] + 2) * F * ((t.abs() + t_off) @ B.abs())
    return y, off + u * (y.abs() + off) + small


# rows quantized inside the product; a split product; blocks of 128 x 64, of 128 x 64 in three groups, of 128 x 256 and of 256 x
# 256; and with them the input gradient in both kinds of block, whole and in slices
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N,R", [(20, 64, 96, 8), (154, 2048, 1280, 32), (300, 640, 5120, 64), (329, 4320, 2512, 40), (600, 1056, 7056, 64),
                                     (2100, 160, 4112, 64), (4200, 416, 4208, 32), (4128, 2080, 496, 32), (2050, 1312, 5136, 64),
                                     (40, 96, 4112, 33)])
def test_low_rank_terms_lose_nothing_in_between(cuda, dtype, M, K, N, R):
    """Over a weight of zeros y is (x A) B and dx is (dy B^T) A^T: sums of mixed signs, most of them far smaller than their terms,
    so a rounding of x A or dy B^T to 16 bits on the way would show."""
    layer, A, B = _layer(K, N, R, dtype, K + N, std=0.1)
    x, dy = _rand(M, K, dtype=dtype, seed=M).requires_grad_(), _rand(M, N, dtype=dtype, seed=N)
    y = layer(x)
    dx, = torch.autograd.grad(y, x, dy)
    _within(y.detach(), *_through(x.detach(), A, B, dtype), "y")
    _within(dx, *_through(dy, B.t(), A.t(), dtype), "dx")
    layer.freeze()
    with torch.no_grad():
        assert torch.equal(layer(x), y)


@pytest.mark.parametrize("dtype", BOTH)
def test_32_bit_low_rank_operands(cuda, dtype):
    """mxfp4_gemm and mxfp4_grad_input take t and dt in fp32 as the layer's own calls do, rows with a stride among them, and
    lowrank_grads takes them in fp32 or as two parts that add up to it."""
    from pyraquant_amd.mxfp4 import lowrank_grads, mxfp4_gemm, mxfp4_grad_input, quant_mxfp4

    M, K, N, R = 70, 96, 80, 32
    x, w, dy = _rand(M, K, dtype=dtype, seed=1), torch.zeros(N, K, device=cuda), _rand(M, N, dtype=dtype, seed=2)
    wide = _rand(M, 36, dtype=torch.float32, seed=3)
    t, l2t, ap = wide[:, :32], _rand(N, R, dtype=dtype, seed=4), _rand(K, R, dtype=dtype, seed=5)
    xq, q8 = quant_mxfp4(x, checkpoint=True)
    wq = quant_mxfp4(w)
    u, small = U[dtype], 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, l in ((mxfp4_gemm(xq, wq, None, dtype, t=t, l2t=l2t), l2t), (mxfp4_grad_input(dy, wq, t.contiguous(), ap), ap)):
        want, terms = t.double() @ l.double().t(), t.double().abs() @ l.double().abs().t()
        off = (u * u + 2 * R * F) * terms + small * l.double().abs().sum(1)
        _within(got, want, off + u * (want.abs() + off) + small, "low-rank term")
    parts = [torch.stack([v.to(dtype), (v - v.to(dtype).float()).to(dtype)]) for v in (t, wide[:, 4:])]
    whole = [p[0].float() + p[1].float() for p in parts]
    a, b = (lowrank_grads(dy, *v, q8, xq.scales, 20) for v in (parts, whole))
    assert all(torch.equal(g, h) for g, h in zip(a, b)) and a[0].dtype == a[1].dtype == dtype


def test_lowrank_grads_checks_both_operands(cuda):
    """t and dt are read through raw pointers: another type or shape of either is refused, whatever is wanted."""
    from pyraquant_amd.mxfp4 import lowrank_grads, quant_mxfp4

    dy, (q, q8) = _rand(4, 32, dtype=torch.bfloat16, seed=1), quant_mxfp4(_rand(4, 64, dtype=torch.bfloat16, seed=2), checkpoint=True)
    good = torch.zeros(2, 4, 32, dtype=torch.bfloat16, device=cuda)
    for bad in (good.float(), good.half(), good[:1], good[:, :, :16], good[:, :3], good[0]):
        with pytest.raises(AssertionError):
            lowrank_grads(dy, bad, good, q8, q.scales, 8)
        with pytest.raises(AssertionError):
            lowrank_grads(dy, good, bad, q8, q.scales, 8)


# ---- infinities and NaNs ------------------------------------------------------------------------------------------

def _same_kind(got, want, what):
    """NaN, an infinity with its sign, or finite: as want is."""
    got = got.detach().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in {int(torch.isnan(got).sum())}, not in {int(torch.isnan(want).sum())} values"
    assert torch.equal(torch.where(torch.isinf(got), got, 0.0).nan_to_num(0, 1, -1), torch.where(torch.isinf(want), want, 0.0).nan_to_num(0, 1, -1)), what


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N,R", [(20, 64, 96, 8), (90, 128, 48, 33), (300, 640, 1040, 64), (2100, 160, 4112, 32), (4128, 2080, 496, 32)])
def test_infinities_stay_infinities(cuda, dtype, M, K, N, R):
    """An infinity in x, dy or a factor gives what the formulas give: infinities of the products' signs, NaN where it meets a zero
    or the other sign. Rows of one or two values make some of t and dt 16-bit values, with nothing left for a second part."""
    from pyraquant_amd.mxfp4 import checkpoint_values, dequant_mxfp4, quant_mxfp4

    layer, A, B = _layer(K, N, R, dtype, K, weight=0.1, std=0.5)
    x, dy = _rand(M, K, dtype=dtype, seed=M), _rand(M, N, dtype=dtype, seed=N)
    x[: M // 2] = torch.where(torch.arange(K, device=cuda) == torch.arange(M // 2, device=cuda).unsqueeze(1) % K, 1.0, 0.0)
    dy[M // 4 : M // 2] = torch.where(torch.arange(N, device=cuda) == torch.arange(M // 2 - M // 4, device=cuda).unsqueeze(1) % N, -0.5, 0.0)
    inf = float("inf")
    for name in ("dy", "x", "A", "B"):
        v = {"x": x.clone(), "dy": dy.clone(), "A": A.clone(), "B": B.clone()}
        for i, j, value in ((1, 3, inf), (M // 3, 17, -inf), (M - 1, 40, inf)):
            rows = v[name].shape[0]
            v[name][i % rows, j % v[name].shape[1]] = value
        with torch.no_grad():
            layer.lr_A.copy_(v["A"])
            layer.lr_B.copy_(v["B"])
        xg = v["x"].requires_grad_()
        y = layer(xg)
        dx, dA, dB = torch.autograd.grad(y, [xg, layer.lr_A, layer.lr_B], v["dy"])
        q, q8 = quant_mxfp4(v["x"].detach(), checkpoint=True)
        X, D, a, b, w = v["x"].detach().double(), v["dy"].double(), v["A"].double(), v["B"].double(), layer.weight(torch.float32).double()
        t, dt = X @ a, D @ b.t()
        want = {"y": dequant_mxfp4(q, torch.float32).double() @ w.t() + t @ b, "dx": D @ w + dt @ a.t(),
                "dA": checkpoint_values(q8, q, torch.float32).double().t() @ dt, "dB": t.t() @ D}
        for k, got in (("y", y), ("dx", dx), ("dA", dA), ("dB", dB)):
            _same_kind(got, want[k], f"{k} of an infinite {name}")


# ---- past the end of fp16 -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,K,N,R", [(20, 64, 96, 8), (90, 128, 48, 33), (300, 640, 1040, 64), (2100, 160, 4112, 32), (4128, 2080, 496, 32),
                                     (329, 4320, 2512, 40), (600, 1056, 7056, 64)])
@pytest.mark.parametrize("which", ("t", "dt"))
def test_low_rank_values_past_fp16(cuda, which, M, K, N, R):
    """x A (or dy B^T) of some 10^5 to 10^7 in most rows and of 1 in others, results inside fp16: they are as exact as elsewhere. A
    row's (in sums over rows, a rank's) values share a scale, so that 2^-25 of 2^15 below its largest may be missing."""
    from pyraquant_amd.mxfp4 import checkpoint_values, quant_mxfp4

    dtype, u, tiny = torch.float16, U[torch.float16], 2.0 ** -25
    large, small = 16000.0, 1e-3 / R ** 0.5
    g = torch.Generator().manual_seed(K)
    layer, *_ = _layer(K, N, R, dtype, 1)
    A = (torch.randn(K, R, generator=g) * (large / K ** 0.5 if which == "t" else small)).half().cuda()
    B = (torch.randn(R, N, generator=g) * (small if which == "t" else large / N ** 0.5)).half().cuda()
    with torch.no_grad():
        layer.lr_A.copy_(A)
        layer.lr_B.copy_(B)
    x, dy = (torch.randn(M, n, generator=g) for n in (K, N))
    far, near = (x, dy) if which == "t" else (dy, x)
    far *= 30.0
    far[::8] *= 10.0
    far[3::8] *= 1e-5
    near *= 0.002 / M ** 0.5
    x, dy = x.half().cuda().requires_grad_(), dy.half().cuda()
    y = layer(x)
    dx, dA, dB = torch.autograd.grad(y, [x, layer.lr_A, layer.lr_B], dy)
    q, q8 = quant_mxfp4(x.detach(), checkpoint=True)
    X, D, a, b = x.detach().double(), dy.double(), A.double(), B.double()
    xt = checkpoint_values(q8, q, torch.float32).double()

    def through(X, a, b):     # (X a) b and its bound, X a and its bounds as rows and as columns share scales
        t = X @ a
        lost = X.shape[1] * F * (X.abs() @ a.abs())
        off = [lost + u * u * (t.abs() + lost) + tiny * (t.abs().amax(d, keepdim=True) * 2.0 ** -15).clamp_min(1) for d in (1, 0)]
        want = t @ b
        bound = off[0] @ b.abs() + 2 * (R + 2) * F * ((t.abs() + off[0]) @ b.abs())
        return want, bound + u * (want.abs() + bound) + tiny, t, off[1]

    def summed(z, t, off):    # z^T t
        want, bound = z.t() @ t, z.abs().t() @ off + 2 * M * F * (z.abs().t() @ (t.abs() + off))
        return want, bound + u * (want.abs() + bound) + tiny

    y_want, y_bound, t, t_off = through(X, a, b)
    dx_want, dx_bound, dt, dt_off = through(D, b.t(), a.t())
    assert float((t if which == "t" else dt).abs().max()) > 1e6 and float(torch.stack([v.abs().max() for v in (y_want, dx_want)]).max()) < 6e4
    _within(y.detach(), y_want, y_bound, "y")
    _within(dx, dx_want, dx_bound, "dx")
    _within(dA, *summed(xt, dt, dt_off), "dA")
    want, bound = summed(D, t, t_off)
    _within(dB, want.t(), bound.t(), "dB")


# ---- autograd beyond a first derivative ---------------------------------------------------------------------------

def test_second_derivatives_raise(cuda):
    """A pass with create_graph gives the same gradients, and differentiating one that depends on what requires a gradient raises:
    never a sum in which this layer's part is missing."""
    dtype = torch.bfloat16
    layer, *_ = _layer(64, 32, 8, dtype, 1, weight=0.1, bias=True)
    x0, scale, dy = _rand(5, 64, dtype=dtype, seed=1), _rand(64, dtype=dtype, seed=2).requires_grad_(), _rand(5, 32, dtype=dtype, seed=3)
    wanted = lambda x: [x, layer.lr_A, layer.lr_B, layer.bias]   # noqa: E731
    x = x0.clone().requires_grad_()
    first = torch.autograd.grad(layer(x), wanted(x), dy)
    grads = torch.autograd.grad(layer(x), wanted(x), dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, grads))
    on = {0: [1, 2], 1: [0, 2], 2: [0, 1], 3: []}      # what each depends on (dy, too, which requires none here)
    for i, g in enumerate(grads):
        assert g.requires_grad == bool(on[i])
        for j in on[i]:
            with pytest.raises(RuntimeError, match="second derivatives"):
                torch.autograd.grad(g.float().square().sum() + wanted(x)[j].float().sum(), wanted(x)[j], retain_graph=True)
    # a gradient penalty through an operation before the layer: the sum of both losses
    y = layer(x * scale)
    dx, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    for wrt in (None, [scale], [x, layer.lr_A]):
        loss = y.float().sum() + dx.float().square().sum()
        with pytest.raises(RuntimeError, match="second derivatives"):
            loss.backward(retain_graph=True) if wrt is None else torch.autograd.grad(loss, wrt, retain_graph=True)
    # nothing that requires a gradient besides x: dx is a constant, and a gradient of dy makes it none
    frozen, *_ = _layer(64, 32, 8, dtype, 1, weight=0.1, trainable=False)
    y = frozen(x)
    assert not torch.autograd.grad(y, x, dy, create_graph=True)[0].requires_grad
    d = dy.clone().requires_grad_()
    dx, = torch.autograd.grad(frozen(x), x, d, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(dx.float().sum(), d)


def test_forward_mode_tangents_raise(cuda):
    """A tangent of x, of a factor or of the bias is never dropped, with or without gradients of the reverse kind."""
    import torch.autograd.forward_ad as fwd

    for trainable in (True, False):
        layer, *_ = _layer(64, 32, 8, torch.bfloat16, 1, weight=0.1, bias=True, trainable=trainable)
        x = _rand(5, 64, dtype=torch.bfloat16, seed=1)
        want = layer(x)
        with fwd.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    layer(fwd.make_dual(x, torch.ones_like(x)))
            if not trainable:
                for name in ("bias", "lr_Af", "lr_Bt"):
                    kept = layer._buffers[name]
                    layer._buffers[name] = fwd.make_dual(kept, torch.ones_like(kept))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        layer(x)
                    layer._buffers[name] = kept
            assert torch.equal(layer(x), want)
        assert torch.equal(layer(x), want)


# ---- every choice of operands -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", BOTH)
def test_lowrank_grads_of_every_choice(cuda, dtype):
    """Each choice of what is wanted, with None for what it does not need: the values that all of them together have."""
    from pyraquant_amd.mxfp4 import lowrank_grads, quant_mxfp4

    M, K, N, rank = 150, 96, 80, 20
    dy, (q, q8) = _rand(M, N, dtype=dtype, seed=1), quant_mxfp4(_rand(M, K, dtype=dtype, seed=2), checkpoint=True)
    t, dt = (torch.nn.functional.pad(_rand(M, rank, dtype=torch.float32, seed=s), (0, 12)) for s in (3, 4))
    parts = torch.stack([dt.to(dtype), (dt - dt.to(dtype).float()).to(dtype)])
    dt = parts[0].float() + parts[1].float()
    every = lowrank_grads(dy, t, dt, q8, q.scales, rank)
    want = dy.double().sum(0)
    assert bool(((every[2].double() - want).abs() <= M * F * dy.double().abs().sum(0)).all())
    for A in (False, True):
        for B in (False, True):
            for b in (False, True):
                # (without a dy the type of the results is that of dt's parts)
                got = lowrank_grads(dy if B or b else None, t if B else None, (dt if B or b else parts) if A else None, q8 if A else None,
                                    q.scales if A else None, rank, A, B, b)
                for g, e, w in zip(got, every, (A, B, b)):
                    assert (g is None) == (not w) and (g is None or (g.dtype == e.dtype and torch.equal(g, e))), (A, B, b)
    for missing in range(5):
        with pytest.raises(AssertionError):
            lowrank_grads(*[None if i == missing else v for i, v in enumerate((dy, t, dt, q8, q.scales))], rank)


def test_scales_that_are_not_contiguous_are_refused(cuda):
    from pyraquant_amd.mxfp4 import Mxfp4Matrix, checkpoint_values, dequant_mxfp4, lowrank_grads, mxfp4_gemm, quant_mxfp4

    q, q8 = quant_mxfp4(_rand(20, 64, dtype=torch.bfloat16, seed=1), checkpoint=True)
    spread = torch.stack([q.scales, q.scales], 1)[:, 0]
    bad, dt = Mxfp4Matrix(q.codes, spread, q.rows, q.cols), torch.zeros(2, 20, 32, dtype=torch.bfloat16, device=cuda)
    for call in (lambda: lowrank_grads(None, None, dt, q8, spread, 8, True, False, False), lambda: dequant_mxfp4(bad),
                 lambda: checkpoint_values(q8, bad), lambda: mxfp4_gemm(bad, quant_mxfp4(torch.zeros(32, 64, device=cuda)), None, torch.bfloat16)):
        with pytest.raises(AssertionError):
            call()


def test_gradient_of_a_bias_without_a_branch(cuda):
    """A frozen layer's bias buffer that requires a gradient, with and without a low-rank branch and a gradient of x."""
    for R in (0, 8):
        layer, *_ = _layer(64, 48, R, torch.bfloat16, 1, weight=0.1, bias=True, trainable=False)
        layer.bias.requires_grad_()
        dy = _rand(70, 48, dtype=torch.bfloat16, seed=1)
        want, bound = dy.double().sum(0), 70 * F * dy.double().abs().sum(0)
        for x in (_rand(70, 64, dtype=torch.bfloat16, seed=2), _rand(70, 64, dtype=torch.bfloat16, seed=2).requires_grad_()):
            g, *dx = torch.autograd.grad(layer(x), [layer.bias] + [x] * x.requires_grad, dy)
            assert g.dtype == torch.float32
            _within(g, want, bound, "dbias")
        layer.bias.requires_grad_(False)
        assert torch.equal(dx[0], torch.autograd.grad(layer(x), x, dy)[0])


def test_an_assigned_bias_counts(cuda):
    """A bias made a parameter, replaced by one or taken away, on a frozen and on a trainable layer."""
    x, dy = _rand(9, 64, dtype=torch.bfloat16, seed=1), _rand(9, 48, dtype=torch.bfloat16, seed=2)
    for trainable in (False, True):
        layer, *_ = _layer(64, 48, 8, torch.bfloat16, 1, weight=0.1, bias=True, trainable=trainable)
        other, *_ = _layer(64, 48, 8, torch.bfloat16, 1, weight=0.1, bias=True, trainable=trainable)
        value = torch.randn(48, generator=torch.Generator().manual_seed(3)).cuda()
        with torch.no_grad():
            other.bias.copy_(value)
        layer.bias = torch.nn.Parameter(value.clone())
        assert torch.equal(layer(x), other(x)) and "bias" in dict(layer.named_parameters())
        g, = torch.autograd.grad(layer(x), layer.bias, dy)
        _within(g, dy.double().sum(0), 9 * F * dy.double().abs().sum(0), "dbias")
        layer.bias = None
        with torch.no_grad():
            other.bias.zero_()
        assert torch.equal(layer(x), other(x))


def test_factors_in_the_kernels_order_take_no_gradient(cuda):
    """lr_Af and lr_Bt are a permutation of padded factors: a gradient in lr_A's own order would be wrong for them."""
    for K in (64, 128):
        layer, *_ = _layer(K, 48, 32, torch.bfloat16, 1, weight=0.1, trainable=False)
        x = _rand(9, K, dtype=torch.bfloat16, seed=1)
        want = layer(x)
        for name in ("lr_Af", "lr_Bt"):
            getattr(layer, name).requires_grad_()
            with pytest.raises(AssertionError):
                layer(x)
            with torch.no_grad():
                assert torch.equal(layer(x), want)
            getattr(layer, name).requires_grad_(False)


# ---- conversion ---------------------------------------------------------------------------------------------------

def test_layers_that_are_not_taken_stay(cuda):
    """A branch of rank 65 or 0, 64-bit weights, sizes that do not fit, in the middle of a model: kept, and the rest converted."""
    from pyraquant_amd.mxfp4 import Mxfp4Linear, convert_linears_to_mxfp4

    for trainable in (False, True):
        lins = [torch.nn.Linear(64, 64).bfloat16() for _ in range(4)] + [torch.nn.Linear(64, 64).double(), torch.nn.Linear(60, 64).bfloat16(),
                                                                            torch.nn.Linear(64, 24).bfloat16()]
        for lin, rank in zip(lins, (64, 65, 0)):
            lin._lowrank_A, lin._lowrank_B = torch.zeros(64, rank).bfloat16(), torch.zeros(rank, 64).bfloat16()
        net = torch.nn.Sequential(*lins)
        stats = convert_linears_to_mxfp4(net, trainable=trainable)
        assert [isinstance(m, Mxfp4Linear) for m in net] == [True, False, False, True, False, False, False]
        assert stats["n_mxfp4_linear"] == 2 and stats["n_bf16_linear_kept"] == 5 and stats["bf16_kept_names"] == ["1", "2", "4", "5", "6"]


# ---- many rows ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,K", [(65536 * 64 + 70, 32), (65536 * 64 + 1, 96)])
def test_input_gradient_of_millions_of_rows(cuda, M, K):
    """More blocks of rows than a grid's second dimension counts."""
    from pyraquant_amd.mxfp4 import dequant_mxfp4, mxfp4_grad_input, quant_mxfp4

    N, R, u = 16, 32, U[torch.bfloat16]
    g = torch.Generator(device=cuda).manual_seed(M)
    dy = torch.randn(M, N, generator=g, device=cuda, dtype=torch.bfloat16)
    dt, ap = torch.randn(M, R, generator=g, device=cuda), torch.randn(K, R, generator=g, device=cuda).bfloat16()
    wq = quant_mxfp4(torch.randn(N, K, generator=g, device=cuda))
    wh = dequant_mxfp4(wq, torch.float32).double()
    got = mxfp4_grad_input(dy, wq, dt, ap)
    for r in range(0, M, 1 << 19):
        d, t = dy[r : r + (1 << 19)].double(), dt[r : r + (1 << 19)].double()
        want, terms = d @ wh + t @ ap.double().t(), d.abs() @ wh.abs() + t.abs() @ ap.double().abs().t()
        off = ((N + 2 * R) * F + u * u) * terms
        _within(got[r : r + (1 << 19)], want, off + u * (want.abs() + off), f"dx from row {r}")


# ---- freezing -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("a_type,b_type", [(torch.float32,) * 2, (torch.bfloat16,) * 2, (torch.float16,) * 2, (torch.bfloat16, torch.float32),
                                           (torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
def test_frozen_layers_answer_as_the_tuned_ones(cuda, dtype, a_type, b_type):
    """Factors of any type, inputs of either: a trainable layer, frozen, gives the same bits, and so does one built frozen; lr_A and
    lr_B come back as they were."""
    from pyraquant_amd.mxfp4 import Mxfp4Linear

    for K, N, R in ((128, 48, 16), (416, 80, 40)):
        g = torch.Generator().manual_seed(K)
        A, B = (torch.randn(K, R, generator=g) * 0.1).to(a_type).cuda(), (torch.randn(R, N, generator=g) * 0.1).to(b_type).cuda()
        lin = torch.nn.Linear(K, N).to(dtype)
        layer = Mxfp4Linear(lin, device="cuda", lowrank=(A, B), trainable=True)
        x = _rand(70, K, dtype=dtype, seed=1)
        with torch.no_grad():
            want = layer(x)
            assert torch.equal(Mxfp4Linear(lin, device="cuda", lowrank=(A, B))(x), want)
            given = Mxfp4Linear(lin, device="cuda", lowrank=(A, B), trainable=True).freeze(dtype)
            assert torch.equal(given(x), want) and given.lr_Af.dtype == given.lr_Bt.dtype == dtype
            layer.freeze()
            assert torch.equal(layer(x), want)
        assert torch.equal(layer.lr_A, A) and torch.equal(layer.lr_B, B) and layer.lr_A.dtype == a_type and layer.lr_B.dtype == b_type


def test_conversion_keeps_factors_in_the_weights_type(cuda):
    from pyraquant_amd.mxfp4 import Mxfp4Linear, convert_linears_to_mxfp4

    for dtype in BOTH:
        lin = torch.nn.Linear(64, 48).to(dtype)
        lin._lowrank_A, lin._lowrank_B = torch.randn(64, 8) * 0.1, torch.randn(8, 48) * 0.1
        net = torch.nn.Sequential(lin)
        convert_linears_to_mxfp4(net)
        assert net[0].lr_Af.dtype == net[0].lr_Bt.dtype == dtype
        x = _rand(9, 64, dtype=dtype, seed=1)
        assert torch.equal(net(x), Mxfp4Linear(lin, device="cuda")(x))


# ---- strides ------------------------------------------------------------------------------------------------------

def test_output_gradients_far_apart(cuda):
    """Rows of dy further apart than the input gradient's kernels address."""
    from pyraquant_amd.mxfp4 import mxfp4_grad_input, quant_mxfp4

    step = 2 ** 21 + 64
    base = torch.zeros(6 * step, dtype=torch.bfloat16, device=cuda)
    far = torch.as_strided(base, (5, 48), (step, 1))
    far.copy_(_rand(5, 48, dtype=torch.bfloat16, seed=1))
    wq = quant_mxfp4(_rand(48, 64, dtype=torch.float32, seed=2))
    assert torch.equal(mxfp4_grad_input(far, wq), mxfp4_grad_input(far.contiguous(), wq))
    layer, *_ = _layer(64, 48, 8, torch.bfloat16, 1, weight=0.1, bias=True)
    x = _rand(5, 64, dtype=torch.bfloat16, seed=3).requires_grad_()
    wanted = [x, layer.lr_A, layer.lr_B, layer.bias]
    for a, b in zip(*(torch.autograd.grad(layer(x), wanted, d) for d in (far, far.contiguous()))):
        assert torch.equal(a, b)


# ---- memory around the outputs, in every kind of block ------------------------------------------------------------

def _framed(M, N, dtype, cuda):
    """An [M, N] window of a larger tensor of sevens, and whether all around it still holds them."""
    big = torch.full((M + 9, N + 24), 7.0, dtype=dtype, device=cuda)
    window = big[4 : 4 + M, 8 : 8 + N]

    def untouched():
        frame = big.clone()
        frame[4 : 4 + M, 8 : 8 + N] = 7.0
        return bool((frame == 7.0).all())

    return window, untouched


# a split product; blocks of 128 x 64, of 128 x 64 in three groups, of 128 x 256 and of 256 x 256, one and several to a workgroup
@pytest.mark.parametrize("M,K,N,R", [(40, 96, 80, 32), (1100, 352, 912, 0), (513, 96, 2064, 64), (329, 4320, 2512, 32), (600, 1056, 7056, 32),
                                     (2100, 160, 4112, 64), (4200, 96, 4208, 32), (8500, 160, 4368, 0)])
def test_products_write_their_output_alone(cuda, M, K, N, R):
    from pyraquant_amd.mxfp4 import dequant_mxfp4, mxfp4_gemm, quant_mxfp4

    for dtype in BOTH:
        g = torch.Generator(device=cuda).manual_seed(M)
        xq, wq = (quant_mxfp4(torch.randn(n, K, generator=g, device=cuda)) for n in (M, N))
        t, bias = torch.randn(M, R, generator=g, device=cuda) if R else None, torch.randn(N, generator=g, device=cuda)
        l2t = torch.randn(N, R, generator=g, device=cuda).to(dtype) if R else None
        out, untouched = _framed(M, N, dtype, cuda)
        mxfp4_gemm(xq, wq, bias, dtype, t=t, l2t=l2t, out=out)
        assert untouched() and torch.equal(out, mxfp4_gemm(xq, wq, bias, dtype, t=t, l2t=l2t))
        xh, wh, u = dequant_mxfp4(xq, torch.float32).double(), dequant_mxfp4(wq, torch.float32).double(), U[dtype]
        want, terms = xh @ wh.t() + bias, xh.abs() @ wh.abs().t() + bias.abs()
        if R:
            want, terms = want + t.double() @ l2t.double().t(), terms + t.double().abs() @ l2t.double().abs().t()
        off = ((K + 2 * R + 2) * F + u * u) * terms + (2.0 ** -25 * l2t.double().abs().sum(1) if R else 0)
        _within(out, want, off + u * (want.abs() + off) + 2.0 ** -25, (dtype, M, K, N))


# 64 x 128 blocks and 256 x 256 blocks, each whole and in slices (slices: whether the call has a workspace)
@pytest.mark.parametrize("M,K,N,slices", [(1000, 1312, 1040, False), (300, 288, 2080, True), (4128, 2080, 496, False), (8300, 1056, 112, False),
                                          (2050, 1312, 5136, True)])
def test_input_gradients_write_their_output_alone(cuda, M, K, N, slices):
    from pyraquant_amd import _lib
    from pyraquant_amd.mxfp4 import dequant_mxfp4, mxfp4_grad_input, quant_mxfp4

    L = _lib.load()
    size = L.pq_mx_grad_input_workspace_size(M, N, K)
    assert (size > 0) == slices
    for dtype in BOTH:
        for R in (0, 32, 64):
            g = torch.Generator(device=cuda).manual_seed(M)
            wq = quant_mxfp4(torch.randn(N, K, generator=g, device=cuda))
            dy = torch.randn(M, N, generator=g, device=cuda).to(dtype)
            dt, ap = (torch.randn(M, R, generator=g, device=cuda), torch.randn(K, R, generator=g, device=cuda).to(dtype)) if R else (None, None)
            dx, untouched = _framed(M, K, dtype, cuda)
            ws = torch.full((size + 256,), 255, dtype=torch.uint8, device=cuda)
            _lib.check(L.pq_mx_grad_input(_lib.ptr(dy), _lib.dtype_code(dtype), N, _lib.ptr(wq.codes), _lib.ptr(wq.scales), _lib.ptr(dt), _lib.ptr(ap),
                                          R, _lib.ptr(dx), dx.stride(0), M, N, K, _lib.ptr(ws), size, _lib.stream_of(dy.device)), "dx")
            assert untouched() and bool((ws[size:] == 255).all())
            assert torch.equal(dx, mxfp4_grad_input(dy, wq, dt, ap))
            wh, u = dequant_mxfp4(wq, torch.float32).double(), U[dtype]
            want, terms = dy.double() @ wh, dy.double().abs() @ wh.abs()
            if R:
                want, terms = want + dt.double() @ ap.double().t(), terms + dt.double().abs() @ ap.double().abs().t()
            off = ((N + 2 * R) * F + u * u) * terms + (2.0 ** -25 * ap.double().abs().sum(1) if R else 0)
            _within(dx, want, off + u * (want.abs() + off) + 2.0 ** -25, (dtype, M, K, N, R))
