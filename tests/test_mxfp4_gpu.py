"""Microscaled 4-bit layers (pyraquant_amd.mxfp4) against their definition in 64 bits (oracle/mxfp4_ref.py).

The values that codes stand for are compared bit for bit. Sums are held to what their arithmetic can lose: with u the unit
roundoff of the 16-bit type (2^-8 for bf16, 2^-11 for fp16: a whole last place, where half a one would do for a single
rounding) and S the sum of the magnitudes of the terms, a sum of n products in fp32 in any order is within n 2^-23 S (twice the
classical bound, for what the matrix instructions lose inside), an intermediate rounded to 16 bits (t, dt) adds u of the
terms that it is part of, and the result's own rounding u of its value."""
import pytest
import torch

from oracle import mxfp4_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BOTH = (torch.bfloat16, torch.float16)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _x(M, K, dtype, seed, std=1.0):
    g = _gen(seed)
    x = torch.randn(M, K, generator=g) * std
    x[:, torch.randperm(K, generator=g)[: max(1, K // 200)]] *= 20
    return x.to(dtype)


def _layer(K, N, R, bias, dtype, seed, trainable=False):
    from pyraquant_amd.mxfp4 import Mxfp4Linear

    g = _gen(seed)
    lin = torch.nn.Linear(K, N, bias=bias)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * 0.02)
        if bias:
            lin.bias.copy_(torch.randn(N, generator=g) * 0.01)
    lin = lin.to(dtype)
    lr = ((torch.randn(K, R, generator=g) * 0.05).to(dtype), (torch.randn(R, N, generator=g) * 0.05).to(dtype)) if R else None
    layer = Mxfp4Linear(lin, device="cuda", lowrank=lr, trainable=trainable)
    b = lin.bias.detach().float() if bias else None
    return layer, lin.weight.detach(), lr or (None, None), b


def _inside(got, want, bound, what):
    """|got - want| <= bound everywhere that want is finite, and NaN where it is NaN"""
    got, bad = got.detach().double().cpu(), torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad), f"{what}: {int((torch.isnan(got) != bad).sum())} values are NaN that should not, or not NaN"
    ratio = ((got - want).abs() / (bound + 1e-30))[~bad]
    assert ratio.numel() == 0 or ratio.max() <= 1, f"{what}: {ratio.max():.3g} of the bound"


def _bounds(x, w, A, B, bias, dy, dtype):
    """Per output, how far the kernels may be from step()'s values."""
    u, f = U[dtype], 2.0 ** -23
    M, K = x.shape
    N = w.shape[0]
    r = ref.step(x, w, A, B, bias, dy)
    xh, wh, xa = ref.four_bits(x).abs(), ref.four_bits(w).abs(), x.double().abs()
    out = {}
    s = xh @ wh.t()
    b = K * f * s
    if A is not None:
        Aa, Ba = A.double().abs(), B.double().abs()
        ta, R = xa @ Aa, A.shape[1]
        t_off = K * f * ta + u * ((x.double() @ A.double()).abs() + K * f * ta)     # of t as the kernels hold it
        b = b + t_off @ Ba + (K + R + 2) * f * ((ta + t_off) @ Ba)
    if bias is not None:
        b = b + 4 * f * (bias.double().abs() + r["y"].abs() + b)
    out["y"] = b + u * (r["y"].abs() + b)
    if dy is not None:
        da = dy.double().abs()
        b = N * f * (da @ wh)
        if A is not None:
            dta = da @ Ba.t()
            dt_off = N * f * dta + u * ((dy.double() @ B.double().t()).abs() + N * f * dta)
            b = b + dt_off @ Aa.t() + (N + R + 2) * f * ((dta + dt_off) @ Aa.t())
            xt = ref.eight_bits(x).abs()
            a = xt.t() @ dt_off + M * f * (xt.t() @ (dta + dt_off))
            out["dA"] = a + u * (r["dA"].abs() + a)
            c = t_off.t() @ da + M * f * ((ta + t_off).t() @ da)
            out["dB"] = c + u * (r["dB"].abs() + c)
        out["dx"] = b + u * (r["dx"].abs() + b)
        out["dbias"] = M * f * da.sum(0)
    if dtype == torch.float16:      # results among the subnormals: half the smallest one
        for k in ("y", "dx", "dA", "dB"):
            if k in out:
                out[k] = out[k] + 2.0 ** -25
    return r, out


# ---- the format -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("M,K", [(1, 32), (1, 128), (3, 96), (16, 128), (17, 160), (33, 2048), (130, 1312)])
def test_codes_stand_for_the_nearest_values(cuda, dtype, M, K):
    from pyraquant_amd.mxfp4 import checkpoint_values, dequant_mxfp4, quant_mxfp4

    x = _x(M, K, dtype, M * K)
    x[0, :32] = 0
    q, q8 = quant_mxfp4(x.cuda(), checkpoint=True)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(dequant_mxfp4(q, out).cpu(), ref.four_bits(x).to(out)), out
    assert torch.equal(checkpoint_values(q8, q, torch.float32).cpu(), ref.eight_bits(x).float())
    # the codes without a checkpoint are the same ones
    alone = quant_mxfp4(x.cuda())
    assert torch.equal(alone.codes, q.codes) and torch.equal(alone.scales, q.scales)


def test_every_tie_and_edge_of_the_grid(cuda):
    """Multiples of 1/16 up to 8 of blocks whose largest value is 4, 6, 7 or just under 8, at scales from the smallest float's to
    the largest's, both signs; blocks of subnormals and of zeros."""
    from pyraquant_amd.mxfp4 import checkpoint_values, dequant_mxfp4, quant_mxfp4

    rows = []
    for top in (4.0, 6.0, 7.0, 7.984375):
        v = torch.arange(0, 128) / 16.0
        v = torch.cat([v[v <= top], -v[v <= top]])
        v = torch.cat([v, torch.zeros(-len(v) % 31)]).reshape(-1, 31)
        rows.append(torch.cat([torch.full((len(v), 1), top), v], 1))
    v = torch.cat(rows)
    for e in (0, -20, 30, -120, -129, -140, 124):
        x = torch.ldexp(v.double(), torch.tensor(e)).float()
        q, q8 = quant_mxfp4(x.cuda(), checkpoint=True)
        assert torch.equal(dequant_mxfp4(q, torch.float32).cpu().double(), ref.four_bits(x)), e
        assert torch.equal(checkpoint_values(q8, q, torch.float32).cpu().double(), ref.eight_bits(x).float().double()), e
    for dtype in BOTH:
        x = (v * 0.125).to(dtype)
        q, q8 = quant_mxfp4(x.cuda(), checkpoint=True)
        assert torch.equal(dequant_mxfp4(q, torch.float32).cpu().double(), ref.four_bits(x)), dtype
        assert torch.equal(checkpoint_values(q8, q, torch.float32).cpu().double(), ref.eight_bits(x)), dtype
    tiny = torch.arange(-16, 16).float().mul(2.0 ** -149).reshape(1, 32)
    assert torch.equal(dequant_mxfp4(quant_mxfp4(tiny.cuda()), torch.float32).cpu().double(), ref.four_bits(tiny))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
def test_blocks_with_infinities_and_nans(cuda, dtype):
    """They are NaN as a whole, and so is every output that sums over them; the others keep their values."""
    from pyraquant_amd.mxfp4 import checkpoint_values, dequant_mxfp4, quant_mxfp4

    x = _x(20, 192, dtype, 7)
    for r, k, v in ((0, 5, "nan"), (3, 64, "inf"), (3, 191, "-inf"), (19, 100, "nan")):
        x[r, k] = float(v)
    q, q8 = quant_mxfp4(x.cuda(), checkpoint=True)
    for got, want in ((dequant_mxfp4(q, torch.float32), ref.four_bits(x)),
                      (checkpoint_values(q8, q, torch.float32), ref.eight_bits(x))):
        assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want)) and int(torch.isnan(want).sum()) == 4 * 32
        assert torch.equal(torch.nan_to_num(got.cpu().double()), torch.nan_to_num(want))


def test_rows_with_strides_offsets_and_signs(cuda):
    """Windows of a larger tensor, rows that do not start on 16 bytes, transposed and expanded inputs, a negated view."""
    from pyraquant_amd.mxfp4 import dequant_mxfp4, quant_mxfp4

    base = torch.randn(70, 330, generator=_gen(1)).to(torch.bfloat16).cuda()
    views = {"window": base[3:40, 8:168], "odd offset": base[:, 3:99], "transposed": base[:64].t()[:60, :64],
             "one row": base[5:6, 1:65], "expanded": base[2:3, :96].expand(19, 96), "column steps": base[:, :192:2],
             "every other row": base[::2, :64]}
    for name, v in views.items():
        assert torch.equal(dequant_mxfp4(quant_mxfp4(v), torch.float32).cpu().double(), ref.four_bits(v.cpu())), name
    neg = torch._neg_view(base[:, :64])
    assert torch.equal(dequant_mxfp4(quant_mxfp4(neg), torch.float32).cpu().double(), ref.four_bits(-base[:, :64].cpu()))


# ---- the layer ------------------------------------------------------------------------------------------------------

# (48, 4224, ..: rows shared by several workgroups; 4128 and 33000 rows: 32 and 64 rows a workgroup of the quantizer with t)
SIZES = [(48, 4224, 32, 32), (1, 32, 16, 0), (1, 1280, 1280, 0), (2, 96, 48, 16), (5, 160, 16, 64), (16, 128, 112, 0), (17, 608, 80, 5), (31, 2080, 144, 32),
         (64, 256, 64, 0), (65, 1024, 272, 40), (129, 384, 400, 32), (257, 544, 528, 0), (300, 1312, 256, 64)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N,R", SIZES)
def test_layer_forward(cuda, dtype, M, K, N, R):
    layer, w, (A, B), bias = _layer(K, N, R, M % 2 == 1, dtype, K + N)
    x = _x(M, K, dtype, M + K)
    with torch.no_grad():
        y = layer(x.cuda())
    assert y.dtype == dtype and tuple(y.shape) == (M, N)
    r, bound = _bounds(x, w, A, B, bias, None, dtype)
    _inside(y, r["y"], bound["y"], "y")


def _grads(layer, x, dy):
    xg = x.cuda().requires_grad_()
    y = layer(xg)
    wanted = {"dx": xg, "dA": layer.lr_A, "dB": layer.lr_B}
    if layer.bias is not None:
        wanted["dbias"] = layer.bias
    got = dict(zip(wanted, torch.autograd.grad(y, list(wanted.values()), dy.cuda())))
    return {"y": y, **got}


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N,R", [s for s in SIZES if s[3]] + [(200, 64, 1040, 32), (1, 64, 32, 1), (515, 288, 96, 33)])
def test_layer_gradients(cuda, dtype, M, K, N, R):
    layer, w, (A, B), bias = _layer(K, N, R, M % 2 == 1, dtype, K + N, trainable=True)
    x = _x(M, K, dtype, M + K)
    dy = (torch.randn(M, N, generator=_gen(M)) * 0.5).to(dtype)
    got = _grads(layer, x, dy)
    r, bound = _bounds(x, w, A, B, bias, dy, dtype)
    for k, g in got.items():
        assert g.dtype == (torch.float32 if k == "dbias" else dtype) and tuple(g.shape) == tuple(r[k].shape), k
        _inside(g, r[k], bound[k], k)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("M,K,N,R", [(40, 64, 96, 8), (515, 288, 208, 33), (1100, 160, 2064, 32), (64, 4224, 2176, 64)])
def test_factor_gradients_lose_nothing_in_between(cuda, dtype, M, K, N, R):
    """dA and dB are sums of products with t and dt, which the kernels hold in two 16-bit parts: u^2 of each may be missing, not
    u. (Sums of mixed signs: most results are far smaller than their terms, and a rounding of t or dt to 16 bits shows.)"""
    layer, w, (A, B), bias = _layer(K, N, R, True, dtype, K + N, trainable=True)
    x, dy = _x(M, K, dtype, M + K), (torch.randn(M, N, generator=_gen(M)) * 0.5).to(dtype)
    got, r, (u, f) = _grads(layer, x, dy), ref.step(x, w, A, B, bias, dy), (U[dtype], 2.0 ** -23)
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    Ad, Bd, xd, dyd, xt = A.double(), B.double(), x.double(), dy.double(), ref.eight_bits(x).abs()
    t_sum, dt_sum = K * f * (xd.abs() @ Ad.abs()), N * f * (dyd.abs() @ Bd.abs().t())
    t_off = t_sum + u * u * ((xd @ Ad).abs() + t_sum) + small
    dt_off = dt_sum + u * u * ((dyd @ Bd.t()).abs() + dt_sum) + small
    a = xt.t() @ dt_off + 2 * M * f * (xt.t() @ ((dyd @ Bd.t()).abs() + dt_off))
    b = t_off.t() @ dyd.abs() + 2 * M * f * (((xd @ Ad).abs() + t_off).t() @ dyd.abs())
    _inside(got["dA"], r["dA"], a + u * (r["dA"].abs() + a) + small, "dA")
    _inside(got["dB"], r["dB"], b + u * (r["dB"].abs() + b) + small, "dB")


@pytest.mark.parametrize("M", (4128, 33000))
def test_many_rows_through_the_low_rank_branch(cuda, M):
    """The quantizer that also takes x lr_A, with more rows a workgroup: codes and checkpoint through y and dA."""
    K, N, R = 96, 32, 40
    layer, w, (A, B), bias = _layer(K, N, R, True, torch.bfloat16, 5, trainable=True)
    x, dy = _x(M, K, torch.bfloat16, 6), torch.randn(M, N, generator=_gen(7)).to(torch.bfloat16)
    got = _grads(layer, x, dy)
    r, bound = _bounds(x, w, A, B, bias, dy, torch.bfloat16)
    for k, g in got.items():
        _inside(g, r[k], bound[k], k)


@pytest.mark.parametrize("M,K,N,split", [(40, 96, 4112, True), (300, 288, 2080, True), (1000, 1312, 1040, False), (4128, 2080, 496, False),
                                         (8300, 1056, 112, False), (2050, 1312, 5136, True), (515, 3104, 9232, True)])
def test_input_gradient_of_every_kind_of_block(cuda, M, K, N, split):
    """Both kinds of block, whole sums and sums cut into slices, ragged in every direction."""
    import pyraquant_amd._lib as L
    from pyraquant_amd.mxfp4 import mxfp4_grad_input, quant_mxfp4

    assert (L.load().pq_mx_grad_input_workspace_size(M, N, K) > 0) == split
    g = torch.Generator(device="cuda").manual_seed(M)
    for dtype, R in ((torch.bfloat16, 32), (torch.float16, 64)):
        w = (torch.randn(N, K, generator=g, device=cuda) * 0.02).to(dtype)
        dy, dt, ap = (torch.randn(*s, generator=g, device=cuda).to(dtype) for s in ((M, N), (M, R), (K, R)))
        got = mxfp4_grad_input(dy, quant_mxfp4(w), dt, ap)
        wh, u = ref.four_bits(w.cpu()).cuda(), U[dtype]      # (the oracle's values; sums in 64 bits on the GPU)
        want = dy.double() @ wh + dt.double() @ ap.double().t()
        terms = dy.double().abs() @ wh.abs() + dt.double().abs() @ ap.double().abs().t()
        off = (N + R) * 2.0 ** -23 * terms
        _inside(got, want.cpu(), (off + u * (want.abs() + off)).cpu() + 2.0 ** -25, (M, K, N, dtype))
        assert torch.equal(got, mxfp4_grad_input(dy, quant_mxfp4(w), dt, ap))


@pytest.mark.parametrize("M,K,N,R", [(2100, 160, 4112, 0), (600, 1056, 7056, 32), (513, 96, 2064, 64), (1100, 352, 912, 32),
                                     (329, 4320, 2512, 32)])
def test_product_of_every_kind_of_block(cuda, M, K, N, R):
    """Sizes whose product runs in blocks of 256 x 256, 128 x 256 and 128 x 64 (n x m), all of them ragged; the last in blocks
    whose stages three groups of waves share, one more stage than a multiple of three."""
    from pyraquant_amd.mxfp4 import mxfp4_gemm, quant_mxfp4

    g = torch.Generator(device="cuda").manual_seed(M)
    for dtype in BOTH:
        x, w = torch.randn(M, K, generator=g, device=cuda).to(dtype), (torch.randn(N, K, generator=g, device=cuda) * 0.02).to(dtype)
        t, l2t = (torch.randn(n, R, generator=g, device=cuda).to(dtype) if R else None for n in (M, N))
        bias = torch.randn(N, generator=g, device=cuda)
        got = mxfp4_gemm(quant_mxfp4(x), quant_mxfp4(w), bias, dtype, t=t, l2t=l2t)
        xh, wh, u = ref.four_bits(x.cpu()).cuda(), ref.four_bits(w.cpu()).cuda(), U[dtype]
        want, terms = xh @ wh.t() + bias, xh.abs() @ wh.abs().t() + bias.abs()
        if R:
            want, terms = want + t.double() @ l2t.double().t(), terms + t.double().abs() @ l2t.double().abs().t()
        off = (K + R + 2) * 2.0 ** -23 * terms
        _inside(got, want.cpu(), (off + u * (want.abs() + off)).cpu() + 2.0 ** -25, (M, K, N, dtype))


def test_gradients_against_differences(cuda):
    """In lr_A, lr_B and the bias the layer is a polynomial: along a direction (a, b, c), the loss sum(dy y) changes by the
    gradients' product with it plus the second-order term sum(dy (x a) b), so central differences of the oracle's y cancel that
    term and leave the derivative. The gradient of lr_A is the oracle's, from 8-bit codes: its distance from the exact x's is at
    most 2^-7 of each block's largest value."""
    M, K, N, R, dtype = 48, 96, 64, 8, torch.float16
    layer, w, (A, B), bias = _layer(K, N, R, True, dtype, 3, trainable=True)
    x, g = _x(M, K, dtype, 4), _gen(5)
    dy = torch.randn(M, N, generator=g).to(dtype)
    got = {k: v.detach().double().cpu() for k, v in _grads(layer, x, dy).items()}
    _, bound = _bounds(x, w, A, B, bias, dy, dtype)

    def loss(A, B, bias):
        return (ref.step(x, w, A, B, bias)["y"] * dy.double()).sum()

    A, B, bias, h = A.double(), B.double(), bias.double(), 2.0 ** -10
    aligned = tuple(got[k].sign() for k in ("dA", "dB", "dbias"))   # along these the derivative is the sum of the magnitudes
    for a, b, c in [tuple(torch.randn(v.shape, generator=g, dtype=torch.float64) for v in (A, B, bias)) for _ in range(4)] + [aligned]:
        diff = (loss(A + h * a, B + h * b, bias + h * c) - loss(A - h * a, B - h * b, bias - h * c)) / (2 * h)
        ours = (got["dA"] * a).sum() + (got["dB"] * b).sum() + (got["dbias"] * c).sum()
        dta = dy.double().abs() @ B.abs().t()
        top = x.double().abs().reshape(M, -1, 32).amax(-1).repeat_interleave(32, 1)
        off = ((bound["dA"] + 2.0 ** -7 * (top.t() @ dta)) * a.abs()).sum() + (bound["dB"] * b.abs()).sum() + \
            (bound["dbias"] * c.abs()).sum()
        assert abs(diff - ours) <= off, (float(diff), float(ours), float(off))


def test_input_gradient_against_differences(cuda):
    """The rounding of x counts as the identity, so dx is the derivative of x -> x wh^T + x A B: of the same loss with the
    unrounded x in the product."""
    M, K, N, R, dtype = 16, 64, 48, 4, torch.bfloat16
    layer, w, (A, B), bias = _layer(K, N, R, True, dtype, 8, trainable=True)
    x, dy = _x(M, K, dtype, 9), torch.randn(M, N, generator=_gen(10)).to(dtype)
    got = _grads(layer, x, dy)["dx"].double().cpu()
    _, bound = _bounds(x, w, A, B, bias, dy, dtype)
    wh = ref.four_bits(w)
    d = torch.randn(M, K, generator=_gen(11), dtype=torch.float64)
    f = lambda x: ((x @ wh.t() + x @ A.double() @ B.double()) * dy.double()).sum()   # noqa: E731
    diff = (f(x.double() + d) - f(x.double() - d)) / 2
    assert abs(diff - (got * d).sum()) <= (bound["dx"] * d.abs()).sum()


def test_rows_of_nan_leave_the_others_alone(cuda):
    """An activation that is NaN makes its row NaN (and, through the sums over rows, the gradients that sum over it); a row of
    zeros gives the bias."""
    layer, w, (A, B), bias = _layer(256, 80, 32, True, torch.bfloat16, 1, trainable=True)
    x = _x(40, 256, torch.bfloat16, 2)
    x[7, 100], x[12] = float("nan"), 0
    dy = torch.randn(40, 80, generator=_gen(3)).to(torch.bfloat16)
    got = _grads(layer, x, dy)
    y = got["y"].detach()
    assert bool(torch.isnan(y[7]).all()) and not bool(torch.isnan(y[torch.arange(40) != 7]).any())
    assert torch.equal(y[12].cpu(), bias.to(torch.bfloat16))
    assert not bool(torch.isnan(got["dx"]).any())                    # dx does not depend on x
    blocks = torch.isnan(got["dA"]).all(1).cpu().reshape(8, 32).all(1)
    assert blocks.tolist() == [k == 100 // 32 for k in range(8)]     # the NaN is its block's alone
    # a weight block that is NaN: its output column
    lin = torch.nn.Linear(256, 80, bias=False)
    with torch.no_grad():
        lin.weight[33, 70] = float("inf")
    from pyraquant_amd.mxfp4 import Mxfp4Linear

    bad = Mxfp4Linear(lin.to(torch.bfloat16), device="cuda")
    xg = torch.ones(5, 256, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = bad(xg)
    assert torch.isnan(y).any(0).nonzero().flatten().tolist() == [33] and bool(torch.isnan(y[:, 33]).all())
    dx, = torch.autograd.grad(y, xg, torch.ones_like(y))
    assert torch.isnan(dx).any(0).nonzero().flatten().tolist() == list(range(64, 96))


def test_empty_and_batched_inputs(cuda):
    layer, w, (A, B), bias = _layer(96, 48, 16, True, torch.bfloat16, 1, trainable=True)
    x = torch.empty(0, 96, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    y = layer(x)
    g = torch.autograd.grad(y, [x, layer.lr_A, layer.lr_B, layer.bias], torch.empty_like(y))
    assert tuple(y.shape) == (0, 48) and tuple(g[0].shape) == (0, 96) and all(not bool(v.any()) for v in g[1:])
    x = _x(42, 96, torch.bfloat16, 3).cuda()
    with torch.no_grad():
        assert torch.equal(layer(x.reshape(2, 3, 7, 96)), layer(x).reshape(2, 3, 7, 48))
        assert torch.equal(layer(x[11]), layer(x[11:12])[0])


def test_output_gradients_of_every_layout(cuda):
    """Expanded (a sum's), transposed and offset output gradients give what a plain copy of them gives."""
    layer, *_ = _layer(128, 64, 16, True, torch.bfloat16, 1, trainable=True)
    x = _x(33, 128, torch.bfloat16, 2)
    wide = torch.randn(33, 90, generator=_gen(4)).to(torch.bfloat16).cuda()
    for dy in (torch.ones((), dtype=torch.bfloat16).expand(33, 64), wide[:, 3:67], wide.t()[:64].t(), wide[:1, :64].expand(33, 64)):
        a, b = _grads(layer, x, dy.cuda()), _grads(layer, x, dy.cuda().clone(memory_format=torch.contiguous_format))
        assert all(torch.equal(a[k], b[k]) for k in a)
    xg = x.cuda().requires_grad_()
    layer(xg).sum().backward()
    assert torch.equal(xg.grad, _grads(layer, x, torch.ones(33, 64, dtype=torch.bfloat16))["dx"])


def test_only_the_wanted_gradients(cuda):
    """Any choice of what requires a gradient: the same values as with all of them, and no others."""
    layer, *_ = _layer(160, 48, 24, True, torch.float16, 5, trainable=True)
    x, dy = _x(50, 160, torch.float16, 6), torch.randn(50, 48, generator=_gen(7)).to(torch.float16)
    every = _grads(layer, x, dy)
    parts = {"dx": None, "dA": layer.lr_A, "dB": layer.lr_B, "dbias": layer.bias}
    for mask in range(1, 16):
        names = [k for i, k in enumerate(parts) if mask >> i & 1]
        xg = x.cuda().requires_grad_("dx" in names)
        for k, p in parts.items():
            if p is not None:
                p.requires_grad_(k in names)
        y = layer(xg)
        got = torch.autograd.grad(y, [xg if k == "dx" else parts[k] for k in names], dy.cuda())
        assert torch.equal(y, every["y"]) and all(torch.equal(g, every[k]) for k, g in zip(names, got)), names
    with torch.no_grad():
        assert torch.equal(layer(x.cuda()), every["y"]) and not layer(x.cuda()).requires_grad


def test_frozen_layer_serves_and_passes_gradients(cuda):
    layer, w, (A, B), bias = _layer(224, 96, 20, True, torch.bfloat16, 5, trainable=True)
    x, dy = _x(37, 224, torch.bfloat16, 6), torch.randn(37, 96, generator=_gen(7)).to(torch.bfloat16)
    before = _grads(layer, x, dy)
    layer.freeze()
    assert not list(layer.parameters()) and torch.equal(layer.lr_A.cpu(), A) and torch.equal(layer.lr_B.cpu(), B)
    xg = x.cuda().requires_grad_()
    y = layer(xg)
    dx, = torch.autograd.grad(y, xg, dy.cuda())
    assert torch.equal(y, before["y"]) and torch.equal(dx, before["dx"])
    # its state dict gives another layer the same results
    other, *_ = _layer(224, 96, 20, True, torch.bfloat16, 99)
    other.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x.cuda()), before["y"])
    # without a low-rank branch or a bias
    plain, w, _, _ = _layer(96, 32, 0, False, torch.bfloat16, 3)
    xg = _x(9, 96, torch.bfloat16, 4).cuda().requires_grad_()
    dy = torch.randn(9, 32, generator=_gen(1)).to(torch.bfloat16)
    dx, = torch.autograd.grad(plain(xg), xg, dy.cuda())
    r, bound = _bounds(xg.detach().cpu(), w, None, None, None, dy, torch.bfloat16)
    _inside(dx, r["dx"], bound["dx"], "dx")


def test_parameters_in_fp32_and_module_casts(cuda):
    """fp32 factors (a master copy) are used in the input's type and get fp32 gradients; .to(dtype) keeps a bias buffer in fp32."""
    from pyraquant_amd.mxfp4 import Mxfp4Linear

    layer, w, (A, B), bias = _layer(128, 64, 16, True, torch.bfloat16, 2, trainable=True)
    x, dy = _x(30, 128, torch.bfloat16, 6), torch.randn(30, 64, generator=_gen(7)).to(torch.bfloat16)
    every = _grads(layer, x, dy)
    layer.lr_A.data, layer.lr_B.data = layer.lr_A.data.float(), layer.lr_B.data.float()
    got = _grads(layer, x, dy)
    assert got["dA"].dtype == torch.float32 and all(torch.equal(got[k].to(every[k].dtype), every[k]) for k in every)
    served, *_ = _layer(128, 64, 16, True, torch.bfloat16, 2)
    served = served.to(torch.float16)
    assert served.bias.dtype == torch.float32 and served.lr_Af.dtype == torch.float16 and served.weight_codes.dtype == torch.uint8
    assert isinstance(served, Mxfp4Linear) and served(x.cuda().to(torch.float16)).dtype == torch.float16


def test_same_results_every_time_and_on_any_stream(cuda):
    """The sums' order depends on the sizes alone; work on another stream than the tensors' own, and in a graph's replays."""
    layer, *_ = _layer(544, 272, 32, True, torch.bfloat16, 5, trainable=True)
    x, dy = _x(700, 544, torch.bfloat16, 6).cuda(), torch.randn(700, 272, generator=_gen(7)).to(torch.bfloat16).cuda()
    first = _grads(layer, x, dy)
    for _ in range(3):
        again = _grads(layer, x, dy)
        assert all(torch.equal(first[k], again[k]) for k in first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _grads(layer, x, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(first[k], other[k]) for k in first)
    served = layer.freeze()
    xin = x.clone()
    with torch.no_grad():
        served(xin)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = served(xin)
        for k in range(4):
            xin.copy_(x * (k + 1))
            graph.replay()
            assert torch.equal(y, served(xin)), k
            torch.cuda.synchronize()


def test_converted_model_and_its_statistics(cuda):
    from pyraquant_amd.mxfp4 import Mxfp4Linear, convert_linears_to_mxfp4

    net = torch.nn.Sequential(torch.nn.Linear(64, 128), torch.nn.GELU(), torch.nn.Linear(128, 64), torch.nn.Linear(64, 7)).to(torch.bfloat16)
    net.x_embedder = torch.nn.Linear(64, 64).to(torch.bfloat16)
    net[0]._lowrank_A, net[0]._lowrank_B = torch.zeros(64, 4, dtype=torch.bfloat16), torch.zeros(4, 128, dtype=torch.bfloat16)
    stats = convert_linears_to_mxfp4(net, trainable=True)
    assert stats["n_mxfp4_linear"] == 2 and sorted(stats["bf16_kept_names"]) == ["3", "x_embedder"]
    assert isinstance(net[0], Mxfp4Linear) and net[0].trainable and not net[2].trainable
    assert {n for n, _ in net[0].named_parameters()} == {"lr_A", "lr_B", "bias"} and not list(net[2].parameters())


# ---- refusals -------------------------------------------------------------------------------------------------------

def test_refusals(cuda):
    from pyraquant_amd.mxfp4 import Mxfp4Linear, Mxfp4Matrix, lowrank_grads, mxfp4_gemm, mxfp4_grad_input, quant_mxfp4

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    q, w = quant_mxfp4(x), quant_mxfp4(torch.zeros(32, 64, device=cuda))
    with pytest.raises(AssertionError):
        quant_mxfp4(x.cpu())
    with pytest.raises(AssertionError):
        quant_mxfp4(x[:, :48])
    with pytest.raises(ValueError):
        quant_mxfp4(x.double())
    with pytest.raises(AssertionError):
        mxfp4_gemm(q, quant_mxfp4(torch.zeros(32, 96, device=cuda)), None, torch.bfloat16)      # another K
    with pytest.raises(AssertionError):
        mxfp4_gemm(q, quant_mxfp4(torch.zeros(24, 64, device=cuda)), None, torch.bfloat16)      # N % 16
    with pytest.raises(ValueError):
        mxfp4_gemm(q, w, None, torch.float32)
    with pytest.raises(AssertionError):
        mxfp4_gemm(q, w, torch.zeros(32, device=cuda, dtype=torch.bfloat16), torch.bfloat16)     # bias not fp32
    with pytest.raises(AssertionError):
        mxfp4_gemm(Mxfp4Matrix(q.codes[:512], q.scales, 4, 64), w, None, torch.bfloat16)         # codes of fewer rows
    t = torch.zeros(4, 16, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(AssertionError):
        mxfp4_gemm(q, w, None, torch.bfloat16, t=t, l2t=torch.zeros(32, 16, dtype=torch.bfloat16, device=cuda))   # rank 16
    with pytest.raises(AssertionError):
        mxfp4_gemm(q, w, None, torch.bfloat16, out=torch.zeros(4, 36, dtype=torch.bfloat16, device=cuda)[:, :32])  # ldc % 8
    with pytest.raises(AssertionError):
        mxfp4_grad_input(torch.zeros(4, 48, dtype=torch.bfloat16, device=cuda), w)
    with pytest.raises(AssertionError):
        lowrank_grads(None, None, t, torch.zeros(4, 64, dtype=torch.int8, device=cuda), q.scales, 16, True, False, False)  # P 16
    layer, *_ = _layer(64, 32, 8, True, torch.bfloat16, 1)
    with pytest.raises(ValueError):
        layer(torch.zeros(4, 64, device=cuda))
    with pytest.raises(AssertionError):
        layer(x.cpu())
    with pytest.raises(AssertionError):
        layer(torch.zeros(4, 96, dtype=torch.bfloat16, device=cuda))
    for K, N, R in ((48, 32, 0), (64, 24, 0), (64, 32, 65)):
        with pytest.raises(AssertionError):
            _layer(K, N, R, False, torch.bfloat16, 1)
    with pytest.raises(AssertionError):
        Mxfp4Linear(torch.nn.Linear(64, 32), device="cuda", trainable=True)


def test_untouched_memory_around_the_outputs(cuda):
    """Rows past M and columns past N of the output's own memory keep what they held."""
    from pyraquant_amd.mxfp4 import mxfp4_gemm, quant_mxfp4

    for M, N in ((5, 16), (33, 80), (130, 272)):
        big = torch.full((M + 9, N + 24), 7.0, dtype=torch.bfloat16, device=cuda)
        q, w = quant_mxfp4(_x(M, 160, torch.bfloat16, 1).cuda()), quant_mxfp4(_x(N, 160, torch.float32, 2).cuda())
        y = mxfp4_gemm(q, w, None, torch.bfloat16, out=big[4 : 4 + M, 8 : 8 + N])
        assert torch.equal(y, mxfp4_gemm(q, w, None, torch.bfloat16))
        edge = big.clone()
        edge[4 : 4 + M, 8 : 8 + N] = 7.0
        assert bool((edge == 7.0).all())


def test_example_tunes_and_serves(cuda):
    """The example end to end, small: tuning lowers the error, and the frozen block answers as the tuned one."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "tune_mxfp4_lowrank.py")
    spec = importlib.util.spec_from_file_location("tune_mxfp4_lowrank", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    bare, started, tuned, served = example.run(dim=256, tokens=512, rank=32, steps=40)
    assert tuned < started and tuned < bare and served == tuned, (bare, started, tuned, served)


@pytest.mark.parametrize("M,K,N,R", [(4200, 32, 4208, 32), (4200, 160, 4208, 0), (8500, 416, 4368, 64), (8500, 2080, 4368, 32)])
def test_large_products_over_several_blocks_a_workgroup(cuda, M, K, N, R):
    """More blocks than compute units, ragged both ways, sums of one stage up to more than the ring holds, over outputs that hold
    NaN: every element is written, and as the same product in two parts gives it (other blocks, other neighbours in time)."""
    from pyraquant_amd.mxfp4 import mxfp4_gemm, quant_mxfp4

    g = torch.Generator(device="cuda").manual_seed(K)
    x, w = torch.randn(M, K, generator=g, device=cuda).bfloat16(), torch.randn(N, K, generator=g, device=cuda).bfloat16()
    t, l2t = (torch.randn(n, R, generator=g, device=cuda).bfloat16() if R else None for n in (M, N))
    bias = torch.randn(N, generator=g, device=cuda)
    xq, wq = quant_mxfp4(x), quant_mxfp4(w)
    for has_bias in (True, False):
        out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=cuda)
        for _ in range(3):
            got = mxfp4_gemm(xq, wq, bias if has_bias else None, torch.bfloat16, t=t, l2t=l2t, out=out)
        xh, wh = (quant.double() for quant in (_values_of(xq), _values_of(wq)))
        want = xh @ wh.t() + (bias if has_bias else 0)
        if R:
            want = want + t.double() @ l2t.double().t()
        terms = xh.abs() @ wh.abs().t() + bias.abs() + (t.double().abs() @ l2t.double().abs().t() if R else 0)
        off = (K + R + 2) * 2.0 ** -23 * terms
        bound = off + U[torch.bfloat16] * (want.abs() + off)
        assert not bool(torch.isnan(got).any()) and bool(((got.double() - want).abs() <= bound).all())
        rows = 160   # few rows: another kernel's blocks
        part = mxfp4_gemm(quant_mxfp4(x[:rows]), wq, bias if has_bias else None, torch.bfloat16, t=None if t is None else t[:rows], l2t=l2t)
        assert bool(((part.double() - want[:rows]).abs() <= bound[:rows]).all())


def _values_of(q):
    from pyraquant_amd.mxfp4 import dequant_mxfp4

    return dequant_mxfp4(q, torch.float32)
