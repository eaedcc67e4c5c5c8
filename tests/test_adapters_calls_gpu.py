"""Calls that adapters answer or refuse beside those of test_adapters_gpu.py, whose problems, formulas and bounds these use."""
import pytest
import torch

from test_adapters_gpu import BOTH, _bank, _near, _problem, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,each,K,N,slots,R", [(1, 9, 72, 40, 3, 8), (2, 77, 264, 136, 4, 16), (6, 50, 136, 264, 5, 24), (5, 1000, 520, 72, 12, 16)])
def test_flat_rows_with_an_id_for_each_request(cuda, n, each, K, N, slots, R, dtype):
    """x [M, K] and y [M, N] with M / each ids: the same bits, forward and back, as a batch of its own dimension."""
    x, y, _, A, B, scale = _problem(n * each, K, N, slots, R, dtype, "one", seed=n)
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-1, slots, (n,), generator=g, device=cuda, dtype=torch.int32)
    dy = torch.randn(n * each, N, device=cuda).to(dtype)
    frozen, tuned = _bank(A, B, scale), _bank(A, B, scale, trainable=True)
    x.requires_grad_()

    def step(*shape):
        out = tuned(x.view(*shape, K), y.view(*shape, N), ids)
        grads = torch.autograd.grad(out, (x, tuned.lr_A, tuned.lr_B), dy.view(*shape, N))
        return (out.detach().view(-1, N), *grads)

    flat = step(n * each)
    assert all(torch.equal(a, b) for a, b in zip(flat, step(n, each)))
    with torch.no_grad():
        assert torch.equal(frozen(x, y, ids), flat[0])
        into = y.clone()
        assert torch.equal(frozen(x, into, ids, out=into), flat[0])
    exact, off = _want(x.detach(), y, ids.repeat_interleave(each), A, B, scale, dy)
    for k, v in zip(("y", "dx", "dA", "dB"), flat):
        _near(v, exact[k], off[k], k)


def test_ids_that_are_no_requests_of_the_rows(cuda):
    x, y, i, A, B, scale = _problem(24, 64, 40, 3, 8, torch.bfloat16, "runs")
    bank = _bank(A, B, scale)
    with torch.no_grad():
        for n in (0, 5, 48):
            with pytest.raises(AssertionError):
                bank(x, y, torch.zeros(n, dtype=torch.int32, device=cuda))
        for bad in ((x[:0], y[:0], i[:3]), (x.view(2, 12, 64), y.view(2, 12, 40), i[:6]), (x[0], y[0], i[:1])):
            with pytest.raises(AssertionError):
                bank(*bad)


def test_layers_take_no_ids_of_flat_rows(cuda):
    """A model's projection whose rows are not the batch's (a table of positions, say) must not take its ids for runs of them."""
    from pyraquant_amd import add_adapters

    net = torch.nn.Sequential(torch.nn.Linear(64, 40)).to(cuda, torch.bfloat16)
    styles = add_adapters(net, 2, 8, whitelist=lambda n: False)
    ids = torch.tensor([0, 1], device=cuda)
    with torch.no_grad(), styles.use(ids):
        assert net(torch.zeros(2, 64, device=cuda, dtype=torch.bfloat16)).shape == (2, 40)
        with pytest.raises(AssertionError):
            net(torch.zeros(6, 64, device=cuda, dtype=torch.bfloat16))


def test_one_row_into_out(cuda):
    """A result of one dimension goes into memory whose values follow each other, and into no other."""
    x, y, _, A, B, scale = _problem(1, 64, 40, 3, 8, torch.bfloat16, "one")
    bank, i = _bank(A, B, scale), torch.tensor(1, device=cuda)
    room = torch.full((160,), 7.0, dtype=torch.bfloat16, device=cuda)
    with torch.no_grad():
        want = bank(x[0], y[0], i)
        assert bank(x[0], y[0], i, out=room[40:80]) is not None and torch.equal(room[40:80], want)
        assert bool((room[:40] == 7).all()) and bool((room[80:] == 7).all())
        room.fill_(7)
        for out in (room[:80:2], room[:1].expand(40), room.view(40, 4)[:, 1], room[1:41]):
            with pytest.raises(AssertionError, match="contiguous|aligned"):
                bank(x[0], y[0], i, out=out)
        assert bool((room == 7).all())


@pytest.mark.parametrize("dtype", (*BOTH, torch.float32))
@pytest.mark.parametrize("K,N,rank", [(8, 8, 1), (136, 264, 20), (1280, 72, 64), (520, 1032, 16)])
def test_factors_laid_out_on_the_gpu(cuda, K, N, rank, dtype):
    """set() and freeze() on the GPU and on the CPU hold the same: ranks below the module's, factors of other types, orders and devices."""
    from pyraquant_amd.adapters import LowRankAdapters

    g = torch.Generator().manual_seed(K)
    here, there = (LowRankAdapters(K, N, 3, rank, dtype=dtype, device=d) for d in (cuda, "cpu"))
    tuned, again = (LowRankAdapters(K, N, 3, rank, dtype=dtype, device=d, trainable=True) for d in (cuda, "cpu"))
    wide_a, wide_b = torch.randn(rank, K + 1, generator=g), torch.randn(N, 2 * rank, generator=g)
    for slot, r, move in ((1, rank, lambda t: t), (0, max(rank - 3, 1), lambda t: t.to(cuda, torch.float16)), (2, 1, lambda t: t.double()),
                          (1, max(rank // 2, 1), lambda t: t.to(cuda))):
        A, B = move(wide_a)[:r, 1:].t(), move(wide_b)[:, ::2].t()[:r]
        for bank in (here, there, tuned, again):
            bank.set(slot, A.requires_grad_(), B, 0.5 + slot)
        assert torch.equal(here.lr_Af.cpu(), there.lr_Af) and torch.equal(here.lr_Bf.cpu(), there.lr_Bf), slot
        assert torch.equal(here.scale.cpu(), there.scale) and torch.equal(here.lr_A[slot, :, :r].cpu(), A.detach().cpu().to(dtype))
    here.set(1, torch._neg_view(torch.ones(K, rank, dtype=dtype, device=cuda)), torch.ones(rank, N, device=cuda))
    assert bool((here.lr_A[1] == -1).all()) and bool((here.lr_B[1] == 1).all()) and torch.equal(here.lr_Af[0].cpu(), there.lr_Af[0])
    for to in (None, torch.float16):
        a, b = (LowRankAdapters(K, N, 3, rank, dtype=dtype, device=m.scale.device, trainable=True) for m in (tuned, again))
        a.load_state_dict(tuned.state_dict())
        b.load_state_dict(again.state_dict())
        a.freeze(to)
        b.freeze(to)
        assert a.lr_Af.dtype == (to or dtype) and torch.equal(a.lr_Af.cpu(), b.lr_Af) and torch.equal(a.lr_Bf.cpu(), b.lr_Bf)


def test_backward_sees_that_factors_were_set(cuda):
    x, y, i, A, B, scale = _problem(24, 64, 40, 3, 8, torch.bfloat16, "runs")
    bank = _bank(A, B, scale)
    out = bank(x.requires_grad_(), y, i)
    bank.set(1, A[0], B[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def _near_small(M, K, N, slots, R, x_std, A_std, B_std, dy_std, ids, spread, seed):
    """fp16 values far below 1: every product of t and dt against 64 bits. Two parts hold a value to 2 u^2 of it, or to half of fp16's smallest
    subnormal, 2^-25, on a scale on which the largest of the values that share one is at least 2^15: those of a row in the products with t or
    dt, those of a rank of the adapter's rows in the sums over rows. So w |v| + 2^-40 max |v|, without the 2^-25 that the values themselves
    would lose."""
    f, u = 2.0 ** -24, 2.0 ** -11
    w, least, tiny = 2 * u * u, 2.0 ** -40, 2.0 ** -25
    x, y, i, A, B, scale = _problem(M, K, N, slots, R, torch.float16, ids, seed=seed)
    dy = torch.randn(M, N, device="cuda")
    x, A, B, dy = x.float() * x_std, A.float() * K ** 0.5 * A_std, B.float() * R ** 0.5 * B_std, dy * dy_std
    if spread:      # ranks of other sizes, and rows that grow
        A = A * 4.0 ** -(torch.arange(R, device="cuda") % 8)
        x = x * torch.logspace(-3, 0, M, device="cuda")[:, None]
        dy = dy * torch.logspace(0, -3, M, device="cuda")[:, None]
    x, A, B, dy, y = x.half(), A.half(), B.half(), dy.half(), y * 0
    bank = _bank(A, B, scale, trainable=True)
    v = x.clone().requires_grad_()
    out = bank(v, y, i)
    got = dict(zip(("dx", "dA", "dB"), torch.autograd.grad(out, (v, bank.lr_A, bank.lr_B), dy)), y=out.detach())
    for s in range(slots):
        rows = torch.nonzero(i == s).flatten()
        if not len(rows):
            continue
        n = len(rows)
        a, b, xs, d, sc = A[s].double(), B[s].double(), x[rows].double(), dy[rows].double(), float(scale[s])
        t, dt = xs @ a * sc, d @ b.t() * sc
        t_off, d_off = sc * (K + 2) * f * (xs.abs() @ a.abs()), sc * (N + 2) * f * (d.abs() @ b.abs().t())
        for name, v0, v_off, other, result in (("y", t, t_off, b, t @ b), ("dx", dt, d_off, a.t(), dt @ a.t())):
            mag = v0.abs() + v_off
            o = (v_off + w * mag + least * mag.amax(1, keepdim=True) + (R + 4) * f * mag) @ other.abs() + 2 * f * result.abs()
            _near(got[name][rows], result, o + u * (result.abs() + o) + tiny, name)
        for name, v0, v_off, z in (("dA", dt, d_off, xs), ("dB", t, t_off, d)):
            mag = v0.abs() + v_off
            result = z.t() @ v0
            o = z.abs().t() @ (v_off + w * mag + least * mag.amax(0, keepdim=True) + (n + 300) * f * mag)
            o = o + u * (result.abs() + o) + tiny
            if name == "dB":
                result, o = result.t(), o.t()
            _near(got[name][s], result, o, name)


@pytest.mark.parametrize("ids", ("one", "runs", "rows"))
@pytest.mark.parametrize("size", [(2051, 520, 808, 3, 32), (1030, 96, 328, 7, 16), (700, 136, 264, 9, 40), (4096, 64, 128, 2, 8)], ids=str)
def test_small_values_in_fp16(cuda, size, ids):
    """t or dt of 1e-6 and 1e-8, as little-scaled gradients and new factors make them, where the sums that they enter are well inside fp16."""
    for x_std, A_std, B_std, dy_std in ((30.0, 1e-2, 4e-6, 1e-2), (1e3, 1e-3, 1e-6, 4e-4), (1e-2, 4e-6, 1e-2, 30.0), (1e-3, 1e-6, 1e-1, 1e3)):
        _near_small(*size, x_std, A_std, B_std, dy_std, ids, False, seed=size[0])


@pytest.mark.parametrize("size", [(2051, 520, 808, 3, 32), (1030, 96, 328, 7, 16), (700, 136, 264, 9, 64), (5000, 64, 128, 2, 8)], ids=str)
def test_sizes_that_differ_in_fp16(cuda, size):
    """Ranks whose values are 2^-14 of others', and rows that grow or fall by a thousand, up to values past fp16's end."""
    for x_std, A_std, B_std, dy_std in ((1.0, 1e-2, 1e-3, 1e-2), (100.0, 10.0, 1e-3, 1.0), (1.0, 1e-3, 10.0, 300.0)):
        for ids in ("one", "runs"):
            _near_small(*size, x_std, A_std, B_std, dy_std, ids, True, seed=size[0] + 1)


def _styles(net, **kw):
    from pyraquant_amd import add_adapters

    styles = add_adapters(net, 3, 8, whitelist=lambda n: False, **kw)
    for bank in styles.layers.values():
        for s in range(3):
            bank.set(s, torch.randn(bank.in_features, 8) * 0.1, torch.randn(8, bank.out_features) * 0.1)
    return styles


@pytest.mark.parametrize("kind", ("linear", "int8", "mxfp4", "split", "split int8"))
def test_what_hooks_keep_stays(cuda, kind):
    """A layer's result that a forward hook keeps, of the layer, of a part of it or of every module, is the layer's own afterwards too."""
    from pyraquant_amd import convert_linears_to_int8, convert_linears_to_mxfp4
    from pyraquant_amd.weights import SplitInLinear

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(256, 128)).to(cuda, torch.bfloat16)
    if "split" in kind:
        net[0] = SplitInLinear(net[0], 128)
    if "int8" in kind:
        convert_linears_to_int8(net, whitelist=lambda n: False)
    if kind == "mxfp4":
        convert_linears_to_mxfp4(net, whitelist=lambda n: False)
    styles = _styles(net.requires_grad_(False))
    layer = net[0].layer
    x = torch.randn(3, 20, 256, device=cuda, dtype=torch.bfloat16)
    ids = torch.tensor([1, -1, 2], device=cuda)
    places = [layer.register_forward_hook, torch.nn.modules.module.register_module_forward_hook]
    if "split" in kind:
        places.append(layer.linears[0].register_forward_hook)
    with torch.no_grad():
        own = layer(x)
        with styles.use(ids):
            want = net(x)
        for place in places:
            seen = []
            handle = place(lambda m, a, out: seen.append((m, out)))
            with styles.use(ids):
                assert torch.equal(net(x), want)
            handle.remove()
            kept = [out for m, out in seen if m is layer]
            if place == places[-1] and "split" in kind:
                kept = [seen[0][1]] if "int8" in kind else []      # (of two parts in one, the first's result is the layer's)
            assert all(torch.equal(out, own) for out in kept) and (kept or place == places[-1])
        layer.forward, inner = lambda v: held, layer.forward     # (a call that was put in the place of the layer's own)
        held = inner(x)
        with styles.use(ids):
            assert torch.equal(net(x), want) and torch.equal(held, own)


def test_a_linear_that_holds_its_result(cuda):
    """An nn.Linear of a class of its own may hand out a tensor that it holds, at any place."""
    class Held(torch.nn.Linear):
        def forward(self, x):
            if not hasattr(self, "out"):
                y = super().forward(x)
                self.out = torch.empty(y.numel() + 1, dtype=y.dtype, device=y.device)[1:].view(y.shape).copy_(y)
            return self.out

    net = torch.nn.Sequential(Held(64, 40)).to(cuda, torch.bfloat16).requires_grad_(False)
    styles = _styles(net)
    x = torch.randn(3, 20, 64, device=cuda, dtype=torch.bfloat16)
    with torch.no_grad():
        plain = net(x).clone()
        with styles.use(torch.tensor([1, -1, 2], device=cuda)):
            first = net(x)
            assert torch.equal(net(x), first) and not torch.equal(first, plain) and torch.equal(net[0].layer.out, plain)


@pytest.mark.parametrize("reentrant", (True, False))
def test_blocks_computed_again_in_the_backward_pass(cuda, reentrant):
    """A checkpointed block gets the choice of its forward pass, where that still holds in the backward pass; else it raises."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(64, 40)).to(cuda, torch.bfloat16).requires_grad_(False)
    styles = _styles(net, trainable=True)
    x = torch.randn(3, 20, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    ids = torch.tensor([1, -1, 2], device=cuda)
    with styles.use(ids):
        net(x).sum().backward()
    want = [p.grad.clone() for p in styles.parameters()]
    for p in styles.parameters():
        p.grad = None
    with styles.use(ids):
        checkpoint(net, x, use_reentrant=reentrant).sum().backward()
    assert all(torch.equal(p.grad, w) for p, w in zip(styles.parameters(), want))
    with styles.use(ids):
        out = checkpoint(net, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="chosen"):
        out.sum().backward()
    with styles.use(ids):
        out = checkpoint(net, x, use_reentrant=reentrant)
    with styles.use(ids):
        out.sum().backward()
    plain = checkpoint(net, x, use_reentrant=reentrant)      # no adapters, in either pass
    x.grad = None
    plain.sum().backward()
    assert torch.equal(x.grad, torch.autograd.grad(net[0].layer(x).sum(), x)[0])
