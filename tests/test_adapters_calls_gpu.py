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
