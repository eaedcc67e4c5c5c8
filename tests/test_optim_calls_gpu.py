"""Calls that AdamW answers or refuses beside those of test_optim_gpu.py, whose bounds these use."""
import copy
import gc

import numpy as np
import pytest
import torch

from oracle import adamw_ref as ref
from test_optim_gpu import TYPES, _before, _check_step, _grads, _opt, _params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", (32, 8))
def test_parameters_that_change_where_they_lie(cuda, bits):
    """A parameter that is shorter, longer, has gaps, or another type than its states' at the same address as before."""
    room = torch.full((4000,), 3.0, device=cuda)
    p = torch.nn.Parameter(room[:1000])
    opt = _opt([p], bits=bits)
    _grads([p], 0)
    opt.step()
    was, state = room.clone(), [t.clone() for t in opt.states()]
    for view, why in ((room[:4], "size"), (room[:2000], "size"), (room[:2000:2], "dense"), (room[:0], "size")):
        p.grad = None
        p.data = view
        assert p.data_ptr() == room.data_ptr() or not p.numel()
        with pytest.raises(AssertionError, match=why):
            opt.step()
        p.grad = torch.ones_like(p)
        with pytest.raises(AssertionError, match=why):
            opt.step()
        assert torch.equal(room, was) and all(torch.equal(a, b) for a, b in zip(opt.states(), state))
    p.grad = None
    p.data = room[:1000]
    _grads([p], 1)
    before = _before(opt)
    opt.step()
    _check_step(opt, before, 2)
    half = torch.nn.Parameter(torch.randn(1000, device=cuda).bfloat16())
    opt = _opt([half], bits=bits)
    _grads([half], 0)
    opt.step()
    at = half.data_ptr()
    half.data, half.grad = half.data.view(torch.float16), None      # (the same bits as values of another type)
    half.data.copy_(torch.randn(1000, device=cuda))
    assert half.data_ptr() == at and half.dtype == torch.float16
    _grads([half], 1)
    before = _before(opt)
    opt.step()
    _check_step(opt, before, 2)
    half.data, half.grad = half.data.double(), None
    with pytest.raises(ValueError, match="dtype"):
        opt.step()


@pytest.mark.parametrize("bits", (32, 8))
def test_a_group_of_empty_parameters(cuda, bits):
    """Parameters without a value, alone in their group, with a gradient and with a limit."""
    empty, full = (torch.nn.Parameter(torch.ones(n, device=cuda)) for n in (0, 100))
    for p in (empty, full):
        p.grad = torch.ones_like(p)
    for groups in ([{"params": [empty]}], [{"params": [empty]}, {"params": [full]}]):
        for limit in (None, 1.0):
            opt = _opt(groups, bits=bits, max_norm=limit)
            opt.step()
            opt.step()
            assert limit is None or abs(float(opt.grad_norm) - 10.0 * (len(groups) - 1)) < 1e-5
            assert all(t.numel() == 0 for t in opt.moments()) and opt.offsets() == [0]
    assert bool((full < 1).all())


def test_a_step_that_was_refused(cuda):
    """What a refused step has seen of parameters that moved counts for nothing: the next one is refused too, or finds all of them."""
    a, b = _params([(1000,), (500,)], torch.float32)
    opt = _opt([a, b])
    _grads([a, b], 0)
    opt.step()
    old, room = a.data, b.data
    was = old.clone()
    a.data = old.clone()
    b.grad, b.data = None, room[:100]
    for _ in range(2):
        with pytest.raises(AssertionError, match="size"):
            opt.step()
    b.data = room
    _grads([a, b], 1)
    before = _before(opt)
    opt.step()
    _check_step(opt, before, 2)
    assert torch.equal(old, was) and not torch.equal(a, was)
    both = torch.zeros(1200, device=cuda)
    a.data, b.data = both[:1000], both[700:]
    _grads([a, b], 2)
    for _ in range(2):
        with pytest.raises(AssertionError, match="share memory"):
            opt.step()
    assert not both.any()


@pytest.mark.parametrize("bits", (32, 8))
def test_captured_steps_keep_rates_and_parameters(cuda, bits):
    """The rate and the parameters' memory that a captured step goes on with are the optimizer's, where nobody else holds them any more."""
    params = _params([(640, 16), (1001,)], torch.float32)
    opt = _opt(params, bits=bits, lr=torch.full((4096,), 1e-3, device=cuda)[0], weight_decay=0.0)
    _grads(params, 0)
    grads = [p.grad for p in params]
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    places = [(p.data_ptr(), p.numel() * 4) for p in params] + [(opt.param_groups[0]["lr"].data_ptr(), 4)]
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))             # (the group's rate is another tensor now)
    for p, g in zip(params, grads):
        p.data = p.data.clone()
        p.grad = g
    opt.step()
    gc.collect()
    junk = [torch.full((n,), 0x7f, dtype=torch.uint8, device=cuda) for n in (4, 512, 4004, 4096, 16384, 40960, 65536) for _ in range(60)]
    for at, n in places:
        assert all(t.data_ptr() + t.numel() <= at or at + n <= t.data_ptr() for t in junk)
    now = [p.detach().clone() for p in params]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params, now)) and all(bool((t == 0x7f).all()) for t in junk)


@pytest.mark.parametrize("nan", (0x7fc00000, -0x400000, 0x7fffffff, -1, -0x7fffff))      # (with the sign bit: from -0x7fffff to -1)
def test_blocks_with_any_nan_are_nan(cuda, nan):
    p = torch.nn.Parameter(torch.ones(128 * 3, device=cuda))
    opt = _opt([p], bits=8)
    g = torch.ones(3, 128, device=cuda)
    g.view(torch.int32)[1, 7] = nan
    assert bool(g[1, 7].isnan())
    p.grad = g.view(-1)
    opt.step()
    for t in opt.moments():
        t = t.view(3, 128)
        assert bool(t[1].isnan().all()) and bool(t[0].isfinite().all()) and bool(t[2].isfinite().all())
    assert int(p.detach().isnan().sum()) == 1
    opt.step()
    for t in opt.moments():
        assert bool(t.view(3, 128)[1].isnan().all())


def test_groups_from_the_end(cuda):
    """A group's number counted from the end is that group, and no other memory."""
    a, b = _params([(300,), (77, 3)], torch.float32)
    opt = _opt([{"params": [a]}, {"params": [b], "bits": 8}])
    _grads([a, b], 0)
    opt.step()
    assert opt.offsets(-1) == opt.offsets(1)
    assert all(x.data_ptr() == y.data_ptr() for x, y in zip(opt.states(-1), opt.states(1)))
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(group=-2), opt.moments(group=0)))
    m, r = opt.moments(group=-1)
    opt.load_moments(m, r, 7, group=-1)
    _grads([a, b], 1)
    before = _before(opt)
    opt.step()
    assert int(opt.state[b]["step"][0]) == 8 and int(opt.state[a]["step"][0]) == 2
    assert opt.state[b]["exp_avg_8bit"].data_ptr() == opt.states(1)[0].data_ptr()
    del before
    for i in (2, -3):
        with pytest.raises(IndexError):
            opt.moments(group=i)


@pytest.mark.parametrize("bits", (32, 8))
def test_states_that_are_taken_away_or_replaced(cuda, bits):
    """opt.state says what a parameter's states are: those that are gone begin anew, others' go on, and given ones count."""
    from collections import defaultdict

    params = _params([(1000,), (33, 7), (2050,)], torch.float32)
    opt = _opt(params, bits=bits, seed=5)

    def step(seed, t):
        _grads(params, seed)
        before = _before(opt)
        opt.step()
        for k, n in enumerate(t):
            assert opt.state[params[k]]["step"].tolist() == [n] * opt.state[params[k]]["step"].numel()
        if len(set(t)) == 1:
            _check_step(opt, before, t[0], seed=5)

    step(0, (1, 1, 1))
    step(1, (2, 2, 2))
    opt.state.clear()
    step(2, (1, 1, 1))
    step(3, (2, 2, 2))
    kept = [t.clone() for t in opt.state[params[0]].values()]
    opt.state.pop(params[1])
    assert not opt.moments()[0][1024:1024 + 231].any() and all(torch.equal(a, b) for a, b in zip(kept, opt.state[params[0]].values()))
    step(4, (3, 1, 3))
    opt.state[params[2]] = {}
    step(5, (4, 2, 1))
    given = {k: v.clone() for k, v in opt.state[params[0]].items()}
    step(6, (5, 3, 2))
    opt.state[params[0]] = given
    step(7, (5, 4, 3))
    opt.state = defaultdict(dict)
    step(8, (1, 1, 1))


def test_states_loaded_on_another_stream(cuda):
    """States that a state dict brings on one stream and a step takes on another, which is behind."""
    p = _params([(1 << 20,)], torch.float32)
    opt, want = _opt(p), _opt(copy.deepcopy(p))
    q = want.param_groups[0]["params"]
    for t in (0, 1):
        for ps, o in ((p, opt), (q, want)):
            _grads(ps, t)
            o.step()
    side = torch.cuda.Stream()
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        opt.step()
    junk = [torch.full((1 << 20,), 1e9, device=cuda) for _ in range(8)]      # (memory that the loaded states may have had)
    torch.cuda.current_stream().wait_stream(side)
    want.step()
    assert torch.equal(p[0], q[0]) and all(torch.equal(a, b) for a, b in zip(opt.states(), want.states()))
    del junk


@pytest.mark.parametrize("dtype", TYPES)
def test_values_do_not_depend_on_their_neighbours(cuda, dtype):
    """With 32-bit states a value's step is the same to the bit whatever else is in its tensor: squares that are subnormal beside it, or infinite."""
    g = torch.Generator().manual_seed(0)
    values, grads = torch.randn(4096, generator=g) * 0.02, torch.randn(2, 4096, generator=g) * 1e-3
    out = []
    for odd in (None, 1e-14, float("inf")):
        p = torch.nn.Parameter(values.to(dtype).to(cuda))
        opt = _opt([p])
        for gr in grads:
            p.grad = gr.to(dtype).to(cuda)
            if odd is not None:
                p.grad[::64] = odd
            opt.step()
        keep = torch.arange(4096, device=cuda) % 64 != 0
        out.append([p.detach()[keep]] + [t[keep] for t in opt.states()])
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


def test_means_beside_a_border_of_their_grid(cuda):
    """8-bit means whose exact value lies a third of fp32's last place below or above a border of the grid (what the hash adds counted in) are held on
    that side of it. The gradients that lead there are found in 64 bits: m' = m + (1 - b1) (g - m) moves by a tenth of g's last place."""
    n, seed, t, b1 = 1 << 16, 3, 1, 0.9
    rng = np.random.default_rng(0)
    m = ref.held(np.where(rng.random(n) < 0.5, 1, -1) * rng.uniform(1e-3, 4e-3, n), 3, 0.5)
    um, _ = ref.dither(np.arange(n), t, seed)
    add = (um * 65536).astype(np.int64) << 4
    bits = np.float32(0.95 * np.abs(m)).view(np.int32).astype(np.int64)
    border = ((bits + add) >> 20 << 20) - add + (1 << 20)                       # the next place in fp32 from which on the sum has one step more
    low = border.astype(np.int32).view(np.float32).astype(np.float64)
    last = np.ldexp(1.0, np.frexp(low)[1] - 24)
    side = np.where(rng.random(n) < 0.5, -1, 1)
    target = np.sign(m) * (low + side * last / 3)
    g = np.float32((target - b1 * m) / (1 - b1))
    exact = b1 * m + (1 - b1) * g.astype(np.float64)
    off = (np.abs(exact) - low) / last
    sure = (off * side > 0.1) & (np.abs(off) < 0.5)                              # (g's own rounding)
    assert sure.mean() > 0.9
    p = torch.nn.Parameter(torch.zeros(n, device=cuda))
    opt = _opt([p], bits=8, seed=seed)
    opt.load_moments(torch.tensor(m, dtype=torch.float32, device=cuda), torch.full((n,), 1e-3, device=cuda), 0)
    assert np.array_equal(opt.moments()[0].double().cpu().numpy(), m)
    p.grad = torch.tensor(g, device=cuda)
    opt.step()
    got, want = opt.moments()[0].double().cpu().numpy(), ref.held(exact, 3, um)
    assert np.array_equal(got[sure], want[sure]), int((got[sure] != want[sure]).sum())


def test_infinite_gradients_where_nothing_is_added(cuda):
    """A block with one infinity is NaN also where the hash adds nothing to it."""
    n = 1 << 22
    places = np.nonzero(ref.dither(np.arange(n), 1, 0)[0] == 0)[0]
    assert len(places) > 20
    for sign in (1.0, -1.0):
        p = torch.nn.Parameter(torch.zeros(n, device=cuda))
        opt = _opt([p], bits=8)
        p.grad = torch.zeros_like(p)
        p.grad[torch.tensor(places, device=cuda)] = sign * float("inf")
        opt.step()
        blocks = torch.zeros(n // 128, dtype=torch.bool, device=cuda)
        blocks[torch.tensor(places // 128, device=cuda)] = True
        for v in opt.moments():
            assert torch.equal(v.view(-1, 128).isnan().all(1), blocks) and not v.view(-1, 128)[~blocks].any()
