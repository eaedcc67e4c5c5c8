"""The optimizer's entries without a GPU: arguments are refused before any HIP call, the oracle's 8-bit values agree with a grid written
out by hand, and the hash is as even as the rounding needs."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw_ref as ref

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(257)


def _lib():
    import pyraquant_amd._lib as L

    return L, L.load()


def _list(L, sizes=(1000, 3000), grads=(256, 256), tensors=P, chunks=P, first=None):
    n = len(sizes)
    counts = [(s + 1023) // 1024 for s in sizes]
    first = first if first is not None else [sum(counts[:i]) for i in range(n + 1)]
    return L.AdamWList(tensors, chunks, (ctypes.c_int64 * (n + 1))(*first), (ctypes.c_void_p * n)(*grads), n)


def test_step_refusals():
    L, lib = _lib()

    def step(lst=None, partials=None, n=0, norm=None, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, most=1.0, m=P, v=P, exps=P, steps=P,
             values=4096, bits=8):
        lst = _list(L) if lst is None else lst
        s, r = L.AdamWStates(m, v, exps, steps, values, bits), L.AdamWRates(lr, b1, b2, eps, wd, most, None, 0)
        return lib.pq_adamw_step(ctypes.byref(lst), ctypes.byref(s), ctypes.byref(r), partials, n, norm, None)

    assert step(m=None) == L.PQ_EINVAL and step(v=None) == L.PQ_EINVAL and step(exps=None) == L.PQ_EINVAL and step(steps=None) == L.PQ_EINVAL
    assert step(bits=16) == L.PQ_EINVAL and step(values=4095) == L.PQ_ESHAPE and step(values=-128) == L.PQ_ESHAPE
    assert step(m=ODD) == L.PQ_EALIGN and step(exps=ODD) == L.PQ_EALIGN
    assert step(lr=-1.0) == L.PQ_EINVAL and step(lr=float("nan")) == L.PQ_EINVAL and step(b1=1.0) == L.PQ_EINVAL and step(b2=-0.1) == L.PQ_EINVAL
    assert step(eps=-1.0) == L.PQ_EINVAL and step(wd=-1.0) == L.PQ_EINVAL
    assert step(n=4) == L.PQ_EINVAL and step(n=4, partials=P, norm=P, most=0.0) == L.PQ_EINVAL and step(n=-1) == L.PQ_ESHAPE
    assert step(_list(L, tensors=None)) == L.PQ_EINVAL and step(_list(L, first=[0, 3, 1])) == L.PQ_ESHAPE
    assert step(_list(L, first=[1, 2, 3])) == L.PQ_ESHAPE
    assert step(_list(L, (), ())) == L.PQ_OK                       # nothing to do
    assert step(_list(L, grads=(None, None))) == L.PQ_OK           # no gradient: no launch
    assert step(_list(L, (0,), (256,))) == L.PQ_OK


def test_norm_and_moments_refusals():
    L, lib = _lib()
    lst = _list(L)
    assert lib.pq_grad_squares_partials(ctypes.byref(lst)) == 1     # four chunks: one workgroup
    assert lib.pq_grad_squares_partials(ctypes.byref(_list(L, grads=(None, None)))) == 0
    many = _list(L, [5000] * 1000, [256] * 1000)
    assert 3 <= lib.pq_grad_squares_partials(ctypes.byref(many)) <= 3 * 2048
    assert lib.pq_grad_squares(ctypes.byref(lst), None, 1, None) == L.PQ_EINVAL
    assert lib.pq_grad_squares(ctypes.byref(many), P, 2, None) == L.PQ_ESHAPE
    join = lib.pq_grad_squares_join
    assert join(None, 4, P, None) == L.PQ_EINVAL and join(P, 4, None, None) == L.PQ_EINVAL and join(P, 0, P, None) == L.PQ_ESHAPE
    s = L.AdamWStates(P, P, P, P, 4096, 8)
    empty = L.AdamWStates(P, P, P, P, 0, 8)
    assert lib.pq_adamw_moments(ctypes.byref(s), None, P, 0, None) == L.PQ_EINVAL
    assert lib.pq_adamw_moments(ctypes.byref(s), P, P, 2, None) == L.PQ_EDTYPE
    assert lib.pq_adamw_moments(ctypes.byref(s), ODD, P, 0, None) == L.PQ_EALIGN
    assert lib.pq_adamw_moments(ctypes.byref(empty), None, None, 0, None) == L.PQ_OK
    assert lib.pq_adamw_load(ctypes.byref(s), P, None, None) == L.PQ_EINVAL and lib.pq_adamw_load(ctypes.byref(s), P, ODD, None) == L.PQ_EALIGN


def test_optimizer_refusals():
    from pyraquant_amd.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(8))
    for kw in (dict(bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(max_norm=0.0), dict(max_norm=-1.0)):
        with pytest.raises(AssertionError):
            AdamW([p], **kw)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(8, dtype=torch.float64))])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(8, dtype=torch.float64))]})
    assert len(opt.param_groups) == 1
    p.grad = torch.ones(8)
    with pytest.raises(AssertionError, match="GPU only"):
        opt.step()


def test_held_values_by_hand():
    """One block whose largest value is 1.9: E = 0, and the grid of means is (1 + i / 8) 2^(j - 15) without its first."""
    grid = sorted((1 + i / 8) * 2.0 ** (j - 15) for i in range(8) for j in range(16))[1:]
    a = np.zeros(128)
    a[:8] = 1.9, -0.3, 2.0 ** -15, 1.06 * 2.0 ** -15, 2.0 ** -15 * 1.07, 2.0 ** -20, 0.4218, 0.4219
    got = ref.held(a, 3, 0.5)
    near = lambda x: min(grid, key=lambda v: abs(v - x))   # noqa: E731
    assert got[0] == 1.875 and got[1] == -near(0.3) and got[2] == 0 and got[3] == 0 and got[4] == 1.125 * 2.0 ** -15 and got[5] == 0
    assert got[6] == 0.40625 and got[7] == 0.4375 and not got[8:].any()
    root = ref.held(np.abs(a), 4, 0.5)
    assert root[5] == 1.0625 * 2.0 ** -15 and root[0] == 1.875 and not root[8:].any()
    # rounding up past the binade, and the block's exponent after it
    a = np.zeros(128)
    a[0], a[1] = 1.99, 2.0 ** -14 * 1.01
    assert ref.held(a, 3, 0.5)[0] == 2.0 and ref.held(a, 3, 0.5)[1] == 0.0 and ref.held(a, 3, 0.0)[0] == 1.875


def test_hash_is_even():
    """2^18 places, 4 steps, 2 seeds: the means of both halves, their covariance and those of neighbouring places, steps and seeds are
    within 5 standard deviations of independent even values (mean 1/2, variance 1/12; a product of two has one of 1/144)."""
    n = 1 << 18
    places = np.arange(n)
    draws = [ref.dither(places, t, s) for s in (0, 1) for t in (1, 2, 100, 101)]
    flat = [h - 0.5 for d in draws for h in d]
    for h in flat:
        assert abs(h.mean()) < 5 * (1 / 12 / n) ** 0.5
        assert abs((h[1:] * h[:-1]).mean()) < 5 / 12 / n ** 0.5 and abs((h[128:] * h[:-128]).mean()) < 5 / 12 / n ** 0.5
    for i, a in enumerate(flat):
        for b in flat[:i]:
            assert abs((a * b).mean()) < 5 / 12 / n ** 0.5
