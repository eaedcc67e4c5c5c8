"""Choices of adapters by threads and in backward passes, and what AdapterSet refuses, without a GPU."""
import copy
import pickle
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from pyraquant_amd.adapters import AdaptedLinear, AdapterSet, LowRankAdapters, add_adapters


class _Thread(threading.Thread):
    """Runs what it is given in turn, and hands results and exceptions back."""

    def __init__(self):
        super().__init__(daemon=True)
        self._todo, self._done, self._go, self._back = None, None, threading.Semaphore(0), threading.Semaphore(0)
        self.start()

    def run(self):
        while True:
            self._go.acquire()
            if self._todo is None:
                return
            try:
                self._done = (self._todo(), None)
            except Exception as e:   # noqa: BLE001
                self._done = (None, e)
            self._back.release()

    def __call__(self, todo):
        self._todo = todo
        self._go.release()
        assert self._back.acquire(timeout=30)
        out, e = self._done
        if e is not None:
            raise e
        return out

    def end(self):
        self._todo = None
        self._go.release()
        self.join(30)


def test_threads_choose_for_themselves():
    styles = AdapterSet({})
    a, b = torch.tensor([0]), torch.tensor([1])
    one, two = _Thread(), _Thread()
    assert styles.ids is None and one(lambda: styles.ids) is None
    with styles.use(a):
        assert styles.ids is a and one(lambda: styles.ids) is a       # (no choice of its own: the only one there is)
        inner = one(lambda: styles.use(b))
        assert styles.ids is a and one(lambda: styles.ids) is b
        with pytest.raises(RuntimeError, match="threads"):
            two(lambda: styles.ids)
        two(lambda: styles.use(None))
        assert two(lambda: styles.ids) is None and styles.ids is a
        one(lambda: inner.__exit__(None, None, None))
        two(lambda: styles.use(a))
        assert one(lambda: styles.ids) is a                            # (all that have chosen have chosen the same)
    assert two(lambda: styles.ids) is a and styles.ids is a
    two.end()
    assert styles.ids is None                                          # (a choice goes with its thread)
    one.end()


def test_choices_nest_and_stay():
    styles = AdapterSet({})
    a, b = torch.tensor([0]), torch.tensor([1])
    styles.use(a)
    with styles.use(b):
        with styles.use(None):
            assert styles.ids is None
        assert styles.ids is b
    assert styles.ids is a
    styles.ids = b
    assert styles.ids is b
    styles.use(None)
    assert styles.ids is None


def test_models_with_adapters_are_copied():
    model = torch.nn.Sequential(torch.nn.Linear(16, 8), torch.nn.Linear(8, 8))
    styles = add_adapters(model, 2, 4, whitelist=lambda n: False)
    ids = torch.tensor([1])
    with styles.use(ids):
        for other, its in (copy.deepcopy((model, styles)), pickle.loads(pickle.dumps((model, styles)))):
            assert its is not styles and its.layers["0"] is other[0].adapters and other[0]._chosen is its and torch.equal(its.ids, ids)
            with its.use(None):
                assert styles.ids is ids and its.ids is None


class _Twice(torch.nn.Module):
    """Stands for adapters, which need a GPU: 2 y, with something kept for the backward pass (what keeps nothing is not computed again)."""

    def forward(self, x, y, ids, out=None):
        return y * torch.full_like(y, 2)


@pytest.mark.parametrize("reentrant", (True, False))
def test_a_block_computed_again_without_its_choice_raises(reentrant):
    styles = AdapterSet({})
    net = torch.nn.Sequential(AdaptedLinear(torch.nn.Linear(4, 4), _Twice(), styles))
    x = torch.randn(3, 4, requires_grad=True)
    ids = torch.tensor([0, 1, 2])
    with styles.use(ids):
        net(x).sum().backward()
        want = x.grad.clone()
        x.grad = None
        checkpoint(net, x, use_reentrant=reentrant).sum().backward()
        assert torch.equal(x.grad, want)
        out = checkpoint(net, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="chosen"):
        out.sum().backward()
    x.grad = None
    checkpoint(net, x, use_reentrant=reentrant).sum().backward()       # without adapters in both passes
    assert torch.equal(2 * x.grad, want)
    styles.use(ids)                                                    # (a choice that stays)
    out = checkpoint(net, x, use_reentrant=reentrant)
    x.grad = None
    out.sum().backward()
    assert torch.equal(x.grad, want)


def test_a_set_that_is_refused_changes_nothing():
    a, b = LowRankAdapters(16, 8, 2, 4), LowRankAdapters(8, 8, 2, 4)
    styles = AdapterSet({"a": a, "b": b})
    good = {"a": (torch.ones(16, 4), torch.ones(4, 8)), "b": (torch.ones(8, 2), torch.ones(2, 8))}
    styles.set(0, good)
    before = [t.clone() for t in (*a.buffers(), *b.buffers())]
    for slot, factors, scale in ((0, {"a": good["b"]}, 1.0), (0, {"a": (good["a"][0] * 2, good["a"][1]), "b": (torch.ones(8, 5), torch.ones(5, 8))}, 1.0),
                                 (2, good, 1.0), (0, {"a": good["a"], "c": good["b"]}, 1.0), (1, {"b": (torch.ones(8), torch.ones(8))}, 1.0),
                                 (1, good, "x")):
        with pytest.raises((AssertionError, ValueError)):
            styles.set(slot, factors, scale)
        assert all(torch.equal(t, o) for t, o in zip((*a.buffers(), *b.buffers()), before))
    with pytest.raises(ValueError, match="dtype"):
        LowRankAdapters(16, 8, 2, 4, trainable=True).freeze(torch.float64)
    with pytest.raises(ValueError, match="dtype"):
        styles.freeze(torch.int8)
