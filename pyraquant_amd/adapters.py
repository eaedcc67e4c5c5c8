"""Low-rank adapters of many requests at once beside one shared projection, for MI355X (gfx950).

  LowRankAdapters(in, out, slots, rank)(x, y, ids)    y + scale[id] (x lr_A[id]) lr_B[id], id the adapter of each row's request
  AdaptedLinear, add_adapters(model, slots, rank)     a model's Linears with adapters beside them
  AdapterSet                                          the handle of a model's adapters: load, clear, and choose them for a batch

The layers of int8_exec and mxfp4 hold one low-rank branch that belongs to the weight. Adapters belong to requests: a model is
quantized once, styles or customers are tuned as small factors, and one batch serves any of them together, or tunes them together.
``ids`` is an integer tensor on the GPU, one for each row or for each of x's leading dimensions (a batch of images: one an image), or, where
LowRankAdapters is called with flat rows, one for each request of M / len(ids) rows that follow each other;
an id that names no adapter (-1) leaves its rows as they are. The kernels read ids, factors and scales when they run, so a
captured graph follows what is written there.

No request's results depend on what the others of its batch hold or choose (the number of rows chooses the kernels, and with them
the last bit). t = x lr_A is held in fp32 and taken to twice the factors' bits. Calls have first
derivatives of the reverse kind (a second one, or a forward-mode tangent, raises; so does a step that is captured while an eager graph of
its leaves lives). Every kernel runs on the caller's
current stream; nothing synchronises. CPU tensors raise AssertionError; a missing library raises at the first call.
"""
from __future__ import annotations

import threading
import weakref
from typing import Callable, Dict, List, Mapping, Optional, Set, Tuple

import torch
import torch.nn as nn
from torch.nn.modules import module as _module

from . import _lib
from .int8_exec import Int8Linear, is_bf16_whitelisted
from .mxfp4 import Mxfp4Linear
from .weights import SplitInLinear

MAX_RANK = 64     # of an adapter (the kernels hold 16, 32 or 64; other ranks run zero-padded)

_adapt = None   # _adapt.so, loaded at the first use


def _load_adapt():
    global _adapt
    _adapt = _lib.load_adapt().adapt
    return _adapt


def _check_dtype(dtype: torch.dtype) -> None:
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"unsupported dtype {dtype} (expected bfloat16, float16 or float32)")


def _padded(rank: int) -> int:
    return 16 if rank <= 16 else 32 if rank <= 32 else 64


def _room(columns: int) -> int:
    return (columns + 127) // 128 * 128


# The kernels' orders (pq_adapter_factors' PQ_ADAPTER_DOWN and PQ_ADAPTER_UP) as views with the axes of a matrix [..., columns, ranks]:
# where a value lies is given by parts of its column and of its rank.
def _down_axes(f: torch.Tensor) -> torch.Tensor:
    """f [..., C, P] in the order of `down` -> [..., C / 32, 4, 8, P / 16, 16], the parts of c and of r"""
    C, P = f.shape[-2:]
    v = f.reshape(*f.shape[:-2], C // 32, P // 16, 4, 16, 8)      # c / 32, r / 16, c / 8 % 4, r % 16, c % 8
    return v.movedim((-5, -3, -1, -4, -2), (-5, -4, -3, -2, -1))


def _up_axes(f: torch.Tensor) -> torch.Tensor:
    """f [..., C, P] in the order of `up` -> [..., C / 128, 16, 8, P / 8, 8], the parts of c and of r"""
    C, P = f.shape[-2:]
    v = f.reshape(*f.shape[:-2], C // 128, 8, P // 8, 16, 8)      # c / 128, c % 8, r / 8, c / 8 % 16, r % 8
    return v.movedim((-5, -2, -4, -3, -1), (-5, -4, -3, -2, -1))


def _write(axes: torch.Tensor, m: torch.Tensor, C: int, P: int) -> None:
    """m [..., c, r] into a factor's order, zeros past its columns and ranks."""
    full = m.new_zeros((*m.shape[:-2], C, P))
    full[..., : m.shape[-2], : m.shape[-1]] = m
    axes.copy_(full.view(axes.shape))


def _lay_out(A: torch.Tensor, B: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> None:
    """A [slots, K, r] and B [slots, r, N] into a and b, [slots, C, P] in the orders of `down` and of `up`: one launch on the GPU for 16 bits. (4096 x
    4096, rank 16, 32 slots set one by one: 1.1 ms, 1.9 with tensor operations; frozen at once 60 us, 119.)"""
    P = a.shape[-1]
    if a.is_cuda and b.device == a.device and b.dtype == a.dtype and a.dtype in (torch.bfloat16, torch.float16) and a.is_contiguous() and b.is_contiguous():
        A, B = A.resolve_neg().contiguous(), B.resolve_neg().contiguous()
        (slots, K, r), N = A.shape, B.shape[2]
        with torch.cuda.device(a.device):
            _lib.check(_lib.load().pq_adapter_factors(_lib.ptr(A), _lib.PQ_ADAPTER_BY_COLUMN, _lib.ptr(B), _lib.PQ_ADAPTER_BY_RANK, slots, K, N, r, P,
                                                      _lib.ptr(a), None, None, _lib.ptr(b), _lib.stream_of(a.device)), "adapters")
        for t in (a, b):
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)
    else:
        _write(_down_axes(a), A, a.shape[1], P)
        _write(_up_axes(b), B.transpose(1, 2), b.shape[1], P)


class LowRankAdapters(nn.Module):
    """``slots`` adapters of a projection: ``adapters(x, y, ids)`` is y + scale[id] (x lr_A[id]) lr_B[id]. x [..., in_features] and y
    [..., out_features] in bf16 or fp16, features multiples of 8, ranks up to 64; ids as the module says. ``out=`` takes the result, y
    itself for one: rows without an adapter are not touched then. (Only where nothing needs a gradient.)

    ``trainable=False`` keeps the factors in the kernels' orders as buffers (``lr_Af`` and ``lr_Bf``, [slots, features rounded up to 128,
    P]; ``lr_A`` and ``lr_B`` give them back). ``trainable=True`` makes ``lr_A`` [slots, K, rank] and ``lr_B`` [slots, rank, N]
    parameters; freeze() turns such a module into the other kind. Factors of another type than x's are cast in each call. ``scale``
    is a buffer in fp32, 0 for an empty slot. Gradients flow to x and y of either kind; adapters without rows get zeros."""

    def __init__(self, in_features: int, out_features: int, slots: int, rank: int, *, dtype: torch.dtype = torch.bfloat16,
                 device=None, trainable: bool = False):
        super().__init__()
        assert in_features > 0 and in_features % 8 == 0, f"in_features {in_features} is not a multiple of 8"
        assert out_features > 0 and out_features % 8 == 0, f"out_features {out_features} is not a multiple of 8"
        assert 1 <= slots <= 65535, f"{slots} adapters (1 to 65535)"
        assert 1 <= rank <= MAX_RANK, f"rank {rank}: adapters take 1 to {MAX_RANK}"
        _check_dtype(dtype)
        self.in_features, self.out_features, self.slots, self.rank = in_features, out_features, slots, rank
        self.trainable = bool(trainable)
        zeros = lambda *shape: torch.zeros(shape, dtype=dtype, device=device)   # noqa: E731
        if trainable:
            self.lr_A = nn.Parameter(zeros(slots, in_features, rank))
            self.lr_B = nn.Parameter(zeros(slots, rank, out_features))
        else:
            P = _padded(rank)
            self.register_buffer("lr_Af", zeros(slots, _room(in_features), P))
            self.register_buffer("lr_Bf", zeros(slots, _room(out_features), P))
        self.register_buffer("scale", torch.zeros(slots, device=device))

    def _slot(self, slot: int) -> int:
        assert 0 <= slot < self.slots, f"slot {slot} of {self.slots}"
        return slot

    def _fitting(self, slot: int, lr_A: torch.Tensor, lr_B: torch.Tensor, scale: float) -> Tuple[int, int, float]:
        r = lr_A.shape[-1] if lr_A.dim() else 0
        assert tuple(lr_A.shape) == (self.in_features, r) and tuple(lr_B.shape) == (r, self.out_features) and 1 <= r <= self.rank, (
            tuple(lr_A.shape), tuple(lr_B.shape), self.in_features, self.out_features, self.rank)
        return self._slot(slot), r, float(scale)

    @torch.no_grad()
    def set(self, slot: int, lr_A: torch.Tensor, lr_B: torch.Tensor, scale: float = 1.0) -> None:
        """An adapter into a slot: lr_A [K, r], lr_B [r, N], r up to the rank (zeros past it). On the current stream; captured graphs
        take it from their next replay on."""
        slot, r, scale = self._fitting(slot, lr_A, lr_B, scale)
        if self.trainable:
            for to, what in ((self.lr_A[slot], lr_A), (self.lr_B[slot].t(), lr_B.t())):
                to[:, :r].copy_(what)
                to[:, r:].zero_()
        else:
            a, b = self.lr_Af, self.lr_Bf
            _lay_out(lr_A[None].to(a.device, a.dtype), lr_B[None].to(b.device, b.dtype), a[slot : slot + 1], b[slot : slot + 1])
        self.scale[slot] = scale

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """An empty slot: its rows get y + 0."""
        slot = self._slot(slot)
        for t in (self.lr_A, self.lr_B) if self.trainable else (self.lr_Af, self.lr_Bf):
            t[slot].zero_()
        self.scale[slot] = 0.0

    def freeze(self, dtype: Optional[torch.dtype] = None) -> "LowRankAdapters":
        """Turns a trainable module into one that serves, in ``dtype`` (give the inputs' type where the factors are in another), with the
        same outputs."""
        if dtype is not None:
            _check_dtype(dtype)
        if self.trainable:
            A, B, P = self.lr_A.detach(), self.lr_B.detach(), _padded(self.rank)
            A, B = A.to(dtype or A.dtype), B.to(dtype or B.dtype)
            del self.lr_A, self.lr_B
            self.trainable = False
            a, b = A.new_zeros((self.slots, _room(self.in_features), P)), B.new_zeros((self.slots, _room(self.out_features), P))
            with torch.no_grad():
                _lay_out(A, B, a, b)
            self.register_buffer("lr_Af", a)
            self.register_buffer("lr_Bf", b)
        return self

    def __getattr__(self, name):
        if name in ("lr_A", "lr_B") and "lr_Af" in self.__dict__.get("_buffers", ()):
            if name == "lr_A":
                return _down_axes(self.lr_Af).reshape(self.lr_Af.shape)[:, : self.in_features, : self.rank].contiguous()
            return _up_axes(self.lr_Bf).reshape(self.lr_Bf.shape)[:, : self.out_features, : self.rank].transpose(1, 2).contiguous()
        return super().__getattr__(name)

    def _apply(self, fn, recurse=True):
        """A module-wide cast leaves the scales in fp32, as the kernels read them."""
        keep = self._buffers["scale"]
        super()._apply(fn, recurse)
        new = self._buffers["scale"]
        if new.dtype != torch.float32:
            self._buffers["scale"] = keep.to(new.device)
        return self

    def forward(self, x: torch.Tensor, y: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        assert x.shape[-1] == self.in_features and y.shape[-1] == self.out_features, (tuple(x.shape), tuple(y.shape), self.in_features, self.out_features)
        if self.trainable:
            p = self._parameters
            A, B = p["lr_A"], p["lr_B"]
        else:
            d = self._buffers
            A, B = d["lr_Af"], d["lr_Bf"]
        dt = x.dtype
        if (A.dtype != dt or B.dtype != dt) and dt in (torch.bfloat16, torch.float16):
            A, B = A.to(dt), B.to(dt)
        return (_adapt or _load_adapt())(x, y, ids, A, B, self._buffers["scale"], self.rank, not self.trainable, out)

    def extra_repr(self) -> str:
        kind = " (trainable)" if self.trainable else ""
        return f"in={self.in_features}, out={self.out_features}, {self.slots} adapters, r={self.rank}{kind} (HIP gfx950)"


class _Choice:
    """What a thread has chosen."""

    __slots__ = ("ids", "__weakref__")

    def __init__(self, ids: Optional[torch.Tensor]):
        self.ids = ids


class AdapterSet:
    """The adapters of a model (add_adapters): one slot in every adapted layer. ``use(ids)`` chooses those of the batches that follow, None
    none of them; as a context manager it puts the earlier choice back.

    A choice is its thread's own. Threads that have made none, autograd's among them, go by the others' while those agree; where they do not,
    ``ids`` raises. A block that is computed again in a backward pass (checkpointed) needs the choice of its forward pass there too; a layer whose
    last call had one raises where none is left."""

    def __init__(self, layers: Dict[str, LowRankAdapters]):
        self.layers = layers
        self._mine = threading.local()
        self._all: Set["weakref.ref[_Choice]"] = set()      # of threads that live (each operation on it is one of the interpreter's)

    def __getstate__(self):
        own = getattr(self._mine, "choice", None)
        return {"layers": self.layers, "ids": own and own.ids}

    def __setstate__(self, state) -> None:
        self.__init__(state["layers"])
        if state["ids"] is not None:
            self.use(state["ids"])

    @property
    def ids(self) -> Optional[torch.Tensor]:
        """What is chosen in this thread."""
        own = getattr(self._mine, "choice", None)
        if own is not None:
            return own.ids
        if not self._all:
            return None
        others = [c.ids for c in (r() for r in list(self._all)) if c is not None]
        for other in others[1:]:
            if other is not others[0]:
                raise RuntimeError("threads have chosen different adapters of a set, and this one has not: use(ids) here too")
        return others[0] if others else None

    @ids.setter
    def ids(self, ids: Optional[torch.Tensor]) -> None:
        self.use(ids)

    def _choose(self, choice: Optional[_Choice]) -> Optional[_Choice]:
        before = getattr(self._mine, "choice", None)
        if before is not None:
            self._all.discard(weakref.ref(before))
        if choice is not None:
            self._all.add(weakref.ref(choice, self._all.discard))
        self._mine.choice = choice
        return before

    def use(self, ids: Optional[torch.Tensor]) -> "_Chosen":
        return _Chosen(self, self._choose(_Choice(ids)))

    def set(self, slot: int, factors: Mapping[str, Tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0) -> None:
        """An adapter of the model into a slot: {layer's name: (lr_A, lr_B)}; layers that it does not name get none."""
        unknown = sorted(set(factors) - set(self.layers))
        assert not unknown, f"not adapted layers: {unknown[:4]}"
        for name, (lr_A, lr_B) in factors.items():      # (all, before any slot changes)
            self.layers[name]._fitting(slot, lr_A, lr_B, scale)
        for name, bank in self.layers.items():
            if name in factors:
                bank.set(slot, *factors[name], scale)
            else:
                bank.clear(slot)

    def get(self, slot: int) -> Dict[str, Tuple[torch.Tensor, torch.Tensor]]:
        """{layer's name: (lr_A, lr_B)} of a slot, as set() takes them."""
        return {name: (bank.lr_A[bank._slot(slot)].detach().clone(), bank.lr_B[slot].detach().clone()) for name, bank in self.layers.items()}

    def clear(self, slot: int) -> None:
        for bank in self.layers.values():
            bank.clear(slot)

    def parameters(self) -> List[nn.Parameter]:
        """What tuning the adapters steps (none of frozen ones)."""
        return [p for bank in self.layers.values() for p in bank.parameters()]

    def freeze(self, dtype: Optional[torch.dtype] = None) -> "AdapterSet":
        for bank in self.layers.values():
            bank.freeze(dtype)
        return self


class _Chosen:
    def __init__(self, adapters: AdapterSet, before: Optional[_Choice]):
        self._adapters, self._before = adapters, before

    def __enter__(self) -> AdapterSet:
        return self._adapters

    def __exit__(self, *exc) -> None:
        self._adapters._choose(self._before)


def _gives_new(layer: nn.Module) -> bool:
    """Whether a layer's result is a new tensor that no hook has seen. (A class of the user's own, or a call in the place of the layer's, may
    hand out anything.)"""
    if layer._forward_hooks or _module._global_forward_hooks or "forward" in layer.__dict__:
        return False
    kind = type(layer)
    return kind in (nn.Linear, Int8Linear, Mxfp4Linear) or kind is SplitInLinear and all(map(_gives_new, layer.linears))


class AdaptedLinear(nn.Module):
    """A projection that requests share and the adapters beside it: layer(x), and what ``chosen.ids`` says is added to it. (Routed
    calls, with rows gathered or scattered, are a TypeError: their rows are not a batch's.)"""

    def __init__(self, layer: nn.Module, adapters: LowRankAdapters, chosen: AdapterSet):
        super().__init__()
        self.layer, self.adapters = layer, adapters
        self._chosen = chosen
        self._adapted = False      # whether the last call had a choice

    @property
    def in_features(self) -> int:
        return self.layer.in_features

    @property
    def out_features(self) -> int:
        return self.layer.out_features

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self.layer(x)
        ids, d = self._chosen.ids, self.__dict__
        if ids is None:
            if d.get("_adapted") and torch.is_grad_enabled() and torch._C._current_graph_task_id() != -1:
                raise RuntimeError("a layer is computed again in a backward pass, and the adapters that its forward pass had are not chosen any more: "
                                   "call backward inside `with use(ids)` where blocks are checkpointed")
            d["_adapted"] = False
            return y
        d["_adapted"] = True
        assert x.dim() != 2 or ids.dim() != 1 or ids.shape[0] == x.shape[0], f"{x.shape[0]} rows and ids of {ids.shape[0]}: a layer's rows are the batch's"
        # without gradients what is added goes into the layer's result, where nobody else can hold that
        return self.adapters(x, y, ids, out=y if not torch.is_grad_enabled() and _gives_new(self.layer) and y.is_contiguous() else None)


def add_adapters(model: nn.Module, slots: int, rank: int, *, dtype: Optional[torch.dtype] = None, trainable: bool = False,
                 whitelist: Callable[[str], bool] = is_bf16_whitelisted) -> AdapterSet:
    """Puts adapters beside the token-level Linears of a model in place (Int8Linear, Mxfp4Linear, SplitInLinear and nn.Linear whose features
    are multiples of 8, but for whitelisted names, as the converters take them; convert first). All slots are empty. ``dtype``: the factors', bf16 if
    not given. Where ``trainable``, the factors are the only parameters added; every other is left as it is."""
    chosen = AdapterSet({})
    inside = set()      # (modules of a layer that is taken)
    made: Dict[nn.Module, AdaptedLinear] = {}
    for name, layer in list(model.named_modules(remove_duplicate=False)):
        if not isinstance(layer, (nn.Linear, Int8Linear, Mxfp4Linear, SplitInLinear)) or whitelist(name) or layer in inside:
            continue
        assert name, "the model is itself a Linear: wrap it in a module"
        if layer.in_features % 8 or layer.out_features % 8:
            continue
        if layer not in made:      # (a layer in several places: one set of adapters, under its first name)
            first = next(iter([*layer.buffers(), *layer.parameters()]))
            bank = LowRankAdapters(layer.in_features, layer.out_features, slots, rank, dtype=dtype or torch.bfloat16, device=first.device,
                                   trainable=trainable)
            made[layer] = AdaptedLinear(layer, bank, chosen)
            inside.update(m for m in layer.modules() if m is not layer)
            chosen.layers[name] = bank
        parent, _, attr = name.rpartition(".")
        setattr(model.get_submodule(parent) if parent else model, attr, made[layer])
    return chosen
