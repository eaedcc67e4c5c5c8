"""Microscaled 4-bit layers for MI355X (gfx950): Linears whose weights and activations are 4-bit floating point with a shared
power of two per 32 values, and the tuning of their low-rank branch over frozen weights.

  quant_mxfp4(x) -> Mxfp4Matrix                     rows to 4-bit codes and scales (and the 8-bit codes of a checkpoint)
  dequant_mxfp4(q, dtype)                            back to values
  checkpoint_values(q8, q, dtype)                    the values of the 8-bit codes
  mxfp4_gemm(xq, wq, bias, out_dtype, t=, l2t=)      the product, with the low-rank term and the bias in its epilogue
  mxfp4_grad_input(dy, wq, dt=, lr_Ap=)              the input's gradient, from the 4-bit weight as it is stored
  lowrank_grads(dy, t, dt, q8, xq, rank)             the gradients of lr_A, lr_B and the bias, from the 8-bit checkpoint
  Mxfp4Linear, convert_linears_to_mxfp4              the layer, and a model's Linears made into it

The format: E = floor(log2(max |x|)) - 2 over 32 consecutive values of a row, each held as the nearest of 0, 0.5, 1, 1.5, 2, 3,
4, 6 times 2^E (ties to an even last bit, saturated at 6). A block with an infinity or a NaN is NaN.

Tuning. ``Mxfp4Linear(lin, lowrank=(A, B), trainable=True)`` keeps the weight in 4 bits and makes lr_A, lr_B and the bias
parameters. What its backward pass keeps of the input are 8-bit codes, rint(x 2^(4 - E)) on the same E, written in the
quantizer's pass over x (half the bytes of x): they give lr_A's gradient. The rounding of x to 4 bits counts as the identity.
The layer has first derivatives of the reverse kind (a second one, or a forward-mode tangent, raises); the functions have none.

Every kernel runs on the caller's current stream; nothing synchronises. CPU tensors raise AssertionError; a missing library
raises at the first call.
"""
from __future__ import annotations

from typing import Callable, Dict, NamedTuple, Optional, Tuple

import torch
import torch.nn as nn

from . import _lib
from .int8_exec import LOWRANK_A_ATTR, LOWRANK_B_ATTR, is_bf16_whitelisted

BLOCK = 32        # values that share a scale
MAX_RANK = 64     # of a low-rank branch (the kernels hold 32 or 64; lower ranks run zero-padded)


class Mxfp4Matrix(NamedTuple):
    """A [rows, cols] matrix in 4 bits: packed codes and scales (flat uint8 tensors, pq_mx_quant's layout)."""

    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    cols: int


_mx = None   # _mx.so, loaded at the first use


def _load_mx():
    global _mx
    _mx = _lib.load_mx()
    return _mx


def _stages(rows: int, cols: int) -> int:
    return (rows + 15) // 16 * ((cols + 127) // 128)


def _check_cuda(*tensors) -> None:
    dev = None
    for t in tensors:
        if t is not None:
            assert t.is_cuda, "the 4-bit layers run on the GPU only (got a CPU tensor)"
            assert dev is None or t.device == dev, f"operands on {dev} and {t.device}"
            dev = t.device


def _check_matrix(q: Mxfp4Matrix) -> None:
    units = _stages(q.rows, q.cols)
    assert q.cols > 0 and q.cols % BLOCK == 0, q.cols
    for t, size in ((q.codes, 1024), (q.scales, 64)):
        assert t.dtype == torch.uint8 and t.is_contiguous() and t.numel() >= units * size, (t.dtype, tuple(t.shape), q.rows, q.cols)


def _dtype16(dt: torch.dtype) -> int:
    return _lib.dtype_code(dt)


def _plain(x: torch.Tensor) -> torch.Tensor:
    x = x.detach()
    return x.resolve_neg() if x.is_neg() else x


def _rows(x2: torch.Tensor, most: Optional[int] = None) -> torch.Tensor:
    """x2 as the kernels read it: rows of consecutive elements, 16-byte aligned, none over another, no further apart than ``most``
    (a copy where not)."""
    x2 = _plain(x2)
    M, K = x2.shape
    if (x2.stride(1) != 1 or x2.data_ptr() % 16
            or M > 1 and (x2.stride(0) < K or x2.stride(0) * x2.element_size() % 16 or most is not None and x2.stride(0) > most)):
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


def _stride(x2: torch.Tensor) -> int:
    """Row stride (that of a single row says nothing)."""
    return x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


# --------------------------------------------------------------------------- quantization
def quant_mxfp4(x2: torch.Tensor, checkpoint: bool = False):
    """x2 [M, K] (bf16, fp16 or fp32, K % 32 == 0) -> Mxfp4Matrix; with ``checkpoint`` (Mxfp4Matrix, q8): q8 [M, K] int8,
    the codes a backward pass keeps, on the same scales. Row-slice views pass without a copy."""
    codes, scales, q8 = (_mx or _load_mx()).quant(x2, checkpoint)
    q = Mxfp4Matrix(codes, scales, *x2.shape)
    return (q, q8) if checkpoint else q


def dequant_mxfp4(q: Mxfp4Matrix, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values a 4-bit matrix holds, [rows, cols] (exact in bf16 and fp32; in fp16 for scales of 2^-22 to 2^13)."""
    return (_mx or _load_mx()).values(q.codes, q.scales, 4, q.rows, q.cols, dtype)


def checkpoint_values(q8: torch.Tensor, q: Mxfp4Matrix, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of a checkpoint's 8-bit codes on the scales of the matrix quantized with them."""
    assert q8.dim() == 2 and tuple(q8.shape) == (q.rows, q.cols), (tuple(q8.shape), q.rows, q.cols)
    return (_mx or _load_mx()).values(q8, q.scales, 8, q.rows, q.cols, dtype)


# --------------------------------------------------------------------------- product and gradients
def mxfp4_gemm(xq: Mxfp4Matrix, wq: Mxfp4Matrix, bias: Optional[torch.Tensor], out_dtype: torch.dtype, *,
               t: Optional[torch.Tensor] = None, l2t: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[M, N] = xq @ wq^T (+ t @ l2t^T) (+ bias), summed in fp32, rounded once. t [M, R] in fp32 (taken to twice out_dtype's
    bits) or out_dtype, l2t [N, R] in out_dtype, R 32 or 64; bias fp32 [N]; N % 16 == 0."""
    _check_matrix(xq)
    _check_matrix(wq)
    _check_cuda(xq.codes, xq.scales, wq.codes, wq.scales, bias, t, l2t, out)
    assert xq.cols == wq.cols, (xq.cols, wq.cols)
    M, N, K = xq.rows, wq.rows, xq.cols
    code = _dtype16(out_dtype)
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.is_contiguous() and bias.numel() == N, (bias.dtype, tuple(bias.shape), N)
    R, ldt = 0, 0
    if t is not None:
        assert l2t is not None and l2t.dtype == out_dtype and t.dtype in (out_dtype, torch.float32) and l2t.is_contiguous()
        assert t.dim() == 2 and t.stride(1) == 1 and t.shape[0] >= M and tuple(l2t.shape) == (N, t.shape[1]), (tuple(t.shape), tuple(l2t.shape), M, N)
        t = _rows(_plain(t).float())   # (as the layer's own is)
        if _stride(t) % 8:
            t = t.contiguous()
        R, ldt = t.shape[1], _stride(t)
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=xq.codes.device)
    assert out.dtype == out_dtype and tuple(out.shape) == (M, N) and out.stride(1) == 1, (out.dtype, tuple(out.shape))
    _lib.check(_lib.load().pq_mx_gemm(_lib.ptr(xq.codes), _lib.ptr(xq.scales), _lib.ptr(wq.codes), _lib.ptr(wq.scales),
                                      _lib.ptr(bias), _lib.ptr(t), ldt, _lib.ptr(l2t), R, _lib.ptr(out), _stride(out), code,
                                      M, N, K, _lib.stream_of(out.device)), "mxfp4_gemm")
    return out


def mxfp4_grad_input(dy: torch.Tensor, wq: Mxfp4Matrix, dt: Optional[torch.Tensor] = None,
                     lr_Ap: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dx [M, K] = dy @ wq (+ dt @ lr_Ap^T): wq's values in dy's type, sums in fp32. dt [M, R] in fp32 or dy's type, lr_Ap
    [K, R] in dy's type, contiguous, R 32 or 64."""
    _check_matrix(wq)
    _check_cuda(dy, wq.codes, wq.scales, dt, lr_Ap)
    assert dy.dim() == 2 and dy.shape[1] == wq.rows, (tuple(dy.shape), wq.rows)
    code = _dtype16(dy.dtype)
    dy = _rows(dy, 1 << 21)   # (pq_mx_grad_input's limit)
    M, N, K = dy.shape[0], wq.rows, wq.cols
    R = 0
    if dt is not None:
        R = dt.shape[1]
        assert lr_Ap is not None and lr_Ap.dtype == dy.dtype and dt.dtype in (dy.dtype, torch.float32) and dt.is_contiguous() and lr_Ap.is_contiguous()
        assert tuple(dt.shape) == (M, R) and tuple(lr_Ap.shape) == (K, R), (tuple(dt.shape), tuple(lr_Ap.shape), M, K)
        dt = _plain(dt).float()
    dx = torch.empty((M, K), dtype=dy.dtype, device=dy.device)
    L = _lib.load()
    size = L.pq_mx_grad_input_workspace_size(M, N, K)
    ws = torch.empty(size, dtype=torch.uint8, device=dy.device) if size else None
    _lib.check(L.pq_mx_grad_input(_lib.ptr(dy), code, _stride(dy), _lib.ptr(wq.codes), _lib.ptr(wq.scales),
                                  _lib.ptr(dt), _lib.ptr(lr_Ap), R, _lib.ptr(dx), K, M, N, K, _lib.ptr(ws), size,
                                  _lib.stream_of(dy.device)), "mxfp4_grad_input")
    return dx


def _ranks(t: torch.Tensor, M: int, P: int, dtype: torch.dtype) -> torch.Tensor:
    """t or dt as lowrank_grads' kernels read it: fp32 [M, P], from that or from its two parts."""
    if t.dim() == 3:
        assert t.dtype == dtype and tuple(t.shape) == (2, M, P), (t.dtype, tuple(t.shape), dtype, M, P)
        t = t[0].float() + t[1].float()
    assert t.dtype == torch.float32 and tuple(t.shape) == (M, P), (t.dtype, tuple(t.shape), M, P)
    return _plain(t).contiguous()


def lowrank_grads(dy: Optional[torch.Tensor], t: Optional[torch.Tensor], dt: Optional[torch.Tensor], q8: Optional[torch.Tensor],
                  x_scales: Optional[torch.Tensor], rank: int, want_A: bool = True, want_B: bool = True, want_bias: bool = True):
    """(dA [K, rank], dB [rank, N], dbias [N] fp32), None for those not wanted: dB = t^T dy, dbias = sum of dy's rows, dA =
    checkpoint^T dt, in dy's type. t and dt are [M, P] in fp32, P 32 or 64 >= rank, zero past rank, or [2, M, P] in the type of
    the results, each the sum of its two parts (the value, and what that rounding left out); q8 and x_scales as quant_mxfp4 gave
    them. What no wanted gradient needs may be None; without a dy, fp32 dt gives dA in bf16."""
    if not (want_A or want_B or want_bias):
        return None, None, None
    _check_cuda(dy, t, dt, q8, x_scales)
    if not want_A:
        dt = q8 = x_scales = None
    if not want_B:
        t = None
    if not (want_B or want_bias):
        dy = None
    for wanted, operands in ((want_A, (dt, q8, x_scales)), (want_B, (dy, t)), (want_bias, (dy,))):
        assert not wanted or all(v is not None for v in operands), "an operand of a wanted gradient is None"
    ranks = dt if want_A else t
    P = _padded_rank(rank) if ranks is None else ranks.shape[-1]
    M, dev = (q8 if want_A else dy).shape[0], (q8 if want_A else dy).device
    dt16 = dy.dtype if dy is not None else dt.dtype if dt.dtype != torch.float32 else torch.bfloat16
    code = _dtype16(dt16)
    K = N = BLOCK
    if want_A:
        dt = _ranks(dt, M, P, dt16)
        assert q8.dim() == 2 and q8.dtype == torch.int8 and q8.is_contiguous(), (q8.dtype, tuple(q8.shape))
        K = q8.shape[1]
        assert x_scales.dtype == torch.uint8 and x_scales.is_contiguous() and x_scales.numel() >= _stages(M, K) * 64
    if want_B:
        t = _ranks(t, M, P, dt16)
    if dy is not None:
        assert dy.dim() == 2 and dy.shape[0] == M, (tuple(dy.shape), M)
        dy = _rows(dy)
        N = dy.shape[1]
    assert 1 <= rank <= P, (rank, P)
    dA = torch.empty((K, rank), dtype=dt16, device=dev) if want_A else None
    dB = torch.empty((rank, N), dtype=dt16, device=dev) if want_B else None
    db = torch.empty(N, dtype=torch.float32, device=dev) if want_bias else None
    if M == 0:
        return tuple(None if g is None else g.zero_() for g in (dA, dB, db))
    L = _lib.load()
    ws = torch.empty(L.pq_mx_grad_factors_workspace_size(M, K, N, P), dtype=torch.uint8, device=dev)
    _lib.check(L.pq_mx_grad_factors(_lib.ptr(dy), code, N if dy is None else _stride(dy), _lib.ptr(t), _lib.ptr(dt),
                                    _lib.ptr(q8), _lib.ptr(x_scales), M, K, N, rank, P, _lib.ptr(dA), _lib.ptr(dB),
                                    _lib.ptr(db), _lib.ptr(ws), ws.numel(), _lib.stream_of(dev)), "lowrank_grads")
    return dA, dB, db


def _padded_rank(R: int) -> int:
    assert 1 <= R <= MAX_RANK, f"rank {R}: the 4-bit layers take 1 to {MAX_RANK}"
    return 32 if R <= 32 else 64


def lay_out_factors(lr_A: torch.Tensor, lr_B: torch.Tensor):
    """lr_A [K, R] and lr_B [R, N] as the forward pass reads them, zero-padded to rank P (32 or 64): (lr_A's fragments
    [ceil(K / 128) * 128, P], pq_mx_factors' order, lr_B's rows [N, P]). Each in its own type."""
    _check_cuda(lr_A, lr_B)
    assert lr_A.dim() == 2 and lr_B.dim() == 2 and lr_A.shape[1] == lr_B.shape[0], (tuple(lr_A.shape), tuple(lr_B.shape))
    A, B = _plain(lr_A).contiguous(), _plain(lr_B).contiguous()
    (K, R), N = A.shape, B.shape[1]
    P = _padded_rank(R)
    if A.dtype != B.dtype or A.dtype not in (torch.bfloat16, torch.float16):   # (the kernel moves 16-bit values)
        Af, Bt = A.new_zeros(((K + 127) // 128 * 128, P)), B.new_zeros((N, P))
        Af[:K, :R], Bt[:, :R] = A, B.t()
        f = Af.reshape(-1, 4, 4, 8, P // 16, 16)    # stage, block, group, k, rank / 16, rank % 16
        return f.permute(0, 2, 4, 1, 5, 3).reshape(Af.shape).contiguous(), Bt
    Af = torch.empty(((K + 127) // 128 * 128, P), dtype=A.dtype, device=A.device)
    Bt = torch.empty((N, P), dtype=A.dtype, device=A.device)
    _lib.check(_lib.load().pq_mx_factors(_lib.ptr(A), R, _lib.PQ_MX_BY_COLUMN, _lib.ptr(B), N, _lib.PQ_MX_BY_RANK, K, N, R, P,
                                         _lib.ptr(Af), None, _lib.ptr(Bt), None, _lib.stream_of(A.device)), "lay_out_factors")
    return Af, Bt


# --------------------------------------------------------------------------- the layer
class Mxfp4Linear(nn.Module):
    """4-bit stand-in for nn.Linear: y = x4 @ w4^T (+ (x @ lr_A) @ lr_B) (+ bias), x4 and w4 the microscaled 4-bit values of x
    and the weight; in_features % 32 == 0, out_features % 16 == 0, low rank up to 64. Inputs are bf16 or fp16, and the
    low-rank factors are used in the input's type.

    Buffers ``weight_codes`` and ``weight_scales`` hold the weight. ``trainable=False`` keeps the bias in fp32 and the low-rank
    branch in the kernels' order as buffers (``lr_Af``, ``lr_Bt``: lay_out_factors; ``lr_A`` and ``lr_B`` give it back), in its own
    type or in ``dtype``: each call casts it where that is not the input's type. ``trainable=True`` (needs a low-rank branch) makes
    ``lr_A`` [K, R], ``lr_B`` [R, N] and ``bias`` parameters; freeze() turns such a layer into the other kind. Gradients flow to the
    input of either."""

    def __init__(self, lin: nn.Linear, device: Optional[torch.device] = None,
                 lowrank: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, trainable: bool = False,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        w = lin.weight.detach()
        if device is not None:
            w = w.to(device)
        self.out_features, self.in_features = N, K = w.shape
        assert N % 16 == 0 and N > 0, f"out_features {N} is not a multiple of 16"
        q = quant_mxfp4(w)
        self.register_buffer("weight_codes", q.codes)
        self.register_buffer("weight_scales", q.scales)
        A, B = lowrank if lowrank is not None else (getattr(lin, LOWRANK_A_ATTR, None), getattr(lin, LOWRANK_B_ATTR, None))
        self.rank = 0
        if A is not None and B is not None:
            A, B = A.detach().to(w.device), B.detach().to(w.device)
            assert A.dim() == 2 and B.dim() == 2 and A.shape[0] == K and B.shape == (A.shape[1], N), (
                tuple(A.shape), tuple(B.shape), K, N)
            self.rank = int(A.shape[1])
            _padded_rank(self.rank)
        assert self.rank or not trainable, "trainable=True tunes a low-rank branch, and the layer has none"
        self.trainable = bool(trainable)
        bias = None if lin.bias is None else lin.bias.detach().to(w.device, torch.float32).contiguous()
        if trainable:
            self.lr_A, self.lr_B = nn.Parameter(A.clone().contiguous()), nn.Parameter(B.clone().contiguous())
            self.register_parameter("bias", None if bias is None else nn.Parameter(bias.clone()))
        else:
            self._keep(A if self.rank else None, B if self.rank else None, bias, dtype)

    def _keep(self, A, B, bias, dtype) -> None:
        """The low-rank branch and the bias as buffers, the branch in the kernels' order."""
        Af = Bt = None
        if A is not None:
            Af, Bt = lay_out_factors(A.to(dtype or A.dtype), B.to(dtype or B.dtype))
        self.register_buffer("lr_Af", Af)
        self.register_buffer("lr_Bt", Bt)
        self.register_buffer("bias", bias)

    def freeze(self, dtype: Optional[torch.dtype] = None) -> "Mxfp4Linear":
        """Turns a trainable layer into one that serves: its low-rank branch laid out once, nothing left to tune, the same outputs.
        Give the inputs' type as ``dtype`` where the factors are in another (fp32 masters), and no call has to cast them."""
        if self.trainable:
            A, B, bias = self.lr_A.detach(), self.lr_B.detach(), self.bias
            del self.lr_A, self.lr_B, self.bias
            self.trainable = False
            self._keep(A, B, None if bias is None else bias.detach().float().contiguous(), dtype)
        return self

    def __getattr__(self, name):
        if name in ("lr_A", "lr_B") and "lr_Af" in self.__dict__.get("_buffers", ()):
            if self.lr_Af is None:
                return None
            if name == "lr_B":
                return self.lr_Bt[:, : self.rank].t().contiguous()
            f = self.lr_Af.reshape(-1, 4, self.lr_Af.shape[1] // 16, 4, 16, 8)    # stage, group, rank / 16, block, rank % 16, k
            return f.permute(0, 3, 1, 5, 2, 4).reshape(self.lr_Af.shape)[: self.in_features, : self.rank].contiguous()
        return super().__getattr__(name)

    def _apply(self, fn, recurse=True):
        """A module-wide cast leaves a bias buffer in fp32, as the kernels read it."""
        keep = self._buffers.get("bias")
        super()._apply(fn, recurse)
        new = self._buffers.get("bias")
        if keep is not None and new.dtype != torch.float32:
            self._buffers["bias"] = keep.to(new.device)
        return self

    def weight(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values of the 4-bit weight, [N, K]."""
        return dequant_mxfp4(Mxfp4Matrix(self.weight_codes, self.weight_scales, self.out_features, self.in_features), dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        assert x.shape[-1] == self.in_features, (tuple(x.shape), self.in_features)
        d, p, trainable = self._buffers, self._parameters, self.trainable
        if trainable:
            A, B = p["lr_A"], p["lr_B"]
        else:
            A, B = d["lr_Af"], d["lr_Bt"]
        bias = d["bias"] if "bias" in d else p["bias"] if "bias" in p else self.bias   # (assigning one makes it a parameter or not)
        dt = x.dtype
        if A is not None and (A.dtype != dt or B.dtype != dt) and dt in (torch.bfloat16, torch.float16):
            A, B = A.to(dt), B.to(dt)
        if bias is not None and bias.dtype != torch.float32:
            bias = bias.float()
        return (_mx or _load_mx()).layer(x, d["weight_codes"], d["weight_scales"], A, B, bias, self.out_features, not trainable)

    def extra_repr(self) -> str:
        lr = f", low-rank r={self.rank}" + (" (trainable)" if self.trainable else "") if self.rank else ""
        return f"in={self.in_features}, out={self.out_features}, mxfp4 W / A{lr} (HIP gfx950)"


# --------------------------------------------------------------------------- model conversion
def convert_linears_to_mxfp4(model: nn.Module, device: Optional[str] = "cuda",
                             whitelist: Callable[[str], bool] = is_bf16_whitelisted,
                             trainable: bool = False) -> Dict[str, object]:
    """Replaces the token-level nn.Linear layers by Mxfp4Linear in place, as convert_linears_to_int8 does by Int8Linear, and
    returns the same kind of statistics. Layers that the 4-bit kernels do not take (in_features % 32, out_features % 16, a
    branch of a rank above 64, 64-bit weights) stay as they are, with the whitelisted ones. A low-rank branch attached under
    LOWRANK_A_ATTR / LOWRANK_B_ATTR is carried over: frozen in the weight's type where that has 16 bits (an nn.Linear's inputs
    have it); with ``trainable`` the branches, as they are, and the biases of the layers that have one become parameters, and every
    other parameter of the model is left as it is."""
    dev = torch.device(device) if device is not None else None
    n4, n_keep, p4, p_keep, kept = 0, 0, 0, 0, []
    for name, lin in [(n, m) for n, m in model.named_modules() if isinstance(m, nn.Linear)]:
        A, B = getattr(lin, LOWRANK_A_ATTR, None), getattr(lin, LOWRANK_B_ATTR, None)
        has_lr = A is not None and B is not None
        if (whitelist(name) or lin.in_features % BLOCK or lin.out_features % 16 or has_lr and not 1 <= A.shape[-1] <= MAX_RANK
                or lin.weight.dtype not in (torch.bfloat16, torch.float16, torch.float32)):
            n_keep += 1
            p_keep += lin.weight.numel()
            kept.append(name)
            continue
        parent_name, _, attr = name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        setattr(parent, attr, Mxfp4Linear(lin, device=dev, trainable=trainable and has_lr,
                                          dtype=lin.weight.dtype if lin.weight.dtype != torch.float32 else None))
        n4 += 1
        p4 += lin.weight.numel()
        del lin
    if dev is not None and dev.type == "cuda":
        torch.cuda.synchronize()
    return {"n_mxfp4_linear": n4, "n_bf16_linear_kept": n_keep, "params_mxfp4": p4, "params_bf16_linear_kept": p_keep,
            "bf16_kept_names": kept, "mxfp4_weight_gib": p4 * (1 / 2 + 1 / BLOCK) / 2**30, "bf16_equiv_gib": p4 * 2 / 2**30}
