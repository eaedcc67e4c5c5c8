"""Microscaled 4-bit entries without a GPU: arguments are refused before any HIP call, and the oracle's format agrees with a
table written out by hand."""
import ctypes

import torch

from oracle import mxfp4_ref as ref

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _lib():
    import pyraquant_amd._lib as L

    return L, L.load()


def test_quant_refusals():
    L, lib = _lib()
    call = lambda x=P, dt=0, M=4, K=64, ldx=64, c=P, s=P, q8=None: lib.pq_mx_quant(x, dt, M, K, ldx, c, s, q8, None)   # noqa: E731
    assert call(K=48, ldx=48) == L.PQ_ESHAPE and call(K=0, ldx=0) == L.PQ_ESHAPE and call(ldx=32) == L.PQ_ESHAPE
    assert call(M=-1) == L.PQ_ESHAPE and call(dt=2) == L.PQ_EDTYPE
    assert call(x=None) == L.PQ_EINVAL and call(c=None) == L.PQ_EINVAL and call(s=None) == L.PQ_EINVAL
    assert call(c=ODD) == L.PQ_EALIGN and call(q8=ODD) == L.PQ_EALIGN and call(x=ctypes.c_void_p(257)) == L.PQ_EALIGN
    assert call(M=1 << 33, K=1 << 12, ldx=1 << 12) == L.PQ_ESHAPE and b"32-bit dispatch" in lib.pq_last_error()
    assert call(M=0, x=None, c=None, s=None) == L.PQ_OK
    vals = lambda bits=4, K=64, ldo=64, dt=0, out=P: lib.pq_mx_values(P, P, bits, 4, K, out, dt, ldo, None)   # noqa: E731
    assert vals(bits=5) == L.PQ_EINVAL and vals(K=40) == L.PQ_ESHAPE and vals(ldo=68) == L.PQ_EALIGN
    assert vals(dt=2) == L.PQ_EDTYPE and vals(out=None) == L.PQ_EINVAL


def test_gemm_and_gradient_refusals():
    L, lib = _lib()

    def gemm(a=P, bias=None, t=None, ldt=0, l2t=None, R=0, c=P, ldc=64, dt=0, M=4, N=64, K=64):
        return lib.pq_mx_gemm(a, P, P, P, bias, t, ldt, l2t, R, c, ldc, dt, M, N, K, None)

    assert gemm(K=48) == L.PQ_ESHAPE and gemm(N=40) == L.PQ_ESHAPE and gemm(ldc=56) == L.PQ_ESHAPE
    assert gemm(dt=3) == L.PQ_EDTYPE and gemm(a=None) == L.PQ_EINVAL and gemm(c=ODD) == L.PQ_EALIGN
    assert gemm(ldc=68) == L.PQ_EALIGN and gemm(bias=ODD) == L.PQ_EALIGN
    assert gemm(t=P, ldt=16, l2t=P, R=16) == L.PQ_ESHAPE and gemm(t=P, ldt=32, R=32) == L.PQ_EINVAL
    assert gemm(t=P, ldt=36, l2t=P, R=32) == L.PQ_EALIGN and gemm(t=P, ldt=16, l2t=P, R=32) == L.PQ_ESHAPE
    assert gemm(M=(1 << 30) + 1) == L.PQ_ESHAPE and gemm(M=0, a=None, c=None) == L.PQ_OK

    def dx(dy=P, ld=64, dt=None, ap=None, R=0, out=P, ldo=64, ty=0, M=4, N=64, K=64):
        return lib.pq_mx_grad_input(dy, ty, ld, P, P, dt, ap, R, out, ldo, M, N, K, None, 0, None)

    assert dx(N=24, ld=24) == L.PQ_ESHAPE and dx(K=33, ldo=40) == L.PQ_ESHAPE and dx(ld=32) == L.PQ_ESHAPE
    assert dx(ty=3) == L.PQ_EDTYPE and dx(dy=None) == L.PQ_EINVAL and dx(dy=ODD) == L.PQ_EALIGN and dx(ldo=68) == L.PQ_EALIGN
    assert dx(dt=P, ap=P, R=48) == L.PQ_ESHAPE and dx(dt=P, R=32) == L.PQ_EINVAL and dx(M=0, dy=None) == L.PQ_OK

    big = dict(M=64, N=12288, K=1280, ld=12288, ldo=1280)      # few rows, a long sum: split, in a workspace
    assert lib.pq_mx_grad_input_workspace_size(64, 12288, 1280) > 0 and dx(**big) == L.PQ_EINVAL
    assert b"workspace" in lib.pq_last_error() and lib.pq_mx_grad_input_workspace_size(65536, 3072, 3072) == 0
    assert dx(ld=(1 << 21) + 8) == L.PQ_ESHAPE

    def factors(dy=P, t=P, dt=P, q8=P, sc=P, M=4, K=64, N=64, R=8, PP=32, dA=P, dB=P, ws=P, size=1 << 40, ty=0):
        return lib.pq_mx_grad_factors(dy, ty, N, t, dt, q8, sc, M, K, N, R, PP, dA, dB, P, ws, size, None)

    assert factors(PP=16) == L.PQ_ESHAPE and factors(R=33) == L.PQ_ESHAPE and factors(M=0) == L.PQ_ESHAPE
    assert factors(ty=3) == L.PQ_EDTYPE and factors(t=None) == L.PQ_EINVAL and factors(q8=None) == L.PQ_EINVAL
    assert factors(dy=ODD) == L.PQ_EALIGN and factors(size=16) == L.PQ_ESHAPE and factors(ws=None) == L.PQ_EINVAL
    assert lib.pq_mx_grad_factors_workspace_size(0, 64, 64, 32) == 0
    small, large = (lib.pq_mx_grad_factors_workspace_size(m, 64, 64, 32) for m in (1, 100000))
    assert 0 < small < large

    def lay(A=P, K=64, N=64, R=8, PP=32, lda=8, ldb=64, ao=0, bo=1, out=P):
        return lib.pq_mx_factors(A, lda, ao, P, ldb, bo, K, N, R, PP, out, P, P, P, None)

    assert lay(R=40) == L.PQ_ESHAPE and lay(PP=48) == L.PQ_ESHAPE and lay(lda=4) == L.PQ_ESHAPE and lay(A=None) == L.PQ_EINVAL
    assert lay(ldb=32) == L.PQ_ESHAPE and lay(ao=3) == L.PQ_EINVAL and lay(out=ODD) == L.PQ_EALIGN
    down = lambda x=P, K=64, ldx=64, R=32, dt=0, t=P: lib.pq_mx_lowrank_down(x, dt, 4, K, ldx, P, R, t, None, 0, None)   # noqa: E731
    assert down(K=24, ldx=24) == L.PQ_ESHAPE and down(R=16) == L.PQ_ESHAPE and down(ldx=32) == L.PQ_ESHAPE
    assert down(dt=3) == L.PQ_EDTYPE and down(x=None) == L.PQ_EINVAL and down(ldx=68) == L.PQ_EALIGN and down(t=ODD) == L.PQ_EALIGN

    def layer(x=P, ldx=64, R=0, l1=None, l2=None, t=None, y=P, codes=P, dt=0, M=4, K=64, N=64):
        return lib.pq_mx_linear(x, dt, M, K, ldx, P, P, None, l1, l2, R, y, N, N, codes, P, None, t, None, 0, None)

    assert layer(K=48) == L.PQ_ESHAPE and layer(N=24) == L.PQ_ESHAPE and layer(R=16) == L.PQ_ESHAPE and layer(ldx=32) == L.PQ_ESHAPE
    assert layer(dt=3) == L.PQ_EDTYPE and layer(x=None) == L.PQ_EINVAL and layer(codes=None) == L.PQ_EINVAL
    assert layer(R=32, l1=P, l2=P) == L.PQ_EINVAL and layer(y=ODD) == L.PQ_EALIGN and layer(ldx=68) == L.PQ_EALIGN
    assert lib.pq_mx_lowrank_workspace_size(512, 12288, 32) > 0 and lib.pq_mx_lowrank_workspace_size(4096, 12288, 32) == 0
    assert layer(M=512, K=12288, ldx=12288, R=32, l1=P, l2=P, t=P) == L.PQ_EINVAL and b"workspace" in lib.pq_last_error()
    assert down(K=12288, ldx=12288) == L.PQ_EINVAL and b"workspace" in lib.pq_last_error()
    assert layer(M=0, x=None, y=None, codes=None) == L.PQ_OK


def test_python_layer_refuses_cpu_tensors():
    import pytest

    from pyraquant_amd.mxfp4 import Mxfp4Linear, quant_mxfp4

    with pytest.raises(AssertionError):
        quant_mxfp4(torch.zeros(4, 64))
    with pytest.raises(AssertionError):
        Mxfp4Linear(torch.nn.Linear(64, 32))


def test_oracle_grid():
    """A block whose largest value is 6: E = 0, and every tie goes to the even neighbour."""
    x = torch.zeros(1, 32, dtype=torch.float64)
    pairs = [(6, 6), (0.25, 0), (0.26, 0.5), (0.75, 1), (1.25, 1), (1.3, 1.5), (1.75, 2), (2.5, 2), (2.6, 3), (3.5, 4), (5, 4),
             (5.1, 6), (-0.75, -1), (-5, -4)]
    x[0, : len(pairs)] = torch.tensor([p[0] for p in pairs], dtype=torch.float64)
    want = torch.tensor([p[1] for p in pairs], dtype=torch.float64)
    assert torch.equal(ref.four_bits(x)[0, : len(pairs)], want)
    assert ref.exponents(x).item() == 0 and ref.exponents(x * 1.3).item() == 0 and ref.exponents(x * 1.4).item() == 1
    assert torch.equal(ref.four_bits(x * 1.3)[0, :1], torch.tensor([6.0], dtype=torch.float64))        # 7.8 saturates
    assert torch.equal(ref.eight_bits(x), (x * 16).round() / 16)
    x[0, 3] = float("inf")
    assert bool(torch.isnan(ref.four_bits(x)).all()) and ref.exponents(torch.zeros(1, 32)).item() == -127
