"""The sums over rows of 4-bit layers where fp16 values of t and dt are small, or of many sizes.

Two parts hold a value to 2 u^2 of it (u = 2^-11), or to half of fp16's smallest subnormal, 2^-25, on a scale on which the largest of a rank's values of
64 rows is at least 2^15: 2^-40 of that. f = 2^-24: M sums and some hundred of slices; u of the result, at least 2^-25 of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F, U = 2.0 ** -24, 2.0 ** -11


@pytest.mark.parametrize("size", (1e-3, 1e-6, 1e-8, 1e5))
@pytest.mark.parametrize("M,K,N,R", [(2050, 160, 336, 32), (700, 544, 48, 20), (4352, 64, 64, 64), (65, 96, 32, 40)])
def test_factor_gradients_of_small_values(cuda, M, K, N, R, size):
    from pyraquant_amd.mxfp4 import checkpoint_values, lowrank_grads, quant_mxfp4

    g = torch.Generator(device="cuda").manual_seed(M)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)   # noqa: E731
    P = 32 if R <= 32 else 64
    ranks = torch.zeros(P, device=cuda)
    ranks[:R] = 4.0 ** -(torch.arange(R, device=cuda) % 8)     # (others are 2^-14 of the largest)
    scale = 1e-3 / size
    x, dy = (r(M, K) * min(scale, 1e3)).half(), (r(M, N) * min(scale, 1e3)).half()
    t, dt = (r(M, P) * size * ranks for _ in range(2))
    q, q8 = quant_mxfp4(x, checkpoint=True)
    dA, dB, _ = lowrank_grads(dy, t, dt, q8, q.scales, R)
    for got, v, z in ((dA.t(), dt, checkpoint_values(q8, q, torch.float32)), (dB, t, dy)):
        v, z = v[:, :R].double(), z.double()
        want = v.t() @ z
        part = 2 * U * U * v.abs() + 2.0 ** -40 * v.abs().amax(0, keepdim=True)
        off = part.t() @ z.abs() + (M + 300) * F * (v.abs().t() @ z.abs())
        off = off + U * (want.abs() + off) + 2.0 ** -25
        fits = want.abs() < 60000
        over = (got.double() - want).abs() - off
        assert bool((over <= 0)[fits].all()), (size, float(over.max()))


def test_infinities_stay_in_their_rank_and_rows(cuda):
    """An infinite or a NaN value of t takes its rank's gradients with it, and no others'; a huge one in other rows costs a rank's no bits."""
    from pyraquant_amd.mxfp4 import lowrank_grads

    g = torch.Generator(device="cuda").manual_seed(0)
    M, N, R = 300, 64, 32
    t, dy = torch.randn(M, R, generator=g, device=cuda) * 1e-6, (torch.randn(M, N, generator=g, device=cuda) * 1e3).half()
    clean = lowrank_grads(dy, t, None, None, None, R, want_A=False, want_bias=False)[1]
    for bad in (float("inf"), float("nan")):
        v = t.clone()
        v[77, 5] = bad
        got = lowrank_grads(dy, v, None, None, None, R, want_A=False, want_bias=False)[1]
        keep = torch.arange(R, device=cuda) != 5
        assert not got[5].isfinite().any() and torch.equal(got[keep], clean[keep])
    v, d = t.clone(), dy.clone()
    v[77, 5], d[77] = 1e9, 0
    want = t.double().t() @ d.double()
    got = lowrank_grads(d, v, None, None, None, R, want_A=False, want_bias=False)[1]
    rows = torch.arange(M, device=cuda) // 64 != 1            # (the 64 rows that share a scale with it)
    part = v.double()[rows].abs().t() @ d.double()[rows].abs()
    lost = 2.0 ** -40 * 1e9 * d.double()[~rows].abs().sum(0)
    off = 2 * U * U * part + (M + 300) * F * (v.double().abs().t() @ d.double().abs())
    off[5] += lost
    off = off + 2 * U * U * (v.double()[~rows].abs().t() @ d.double()[~rows].abs()) + 2.0 ** -40 * 1e-5 * d.double().abs().sum(0)
    assert bool(((got.double() - want).abs() <= off + U * (want.abs() + off) + 2.0 ** -25).all())
