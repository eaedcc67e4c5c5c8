"""Adapters' entries without a GPU: arguments are refused before any HIP call, and the modules' own checks."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _lib():
    import pyraquant_amd._lib as L

    return L, L.load()


def test_down_and_up_refusals():
    L, lib = _lib()

    def down(x=P, ty=0, M=4, K=64, ldx=64, f=P, slots=2, PP=16, ids=P, bits=32, each=1, part=P):
        return lib.pq_adapter_down(x, ty, M, K, ldx, f, slots, PP, ids, bits, each, part, None)

    assert down(K=60, ldx=60) == L.PQ_ESHAPE and down(K=0) == L.PQ_ESHAPE and down(ldx=56) == L.PQ_ESHAPE and down(M=-1) == L.PQ_ESHAPE
    assert down(PP=8) == L.PQ_ESHAPE and down(PP=128) == L.PQ_ESHAPE and down(M=(1 << 30) + 1) == L.PQ_ESHAPE and down(K=1 << 25, ldx=1 << 25) == L.PQ_ESHAPE
    assert down(ty=3) == L.PQ_EDTYPE and down(bits=16) == L.PQ_EDTYPE
    assert down(slots=0) == L.PQ_ESHAPE and down(slots=65536) == L.PQ_ESHAPE and down(each=0) == L.PQ_ESHAPE and down(each=3) == L.PQ_ESHAPE
    assert down(x=None) == L.PQ_EINVAL and down(f=None) == L.PQ_EINVAL and down(ids=None) == L.PQ_EINVAL and down(part=None) == L.PQ_EINVAL
    assert down(x=ODD) == L.PQ_EALIGN and down(ldx=68) == L.PQ_EALIGN and down(f=ODD) == L.PQ_EALIGN and down(ids=ctypes.c_void_p(258)) == L.PQ_EALIGN
    assert down(ids=ctypes.c_void_p(260), bits=64) == L.PQ_EALIGN
    assert down(M=0, x=None, f=None, ids=None, part=None) == L.PQ_OK

    def up(part=P, slices=1, scale=P, g=P, slots=2, C=64, R=8, PP=16, ids=P, bits=32, each=1, base=P, ldb=64, out=P, ldo=64, joined=None, ty=0, M=4):
        return lib.pq_adapter_up(part, slices, scale, g, slots, C, R, PP, ids, bits, each, base, ldb, out, ldo, joined, ty, M, None)

    assert up(C=60) == L.PQ_ESHAPE and up(ldo=56) == L.PQ_ESHAPE and up(ldb=56) == L.PQ_ESHAPE and up(R=17) == L.PQ_ESHAPE and up(R=0) == L.PQ_ESHAPE
    assert up(slices=0) == L.PQ_ESHAPE and up(slices=17) == L.PQ_ESHAPE and up(ty=3) == L.PQ_EDTYPE and up(ldb=72) == L.PQ_ESHAPE
    assert up(ldo=(1 << 30) + 8) == L.PQ_ESHAPE and up(base=ctypes.c_void_p(512), ldb=(1 << 30) + 8) == L.PQ_ESHAPE
    assert up(part=None) == L.PQ_EINVAL and up(scale=None) == L.PQ_EINVAL and up(g=None) == L.PQ_EINVAL and up(out=None) == L.PQ_EINVAL
    assert up(out=None, joined=P) == L.PQ_EINVAL and up(joined=ODD) == L.PQ_EALIGN       # (a base without a result)
    assert up(out=ODD) == L.PQ_EALIGN and up(base=ODD) == L.PQ_EALIGN and up(ldo=68) == L.PQ_EALIGN and up(base=ctypes.c_void_p(512), ldb=68) == L.PQ_EALIGN
    assert up(M=0, part=None, out=None) == L.PQ_OK

    def rows(x=P, ty=0, M=4, K=64, ldx=64, f=P, scale=P, g=P, slots=2, C=64, R=8, PP=16, ids=P, bits=32, each=1, base=P, ldb=64, out=P, ldo=64, joined=None):
        return lib.pq_adapter_rows(x, ty, M, K, ldx, f, scale, g, slots, C, R, PP, ids, bits, each, base, ldb, out, ldo, joined, None)

    far = ctypes.c_void_p(512)
    assert rows(K=60) == L.PQ_ESHAPE and rows(C=60) == L.PQ_ESHAPE and rows(ldx=56) == L.PQ_ESHAPE and rows(ldo=56) == L.PQ_ESHAPE and rows(ldb=56) == L.PQ_ESHAPE
    assert rows(M=-1) == L.PQ_ESHAPE and rows(M=(1 << 16) + 1) == L.PQ_ESHAPE and rows(R=17) == L.PQ_ESHAPE and rows(PP=8) == L.PQ_ESHAPE
    assert rows(each=3) == L.PQ_ESHAPE and rows(slots=0) == L.PQ_ESHAPE and rows(ldb=72) == L.PQ_ESHAPE and rows(ty=2) == L.PQ_EDTYPE and rows(bits=8) == L.PQ_EDTYPE
    assert all(rows(**{k: None}) == L.PQ_EINVAL for k in ("x", "f", "scale", "g", "ids")) and rows(out=None) == L.PQ_EINVAL
    assert rows(out=None, joined=P) == L.PQ_EINVAL and rows(out=None, base=None) == L.PQ_EINVAL
    assert all(rows(**{k: ODD}) == L.PQ_EALIGN for k in ("x", "f", "g", "base", "out", "joined"))
    assert rows(ldx=68) == L.PQ_EALIGN and rows(base=far, ldb=68) == L.PQ_EALIGN and rows(base=far, ldo=68) == L.PQ_EALIGN
    assert rows(M=0, x=None, out=None) == L.PQ_OK
    fit = lib.pq_adapter_rows_fit
    assert fit(1, 1280, 1280, 16, 1) and fit(154, 2048, 1280, 16, 77) and not fit(8192, 640, 640, 16, 1) and not fit(1, 1 << 20, 64, 16, 1) and not fit(1, 60, 64, 16, 1)


def test_gradient_and_order_refusals():
    L, lib = _lib()

    def grads(x=P, ldx=64, dy=P, lddy=64, ty=0, t=P, dt=P, ids=P, bits=32, each=1, M=4, K=64, N=64, slots=2, R=8, PP=16,
              dA=P, dB=P, ws=P, size=1 << 40):
        return lib.pq_adapter_grads(x, ldx, dy, lddy, ty, t, dt, ids, bits, each, M, K, N, slots, R, PP, dA, dB, ws, size, None)

    assert grads(K=60) == L.PQ_ESHAPE and grads(N=4) == L.PQ_ESHAPE and grads(ldx=56) == L.PQ_ESHAPE and grads(lddy=56) == L.PQ_ESHAPE
    assert grads(R=17) == L.PQ_ESHAPE and grads(size=64) == L.PQ_ESHAPE
    assert grads(ty=2) == L.PQ_EDTYPE and grads(bits=8) == L.PQ_EDTYPE and grads(each=3) == L.PQ_ESHAPE
    assert grads(x=None) == L.PQ_EINVAL and grads(t=None) == L.PQ_EINVAL and grads(dt=None) == L.PQ_EINVAL and grads(dy=None) == L.PQ_EINVAL
    assert grads(ws=None) == L.PQ_EINVAL
    assert grads(x=ODD) == L.PQ_EALIGN and grads(lddy=68) == L.PQ_EALIGN and grads(ws=ODD) == L.PQ_EALIGN
    assert grads(dA=None, dB=None) == L.PQ_OK
    size = lib.pq_adapter_grads_workspace_size
    assert size(4, 60, 64, 2, 16, 1) == 0 and size(4, 64, 64, 0, 16, 1) == 0 and size(4, 64, 64, 2, 16, 3) == 0
    assert 0 < size(4, 64, 64, 2, 16, 1) < size(100000, 64, 64, 2, 16, 1)
    assert 1 <= lib.pq_adapter_slices(1, 65536) <= 16 and lib.pq_adapter_slices(1 << 20, 64) == 1 and lib.pq_adapter_slices(0, 64) == 1
    lay = lambda A=P, B=P, slots=2, K=64, N=64, R=8, PP=16, at=P, bt=P, oa=0, ob=1: lib.pq_adapter_factors(   # noqa: E731
        A, oa, B, ob, slots, K, N, R, PP, at, None, None, bt, None)
    assert lay(oa=4) == L.PQ_EINVAL and lay(ob=-1) == L.PQ_EINVAL and lay(A=ODD, oa=2) == L.PQ_EALIGN
    assert lib.pq_adapter_factor_size(136, 32) == 256 * 32 and lib.pq_adapter_factor_size(60, 32) == 0 and lib.pq_adapter_factor_size(64, 8) == 0
    assert lay(K=4) == L.PQ_ESHAPE and lay(R=17) == L.PQ_ESHAPE and lay(slots=0) == L.PQ_ESHAPE
    assert lay(A=None) == L.PQ_EINVAL and lay(B=None) == L.PQ_EINVAL and lay(A=None, B=None, at=None, bt=None) == L.PQ_OK and lay(at=ODD) == L.PQ_EALIGN


def test_module_refusals():
    from pyraquant_amd.adapters import AdapterSet, LowRankAdapters, add_adapters

    for args in ((60, 64, 2, 8), (64, 4, 2, 8), (64, 64, 0, 8), (64, 64, 65536, 8), (64, 64, 2, 0), (64, 64, 2, 65)):
        with pytest.raises(AssertionError):
            LowRankAdapters(*args)
    with pytest.raises(ValueError):
        LowRankAdapters(64, 64, 2, 8, dtype=torch.float64)
    bank = LowRankAdapters(64, 32, 2, 8)
    for slot, A, B in ((2, (64, 8), (8, 32)), (-1, (64, 8), (8, 32)), (0, (64, 9), (9, 32)), (0, (64, 8), (4, 32)), (0, (32, 8), (8, 32))):
        with pytest.raises(AssertionError):
            bank.set(slot, torch.zeros(A), torch.zeros(B))
    x, y = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="GPU only"):
        bank(x, y, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(AssertionError):
        AdapterSet({"a": bank}).set(0, {"b": (torch.zeros(64, 8), torch.zeros(8, 32))})
    with pytest.raises(AssertionError, match="itself a Linear"):
        add_adapters(torch.nn.Linear(64, 32), 2, 8)


@pytest.mark.parametrize("trainable", (False, True))
def test_slots_hold_what_was_set(trainable):
    """Factors in and out of either kind, ranks below the module's, a cleared slot, a cast, freeze(), a state dict."""
    from pyraquant_amd.adapters import LowRankAdapters

    bank = LowRankAdapters(64, 40, 3, 20, trainable=trainable)
    A, B = torch.randn(64, 12).bfloat16(), torch.randn(12, 40).bfloat16()
    bank.set(1, A, B, 0.5)
    bank.set(2, A, B)
    bank.clear(2)
    assert bank.scale.tolist() == [0.0, 0.5, 0.0]
    assert torch.equal(bank.lr_A[1, :, :12], A) and torch.equal(bank.lr_B[1, :12], B) and not bank.lr_A[1, :, 12:].any() and not bank.lr_B[2].any()
    assert (len(list(bank.parameters())) == 2) == trainable
    other = LowRankAdapters(64, 40, 3, 20, trainable=trainable)
    other.load_state_dict(bank.state_dict())
    assert torch.equal(other.lr_A, bank.lr_A) and torch.equal(other.scale, bank.scale)
    bank.half()
    assert bank.scale.dtype == torch.float32 and bank.lr_A.dtype == torch.float16
    frozen = bank.freeze()
    assert not list(frozen.parameters()) and not frozen.trainable and torch.equal(frozen.lr_B[1, :12], B.half())


def test_a_models_layers_get_adapters():
    from pyraquant_amd.adapters import AdaptedLinear, add_adapters
    from pyraquant_amd.weights import SplitInLinear

    model = torch.nn.ModuleDict({"up": torch.nn.Linear(64, 128), "proj_out": torch.nn.Linear(64, 64), "odd": torch.nn.Linear(60, 64),
                                 "split": SplitInLinear(torch.nn.Linear(128, 64), 48), "deep": torch.nn.Sequential(torch.nn.Linear(32, 64))})
    kept = {k: list(p.shape) for k, p in model.named_parameters()}
    styles = add_adapters(model, 4, 8, trainable=True, whitelist=lambda n: n == "proj_out")
    assert sorted(styles.layers) == ["deep.0", "split", "up"]
    assert isinstance(model["split"], AdaptedLinear) and isinstance(model["split"].layer, SplitInLinear)
    assert isinstance(model["odd"], torch.nn.Linear) and isinstance(model["proj_out"], torch.nn.Linear) and model["up"].out_features == 128
    assert len(styles.parameters()) == 6 and len(list(model.parameters())) == len(kept) + 6
    x = torch.randn(3, 64)
    assert torch.equal(model["up"](x), model["up"].layer(x))          # nothing chosen
    styles.set(1, {"up": (torch.ones(64, 3), torch.ones(3, 128))}, 2.0)
    got = styles.get(1)
    assert sorted(got) == ["deep.0", "split", "up"] and not got["split"][0].any() and got["up"][1].shape == (8, 128)
    ids = torch.tensor([0, 1])
    with styles.use(ids) as s:
        assert s.ids is ids
        with styles.use(None):
            assert styles.ids is None
        assert styles.ids is ids
    assert styles.ids is None
    styles.freeze()
    assert not styles.parameters()


def test_a_layer_in_two_places_gets_one_set():
    from pyraquant_amd.adapters import AdaptedLinear, add_adapters

    tied = torch.nn.Linear(64, 64)
    model = torch.nn.ModuleDict({"a": tied, "b": torch.nn.Sequential(tied), "c": torch.nn.Linear(64, 64)})
    styles = add_adapters(model, 2, 8, whitelist=lambda n: False)
    assert sorted(styles.layers) == ["a", "c"] and model["b"][0] is model["a"] and isinstance(model["a"], AdaptedLinear)
    assert model["a"].layer is tied
