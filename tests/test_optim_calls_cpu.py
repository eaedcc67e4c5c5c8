"""What AdamW does without a kernel: hooks of a state dict that is loaded, groups' numbers."""
import copy

import pytest
import torch

from pyraquant_amd.optim import AdamW


def test_states_without_values():
    """Null pointers where there are no states, and then no list that has values."""
    import ctypes

    import pyraquant_amd._lib as L

    lib, P = L.load(), ctypes.c_void_p(256)
    for bits in (8, 32):
        s, r = L.AdamWStates(None, None, None, None, 0, bits), L.AdamWRates(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None, 0)
        for size, want in ((0, L.PQ_OK), (1000, L.PQ_ESHAPE)):
            lst = L.AdamWList(P, P, (ctypes.c_int64 * 2)(0, (size + 1023) // 1024), (ctypes.c_void_p * 1)(256), 1)
            assert lib.pq_adamw_step(ctypes.byref(lst), ctypes.byref(s), ctypes.byref(r), None, 0, None, None) == want
        assert lib.pq_adamw_moments(ctypes.byref(s), None, None, 0, None) == L.PQ_OK and lib.pq_adamw_load(ctypes.byref(s), None, None, None) == L.PQ_OK


def _saved(opt, n=8):
    state = {0: {"step": torch.tensor([3], dtype=torch.int32), "exp_avg": torch.arange(n, dtype=torch.float32), "exp_avg_sq": torch.full((n,), 2.0 ** -40)}}
    return {"state": state, "param_groups": copy.deepcopy(opt.state_dict()["param_groups"])}


def test_load_hooks_see_the_states():
    """Hooks before the load get the whole state dict and may give another one; hooks after it find the states, in their own types."""
    p = torch.nn.Parameter(torch.zeros(8, dtype=torch.bfloat16))
    opt = AdamW([p], lr=1e-3)
    saved, seen = _saved(opt), []

    def first(o, d):
        seen.append(sorted(d["state"][0]))
        d = copy.deepcopy(d)
        d["state"][0]["exp_avg"] += 1
        d["param_groups"][0]["lr"] = 0.5
        return d

    opt.register_load_state_dict_pre_hook(first)
    opt.register_load_state_dict_pre_hook(lambda o, d: seen.append(float(d["state"][0]["exp_avg"][0])))
    opt.register_load_state_dict_post_hook(lambda o: seen.append({k: v.clone() for k, v in o.state[p].items()}))
    opt.load_state_dict(saved)
    names, value, after = seen
    assert names == ["exp_avg", "exp_avg_sq", "step"] and value == 1.0
    assert torch.equal(after["exp_avg"], torch.arange(8.0) + 1) and after["exp_avg_sq"].dtype == torch.float32
    assert float(after["exp_avg_sq"][0]) == 2.0 ** -40 and after["step"].dtype == torch.int32 and opt.param_groups[0]["lr"] == 0.5
    assert saved["state"][0]["exp_avg"][0] == 0 and opt.state[p]["exp_avg"] is not saved["state"][0]["exp_avg"]
    later = opt.state_dict()
    assert torch.equal(later["state"][0]["exp_avg"], after["exp_avg"])
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 2      # (none of the load's own is left)
    other = AdamW([torch.nn.Parameter(torch.zeros(8))])
    with pytest.raises(ValueError):
        other.load_state_dict({"state": {}, "param_groups": []})
    assert not other._optimizer_load_state_dict_pre_hooks and not other.state


def test_hooks_see_every_groups_states():
    a, b = (torch.nn.Parameter(torch.zeros(8)) for _ in range(2))
    opt = AdamW([{"params": [a]}, {"params": [b]}], lr=1e-3)
    d = _saved(opt)
    d["state"][1] = {k: v + 1 for k, v in d["state"][0].items()}
    opt.load_state_dict(d)
    assert int(opt.state[a]["step"]) == 3 and int(opt.state[b]["step"]) == 4 and len(opt.state) == 2
    other = AdamW([{"params": [b]}, {"params": [a]}], lr=1e-3)
    other.load_state_dict(opt.state_dict())
    assert int(other.state[b]["step"]) == 3 and int(other.state[a]["step"]) == 4
