"""CPU: states, settings and sizes of the token-level operators that are unusual, as far as they can be seen without a device."""
import copy

import pytest
import torch


def _params():
    return [torch.nn.Parameter(torch.zeros(6, 4)), torch.nn.Parameter(torch.zeros(6)), torch.nn.Parameter(torch.zeros(9, 6))]


def _adamw_state(make):
    """A state with AdamW's entries for every parameter, in the groups of ``make``."""
    opt = make()
    for group in opt.param_groups:
        for p in group["params"]:
            opt.state[p] = {"step": torch.tensor(3.0), "exp_avg": torch.ones_like(p), "exp_avg_sq": torch.ones_like(p)}
    return copy.deepcopy(opt.state_dict())


@pytest.mark.parametrize("source", ["fused", "torch"])
def test_a_group_keeps_its_muon_settings_when_an_adamw_state_is_loaded(source):
    from ssecg.optim import FusedAdamW, FusedMuon
    a, b, head = _params()
    muon = FusedMuon([{"params": [a, b], "momentum": 0.8, "ns_steps": 3, "adjust_lr": "original", "nesterov": False, "ns_eps": 1e-6},
                      {"params": [head], "muon": False}], lr=0.3)
    kind = FusedAdamW if source == "fused" else torch.optim.AdamW
    muon.load_state_dict(_adamw_state(lambda: kind([{"params": _params()[:2]}, {"params": _params()[2:], "lr": 0.07}], lr=1e-2)))
    body, rest = muon.param_groups
    assert (body["muon"], body["momentum"], body["ns_steps"], body["adjust_lr"], body["nesterov"], body["ns_eps"]) == (True, 0.8, 3, "original", False, 1e-6)
    assert rest["muon"] is False and rest["momentum"] == 0.95
    assert body["lr"] == 1e-2 and rest["lr"] == 0.07                     # what the state has comes from the state
    assert set(muon.state[head]) == set(muon.state[b]) == {"step", "exp_avg", "exp_avg_sq"}
    assert not muon.state[a]                                             # the matrix starts anew and keeps no AdamW tensors


def test_a_muon_state_brings_its_settings():
    from ssecg.optim import FusedMuon
    a, b, head = _params()
    first = FusedMuon([{"params": [a, b], "momentum": 0.7}, {"params": [head], "muon": False}])
    first.state[a]["momentum_buffer"] = torch.full_like(a, 2.0)
    c, d, other = _params()
    second = FusedMuon([{"params": [c, d]}, {"params": [other]}])
    second.load_state_dict(copy.deepcopy(first.state_dict()))
    assert [(g["muon"], g["momentum"]) for g in second.param_groups] == [(True, 0.7), (False, 0.95)]
    assert torch.equal(second.state[c]["momentum_buffer"], torch.full_like(c, 2.0))


def test_a_state_that_a_group_cannot_take_is_refused_whole():
    from ssecg.optim import FusedMuon
    big, small = torch.nn.Parameter(torch.empty((1 << 20) + 1, 2)), torch.nn.Parameter(torch.zeros(4, 2))
    opt = FusedMuon([{"params": [small]}, {"params": [big], "muon": False}], lr=0.1)
    for at, change in ((1, {"muon": True}), (0, {"momentum": 1.5}), (0, {"adjust_lr": "other"}), (0, {"ns_steps": 0})):
        state = copy.deepcopy(opt.state_dict())
        state["param_groups"][at].update(change, lr=0.9)
        with pytest.raises(ValueError):
            opt.load_state_dict(state)
        assert [g["lr"] for g in opt.param_groups] == [0.1, 0.1] and opt.param_groups[1]["muon"] is False
    state = copy.deepcopy(opt.state_dict())
    state["param_groups"].pop()
    with pytest.raises(ValueError):
        opt.load_state_dict(state)


def test_muon_entry_with_its_scalars_on_the_device_refuses_bad_arguments():
    import ctypes
    from ssecg.lib import lib
    L = lib()
    one = (ctypes.c_int64 * 5)(256, 256, 256, 64, 192)
    n = L.ssecg_orthogonalize_workspace(one, 1)
    ok = [one, 1, 256, 1, 1, 5, 1e-7, None, 256, n, None]
    for at, bad in ((0, None), (1, 0), (2, None), (4, 2), (4, -1), (5, 0), (5, 101), (6, -1.0), (6, float("nan")), (8, None), (8, 264)):
        args = list(ok)
        args[at] = bad
        assert L.ssecg_muon_multi_scalars(*args) == -1, at
    assert L.ssecg_muon_multi_scalars(*(ok[:9] + [n - 1, None])) == -2
    assert L.ssecg_muon_multi_scalars(*([(ctypes.c_int64 * 5)(256, 256, 0, 64, 192)] + ok[1:])) == -1      # no momentum


def test_muon_refuses_settings_it_does_not_know():
    """A misspelt setting of the YAML is an error, not the default."""
    from utils.optimizer import get_optimizer_from_config
    conf = {"optimizer": "muon", "lr": 1e-3, "weight_decay": 0.05}
    known = {"momentum": 0.9, "nesterov": False, "ns_steps": 4, "ns_eps": 1e-6, "adjust_lr": "original", "betas": [0.8, 0.9], "eps": 1e-6}
    group = get_optimizer_from_config({**conf, "optimizer_kwargs": known}, _params()).param_groups[0]
    assert {k: group[k] for k in known} == {**known, "betas": (0.8, 0.9)}
    for name in ("momentun", "muon", "adjust"):
        with pytest.raises(ValueError, match=name):
            get_optimizer_from_config({**conf, "optimizer_kwargs": {name: 0.5}}, _params())
    for empty in ({}, None):
        assert get_optimizer_from_config({**conf, "optimizer_kwargs": empty}, _params()).param_groups[0]["momentum"] == 0.95


def test_layer_norm_backward_entry_needs_something_to_make():
    from ssecg.lib import lib
    L = lib()
    assert L.ssecg_layer_norm_bwd(8, 8, 8, 8, None, 0, 4, 8, None, None, None, None, 0, None) == -1
    assert L.ssecg_layer_norm_bwd(8, 8, 8, 8, None, 0, 4, 8, None, 8, None, None, 0, None) == -2          # dweight alone: its workspace is missing
