"""CPU: the token-level operators refuse what they cannot take before any launch (C entries and Python wrappers)."""
import ctypes

import pytest
import torch


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_c_entries_refuse_bad_arguments():
    from ssecg.lib import lib
    L = lib()
    assert L.ssecg_layer_norm_fwd(None, None, None, 0, 1, 8, 1e-5, 8, 8, 8, None) == -1
    assert L.ssecg_layer_norm_fwd(8, None, None, 3, 1, 8, 1e-5, 8, 8, 8, None) == -1          # no such type
    assert L.ssecg_layer_norm_fwd(8, None, None, 0, 0, 8, 1e-5, 8, 8, 8, None) == -1          # no rows
    assert L.ssecg_layer_norm_fwd(8, None, None, 0, 1, 8, -1.0, 8, 8, 8, None) == -1          # negative eps
    assert L.ssecg_layer_norm_fwd(8, None, None, 0, 1, 8, float("nan"), 8, 8, 8, None) == -1
    assert L.ssecg_layer_norm_bwd(8, 8, 8, 8, None, 0, 4, 8, 8, 8, 8, None, 0, None) == -2    # parameter gradients need a workspace
    assert L.ssecg_layer_norm_bwd_workspace(0, 4, 8) > 0 and L.ssecg_layer_norm_bwd_workspace(0, 0, 8) == 0
    n = L.ssecg_linear_ce_fwd_workspace(1, 100, 64, 1000)
    assert n > 0 and L.ssecg_linear_ce_fwd_workspace(1, 0, 64, 1000) == 0
    ok = [256, 256, None, 256, None, 0.0, -100, 1, 100, 64, 1000, 1, 256, 256, 256, 256, None, 0, 256, n, None]
    for at, bad in ((0, None), (1, None), (3, None), (7, 5), (8, 0), (9, 0), (10, 0), (11, 3), (12, None), (16, 8), (18, None), (18, 264)):
        args = list(ok)
        args[at] = bad
        assert L.ssecg_linear_ce_fwd(*args) == -1, at
    assert L.ssecg_linear_ce_fwd(*(ok[:19] + [n - 1, None])) == -2
    assert L.ssecg_linear_ce_fwd(*([264] + ok[1:])) == -2            # x is not 16-byte aligned: its copy has no place
    assert L.ssecg_linear_ce_packed_bytes(256, 256, 1, 100, 64, 1000) == 0 < L.ssecg_linear_ce_packed_bytes(256, 256, 0, 100, 64, 1000)
    n = L.ssecg_linear_ce_bwd_workspace(1, 100, 64, 1000, 1, 1, 0)
    ok = [256, 256, 256, None, 256, 256, 256, 256, 1, 100, 64, 1000, 1, 256, 256, None, None, 0, 256, n, None]
    for at, bad in ((0, None), (5, None), (8, 7), (9, -1), (12, -1), (18, None)):
        args = list(ok)
        args[at] = bad
        assert L.ssecg_linear_ce_bwd(*args) == -1, at
    assert L.ssecg_linear_ce_bwd(*(ok[:13] + [None, None, None, None, 0, 256, n, None])) == -1          # nothing wanted
    assert L.ssecg_linear_ce_bwd(*(ok[:19] + [n - 1, None])) == -2
    one = _i64(256, 256, 256, 64, 192)
    n = L.ssecg_orthogonalize_workspace(one, 1)
    assert n > 0 and L.ssecg_orthogonalize_workspace(_i64(0, 0, 0, 0, 4), 1) == 0
    assert L.ssecg_orthogonalize_multi(one, 0, 0, 5, 1e-7, 256, n, None) == -1
    assert L.ssecg_orthogonalize_multi(one, 1, 0, 0, 1e-7, 256, n, None) == -1                 # steps
    assert L.ssecg_orthogonalize_multi(one, 1, 0, 5, 1e-7, 256, n - 1, None) == -2
    assert L.ssecg_orthogonalize_multi(_i64(0, 256, 0, 4, 4), 1, 0, 5, 1e-7, 256, n, None) == -1
    assert L.ssecg_muon_multi(_i64(256, 256, 0, 4, 4), 1, 0.1, 0.9, 1, 0.0, 1, 5, 1e-7, None, None, 256, n, None) == -1   # no momentum
    assert L.ssecg_muon_multi(one, 1, 0.1, 1.0, 1, 0.0, 1, 5, 1e-7, None, None, 256, n, None) == -1
    assert L.ssecg_muon_multi(one, 1, 0.1, 0.9, 1, 0.0, 2, 5, 1e-7, None, None, 256, n, None) == -1


def test_workspaces_grow_with_the_matrices_of_one_chain():
    from ssecg.lib import lib
    L = lib()
    rows = _i64(*([0, 0, 0, 64, 64] * 40))
    w1, w32, w40 = (L.ssecg_orthogonalize_workspace(rows, k) for k in (1, 32, 40))
    assert w1 < w32 == w40           # 40 matrices are a chain of 32 and one of 8


def test_wrappers_refuse_cpu_tensors_and_bad_arguments():
    from ssecg import ops
    from ssecg.lib import SsecgError
    x, w, t = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.layer_norm_fwd(x), lambda: ops.linear_ce_fwd(x, w, t), lambda: ops.orthogonalize(x), lambda: ops.orthogonalize([x])):
        with pytest.raises(SsecgError):
            call()
    assert ops.orthogonalize([]) == []
    with pytest.raises(SsecgError):
        ops.orthogonalize(x, steps=0)


def test_muon_hyper_parameters():
    from ssecg.lib import SsecgError
    from ssecg.optim import FusedMuon
    from utils.optimizer import get_optimizer_from_config
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for bad in (dict(momentum=1.0), dict(ns_steps=0), dict(adjust_lr="other"), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            FusedMuon([p], **bad)
    opt = get_optimizer_from_config({"optimizer": "muon", "lr": 1e-3, "weight_decay": 0.05, "optimizer_kwargs": {"momentum": 0.9, "betas": [0.9, 0.95]}}, [p])
    g = opt.param_groups[0]
    assert isinstance(opt, FusedMuon) and g["momentum"] == 0.9 and g["betas"] == (0.9, 0.95) and g["muon"] is True
    opt.step()                       # no gradient: nothing to do, nothing refused
    p.grad = torch.zeros(4, 4)
    with pytest.raises(SsecgError):
        opt.step()                   # a CPU parameter


def test_limits_are_refused_before_anything_is_sized():
    from ssecg.lib import lib
    from ssecg.optim import FusedMuon
    L = lib()
    assert L.ssecg_linear_ce_fwd_workspace(1, 1 << 21, 64, 1 << 17) > 0
    for N, C, V in ((1 << 21, 64, (1 << 17) + 1), ((1 << 21) + 1, 64, 8), (8, (1 << 16) + 1, 8), (8, 8, (1 << 24) + 1)):
        assert L.ssecg_linear_ce_fwd_workspace(1, N, C, V) == 0 == L.ssecg_linear_ce_bwd_workspace(1, N, C, V, 1, 1, 1)
        assert L.ssecg_linear_ce_fwd(256, 256, None, 256, None, 0.0, -100, 1, N, C, V, 1, 256, 256, 256, 256, None, 0, 256, 1 << 40, None) == -1
    assert L.ssecg_layer_norm_bwd_workspace(0, 4, (1 << 24) + 1) == 0
    assert L.ssecg_orthogonalize_workspace(_i64(0, 0, 0, (1 << 20) + 1, 4), 1) == 0
    big, small = torch.nn.Parameter(torch.empty((1 << 20) + 1, 2)), torch.nn.Parameter(torch.empty(4, 2))
    with pytest.raises(ValueError):
        FusedMuon([big])
    opt = FusedMuon([{"params": [big], "muon": False}, {"params": [small]}])
    for bad in (dict(ns_steps=101), dict(momentum=-0.1), dict(ns_eps=float("nan")), dict(adjust_lr=1)):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[torch.nn.Parameter(torch.empty(2, 2))], **bad))
    assert len(opt.param_groups) == 2


def test_every_piece_of_the_vocabulary_is_covered_once():
    """The backward workspace holds a bounded piece of the gradient of the logits, whatever the vocabulary."""
    from ssecg.lib import lib
    L = lib()
    whole = L.ssecg_linear_ce_bwd_workspace(1, 8192, 1024, 65536, 1, 1, 0)
    assert (1 << 30) <= whole < (1 << 30) + (1 << 28)
    assert L.ssecg_linear_ce_bwd_workspace(1, 8192, 1024, 1 << 20, 1, 1, 0) < 2 * whole
