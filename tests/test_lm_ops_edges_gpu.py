"""GPU: the token-level operators where their values, sizes or callers are unusual - logits far from zero, operands of very different
sizes, rare classes, several pieces, large constant rows, saved tensors that move, captured hyper-parameters (bounds: tests/lm_close.py
and tests/lm_ref.py, derived from the arithmetic)."""
import pytest
import torch

import lm_close as K
import lm_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ce_case(seed, N, C, V, dtype):
    g = _gen(seed)
    return _normal(g, N, C, dtype=dtype), _normal(g, V, C, scale=C ** -0.5, dtype=dtype), torch.randint(0, V, (N,), generator=g, device="cuda")


def _ce_check(x, w, t, b=None, dloss=None, reduction="mean", what=""):
    from ssecg import ops
    loss, saved = ops.linear_ce_fwd(x, w, t, b, reduction=reduction)
    got = (loss, *ops.linear_ce_bwd(saved, dloss))
    want, bound = K.linear_ce(x, w, t, b, reduction=reduction, dloss=dloss)
    for p, v, e, name in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        if p is not None:
            R.within(p, v, e, (what, name))
    return got


# ------------------------------------------------------------------------------------------------ logits far from zero
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["first", "middle", "last", "all but one", "all"])
@pytest.mark.parametrize("low", [-1e4, float("-inf")])
def test_linear_ce_classes_that_a_bias_rules_out(low, where, dtype):
    """Padding or forbidden classes at -10000 (or -inf), in whole tiles and parts of them; shared by all classes it cancels."""
    N, C, V = 37, 64, 1100
    x, w, t = _ce_case(101, N, C, V, dtype)
    b = torch.zeros(V, device="cuda")
    if where == "first":
        b[:520] = low
        t = 520 + t % (V - 520)
    elif where == "middle":
        b[260:900] = low
        t = t % 260
    elif where == "last":
        b[512:] = low
        t = t % 512
    elif where == "all but one":
        b[:] = low
        b[777] = 0
        t[:] = 777
    else:
        b[:] = -1e4
    _ce_check(x, w, t, b, what=where)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C,V", [(3, 8, 1), (5, 16, 2), (40, 24, 3), (2, 64, 5), (9, 64, 300), (300, 48, 2003), (2, 32, 40000)])
@pytest.mark.parametrize("shift", [-200.0, -100.0, 100.0, 1000.0])
def test_linear_ce_of_shifted_logits(shift, N, C, V, dtype):
    x, w, t = _ce_case(N + C + V, N, C, V, dtype)
    _ce_check(x, w, t, torch.full((V,), shift, device="cuda"), what=shift)


def test_linear_ce_nan_logits_are_not_hidden_by_ruled_out_classes():
    from ssecg import ops
    x, w, t = _ce_case(102, 12, 64, 700, torch.float32)
    b = torch.zeros(700, device="cuda")
    b[:300] = -1e4
    for at in (10, 650):
        w2 = w.clone()
        w2[at, 3] = float("nan")
        assert torch.isnan(ops.linear_ce_fwd(x, w2, t, b)[0])
    assert torch.isnan(ops.linear_ce_fwd(x, w, t, torch.full_like(b, float("-inf")))[0])       # no class is left: 0 / 0, as a softmax has it


# ------------------------------------------------------------------------------------------------ the optimiser's states
def test_muon_excluded_group_continues_adamw_after_a_load():
    from ssecg.optim import FusedAdamW, FusedMuon
    import copy
    g = _gen(120)
    tensors = [_normal(g, 30, 20), _normal(g, 9), _normal(g, 50, 30)]
    make = lambda: [torch.nn.Parameter(t.clone()) for t in tensors]   # noqa: E731
    a, b = make(), make()
    adam = FusedAdamW([{"params": a[:2]}, {"params": a[2:]}], lr=1e-2)
    muon = FusedMuon([{"params": b[:2]}, {"params": b[2:], "muon": False}], lr=0.3)
    for p in a:
        p.grad = torch.ones_like(p)
    adam.step()
    muon.load_state_dict(copy.deepcopy(adam.state_dict()))
    with torch.no_grad():
        for p, q in zip(b, a):
            p.copy_(q)
    for _ in range(2):
        for p, q in zip(a, b):
            p.grad = _normal(g, *p.shape)
            q.grad = p.grad.clone()
        adam.step(), muon.step()
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2]) and not torch.equal(a[0], b[0])
    assert set(muon.state[b[0]]) == {"momentum_buffer"}
    muon.param_groups[0]["muon"] = False                     # from now on AdamW for the matrix too: its own first step
    del muon.state[b[1]]
    muon.step()
    assert {"step", "exp_avg", "exp_avg_sq"} <= set(muon.state[b[0]])
