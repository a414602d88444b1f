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


# ------------------------------------------------------------------------------------------------ fp32 operands of very different sizes
@pytest.mark.parametrize("big", [1e6, 1e12, 1e30])
@pytest.mark.parametrize("N,C,V", [(40, 64, 300), (300, 771, 2003)])
def test_linear_ce_fp32_one_large_row_leaves_the_others_alone(N, C, V, big):
    """A position (and a class) far larger than the others: every other row of the logits, the loss and the gradients keeps its own bound."""
    x, w, t = _ce_case(130 + N, N, C, V, torch.float32)
    x[7] *= big
    w[:, :] /= big if big > 1e20 else 1                      # keep the large row's logits finite
    b = torch.zeros(V, device="cuda")
    dloss = torch.ones(N, device="cuda")
    _ce_check(x, w, t, b, dloss, "none", what="row")
    x, w, t = _ce_case(131 + N, N, C, V, torch.float32)
    w[11] *= -big                                            # a class whose logits are huge and negative or positive
    x[:, 1:] = 0
    x[:, 0] = x[:, 0].abs() + 0.5
    w[:, 0] = w[:, 0].abs() + 0.1
    w[11, 0] = -big
    t[t == 11] = 12
    _ce_check(x, w, t, b, dloss, "none", what="class")


def test_linear_ce_fp32_largest_and_smallest_values():
    g = _gen(132)
    x, w, t = _ce_case(132, 20, 64, 130, torch.float32)
    x[3, 5], w[:, 5] = torch.finfo(torch.float32).max, 0.0   # rounds to infinity in 16 bits, counts for nothing here
    x[4] = _normal(g, 64, scale=1e-30)
    w[9] = _normal(g, 64, scale=1e-30)
    _ce_check(x, w, t, None, torch.ones(20, device="cuda"), "none")


@pytest.mark.parametrize("dtype,low", [(torch.float32, -20.0), (torch.float32, -30.0), (torch.float32, -60.0), (torch.bfloat16, -30.0),
                                       (torch.bfloat16, -60.0), (torch.float16, -12.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_linear_ce_rare_classes_keep_their_precision(reduction, dtype, low):
    """Classes that are no label and have a probability of e^low in every position: their rows of dW to their own bound (fp16: as far as
    its exponents go)."""
    N, C, V = 90, 64, 700
    x, w, t = _ce_case(133, N, C, V, dtype)
    b = torch.zeros(V, device="cuda")
    b[200:520] = low
    t = torch.where((t >= 200) & (t < 520), t % 200, t)
    scale = 2.0 ** 12 if dtype == torch.float16 else 1.0
    _ce_check(x, w, t, b, torch.full((N,) if reduction == "none" else (), scale, device="cuda"), reduction)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_ce_small_upstream_gradients_beside_large_ones(dtype):
    N = 60
    x, w, t = _ce_case(134, N, 64, 300, dtype)
    dloss = torch.logspace(0, -18, N, device="cuda")[torch.randperm(N, generator=_gen(135), device="cuda")]
    _ce_check(x, w, t, torch.zeros(300, device="cuda"), dloss, "none")


# ------------------------------------------------------------------------------------------------ several pieces of the vocabulary
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_linear_ce_in_pieces_with_bias(reduction, dtype):
    """More classes than a piece of the gradient of the logits holds (1 GiB: 10922 classes in fp32, 32768 in 16 bits at 16384 positions):
    every class of dW and db and every position of dx against 64 bits."""
    N, C, V = 16384, 64, (24001 if dtype == torch.float32 else 40001)
    x, w, t = _ce_case(136, N, C, V, dtype)
    t[::5] = V - 1 - torch.arange(len(t[::5]), device="cuda") % 9000        # labels in the last piece too
    t[100:300] = -100
    b = _normal(_gen(137), V, scale=0.3)
    dloss = torch.rand(N, generator=_gen(138), device="cuda") if reduction == "none" else torch.tensor(256.0, device="cuda")
    _ce_check(x, w, t, b, dloss, reduction)


@pytest.mark.parametrize("shapes", [[(40, 20), (7,)], [(200, 300), (64, 64), (7,)]])
def test_captured_muon_step_follows_its_hyper_parameters(shapes):
    """lr, weight decay and momentum that change between replays; the settings that a captured launch holds are refused."""
    from ssecg.graph import StepGraph
    from ssecg.lib import SsecgError
    from ssecg.optim import FusedMuon
    start = [_normal(_gen(140 + k), *s) for k, s in enumerate(shapes)]
    grads = [[_normal(_gen(150 + 10 * n + k), *s) for k, s in enumerate(shapes)] for n in range(8)]

    def build():
        ps = [torch.nn.Parameter(t.clone()) for t in start]
        opt = FusedMuon(ps, lr=1e-2)

        def step(*gs):
            for p, g in zip(ps, gs):
                p.grad = g * 1.0
            opt.step()
            opt.zero_grad()
            return (ps[0].detach().sum(),)
        return ps, opt, step
    ps_e, opt_e, step_e = build()
    ps_g, opt_g, step_g = build()
    graph = StepGraph(step_g)
    for n, gs in enumerate(grads):
        for o in (opt_e, opt_g):
            o.param_groups[0].update(lr=1e-2 / (n + 1), weight_decay=0.02 * n, momentum=0.5 + 0.06 * n)
        step_e(*gs), graph(*gs)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps_e, ps_g)), n
    assert graph.replays >= 5 and not graph.disabled
    steps = float(opt_g.state[ps_g[-1]]["step"])
    for change in (dict(nesterov=False), dict(ns_steps=4), dict(ns_eps=1e-3), dict(adjust_lr="original"), dict(muon=False), dict(momentum=1.0),
                   dict(betas=(0.8, 0.99)), dict(eps=1e-6)):
        old = {k: opt_g.param_groups[0][k] for k in change}
        opt_g.param_groups[0].update(change)
        with pytest.raises((SsecgError, ValueError)):
            graph(*grads[0])
        opt_g.param_groups[0].update(old)
    step_e(*grads[0]), graph(*grads[0])                      # a refused call has moved nothing
    assert float(opt_g.state[ps_g[-1]]["step"]) == steps + 1
    assert all(torch.equal(p, q) for p, q in zip(ps_e, ps_g))


# ------------------------------------------------------------------------------------------------ layer norm: sizes and values
def test_layer_norm_refuses_rows_longer_than_it_counts():
    """2^24 columns are the limit; 2^32 + 512 is not 512."""
    from ssecg import ops
    from ssecg.lib import SsecgError
    one = torch.zeros(1, device="cuda")
    for C in ((1 << 24) + 1, (1 << 32) + 512):
        x = torch.empty(1, C, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(SsecgError):
            ops.layer_norm_fwd(x)
        with pytest.raises(SsecgError):
            ops.layer_norm_bwd(x, x, one, one)
        del x


def test_layer_norm_of_infinite_and_nan_rows_keeps_their_mean():
    from ssecg import ops
    x = _normal(_gen(182), 4, 300)
    x[0, 3], x[1, 4], x[2, 5] = float("inf"), float("-inf"), float("nan")
    y, mean, rstd = ops.layer_norm_fwd(x)
    assert mean[0] == float("inf") and mean[1] == float("-inf") and torch.isnan(mean[2])
    assert torch.isnan(y[:3]).all() and torch.isnan(rstd[:3]).all() and torch.isfinite(y[3]).all()


# ------------------------------------------------------------------------------------------------ what autograd keeps
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_keeps_everything_as_saved_tensors(dtype):
    """Hooks see every byte that the node keeps, wherever they put it back (off any boundary too), and nothing is left after the backward
    pass."""
    from ssecg import functional as SF
    N, C, V = 512, 200, 4096                                 # C is no whole stage: copies in every type
    x, w, t = _ce_case(160, N, C, V, dtype)
    x.requires_grad_(True), w.requires_grad_(True)
    b = torch.zeros(V, device="cuda", dtype=dtype, requires_grad=True)
    plain = torch.autograd.grad(SF.linear_cross_entropy(x, w, t, bias=b), (x, w, b))
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()

    def moved(s):
        return torch.empty(s.numel() + 1, dtype=s.dtype, device=s.device)[1:].view(s.shape).copy_(s)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.detach().cpu(), lambda s: moved(s.cuda())):
        loss = SF.linear_cross_entropy(x, w, t, bias=b)
    assert torch.cuda.memory_allocated() - start <= 4096     # the loss; all else went with the hooks
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(loss, (x, w, b)), plain))
    loss = SF.linear_cross_entropy(x, w, t, bias=b)
    assert torch.cuda.memory_allocated() - start >= (N + V) * 256 * 2
    grads = torch.autograd.grad(loss, (x, w, b))
    del grads
    assert torch.cuda.memory_allocated() - start <= 8192     # the node still lives with the loss, what it kept does not


def test_linear_ce_notices_operands_that_changed():
    from ssecg import functional as SF
    x, w, t = _ce_case(161, 16, 64, 50, torch.float32)
    w.requires_grad_(True)
    loss = SF.linear_cross_entropy(x, w, t)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(300, 64), (70, 777), (5, 20001)])
def test_layer_norm_makes_only_the_gradients_that_are_wanted(rows, C, dtype):
    from ssecg import functional as SF, ops
    g = _gen(170)
    x, dy = _normal(g, rows, C, dtype=dtype), _normal(g, rows, C, dtype=dtype)
    w, b = (1 + _normal(g, C, scale=0.2)).requires_grad_(True), _normal(g, C).requires_grad_(True)
    _, mean, rstd = ops.layer_norm_fwd(x, w.detach(), b.detach())
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w.detach())
    part = ops.layer_norm_bwd(dy, x, mean, rstd, w.detach(), want_dx=False)
    assert part[0] is None and torch.equal(part[1], dw) and torch.equal(part[2], db)
    part = ops.layer_norm_bwd(dy, x, mean, rstd, w.detach(), want_params=False)
    assert torch.equal(part[0], dx) and part[1] is None and part[2] is None
    assert ops.layer_norm_bwd(dy, x, mean, rstd, w.detach(), want_params=False, want_dx=False) == (None, None, None)
    y = SF.layer_norm(x, w, b)                               # the data need no gradient
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    got = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(got[0], dw) and torch.equal(got[1], db)
    if rows == 300:                                          # (the others' column sums need more than dx)
        nbytes = ops.lib().ssecg_layer_norm_bwd_workspace({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], rows, C)
        assert torch.cuda.max_memory_allocated() - start <= nbytes + 3 * 1024


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [7, 49, 100, 777, 2049, 6000, 20001])
def test_layer_norm_of_rows_of_equal_and_nearly_equal_large_values(C, dtype):
    """Equal values: no deviation, y = bias exactly and the mean is the value.  Nearly equal ones, a step apart: fp32's mean may be half a
    step of x off, no more."""
    from ssecg import ops
    top = 6e4 if dtype == torch.float16 else 3e7
    v = torch.tensor([3.0, 1000.3, 12345.6, 60000.0, 123456.7, 1e6, 3e7, -1e6], device="cuda").clamp(max=top, min=-top).to(dtype)
    x = v[:, None].expand(-1, C).contiguous()
    b = _normal(_gen(180), C)
    y, mean, rstd = ops.layer_norm_fwd(x, None, b)
    assert torch.equal(mean, v.float()) and torch.equal(y, b.to(dtype).expand_as(y))
    dx, dw, db = ops.layer_norm_bwd(torch.ones_like(x), x, mean, rstd)
    assert not dw.any() and torch.isfinite(dx).all()
    if dtype == torch.float32:
        step = 2.0 ** -23 * 2.0 ** torch.floor(torch.log2(v.abs()))
        x = x + step[:, None] * torch.randint(-3, 4, (8, C), generator=_gen(181), device="cuda")
        y, mean, rstd = ops.layer_norm_fwd(x)
        x64 = x.double()
        mu, var = x64.mean(1, keepdim=True), x64.var(1, unbiased=False, keepdim=True)
        rs = 1 / torch.sqrt(var + 1e-5)
        assert ((mean.double() - mu[:, 0]).abs() <= 0.5 * 1.001 * step.double()).all()
        # the mean half a step off (and once more where rstd's variance takes it in: at most (step / 2)^2 of it), then fp32's roundings
        off = 0.5 * 1.001 * step[:, None].double() * rs
        R.within(y, (x64 - mu) * rs, off + 32 * R.U * ((x64 - mu) * rs).abs() + 32 * R.U, "y")
        R.within(rstd, rs[:, 0], 64 * R.U * rs[:, 0], "rstd")


@pytest.mark.parametrize("chain", [False, True])
def test_orthogonalize_is_as_near_to_64_bits_as_32_bit_products(chain):
    """300 matrices of up to 64 rows, alone and beside a larger one (which sends them through the chain of launches): against the plain form
    in 32 bits.  Both errors are a few roundings that the iteration amplifies, so either form is the nearer one by chance.  Where one is
    1.5 times as far off as the other (and beyond 1e-6), a fair coin decides which: of n such matrices the kernel has at most
    n / 2 + 3 sqrt(n) / 2."""
    import math
    import random
    from ssecg import ops
    rng = random.Random(5)
    larger = _normal(_gen(199), 300, 400)
    further = nearer = 0
    for k in range(300):
        m, n = (int(round(math.exp(rng.uniform(0, math.log(top))))) for top in (64, 4096))
        g, r = _gen(k), max(1, min(m, n) // 8)
        x = ((_normal(g, m, r) @ _normal(g, r, n)) / math.sqrt(r) + _normal(g, m, n, scale=0.5)) * 1e-3
        want, plain = R.orthogonal(x), R.orthogonal(x, dtype=torch.float32)
        got = ops.orthogonalize([x, larger])[0] if chain else ops.orthogonalize(x)
        own, off = ((v.double() - want).norm() / want.norm() for v in (plain, got))
        further += int(off > max(1e-6, 1.5 * own))
        nearer += int(own > max(1e-6, 1.5 * off))
    count = further + nearer
    assert further <= count / 2 + 1.5 * math.sqrt(count), (further, nearer)
