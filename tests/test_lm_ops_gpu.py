"""GPU: layer norm, classifier + cross entropy over a large vocabulary, orthogonalised updates - against their plain forms in 64
bits, at the sizes, types, masks and strides where they can go wrong (bounds: tests/lm_ref.py, derived from the arithmetic)."""
import copy

import pytest
import torch

import lm_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 7), (3, 64), (1008, 512), (67, 513), (130, 777), (17, 2048), (9, 2049), (33, 4096), (5, 8191),
                                    (6, 16384), (3, 16385), (2, 40000), (2100, 24)])
def test_layer_norm(rows, C, dtype):
    from ssecg import ops
    g = _gen(rows * 100003 + C)
    x = _normal(g, rows, C, dtype=dtype) * 2 + _normal(g, rows, 1, dtype=dtype)
    dy = _normal(g, rows, C, dtype=dtype)
    w, b = 1 + _normal(g, C, scale=0.2), _normal(g, C, scale=0.2)
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, 1e-5)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    want, bound = R.layer_norm(x, dy, w, b, 1e-5)
    for got, v, t, what in zip((y, dx, dw, db), want, bound, ("y", "dx", "dw", "db")):
        R.within(got, v, t, what)
    again = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


# ------------------------------------------------------------------------------------------------ classifier + cross entropy
def _ce_case(seed, N, C, V, dtype, bias, gate, ignore=0.2):
    g = _gen(seed)
    x = _normal(g, N, C, dtype=dtype)
    w = _normal(g, V, C, scale=C ** -0.5, dtype=dtype)
    b = _normal(g, V, scale=0.3) if bias else None
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    if ignore:
        t[torch.rand((N,), generator=g, device="cuda") < ignore] = -100
    conf = torch.rand((N,), generator=g, device="cuda") if gate else None
    return x, w, b, t, conf


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C,V,bias,gate", [(1, 8, 2, True, False), (1, 64, 300, False, False), (5, 65, 33, True, True), (126, 512, 1000, True, False),
                                             (257, 128, 129, False, True), (300, 771, 2003, True, True), (1999, 64, 4, True, True),
                                             (2, 1024, 8192, False, False)])
def test_linear_ce(N, C, V, bias, gate, dtype):
    from ssecg import ops
    x, w, b, t, conf = _ce_case(N + 7 * C + 31 * V, N, C, V, dtype, bias, gate)
    dloss = torch.full((), 1024.0, device="cuda")
    loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.4)
    got = (loss, *ops.linear_ce_bwd(saved, dloss))
    want, bound = R.linear_ce(x, w, t, b, conf, 0.4, dloss=dloss)
    for p, v, e, what in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        if p is not None:
            R.within(p, v, e, what)


# ------------------------------------------------------------------------------------------------ orthogonalised updates
def _near(got, g, what, steps=5):
    """No further from 64 bits than eight times what the plain form in fp32 is (operands are held in 22 bits and more against 24, and
    the product of the low halves is dropped: 2^-22 against 2^-24 per product), plus the result's own rounding."""
    want, plain = R.orthogonal(g, steps), R.orthogonal(g.float(), steps, dtype=torch.float32)
    norm = want.norm()
    off, own = (got.double() - want).norm() / norm, (plain.double() - want).norm() / norm
    # 16-bit results: a rounding is at most half a step of each element
    assert off <= 8 * own + 2.0 ** -20 + (R.half_step(got.dtype) if got.dtype != torch.float32 else 0), (what, float(off), float(own))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [[(1, 1)], [(64, 192)], [(1, 515), (515, 1)], [(33, 65), (65, 33), (7, 300)], [(512, 1536), (100, 1000), (4, 128)],
                                    [(1000, 777)], [(2100, 2051)]])
def test_orthogonalize(shapes, dtype):
    from ssecg import ops
    g = _gen(sum(m * 1000 + n for m, n in shapes))
    mats = [_normal(g, m, n, scale=1e-3, dtype=dtype) for m, n in shapes]
    for m, o in zip(mats, ops.orthogonalize(mats)):
        _near(o, m, tuple(m.shape))


# ------------------------------------------------------------------------------------------------ layer norm: the calls around it
def test_layer_norm_autograd_strided_and_without_parameters():
    from ssecg import functional as SF
    g = _gen(1)
    base = _normal(g, 6, 40, 33)
    x = base.transpose(1, 2).requires_grad_(True)            # (6, 33, 40), strided
    w, b = (1 + _normal(g, 40, scale=0.2)).requires_grad_(True), _normal(g, 40).requires_grad_(True)
    dy = _normal(g, 6, 40, 33).transpose(1, 2)
    y = SF.layer_norm(x, w, b, 1e-3)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want, bound = R.layer_norm(x.detach(), dy, w.detach(), b.detach(), 1e-3)
    for got, v, t, what in zip((y.detach(), dx, dw, db), want, bound, ("y", "dx", "dw", "db")):
        R.within(got, v, t, what)
    y = SF.layer_norm(x, None, None, 1e-3)
    (dx,) = torch.autograd.grad(y, x, dy)
    want, bound = R.layer_norm(x.detach(), dy, None, None, 1e-3)
    R.within(y.detach(), want[0], bound[0], "y")
    R.within(dx, want[1], bound[1], "dx")


def test_layer_norm_16_bit_parameters_and_module():
    from ssecg import functional as SF
    from ssecg.nn import LayerNorm
    g = _gen(2)
    x = _normal(g, 30, 100, dtype=torch.bfloat16).requires_grad_(True)
    m = LayerNorm(100).cuda().to(torch.bfloat16)
    dy = _normal(g, 30, 100, dtype=torch.bfloat16)
    with torch.no_grad():
        m.weight.copy_(1 + _normal(g, 100, scale=0.2))
    y = m(x)
    dx, dw, db = torch.autograd.grad(y, (x, m.weight, m.bias), dy)
    assert dw.dtype == db.dtype == torch.bfloat16
    want, bound = R.layer_norm(x.detach(), dy, m.weight.detach(), m.bias.detach(), m.eps)
    R.within(y.detach(), want[0], bound[0], "y")
    R.within(dx, want[1], bound[1], "dx")
    R.within(dw, want[2], bound[2] + R.rounded(want[2], torch.bfloat16), "dw")
    with pytest.raises(ValueError):
        m(x[:, :50])
    assert set(LayerNorm(8).state_dict()) == {"weight", "bias"} and SF.layer_norm(x[:0].detach()).shape == (0, 100)


def test_layer_norm_no_rows_and_bad_rows():
    from ssecg import ops
    y, mean, rstd = ops.layer_norm_fwd(torch.empty(0, 16, device="cuda"))
    dx, dw, db = ops.layer_norm_bwd(y, y, mean, rstd)
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    g = _gen(3)
    x, dy = _normal(g, 9, 300), _normal(g, 9, 300)
    x[2, 7], x[5, 0] = float("inf"), float("nan")
    y, mean, rstd = ops.layer_norm_fwd(x)
    dx, _, _ = ops.layer_norm_bwd(dy, x, mean, rstd)
    good = [0, 1, 3, 4, 6, 7, 8]
    want, bound = R.layer_norm(x[good], dy[good], None, None, 1e-5)
    R.within(y[good], want[0], bound[0], "y")                # a row's values stay in the row
    R.within(dx[good], want[1], bound[1], "dx")
    assert torch.isnan(y[2]).any() and torch.isnan(y[5]).all()
    c = torch.full((4, 64), 3.0, device="cuda")              # no variance: y = b, finite
    y, mean, rstd = ops.layer_norm_fwd(c, None, torch.ones(64, device="cuda"))
    assert torch.equal(y, torch.ones_like(y)) and torch.isfinite(rstd).all()


def test_layer_norm_gradient_against_differences():
    """<dx, d> against (f(x + h d) - f(x - h d)) / 2h for f = sum y dy.  The quotient of the kernel's forward pass is held to the
    quotient of the 64-bit form at the same h (no truncation in between): each f is off by at most the sum of y's bounds."""
    from ssecg import ops
    g = _gen(4)
    x, dy, d = _normal(g, 5, 64), _normal(g, 5, 64), _normal(g, 5, 64)
    h = 2.0 ** -8
    xp, xm = x + h * d, x - h * d
    (yp, _, _), (ym, _, _) = ops.layer_norm_fwd(xp), ops.layer_norm_fwd(xm)
    (wp, tp), (wm, tm) = R.layer_norm(xp, dy, None, None, 1e-5), R.layer_norm(xm, dy, None, None, 1e-5)
    q = ((yp.double() - ym.double()) * dy.double()).sum() / (2 * h)
    q64 = ((wp[0] - wm[0]) * dy.double()).sum() / (2 * h)
    assert abs(q - q64) <= ((tp[0] + tm[0]) * dy.double().abs()).sum() / (2 * h)
    y, mean, rstd = ops.layer_norm_fwd(x)
    dx, _, _ = ops.layer_norm_bwd(dy, x, mean, rstd)
    # truncation h^2 / 6 f''': third differences of the 64-bit form bound f''' (twice as wide a step on both sides)
    f = [(R.layer_norm(x + k * h * d, dy, None, None, 1e-5)[0][0] * dy.double()).sum() for k in (-2, -1, 1, 2)]
    third = abs(f[3] - 2 * f[2] + 2 * f[1] - f[0]) / (2 * h ** 3)
    want, bound = R.layer_norm(x, dy, None, None, 1e-5)
    assert abs((dx.double() * d.double()).sum() - q64) <= h * h / 3 * third + (bound[1] * d.double().abs()).sum()


# ------------------------------------------------------------------------------------------------ classifier + cross entropy: around it
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_linear_ce_reductions(reduction, dtype):
    from ssecg import ops
    x, w, b, t, conf = _ce_case(11, 77, 128, 500, dtype, True, True)
    dloss = torch.tensor(3.0, device="cuda") if reduction == "sum" else 64 * (torch.rand(77, generator=_gen(5), device="cuda") - 0.3)
    loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.3, reduction=reduction)
    got = (loss, *ops.linear_ce_bwd(saved, dloss))
    want, bound = R.linear_ce(x, w, t, b, conf, 0.3, reduction=reduction, dloss=dloss)
    if reduction == "none":      # E is held times a power of two >= max |dloss|: the smallest step of fp16 there, 2^-25 / 2^14 of it
        top = 2 * dloss.abs().max().double()
        extra = 2.0 ** -39 * top
        bound = (bound[0], bound[1] + extra * w.double().abs().sum(0), bound[2] + extra * x.double().abs().sum(0), bound[3])
    for p, v, e, what in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        R.within(p, v, e, what)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_rows_that_do_not_count_may_hold_anything(dtype):
    from ssecg import ops
    x, w, b, t, conf = _ce_case(12, 65, 64, 90, dtype, True, True, ignore=0.0)
    t[3] = t[64] = -100
    conf[7] = float("nan")
    clean = x.clone()
    x[3], x[64], x[7] = float("nan"), float("inf"), torch.finfo(dtype).max
    clean[[3, 64, 7]] = 0
    loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.2)
    got = (loss, *ops.linear_ce_bwd(saved))
    want, bound = R.linear_ce(clean, w, t, b, conf, 0.2)
    for p, v, e, what in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        R.within(p, v, e, what)
    assert not got[1][[3, 64, 7]].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_nothing_counts(dtype):
    from ssecg import ops
    x, w, b, t, _ = _ce_case(13, 10, 40, 30, dtype, True, False)
    for target, conf in ((torch.full_like(t, -100), None), (t, torch.zeros(10, device="cuda"))):
        for reduction in ("mean", "sum", "none"):
            loss, saved = ops.linear_ce_fwd(x, w, target, b, conf, 0.5, reduction=reduction)
            dx, dw, db = ops.linear_ce_bwd(saved)
            assert not loss.any() and not dx.any() and not dw.any() and not db.any()
    loss, saved = ops.linear_ce_fwd(x[:0], w, t[:0], b)
    dx, dw, db = ops.linear_ce_bwd(saved)
    assert loss.item() == 0 and dx.shape == (0, 40) and not dw.any() and not db.any()


def test_linear_ce_label_outside_the_vocabulary_is_nan_in_its_row():
    from ssecg import ops
    x, w, _, t, _ = _ce_case(14, 20, 64, 30, torch.float32, False, False, ignore=0.0)
    t[4], t[9] = 30, -1
    loss, saved = ops.linear_ce_fwd(x, w, t, reduction="none")
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[[4, 9]] = True
    assert torch.equal(torch.isnan(loss), bad)
    dx, _, _ = ops.linear_ce_bwd(saved)
    assert torch.equal(torch.isnan(dx).any(1), bad)
    want, bound = R.linear_ce(x[~bad], w, t[~bad], reduction="none")
    R.within(loss[~bad], want[0], bound[0], "loss")
    R.within(dx[~bad], want[1], bound[1], "dx")


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_strides_alignment_and_autograd(dtype):
    from ssecg import functional as SF
    g = _gen(15)
    B, L, C, V = 3, 21, 64, 70
    x = _normal(g, B, C, L, dtype=dtype).transpose(1, 2).requires_grad_(True)            # (B, L, C) of a (B, C, L) tensor
    w = _normal(g, V * C + 1, scale=0.125, dtype=dtype)[1:].view(V, C).requires_grad_(True)   # not 16-byte aligned
    b = _normal(g, V, dtype=dtype).requires_grad_(True)
    t = torch.randint(0, V, (B, L), generator=g, device="cuda")
    t[0, :5] = 7
    loss = SF.linear_cross_entropy(x, w, t, bias=b, ignore_index=7)
    dx, dw, db = torch.autograd.grad(loss, (x, w, b), torch.tensor(8.0, device="cuda"))
    assert dx.shape == x.shape and db.dtype == dtype
    want, bound = R.linear_ce(x.detach().reshape(-1, C), w.detach(), t.flatten(), b.detach(), ignore=7, dloss=torch.tensor(8.0, device="cuda"))
    R.within(loss.detach(), want[0], bound[0], "loss")
    R.within(dx.reshape(-1, C), want[1], bound[1], "dx")
    R.within(dw, want[2], bound[2], "dw")
    R.within(db, want[3], bound[3] + R.rounded(want[3], dtype), "db")
    only = SF.linear_cross_entropy(x.detach(), w, t, ignore_index=7, reduction="none")   # weight's gradient alone
    assert only.shape == (B, L)
    (dw2,) = torch.autograd.grad(only, w, torch.ones_like(only))
    want, bound = R.linear_ce(x.detach().reshape(-1, C), w.detach(), t.flatten(), ignore=7, reduction="sum")
    R.within(dw2, want[2], bound[2], "dw")


def test_linear_ce_in_two_pieces_is_the_same_everywhere():
    """More than 1 GiB of E: two pieces of the vocabulary, dx summed over both."""
    from ssecg import ops
    N, C, V = 16384, 64, 40000
    x, w, _, t, _ = _ce_case(16, N, C, V, torch.bfloat16, False, False, ignore=0.0)
    t[:4096] = -100
    loss, saved = ops.linear_ce_fwd(x, w, t)
    dx, dw, _ = ops.linear_ce_bwd(saved)
    rows = torch.arange(4000, 4200, device="cuda")           # dx of some rows; its scale is the whole batch's
    want, bound = R.linear_ce(x[rows], w, t[rows], reduction="sum", dloss=torch.tensor(1.0 / 12288, device="cuda", dtype=torch.float64))
    R.within(dx[rows], want[1], bound[1], "dx")
    cols = torch.cat([torch.arange(0, 20), torch.arange(20470, 20490), torch.arange(V - 20, V)]).cuda()
    p = torch.empty(N, 60, dtype=torch.float64, device="cuda")
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for r in range(0, N, 2048):
        z = x[r:r + 2048].double() @ w.double().T
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        p[r:r + 2048] = lp[:, cols].exp()
        if r >= 4096:
            total -= lp.gather(1, t[r:r + 2048, None]).sum()
    E = (p - (t[:, None] == cols).double()) * (t != -100)[:, None] / 12288
    want = E.T @ x.double()
    # E's rounding to bf16 (half a step), its exponent's error, dw's rounding
    bound = (R.half_step(torch.bfloat16) + 2.0 ** -16) * (E.abs().T @ x.double().abs()) + R.rounded(want, torch.bfloat16)
    R.within(dw[cols], want, bound, "dw")
    assert abs(loss.double() - total / 12288) <= 2.0 ** -18 * (total / 12288)


def test_linear_ce_weights_beyond_2_31_elements():
    from ssecg import ops
    C, V = 1024, (1 << 21) + 3000                            # 2.15e9 weights, two pieces
    g = _gen(17)
    w = torch.empty(V, C, dtype=torch.bfloat16, device="cuda")
    for r in range(0, V, 1 << 18):
        w[r:r + (1 << 18)] = _normal(g, min(1 << 18, V - r), C, scale=1 / 32, dtype=torch.bfloat16)
    x = _normal(g, 3, C, dtype=torch.bfloat16)
    t = torch.tensor([V - 1, 0, 1 << 21], device="cuda")
    loss, saved = ops.linear_ce_fwd(x, w, t, reduction="sum")
    dx, dw, _ = ops.linear_ce_bwd(saved)
    z = torch.cat([x.double() @ w[r:r + (1 << 18)].double().T for r in range(0, V, 1 << 18)], 1)
    lse = torch.logsumexp(z, 1)
    R.within(loss, (lse - z.gather(1, t[:, None])[:, 0]).sum(), 2.0 ** -16 * lse.sum(), "loss")
    for r in (0, 5, 1 << 21, V - 2, V - 1):
        E = (z[:, r] - lse).exp() - (t == r).double()
        want = E @ x.double()
        R.within(dw[r], want, (R.half_step(torch.bfloat16) + 2.0 ** -16) * (E.abs() @ x.double().abs()) + R.rounded(want, torch.bfloat16), f"dw[{r}]")
    p = (z - lse[:, None]).exp()
    want = sum(p[:, r:r + (1 << 18)] @ w[r:r + (1 << 18)].double() for r in range(0, V, 1 << 18)) - w[t].double()
    # p w sums over two million classes of random sign, each off by half a bf16 step: 8 standard deviations of that, and the roundings
    noise = 8 * R.half_step(torch.bfloat16) * torch.stack([(p[i] ** 2).sum().sqrt() for i in range(3)])[:, None] * w[:1000].double().abs().max()
    R.within(dx, want, noise + R.rounded(want, torch.bfloat16) + 2.0 ** -12 * want.abs(), "dx")


def test_linear_ce_is_reproducible_and_runs_on_its_callers_stream():
    from ssecg import ops
    x, w, b, t, conf = _ce_case(18, 300, 96, 1500, torch.float32, True, True)
    loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.3)
    first = (loss, *ops.linear_ce_bwd(saved))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.3)
        again = (loss, *ops.linear_ce_bwd(saved))
        y, mean, rstd = ops.layer_norm_fwd(x)
        o = ops.orthogonalize(w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    assert torch.equal(y, ops.layer_norm_fwd(x)[0]) and torch.equal(o, ops.orthogonalize(w))


def test_linear_ce_gradient_against_differences():
    """As for the norm: the quotient of the kernel's losses against that of the 64-bit losses, and <dx, d> against it."""
    from ssecg import ops
    x, w, b, t, _ = _ce_case(19, 9, 32, 50, torch.float32, True, False)
    d, h = _normal(_gen(20), 9, 32), 2.0 ** -7
    at = [R.linear_ce(x + k * h * d, w, t, b) for k in (-2, -1, 1, 2)]
    f = [a[0][0] for a in at]
    q64 = (f[2] - f[1]) / (2 * h)
    q = (ops.linear_ce_fwd(x + h * d, w, t, b)[0].double() - ops.linear_ce_fwd(x - h * d, w, t, b)[0].double()) / (2 * h)
    assert abs(q - q64) <= (at[1][1][0] + at[2][1][0]) / (2 * h)
    third = abs(f[3] - 2 * f[2] + 2 * f[1] - f[0]) / (2 * h ** 3)
    _, saved = ops.linear_ce_fwd(x, w, t, b)
    dx, _, _ = ops.linear_ce_bwd(saved)
    bound = R.linear_ce(x, w, t, b)[1][1]
    assert abs((dx.double() * d.double()).sum() - q64) <= h * h / 3 * third + (bound * d.double().abs()).sum()


# ------------------------------------------------------------------------------------------------ orthogonalised updates: around them
def test_orthogonalize_zero_nan_one_and_none():
    from ssecg import ops
    assert not ops.orthogonalize(torch.zeros(40, 50, device="cuda")).any()
    assert not ops.orthogonalize(torch.zeros(300, 200, device="cuda")).any()
    assert [o.shape for o in ops.orthogonalize([torch.empty(0, 5, device="cuda"), torch.ones(2, 2, device="cuda")])] == [(0, 5), (2, 2)]
    for shape in ((20, 30), (200, 300)):
        x = _normal(_gen(21), *shape)
        x[3, 4] = float("nan")
        assert torch.isnan(ops.orthogonalize(x)).all()
        x[3, 4] = float("inf")
        assert torch.isnan(ops.orthogonalize(x)).any()
    x = _normal(_gen(22), 96, 64).t()                        # strided
    _near(ops.orthogonalize(x), x, "strided")
    big, tiny = _normal(_gen(23), 70, 90) * 1e25, _normal(_gen(24), 70, 90) * 1e-3
    _near(ops.orthogonalize(big), big, "large")              # the norm is a sum in 64 bits
    _near(ops.orthogonalize(tiny, steps=3), tiny, "three steps", steps=3)


def test_orthogonalize_many_matrices_and_their_singular_values():
    from ssecg import ops
    g = _gen(25)
    mats = [_normal(g, 3 + 5 * k, 60 + k) for k in range(40)]      # a chain of 32 matrices and one of 8
    out = ops.orthogonalize(mats)
    for k in (0, 7, 31, 32, 39):
        _near(out[k], mats[k], k)
        s = torch.linalg.svdvals(out[k].double())
        assert 0.3 < s.min() and s.max() < 1.3
    alone = ops.orthogonalize([mats[k] for k in (1, 2)])
    _near(alone[1], mats[2], "alone")


def _optimizer_case(shapes, seed, **kw):
    from ssecg.optim import FusedMuon
    g = _gen(seed)
    ps = [torch.nn.Parameter(_normal(g, *s, scale=0.1)) for s in shapes]
    return ps, FusedMuon(ps, **kw), g


@pytest.mark.parametrize("adjust,nesterov", [("match_rms_adamw", True), ("original", False)])
@pytest.mark.parametrize("shapes", [[(64, 12, 7), (20, 9)], [(128, 64, 3), (64, 128, 1), (200, 40), (300, 300)]])
def test_muon_steps(shapes, adjust, nesterov):
    ps, opt, g = _optimizer_case(shapes, 26, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust)
    ref = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64)) for p in ps]
    plain = [(p.detach().clone(), torch.zeros_like(p)) for p in ps]
    for step in range(3):
        for grp in opt.param_groups:
            grp["lr"] = 0.02 / (step + 1)
        for p in ps:
            p.grad = _normal(g, *p.shape, scale=1e-2)
        opt.step()
        args = (0.02 / (step + 1), 0.9, nesterov, 0.1, adjust)
        ref = [R.muon_step(q, p.grad, v, *args) for p, (q, v) in zip(ps, ref)]
        plain = [R.muon_step(q, p.grad, v, *args, dtype=torch.float32) for p, (q, v) in zip(ps, plain)]
    for p, (q, v), (qp, _) in zip(ps, ref, plain):
        # the update's error is at most 8 times the plain form's (as for the orthogonalisation), and p is rounded three times
        off, own = (p.detach().double() - q).norm(), (qp.double() - q).norm()
        assert off <= 8 * own + 4 * R.U * q.norm(), (tuple(p.shape), float(off), float(own))
        R.within(opt.state[p]["momentum_buffer"], v, 8 * R.U * v.abs().max(), "momentum")


def test_muon_vectors_take_adamw_and_groups_choose():
    from ssecg.optim import FusedAdamW, FusedMuon
    g = _gen(27)
    make = lambda: [torch.nn.Parameter(t.clone()) for t in tensors]   # noqa: E731
    tensors = [_normal(g, 33), _normal(g, 40, 20)]
    grads = [_normal(g, 33), _normal(g, 40, 20)]
    a, b = make(), make()
    muon = FusedMuon([{"params": [a[0]]}, {"params": [a[1]], "muon": False}], lr=1e-2, weight_decay=0.05)
    adam = FusedAdamW(b, lr=1e-2, weight_decay=0.05)
    for _ in range(2):
        for p, q, gr in zip(a, b, grads):
            p.grad, q.grad = gr.clone(), gr.clone()
        muon.step()
        adam.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert set(muon.state[a[1]]) == {"step", "exp_avg", "exp_avg_sq"}


@pytest.mark.parametrize("shapes", [[(40, 20), (7,)], [(200, 300), (7,)]])
def test_muon_skipped_step_touches_nothing_and_checkpoints(shapes):
    ps, opt, g = _optimizer_case(shapes, 28, lr=0.01)
    for p in ps:
        p.grad = _normal(g, *p.shape)
    opt.step(found_inf=torch.zeros(1, device="cuda"))
    before = [p.detach().clone() for p in ps]
    v = opt.state[ps[0]]["momentum_buffer"].clone()
    for p in ps:
        p.grad = torch.full_like(p, float("nan"))
    opt.step(found_inf=torch.ones(1, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(ps, before)) and torch.equal(opt.state[ps[0]]["momentum_buffer"], v)
    sd = copy.deepcopy(opt.state_dict())                     # (a loaded state would share its tensors)
    twins, other, _ = _optimizer_case(shapes, 29, lr=0.5)
    other.load_state_dict(sd)
    assert other.param_groups[0]["lr"] == 0.01 and torch.equal(other.state[twins[0]]["momentum_buffer"], v)
    with torch.no_grad():
        for p, q in zip(twins, ps):
            p.copy_(q)
    for p, q in zip(twins, ps):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step(found_inf=torch.zeros(1, device="cuda"))
    other.step(found_inf=torch.zeros(1, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(twins, ps))


# ------------------------------------------------------------------------------------------------ together, captured, in the plugins
class _Head(torch.nn.Module):
    """What a token model ends in: a matrix, the norm, the classifier."""

    def __init__(self, C, V, dtype):
        from ssecg.nn import LayerNorm
        super().__init__()
        g = torch.Generator().manual_seed(3)
        self.mix = torch.nn.Parameter(torch.randn(C, C, generator=g) / C ** 0.5)
        self.norm = LayerNorm(C)
        self.weight = torch.nn.Parameter(torch.randn(V, C, generator=g) / C ** 0.5)
        self.bias = torch.nn.Parameter(torch.zeros(V))
        self.dtype = dtype

    def forward(self, x, t, conf):
        from ssecg import functional as SF
        h = self.norm((x @ self.mix).to(self.dtype))
        return SF.masked_linear_cross_entropy(h, self.weight.to(self.dtype), t, conf, 0.3, bias=self.bias)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_of_all_together(dtype):
    from ssecg.optim import FusedMuon
    C, V, N = 64, 300, 130
    g = _gen(30)
    x, t, conf = _normal(g, N, C), torch.randint(0, V, (N,), generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    t[:9] = -100
    head = _Head(C, V, dtype).cuda()
    twin = {k: v.detach().double().requires_grad_(True) for k, v in head.named_parameters()}
    opt = FusedMuon([{"params": [head.mix, *head.norm.parameters(), head.bias]}, {"params": [head.weight], "muon": False}], lr=1e-2)
    loss = head(x, t, conf)
    loss.backward()
    h = torch.nn.functional.layer_norm(x.double() @ twin["mix"], (C,), twin["norm.weight"], twin["norm.bias"])
    z = h @ twin["weight"].T + twin["bias"]
    row = torch.nn.functional.cross_entropy(z, t, reduction="none", ignore_index=-100)
    want = (row * (conf >= 0.3)).sum() / (t != -100).sum()
    grads = torch.autograd.grad(want, list(twin.values()))
    # each value is rounded to the type about four times on its way (h, y, E, the gradient), each by half a step: relative to the norm
    tol = 8 * R.half_step(dtype) + 2.0 ** -18
    assert abs(loss.double() - want) <= tol * abs(want)
    for (k, p), gr in zip(head.named_parameters(), grads):
        assert (p.grad.double() - gr).norm() <= tol * gr.norm(), k
    before = {k: p.detach().clone() for k, p in head.named_parameters()}
    opt.step()
    for k, p in head.named_parameters():
        step = (p.detach() - before[k]).norm()
        assert torch.isfinite(p).all() and step > 0, k
    u = 1.95 * head.mix.grad                                 # nesterov, first step: g + 0.95 g
    o = R.orthogonal(u)
    want = before["mix"].double() * (1 - 1e-2 * 0.1) - 1e-2 * 0.2 * C ** 0.5 * o
    assert (head.mix.detach().double() - want).norm() <= 2.0 ** -18 * want.norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step_is_the_eager_step(dtype):
    """Norm, classifier and optimiser in one captured step, replayed with eager steps of another model between the replays."""
    from ssecg.graph import StepGraph
    from ssecg.optim import FusedMuon
    C, V, N = 64, 200, 96
    g = _gen(31)
    batches = [(_normal(g, N, C), torch.randint(0, V, (N,), generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")) for _ in range(7)]

    def build():
        torch.manual_seed(0)
        head = _Head(C, V, dtype).cuda()
        opt = FusedMuon(head.parameters(), lr=1e-2)

        def step(x, t, conf):
            loss = head(x, t, conf)
            loss.backward()
            opt.step()
            opt.zero_grad()
            return (loss.detach(),)
        return head, opt, step
    eager, opt_e, step_e = build()
    other, _, step_o = build()
    graphed, opt_g, step_g = build()
    graph = StepGraph(step_g)
    for k, batch in enumerate(batches):
        for o in (opt_e, opt_g):
            o.param_groups[0]["lr"] = 1e-2 / (k + 1)
        (le,), (lg,) = step_e(*batch), graph(*batch)
        step_o(*batches[-1 - k])
        torch.cuda.synchronize()
        assert torch.equal(le, lg), k
        for (n, p), q in zip(eager.named_parameters(), graphed.parameters()):
            assert torch.equal(p, q), (k, n)
    assert graph.replays >= 4 and not graph.disabled


def test_fixmatch_trains_with_muon():
    from helpers import TRAIN_CFG, build_hip_model, to_dev
    import algorithms.fixmatch as A_fm
    from ssecg import synth
    from ssecg.optim import FusedMuon
    from utils.misc import NativeScalerWithGradNormCount
    from utils.optimizer import get_optimizer_from_config
    dev = torch.device("cuda:0")
    model = build_hip_model(2, synth.model_state(5, 2, trained=True, sharpen=16.0), dev)
    opt = get_optimizer_from_config(dict(TRAIN_CFG, optimizer="muon"), model.parameters())
    assert isinstance(opt, FusedMuon)
    b = to_dev(synth.fixmatch_batch(6, 2, 2, 500), dev)
    before = {k: v.detach().clone() for k, v in model.named_parameters()}
    stats = A_fm.train_one_epoch(model, [b["labeled"]] * 3, [b["unlabeled"]] * 3, opt, dev, 3, NativeScalerWithGradNormCount(), None, False,
                                 dict(TRAIN_CFG))
    assert all(v == v for v in stats.values())
    for k, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[k]), k
    convs = [p for p in model.parameters() if p.dim() >= 2]
    assert all("momentum_buffer" in opt.state[p] for p in convs) and all("exp_avg" in opt.state[p] for p in model.parameters() if p.dim() < 2)


# ------------------------------------------------------------------------------------------------ calls at once, other callers' habits
def test_two_streams_and_two_graphs_share_nothing():
    """The same operators on two streams at once and in two captured graphs replayed in turn: every result is the one alone."""
    from ssecg import ops
    cases = [_ce_case(40 + k, 200 + 31 * k, 96, 700, torch.bfloat16, True, True) for k in range(2)]
    mats = [_normal(_gen(42 + k), 130 + k, 260) for k in range(2)]

    def work(k):
        x, w, b, t, conf = cases[k]
        loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.3)
        y, mean, rstd = ops.layer_norm_fwd(x)
        return (loss, *ops.linear_ce_bwd(saved), y, *ops.layer_norm_bwd(x, x, mean, rstd), ops.orthogonalize(mats[k]))
    alone = [work(k) for k in range(2)]
    torch.cuda.synchronize()
    streams, both = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                both[k] = work(k)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for k in range(2) for p, q in zip(both[k], alone[k]))
    graphs, held = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(work(k))
        graphs.append(g)
    for _ in range(3):
        for k in (1, 0):
            for p in held[k]:
                p.zero_()
            graphs[k].replay()
            work(1 - k)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(held[k], alone[k]))


def test_linear_ce_summed_per_position_and_twice_backward():
    from ssecg import functional as SF
    x, w, b, t, conf = _ce_case(50, 33, 64, 129, torch.float32, True, True)
    x.requires_grad_(True), w.requires_grad_(True)
    per = SF.masked_linear_cross_entropy(x, w, t, conf, 0.4, bias=b, reduction="none")
    total = SF.masked_linear_cross_entropy(x, w, t, conf, 0.4, bias=b, reduction="sum")
    first = torch.autograd.grad(per.sum(), (x, w), retain_graph=True)      # dloss arrives expanded, stride 0
    again = torch.autograd.grad(per.sum(), (x, w))
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    want, bound = R.linear_ce(x.detach(), w.detach(), t, b, conf, 0.4, reduction="sum")
    for got, v, e, what in zip((total.detach(), *first), want, bound, ("loss", "dx", "dw")):
        R.within(got, v, e, what)
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(total, x, create_graph=True)[0]
        g.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_saved_tensors_may_move(dtype):
    """Saved tensors that come back elsewhere in memory, off a 16-byte boundary too (offloading hooks)."""
    from ssecg import functional as SF
    x, w, b, t, _ = _ce_case(51, 40, 64, 100, dtype, True, False)
    x = torch.empty(40 * 64 + 1, dtype=dtype, device="cuda")[1:].view(40, 64).copy_(x).requires_grad_(True)
    w.requires_grad_(True)
    plain = torch.autograd.grad(SF.linear_cross_entropy(x, w, t, bias=b), (x, w))

    def moved(s):
        return torch.empty(s.numel() + 1, dtype=s.dtype, device=s.device)[1:].view(s.shape).copy_(s)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.detach().clone(), moved):
        loss = SF.linear_cross_entropy(x, w, t, bias=b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(loss, (x, w)), plain))


def test_linear_ce_wants_only_what_is_asked_for():
    from ssecg import ops
    x, w, b, t, _ = _ce_case(52, 70, 48, 90, torch.bfloat16, True, False)
    _, saved = ops.linear_ce_fwd(x, w, t, b)
    whole = ops.linear_ce_bwd(saved)
    for k in range(3):
        want = [k == i for i in range(3)]
        part = ops.linear_ce_bwd(saved, None, *want)
        assert [p is not None for p in part] == want and torch.equal(part[k], whole[k])
    assert ops.linear_ce_bwd(saved, None, False, False, False) == (None, None, None)


def test_refusals_on_the_device():
    from ssecg import ops
    from ssecg.lib import SsecgError
    x, w, b, t, conf = _ce_case(53, 12, 64, 30, torch.float32, True, True)
    y, mean, rstd = ops.layer_norm_fwd(x)
    for call in (lambda: ops.linear_ce_fwd(x, w.bfloat16(), t), lambda: ops.linear_ce_fwd(x, w[:, :32], t), lambda: ops.linear_ce_fwd(x, w, t[:5]),
                 lambda: ops.linear_ce_fwd(x, w, t.int()), lambda: ops.linear_ce_fwd(x, w, t, b[:3]), lambda: ops.linear_ce_fwd(x, w, t, b.cpu()),
                 lambda: ops.linear_ce_fwd(x, w, t, conf=conf[:2]), lambda: ops.linear_ce_fwd(x, w, t, conf=conf.half()),
                 lambda: ops.linear_ce_fwd(x, w, t, reduction="avg"), lambda: ops.linear_ce_fwd(x.double(), w.double(), t),
                 lambda: ops.linear_ce_bwd(ops.linear_ce_fwd(x, w, t)[1], torch.ones(12, device="cuda")),
                 lambda: ops.linear_ce_bwd(ops.linear_ce_fwd(x, w, t, reduction="none")[1], torch.ones(1, device="cuda")),
                 lambda: ops.layer_norm_fwd(x, w[0][:5]), lambda: ops.layer_norm_fwd(x, eps=-1.0), lambda: ops.layer_norm_fwd(x[:, :0]),
                 lambda: ops.layer_norm_bwd(y.half(), x, mean, rstd), lambda: ops.layer_norm_bwd(y[:5], x, mean, rstd),
                 lambda: ops.layer_norm_bwd(y, x, mean[:5], rstd), lambda: ops.layer_norm_bwd(y, x, mean.double(), rstd),
                 lambda: ops.orthogonalize(x[0]), lambda: ops.orthogonalize([x, x.half()]), lambda: ops.orthogonalize(x, eps=-1.0),
                 lambda: ops.orthogonalize(x, steps=101), lambda: ops.orthogonalize([x, x.cpu()])):
        with pytest.raises(SsecgError):
            call()


def test_muon_takes_an_adamw_state():
    from ssecg.optim import FusedAdamW, FusedMuon
    g = _gen(54)
    make = lambda: [torch.nn.Parameter(t.clone()) for t in tensors]   # noqa: E731
    tensors = [_normal(g, 30, 20), _normal(g, 9)]
    a, b = make(), make()
    adam, muon = FusedAdamW(a, lr=1e-2), FusedMuon(b, lr=0.3)
    for p in a:
        p.grad = torch.ones_like(p)
    adam.step()
    muon.load_state_dict(copy.deepcopy(adam.state_dict()))
    with torch.no_grad():
        for p, q in zip(b, a):
            p.copy_(q)
    for p, q in zip(a, b):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    adam.step(), muon.step()
    assert torch.equal(a[1], b[1]) and not torch.equal(a[0], b[0])     # the vector continues AdamW, the matrix starts its momentum
    assert torch.equal(muon.state[b[0]]["momentum_buffer"], torch.ones_like(b[0]))


# ------------------------------------------------------------------------------------------------ sizes at which other tiles are chosen
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C,V", [(2990, 1501, 3001), (4500, 2100, 301), (301, 2101, 4501), (601, 209, 4091), (2500, 130, 9001), (2001, 511, 8193)])
def test_linear_ce_larger(N, C, V, dtype):
    from ssecg import ops
    x, w, b, t, conf = _ce_case(N + C + V, N, C, V, dtype, True, True)
    loss, saved = ops.linear_ce_fwd(x, w, t, b, conf, 0.3)
    got = (loss, *ops.linear_ce_bwd(saved))
    want, bound = R.linear_ce(x, w, t, b, conf, 0.3)
    for p, v, e, what in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        R.within(p, v, e, what)


@pytest.mark.parametrize("shapes", [[(2600, 2750)], [(3500, 3001)], [(4090, 4097)], [(5200, 5100)], [(1024, 1030)] * 8])
def test_orthogonalize_larger(shapes):
    from ssecg import ops
    g = _gen(sum(m * 1000 + n for m, n in shapes))
    mats = [_normal(g, m, n) for m, n in shapes]
    for m, o in zip(mats[:2], ops.orthogonalize(mats)):
        _near(o, m, tuple(m.shape))


def test_layer_norm_beyond_2_31_elements():
    from ssecg import ops
    C, rows = 4096, (1 << 19) + 9
    g = _gen(60)
    x = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda")
    piece = _normal(g, 1 << 14, C, dtype=torch.bfloat16)
    for r in range(0, rows, 1 << 14):
        x[r:r + (1 << 14)] = piece[:min(1 << 14, rows - r)]
    w = 1 + _normal(g, C, scale=0.1)
    y, mean, rstd = ops.layer_norm_fwd(x, w)
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd, w)
    few, m, r = ops.layer_norm_fwd(piece[:9], w)
    assert torch.equal(y[-9:], few) and torch.equal(y[:9], few) and torch.equal(mean[-9:], m) and torch.equal(rstd[-9:], r)
    assert torch.equal(dx[-9:], ops.layer_norm_bwd(piece[:9], piece[:9], m, r, w)[0])
    p = piece.double()
    xh = (p - p.mean(1, keepdim=True)) / torch.sqrt(p.var(1, unbiased=False, keepdim=True) + 1e-5)
    for got, terms in ((dw, p * xh), (db, p)):
        want = 32 * terms.sum(0) + terms[:9].sum(0)
        # at most 2049 rows one after the other (of 256 workgroups, or more of them), then their partial sums; the terms' own errors
        bound = R.U * (2049 + 512) * (32 * terms.abs().sum(0) + terms[:9].abs().sum(0))
        R.within(got, want, bound, "column sums")
