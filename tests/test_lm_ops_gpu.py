"""GPU: layer norm, classifier + cross entropy over a large vocabulary, orthogonalised updates - against their plain forms in 64
bits, at the sizes, types, masks and strides where they can go wrong (bounds: tests/lm_ref.py, derived from the arithmetic)."""
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
