"""Plain 64-bit forms of the token-level operators, and error bounds of a computation in 32 bits (test infrastructure).

u = 2^-24 is the unit roundoff of fp32.  A sum of n terms in fp32 is off by at most D u sum|terms|, D the longest chain of
additions; for long products the bound below takes 8 sqrt(n) u (rounding errors of random sign; 8 standard deviations)."""
import torch

U = 2.0 ** -24
COEF = (3.4445, -4.7750, 2.0315)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(v, dtype):
    """How far a rounding of v to ``dtype`` may be off: half a step, eps / 2 of a normal value; below the smallest normal number (tiny)
    the steps no longer shrink: the spacing there is tiny * eps, so half a step is tiny * eps / 2 (fp16: 2^-14 2^-10 / 2 = 2^-25)."""
    f = torch.finfo(dtype)
    return (f.eps / 2 * v.abs()).clamp(min=f.tiny * f.eps / 2)


def layer_norm(x, dy, w, b, eps):
    """-> ((y, dx, dw, db) in 64 bits, the bound of each for outputs of x's type)."""
    x64, dy64 = x.double(), dy.double()
    C = x.shape[-1]
    w64 = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x64.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt((x64 - mu).square().mean(-1, keepdim=True) + eps)
    xh = (x64 - mu) * rs
    y = xh * w64 + b64
    g = dy64 * w64
    dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    dw, db = (dy64 * xh).flatten(0, -2).sum(0), dy64.flatten(0, -2).sum(0)
    # a row's sums: at most 32 terms by one thread, 6 steps within a wave, 16 waves -> D = 64 with the roundings of the terms
    D = 64
    ah = x64.abs().amax(-1, keepdim=True) * rs            # |xh| before the mean cancels: the error of xh is 2 D u of this
    ty = rounded(y, x.dtype) + 4 * D * U * (ah * w64.abs() + y.abs() + b64.abs())
    G = g.abs().amax(-1, keepdim=True)
    tx = rounded(dx, x.dtype) + 8 * D * U * rs * G * (2 + ah * ah.clamp(min=1))
    rows = max(1, x.numel() // C)
    Dr = min(rows, 256) + 64                              # rows of a workgroup one after the other, then its partial sums
    tw = (Dr + 4 * D) * U * (dy64.abs() * ah).flatten(0, -2).sum(0)
    tb = Dr * U * dy64.abs().flatten(0, -2).sum(0)
    return (y, dx, dw, db), (ty, tx, tw, tb)


def linear_ce(x, w, target, bias=None, conf=None, thresh=0.0, ignore=-100, reduction="mean", dloss=None):
    """-> ((loss, dx, dw, db), bounds).  Rows that do not count enter as zeros."""
    N, C = x.shape
    V = w.shape[0]
    kept = target != ignore
    gate = kept if conf is None else kept & (conf >= thresh)
    count = max(1, int(kept.sum()))
    x64 = torch.where(gate[:, None], x, torch.zeros_like(x)).double()
    w64 = w.double()
    z = x64 @ w64.T
    if bias is not None:
        z = z + bias.double()
    lse = torch.logsumexp(z, 1)
    t = torch.where(kept, target, torch.zeros_like(target))
    row = torch.where(gate, lse - z.gather(1, t[:, None])[:, 0], torch.zeros_like(lse))
    d = torch.ones(N if reduction == "none" else (), dtype=torch.float64, device=x.device) if dloss is None else dloss.double()
    f = d / count if reduction == "mean" else d
    p = torch.softmax(z, 1)
    onehot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    E = (p - onehot) * gate[:, None] * (f[:, None] if f.dim() else f)
    loss = row if reduction == "none" else (row.sum() / count if reduction == "mean" else row.sum())
    # logits: fp32 accumulation of C products, operands exact (16-bit) or held in 22 bits and more (2^-23 each, lo lo 2^-22)
    az = x64.abs() @ w64.abs().T
    dz = 8 * C ** 0.5 * U * az + (2.0 ** -21 * az if x.dtype == torch.float32 else 0) + 4 * U * z.abs()
    dzm = dz.amax(1)
    trow = torch.where(gate, 2 * dzm + 16 * U * (lse.abs() + 1), torch.zeros_like(lse))
    tl = trow if reduction == "none" else (trow.sum() / count if reduction == "mean" else trow.sum()) + 16 * U * loss.abs()
    # E: relative error of exp(z - lse) plus its rounding to the held type (fp32: 22 bits); a target's entry rounds as a whole
    held = 2.0 ** -22 if x.dtype == torch.float32 else half_step(x.dtype)
    spread = (z - lse[:, None]).abs()
    ef = (f.abs()[:, None] if f.dim() else f.abs()) * gate[:, None]
    tE = held * E.abs() + ef * p * ((dz + dzm[:, None]) + 4 * U * (1 + spread)) + ef * 2.0 ** -38
    rep = 2.0 ** -21 if x.dtype == torch.float32 else 0.0
    dx, dw, db = E @ w64, E.T @ x64, E.sum(0)
    tx = tE @ w64.abs() + (8 * V ** 0.5 * U + rep) * (E.abs() @ w64.abs()) + rounded(dx, x.dtype)
    tw = tE.T @ x64.abs() + (8 * N ** 0.5 * U + rep) * (E.abs().T @ x64.abs()) + rounded(dw, x.dtype)
    tb = (tE + 8 * N ** 0.5 * U * E.abs()).sum(0)
    return (loss, dx, dw, db), (tl, tx, tw, tb)


def orthogonal(g, steps=5, eps=1e-7, dtype=torch.float64):
    a, b, c = COEF
    x = g.to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (torch.sqrt((x * x).sum()) + eps)
    for _ in range(steps):
        A = x @ x.T
        x = a * x + (b * A + c * (A @ A)) @ x
    return (x.T if tall else x).contiguous()


def muon_step(p, g, v, lr, momentum, nesterov, wd, adjust, steps=5, dtype=torch.float64):
    """-> (p, v) after one step."""
    m, n = p.shape[0], p.numel() // p.shape[0]
    v = momentum * v.to(dtype) + g.to(dtype)
    u = (g.to(dtype) + momentum * v) if nesterov else v
    o = orthogonal(u.reshape(m, n), steps, dtype=dtype).reshape(p.shape)
    s = 0.2 * max(m, n) ** 0.5 if adjust == "match_rms_adamw" else max(1.0, m / n) ** 0.5
    return p.to(dtype) * (1 - lr * wd) - lr * s * o, v


def within(got, want, bound, what):
    """Every element within its bound; NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    off = torch.where(got == want, torch.zeros_like(got), (got - want).abs()).nan_to_num(0.0)
    bad = off > bound
    if bool(bad.any()):
        k = int(torch.argmax((off / bound.clamp(min=1e-300) if torch.is_tensor(bound) else off / bound).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound; worst at {k}: {got.flatten()[k].item()!r} "
                             f"for {want.flatten()[k].item()!r}")
