"""Element-wise bounds of the classifier loss for operands of any range (test infrastructure): each row of logits is held to its own
size, each class's row of dW to its own probabilities, so nothing far larger elsewhere excuses an error.

u = 2^-24 is the unit roundoff of fp32.  A product summed over n terms is off by at most 8 sqrt(n) u sum|a||b| (rounding errors of random
sign, eight standard deviations).  fp32 operands that enter as three 8-bit parts are exact, and of nine products of parts the three
smallest, below 2^-26 of |a||b| together (2^-9 2^-18 twice and 2^-36), are left out."""
import torch

from lm_ref import U, half_step, rounded


def linear_ce(x, w, target, bias=None, conf=None, thresh=0.0, ignore=-100, reduction="mean", dloss=None, held=None):
    """-> ((loss, dx, dw, db), bounds) in 64 bits; rows that do not count enter as zeros.  ``held``: half a step of the type the gradient of
    the logits is held in (default: the operands', fp32: exact)."""
    N, C = x.shape
    V = w.shape[0]
    kept = target != ignore
    gate = kept if conf is None else kept & (conf >= thresh)
    count = max(1, int(kept.sum()))
    x64, w64 = torch.where(gate[:, None], x, torch.zeros_like(x)).double(), w.double()
    z = x64 @ w64.T
    if bias is not None:
        z = z + bias.double()
    lse = torch.logsumexp(z, 1)
    t = torch.where(kept, target, torch.zeros_like(target))[:, None]
    zt = z.gather(1, t)[:, 0]
    row = torch.where(gate, lse - zt, torch.zeros_like(lse))
    d = torch.ones(N if reduction == "none" else (), dtype=torch.float64, device=x.device) if dloss is None else dloss.double()
    f = d / count if reduction == "mean" else d
    f = f[:, None] if f.dim() else f
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, t, 1.0)
    G = gate[:, None].double()
    E = (p - onehot) * G * f
    loss = row if reduction == "none" else (row.sum() / count if reduction == "mean" else row.sum())
    # logits: the product, the bias added to it; a class at -inf is exact.  lse: the classes' errors by their weight, the sum of V
    # exponentials (each within 2 u; chains of at most 512 additions), its own rounding, once in the forward pass and once as it is read
    dz = (8 * C ** 0.5 * U + 2.0 ** -26) * (x64.abs() @ w64.abs().T) + 2 * U * torch.where(torch.isinf(z), torch.zeros_like(z), z.abs())
    dlse = (p * dz).sum(1) + 32 * U + 2 * U * lse.abs()
    trow = torch.where(gate, dlse + dz.gather(1, t)[:, 0] + U * row.abs(), torch.zeros_like(lse))
    tl = trow if reduction == "none" else (trow.sum() / count if reduction == "mean" else trow.sum()) + 2 * U * loss.abs()
    # E: exp(z - lse), whose argument is rounded twice and which is off by 2 u itself; 1 - p; its rounding to the held type
    own = (0.0 if x.dtype == torch.float32 else half_step(x.dtype)) if held is None else held
    arg = torch.where(torch.isinf(z), torch.zeros_like(z), (z - lse[:, None]).abs())
    tE = G * f.abs() * (p * (dz + dlse[:, None] + 4 * U * (1 + arg)) + onehot * U) + (own + 2 * U) * E.abs()
    dx, dw, db = E @ w64, E.T @ x64, E.sum(0)
    rep = 2.0 ** -26 if x.dtype == torch.float32 else 0.0
    tx = tE @ w64.abs() + (8 * V ** 0.5 * U + rep) * (E.abs() @ w64.abs()) + 2 * U * dx.abs() + rounded(dx, x.dtype)
    tw = tE.T @ x64.abs() + (8 * N ** 0.5 * U + rep) * (E.abs().T @ x64.abs()) + 2 * U * dw.abs() + rounded(dw, x.dtype)
    tb = (tE + 8 * N ** 0.5 * U * E.abs()).sum(0) + 2 * U * db.abs() + rounded(db, torch.float32)
    return (loss, dx, dw, db), (tl, tx, tw, tb)
