"""The mixture-of-experts layer's definition in 64 bits, and how far a result may be from it (shared by the CPU and GPU
tests).

The kernel's arithmetic: g, u, y are fp32 sums of exact products, 16 at a time; a step loses at most 2^-22 of the sum of
the products' magnitudes so far, so a sum over K products with n partials is within (K / 16 + n) 2^-22 of A, the sum of
all magnitudes.  p: the logits are sums of D / 32 + 5 roundings of 2^-24 of their magnitudes; an error d in each logit
changes p by a factor within exp(2 d); the exponential and the division add 2^-20.  h = p silu(g) u is rounded to the
operands' type: eps / 2 of it (fp16: at least 2^-25); |silu'| <= 1.1; the fast exponential and the products' roundings
are within (8 + 3 |g|) 2^-23.  y is rounded once."""
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def route(X, R, k, renormalize=True):
    """(ids, weights, bound on the weights' relative error): equal logits go to the lower index."""
    x, r = X.double(), R.double()
    logits = x @ r.t()
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    ids, v = order.indices[:, :k], order.values[:, :k]
    e = torch.exp(v - v[:, :1])
    total = e.sum(1, keepdim=True) if renormalize else torch.exp(logits - v[:, :1]).sum(1, keepdim=True)
    d = (x.shape[1] / 32 + 5) * 2.0 ** -24 * (x.abs() @ r.abs().t()).amax(1, keepdim=True)
    return ids, e / total, torch.expm1(2 * d) + 2.0 ** -20


def layer(X, ids, weights, w_err, W1, W2):
    """(y, tolerance) in 64 bits for the given choice and weights."""
    T, D = X.shape
    F = W2.shape[2]
    x = X.double()
    y, tol, mag = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    unit = 2.0 ** -22
    active = torch.unique(ids).tolist()
    for e in active:
        tok, j = torch.nonzero(ids == e, as_tuple=True)
        p = weights[tok, j][:, None].double()
        w1, w2 = W1[e].double(), W2[e].double()
        gu, au = x[tok] @ w1.t(), (x[tok].abs() @ w1.abs().t()) * (D / 16 + 8) * unit
        g, u, dg, du = gu[:, :F], gu[:, F:], au[:, :F], au[:, F:]
        silu = g * torch.sigmoid(g)
        h = p * silu * u
        dh = p * (1.1 * dg * (u.abs() + du) + silu.abs() * du) + h.abs() * (
            HALF[X.dtype] + (8 + 3 * g.abs()) * 2.0 ** -23 + w_err[tok]) + TINY[X.dtype]
        y[tok] += h @ w2.t()
        tol[tok] += dh @ w2.abs().t()
        mag[tok] += (h.abs() + dh) @ w2.abs().t()
    tol += mag * (len(active) * F / 16 + 160) * unit
    return y, tol + (y.abs() + tol) * HALF[X.dtype] + TINY[X.dtype]
