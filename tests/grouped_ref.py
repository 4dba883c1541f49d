"""The grouped and 8-bit floating-point products' definitions in 64 bits, and how far a result may be from them (shared by the
CPU and GPU tests).

A sum of K products in the tensor core: the products are exact in fp32; an MMA adds 16 (fp16, bf16) or 32 (e4m3) of them to
the accumulator, at most one fp32 step (2^-23 of the terms' magnitudes) lost per addition and per term, so
(K / 16 + 16) 2^-23 of the sum of magnitudes bounds a 16-bit sum, (4 + 32) 2^-23 a block of 128 e4m3 products.  A block's sum
is multiplied by the rounded product of two scales (2 2^-24) and added (2^-24 of the running sum's magnitude, one per block).
Parts of a tile split along K are added in fp32: at most 16 more additions here.  With the activation, silu(g) u: the errors
of g and u pass through (|silu'| <= 1.1), and the fast exponential and the products add (6 + 3 |g|) 2^-23 of the result.  Then
half a step of the result's type: eps / 2 of it."""
import torch

BLOCK = 128
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FLOOR = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}  # half the smallest step


def offsets_of(counts, first=0, device="cpu"):
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.tensor(counts, dtype=torch.int64), 0).to(torch.int32)
    return (off + first).to(torch.int32).to(device)


def e4m3(v):
    """v (float64) rounded to e4m3's values, ties to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 4, min=-9))
    return torch.clamp(torch.round(v / step) * step, -448, 448)


def _rounded32(v):
    return v.float().double()


def _quantize(x, top):
    """x (float64) by its group's largest magnitude `top` (broadcast): (e4m3 values, scale).  448 / top is taken out of fp32's
    range's reach by a power of two, which changes no rounding."""
    up = torch.where(top < 2.0 ** -100, 2.0 ** 100, 1.0).to(torch.float64)
    inv = _rounded32(448.0 / (top * up))
    q = e4m3(_rounded32(x * up * inv))
    bad = ~torch.isfinite(top)
    q = torch.where(bad | (top == 0), torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(top, float("nan")), _rounded32(top / 448.0))
    return q, scale


def quantize_rows(x):
    x = x.double()
    M, K = x.shape
    kb = -(-K // BLOCK)
    pad = torch.nn.functional.pad(x, (0, kb * BLOCK - K)).view(M, kb, BLOCK)
    top = pad.abs().amax(dim=2, keepdim=True)
    top = torch.where(torch.isnan(pad).any(dim=2, keepdim=True), torch.full_like(top, float("nan")), top)
    q, s = _quantize(pad, top)
    return q.reshape(M, -1)[:, :K], s[:, :, 0]


def quantize_blocks(w):
    w = w.double()
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    pad = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    top = pad.abs().amax(dim=(1, 3), keepdim=True)
    top = torch.where(torch.isnan(pad).any(dim=3, keepdim=True).any(dim=1, keepdim=True), torch.full_like(top, float("nan")), top)
    q, s = _quantize(pad, top)
    return q.reshape(nb * BLOCK, kb * BLOCK)[:N, :K], s[:, 0, :, 0]


def product16(x, w):
    """(x w^T, a bound on its error before the last rounding): x (rows x K), w (N x K)."""
    x, w = x.double(), w.double()
    K = x.shape[1]
    return x @ w.t(), (x.abs() @ w.abs().t()) * ((K / 16 + 16 + 16) * 2.0 ** -23)


def product8(q, s, w, t):
    """The same for e4m3 values q (rows x K), scales s (rows x blocks), w (N x K), t (blocks of rows x blocks)."""
    q, s, w, t = q.double(), s.double(), w.double(), t.double()
    K, N = q.shape[1], w.shape[0]
    x = q * s.repeat_interleave(BLOCK, 1)[:, :K]
    v = w * t.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    return x @ v.t(), (x.abs() @ v.abs().t()) * ((36 + 2 + s.shape[1] + 16) * 2.0 ** -23)


def glu(y, err, blocks):
    """silu(gate) * up of column pairs: in groups of 128 gate and 128 up columns, or the halves."""
    if blocks:
        y, err = (v.reshape(v.shape[0], -1, 2, BLOCK) for v in (y, err))
        (g, u), (eg, eu) = ((v[:, :, 0].flatten(1), v[:, :, 1].flatten(1)) for v in (y, err))
    else:
        n = y.shape[1] // 2
        (g, u), (eg, eu) = ((v[:, :n], v[:, n:]) for v in (y, err))
    a = g * torch.sigmoid(g)
    out = a * u
    return out, 1.1 * eg * (u.abs() + eu) + (a.abs() + 1.1 * eg) * eu + out.abs() * (6 + 3 * g.abs()) * 2.0 ** -23


def grouped(x, off, weight, n, product):
    """Rows of each expert times its weights: (y, error bound, covered rows)."""
    y = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
    err, covered = torch.zeros_like(y), torch.zeros(x.shape[0], dtype=torch.bool, device=x.device)
    o = off.tolist()
    for e in range(len(o) - 1):
        if o[e] < o[e + 1]:
            r = slice(o[e], o[e + 1])
            y[r], err[r] = product(r, e)
            covered[r] = True
    return y, err, covered


def weight_gradient(dY, X, off):
    """(dW, error bound): E x N x K."""
    o = off.tolist()
    E = len(o) - 1
    y = torch.zeros((E, dY.shape[1], X.shape[1]), dtype=torch.float64, device=X.device)
    err = torch.zeros_like(y)
    for e in range(E):
        r = slice(o[e], o[e + 1])
        if o[e] < o[e + 1]:
            y[e], err[e] = product16(dY[r].t(), X[r].t())
    return y, err


def close(got, y, err):
    """Whether every element is within the bound (NaN where the definition is NaN)."""
    tol = err + (y.abs() + err) * HALF_STEP[got.dtype] + FLOOR[got.dtype]
    g = got.double()
    ok = ((g - y).abs() <= tol) | (torch.isnan(g) & torch.isnan(y)) | (g == y)
    return bool(ok.all()), float(((g - y).abs() / tol).nan_to_num(0).max()) if g.numel() else 0.0
