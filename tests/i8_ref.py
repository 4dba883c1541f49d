"""The 8-bit operators' definition in 64 bits, and how far a result may be from it (shared by the CPU and GPU tests).

A value is float(s) * row scale * column scale: three roundings of 2^-24 of it, a fourth where the row scale itself was
rounded (a / 127), then half a step of C's type, eps / 2 of
it (for fp16 at least 2^-25, half its smallest step).  With the activation, silu(g) u: the fast exponential's
(2 + 1.16 |g|) 2^-23, g's own three roundings through exp (3 |g| 2^-24), u's three, the division's and the products'
three: (6 + 3 |g|) 2^-23 in all; below g = -88, where exp(-g) leaves fp32, the result is 0 for up to 2^-120 |u|."""
import numpy as np

HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
FLOOR = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 2.0 ** -150}


def quantize_exact(x):
    """(q, scale) of rows x (float64 holding fp16 or bf16 values): half-way cases settled in integers."""
    a = np.abs(x).max(axis=1, keepdims=True)
    bad = ~np.isfinite(a)
    safe = np.where(bad | (a == 0), 1.0, a)
    xs = np.where(bad, 0.0, x)
    n = np.floor(127.0 * np.abs(xs) / safe)  # then corrected: the remainder is exact in 64 bits
    rem = 127.0 * np.abs(xs) - n * safe
    n = np.where(rem < 0, n - 1, np.where(rem >= safe, n + 1, n))
    rem = 127.0 * np.abs(xs) - n * safe
    up = (2 * rem > safe) | ((2 * rem == safe) & (n % 2 == 1))
    q = np.sign(xs) * (n + up)
    return q, np.where(bad[:, 0], np.nan, a[:, 0] / 127.0)


def product(q, qs, w, ws):
    return (q.astype(np.float64) @ w.astype(np.float64).T) * qs.astype(np.float64)[:, None] * ws.astype(np.float64)


def swiglu(y):
    M, N = y.shape
    y = y.reshape(M, N // 256, 2, 128)
    g, u = y[:, :, 0].reshape(M, N // 2), y[:, :, 1].reshape(M, N // 2)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u, g, u


def outside(got, y, kind, activation=False):
    """The elements of `got` farther from the definition than the arithmetic above allows."""
    if activation:
        ref, g, u = swiglu(y)
        tol = np.abs(ref) * (HALF_STEP[kind] + (6 + 3 * np.abs(g)) * 2.0 ** -23) + np.where(g < -87, 2.0 ** -120, 0) * np.abs(u)
    else:
        ref = y
        tol = np.abs(ref) * (HALF_STEP[kind] + 4 * 2.0 ** -24)
    # a value past C's largest rounds to infinity there
    top = {"fp16": 65520.0, "bf16": 3.396e38, "fp32": 3.403e38}[kind]
    ok = (np.abs(got - ref) <= tol + FLOOR[kind]) | (np.isinf(got) & (np.abs(ref) * (1 + 2.0 ** -20) >= top))
    return np.argwhere(~ok)
