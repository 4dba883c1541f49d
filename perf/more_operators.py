"""Products grouped by expert and products in 8-bit floating point as measured operators: their cases, their inputs and
their plain forms (elementary torch operations in 32 bits), beside the calls a user makes of the library.

Operators
  grouped     rows of X (R x K, fp16 or bf16) sorted by expert, expert e's rows being offsets[e] .. offsets[e + 1] - 1:
                tn      Y_r = X_r W_e^T, W: E x N x K (a layer's forward product)
                nn      Y_r = X_r W_e, W: E x K x N (the gradient of its input)
                swiglu  silu(X_r G_e^T) * (X_r U_e^T), W: E x 2F x K, the gate rows G_e then the up rows U_e
  grouped_dw  dW_e = dY_e^T X_e over expert e's rows, E x N x K (the gradient of the weights; 0 without rows)
  quantize    fp16 or bf16 to e4m3 with a scale a / 448 for each group (a the group's largest magnitude, s = fl32(a / 448)):
                q = e4m3(fl32(x fl32(448 / a))), rounded to nearest, ties to even
                rows    groups of 128 along a row (activations)
                blocks  128 x 128 blocks (weights)
  linear_f8   Y = X W^T in X's type: X quantised as `rows`, W given as `blocks` gives it,
                y_mn = sum over blocks b of 128 of K: s_mb t_{n / 128, b} sum_{k in b} q_mk w_nk
              swiglu: W's rows in groups of 128 gate and 128 up rows, silu(gate) * up, N / 2 columns.
              E > 0: grouped by expert as above, W: E x N x K (swiglu: gate rows then up rows).
"""
import math
import os
import sys

import torch

own = False  # True: run() calls the library's operators

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemm-ladder_b200")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
TOP = 448.0  # e4m3's largest value
BLOCK = 128


def _bwgemm():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import bwgemm

    return bwgemm


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode batch routed over many small experts, most with one row or none: the stream of the active weights
        {"name": "grouped_few", "op": "grouped", "form": "tn", "R": 24, "E": 64, "N": 2048, "K": 1024, "dtype": "bf16"},
        # a prefill chunk through wide experts, gate and up with the activation; a ragged number of rows everywhere
        {"name": "grouped_swiglu", "op": "grouped", "form": "swiglu", "R": 8191, "E": 32, "N": 5760, "K": 2880,
         "dtype": "fp16"},
        # a training step's input gradient over many experts
        {"name": "grouped_dx", "op": "grouped", "form": "nn", "R": 16384, "E": 64, "N": 2048, "K": 2816, "dtype": "bf16"},
        # the weight gradient of few rows and odd sizes: the write of the gradient
        {"name": "grouped_dw_few", "op": "grouped_dw", "R": 1000, "E": 16, "N": 1352, "K": 2048, "dtype": "fp16"},
        # a training step's weight gradient
        {"name": "grouped_dw", "op": "grouped_dw", "R": 16384, "E": 64, "N": 2816, "K": 2048, "dtype": "bf16"},
        # a prefill chunk's activations, a width that ends inside a group
        {"name": "quantize_rows", "op": "quantize", "form": "rows", "M": 4099, "K": 7184, "dtype": "bf16"},
        # a weight matrix
        {"name": "quantize_blocks", "op": "quantize", "form": "blocks", "M": 10240, "K": 8192, "dtype": "bf16"},
        # one decode step of one sequence through a qkv projection: the launches and the stream of the weights
        {"name": "f8_m1", "op": "linear_f8", "form": "tn", "M": 1, "E": 0, "N": 10240, "K": 8192, "dtype": "bf16"},
        # an odd decode batch through a down projection: a long K, few output columns
        {"name": "f8_m17_down", "op": "linear_f8", "form": "tn", "M": 17, "E": 0, "N": 8192, "K": 28672, "dtype": "fp16"},
        # a prefill chunk of odd length through the gate and up projections of a gated MLP
        {"name": "f8_swiglu_m1001", "op": "linear_f8", "form": "swiglu", "M": 1001, "E": 0, "N": 28672, "K": 4112,
         "dtype": "bf16"},
        # the square shape of the ladder: the tensor cores' rate
        {"name": "f8_ladder", "op": "linear_f8", "form": "tn", "M": 8192, "E": 0, "N": 8192, "K": 8192, "dtype": "bf16"},
        # a prefill chunk routed over many experts in 8 bits
        {"name": "f8_grouped", "op": "linear_f8", "form": "tn", "M": 8192, "E": 64, "N": 4096, "K": 2048, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["grouped", "grouped", "grouped_dw", "quantize", "linear_f8", "linear_f8", "linear_f8"])
    while True:
        if op in ("grouped", "grouped_dw"):
            form = rng.choice(["tn", "nn", "swiglu"]) if op == "grouped" else "dw"
            c = {"op": op, "form": form, "R": _log_int(rng, 1, 32768), "E": rng.choice([1, 4, 8, 16, 24, 32, 60, 64, 128, 160]),
                 "N": _log_int(rng, 256, 8192, 16), "K": _log_int(rng, 128, 8192, 8), "dtype": dtype}
            if c["R"] * c["N"] * c["K"] <= 1.6e11 and c["E"] * c["N"] * c["K"] <= 9e8:
                return c
        elif op == "quantize":
            c = {"op": op, "form": rng.choice(["rows", "blocks"]), "M": _log_int(rng, 1, 16384),
                 "K": _log_int(rng, 128, 28672, 16), "dtype": dtype}
            if c["M"] * c["K"] <= 1.2e8:
                return c
        else:
            form = rng.choice(["tn", "tn", "swiglu"])
            c = {"op": op, "form": form, "M": _log_int(rng, 1, 16384),
                 "E": rng.choice([0, 0, 0, 8, 16, 32, 64, 128]), "N": _log_int(rng, 256, 32768, 256 if form == "swiglu" else 16),
                 "K": _log_int(rng, 128, 28672, 16), "dtype": dtype}
            if c["M"] * c["N"] * c["K"] <= 4e11 and max(1, c["E"]) * c["N"] * c["K"] <= 9e8:
                return c


# ------------------------------------------------------------------ the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, cols, dtype, g):
    """Rows as a transformer's hidden states are: unit variance, a few channels several times larger."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    loud = 1.0 + 7.0 * (torch.rand((cols,), generator=g, device="cuda") < 0.004).float()
    return (x * loud).to(dtype)


def _popularity(E):
    """How often each expert is chosen: a few several times as often as the rest."""
    return [1.0 / (3.0 + (7 * e) % E) + 0.5 / E for e in range(E)]


def _offsets(rows, E, g):
    """The rows' experts drawn by popularity, as prefix sums of the experts' numbers of rows."""
    p = torch.tensor(_popularity(E), device="cuda")
    ids = torch.multinomial(p, rows, replacement=True, generator=g)
    off = torch.zeros((E + 1,), dtype=torch.int32, device="cuda")
    off[1:] = torch.cumsum(torch.bincount(ids, minlength=E), 0).to(torch.int32)
    return off


def _weights(E, N, K, dtype, g):
    w = torch.empty((E, N, K), dtype=dtype, device="cuda")
    for e in range(E):
        w[e] = torch.randn((N, K), generator=g, device="cuda") * (1.0 / math.sqrt(K))
    return w


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    op, s = case["op"], dict(case)
    if op == "quantize":
        s["X"] = _activations(case["M"], case["K"], dtype, g)
    elif op == "grouped_dw":
        s["dY"] = torch.randn((case["R"], case["N"]), generator=g, device="cuda").to(dtype)
        s["X"] = _activations(case["R"], case["K"], dtype, g)
        s["offsets"] = _offsets(case["R"], case["E"], g)
    elif op == "grouped":
        s["X"] = _activations(case["R"], case["K"], dtype, g)
        s["offsets"] = _offsets(case["R"], case["E"], g)
        E, N, K = case["E"], case["N"], case["K"]
        s["W"] = _weights(E, K, N, dtype, g) if case["form"] == "nn" else _weights(E, N, K, dtype, g)
    else:
        M, E, N, K = case["M"], case["E"], case["N"], case["K"]
        s["X"] = _activations(M, K, dtype, g)
        if E:
            s["offsets"] = _offsets(M, E, g)
        nb, kb = -(-N // BLOCK), -(-K // BLOCK)
        q = torch.empty((max(1, E), N, K), dtype=F8, device="cuda")
        t = torch.empty((max(1, E), nb, kb), dtype=torch.float32, device="cuda")
        for e in range(max(1, E)):  # each expert's weights quantised block by block
            w = (torch.randn((N, K), generator=g, device="cuda") * (1.0 / math.sqrt(K))).to(dtype)
            q[e], t[e] = _quantize_blocks_plain(w)
        s["W"], s["w_scale"] = (q, t) if E else (q[0], t[0])
    return s


# ------------------------------------------------------------------ one pass
def _scales_plain(amax):
    """(448 / amax, amax / 448), each the 32-bit quotient (a Python number in their place would be multiplied by its
    counterpart's reciprocal)."""
    top = torch.full_like(amax, TOP)
    return torch.where(amax > 0, top / amax, torch.zeros_like(amax)), amax / top


def _quantize_rows_plain(x):
    M, K = x.shape
    kb = -(-K // BLOCK)
    xf = torch.zeros((M, kb * BLOCK), dtype=torch.float32, device=x.device)
    xf[:, :K] = x.float()
    xf = xf.view(M, kb, BLOCK)
    inv, scale = _scales_plain(xf.abs().amax(dim=2))
    q = (xf * inv[:, :, None]).to(F8)
    return q.view(M, kb * BLOCK)[:, :K].contiguous(), scale


def _quantize_blocks_plain(w):
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    wf = torch.zeros((nb * BLOCK, kb * BLOCK), dtype=torch.float32, device=w.device)
    wf[:N, :K] = w.float()
    wf = wf.view(nb, BLOCK, kb, BLOCK)
    inv, scale = _scales_plain(wf.abs().amax(dim=(1, 3)))
    q = (wf * inv[:, None, :, None]).to(F8)
    return q.view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous(), scale


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _spread(t, rows, cols):
    """A scale per 128 x 128 block as a factor per element."""
    return t.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _grouped_plain(x, offsets, n, weight):
    """Rows of each expert times weight(e) (K x n), in 32 bits."""
    y = torch.empty((x.shape[0], n), dtype=torch.float32, device=x.device)
    off = offsets.tolist()
    for e in range(len(off) - 1):
        a, b = off[e], off[e + 1]
        if a < b:
            y[a:b] = x[a:b] @ weight(e)
    return y


def run(s):
    op, form = s["op"], s.get("form")
    if own:
        bw = _bwgemm()
        if op == "grouped":
            if form == "nn":
                return bw.gemm_grouped(s["X"], s["W"], s["offsets"])
            return bw.gemm_grouped_tn(s["X"], s["W"], s["offsets"], swiglu=form == "swiglu")
        if op == "grouped_dw":
            return bw.gemm_grouped_dw(s["dY"], s["X"], s["offsets"])
        if op == "quantize":
            q, t = bw.quantize_f8(s["X"]) if form == "rows" else bw.quantize_blocks_f8(s["X"])
            return q, t
        return bw.linear_f8(s["X"], s["W"], s["w_scale"], offsets=s.get("offsets"), swiglu=form == "swiglu")
    dtype = s["X"].dtype
    if op == "quantize":
        return _quantize_rows_plain(s["X"]) if form == "rows" else _quantize_blocks_plain(s["X"])
    if op == "grouped_dw":
        off = s["offsets"].tolist()
        dw = torch.zeros((s["E"], s["N"], s["K"]), dtype=dtype, device=s["X"].device)
        for e in range(s["E"]):
            a, b = off[e], off[e + 1]
            if a < b:
                dw[e] = (s["dY"][a:b].float().t() @ s["X"][a:b].float()).to(dtype)
        return dw
    N, K, w = s["N"], s["K"], s["W"]
    if op == "grouped":
        x = s["X"].float()
        y = _grouped_plain(x, s["offsets"], N, lambda e: w[e].float() if form == "nn" else w[e].float().t())
    else:
        q, t = _quantize_rows_plain(s["X"])
        x = q.float() * t.repeat_interleave(BLOCK, 1)[:, :K]
        if s["E"]:
            y = _grouped_plain(x, s["offsets"], N, lambda e: (w[e].float() * _spread(s["w_scale"][e], N, K)).t())
        else:
            y = x @ (w.float() * _spread(s["w_scale"], N, K)).t()
    if form == "swiglu":
        if op == "linear_f8" and not s["E"]:
            y = y.view(-1, N // 256, 2, 128)
            y = (_silu(y[:, :, 0]) * y[:, :, 1]).reshape(-1, N // 2)
        else:
            y = _silu(y[:, :N // 2]) * y[:, N // 2:]
    return y.to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "quantize":
        M, K = case["M"], case["K"]
        groups = M * -(-K // BLOCK) if case["form"] == "rows" else -(-M // BLOCK) * -(-K // BLOCK)
        return {"bytes": 3.0 * M * K + 4.0 * groups, "flops": 2.0 * M * K}
    rows, E, N, K = case.get("R", case.get("M")), case["E"], case["N"], case["K"]
    if op == "grouped_dw":
        return {"bytes": 2.0 * rows * (N + K) + 2.0 * E * N * K, "flops": 2.0 * rows * N * K}
    active = 1.0
    if E:  # expected experts that some row chooses
        p = _popularity(E)
        active = sum(1.0 - (1.0 - v / sum(p)) ** rows for v in p)
    out = N // 2 if case["form"] == "swiglu" else N
    size = 2.0 if op == "grouped" else 1.0 + 4.0 / BLOCK ** 2
    return {"bytes": 2.0 * rows * (K + out) + size * active * N * K, "flops": 2.0 * rows * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def _e4m3_exact(v):
    """v (float64) rounded to e4m3's values: 4 significant bits down to 2^-6, steps of 2^-9 below; ties to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 4, min=-9))
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _groups_exact(x, rows):
    """(values e4m3 holds, scales), groups of `rows` rows x 128 columns.  The definition's own roundings to 32 bits are made
    by converting; a conversion of a 64-bit quotient or product of 32-bit values is the correctly rounded one."""
    M, K = x.shape
    q = torch.empty((M, K), dtype=torch.float64, device=x.device)
    scales = []
    for k in range(0, K, BLOCK):
        part = x[:, k:k + BLOCK].double()
        top = part.abs().max(dim=1).values
        if rows > 1:
            pad = torch.nn.functional.pad(top, (0, -M % rows)).view(-1, rows)
            each = pad.max(dim=1).values
            top = each.repeat_interleave(rows)[:M]
        else:
            each = top
        scales.append((each / TOP).float().double())
        inv = (TOP / top).float().double()
        inv[top == 0] = 0.0
        q[:, k:k + BLOCK] = _e4m3_exact((part * inv[:, None]).float().double())
    return q, torch.stack(scales, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    op, form = s["op"], s.get("form")
    if op == "quantize":
        return _groups_exact(s["X"], 1 if form == "rows" else BLOCK)
    if op == "grouped_dw":
        off = s["offsets"].cpu().numpy()
        dw = torch.zeros((s["E"], s["N"], s["K"]), dtype=torch.float64, device="cuda")
        for e in range(s["E"]):
            rows = slice(int(off[e]), int(off[e + 1]))
            dw[e] = torch.einsum("tn,tk->nk", s["dY"][rows].double(), s["X"][rows].double())
        return dw
    N, K, E = s["N"], s["K"], s["E"]
    if op == "grouped":
        x = s["X"].double()
    else:
        q, t = _groups_exact(s["X"], 1)
        x = q * torch.repeat_interleave(t, BLOCK, dim=1)[:, :K]
    y = torch.empty((x.shape[0], N), dtype=torch.float64, device="cuda")
    off = s["offsets"].cpu().numpy() if E else (0, x.shape[0])
    for e in range(max(1, E)):
        rows = slice(int(off[e]), int(off[e + 1]))
        w = s["W"][e] if s["W"].dim() == 3 else s["W"]
        for n in range(0, N, BLOCK):
            if op == "linear_f8":
                t = s["w_scale"][e] if s["w_scale"].dim() == 3 else s["w_scale"]
                wn = w[n:n + BLOCK].double() * torch.repeat_interleave(t[n // BLOCK].double(), BLOCK)[:K]
            elif form == "nn":
                wn = w[:, n:n + BLOCK].t().double()
            else:
                wn = w[n:n + BLOCK].double()
            y[rows, n:n + BLOCK] = torch.einsum("tk,nk->tn", x[rows], wn)
    if form == "swiglu":
        if op == "linear_f8" and not E:
            y = y.reshape(-1, N // 256, 256)
            gate, up = y[..., :128], y[..., 128:]
        else:
            gate, up = y[:, :N // 2], y[:, N // 2:]
        y = (gate * torch.sigmoid(gate) * up).reshape(x.shape[0], N // 2)
    return y
