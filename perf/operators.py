"""The 8-bit linear layers and the mixture-of-experts MLP of few tokens as measured operators: their cases, their inputs
and their plain forms (elementary torch operations in 32 bits), beside the calls a user makes of the library.

Operators
  linear_i8         Y = X W^T with 8-bit integers: each row of X (fp16 or bf16) quantised to int8 with one scale, W given
                    as int8 rows with one scale each (an output channel), products summed exactly in 32-bit integers.
                      s_m = max_k |x_mk| / 127,  q_mk = round-half-even(127 x_mk / max_k |x_mk|)
                      y_mn = s_m t_n sum_k q_mk w_nk
  linear_i8_swiglu  the same with W's rows in groups of 128 gate and 128 up rows: silu(gate) * up, N / 2 columns.
  moe               a mixture-of-experts MLP layer: router logits X R^T, the top_k experts of each token (ties to the
                    lower index) with softmax weights over the chosen, per expert silu(X G^T) * (X U^T) and the down
                    product, summed over the token's experts with their weights.
"""
import math
import os
import sys

import torch

own = False  # True: run() calls the library's operators

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemm-ladder_b200")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _bwgemm():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import bwgemm

    return bwgemm


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of one sequence through a qkv projection: the launch and the stream of the weights
        {"name": "linear_m1", "op": "linear_i8", "M": 1, "N": 10240, "K": 8192, "dtype": "fp16"},
        # a decode batch of 16 through a down projection: a long K, few output columns
        {"name": "linear_m16_down", "op": "linear_i8", "M": 16, "N": 8192, "K": 28672, "dtype": "bf16"},
        # a chunk of prompts of odd length through a small layer whose K is no multiple of a tile
        {"name": "linear_m1001_small", "op": "linear_i8", "M": 1001, "N": 2304, "K": 1104, "dtype": "fp16"},
        # a prefill chunk through a qkv projection
        {"name": "linear_m2048", "op": "linear_i8", "M": 2048, "N": 10240, "K": 8192, "dtype": "bf16"},
        # the square shape of the ladder: the tensor cores' rate
        {"name": "linear_ladder", "op": "linear_i8", "M": 8192, "N": 8192, "K": 8192, "dtype": "fp16"},
        # a decode batch through the gate and up projections of a gated MLP
        {"name": "swiglu_m16", "op": "linear_i8_swiglu", "M": 16, "N": 57344, "K": 8192, "dtype": "bf16"},
        # a prefill chunk of odd length through the same
        {"name": "swiglu_m1999", "op": "linear_i8_swiglu", "M": 1999, "N": 57344, "K": 8192, "dtype": "fp16"},
        # one token through a layer of many small experts: latency
        {"name": "moe_t1", "op": "moe", "T": 1, "E": 64, "k": 8, "D": 2048, "F": 1024, "dtype": "bf16"},
        # a small decode batch over many experts whose width ends inside a tile
        {"name": "moe_t8", "op": "moe", "T": 8, "E": 128, "k": 8, "D": 4096, "F": 1344, "dtype": "fp16"},
        # an odd decode batch over few wide experts: every expert's weights are read
        {"name": "moe_t33_wide", "op": "moe", "T": 33, "E": 8, "k": 2, "D": 4096, "F": 14336, "dtype": "bf16"},
        # the largest batches the layer takes: nearly every expert is active
        {"name": "moe_t64", "op": "moe", "T": 64, "E": 128, "k": 8, "D": 4096, "F": 1280, "dtype": "bf16"},
        {"name": "moe_t128", "op": "moe", "T": 128, "E": 32, "k": 4, "D": 2880, "F": 2880, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["linear_i8", "linear_i8", "linear_i8_swiglu", "moe", "moe", "moe"])
    while op == "moe":
        c = {"op": op, "T": _log_int(rng, 1, 128), "E": rng.choice([4, 8, 16, 24, 32, 60, 64, 96, 128, 160, 256]),
             "k": rng.choice([1, 2, 2, 3, 4, 4, 6, 8, 8]), "D": _log_int(rng, 256, 8192, 64),
             "F": _log_int(rng, 128, 14336, 64), "dtype": dtype}
        if c["k"] <= c["E"] and 6 * c["E"] * c["D"] * c["F"] <= 2.8e9:
            return c
    while True:
        n_step = 256 if op == "linear_i8_swiglu" else 64
        c = {"op": op, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 256, 57344, n_step),
             "K": _log_int(rng, 128, 28672, 16), "dtype": dtype}
        if c["M"] * c["N"] * c["K"] <= 5e11 and c["N"] * c["K"] <= 4.7e8:
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


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "moe":
        T, E, D, F = case["T"], case["E"], case["D"], case["F"]
        state["X"] = torch.randn((T, D), generator=g, device="cuda").to(dtype)
        state["R"] = (torch.randn((E, D), generator=g, device="cuda") * (1.5 / math.sqrt(D))).to(dtype)
        W1 = torch.empty((E, 2 * F, D), dtype=dtype, device="cuda")
        W2 = torch.empty((E, D, F), dtype=dtype, device="cuda")
        for e in range(E):
            W1[e] = torch.randn((2 * F, D), generator=g, device="cuda") * (1.0 / math.sqrt(D))
            W2[e] = torch.randn((D, F), generator=g, device="cuda") * (2.0 / math.sqrt(F))
        state["W1"], state["W2"] = W1, W2
        return state
    M, N, K = case["M"], case["N"], case["K"]
    state["X"] = _activations(M, K, dtype, g)
    w = torch.empty((N, K), dtype=torch.int8, device="cuda")
    scale = torch.empty((N,), dtype=torch.float32, device="cuda")
    for n0 in range(0, N, 4096):  # each output channel quantised with its own scale
        f = torch.randn((min(4096, N - n0), K), generator=g, device="cuda") * (1.0 / math.sqrt(K))
        s = f.abs().amax(dim=1) / 127.0
        w[n0:n0 + f.shape[0]] = torch.round(f / s[:, None]).clamp(-127, 127).to(torch.int8)
        scale[n0:n0 + f.shape[0]] = s
    state["W"], state["w_scale"] = w, scale
    return state


# ------------------------------------------------------------------ one pass
def _linear_plain(x, w, w_scale):
    xf = x.float()
    amax = xf.abs().amax(dim=1, keepdim=True)
    q = torch.round(xf * 127.0 / amax)  # rows of activations are never all zero
    return (q @ w.float().t()) * (amax / 127.0) * w_scale[None, :]


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _moe_plain(x, r, w1, w2, top_k):
    xf = x.float()
    F = w2.shape[2]
    # the choice of experts is a comparison of near values: logits in 64 bits
    logits = x.double() @ r.double().t()
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    ids, chosen = order.indices[:, :top_k], order.values[:, :top_k]
    e = torch.exp(chosen - chosen[:, :1])
    weights = (e / e.sum(dim=1, keepdim=True)).float()
    y = torch.zeros_like(xf)
    for ex in torch.unique(ids).tolist():
        tok, slot = torch.nonzero(ids == ex, as_tuple=True)
        h = xf[tok] @ w1[ex].float().t()
        h = _silu(h[:, :F]) * h[:, F:] * weights[tok, slot][:, None]
        y[tok] += h @ w2[ex].float().t()
    return y


def run(state):
    if own:
        bw = _bwgemm()
        if state["op"] == "moe":
            return bw.moe_mlp(state["X"], state["R"], state["W1"], state["W2"], state["k"])
        return bw.linear_i8(state["X"], state["W"], state["w_scale"], swiglu=state["op"] == "linear_i8_swiglu")
    dtype = state["X"].dtype
    if state["op"] == "moe":
        return _moe_plain(state["X"], state["R"], state["W1"], state["W2"], state["k"]).to(dtype)
    y = _linear_plain(state["X"], state["W"], state["w_scale"])
    if state["op"] == "linear_i8_swiglu":
        M, N = y.shape
        y = y.view(M, N // 256, 2, 128)
        y = (_silu(y[:, :, 0]) * y[:, :, 1]).reshape(M, N // 2)
    return y.to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "moe":
        T, E, k, D, F = (case[n] for n in ("T", "E", "k", "D", "F"))
        active = E * (1.0 - (1.0 - k / E) ** T)  # expected experts that some token chooses
        return {"bytes": 2.0 * (active * 3 * D * F + E * D + 2 * T * D),
                "flops": 2.0 * T * (k * 3 * D * F + E * D)}
    M, N, K = case["M"], case["N"], case["K"]
    out = N // 2 if case["op"] == "linear_i8_swiglu" else N
    return {"bytes": 2.0 * M * K + 1.0 * N * K + 4.0 * N + 2.0 * M * out, "flops": 2.0 * M * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s["X"].double()
    if case["op"] == "moe":
        k, F = case["k"], case["F"]
        scores = torch.einsum("td,ed->te", x, s["R"].double())
        T, E = scores.shape
        y = torch.zeros_like(x)
        left = scores.clone()
        gate = torch.zeros_like(scores)
        index = torch.arange(E, device=x.device)
        for _ in range(k):  # the largest score left, the lowest index among equals
            best = left.amax(dim=1, keepdim=True)
            first = torch.where(left == best, index, E).amin(dim=1, keepdim=True)
            gate.scatter_(1, first, 1.0)
            left.scatter_(1, first, -math.inf)
        p = torch.softmax(torch.where(gate > 0, scores, torch.full_like(scores, -math.inf)), dim=1)
        for e in range(E):
            rows = gate[:, e] > 0
            if not bool(rows.any()):
                continue
            xe = x[rows]
            g = torch.einsum("td,fd->tf", xe, s["W1"][e, :F].double())
            u = torch.einsum("td,fd->tf", xe, s["W1"][e, F:].double())
            h = g * torch.sigmoid(g) * u
            y[rows] += p[rows, e][:, None] * torch.einsum("tf,df->td", h, s["W2"][e].double())
        return y
    N = case["N"]
    peak = x.abs().max(dim=1).values
    steps = torch.round(x / peak[:, None] * 127.0)
    # x / peak * 127 rounds twice: settle the quotients that land next to a half with integers
    twice = 2.0 * (x * 127.0 - steps * peak[:, None])
    steps = steps + (twice > peak[:, None]).double() - (twice < -peak[:, None]).double()
    tie = twice.abs() == peak[:, None]
    steps = torch.where(tie & (steps % 2 != 0), steps + torch.sign(twice), steps)
    out = torch.empty((case["M"], N), dtype=torch.float64, device=x.device)
    for n0 in range(0, N, 8192):
        n1 = min(N, n0 + 8192)
        out[:, n0:n1] = torch.einsum("mk,nk->mn", steps, s["W"][n0:n1].double())
        out[:, n0:n1] *= s["w_scale"][n0:n1].double()
    out *= peak[:, None] / 127.0
    if case["op"] == "linear_i8_swiglu":
        g = out.view(case["M"], N // 256, 256)
        gate_part, up = g[..., :128], g[..., 128:]
        out = (gate_part * torch.sigmoid(gate_part) * up).reshape(case["M"], N // 2)
    return out
