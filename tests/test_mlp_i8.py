"""The gated MLP block in 8 bits (tp_mlp.TPMLPI8): over two CPU ranks (gloo, plain products standing in for the kernels) it
equals the block computed whole with the same shards' scales; on a B200 the kernels' block equals the same chain of
operations in 64 bits, step by step, and the fp16 block it stands for within the quantisation's own error."""
import os
import socket

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import torch.distributed as dist  # noqa: E402
import torch.multiprocessing as mp  # noqa: E402

import i8_ref  # noqa: E402
import tp_mlp  # noqa: E402


def quantize_rows(X):
    q, s = i8_ref.quantize_exact(X.double().numpy())
    return torch.from_numpy(q).to(torch.int8), torch.from_numpy(s).float()


def gemm_f32(q, qs, B, bs):
    return ((q.double() @ B.double().t()) * qs.double()[:, None] * bs.double()).float()


def linear(group):
    def f(X, B, bs, swiglu=False):
        y = gemm_f32(*quantize_rows(X), B, bs).double()
        if swiglu:
            y = y.view(y.shape[0], -1, 2, group)
            y = (torch.nn.functional.silu(y[:, :, 0]) * y[:, :, 1]).reshape(y.shape[0], -1)
        return y.to(X.dtype)
    return f


def weights(hidden, f, dtype, device="cpu"):
    g = torch.Generator().manual_seed(7)
    X = torch.randn((32, hidden), generator=g).to(dtype)
    W1 = (torch.randn((hidden, 2 * f), generator=g) / hidden ** 0.5).to(dtype)
    W2 = (torch.randn((f, hidden), generator=g) / f ** 0.5).to(dtype)
    return X.to(device), W1.to(device), W2.to(device)


def reduce_scatter_gloo(out, inp):
    full = inp.clone()
    dist.all_reduce(full)
    rows = out.shape[0]
    out.copy_(full[dist.get_rank() * rows:(dist.get_rank() + 1) * rows])


def worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        X, W1, W2 = weights(64, 96, torch.float16)
        w1, w2 = tp_mlp.quantize_shards(W1, W2, rank, world, quantize_rows, group=16)
        blk = tp_mlp.TPMLPI8(w1, w2, rank, world, linear(16), quantize_rows, gemm_f32, reduce_scatter_gloo)
        Y = blk.forward(X)
        # the same block whole: every rank's shard on one process, summed
        total = torch.zeros((32, 64), dtype=torch.float64)
        for r in range(world):
            a1, a2 = tp_mlp.quantize_shards(W1, W2, r, world, quantize_rows, group=16)
            total += gemm_f32(*quantize_rows(linear(16)(X, *a1, swiglu=True)), *a2).double()
        want = total[rank * 16:(rank + 1) * 16]
        # fp32 partials and their sum (world roundings of 2^-24 of the partials, each below a few units), fp16 result
        q.put((rank, ((Y.double() - want).abs() - want.abs() * 2.0 ** -11).max().item()))
    finally:
        dist.destroy_process_group()


def test_two_cpu_ranks_equal_the_whole_block():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    for _ in range(2):
        rank, over = q.get(timeout=5)
        assert over <= 2.0 ** -20, (rank, over)


def test_shards_must_agree():
    X, W1, W2 = weights(64, 96, torch.float16)
    w1, w2 = tp_mlp.quantize_shards(W1, W2, 0, 2, quantize_rows, group=16)
    with pytest.raises(ValueError):
        tp_mlp.TPMLPI8(w1, tp_mlp.quantize_shards(W1, W2, 0, 1, quantize_rows, group=16)[1], 0, 2, None)
    with pytest.raises(ValueError):
        tp_mlp.TPMLPI8(w1, w2, 0, 2, linear(16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("graph", [False, True])
def test_block_on_the_gpu(dtype, graph):
    import bwgemm

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hidden, f = 512, 1280
    X, W1, W2 = weights(hidden, f, dtype, "cuda")
    w1, w2 = tp_mlp.quantize_shards(W1, W2, 0, 1, bwgemm.quantize_rows)
    blk = tp_mlp.TPMLPI8(w1, w2, 0, 1, bwgemm.linear_i8)
    Y = blk.forward(X)
    if graph:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            Y = blk.forward(X)
        X.copy_(X.roll(1, 0))
        g.replay()
    torch.cuda.synchronize()
    kind = {torch.float16: "fp16", torch.bfloat16: "bf16"}[dtype]
    # step by step: each step's own inputs, the definition in 64 bits
    A = bwgemm.linear_i8(X, *w1, swiglu=True)
    for inp, w, out, act in ((X, w1, A, True), (A, w2, Y, False)):
        q, qs = i8_ref.quantize_exact(inp.double().cpu().numpy())
        y = i8_ref.product(q, qs, w[0].cpu().numpy(), w[1].cpu().numpy())
        assert len(i8_ref.outside(out.double().cpu().numpy(), y, kind, act)) == 0
    # over ranks, down runs as quantiser and fp32 product: the same values before C's rounding
    P = bwgemm.gemm_i8(*bwgemm.quantize_rows(A), *w2, dtype=torch.float32)
    assert torch.equal(P.to(dtype), Y)
    # the block it stands for: every quantisation is off by at most half a step (1 / 254 of a row's maximum) per operand
    H = X.double() @ W1.double()
    ref = (torch.nn.functional.silu(H[:, :f]) * H[:, f:]) @ W2.double()
    rel = ((Y.double() - ref).norm() / ref.norm()).item()
    # relative noise of a row of normal values with maximum about 3.5 to 4.5 sigma: 4.5 / 254 / sqrt(3) = 1.0 % per
    # operand; six quantised operands (X twice, gate, up, A, W2), the activation's slope at most 1.1: below 3 %
    assert rel < 0.03, rel
