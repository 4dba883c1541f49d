"""The grouped and 8-bit floating-point products on a B200 against their definitions in 64 bits (tests/grouped_ref.py), at the
sizes and values where they can go wrong."""
import pytest

torch = pytest.importorskip("torch")

import bwgemm  # noqa: E402
import grouped_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    bwgemm.clear_status()
    yield
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0, bwgemm.status()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(T, K, dtype, seed, pad=0):
    return torch.randn((T, K + pad), generator=gen(seed), device="cuda").to(dtype)[:, :K]


def weights(E, N, K, dtype, seed, mn=False):
    shape = (E, K, N) if mn else (E, N, K)
    return (torch.randn(shape, generator=gen(seed), device="cuda") / K ** 0.5).to(dtype)


def check(got, y, err):
    ok, worst = ref.close(got, y, err)
    assert ok, f"{worst:.3f} of the bound"


def reference16(X, W, off, N, mn=False, swiglu=False):
    y, err, covered = ref.grouped(X, off, W, N, lambda r, e: ref.product16(X[r], W[e].t() if mn else W[e]))
    return (*ref.glu(y, err, False), covered) if swiglu else (y, err, covered)


COUNTS = [
    [1], [0, 0, 1], [5, 0, 31, 32, 33, 0], [64, 1, 129], [255, 256, 257], [700, 3], [0, 0], [16] * 40 + [0] * 5 + [90],
    [2000, 1500, 7],
]
SIZES = [(64, 64), (256, 512), (1352, 200), (520, 1544)]


@pytest.mark.parametrize("form", ["tn", "nn", "swiglu"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:6])))
def test_grouped(form, dtype, counts):
    for N, K in SIZES:
        if form == "swiglu" and N % 16:
            continue
        T = sum(counts) + 5
        X = rows(T, K, dtype, N + T, pad=16)
        off = ref.offsets_of(counts, 2, "cuda")
        W = weights(len(counts), N, K, dtype, K, form == "nn")
        C = torch.full((T, N // 2 if form == "swiglu" else N), float("nan"), dtype=dtype, device="cuda")
        if form == "nn":
            out = bwgemm.gemm_grouped(X, W, off, C)
        else:
            out = bwgemm.gemm_grouped_tn(X, W, off, C, swiglu=form == "swiglu")
        assert out is C
        y, err, covered = reference16(X, W, off, N, form == "nn", form == "swiglu")
        check(C[covered], y[covered], err[covered])
        assert torch.isnan(C[~covered]).all(), "rows of no expert were written"


@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts", COUNTS + [[9000]], ids=lambda c: "-".join(map(str, c[:6])))
def test_weight_gradient(dtype, out, counts):
    for N, K in SIZES:
        T, E = sum(counts) + 5, len(counts)
        dY, X = rows(T, N, dtype, N + T, pad=8), rows(T, K, dtype, K + T + 1, pad=16)
        off = ref.offsets_of(counts, 2, "cuda")
        for v in (dY, X):  # rows of no expert reach no gradient
            v[:2] = float("nan")
            v[T - 3:] = float("inf")
        dW = torch.full((E, N, K), float("nan"), dtype=out or dtype, device="cuda")
        assert bwgemm.gemm_grouped_dw(dY, X, off, dW, dtype=out) is dW
        check(dW, *ref.weight_gradient(dY, X, off))


def f8_operands(T, E, N, K, dtype, seed):
    X = rows(T, K, dtype, seed)
    W = weights(max(1, E), N, K, dtype, seed + 1)
    if not E:
        W = W[0]
    return X, *bwgemm.quantize_f8(X), *bwgemm.quantize_blocks_f8(W)


def reference8(Q, s, B, t, off, N, swiglu):
    if off is None:
        y, err = ref.product8(Q, s, B, t)
        covered = torch.ones(Q.shape[0], dtype=torch.bool, device="cuda")
    else:
        y, err, covered = ref.grouped(Q, off, B, N, lambda r, e: ref.product8(Q[r], s[r], B[e], t[e]))
    return (*ref.glu(y, err, off is None), covered) if swiglu else (y, err, covered)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("shape", [(1, 256, 128), (1, 10240, 2048), (3, 512, 144), (17, 8192, 4112), (33, 768, 1040),
                                   (130, 1280, 2000), (257, 512, 400), (1001, 2560, 1552), (2100, 512, 8192)])
def test_f8(dtype, swiglu, shape):
    M, N, K = shape
    X, Q, s, B, t = f8_operands(M, 0, N, K, BF16, M + N)
    C = bwgemm.gemm_f8(Q, s, B, t, dtype=dtype, swiglu=swiglu)
    y, err, _ = reference8(Q, s, B, t, None, N, swiglu)
    check(C, y, err)


@pytest.mark.parametrize("N", [8, 72, 136, 264, 392])
def test_f8_columns_that_end_inside_a_tile(N):
    X, Q, s, B, t = f8_operands(37, 0, N, 272, F16, N)
    check(bwgemm.gemm_f8(Q, s, B, t, dtype=F32), *reference8(Q, s, B, t, None, N, False)[:2])


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:6])))
def test_f8_grouped(swiglu, counts):
    for N, K in [(256, 128), (512, 400), (1280, 1040)]:
        T, E = sum(counts) + 7, len(counts)
        X, Q, s, B, t = f8_operands(T, E, N, K, F16, N + T)
        off = ref.offsets_of(counts, 3, "cuda")
        C = torch.full((T, N // 2 if swiglu else N), float("nan"), dtype=BF16, device="cuda")
        bwgemm.gemm_f8(Q, s, B, t, offsets=off, C=C, dtype=BF16, swiglu=swiglu)
        y, err, covered = reference8(Q, s, B, t, off, N, swiglu)
        check(C[covered], y[covered], err[covered])
        assert torch.isnan(C[~covered]).all(), "rows of no expert were written"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", [(1, 128), (1, 16), (5, 144), (31, 4112), (33, 256), (257, 272), (1000, 7184)])
def test_quantizers(dtype, shape):
    M, K = shape
    X = rows(M, K, dtype, M + K, pad=8)
    if M > 3:  # a group of zeros, one of subnormal values, a large one
        X[1, :128] = 0
        X[2, :128] *= 2.0 ** -24 if dtype == F16 else 2.0 ** -126
        X[3, :] *= 2.0 ** 10
    Q, s = bwgemm.quantize_f8(X)
    q, sc = ref.quantize_rows(X)
    assert torch.equal(Q.double(), q) and torch.equal(s.double(), sc)
    W = X.contiguous()
    Q, s = bwgemm.quantize_blocks_f8(W)
    q, sc = ref.quantize_blocks(W)
    assert torch.equal(Q.double(), q) and torch.equal(s.double(), sc)
    W3 = torch.stack([W, W.flip(0)]).contiguous()
    Q3, s3 = bwgemm.quantize_blocks_f8(W3)
    assert torch.equal(Q3[0].view(torch.uint8), Q.view(torch.uint8)) and torch.equal(s3[0], s)
    q1, sc1 = ref.quantize_blocks(W3[1])
    assert torch.equal(Q3[1].double(), q1) and torch.equal(s3[1].double(), sc1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("E", [0, 5])
def test_linear_f8_is_its_parts(dtype, E):
    M, N, K = 77, 512, 1040
    X = rows(M, K, dtype, 1, pad=24)
    W = weights(max(1, E), N, K, dtype, 2)
    B, t = bwgemm.quantize_blocks_f8(W if E else W[0])
    off = ref.offsets_of([10, 0, 60, 1, 6], 0, "cuda") if E else None
    Q, s = bwgemm.quantize_f8(X)
    for swiglu in (False, True):
        a = bwgemm.linear_f8(X, B, t, offsets=off, swiglu=swiglu)
        b = bwgemm.gemm_f8(Q, s, B, t, offsets=off, dtype=dtype, swiglu=swiglu)
        assert torch.equal(a, b)


def test_the_same_bits_every_time():
    """Whole tiles go to whichever pair asks first and split tiles' parts are summed by the last: neither shows."""
    counts = [300, 0, 1, 700, 64, 130, 33]
    off = ref.offsets_of(counts, 0, "cuda")
    T, E, N, K = sum(counts), len(counts), 1352, 1544
    X, W = rows(T, K, F16, 1), weights(E, N, K, F16, 2)
    dY = rows(T, N, F16, 3)
    Q, s = bwgemm.quantize_f8(rows(700, 4112, BF16, 4))
    B, t = bwgemm.quantize_blocks_f8(weights(1, 2560, 4112, BF16, 5)[0])
    calls = [lambda: bwgemm.gemm_grouped_tn(X, W, off), lambda: bwgemm.gemm_grouped_dw(dY, X, off),
             lambda: bwgemm.gemm_f8(Q, s, B, t), lambda: bwgemm.gemm_f8(Q[:9], s[:9], B, t, swiglu=True)]
    for call in calls:
        want = call()
        for _ in range(8):
            assert torch.equal(call(), want)


def test_streams_graphs_and_a_gemm_beside():
    """Calls that overlap on two streams and beside a long product, and graphs replayed at once with new contents."""
    A = torch.randn((8192, 4096), device="cuda").half()
    Bm = torch.randn((4096, 8192), device="cuda").half()
    counts = [20, 0, 5, 300]
    off = ref.offsets_of(counts, 0, "cuda")
    T, N, K = sum(counts), 512, 1040
    X, W = rows(T, K, BF16, 1), weights(4, N, K, BF16, 2)
    B8, t8 = bwgemm.quantize_blocks_f8(weights(1, N, K, BF16, 3)[0])
    fs = [lambda st=None: bwgemm.gemm_grouped_tn(X, W, off, swiglu=True, stream=st),
          lambda st=None: bwgemm.linear_f8(X, B8, t8, stream=st)]
    want = [f() for f in fs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        bwgemm.gemm(A, Bm)
        for i in range(2):
            got[i].append(fs[i](side[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    graphs, out = [], []
    for f in fs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append((f(), f()))
        graphs.append(g)
    for _ in range(5):
        X.copy_(torch.randn_like(X))
        c = torch.randint(0, T, (3,)).sort().values.tolist()
        off.copy_(torch.tensor([0, *c, T], dtype=torch.int32))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            y = fs[i]()
            assert torch.equal(out[i][0], y) and torch.equal(out[i][1], y)


def test_a_kernel_ahead_writes_the_inputs():
    """Offsets, weights and rows written on the stream right before the call."""
    T, N, K = 400, 512, 512
    X0, W0 = rows(T, K, F16, 1), weights(3, N, K, F16, 2)
    o0 = ref.offsets_of([100, 250, 50], 0, "cuda")
    want = bwgemm.gemm_grouped_tn(X0, W0, o0)
    B0, t0 = bwgemm.quantize_blocks_f8(W0[0])
    want8 = bwgemm.linear_f8(X0, B0, t0)
    X, W, off, B, t = (torch.zeros_like(v) for v in (X0, W0, o0, B0, t0))
    for _ in range(10):
        for to, v in ((X, X0), (W, W0), (off, o0), (t, t0)):
            to.zero_()
            to.copy_(v)
        B.view(torch.uint8).zero_()
        B.view(torch.uint8).copy_(B0.view(torch.uint8))
        a = bwgemm.gemm_grouped_tn(X, W, off)
        for to in (W, t):
            to.zero_()
        W.copy_(W0)
        t.copy_(t0)
        b = bwgemm.linear_f8(X, B, t)
        X.zero_()
        assert torch.equal(a, want) and torch.equal(b, want8)


def test_nan_and_infinity_stay_where_they_belong():
    counts = [40, 70, 30]
    off = ref.offsets_of(counts, 0, "cuda")
    T, N, K = sum(counts), 256, 272
    X, W = rows(T, K, F16, 1), weights(3, N, K, F16, 2)
    dY = rows(T, N, F16, 3)
    clean, grad = bwgemm.gemm_grouped_tn(X, W, off), bwgemm.gemm_grouped_dw(dY, X, off)
    Q, s = bwgemm.quantize_f8(X)
    B, t = bwgemm.quantize_blocks_f8(W)
    clean8 = [bwgemm.gemm_f8(Q, s, B, t, offsets=off), bwgemm.gemm_f8(Q[:9], s[:9], B[0], t[0])]
    X2, W2 = X.clone(), W.clone()
    X2[45, 7] = float("nan")
    X2[60, 130] = float("inf")
    W2[2, 5, 3] = float("nan")
    Y = bwgemm.gemm_grouped_tn(X2, W2, off)
    bad = torch.zeros((T, N), dtype=torch.bool, device="cuda")
    bad[45] = bad[60] = True
    bad[110:, 5] = True
    assert torch.isfinite(Y[~bad]).all() and torch.equal(Y[~bad], clean[~bad]) and not torch.isfinite(Y[bad]).any()
    G = bwgemm.gemm_grouped_dw(dY, X2, off)
    assert torch.isnan(G[1, :, 7]).all() and not torch.isfinite(G[1, :, 130]).any()
    keep = torch.ones_like(G, dtype=torch.bool)
    keep[1, :, 7] = keep[1, :, 130] = False
    assert torch.equal(G[keep], grad[keep])
    Q2, s2 = bwgemm.quantize_f8(X2)
    assert torch.isnan(s2[45, 0]) and torch.isnan(s2[60, 1]) and torch.isfinite(s2).sum() == s2.numel() - 2
    Y8 = bwgemm.gemm_f8(Q2, s2, B, t, offsets=off)
    hit = torch.zeros(T, dtype=torch.bool, device="cuda")
    hit[45] = hit[60] = True
    assert torch.isnan(Y8[hit]).all() and torch.equal(Y8[~hit], clean8[0][~hit])
    B2, t2 = bwgemm.quantize_blocks_f8(W2)
    assert torch.isnan(t2[2, 0, 0]) and torch.isfinite(t2).sum() == t2.numel() - 1
    s9 = s[:9].clone(memory_format=torch.preserve_format)
    s9[4, 1] = float("nan")
    Y9 = bwgemm.gemm_f8(Q[:9], s9, B[0], t[0])
    assert torch.isnan(Y9[4]).all() and torch.equal(Y9[[0, 1, 2, 3, 5, 6, 7, 8]], clean8[1][[0, 1, 2, 3, 5, 6, 7, 8]])


BAD = [([-5, 30, 20, 900], [0, 30, 30, 120]), ([40, 40, 1000, 70], [40, 40, 120, 120]), ([2 ** 31 - 1, 0, 5, 6], [120] * 4)]


@pytest.mark.parametrize("bad,taken", BAD)
def test_row_numbers_out_of_order_lead_nowhere(bad, taken):
    T, N, K = 120, 256, 144
    X, W, dY = rows(T, K, F16, 1), weights(3, N, K, F16, 2), rows(T, N, F16, 3)
    off, want = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (bad, taken))
    C = [torch.full((T, N), -7.0, dtype=F16, device="cuda") for _ in range(2)]
    assert torch.equal(bwgemm.gemm_grouped_tn(X, W, off, C[0]), bwgemm.gemm_grouped_tn(X, W, want, C[1]))
    assert torch.equal(bwgemm.gemm_grouped_dw(dY, X, off), bwgemm.gemm_grouped_dw(dY, X, want))
    B, t = bwgemm.quantize_blocks_f8(W)
    assert torch.equal(bwgemm.linear_f8(X, B, t, off, C[0]), bwgemm.linear_f8(X, B, t, want, C[1]))


def test_no_rows():
    X, W = rows(0, 128, F16, 1), weights(3, 64, 128, F16, 2)
    off = ref.offsets_of([0, 0, 0], 0, "cuda")
    assert bwgemm.gemm_grouped_tn(X, W, off).shape == (0, 64)
    assert bwgemm.gemm_grouped(rows(0, 64, F16, 1), W, off).shape == (0, 128)
    dW = torch.full((3, 64, 128), float("nan"), dtype=F32, device="cuda")
    assert not bwgemm.gemm_grouped_dw(rows(0, 64, F16, 1), X, off, dW, dtype=F32).any()
    Q, s = bwgemm.quantize_f8(X)
    B, t = bwgemm.quantize_blocks_f8(W)
    assert Q.shape == (0, 128) and s.shape == (0, 1)
    assert bwgemm.gemm_f8(Q, s, B[0], t[0]).shape == (0, 64) and bwgemm.linear_f8(X, B, t, off).shape == (0, 64)


def test_offsets_past_32_bits():
    """C, X and dW of more than 2^32 bytes and 2^31 elements: the last rows are right."""
    T, N, K = 70000, 32768, 128
    X, W = rows(T, K, F16, 1), weights(2, N, K, F16, 2)
    off = ref.offsets_of([T - 100, 100], 0, "cuda")
    C = bwgemm.gemm_grouped_tn(X, W, off)
    B, t = bwgemm.quantize_blocks_f8(W[0])
    C8 = bwgemm.linear_f8(X, B, t)
    Q, s = bwgemm.quantize_f8(X[-40:])
    for e, r in ((0, slice(0, 40)), (0, slice(T - 140, T - 100)), (1, slice(T - 40, T))):
        check(C[r], *ref.product16(X[r], W[e]))
    check(C8[-40:], *ref.product8(Q, s, B, t))
    del C, C8
    E, N, K = 40, 8192, 8192
    counts = [0] * (E - 1) + [33]
    dY, X = rows(33, N, F16, 3), rows(33, K, F16, 4)
    dW = bwgemm.gemm_grouped_dw(dY, X, ref.offsets_of(counts, 0, "cuda"))
    y, err = ref.weight_gradient(dY, X, ref.offsets_of([33], 0, "cuda"))
    check(dW[-1:], y, err)
    assert not dW[:-1].any()


def test_refused_tensors():
    X, W = rows(20, 128, F16, 1), weights(3, 256, 128, F16, 2)
    off = ref.offsets_of([5, 5, 10], 0, "cuda")
    Q, s = bwgemm.quantize_f8(X)
    B, t = bwgemm.quantize_blocks_f8(W)
    g, d, f, q = bwgemm.gemm_grouped_tn, bwgemm.gemm_grouped_dw, bwgemm.gemm_f8, bwgemm.linear_f8
    new = lambda *a, **k: torch.empty(*a, device="cuda", **k)
    for call in (lambda: g(X.float(), W, off), lambda: g(X, W.bfloat16(), off), lambda: g(X, W.transpose(1, 2), off),
                 lambda: g(X, W[0], off), lambda: g(X[:, :64], W, off), lambda: g(X, W, off.long()), lambda: g(X, W, off[:3]),
                 lambda: g(X, W, off.cpu()), lambda: g(X.t(), W, off), lambda: g(X, W, off, new((20, 128), dtype=F16)),
                 lambda: g(X, W, off, new((20, 256), dtype=F32)), lambda: bwgemm.gemm_grouped(X, W, off),
                 lambda: d(X, X[:10], off), lambda: d(X, X.bfloat16(), off), lambda: d(X, X, off.float()), lambda: d(X, X, off[:1]),
                 lambda: d(X, X, off, dtype=torch.float64), lambda: d(X, X, off, new((3, 128, 64), dtype=F16)),
                 lambda: d(X, X, off, new((3, 128, 128), dtype=F16), dtype=F32),
                 lambda: f(X, s, B[0], t[0]), lambda: f(Q, s.contiguous(), B[0], t[0]) if s.shape[1] > 1 else g(X, W, off.long()),
                 lambda: f(Q, s[:10], B[0], t[0]), lambda: f(Q, s.half(), B[0], t[0]), lambda: f(Q, s, B, t),
                 lambda: f(Q, s, B[0], t[0], off), lambda: f(Q, s, B[0], t), lambda: f(Q, s, B[0][:, :64], t[0]),
                 lambda: f(Q, s, B[0], t[0].half()), lambda: f(Q, s, B[0], t[0], dtype=torch.int8),
                 lambda: f(Q, s, B[0], t[0], C=new((20, 256), dtype=BF16)), lambda: q(X.float(), B[0], t[0]),
                 lambda: q(X, B[0].view(torch.int8), t[0]), lambda: q(X, B, t, off[:2]), lambda: bwgemm.quantize_f8(X.float()),
                 lambda: bwgemm.quantize_f8(X, Q=new((20, 64), dtype=torch.float8_e4m3fn)),
                 lambda: bwgemm.quantize_f8(X, scale=new((20, 2))), lambda: bwgemm.quantize_blocks_f8(W.transpose(1, 2)),
                 lambda: bwgemm.quantize_blocks_f8(W, scale=new((3, 2, 2)))):
        with pytest.raises(ValueError):
            call()
    X3, W3 = rows(20, 100, F16, 1), weights(3, 256, 100, F16, 2)
    for call in (lambda: g(X, weights(3, 100, 128, F16, 1), off), lambda: g(rows(20, 104, F16, 1), weights(3, 12, 104, F16, 1), off),
                 lambda: g(X, weights(3, 264, 128, F16, 1), off, swiglu=True), lambda: g(X, W, off, new(20 * 256 + 4, dtype=F16)[4:].view(20, 256)),
                 lambda: q(rows(20, 72, F16, 1), B[0][:, :72].contiguous(), t[0]), lambda: q(X, B[0][:128], t[0][:1], swiglu=True),
                 lambda: bwgemm.quantize_f8(rows(20, 72, F16, 1)), lambda: g(X, W.repeat(400, 1, 1), ref.offsets_of([0] * 1200, 0, "cuda"))):
        with pytest.raises(bwgemm.BwError):
            call()
    with pytest.raises(ValueError):  # rows that do not start on 16 bytes
        g(X3, W3, off)


def expert_layer(X, ids, p, W1, W2, products):
    """A mixture-of-experts layer's forward and backward over given routing, as a training step makes it: rows gathered by
    expert, gate and up, the activation, down, the weighted sum back; then the gradients for dL/dY = Y."""
    up, down, dx_up, dx_down, dw = products
    T, k = ids.shape
    E, F = W1.shape[0], W2.shape[2]
    order = torch.argsort(ids.flatten(), stable=True)
    tok, w = order // k, p.flatten()[order][:, None]
    off = torch.zeros(E + 1, dtype=torch.int32, device=X.device)
    off[1:] = torch.cumsum(torch.bincount(ids.flatten(), minlength=E), 0)
    Xe = X[tok].contiguous()
    gu = up(Xe, W1, off)
    g, u = gu[:, :F].double(), gu[:, F:].double()
    sg = torch.sigmoid(g)
    a = (g * sg * u).to(X.dtype)
    h = down(a, W2, off)
    Y = torch.zeros(X.shape, dtype=torch.float64, device=X.device).index_add_(0, tok, h.double() * w)
    dh = (Y[tok] * w).to(X.dtype)
    da = dx_down(dh, W2, off).double()
    dgu = torch.cat([da * u * (sg + g * sg * (1 - sg)), da * g * sg], 1).to(X.dtype)
    dX = torch.zeros_like(Y).index_add_(0, tok, dx_up(dgu, W1, off).double())
    return Y, dX, dw(dgu, Xe, off), dw(dh, a, off)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_an_expert_layer_with_its_gradients(dtype):
    """The products together as a layer uses them against the same chain in 64 bits, and that chain against differences."""
    T, E, k, D, F = 200, 8, 2, 256, 320
    X, W1 = rows(T, D, dtype, 1), weights(E, 2 * F, D, dtype, 2)
    W2 = weights(E, D, F, dtype, 3)
    logits = torch.randn((T, E), generator=gen(4), device="cuda")
    logits[:, 5] = -100  # an expert that nobody chooses
    top = torch.topk(logits, k, dim=1)
    ids, p = top.indices, torch.softmax(top.values.double(), 1)

    def each(f):
        def run(a, b, off):
            o = off.tolist()
            return torch.cat([f(a[o[e]:o[e + 1]].double(), b[e].double()) for e in range(E)])
        return run

    def grad(a, b, off):
        o = off.tolist()
        return torch.stack([a[o[e]:o[e + 1]].double().t() @ b[o[e]:o[e + 1]].double() for e in range(E)])

    exact = (each(lambda a, b: a @ b.t()), each(lambda a, b: a @ b.t()), each(lambda a, b: a @ b), each(lambda a, b: a @ b), grad)
    own = (bwgemm.gemm_grouped_tn, bwgemm.gemm_grouped_tn, bwgemm.gemm_grouped, bwgemm.gemm_grouped,
           lambda a, b, off: bwgemm.gemm_grouped_dw(a, b, off, dtype=F32))
    got, want = expert_layer(X, ids, p, W1, W2, own), expert_layer(X, ids, p, W1, W2, exact)
    # each of the chain's at most 6 roundings to `dtype` (gu, a, h, dh, da, dgu) is off by half a step of its value; as
    # independent errors of uniform size they make sqrt(6 / 3) half steps of the norm, the sums' own errors are far below
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 2.0 * ref.HALF_STEP[dtype] * b.norm()
    # the formulas against differences in 64 bits: L = |Y|^2 / 2
    d = lambda v: v.double()
    _, dX, dW1, dW2 = expert_layer(d(X), ids, p, d(W1), d(W2), exact)
    loss = lambda *a: 0.5 * expert_layer(a[0], ids, p, a[1], a[2], exact)[0].square().sum()
    args = [d(X), d(W1), d(W2)]
    for i, gr in enumerate((dX, dW1, dW2)):
        v = torch.randn(args[i].shape, generator=gen(9 + i), device="cuda", dtype=torch.float64)
        step = 1e-5
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + step * v, args[i] - step * v
        diff = (loss(*hi) - loss(*lo)) / (2 * step)
        assert abs(diff - (gr * v).sum()) <= 1e-6 * abs(diff) + 1e-6


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 32, 300])
def test_mlp_block_in_8_bit_floating_point(dtype, M):
    """The tensor-parallel block's 8-bit form over these operators: each step against its definition, in a graph, and the block
    that it stands for."""
    import tp_mlp

    hidden, f = 512, 1280
    X = rows(M, hidden, dtype, 1)
    W1 = (torch.randn((hidden, 2 * f), generator=gen(2), device="cuda") / hidden ** 0.5).to(dtype)
    W2 = (torch.randn((f, hidden), generator=gen(3), device="cuda") / f ** 0.5).to(dtype)
    w1, w2 = tp_mlp.quantize_shards(W1, W2, 0, 1, bwgemm.quantize_blocks_f8)
    blk = tp_mlp.TPMLPI8(w1, w2, 0, 1, bwgemm.linear_f8)
    blk.forward(X)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Y = blk.forward(X)
    X.copy_(X.roll(1, 0))
    g.replay()
    A = bwgemm.linear_f8(X, *w1, swiglu=True)
    for inp, w, out, act in ((X, w1, A, True), (A, w2, Y, False)):
        q, s = ref.quantize_rows(inp)
        y, err, _ = reference8(q, s, w[0], w[1], None, w[0].shape[0], act)
        check(out, y, err)
    # over ranks, down runs as quantiser and fp32 product: the same values before the last rounding
    P = bwgemm.gemm_f8(*bwgemm.quantize_f8(A), *w2, dtype=F32)
    assert torch.equal(P.to(dtype), Y)
    H = X.double() @ W1.double()
    want = (torch.nn.functional.silu(H[:, :f]) * H[:, f:]) @ W2.double()
    # e4m3's rounding is at most 2^-4 of a value, as a uniform error 2^-4 / sqrt(3) = 3.6 %, about 2.6 % over the values of a
    # step; six quantised operands (X twice, gate, up, A, W2), the activation's slope at most 1.1: below 9 %
    assert (Y.double() - want).norm() <= 0.09 * want.norm()


@pytest.mark.parametrize("N", [8, 72, 136, 264, 392])
def test_f8_columns_that_end_inside_a_tile_of_many_tokens(N):
    for M, K in ((300, 272), (129, 4112)):
        X, Q, s, B, t = f8_operands(M, 0, N, K, F16, N)
        for dtype in (F16, F32):
            check(bwgemm.gemm_f8(Q, s, B, t, dtype=dtype), *reference8(Q, s, B, t, None, N, False)[:2])


@pytest.mark.parametrize("most", [4, 120])
def test_as_many_experts_as_there_may_be(most):
    E, N, K = bwgemm.GROUP_MAX_EXPERTS, 72, 144
    counts = torch.randint(0, most, (E,), generator=torch.Generator().manual_seed(most)).tolist()
    T = sum(counts) + 5
    off = ref.offsets_of(counts, 2, "cuda")
    X, dY = rows(T, K, BF16, 1), rows(T, N, BF16, 2)
    for mn in (False, True):
        W = weights(E, N, K, BF16, 3, mn)
        C = (bwgemm.gemm_grouped if mn else bwgemm.gemm_grouped_tn)(X, W, off)
        y, err, covered = reference16(X, W, off, N, mn)
        check(C[covered], y[covered], err[covered])
    check(bwgemm.gemm_grouped_dw(dY, X, off), *ref.weight_gradient(dY, X, off))
    Q, s = bwgemm.quantize_f8(X)
    B, t = bwgemm.quantize_blocks_f8(weights(E, N, K, BF16, 4))
    C = bwgemm.gemm_f8(Q, s, B, t, offsets=off, dtype=BF16)
    y, err, covered = reference8(Q, s, B, t, off, N, False)
    check(C[covered], y[covered], err[covered])


@pytest.mark.parametrize("N,K", [(8, 8), (16, 8), (8, 16), (24, 40)])
def test_the_smallest_widths(N, K):
    counts = [3, 0, 1, 70]
    T, E = sum(counts) + 4, len(counts)
    off = ref.offsets_of(counts, 2, "cuda")
    X, dY = rows(T, K, F16, 1), rows(T, N, F16, 2)
    for mn in (False, True):
        W = weights(E, N, K, F16, 3, mn)
        C = (bwgemm.gemm_grouped if mn else bwgemm.gemm_grouped_tn)(X, W, off)
        y, err, covered = reference16(X, W, off, N, mn)
        check(C[covered], y[covered], err[covered])
    check(bwgemm.gemm_grouped_dw(dY, X, off, dtype=F32), *ref.weight_gradient(dY, X, off))
    for M in (1, 200):
        X, Q, s, B, t = f8_operands(M, 0, N, 16 * K, F16, N)
        check(bwgemm.gemm_f8(Q, s, B, t), *reference8(Q, s, B, t, None, N, False)[:2])
        X, Q, s, B, t = f8_operands(M, 0, N, 16, F16, N)
        check(bwgemm.gemm_f8(Q, s, B, t), *reference8(Q, s, B, t, None, N, False)[:2])
