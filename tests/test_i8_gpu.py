"""The 8-bit integer operators on a B200, through the public entry points, against the definition in 64 bits
(tests/i8_ref.py derives how far a result may be from it): every plan form, ragged tokens, K that ends inside a stage,
strided rows, rows of zeros, infinities and NaN, half-way quotients; streams, CUDA graphs that overlap, the largest
magnitudes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bwgemm  # noqa: E402
import i8_ref  # noqa: E402

pytestmark = pytest.mark.gpu

KIND = {torch.float16: "fp16", torch.bfloat16: "bf16", torch.float32: "fp32"}


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    bwgemm.clear_status()
    yield
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def weight(N, K, seed):
    g = gen(seed)
    B = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand((N,), generator=g, device="cuda") * 2e-3 + 1e-4
    return B, s


def product64(q, qs, B, bs):
    """The exact scaled products (the sums are below 2^53)."""
    return (q.double() @ B.double().t()) * qs.double()[:, None] * bs.double()


def check(C, y64, activation=False):
    bad = i8_ref.outside(C.double().cpu().numpy(), y64.cpu().numpy(), KIND[C.dtype], activation)
    assert len(bad) == 0, f"{len(bad)} elements outside, first {bad[:3].tolist()}"


# ------------------------------------------------------------------ the quantiser
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,ld", [(1, 16, 16), (7, 48, 64), (9, 512, 512), (3, 1104, 1112), (17, 2048, 2048),
                                          (2, 2064, 2064), (5, 8192, 8200), (1, 28672, 28672), (2, 32784, 32784),
                                          (1, 100000, 100000), (1000, 320, 320)])
def test_quantize_rows_is_the_exact_rounding(rows, cols, ld, dtype):
    g = gen(rows * 131 + cols)
    full = torch.randn((rows, ld), generator=g, device="cuda") * 3
    full[0, :8] = torch.tensor([0.0, -0.0, 1.0, -1.0, 0.5, 127.0, -127.0, 63.5])  # half-way quotients of 127
    X = full.to(dtype)[:, :cols]
    before = X.clone()
    Q, s = bwgemm.quantize_rows(X)
    q, qs = i8_ref.quantize_exact(X.double().cpu().numpy())
    assert np.array_equal(Q.cpu().numpy(), q)
    assert np.all(np.abs(s.double().cpu().numpy() - qs) <= qs * 2.0 ** -24)
    assert torch.equal(X, before)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_every_value_against_many_maxima(dtype):
    """Every finite value of the type up to the row's maximum, for maxima whose significand makes half-way quotients
    (127 divides it), subnormal, the smallest, the largest."""
    every = torch.arange(0, 32768, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    every = every[torch.isfinite(every.float())]
    top = torch.finfo(dtype)
    maxima = [1.0, 127.0, 254.0, 254.0 * 2 ** -10, 508.0 * 2 ** 3, 1.9921875, 1016.0, top.max, top.tiny, top.tiny / 4,
              float(every[1]), 2.0 ** -20, 3.0]
    for a in maxima:
        a = torch.tensor(a, dtype=dtype, device="cuda")
        row = every[every <= a]
        row = torch.cat([row, -row, a[None], torch.zeros((-(2 * len(row) + 1)) % 16, dtype=dtype, device="cuda")])[None]
        Q, s = bwgemm.quantize_rows(row.contiguous())
        q, _ = i8_ref.quantize_exact(row.double().cpu().numpy())
        assert np.array_equal(Q.cpu().numpy(), q), float(a)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 4096])
def test_quantize_zero_infinite_and_nan_rows(dtype, cols):
    X = torch.randn((6, cols), generator=gen(1), device="cuda").to(dtype)
    X[1] = 0
    X[2, 5] = float("inf")
    X[3, cols - 1] = float("-inf")
    X[4, 7] = float("nan")
    Q, s = bwgemm.quantize_rows(X)
    assert s[1] == 0 and torch.isnan(s[2:5]).all() and torch.isfinite(s[[0, 5]]).all()
    assert (Q[1:5] == 0).all()
    B, bs = weight(64, cols, 2)
    C = bwgemm.linear_i8(X, B, bs)
    assert (C[1] == 0).all() and torch.isnan(C[2:5]).all() and torch.isfinite(C[[0, 5]]).all()


def test_quantize_into_given_tensors():
    X = torch.randn((5, 64), generator=gen(3), device="cuda").half()
    Q, s = torch.empty((5, 64), dtype=torch.int8, device="cuda"), torch.empty((5,), device="cuda")
    Q2, s2 = bwgemm.quantize_rows(X, Q, s)
    assert Q2 is Q and s2 is s and torch.equal(Q, bwgemm.quantize_rows(X)[0])
    with pytest.raises(ValueError):
        bwgemm.quantize_rows(X, Q[:, :32], s)
    with pytest.raises(ValueError):
        bwgemm.quantize_rows(X.t())
    with pytest.raises(ValueError):
        bwgemm.quantize_rows(X[:, 1:49])  # off 16 bytes
    with pytest.raises(bwgemm.BwError):
        bwgemm.quantize_rows(X[:, :40])


# ------------------------------------------------------------------ the products
SHAPES = [(1, 64, 16), (1, 8192, 8192), (3, 256, 2048), (8, 10240, 1024), (16, 57344, 256), (16, 8192, 28672),
          (33, 1088, 576), (64, 38080, 128), (100, 10240, 1040), (128, 512, 4096), (129, 256, 128), (200, 512, 1024),
          (272, 5376, 128), (512, 8192, 1024), (1001, 2304, 1104), (2049, 4864, 144), (4599, 5632, 208)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gemm_i8(shape, dtype):
    M, N, K = shape
    A, a_s = weight(M, K, 11)
    B, b_s = weight(N, K, 12)
    a_s *= 10
    C = torch.full((M, N), float("nan"), dtype=dtype, device="cuda")
    bwgemm.gemm_i8(A, a_s, B, b_s, C, dtype=dtype)
    check(C, product64(A, a_s, B, b_s))
    again = bwgemm.gemm_i8(A, a_s, B, b_s, dtype=dtype)
    assert torch.equal(C, again), "calls differ"


def test_gemm_i8_sums_are_exact_at_the_largest_magnitudes():
    K = 131056
    A = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    B = torch.full((64, K), -128, dtype=torch.int8, device="cuda")
    B[1] = 127
    one = torch.ones((64,), device="cuda")
    C = bwgemm.gemm_i8(A, one[:2].contiguous(), B, one, dtype=torch.float32)
    assert (C[:, 0].double() == float(np.float32(128 * 128 * K))).all()
    assert (C[:, 1].double() == float(np.float32(-128 * 127 * K))).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 256, 64), (16, 57344, 272), (7, 4096, 1024), (100, 1280, 144), (128, 512, 4096),
                                   (129, 256, 128), (1001, 2304, 1104), (300, 57344, 256)])
def test_gemm_i8_swiglu(M, N, K, dtype):
    A, a_s = weight(M, K, 21)
    B, b_s = weight(N, K, 22)
    a_s *= 4.0 / np.sqrt(K)
    C = torch.full((M, N // 2), float("nan"), dtype=dtype, device="cuda")
    bwgemm.gemm_i8_swiglu(A, a_s, B, b_s, C, dtype=dtype)
    check(C, product64(A, a_s, B, b_s), activation=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,N,K,pad", [(1, 10240, 8192, 0), (5, 512, 2064, 8), (16, 8192, 28672, 0), (77, 57344, 512, 16),
                                       (1001, 2304, 1104, 8), (2048, 2560, 8192, 0)])
def test_linear_i8(M, N, K, pad, swiglu, dtype):
    X = torch.randn((M, K + pad), generator=gen(M + K), device="cuda").to(dtype)[:, :K]
    B, b_s = weight(N, K, 31)
    b_s *= 4.0 / np.sqrt(K)
    C = bwgemm.linear_i8(X, B, b_s, swiglu=swiglu)
    assert C.dtype == dtype
    q, qs = i8_ref.quantize_exact(X.double().cpu().numpy())
    q, qs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    check(C, product64(q, qs, B, b_s), activation=swiglu)
    assert torch.equal(C, bwgemm.linear_i8(X, B, b_s, swiglu=swiglu)), "calls differ"


def test_no_tokens():
    B, b_s = weight(256, 64, 5)
    X = torch.empty((0, 64), dtype=torch.float16, device="cuda")
    assert bwgemm.linear_i8(X, B, b_s).shape == (0, 256) and bwgemm.linear_i8(X, B, b_s, swiglu=True).shape == (0, 128)
    Q, s = bwgemm.quantize_rows(X)
    assert bwgemm.gemm_i8(Q, s, B, b_s).shape == (0, 256)


def test_rows_past_m_are_left_alone():
    M, N, K = 37, 512, 256
    A, a_s = weight(64, K, 6)
    B, b_s = weight(N, K, 7)
    C = torch.full((64, N), 7.0, dtype=torch.float16, device="cuda")
    bwgemm.gemm_i8(A[:M], a_s[:M], B, b_s, C[:M])
    assert (C[M:] == 7.0).all() and torch.equal(C[:M], bwgemm.gemm_i8(A, a_s, B, b_s)[:M])


# ------------------------------------------------------------------ streams, graphs, overlap
SPLIT = (16, 57344, 1024)  # stream-K: partials and counters in the workspace


def test_another_stream_and_two_at_once():
    M, N, K = SPLIT
    X = [torch.randn((M, K), generator=gen(i), device="cuda").half() for i in range(2)]
    B, b_s = weight(N, K, 8)
    want = [bwgemm.linear_i8(x, B, b_s) for x in X]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):  # both streams hold calls at once, each with its own workspace
        for i in range(2):
            got[i].append(bwgemm.linear_i8(X[i], B, b_s, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(c, want[i]) for c in got[i])


def test_two_captured_graphs_replayed_at_once():
    M, N, K = SPLIT
    X = [torch.randn((M, K), generator=gen(i), device="cuda").bfloat16() for i in range(2)]
    B, b_s = weight(N, K, 9)
    graphs, out = [], []
    bwgemm.linear_i8(X[0], B, b_s)
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(bwgemm.linear_i8(X[i], B, b_s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                X[i].copy_(torch.randn((M, K), generator=gen(100 + rep * 2 + i), device="cuda"))  # new contents
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(out[i], bwgemm.linear_i8(X[i], B, b_s))


def test_workspace_too_small_is_refused():
    import ctypes

    M, N, K = SPLIT
    A, a_s = weight(M, K, 1)
    B, b_s = weight(N, K, 2)
    C = torch.empty((M, N), dtype=torch.float16, device="cuda")
    n = ctypes.c_size_t()
    L = bwgemm.lib()
    assert L.bw_gemm_i8_work_bytes(M, N, K, 0, 0, 0, ctypes.byref(n)) == 0 and n.value > 0
    rc = L.bw_gemm_i8(A.data_ptr(), a_s.data_ptr(), B.data_ptr(), b_s.data_ptr(), C.data_ptr(), M, N, K, 0,
                      C.data_ptr(), n.value - 1, None)
    assert rc == bwgemm.BW_ERR_SCRATCH


def test_refused_tensors():
    B, b_s = weight(256, 64, 5)
    X = torch.randn((4, 64), device="cuda").half()
    for call in (lambda: bwgemm.linear_i8(X.float(), B, b_s), lambda: bwgemm.linear_i8(X, B.t(), b_s),
                 lambda: bwgemm.linear_i8(X, B, b_s[:128]), lambda: bwgemm.linear_i8(X, B, b_s.double()),
                 lambda: bwgemm.linear_i8(X[:, ::2], B, b_s), lambda: bwgemm.linear_i8(X, B[:, :32].contiguous(), b_s),
                 lambda: bwgemm.linear_i8(X.expand(4, 64)[:1].expand(4, 64), B, b_s),
                 lambda: bwgemm.linear_i8(X, B, b_s, C=torch.empty((4, 128), dtype=torch.float16, device="cuda")),
                 lambda: bwgemm.linear_i8(X, B, b_s, C=torch.empty((4, 256), device="cuda"))):
        with pytest.raises(ValueError):
            call()
