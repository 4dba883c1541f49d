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
