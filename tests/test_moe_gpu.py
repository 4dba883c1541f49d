"""The mixture-of-experts layer on a B200, through the public entry point, against the definition in 64 bits
(tests/moe_ref.py derives how far a result may be from it): one token to 128, one expert to 512, ragged widths, ties,
all tokens on one expert; strided rows, streams, overlapping calls and graphs, a stall's status."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import bwgemm  # noqa: E402
import moe_ref  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    bwgemm.clear_status()
    yield
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0


def inputs(T, E, D, F, dtype, seed=0, pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    X = randn(T, D + pad).to(dtype)[:, :D]
    R = (randn(E, D) * (1.5 / D ** 0.5)).to(dtype)
    W1 = (randn(E, 2 * F, D) / D ** 0.5).to(dtype)
    W2 = (randn(E, D, F) * (2 / F ** 0.5)).to(dtype)
    return X, R, W1, W2


def check(Y, X, R, W1, W2, k, renormalize=True):
    ids, weights, err = moe_ref.route(X, R, k, renormalize)
    y, tol = moe_ref.layer(X, ids, weights, err, W1, W2)
    bad = ((Y.double() - y).abs() > tol) | ~torch.isfinite(Y.double())
    assert not bad.any(), f"{int(bad.sum())} elements outside, first {bad.nonzero()[:3].tolist()}"
    return ids, weights, err


CASES = [  # T, E, k, D, F
    (1, 1, 1, 64, 64), (1, 8, 2, 256, 128), (1, 64, 8, 2048, 1024), (2, 60, 4, 512, 192), (3, 4, 4, 128, 64),
    (5, 16, 3, 4096, 128), (8, 128, 8, 1024, 448), (16, 8, 1, 320, 1344), (17, 8, 2, 2112, 320), (33, 8, 2, 1024, 1792),
    (64, 128, 8, 512, 256), (77, 512, 6, 192, 64), (100, 32, 32, 256, 128), (128, 32, 4, 1472, 704), (128, 2, 2, 64, 4096)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_layer(case, dtype):
    T, E, k, D, F = case
    X, R, W1, W2 = inputs(T, E, D, F, dtype, seed=T + E + D, pad=8 if T % 2 else 0)
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    weights = torch.full((T, k), float("nan"), device="cuda")
    buf = torch.full((T + 4, D), float("nan"), dtype=dtype, device="cuda")
    Y = bwgemm.moe_mlp(X, R, W1, W2, k, Y=buf[:T], ids=ids, weights=weights)
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0, bwgemm.status()
    want, p, err = check(Y, X, R, W1, W2, k)
    assert torch.equal(ids.long(), want)
    assert ((weights.double() - p).abs() <= p * err).all()
    assert torch.isnan(buf[T:]).all()
    assert torch.equal(Y, bwgemm.moe_mlp(X, R, W1, W2, k)), "calls differ"


@pytest.mark.parametrize("renormalize", [True, False])
def test_weights_over_the_chosen_or_over_all(renormalize):
    X, R, W1, W2 = inputs(6, 40, 256, 128, torch.bfloat16, 3)
    weights = torch.empty((6, 4), device="cuda")
    Y = bwgemm.moe_mlp(X, R, W1, W2, 4, renormalize=renormalize, weights=weights)
    check(Y, X, R, W1, W2, 4, renormalize)
    assert (weights.sum(1) - 1).abs().max() < 1e-5 if renormalize else (weights.sum(1) < 1).all()


def test_equal_logits_go_to_the_lower_index():
    X, R, W1, W2 = inputs(9, 100, 256, 64, torch.float16, 4)
    R[:] = R[torch.arange(100, device="cuda") % 7]  # every logit about 14 times
    X[4] = 0  # every logit equal
    ids = torch.empty((9, 5), dtype=torch.int32, device="cuda")
    Y = bwgemm.moe_mlp(X, R, W1, W2, 5, ids=ids)
    want, _, _ = check(Y, X, R, W1, W2, 5)
    assert torch.equal(ids.long(), want)
    assert ids[4].tolist() == [0, 1, 2, 3, 4] and (Y[4] == 0).all()


def test_every_token_on_one_expert():
    X, R, W1, W2 = inputs(50, 16, 512, 320, torch.bfloat16, 5)
    X = X.abs() + 0.1
    R[:] = 0
    R[11] = 1
    ids = torch.empty((50, 1), dtype=torch.int32, device="cuda")
    Y = bwgemm.moe_mlp(X, R, W1, W2, 1, ids=ids)
    check(Y, X, R, W1, W2, 1)
    assert (ids == 11).all()


def test_a_token_with_nan_or_infinity_reaches_no_other_token():
    X, R, W1, W2 = inputs(20, 16, 256, 128, torch.float16, 6)
    want = bwgemm.moe_mlp(X, R, W1, W2, 3)
    X[7, 3] = float("nan")
    X[13, 100] = float("inf")
    ids = torch.empty((20, 3), dtype=torch.int32, device="cuda")
    got = bwgemm.moe_mlp(X, R, W1, W2, 3, ids=ids)
    others = [t for t in range(20) if t not in (7, 13)]
    assert torch.isnan(got[7]).all()
    assert torch.equal(got[others], want[others])
    assert ((ids >= 0) & (ids < 16)).all()


def test_inactive_experts_weights_are_not_met():
    X, R, W1, W2 = inputs(4, 32, 256, 128, torch.bfloat16, 7)
    ids, _, _ = moe_ref.route(X, R, 2)
    want = bwgemm.moe_mlp(X, R, W1, W2, 2)
    idle = [e for e in range(32) if e not in set(ids.flatten().tolist())]
    W1[idle] = float("nan")
    W2[idle] = float("nan")
    assert torch.equal(bwgemm.moe_mlp(X, R, W1, W2, 2), want)


def test_inputs_are_left_alone():
    a = inputs(12, 16, 512, 192, torch.float16, 8)
    before = [t.clone() for t in a]
    bwgemm.moe_mlp(*a, 4)
    assert all(torch.equal(x, y) for x, y in zip(a, before))


def test_no_tokens():
    X, R, W1, W2 = inputs(1, 4, 64, 64, torch.float16)
    assert bwgemm.moe_mlp(X[:0], R, W1, W2, 2).shape == (0, 64)


def test_streams_and_overlapping_calls():
    sets = [inputs(t, 32, 1024, 512, torch.bfloat16, 20 + t) for t in (3, 24)]
    want = [bwgemm.moe_mlp(*a, 4) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):  # cooperative launches on both streams
        for i in range(2):
            got[i].append(bwgemm.moe_mlp(*sets[i], 4, stream=streams[i]))
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0, bwgemm.status()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_beside_a_long_gemm():
    """The blocks of a GEMM on another stream hold the SMs: the layer's blocks start once all of them fit."""
    A = torch.randn((8192, 8192), device="cuda").half()
    a = inputs(8, 32, 1024, 512, torch.float16, 31)
    want = bwgemm.moe_mlp(*a, 4)
    C = bwgemm.gemm(A, A)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = []
    for _ in range(8):
        C2 = bwgemm.gemm(A, A)
        out.append(bwgemm.moe_mlp(*a, 4, stream=side))
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0
    assert all(torch.equal(y, want) for y in out) and torch.equal(C, C2)


def test_graphs_with_new_contents_replayed_at_once():
    sets = [inputs(t, 32, 512, 256, torch.bfloat16, 40 + t) for t in (1, 16)]
    for a in sets:
        bwgemm.moe_mlp(*a, 4)
    torch.cuda.synchronize()
    graphs, out = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(bwgemm.moe_mlp(*a, 4))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(10):
        for a in sets:
            a[0].copy_(torch.randn_like(a[0]))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert bwgemm.status()[0] == 0, bwgemm.status()
        for i in range(2):
            assert torch.equal(out[i], bwgemm.moe_mlp(*sets[i], 4))


def test_refused_tensors():
    X, R, W1, W2 = inputs(4, 8, 128, 64, torch.float16, 9)
    for call in (lambda: bwgemm.moe_mlp(X.float(), R, W1, W2, 2), lambda: bwgemm.moe_mlp(X, R.bfloat16(), W1, W2, 2),
                 lambda: bwgemm.moe_mlp(X, R, W1[:, :64], W2, 2), lambda: bwgemm.moe_mlp(X, R, W1, W2.transpose(1, 2), 2),
                 lambda: bwgemm.moe_mlp(X, R[:4], W1, W2, 2), lambda: bwgemm.moe_mlp(X[:, :64], R, W1, W2, 2),
                 lambda: bwgemm.moe_mlp(X, R, W1, W2, 2, ids=torch.empty((4, 3), dtype=torch.int32, device="cuda")),
                 lambda: bwgemm.moe_mlp(X, R, W1, W2, 2, weights=torch.empty((4, 2), dtype=torch.float64, device="cuda")),
                 lambda: bwgemm.moe_mlp(X, R, W1, W2, 2, Y=torch.empty((4, 64), dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: bwgemm.moe_mlp(X, R, W1, W2, 0), lambda: bwgemm.moe_mlp(X, R, W1, W2, 9),
                 lambda: bwgemm.moe_mlp(X.repeat(33, 1), R, W1, W2, 2)):
        with pytest.raises(bwgemm.BwError):
            call()
    n = ctypes.c_size_t()
    L = bwgemm.lib()
    assert L.bw_moe_work_bytes(4, 8, 2, 128, 64, ctypes.byref(n)) == 0
    w = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    rc = L.bw_moe_mlp(X.data_ptr(), 128, R.data_ptr(), W1.data_ptr(), W2.data_ptr(), X.data_ptr(), 4, 8, 2, 128, 64, 0, 1,
                      None, None, w.data_ptr(), n.value - 1, None)
    assert rc == bwgemm.BW_ERR_SCRATCH


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,D,F", [(1, 8, 2, 512, 1024), (3, 256, 8, 1152, 576), (8, 32, 8, 1024, 704)])
def test_few_tokens_are_as_exact_as_one_rounding(T, E, k, D, F, dtype):
    """Up to 8 tokens h is kept as two values, to 2^-16 (bf16) or 2^-22 (fp16) of it: what is left beside the rounding of Y
    is that (for bf16 1 / 128 of Y's own rounding, added in quadrature) and fp32 sums, 2^-20 of Y's norm at these sizes."""
    a = inputs(T, E, D, F, dtype, seed=77)
    Y = bwgemm.moe_mlp(*a, k)
    ids, weights, err = moe_ref.route(a[0], a[1], k)
    y, _ = moe_ref.layer(a[0], ids, weights, err, a[2], a[3])
    rounded = (y.to(dtype).double() - y).norm()
    assert (Y.double() - y).norm() <= 1.02 * rounded + 2.0 ** -18 * y.norm()


def close_to_one_rounding(Y, X, R, W1, W2, k):
    """As test_moe_cpu.close_to_one_rounding derives it: h is off by 2^-16 (bf16) or 2^-22 (fp16) of itself or, in fp16, by up
    to 2^-28 (independent errors, whose sum has at most 2^-28 / sqrt(3) of the norm of W2's row as its standard deviation);
    the sums are fp32, 2^-20 of Y's norm at these sizes."""
    ids, weights, err = moe_ref.route(X, R, k)
    y, _ = moe_ref.layer(X, ids, weights, err, W1, W2)
    rounded = (y.to(X.dtype).double() - y).norm()
    tiny = 0.0
    if X.dtype == torch.float16:
        rows = torch.stack([w.double().norm() for w in W2])  # over an expert's D rows
        tiny = 2.0 ** -28 * float(rows[ids].norm())
    assert torch.isfinite(Y).all()
    assert (Y.double() - y).norm() <= 1.02 * rounded + 2.0 ** -18 * y.norm() + tiny


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,D,F", [(9, 16, 4, 512, 704), (17, 8, 2, 2112, 320), (48, 32, 4, 256, 512), (64, 8, 2, 1024, 576),
                                       (65, 8, 2, 512, 1344), (96, 4, 1, 320, 64), (128, 32, 4, 1472, 704)])
def test_any_number_of_tokens_is_as_exact_as_one_rounding(T, E, k, D, F, dtype):
    a = inputs(T, E, D, F, dtype, seed=T)
    close_to_one_rounding(bwgemm.moe_mlp(*a, k), *a, k)


@pytest.mark.parametrize("scale", [2.0 ** 8, 2.0 ** -9])
@pytest.mark.parametrize("T", [3, 20, 80])
def test_activations_beyond_the_range_of_fp16(T, scale):
    """h up to some 2^20 with small W2, where fp16 ends at 65504; h around 2^-19, below its smallest normal, with large W2."""
    X, R, W1, W2 = inputs(T, 8, 256, 512, torch.float16, T)
    W1, W2 = (W1.float() * scale).half(), (W2.float() / scale ** 1.5).half()
    close_to_one_rounding(bwgemm.moe_mlp(X, R, W1, W2, 2), X, R, W1, W2, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,D,F", [(1, 8, 2, 256, 128), (7, 16, 4, 512, 704), (33, 8, 2, 1024, 1792), (128, 32, 4, 1472, 704),
                                       (20, 2, 1, 64, 64)])
def test_infinity_or_nan_in_w2_reaches_the_tokens_of_its_expert(T, E, k, D, F, dtype):
    """As test_moe_cpu.check_w2: in its own column, the tokens that chose its expert; every other element is what it is
    without (in those columns up to the order of its sum)."""
    X, R, W1, W2 = inputs(T, E, D, F, dtype, seed=T + 9)
    clean = bwgemm.moe_mlp(X, R, W1, W2, k)
    ids, weights, err = moe_ref.route(X, R, k)
    e, cols = int(ids[0, 0]), [3, D - 1, 17]
    W2[e, 3, F // 2] = float("inf")
    W2[e, D - 1, 0] = float("nan")
    W2[e, 17, 5], W2[e, 17, 40] = float("inf"), float("-inf")
    Y = bwgemm.moe_mlp(X, R, W1, W2, k)
    y, _ = moe_ref.layer(X, ids, weights, err, W1, W2)
    y0, tol = moe_ref.layer(X, ids, weights, err, W1, torch.nan_to_num(W2, 0.0, 0.0, 0.0))
    rest = [c for c in range(D) if c not in cols]
    assert torch.equal(Y[:, rest], clean[:, rest])
    Y, fine = Y.double(), torch.isfinite(y)
    assert not fine[0, cols].any()
    assert ((Y - y0).abs() <= tol)[fine].all() and torch.isfinite(Y[fine]).all()
    assert torch.equal(torch.isnan(Y), torch.isnan(y)) and torch.equal(Y[torch.isinf(y)], y[torch.isinf(y)])


def test_a_weight_tensor_full_of_nan():
    """Every result is summed again: slower, and still the definition's (an expert that nobody chose is not met)."""
    X, R, W1, W2 = inputs(64, 8, 512, 1024, torch.bfloat16, 51)
    ids, _, _ = moe_ref.route(X, R, 2)
    bwgemm.moe_mlp(X, R, W1, W2, 2)
    W2[:] = float("nan")
    assert torch.isnan(bwgemm.moe_mlp(X, R, W1, W2, 2)).all()
    torch.cuda.synchronize()
    assert bwgemm.status()[0] == 0


def test_a_stalls_status_stays_until_it_is_cleared():
    """A wait that ran out elsewhere (the library's own check) is still in the status word after a call of the layer, whose
    result does not depend on it."""
    a = inputs(5, 16, 256, 128, torch.float16, 61)
    want = bwgemm.moe_mlp(*a, 4)
    try:
        assert bwgemm.wait_selftest(50_000_000) == bwgemm.BW_ERR_TIMEOUT
        before = bwgemm.status()
        assert before[0] == bwgemm.BW_ERR_TIMEOUT
        assert torch.equal(bwgemm.moe_mlp(*a, 4), want)
        torch.cuda.synchronize()
        assert bwgemm.status() == before
    finally:
        bwgemm.clear_status()
    assert bwgemm.status()[0] == 0


def test_weights_whose_offsets_pass_32_bits():
    """W1 of 2.35e9 elements; the chosen experts are the last ones, and an infinity in the last one's W2 takes the second
    summation there."""
    E, D, F = 160, 4096, 1792
    X, R, _, _ = inputs(2, E, D, 64, torch.bfloat16, 71)
    W1 = torch.zeros((E, 2 * F, D), dtype=torch.bfloat16, device="cuda")
    W2 = torch.zeros((E, D, F), dtype=torch.bfloat16, device="cuda")
    assert W1.numel() > 2 ** 31
    g = torch.Generator(device="cuda")
    g.manual_seed(72)
    for e in (E - 2, E - 1):
        W1[e] = torch.randn((2 * F, D), generator=g, device="cuda") / D ** 0.5
        W2[e] = torch.randn((D, F), generator=g, device="cuda") * (2 / F ** 0.5)
    R[:] = 0
    R[E - 1], R[E - 2] = X[0] / D, X[1] / D  # token 0: the last expert, token 1: the one before
    Y = bwgemm.moe_mlp(X, R, W1, W2, 1)
    ids, _, _ = check(Y, X, R, W1, W2, 1)
    assert ids.flatten().tolist() == [E - 1, E - 2]
    W2[E - 1, D - 1, F - 1] = float("inf")
    got = bwgemm.moe_mlp(X, R, W1, W2, 1)
    assert torch.isinf(got[0, D - 1])
    assert torch.equal(got[1], Y[1]) or ((got[1, D - 1] - Y[1, D - 1]).abs() <= 2.0 ** -7 * Y[1, D - 1].abs() and
                                         torch.equal(got[1, :-1], Y[1, :-1]))
    assert torch.equal(got[0, :-1], Y[0, :-1])
