"""The 8-bit integer operators without a GPU: their argument checks through the C ABI (refused before any CUDA call), and
the kernels' own source on the host emulator (tests/test_emulator.py describes it) against the definition in 64 bits:
swap-AB with the K split over clusters, stream-K, whole tiles; pair tiles whole, with a split-K tail and with stream-K;
the SwiGLU epilogue; ragged M, K that ends inside a stage, the largest magnitudes."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import bwgemm
import i8_ref
from test_emulator import CUDA_INCLUDE, PKG, ROOT

F16, BF16, F32 = bwgemm.BW_TYPE_F16, bwgemm.BW_TYPE_BF16, bwgemm.BW_TYPE_F32


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    if not os.path.isdir(CUDA_INCLUDE):
        pytest.skip("no CUDA headers")
    lib = str(tmp_path_factory.mktemp("emu_ops") / "libbwemu_ops.so")
    subprocess.check_call(["g++", "-std=c++20", "-O2", "-pthread", "-DBW_EMULATE", "-fPIC", "-shared", "-w",
                           f"-I{CUDA_INCLUDE}", f"-I{os.path.join(ROOT, 'include')}", f"-I{os.path.join(PKG, 'csrc')}",
                           os.path.join(PKG, "emu", "emu_ops.cpp"), "-o", lib])
    return ctypes.CDLL(lib)


def to_f32(bits, out_type):
    if out_type == F32:
        return bits
    if out_type == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def emulate_i8(L, A, sa, B, sb, sms, out_type, swiglu):
    M, K = A.shape
    N = B.shape[0]
    cols = N // 2 if swiglu else N
    # 16 rows of padding after row M: written nowhere
    C = np.full((M + 16, cols), np.nan, np.float32) if out_type == F32 else np.full((M + 16, cols), 0xFFFF, np.uint16)
    st, dirty, nf = (ctypes.c_uint * 4)(), ctypes.c_int(), ctypes.c_int()
    msg = ctypes.create_string_buffer(512)
    vp = ctypes.c_void_p
    rc = L.bw_emu_gemm_i8(vp(A.ctypes.data), vp(sa.ctypes.data), vp(B.ctypes.data), vp(sb.ctypes.data), vp(C.ctypes.data),
                          M, N, K, sms, out_type, swiglu, st, ctypes.byref(dirty), ctypes.byref(nf), msg, 512)
    assert rc == 0, rc
    assert nf.value == 0, msg.value.decode()
    assert st[0] == 0 and dirty.value == 0
    pad = C[M:]
    assert np.isnan(pad).all() if out_type == F32 else (pad == 0xFFFF).all(), "rows past M written"
    return to_f32(C[:M], out_type)


CASES = [  # M, N, K, SMs, type, swiglu
    (1, 256, 64, 8, F16, 0),        # one token; K ends inside the first stage
    (16, 1024, 1024, 8, BF16, 0),   # stream-K swap-AB
    (8, 256, 2048, 8, F16, 0),      # the K split over a cluster
    (100, 448, 1040, 8, F16, 0),    # ragged tokens, a half tile in N, K % 128 != 0
    (130, 512, 272, 8, BF16, 0),    # pair tiles, ragged rows
    (300, 1280, 896, 8, F16, 0),    # pair tiles with split K
    (300, 512, 208, 8, F32, 0),
    (5, 256, 512, 8, F32, 0),       # fp32 at few tokens: pair tiles
    (16, 1280, 512, 4, F16, 1),     # the activation, swap-AB
    (33, 512, 144, 8, BF16, 1),
    (200, 512, 256, 8, BF16, 1),    # the activation, pair tiles
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_emulated_product(emu, case):
    M, N, K, sms, out_type, swiglu = case
    rng = np.random.default_rng(M * 7 + N + K)
    A = rng.integers(-127, 128, (M, K), dtype=np.int8)
    B = rng.integers(-128, 128, (N, K), dtype=np.int8)
    A[0] = 127  # the largest sums of one sign in a corner
    B[0] = -128
    sa = (rng.random(M) * 2e-2 + 1e-3).astype(np.float32)
    sb = (rng.random(N) * 2e-3 + 1e-4).astype(np.float32)
    got = emulate_i8(emu, A, sa, B, sb, sms, out_type, swiglu)
    kind = {F16: "fp16", BF16: "bf16", F32: "fp32"}[out_type]
    bad = i8_ref.outside(got, i8_ref.product(A, sa, B, sb), kind, bool(swiglu))
    assert len(bad) == 0, bad[:4]


# ------------------------------------------------------------------ refusals, before any CUDA call
@pytest.mark.parametrize("M,N,K", [(16, 32, 64), (16, 64, 24), (16, 64, 0), (-1, 64, 64), (16, 64, 131072)])
def test_bad_shapes(M, N, K):
    L = bwgemm.lib()
    assert L.bw_gemm_i8(256, 256, 256, 256, 256, M, N, K, F16, None, 0, None) == bwgemm.BW_ERR_SHAPE
    assert L.bw_linear_i8(256, F16, max(K, 16), 256, 256, 256, M, N, K, 0, 256, 1 << 30, None) == bwgemm.BW_ERR_SHAPE
    n = ctypes.c_size_t(7)
    assert L.bw_gemm_i8_work_bytes(M, N, K, F16, 0, 1, ctypes.byref(n)) == bwgemm.BW_ERR_SHAPE and n.value == 0


def test_swiglu_needs_whole_groups_and_a_16_bit_result():
    L = bwgemm.lib()
    assert L.bw_gemm_i8_swiglu(256, 256, 256, 256, 256, 16, 320, 64, F16, None, 0, None) == bwgemm.BW_ERR_SHAPE
    assert L.bw_gemm_i8_swiglu(256, 256, 256, 256, 256, 16, 256, 64, F32, None, 0, None) == bwgemm.BW_ERR_ARG
    assert L.bw_linear_i8(256, F16, 64, 256, 256, 256, 16, 320, 64, 1, 256, 1 << 30, None) == bwgemm.BW_ERR_SHAPE


def test_bad_arguments():
    L = bwgemm.lib()
    ok = [256, 256, 256, 256, 256]  # A, a_scale, B, b_scale, C
    for i, bad in [(0, 0), (0, 8), (1, 0), (1, 2), (2, 0), (2, 8), (3, 0), (3, 4), (4, 0), (4, 8)]:
        a = list(ok)
        a[i] = bad
        assert L.bw_gemm_i8(*a, 16, 64, 64, F16, None, 0, None) == bwgemm.BW_ERR_ARG, (i, bad)
    assert L.bw_gemm_i8(*ok, 16, 64, 64, 3, None, 0, None) == bwgemm.BW_ERR_ARG
    assert L.bw_gemm_i8(*ok, 16, 64, 64, F16, 128, 4096, None) == bwgemm.BW_ERR_ARG  # a workspace off 256 bytes
    assert L.bw_linear_i8(256, F32, 64, 256, 256, 256, 16, 64, 64, 0, 256, 1 << 20, None) == bwgemm.BW_ERR_ARG
    assert L.bw_linear_i8(256, F16, 64, 256, 256, 256, 16, 64, 64, 2, 256, 1 << 20, None) == bwgemm.BW_ERR_ARG
    assert L.bw_linear_i8(256, F16, 64, 256, 256, 256, 16, 64, 64, 0, None, 0, None) == bwgemm.BW_ERR_ARG
    assert L.bw_gemm_i8_work_bytes(16, 64, 64, F16, 0, 0, None) == bwgemm.BW_ERR_ARG


def test_bad_rows_to_quantise():
    L = bwgemm.lib()
    q = lambda x=256, t=F16, ld=64, Q=256, s=256, r=4, c=64: L.bw_quant_rows_i8(x, t, ld, Q, s, r, c, None)  # noqa: E731
    assert q(c=24) == q(ld=56) == q(ld=68) == q(r=-1) == q(c=0) == bwgemm.BW_ERR_SHAPE
    assert q(x=8) == q(x=0) == q(t=F32) == q(Q=8) == q(Q=0) == q(s=0) == q(s=2) == bwgemm.BW_ERR_ARG


def test_no_rows_is_a_call_that_does_nothing():
    L = bwgemm.lib()
    assert L.bw_quant_rows_i8(None, F16, 64, None, None, 0, 64, None) == bwgemm.BW_OK
    assert L.bw_gemm_i8(None, None, None, None, None, 0, 64, 64, F16, None, 0, None) == bwgemm.BW_OK
    assert L.bw_linear_i8(None, BF16, 64, None, None, None, 0, 64, 64, 0, None, 0, None) == bwgemm.BW_OK
    n = ctypes.c_size_t(7)
    assert L.bw_gemm_i8_work_bytes(0, 64, 64, F16, 0, 1, ctypes.byref(n)) == bwgemm.BW_OK and n.value == 0


def test_python_refuses_tensors_it_cannot_pass_on():
    torch = pytest.importorskip("torch")
    x = torch.zeros((4, 64), dtype=torch.float16)
    w, s = torch.zeros((64, 64), dtype=torch.int8), torch.zeros(64)
    for call in (lambda: bwgemm.quantize_rows(x), lambda: bwgemm.linear_i8(x, w, s),
                 lambda: bwgemm.gemm_i8(w, s, w, s), lambda: bwgemm.gemm_i8_swiglu(w, s, w, s, dtype=torch.float32),
                 lambda: bwgemm.gemm_i8(w, s, w, s, dtype=torch.float64)):
        with pytest.raises(ValueError):  # host tensors, types
            call()


@pytest.mark.parametrize("late", [0, 1])
@pytest.mark.parametrize("force", [2 * 16 + 1, 3 * 16 + 2, 5 * 16 + 1, 6 * 16 + 2, 8 * 16 + 1])
def test_emulated_k_split_into_the_buffer_or_the_ring(emu, force, late):
    """Clusters of up to 5 blocks send their parts into a buffer that is expected from the start; larger ones into the idle
    ring, once it is.  late: the first block of every cluster starts late, so that the others' parts are sent before it
    runs."""
    c, wm = force // 16, force % 16
    rng = np.random.default_rng(force)
    M, N, K = 11, 256 * wm, 4096
    A = rng.integers(-127, 128, (M, K), dtype=np.int8)
    B = rng.integers(-127, 128, (N, K), dtype=np.int8)
    sa, sb = np.full(M, 1e-2, np.float32), np.full(N, 1e-3, np.float32)
    emu.bw_emu_set(b"force_ksplit", ctypes.c_longlong(force))
    emu.bw_emu_set(b"lead_skew_us", ctypes.c_longlong(200000 * late))
    try:
        got = emulate_i8(emu, A, sa, B, sb, 2 * c, F16, 0)
    finally:
        emu.bw_emu_set(b"force_ksplit", ctypes.c_longlong(0))
        emu.bw_emu_set(b"lead_skew_us", ctypes.c_longlong(0))
    assert len(i8_ref.outside(got, i8_ref.product(A, sa, B, sb), "fp16")) == 0


@pytest.mark.parametrize("force", [2 * 16 + 1, 3 * 16 + 2, 5 * 16 + 1])
def test_a_block_that_gives_up_leaves_after_the_parts_sent_to_it(emu, force):
    """The last block of a cluster owns a run of the tile's columns; its accumulator's completion never arrives, so
    its epilogue gives up, while the other blocks' parts of those columns are on their way into
    its buffer (expected from the start, so nobody asks).  They land before it leaves."""
    c, wm = force // 16, force % 16
    rng = np.random.default_rng(force)
    M, N, K = 11, 256 * wm, 128 * 4 * c  # 4 stages a block: commits 0 to 3 free them, 4 is the accumulator's
    A = rng.integers(-127, 128, (M, K), dtype=np.int8)
    B = rng.integers(-127, 128, (N, K), dtype=np.int8)
    C = np.zeros((M, N), np.uint16)
    sa, sb = np.ones(M, np.float32), np.ones(N, np.float32)
    st, dirty, nf = (ctypes.c_uint * 4)(), ctypes.c_int(), ctypes.c_int()
    msg, vp = ctypes.create_string_buffer(512), ctypes.c_void_p
    # a part takes about half a second to cross; the accumulator's wait (kind 2) gives up after 0.3 s, others after 3
    knobs = dict(force_ksplit=force, wait_ns=3_000_000_000, short_kind=2, engine_delay_us=2000, drop_block=c - 1, drop_commit=4)
    for name, value in knobs.items():
        assert emu.bw_emu_set(name.encode(), ctypes.c_longlong(value)) == 0
    try:
        emu.bw_emu_gemm_i8(vp(A.ctypes.data), vp(sa.ctypes.data), vp(B.ctypes.data), vp(sb.ctypes.data), vp(C.ctypes.data),
                           M, N, K, 2 * c, F16, 0, st, ctypes.byref(dirty), ctypes.byref(nf), msg, 512)
    finally:
        for name, value in dict(force_ksplit=0, wait_ns=60_000_000_000, short_kind=-1, engine_delay_us=20, drop_block=-1,
                                drop_commit=-1).items():
            emu.bw_emu_set(name.encode(), ctypes.c_longlong(value))
    assert st[0] == 3, "no wait gave up"
    assert nf.value == 0, msg.value.decode()


@pytest.mark.parametrize("M,N,K,sms,out_type,swiglu", [(9, 256, 256, 4, F16, 0), (20, 512, 256, 4, BF16, 1),
                                                       (130, 512, 256, 8, F16, 0), (130, 256, 256, 4, F32, 0)])
def test_the_scales_are_no_constants_of_the_product(emu, M, N, K, sms, out_type, swiglu):
    """In the linear layer's one call the product starts while the quantiser still writes the row scales, and with
    BWGEMM_PDL=1 so may a product whose column scales a kernel ahead writes: neither may be read through the non-coherent
    path (the emulator reports such a load)."""
    A, B = np.ones((M, K), np.int8), np.ones((N, K), np.int8)
    s = np.ones(max(M, N), np.float32)
    got = emulate_i8(emu, A, s[:M].copy(), B, s[:N].copy(), sms, out_type, swiglu)
    assert (got == (K * K if swiglu else K)).all()
