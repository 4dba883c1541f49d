"""The mixture-of-experts router's own source on the host emulator (tests/test_emulator.py describes it): a cluster of 8
blocks per token, or per four, its choices, weights and laid-out tokens against the definition in 64 bits
(tests/moe_ref.py), and that no block touches another's shared memory before the cluster's blocks have met."""
import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

import moe_ref  # noqa: E402
from test_emulator import CUDA_INCLUDE, PKG, ROOT  # noqa: E402


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    if not os.path.isdir(CUDA_INCLUDE):
        pytest.skip("no CUDA headers")
    lib = str(tmp_path_factory.mktemp("emu_router") / "libbwemu_router.so")
    subprocess.check_call(["g++", "-std=c++20", "-O2", "-pthread", "-DBW_EMULATE", "-DBW_EMU_THREADS=512", "-fPIC",
                           "-shared", "-w", f"-I{CUDA_INCLUDE}", f"-I{os.path.join(ROOT, 'include')}",
                           f"-I{os.path.join(PKG, 'csrc')}", os.path.join(PKG, "emu", "emu_router.cpp"), "-o", lib])
    return ctypes.CDLL(lib)


def emulate(L, X, R, k, renormalize=True):
    T, D = X.shape
    ids = torch.full((T + 1, k), -1, dtype=torch.int32)
    weights = torch.full((T + 1, k), float("nan"))
    xt = torch.full((T * D,), float("nan"), dtype=X.dtype)
    zero = torch.full((77,), 5, dtype=torch.int32)
    nf, msg, vp = ctypes.c_int(), ctypes.create_string_buffer(512), ctypes.c_void_p
    L.bw_emu_router(vp(X.data_ptr()), ctypes.c_longlong(X.stride(0)), vp(R.data_ptr()), T, R.shape[0], k, D,
                    int(X.dtype == torch.bfloat16), int(renormalize), vp(ids.data_ptr()), vp(weights.data_ptr()),
                    vp(xt.data_ptr()), vp(zero.data_ptr()), 76, ctypes.byref(nf), msg, 512)
    assert nf.value == 0, msg.value.decode()
    assert (ids[T] == -1).all() and torch.isnan(weights[T]).all(), "rows past T written"
    assert (zero[:76] == 0).all() and zero[76] == 5
    # K-blocks of 64 values, T rows of 128 bytes, a row's 16-byte chunk c at c ^ (t % 8)
    at = torch.arange(8)[None, :] ^ (torch.arange(T)[:, None] % 8)
    laid = xt.view(D // 64, T, 8, 8).gather(2, at[None, :, :, None].expand(D // 64, T, 8, 8))
    assert torch.equal(laid.permute(1, 0, 2, 3).reshape(T, D).view(torch.int16), X.contiguous().view(torch.int16))
    return ids[:T].long(), weights[:T]


CASES = [  # T, E, k, D, type
    (1, 1, 1, 64, torch.float16),      # blocks without an expert
    (2, 40, 8, 64, torch.bfloat16),    # fewer vectors than lanes
    (1, 129, 32, 320, torch.float16),  # two experts past a power of two
    (17, 9, 2, 192, torch.bfloat16),   # four tokens per cluster, the last of one
    (19, 512, 5, 128, torch.float16),  # more than one round of experts
]


@pytest.mark.parametrize("skew", [0, 50000])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_emulated_router(emu, case, skew):
    """skew: the block that chooses for the first token starts late, after the others have their logits."""
    T, E, k, D, dtype = case
    g = torch.Generator()
    g.manual_seed(T + E)
    X = torch.randn((T, D + 8), generator=g).to(dtype)[:, :D]
    R = (torch.randn((E, D), generator=g) * (1.5 / D ** 0.5)).to(dtype)
    emu.bw_emu_router_set(b"lead_skew_us", ctypes.c_longlong(skew))
    try:
        for renormalize in (True, False):
            ids, weights = emulate(emu, X, R, k, renormalize)
            want, p, err = moe_ref.route(X, R, k, renormalize)
            assert torch.equal(ids, want)
            assert ((weights.double() - p).abs() <= p * err).all()
    finally:
        emu.bw_emu_router_set(b"lead_skew_us", ctypes.c_longlong(0))


def test_equal_logits_go_to_the_lower_index(emu):
    X = torch.zeros((3, 128), dtype=torch.float16)
    X[1] = 1
    R = torch.ones((70, 128), dtype=torch.float16)
    ids, _ = emulate(emu, X, R, 6)
    assert (ids == torch.arange(6)).all()
