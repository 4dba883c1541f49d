"""The grouped and 8-bit floating-point products without a GPU: the cut into tiles and parts (grouped_sched.h, through a small
program), the argument checks through the C ABI, and the kernels' own source on the host emulator (tests/test_emulator.py
describes it) against the definitions in 64 bits (tests/grouped_ref.py)."""
import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

import grouped_ref as ref  # noqa: E402
from test_emulator import CUDA_INCLUDE, PKG, ROOT  # noqa: E402


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    if not os.path.isdir(CUDA_INCLUDE):
        pytest.skip("no CUDA headers")
    lib = str(tmp_path_factory.mktemp("emu_grouped") / "libbwemu_grouped.so")
    subprocess.check_call(["g++", "-std=c++20", "-O2", "-pthread", "-DBW_EMULATE", "-DBW_EMU_THREADS=384", "-fPIC",
                           "-shared", "-w", f"-I{CUDA_INCLUDE}", f"-I{os.path.join(ROOT, 'include')}",
                           f"-I{os.path.join(PKG, 'csrc')}", os.path.join(PKG, "emu", "emu_grouped.cpp"), "-o", lib])
    return ctypes.CDLL(lib)


OUT = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
vp, i32, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


def emulate(L, X, W, off, N, pairs, xs=None, ws=None, mn=False, glu=0, out=None, cap=32, stages=0):
    """The kernel's form by cap: 8-bit operands with 256 tokens a tile have the tokens as the MMA's M."""
    kind = 0 if xs is None else 2 if cap == 256 else 1
    T, K = X.shape
    E = 1 if off is None else off.numel() - 1
    out = X.dtype if out is None else out
    C = torch.full((T + 8, N // 2 if glu else N), float("nan"), dtype=out)  # rows past T: written nowhere
    st, dirty, nf, msg = (ctypes.c_uint * 4)(), i32(), i32(), ctypes.create_string_buffer(512)
    ptr = lambda t: vp(t.data_ptr()) if t is not None else None
    L.bw_emu_grouped(ptr(X), ll(X.stride(0)), ptr(xs), ll(xs.stride(1) if xs is not None else 0), ptr(W), ptr(ws), ptr(off),
                     ptr(C), E, T, N, K, pairs, kind, int(X.dtype == torch.bfloat16), int(mn), glu,
                     OUT[out], cap, stages, st, ctypes.byref(dirty), ctypes.byref(nf), msg, 512)
    assert nf.value == 0, msg.value.decode()
    return C, list(st)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def inputs16(counts, N, K, dtype, seed, mn=False, pad=0, first=0, tail=0):
    g = gen(seed)
    T = first + sum(counts) + tail
    X = torch.randn((T, K + pad), generator=g).to(dtype)[:, :K]
    shape = (len(counts), K, N) if mn else (len(counts), N, K)
    W = (torch.randn(shape, generator=g) / K ** 0.5).to(dtype)
    return X, W, ref.offsets_of(counts, first)


CASES16 = [  # counts, N, K, pairs, type, W as E x K x N, activation, cap
    ([5], 64, 64, 1, torch.float16, False, 0, 32),
    ([0, 7, 0, 40, 1], 328, 200, 2, torch.bfloat16, False, 0, 32),      # empty experts, ragged everything
    ([33, 70], 256, 136, 2, torch.float16, True, 0, 64),
    ([3, 0, 66], 264, 328, 3, torch.bfloat16, True, 0, 64),             # split tiles
    ([9, 20], 400, 128, 2, torch.float16, False, 2, 32),                # gate and up halves, 200 columns
    ([1, 2, 3], 512, 72, 1, torch.bfloat16, False, 1, 32),
    ([260], 256, 64, 2, torch.float16, False, 0, 256),                  # the widest runs
    ([17], 256, 576, 4, torch.bfloat16, False, 2, 32),                  # one tile split over several pairs, activation
]


@pytest.mark.parametrize("case", CASES16, ids=lambda c: "-".join(map(str, c[0])) + "x%dx%d" % (c[1], c[2]))
def test_emulated_grouped(emu, case):
    counts, N, K, pairs, dtype, mn, glu, cap = case
    X, W, off = inputs16(counts, N, K, dtype, N + K, mn, pad=8, first=2, tail=3)
    C, st = emulate(emu, X, W, off, N, pairs, mn=mn, glu=glu, cap=cap)
    assert st[0] == 0, st
    y, err, rows = ref.grouped(X, off, W, N, lambda r, e: ref.product16(X[r], W[e].t() if mn else W[e]))
    if glu:
        y, err = ref.glu(y, err, glu == 1)
    T = X.shape[0]
    ok, worst = ref.close(C[:T][rows], y[rows], err[rows])
    assert ok, worst
    assert torch.isnan(C[:T][~rows]).all() and torch.isnan(C[T:]).all(), "rows of no expert were written"


def inputs8(counts, N, K, dtype, seed, first=0, tail=0):
    g = gen(seed)
    T = first + sum(counts) + tail
    X = torch.randn((T, K), generator=g).to(dtype)
    q, s = ref.quantize_rows(X)
    ld = (T + 3) // 4 * 4
    buf = torch.full((s.shape[1], ld), float("nan"))
    buf[:, :T] = s.t().float()
    E = len(counts)
    w8, ws = [], []
    for e in range(E):
        a, b = ref.quantize_blocks((torch.randn((N, K), generator=g) / K ** 0.5).to(dtype))
        w8.append(a)
        ws.append(b)
    w8, ws = torch.stack(w8), torch.stack(ws).float().contiguous()
    f8 = lambda t: t.float().to(torch.float8_e4m3fn).contiguous()
    return f8(q), buf.t()[:T], f8(w8), ws, ref.offsets_of(counts, first)


CASES8 = [  # counts (None offsets: one), N, K, pairs, out, activation, cap
    ([1], 64, 128, 1, torch.bfloat16, 0, 32, False),
    ([19], 328, 272, 2, torch.float32, 0, 32, False),                   # K and N end inside a block
    ([5, 0, 38, 1], 264, 400, 2, torch.float16, 0, 32, True),
    ([66, 3], 512, 160, 3, torch.bfloat16, 2, 64, True),
    ([18], 512, 1040, 3, torch.bfloat16, 1, 32, False),                 # split tiles with the activation
    ([100], 256, 144, 1, torch.float16, 0, 128, False),
    ([200], 256, 144, 1, torch.float16, 0, 256, False),                 # the tokens as the MMA's M from here on
    ([130, 0, 300], 328, 400, 2, torch.float32, 0, 256, True),
    ([5], 264, 1168, 3, torch.bfloat16, 0, 256, False),                 # split tiles
    ([290], 512, 272, 2, torch.bfloat16, 1, 256, False),
    ([3, 140], 512, 400, 3, torch.float16, 2, 256, True),
]


@pytest.mark.parametrize("case", CASES8, ids=lambda c: "-".join(map(str, c[0])) + "x%dx%d" % (c[1], c[2]))
def test_emulated_f8(emu, case):
    counts, N, K, pairs, out, glu, cap, grouped = case
    Q, s, W, ws, off = inputs8(counts, N, K, torch.bfloat16, N + K, first=3 if grouped else 0, tail=2 if grouped else 0)
    C, st = emulate(emu, Q, W, off if grouped else None, N, pairs, xs=s, ws=ws, glu=glu, out=out, cap=cap)
    assert st[0] == 0, st
    y, err, rows = ref.grouped(Q, off, W, N, lambda r, e: ref.product8(Q[r], s[r], W[e], ws[e]))
    if glu:
        y, err = ref.glu(y, err, glu == 1)
    T = Q.shape[0]
    ok, worst = ref.close(C[:T][rows], y[rows], err[rows])
    assert ok, worst
    assert torch.isnan(C[:T][~rows].float()).all() and torch.isnan(C[T:].float()).all(), "rows of no expert were written"


CASES_DW = [  # counts, N, K, pairs, type, out
    ([5], 64, 64, 1, torch.float16, torch.float16),
    ([0, 7, 0, 64, 81], 136, 200, 2, torch.bfloat16, torch.float32),    # empty experts, one whole stage, a tail of 1
    ([3, 66, 16, 0], 264, 72, 3, torch.float16, torch.float16),
    ([300, 0], 256, 328, 3, torch.bfloat16, torch.bfloat16),            # split tiles
    ([1] * 7 + [130], 72, 296, 1, torch.bfloat16, torch.bfloat16),      # more tiles than a pair splits
]


@pytest.mark.parametrize("case", CASES_DW, ids=lambda c: "-".join(map(str, c[0])) + "x%dx%d" % (c[1], c[2]))
def test_emulated_weight_gradient(emu, case):
    counts, N, K, pairs, dtype, out = case
    g = gen(N + K)
    first, tail = 2, 3
    T = first + sum(counts) + tail
    dY, X = (torch.randn((T, n + 8), generator=g).to(dtype)[:, :n] for n in (N, K))
    off = ref.offsets_of(counts, first)
    # rows of no expert hold infinities and NaN: they reach nothing
    for v in (dY, X):
        v[:first] = float("nan")
        v[T - tail:] = float("inf")
    E = len(counts)
    dW = torch.full((E + 1, N, K), float("nan"), dtype=out)
    st, nf, msg = (ctypes.c_uint * 4)(), i32(), ctypes.create_string_buffer(512)
    emu.bw_emu_grouped_dw(vp(dY.data_ptr()), ll(dY.stride(0)), vp(X.data_ptr()), ll(X.stride(0)), vp(off.data_ptr()),
                          vp(dW.data_ptr()), E, T, N, K, pairs, int(dtype == torch.bfloat16), OUT[out], 0, st,
                          ctypes.byref(nf), msg, 512)
    assert nf.value == 0, msg.value.decode()
    assert st[0] == 0, list(st)
    y, err = ref.weight_gradient(dY, X, off)
    ok, worst = ref.close(dW[:E], y, err)
    assert ok, worst
    assert torch.isnan(dW[E]).all()
