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


BAD_OFFSETS = [  # what the caller wrote, what it is taken as (12 rows)
    ([-5, 3, 2, 40], [0, 3, 3, 12]),
    ([4, 4, 100, 7], [4, 4, 12, 12]),
    ([2 ** 31 - 1, 0, 5, 6], [12, 12, 12, 12]),
    ([-2 ** 31, -1, 12, 12], [0, 0, 12, 12]),
]


@pytest.mark.parametrize("bad,taken", BAD_OFFSETS)
def test_row_numbers_out_of_order_lead_nowhere(emu, bad, taken):
    """Through every form: the rows are those of the nearest ascending numbers, and no access leaves X, C or dW."""
    g = gen(5)
    N, K, E = 64, 144, 3
    X = torch.randn((12, K), generator=g).half()
    W = torch.randn((E, N, K), generator=g).half()
    off, want = torch.tensor(bad, dtype=torch.int32), torch.tensor(taken, dtype=torch.int32)
    C, st = emulate(emu, X, W, off, N, 2)
    assert st[0] == 0
    y, err, rows = ref.grouped(X, want, W, N, lambda r, e: ref.product16(X[r], W[e]))
    assert ref.close(C[:12][rows], y[rows], err[rows])[0] and torch.isnan(C[:12][~rows]).all() and torch.isnan(C[12:]).all()
    Q, s, W8, ws, _ = inputs8([4, 4, 4], N, K, torch.float16, 6)
    for cap in (32, 256):
        C, st = emulate(emu, Q, W8, off, N, 2, xs=s, ws=ws, out=torch.float16, cap=cap)
        assert st[0] == 0
        y, err, rows = ref.grouped(Q, want, W8, N, lambda r, e: ref.product8(Q[r], s[r], W8[e], ws[e]))
        assert ref.close(C[:12][rows], y[rows], err[rows])[0] and torch.isnan(C[:12][~rows]).all() and torch.isnan(C[12:]).all()
    dY = torch.randn((12, N), generator=g).half()
    dW = torch.full((E + 1, N, K), float("nan"), dtype=torch.float32)
    st, nf, msg = (ctypes.c_uint * 4)(), i32(), ctypes.create_string_buffer(512)
    emu.bw_emu_grouped_dw(vp(dY.data_ptr()), ll(N), vp(X.data_ptr()), ll(K), vp(off.data_ptr()), vp(dW.data_ptr()), E, 12, N, K,
                          2, 0, 2, 0, st, ctypes.byref(nf), msg, 512)
    assert nf.value == 0 and st[0] == 0, msg.value.decode()
    assert ref.close(dW[:E], *ref.weight_gradient(dY, X, want))[0] and torch.isnan(dW[E]).all()


def test_blocks_out_of_step(emu):
    """The first block of every pair starts late and the engines lag: the waits order the blocks, not luck; the results of
    split tiles are the same bits."""
    Q, s, W, ws, off = inputs8([18], 512, 1040, torch.bfloat16, 9)
    X, W16, o16 = inputs16([9, 0, 70], 264, 328, torch.bfloat16, 10)
    want = [emulate(emu, Q, W, None, 512, 3, xs=s, ws=ws, glu=1, out=torch.bfloat16, cap=c)[0] for c in (32, 256)]
    want16 = emulate(emu, X, W16, o16, 264, 3)[0]
    emu.bw_emu_grouped_set(b"lead_skew_us", ll(30000))
    emu.bw_emu_grouped_set(b"engine_delay_us", ll(300))
    try:
        for c, w in zip((32, 256), want):
            C, st = emulate(emu, Q, W, None, 512, 3, xs=s, ws=ws, glu=1, out=torch.bfloat16, cap=c)
            assert st[0] == 0 and torch.equal(C.view(torch.int16), w.view(torch.int16))
        C, st = emulate(emu, X, W16, o16, 264, 3)
        assert st[0] == 0 and torch.equal(C.view(torch.int16), want16.view(torch.int16))
    finally:
        emu.bw_emu_grouped_set(b"lead_skew_us", ll(0))
        emu.bw_emu_grouped_set(b"engine_delay_us", ll(20))


@pytest.mark.parametrize("form", ["fp16", "e4m3 weights", "e4m3 tokens", "gradient"])
def test_a_load_that_never_lands_ends_the_kernel_with_a_status(emu, form):
    emu.bw_emu_grouped_set(b"wait_ns", ll(500_000_000))
    emu.bw_emu_grouped_set(b"drop_tma", ll(5))
    try:
        st, nf, msg = (ctypes.c_uint * 4)(), i32(), ctypes.create_string_buffer(512)
        X, W, off = inputs16([40, 50], 256, 200, torch.float16, 1)
        if form == "fp16":
            _, st = emulate(emu, X, W, off, 256, 2, glu=2)
        elif form == "gradient":
            dW = torch.empty((2, 200, 200), dtype=torch.float16)
            emu.bw_emu_grouped_dw(vp(X.data_ptr()), ll(200), vp(X.data_ptr()), ll(200), vp(off.data_ptr()), vp(dW.data_ptr()), 2,
                                  90, 200, 200, 2, 0, 0, 0, st, ctypes.byref(nf), msg, 512)
            assert nf.value == 0, msg.value.decode()
        else:
            Q, s, W8, ws, o8 = inputs8([40, 50], 512, 400, torch.float16, 2)
            _, st = emulate(emu, Q, W8, o8, 512, 2, xs=s, ws=ws, glu=2, out=torch.float16, cap=256 if "tokens" in form else 32)
        assert st[0] == 3, "no wait gave up"
    finally:
        emu.bw_emu_grouped_set(b"wait_ns", ll(60_000_000_000))
        emu.bw_emu_grouped_set(b"drop_tma", ll(-1))


SCHED_CHECK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "grouped_sched.h"
using namespace bw;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
// every K-block of every tile exactly once; the parts of a split tile, their slots and their number as its blocks take them
int main()
{
    long long n = 0;
    for (int pairs : {1, 2, 3, 74})
        for (int nt : {1, 2, 5, 40})
            for (int kb : {1, 3, 4, 33, 224})
                for (int runs : {0, 1, 2, 7, 73, 74, 75, 200}) {
                    const GroupSched s = group_sched(nt, kb, pairs, runs);
                    CHECK(s.tiles == nt * runs && s.split < (pairs > 1 ? pairs : 1) + (pairs == 1));
                    CHECK((s.tiles - s.split) % pairs == 0);
                    std::vector<std::vector<int>> owner(s.tiles, std::vector<int>(kb, -1));
                    for (int c = 0; c < pairs; ++c) {
                        GroupWalk w(s, c);
                        GroupSeg g;
                        std::vector<int> slots;
                        while (w.next(s, g)) {
                            CHECK(g.tile >= 0 && g.tile < s.tiles && g.k0 < g.k1 && g.k1 <= kb);
                            for (int k = g.k0; k < g.k1; ++k) {
                                CHECK(owner[g.tile][k] < 0);
                                owner[g.tile][k] = c;
                                ++n;
                            }
                            if (g.k0 != 0 || g.k1 != kb) {
                                CHECK(g.tile < s.split);
                                const int slot = part_slot(s, c, g.tile);
                                CHECK(slot >= 2 * c && slot < 2 * c + 2);
                                for (int o : slots) CHECK(o != slot);
                                slots.push_back(slot);
                                CHECK(c >= tile_first_part(s, g.tile) && c <= tile_last_part(s, g.tile));
                            }
                        }
                    }
                    for (int t = 0; t < s.tiles; ++t) {
                        int parts = 1;
                        for (int k = 0; k < kb; ++k) {
                            CHECK(owner[t][k] >= 0);
                            if (k) {
                                CHECK(t >= s.split || owner[t][k] >= owner[t][k - 1]);  // in the order of K
                                parts += owner[t][k] != owner[t][k - 1];
                            }
                        }
                        if (t < s.split) CHECK(parts == tile_last_part(s, t) - tile_first_part(s, t) + 1);
                        else CHECK(parts == 1);
                    }
                }
    // an expert's runs: all of its rows, none empty, none above the cap
    for (int cap : {32, 64, 128, 256})
        for (int a : {0, 5})
            for (int b = a; b < a + 2100; b += b < a + 300 ? 1 : 37) {
                const int r = group_runs(a, b, cap);
                CHECK((r == 0) == (a == b));
                if (!r) continue;
                const int rows = group_run_rows(a, b, r);
                CHECK(rows % 32 == 0 && rows <= cap && a + (r - 1) * rows < b && a + r * rows >= b);
            }
    // places: every (run, weight tile) of an expert once
    for (int nt : {1, 3, 40})
        for (int runs : {1, 7, 8, 9, 30}) {
            std::vector<char> seen(nt * runs, 0);
            for (int j = 0; j < nt * runs; ++j) {
                int m, w;
                group_place(j, nt, runs, m, w);
                CHECK(m >= 0 && m < runs && w >= 0 && w < nt && !seen[w * runs + m]);
                seen[w * runs + m] = 1;
            }
        }
    // the gradient: every unit of every tile once, whole tiles left for the counter, parts and slots as above
    unsigned rng = 1;
    for (int pairs : {1, 3, 74})
        for (int E : {1, 4, 33})
            for (int per : {1, 6, 88})
                for (int kind = 0; kind < 4; ++kind) {
                    std::vector<int> off(E + 1, 0), cum(E + 1, 0);
                    for (int e = 0; e < E; ++e) {
                        rng = rng * 1664525u + 1013904223u;
                        const int rows = kind == 0 ? 0 : kind == 1 ? (int)(rng >> 20) % 3 : kind == 2 ? (int)(rng >> 20) % 700 : 64 * ((int)(rng >> 24) % 4);
                        off[e + 1] = off[e] + rows;
                        cum[e + 1] = cum[e] + dw_blocks(rows);
                    }
                    const DwSched s = dw_sched(off.data(), cum.data(), E, per, pairs);
                    CHECK(s.tiles == E * per && (s.split == s.tiles || (s.tiles - s.split) % pairs == 0));
                    std::vector<std::vector<int>> owner(s.tiles);
                    for (int t = 0; t < s.tiles; ++t) owner[t].assign(dw_blocks(off[t / per + 1] - off[t / per]), -1);
                    for (int c = 0; c < pairs; ++c) {
                        DwWalk w(s, c);
                        DwSeg g;
                        std::vector<int> slots;
                        while (w.next_part(s, off.data(), cum.data(), g)) {
                            CHECK(g.tile < s.split && g.e == g.tile / per && g.kb == (int)owner[g.tile].size() && g.k0 < g.k1 && g.k1 <= g.kb);
                            CHECK(g.u0 == dw_tile_unit(off.data(), cum.data(), per, g.tile, E));
                            for (int k = g.k0; k < g.k1; ++k) {
                                CHECK(owner[g.tile][k] < 0);
                                owner[g.tile][k] = c;
                                ++n;
                            }
                            if (g.k0 != 0 || g.k1 != g.kb) {
                                const int slot = dw_slot(s, c, g.u0);
                                CHECK(slot >= 2 * c && slot < 2 * c + 2);
                                for (int o : slots) CHECK(o != slot);
                                slots.push_back(slot);
                                CHECK(c >= dw_part_of(s, g.u0) && c <= dw_part_of(s, g.u0 + g.kb - 1));
                            }
                        }
                    }
                    for (int t = 0; t < s.split; ++t) {
                        int parts = 1;
                        for (size_t k = 0; k < owner[t].size(); ++k) {
                            CHECK(owner[t][k] >= 0);
                            if (k) {
                                CHECK(owner[t][k] >= owner[t][k - 1]);
                                parts += owner[t][k] != owner[t][k - 1];
                            }
                        }
                        const long long u0 = dw_tile_unit(off.data(), cum.data(), per, t, E);
                        CHECK(parts == dw_part_of(s, u0 + (long long)owner[t].size() - 1) - dw_part_of(s, u0) + 1);
                    }
                }
    printf("OK %lld\n", n);
    return 0;
}
"""


def test_schedule(tmp_path):
    src, exe = tmp_path / "check.cpp", str(tmp_path / "check")
    src.write_text(SCHED_CHECK)
    subprocess.check_call(["g++", "-std=c++17", "-O2", f"-I{os.path.join(PKG, 'csrc')}", str(src), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("OK"), out.stdout


P = 1 << 20  # an aligned address that nothing is read from: every call below is refused before


@pytest.fixture(scope="module")
def abi():
    import bwgemm

    return bwgemm.lib(), bwgemm


def test_refusals_of_the_grouped_entries(abi):
    L, b = abi
    n = ctypes.c_size_t()

    def call(E=4, M=100, N=256, K=128, ldx=128, type=0, layout=1, swiglu=0, X=P, B=P, off=P, C=P, work=P):
        return L.bw_gemm_grouped(X, ldx, B, off, C, E, M, N, K, type, layout, swiglu, work, 1 << 30, None)

    for bad in (dict(E=0), dict(E=1025), dict(M=-1), dict(M=2 ** 30 + 1), dict(N=0), dict(N=12), dict(K=0), dict(K=100), dict(K=-8),
                dict(ldx=120), dict(ldx=129), dict(ldx=2 ** 33), dict(N=264, swiglu=1), dict(N=2 ** 20 + 8),
                dict(M=2 ** 30, N=2 ** 20)):
        assert call(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(type=2), dict(type=-1), dict(layout=2), dict(swiglu=2), dict(layout=0, swiglu=1), dict(X=0), dict(X=P + 8),
                dict(B=0), dict(B=P + 2), dict(C=P + 4), dict(off=0), dict(off=P + 2), dict(work=0), dict(work=P + 16)):
        assert call(**bad) == b.BW_ERR_ARG, bad
    assert call(M=0) == b.BW_OK and call(M=0, X=0, off=0, work=0) == b.BW_OK
    assert L.bw_gemm_grouped_work_bytes(4, 100, 256, 128, 1, 0, None) == b.BW_ERR_ARG
    assert L.bw_gemm_grouped_work_bytes(4, 0, 256, 128, 1, 0, ctypes.byref(n)) == b.BW_OK and n.value == 0

    def dw(E=4, M=100, N=256, K=128, ldy=256, ldx=128, type=0, out=0, dY=P, X=P, off=P, dW=P, work=P):
        return L.bw_gemm_grouped_dw(dY, ldy, X, ldx, off, dW, E, M, N, K, type, out, work, 1 << 30, None)

    for bad in (dict(E=0), dict(M=-1), dict(N=4), dict(K=12), dict(ldy=248), dict(ldy=257), dict(ldx=64), dict(E=1024, N=2 ** 20, K=2 ** 20)):
        assert dw(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(type=2), dict(out=3), dict(out=-1), dict(dY=0), dict(X=P + 8), dict(off=0), dict(dW=0), dict(dW=P + 8), dict(work=0)):
        assert dw(**bad) == b.BW_ERR_ARG, bad


def test_refusals_of_the_f8_entries(abi):
    L, b = abi
    n = ctypes.c_size_t()

    def gemm(E=0, M=100, N=256, K=128, lds=100, out=0, swiglu=0, A=P, s=P, B=P, t=P, off=None, C=P, work=P):
        return L.bw_gemm_f8(A, s, lds, B, t, off, E, C, M, N, K, out, swiglu, work, 1 << 30, None)

    for bad in (dict(E=-1), dict(E=1025, off=P), dict(M=-1), dict(N=4), dict(K=8), dict(K=72), dict(lds=99), dict(N=384, swiglu=1)):
        assert gemm(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(out=3), dict(swiglu=-1), dict(A=0), dict(A=P + 8), dict(s=P + 2), dict(B=P + 8), dict(t=0), dict(C=P + 8),
                dict(work=P + 128), dict(E=2), dict(E=2, off=P + 1)):
        assert gemm(**bad) == b.BW_ERR_ARG, bad
    assert gemm(M=0) == b.BW_OK

    def linear(E=0, M=100, N=256, K=128, ld=128, type=0, swiglu=0, X=P, B=P, t=P, off=None, C=P, work=P):
        return L.bw_linear_f8(X, type, ld, B, t, off, E, C, M, N, K, swiglu, work, 1 << 30, None)

    for bad in (dict(ld=120), dict(ld=130), dict(K=72), dict(N=257)):
        assert linear(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(type=2), dict(type=3), dict(X=P + 8), dict(B=0), dict(C=0), dict(work=0), dict(E=3)):
        assert linear(**bad) == b.BW_ERR_ARG, bad
    assert linear(M=0) == b.BW_OK

    def quant(type=0, ld=128, Q=P, s=P, lds=100, rows=100, cols=128, X=P):
        return L.bw_quant_f8(X, type, ld, Q, s, lds, rows, cols, None)

    for bad in (dict(ld=120), dict(ld=132), dict(lds=99), dict(rows=-1), dict(cols=0), dict(cols=24, ld=24),
                dict(rows=2 ** 30 + 1, lds=2 ** 31)):
        assert quant(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(type=2), dict(X=P + 8), dict(Q=P + 8), dict(s=0)):
        assert quant(**bad) == b.BW_ERR_ARG, bad
    assert quant(rows=0) == b.BW_OK

    def blocks(type=0, Q=P, s=P, E=1, N=100, K=128, W=P):
        return L.bw_quant_blocks_f8(W, type, Q, s, E, N, K, None)

    for bad in (dict(E=-1), dict(E=65536), dict(N=0), dict(K=8), dict(K=2 ** 20 + 16)):
        assert blocks(**bad) == b.BW_ERR_SHAPE, bad
    for bad in (dict(type=2), dict(W=P + 8), dict(Q=0), dict(s=P + 2)):
        assert blocks(**bad) == b.BW_ERR_ARG, bad
    assert blocks(E=0) == b.BW_OK
    assert L.bw_gemm_f8_work_bytes(0, 0, 256, 128, 0, 0, 1, ctypes.byref(n)) == b.BW_OK and n.value == 0
