"""The mixture-of-experts layer without a GPU: its work split (moe_sched.h, through a small program), its argument checks
through the C ABI, and the experts kernel's own source on the host emulator (tests/test_emulator.py describes it; here
every block of the grid runs at once) against the definition in 64 bits (tests/moe_ref.py)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import moe_ref  # noqa: E402
from test_emulator import CUDA_INCLUDE, PKG, ROOT  # noqa: E402


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    if not os.path.isdir(CUDA_INCLUDE):
        pytest.skip("no CUDA headers")
    lib = str(tmp_path_factory.mktemp("emu_moe") / "libbwemu_moe.so")
    subprocess.check_call(["g++", "-std=c++20", "-O2", "-pthread", "-DBW_EMULATE", "-DBW_EMU_THREADS=352", "-fPIC",
                           "-shared", "-w", f"-I{CUDA_INCLUDE}", f"-I{os.path.join(ROOT, 'include')}",
                           f"-I{os.path.join(PKG, 'csrc')}", os.path.join(PKG, "emu", "emu_moe.cpp"), "-o", lib])
    return ctypes.CDLL(lib)


def emulate(L, X, W1, W2, ids, weights, grid):
    T, D = X.shape
    E, _, F = W2.shape[0], None, W2.shape[2]
    Y = torch.full((T + 8, D), float("nan"), dtype=X.dtype)  # rows past T: written nowhere
    ids, weights = ids.to(torch.int32).contiguous(), weights.float().contiguous()
    st, nf, msg = (ctypes.c_uint * 4)(), ctypes.c_int(), ctypes.create_string_buffer(512)
    vp = ctypes.c_void_p
    L.bw_emu_moe(vp(X.data_ptr()), ctypes.c_longlong(X.stride(0)), vp(W1.data_ptr()), vp(W2.data_ptr()), vp(Y.data_ptr()),
                 vp(ids.data_ptr()), vp(weights.data_ptr()), T, E, ids.shape[1], D, F, grid,
                 int(X.dtype == torch.bfloat16), st, ctypes.byref(nf), msg, 512)
    return Y, list(st), nf.value, msg.value.decode()


def inputs(T, E, D, F, dtype, seed, pad=0):
    g = torch.Generator()
    g.manual_seed(seed)
    X = torch.randn((T, D + pad), generator=g).to(dtype)[:, :D]
    R = (torch.randn((E, D), generator=g) / D ** 0.5).to(dtype)
    W1 = (torch.randn((E, 2 * F, D), generator=g) / D ** 0.5).to(dtype)
    W2 = (torch.randn((E, D, F), generator=g) / F ** 0.5).to(dtype)
    return X, R, W1, W2


CASES = [  # T, E, k, D, F, grid, type
    (1, 4, 1, 64, 64, 4, torch.float16),      # fewer K-blocks than shares take
    (1, 8, 2, 256, 128, 4, torch.bfloat16),   # split tiles of both products
    (3, 4, 4, 128, 192, 3, torch.float16),    # every expert active; F ends inside a tile
    (17, 6, 2, 320, 128, 5, torch.bfloat16),  # ragged tokens, a ragged output tile
    (5, 2, 1, 576, 64, 2, torch.float16),     # more output tiles than blocks: whole tiles of both products
    (40, 3, 3, 128, 128, 7, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_emulated_layer(emu, case):
    T, E, k, D, F, grid, dtype = case
    X, R, W1, W2 = inputs(T, E, D, F, dtype, T + D, pad=8)
    ids, weights, err = moe_ref.route(X, R, k)
    Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, grid)
    assert findings == 0, msg
    assert st[0] == 0, st
    y, tol = moe_ref.layer(X, ids, weights, err, W1, W2)
    assert ((Y[:T].double() - y).abs() <= tol).all()
    assert torch.isnan(Y[T:]).all()


def test_emulated_layer_with_blocks_out_of_step(emu):
    """The blocks start one after the other and the engines lag: the waits between the blocks, not luck, order them."""
    X, R, W1, W2 = inputs(9, 5, 256, 192, torch.bfloat16, 3)
    ids, weights, err = moe_ref.route(X, R, 2)
    y, tol = moe_ref.layer(X, ids, weights, err, W1, W2)
    emu.bw_emu_moe_set(b"block_ramp_us", ctypes.c_longlong(20000))
    emu.bw_emu_moe_set(b"engine_delay_us", ctypes.c_longlong(300))
    try:
        first = None
        for _ in range(2):
            Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, 6)
            assert findings == 0 and st[0] == 0, (msg, st)
            assert ((Y[:9].double() - y).abs() <= tol).all()
            assert first is None or torch.equal(first, Y[:9]), "the order of the blocks shows in the result"
            first = Y[:9]
    finally:
        emu.bw_emu_moe_set(b"block_ramp_us", ctypes.c_longlong(0))
        emu.bw_emu_moe_set(b"engine_delay_us", ctypes.c_longlong(20))


def test_a_token_with_nan_reaches_no_other_token(emu):
    X, R, W1, W2 = inputs(4, 4, 128, 128, torch.float16, 5)
    ids, weights, err = moe_ref.route(X, R, 2)
    want, _, _, _ = emulate(emu, X, W1, W2, ids, weights, 4)
    X[2, 7] = float("nan")
    got, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, 4)
    assert findings == 0 and st[0] == 0
    assert torch.isnan(got[2]).all() and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


def test_a_load_that_never_lands_ends_the_kernel_with_a_status(emu):
    X, R, W1, W2 = inputs(2, 4, 128, 128, torch.float16, 6)
    ids, weights, _ = moe_ref.route(X, R, 2)
    emu.bw_emu_moe_set(b"wait_ns", ctypes.c_longlong(300_000_000))
    emu.bw_emu_moe_set(b"drop_tma", ctypes.c_longlong(3))
    try:
        _, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, 4)
        assert findings == 0, msg
        assert st[0] == 3, "no wait gave up"
    finally:
        emu.bw_emu_moe_set(b"wait_ns", ctypes.c_longlong(60_000_000_000))
        emu.bw_emu_moe_set(b"drop_tma", ctypes.c_longlong(-1))


SCHED_CHECK = r"""
#include <cstdio>
#include <vector>
#include <set>
#include <cstdlib>
#include "moe_sched.h"
using namespace bw;
// every K-block of every tile of both products exactly once, in shares that differ by one; a split tile's segments,
// counters and slots as its writers and readers take them to be
int main()
{
    long long checked = 0;
    for (int grid : {1, 2, 3, 8, 74, 148})
        for (int active : {1, 2, 3, 8, 60})
            for (int D : {64, 128, 576, 2048})
                for (int F : {64, 192, 1344}) {
                    const MoeSched s = moe_sched(5, D, F, active, grid);
                    const int tiles[2] = {active * s.f_tiles, s.d_tiles}, kbs[2] = {s.kb1, active * s.kbf};
                    std::vector<std::vector<char>> seen[2];
                    std::vector<int> parts[2], counter[2];
                    std::set<int> slots, counters;
                    for (int ph = 0; ph < 2; ++ph) {
                        seen[ph].assign(tiles[ph], std::vector<char>(kbs[ph], 0));
                        parts[ph].assign(tiles[ph], 0);
                        counter[ph].assign(tiles[ph], -1);
                    }
                    for (int c = 0; c < grid; ++c) {
                        MoeIter it(s, c);
                        MoeSeg g;
                        int last_phase = 0, split2 = 0;
                        while (it.next(s, g)) {
                            if (g.phase < last_phase || g.k0 >= g.k1 || g.tile >= tiles[g.phase]) return 1;
                            last_phase = g.phase;
                            for (int k = g.k0; k < g.k1; ++k)
                                if (k >= kbs[g.phase] || seen[g.phase][g.tile][k]++) return 2;
                            const bool whole = g.k0 == 0 && g.k1 == kbs[g.phase];
                            if (whole != (g.nseg == 1)) return 3;
                            if (c < g.first || c >= g.first + g.nseg) return 4;
                            ++parts[g.phase][g.tile];
                            if (g.nseg > 1) {
                                if (moe_slot(g, c) / 4 != c || !slots.insert(moe_slot(g, c)).second) return 5;
                                if (counter[g.phase][g.tile] < 0) {
                                    counter[g.phase][g.tile] = moe_counter(g);
                                    if (moe_counter(g) >= 2 * grid || !counters.insert(moe_counter(g)).second) return 6;
                                } else if (counter[g.phase][g.tile] != moe_counter(g)) return 7;
                                if (g.phase == 1 && ++split2 > 2) return 8;
                            }
                            const int b = g.first + g.nseg - 1;  // the last block of the tile
                            if (g.nseg > 1 && (c == b) != (g.k1 == kbs[g.phase])) return 9;
                            ++checked;
                        }
                    }
                    for (int ph = 0; ph < 2; ++ph)
                        for (int t = 0; t < tiles[ph]; ++t)
                            for (char v : seen[ph][t])
                                if (v != 1) return 10;
                }
    printf("%lld\n", checked);
    return checked > 1000 ? 0 : 11;
}
"""


def test_the_work_split(tmp_path):
    src = tmp_path / "check.cpp"
    src.write_text(SCHED_CHECK)
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O2", f"-I{os.path.join(PKG, 'csrc')}", str(src), "-o", exe])
    r = subprocess.run([exe], capture_output=True)
    assert r.returncode == 0, r.returncode


# ------------------------------------------------------------------ refusals, before any CUDA call
def moe_call(T=4, E=8, k=2, D=128, F=64, type=0, ldx=None, renormalize=1, X=256, R=256, W1=256, W2=256, Y=256, ids=None,
             weights=None, work=256):
    import bwgemm

    return bwgemm.lib().bw_moe_mlp(X, D if ldx is None else ldx, R, W1, W2, Y, T, E, k, D, F, type, renormalize, ids,
                                   weights, work, 1 << 40, None)


@pytest.mark.parametrize("bad", [dict(T=129), dict(T=-1), dict(E=0), dict(E=513), dict(k=0), dict(k=9), dict(E=64, k=33),
                                 dict(D=96), dict(D=0), dict(F=32), dict(F=0), dict(ldx=64), dict(ldx=132)], ids=str)
def test_bad_shapes(bad):
    import bwgemm

    assert moe_call(**bad) == bwgemm.BW_ERR_SHAPE


@pytest.mark.parametrize("bad", [dict(type=2), dict(type=-1), dict(renormalize=2), dict(X=0), dict(X=8), dict(R=0),
                                 dict(W1=8), dict(W2=0), dict(Y=0), dict(Y=1), dict(work=0), dict(work=128), dict(ids=2),
                                 dict(weights=6)], ids=str)
def test_bad_arguments(bad):
    import bwgemm

    assert moe_call(**bad) == bwgemm.BW_ERR_ARG


def test_no_tokens_and_the_workspace_query():
    import bwgemm

    n = ctypes.c_size_t(7)
    assert moe_call(T=0, X=0, work=0) == bwgemm.BW_OK
    assert bwgemm.lib().bw_moe_work_bytes(0, 8, 2, 128, 64, ctypes.byref(n)) == bwgemm.BW_OK and n.value == 0
    assert bwgemm.lib().bw_moe_work_bytes(4, 8, 9, 128, 64, ctypes.byref(n)) == bwgemm.BW_ERR_SHAPE
    assert bwgemm.lib().bw_moe_work_bytes(4, 8, 2, 128, 64, None) == bwgemm.BW_ERR_ARG


# ------------------------------------------------------------------ what of h reaches the down product
def close_to_one_rounding(Y, X, ids, weights, err, W1, W2):
    """h = p silu(g) u goes to the down product as two values of the type, together within 2^-16 (bf16) or 2^-22 (fp16) of it
    and, in fp16, at worst 2^-28 off (half the second value's smallest step, its scale counted): independent errors, whose
    sum over an expert's F has at most 2^-28 / sqrt(3) of the norm of W2's row as its standard deviation.  The sums are fp32
    (2^-20 of Y's norm at these sizes).  Beside Y's own rounding that is (for bf16 1 / 128 of the rounding, added in quadrature)."""
    y, _ = moe_ref.layer(X, ids, weights, err, W1, W2)
    rounded = (y.to(X.dtype).double() - y).norm()
    tiny = torch.zeros_like(y)
    if X.dtype == torch.float16:
        for t in range(X.shape[0]):
            for e in ids[t].tolist():
                tiny[t] += (2.0 ** -28 * W2[e].double().norm(dim=1)) ** 2
    assert torch.isfinite(Y.double()).all()
    got = (Y.double() - y).norm()
    assert got <= 1.02 * rounded + 2.0 ** -18 * y.norm() + tiny.sum().sqrt(), float(got / rounded)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,D,F,grid", [(8, 4, 2, 128, 128, 4), (9, 4, 2, 128, 192, 3), (40, 3, 3, 128, 128, 7),
                                            (64, 2, 1, 64, 128, 2), (65, 2, 1, 320, 64, 3), (128, 2, 2, 64, 192, 2)])
def test_emulated_layer_is_as_exact_as_one_rounding(emu, T, E, k, D, F, grid, dtype):
    X, R, W1, W2 = inputs(T, E, D, F, dtype, T + F)
    ids, weights, err = moe_ref.route(X, R, k)
    Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, grid)
    assert findings == 0 and st[0] == 0, (msg, st)
    assert torch.isnan(Y[T:]).all()
    close_to_one_rounding(Y[:T], X, ids, weights, err, W1, W2)


@pytest.mark.parametrize("scale", [2.0 ** 8, 2.0 ** -9])
@pytest.mark.parametrize("T", [3, 20, 80])
def test_emulated_activations_beyond_the_range_of_fp16(emu, T, scale):
    """h up to some 2^20 with small W2, where fp16 ends at 65504; h around 2^-19, below its smallest normal, with large W2."""
    D, F = 128, 128
    X, R, W1, W2 = inputs(T, 4, D, F, torch.float16, T)
    W1, W2 = (W1.float() * scale).half(), (W2.float() / scale ** 1.5).half()
    ids, weights, err = moe_ref.route(X, R, 2)
    Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, 4)
    assert findings == 0 and st[0] == 0, (msg, st)
    close_to_one_rounding(Y[:T], X, ids, weights, err, W1, W2)


# ------------------------------------------------------------------ infinities and NaN in the weights
def check_w2(Y, clean, X, ids, weights, err, W1, W2, cols):
    """An infinity or a NaN of W2 reaches, in its own column, the tokens that chose its expert, as the definition has it;
    every other element is what it is without (in those columns up to the order of its sum)."""
    y, _ = moe_ref.layer(X, ids, weights, err, W1, W2)
    y0, tol = moe_ref.layer(X, ids, weights, err, W1, torch.nan_to_num(W2, 0.0, 0.0, 0.0))
    Y, fine = Y.double(), torch.isfinite(y)
    assert (~fine).any() and fine[:, cols].any(), "the case shows nothing"
    rest = [c for c in range(Y.shape[1]) if c not in cols]
    assert torch.equal(Y[:, rest], clean.double()[:, rest])
    assert torch.isfinite(Y[fine]).all()
    assert ((Y - y0).abs() <= tol)[fine].all()
    assert torch.equal(torch.isnan(Y), torch.isnan(y)) and torch.equal(Y[torch.isinf(y)], y[torch.isinf(y)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,D,F,grid", [(2, 8, 2, 256, 128, 4), (5, 4, 1, 576, 64, 2), (12, 6, 2, 320, 192, 3),
                                            (70, 4, 1, 64, 64, 2)])
def test_emulated_infinity_or_nan_in_w2_reaches_the_tokens_of_its_expert(emu, T, E, k, D, F, grid, dtype):
    X, R, W1, W2 = inputs(T, E, D, F, dtype, T + 11)
    ids, weights, err = moe_ref.route(X, R, k)
    clean, _, _, _ = emulate(emu, X, W1, W2, ids, weights, grid)
    e = int(ids[0, 0])
    W2[e, 3, F // 2] = float("inf")
    W2[e, D - 1, 0] = float("nan")
    W2[e, 17, 5], W2[e, 17, 40] = float("inf"), float("-inf")
    Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, grid)
    assert findings == 0 and st[0] == 0, (msg, st)
    assert torch.isnan(Y[T:]).all()
    check_w2(Y[:T], clean[:T], X, ids, weights, err, W1, W2, [3, D - 1, 17])


def test_a_chosen_expert_whose_weight_underflowed_still_passes_nan_on(emu):
    """p = 0 of an expert that was chosen (a softmax weight below fp32) is a factor, 0 x NaN; of one that was not, no term."""
    X, R, W1, W2 = inputs(5, 4, 128, 64, torch.bfloat16, 15)
    ids = torch.tensor([[0, 1], [0, 2], [1, 2], [3, 2], [2, 0]])
    weights = torch.tensor([[1.0, 0.0], [1.0, 0.0], [0.5, 0.5], [1.0, 0.0], [0.25, 0.75]])
    want, _, _, _ = emulate(emu, X, W1, W2, ids, weights, 3)
    W1[1, 7] = float("nan")
    Y, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, 3)
    assert findings == 0 and st[0] == 0, (msg, st)
    assert torch.isnan(Y[[0, 2]]).all() and torch.equal(Y[[1, 3, 4]], want[[1, 3, 4]])


@pytest.mark.parametrize("what,D,grid,role,kind", [("drop_bulk", 512, 1, 1, 12), ("drop_red", 64, 4, 3, 10),
                                                   ("drop_atom", 64, 4, 2, 11)])
def test_a_stall_is_recorded_where_it_was_seen(emu, what, D, grid, role, kind):
    """A stage's tokens that never land (one block, more stages than its ring holds), a gate/up tile that is never counted, a
    part of a split down tile that is never counted (D = 64: no gate/up tile is split): the wait that gave up first is in the
    status word, and every block leaves."""
    X, R, W1, W2 = inputs(2, 4, D, 256, torch.float16, 16)
    ids, weights, _ = moe_ref.route(X, R, 2)
    emu.bw_emu_moe_set(b"first_kind", ctypes.c_longlong(kind))
    emu.bw_emu_moe_set(b"wait_ns", ctypes.c_longlong(1_000_000_000))
    emu.bw_emu_moe_set(what.encode(), ctypes.c_longlong(1))
    try:
        _, st, findings, msg = emulate(emu, X, W1, W2, ids, weights, grid)
    finally:
        emu.bw_emu_moe_set(b"first_kind", ctypes.c_longlong(-1))
        emu.bw_emu_moe_set(b"wait_ns", ctypes.c_longlong(60_000_000_000))
        emu.bw_emu_moe_set(what.encode(), ctypes.c_longlong(-1))
    assert findings == 0, msg
    assert st[0] == 3 and st[1] >> 8 == role << 8 | kind, [hex(v) for v in st]
