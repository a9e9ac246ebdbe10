"""GPU: the tile kernels of the dense operators, by sizes that provably take them (captured.py), against the formulas in 64 bits
with the tolerances that test_gpu_dense.py derives: every storage of the operands and every tile shape, whole and cut, with
reductions that end inside a step, padded and offset rows, rows beyond 32 bits, infinities and NaN."""
import math
import re

import pytest
import torch

from captured import kernels_of
from test_gpu_dense import (D, TYPES, act64, check_backward, check_forward, check_gated, check_gated_backward, close, matrix, product_tol, run_backward,
                            run_forward, run_gated, run_gated_backward, slope64)

pytestmark = pytest.mark.gpu
NAMES = {"f32": "dense_tile_f32_kernel", "bf16": "dense_tile_kernel"}
STORAGE = {"ss": "false, false", "st": "false, true", "tt": "true, true"}


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    torch.cuda.set_device(0)


def kernels(kind, op, n, ic, oc):
    """The kernels of one dense call of these sizes (SiLU; every output wanted)."""
    code, dtype = TYPES[kind]

    def e(*shape):
        return torch.empty(shape, dtype=dtype, device="cuda")
    x, wg, wu, a, b, c, dx, dwg, dwu, db, dbu = e(n, ic), e(oc, ic), e(oc, ic), e(n, oc), e(n, oc), e(n, oc), e(n, ic), e(oc, ic), e(oc, ic), e(oc), e(oc)
    query = {"forward": D.matMul_fused_workspace, "gated": D.gatedMatMul_workspace, "backward": D.dmatMul_fused_workspace, "gated_backward": D.dgatedMatMul_workspace}[op]
    size = query(code, n, ic, oc)
    ws = torch.empty(max(size, 256), dtype=torch.uint8, device="cuda")
    p = torch.Tensor.data_ptr
    calls = {
        "forward": lambda s: D.matMul_fused([s], 1, code, p(x), ic, p(wg), ic, 0, D.ACT_SILU, 0.0, 0, 0, 0, 0, p(a), oc, n, ic, oc, p(ws), size),
        "gated": lambda s: D.gatedMatMul([s], 1, code, p(x), ic, p(wg), ic, 0, p(wu), ic, 0, D.ACT_SILU, 0.0, 0, 0, 0, 0, p(a), oc, n, ic, oc, p(ws), size),
        "backward": lambda s: D.dmatMul_fused([s], 1, code, p(a), oc, p(b), oc, D.ACT_SILU, 0.0, p(x), ic, p(wg), ic, p(dx), ic, p(dwg), ic, p(db), n, ic, oc,
                                              p(ws), size),
        "gated_backward": lambda s: D.dgatedMatMul([s], 1, code, p(a), oc, p(b), oc, p(c), oc, D.ACT_SILU, 0.0, p(x), ic, p(wg), ic, p(wu), ic, p(dx), ic,
                                                   p(dwg), ic, p(dwu), ic, p(db), p(dbu), n, ic, oc, p(ws), size),
    }
    return kernels_of(calls[op])


def taken(kind, op, n, ic, oc):
    """{(storage, rows, columns of the tile, cut)} of a call's tile kernels; `cut`: their pieces are joined by the next kernel."""
    found, names = set(), [k for k, _ in kernels(kind, op, n, ic, oc)]
    for i, k in enumerate(names):
        m = re.search(NAMES[kind] + r"<(\w+, \w+), \w+, (\d+), (\d+)", k)
        if m:
            storage = {v: key for key, v in STORAGE.items()}[m.group(1)]
            found.add((storage, int(m.group(2)), int(m.group(3)), i + 1 < len(names) and "dense_pieces_kernel" in names[i + 1]))
    return found


def must_take(kind, op, n, ic, oc, *want):
    got = taken(kind, op, n, ic, oc)
    assert set(want) <= got, "%s takes %s" % ((kind, op, n, ic, oc), sorted(got))


# ---- values ----------------------------------------------------------------------------------------------------------
# kind, sizes, the tile (storage, rows, columns, cut) that it is about
FORWARD = [
    ("f32", 4745, 49, 537, ("ss", 128, 128, False)), ("f32", 777, 3001, 1025, ("ss", 128, 128, True)),
    ("f32", 1615, 121, 2953, ("ss", 256, 128, False)), ("f32", 4100, 517, 4097, ("ss", 256, 128, True)),
    ("bf16", 1500, 777, 1300, ("ss", 128, 128, False)), ("bf16", 777, 3001, 1025, ("ss", 128, 128, True)), ("bf16", 777, 3000, 1025, ("ss", 128, 128, True)),
    ("bf16", 4037, 1421, 1105, ("ss", 256, 128, False)), ("bf16", 3457, 5288, 635, ("ss", 256, 128, True)),
    ("bf16", 4183, 104, 2097, ("ss", 256, 256, False)), ("bf16", 5000, 2001, 5001, ("ss", 256, 256, False)),
]
GATED = [
    ("f32", 5245, 97, 277, ("ss", 128, 128, False)), ("f32", 115, 1703, 1381, ("ss", 128, 128, True)),
    ("f32", 2001, 515, 2001, ("ss", 256, 128, False)), ("f32", 2711, 381, 3013, ("ss", 256, 128, True)),
    ("bf16", 1500, 777, 1300, ("ss", 128, 128, False)), ("bf16", 77, 4051, 2971, ("ss", 128, 128, True)), ("bf16", 2418, 2840, 1449, ("ss", 256, 128, False)),
    ("bf16", 3377, 93, 1671, ("ss", 256, 256, False)), ("bf16", 5379, 1549, 3103, ("ss", 256, 256, True)),
]
BACKWARD = [
    ("f32", 3597, 4385, 169, ("st", 128, 128, False)), ("f32", 1500, 777, 1300, ("st", 128, 128, True), ("tt", 128, 128, True)),
    ("f32", 2715, 2313, 41, ("st", 256, 128, False)), ("f32", 2049, 1001, 2050, ("st", 256, 128, True), ("tt", 256, 128, True)),
    ("f32", 777, 3001, 1025, ("tt", 128, 128, False)), ("f32", 53, 1271, 3239, ("tt", 256, 128, False)),
    ("bf16", 2049, 1001, 2050, ("st", 128, 128, False), ("tt", 128, 128, False)), ("bf16", 231, 592, 4576, ("st", 128, 128, True)),
    ("bf16", 2319, 2465, 3649, ("st", 256, 128, False)), ("bf16", 2001, 515, 2001, ("tt", 128, 128, True)),
    ("bf16", 5000, 2001, 5001, ("st", 256, 256, False), ("tt", 256, 256, False)),
]
GATED_BACKWARD = [
    ("f32", 3587, 2995, 39, ("st", 128, 128, False)), ("f32", 245, 1497, 625, ("st", 128, 128, True)), ("f32", 133, 301, 4483, ("tt", 128, 128, False)), ("f32", 2489, 71, 1797, ("tt", 128, 128, True)),
    ("f32", 2149, 491, 4585, ("st", 256, 128, True)), ("f32", 2001, 515, 2001, ("tt", 256, 128, True)), ("f32", 75, 1841, 1177, ("tt", 256, 128, False)),
    ("bf16", 1500, 777, 1300, ("st", 128, 128, True)), ("bf16", 2481, 599, 3875, ("st", 256, 128, True)), ("bf16", 4873, 2199, 311, ("st", 256, 256, False)),
    ("bf16", 678, 3609, 4841, ("st", 256, 256, True)), ("bf16", 4001, 24, 4007, ("tt", 128, 128, True)), ("bf16", 851, 673, 2753, ("tt", 256, 128, False)),
    ("bf16", 165, 4901, 2601, ("tt", 256, 256, False)), ("bf16", 5001, 2001, 5001, ("tt", 256, 256, True)),
]
ROWS = [(0, 0), (3, 1), (8, 8)]      # pad and offset in elements


@pytest.mark.parametrize("case", FORWARD, ids=str)
@pytest.mark.parametrize("pad,offset", ROWS)
def test_forward_tiles(case, pad, offset):
    kind, n, ic, oc, *want = case
    must_take(kind, "forward", n, ic, oc, *want)
    check_forward(kind, n, ic, oc, act=D.ACT_SILU, bias=True, residual=True, save=True, pad=pad, offset=offset)


@pytest.mark.parametrize("case", GATED, ids=str)
@pytest.mark.parametrize("pad,offset,wu_pad", [(0, 0, 0), (3, 1, 3), (8, 8, 16)])
def test_gated_tiles(case, pad, offset, wu_pad):
    kind, n, ic, oc, *want = case
    must_take(kind, "gated", n, ic, oc, *want)
    check_gated(kind, n, ic, oc, pad=pad, offset=offset, wu_pad=wu_pad)


@pytest.mark.parametrize("case", BACKWARD, ids=str)
@pytest.mark.parametrize("pad,offset", ROWS)
def test_backward_tiles(case, pad, offset):
    kind, n, ic, oc, *want = case
    must_take(kind, "backward", n, ic, oc, *want)
    check_backward(kind, n, ic, oc, act=D.ACT_SILU, pad=pad, offset=offset)
    check_backward(kind, n, ic, oc, act=D.ACT_NONE, want=("dx", "dw"), pad=pad, offset=offset)


@pytest.mark.parametrize("case", GATED_BACKWARD, ids=str)
@pytest.mark.parametrize("pad,offset,wu_pad", [(0, 0, 0), (3, 1, 3), (8, 8, 16)])
def test_gated_backward_tiles(case, pad, offset, wu_pad):
    kind, n, ic, oc, *want = case
    must_take(kind, "gated_backward", n, ic, oc, *want)
    check_gated_backward(kind, n, ic, oc, pad=pad, offset=offset, wu_pad=wu_pad)


@pytest.mark.parametrize("ic", [8, 16, 24, 32, 40])
@pytest.mark.parametrize("pad", [0, 8])
def test_rows_closer_than_a_step(ic, pad):
    """bf16 rows of 8 to 40 elements, read in place, and a tile that has fewer rows than it could."""
    for n, oc in ((4001, 4007), (4225, 4129)):
        assert any(t[0] == "ss" for t in taken("bf16", "forward", n, ic, oc)) and any(t[0] == "ss" for t in taken("bf16", "gated", n, ic, oc))
        check_forward("bf16", n, ic, oc, pad=pad)
        check_gated("bf16", n, ic, oc, pad=pad)


@pytest.mark.parametrize("n,ic", [(1500, 777), (4100, 517), (4097, 1003)])
def test_fp32_tile_products_with_an_identity_are_exact(n, ic):
    """X I = X and I X^T = X^T bit for bit: all 24 bits of an operand pass the split, also at the ends of the range."""
    for rows, columns in ((n, ic), (ic, n)):
        got = taken("f32", "forward", rows, ic, columns)
        assert any(t[0] == "ss" for t in got), (rows, ic, columns)
    x = matrix(n, ic, torch.float32, 9)
    x[0, :8] = torch.tensor([3.4e38, -3.4028234e38, 3.39e38, 1e-30, -1.1754944e-38, 0.0, 1 + 2.0 ** -23, 2.0 ** 100 * (1 + 2.0 ** -20)])
    eye = torch.eye(ic, device="cuda")
    y, _ = run_forward("f32", x, eye, None, 0, None, False)
    assert torch.equal(y, x)
    y, _ = run_forward("f32", eye, x, None, 0, None, False)
    assert torch.equal(y, x.t())


@pytest.mark.parametrize("exponent", [-100, -109, -110, -111, -113, -116, -120, -126])
def test_fp32_tile_products_of_small_operands(exponent):
    """All bits of an operand of 2^-110 and more; below, what is left of it behind three bf16 parts is at most half of the last
    subnormal, 2^-134. (The other operand is a power of two, so the product adds nothing.)"""
    n, ic = 4097, 1003
    must_take("f32", "forward", n, ic, ic, ("ss", 128, 128, True))
    x = matrix(n, ic, torch.float32, 9)
    x = (1 + x.abs().clamp(max=0.999)) * 2.0 ** exponent
    y, _ = run_forward("f32", x, torch.eye(ic, device="cuda") * 2.0 ** 100, None, 0, None, False)
    off = (y.double() * 2.0 ** -100 - x.double()).abs().max()
    assert float(off) <= (0.0 if exponent >= -110 else 2.0 ** -134)


# ---- rows beyond 32 bits ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", TYPES)
def test_rows_of_the_largest_stride(kind):
    """Rows 2^22 elements apart: a tile's descriptor covers up to 2^31 (bf16) and 2^32 bytes (fp32), and the operands 12 to 25 GB."""
    dtype = TYPES[kind][1]
    n, ic, oc, far = 1500, 776, 1304, 1 << 22
    must_take(kind, "forward", n, ic, oc, ("ss", 128, 128, False))
    assert {t[0] for t in taken(kind, "backward", n, ic, oc)} >= ({"st", "tt"} if kind == "f32" else set())

    def wide(rows, cols, seed, std=1.0):
        flat = torch.empty((rows - 1) * far + cols, dtype=dtype, device="cuda")
        v = flat.as_strided((rows, cols), (far, 1))
        v.copy_(matrix(rows, cols, dtype, seed, std))
        return v
    x, w = wide(n, ic, 1), wide(oc, ic, 2, ic ** -0.5)
    x64, w64 = x.double(), w.double()
    y, _ = run_forward(kind, x, w, None, 0, None, False)
    close(y, x64 @ w64.t(), product_tol(x64, w64, dtype), "far rows")
    dy = wide(n, oc, 3)
    got = run_backward(kind, dy, None, D.ACT_NONE, x, w, ("dx", "dw"))
    dy64 = dy.double()
    close(got["dx"], dy64 @ w64, product_tol(dy64, w64.t(), dtype), "far rows dx")
    close(got["dw"], dy64.t() @ x64, product_tol(dy64.t(), x64.t(), dtype), "far rows dw")


# ---- infinities and NaN ----------------------------------------------------------------------------------------------
INF, NAN = float("inf"), float("nan")


def spoil(t, places):
    for (r, c), v in places.items():
        t[r % t.shape[0], c % t.shape[1]] = v


def same_pattern(got, want, what):
    """Infinities and NaN where the formula has them, of the same sign."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want)), what


def finite_part(got, want, tol, what):
    fine = torch.isfinite(want)
    zero = torch.zeros((), dtype=want.dtype, device=want.device)
    close(torch.where(fine, got, zero.to(got.dtype)), torch.where(fine, want, zero), tol, what)


def tame(t):
    return torch.where(torch.isfinite(t), t, torch.zeros_like(t)).double()


def clamped(t):
    """Sums beyond fp32 are infinite in fp32."""
    top = torch.finfo(torch.float32).max
    return torch.where(t.abs() > top, torch.sign(t) * INF, t)


X_PLACES = {(1, 7): INF, (2, 11): NAN, (3, 12): INF, (3, 13): INF, (-1, -1): -INF, (40, 30): -INF, (41, 9): INF, (130, 0): NAN}
W_PLACES = {(3, 7): 0.0, (5, 9): -INF, (-1, -2): INF, (70, 12): 0.0, (71, 13): -INF, (-2, 30): 0.0}


@pytest.mark.parametrize("case", [c for c in FORWARD if c[1] * c[2] * c[3] < 5e9], ids=str)
def test_forward_tiles_with_infinities_and_nans(case):
    kind, n, ic, oc, *want = case
    must_take(kind, "forward", n, ic, oc, *want)
    x, w = matrix(n, ic, TYPES[kind][1], 1, pad=3), matrix(oc, ic, TYPES[kind][1], 2, 0.1, pad=1)
    spoil(x, X_PLACES)
    spoil(w, W_PLACES)
    if kind == "f32":     # near the end of the range: rounded up to bf16 these are infinite, and products of parts overflow
        x[4, 20], x[6, :], w[8, 31] = 3.4e38, 0.0, 2.0 ** 63
        x[6, 31] = 1.998 * 2.0 ** 64
        w[:, 20].clamp_(-0.5, 0.5)
    y, _ = run_forward(kind, x, w, None, 0, None, False)
    exact = x.double() @ w.double().t()
    if kind == "f32":
        exact = clamped(exact)
        assert float(y[6, 8]) == float(x[6, 31]) * 2.0 ** 63
    same_pattern(y, exact, case)
    finite_part(y, exact, product_tol(tame(x), tame(w), TYPES[kind][1]), case)


@pytest.mark.parametrize("case", [c for c in GATED if c[1] * c[2] * c[3] < 5e9 and c[0] == "f32"], ids=str)
def test_gated_tiles_with_infinities_and_nans(case):
    kind, n, ic, oc, *want = case
    must_take(kind, "gated", n, ic, oc, *want)
    x, wg, wu = matrix(n, ic, torch.float32, 1, pad=3), matrix(oc, ic, torch.float32, 2, 0.1, pad=1), matrix(oc, ic, torch.float32, 3, 0.1, pad=1)
    spoil(x, {k: v for k, v in X_PLACES.items() if not math.isnan(v)})
    x[9, 5] = NAN
    spoil(wg, W_PLACES)
    spoil(wu, {(17, 3): INF, (-1, 7): 0.0})
    h, g, u = run_gated(kind, x, wg, wu, None, None, D.ACT_LEAKY_RELU, "gu")
    g64, u64 = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    for name, got, exact in (("G", g, g64), ("U", u, u64), ("H", h, act64(D.ACT_LEAKY_RELU, g64) * u64)):
        same_pattern(got, exact, (name, case))
    finite_part(g, g64, product_tol(tame(x), tame(wg), torch.float32), case)
    finite_part(u, u64, product_tol(tame(x), tame(wu), torch.float32), case)


DY_PLACES = {(1, 7): INF, (2, 11): NAN, (3, 12): INF, (3, 13): -INF, (-1, -1): -INF, (33, 30): INF}


@pytest.mark.parametrize("case", [c for c in BACKWARD if c[1] * c[2] * c[3] < 5e9 and c[0] == "f32"], ids=str)
@pytest.mark.parametrize("act", [D.ACT_NONE, D.ACT_LEAKY_RELU])
def test_backward_tiles_with_infinities_and_nans(case, act):
    kind, n, ic, oc, *want = case
    must_take(kind, "backward", n, ic, oc, *want)
    x, w, dy = matrix(n, ic, torch.float32, 1, pad=3), matrix(oc, ic, torch.float32, 2, 0.1, pad=1), matrix(n, oc, torch.float32, 3, pad=5)
    z = matrix(n, oc, torch.float32, 4) if act != D.ACT_NONE else None
    spoil(dy, DY_PLACES)
    spoil(x, {(1, 5): 0.0, (3, 8): INF, (-1, -1): 0.0, (29, 6): -INF})
    spoil(w, {(7, 2): 0.0, (12, 4): -INF, (-1, -1): INF, (30, 3): 0.0})
    got = run_backward(kind, dy, z, act, x, w)
    dz = dy.double() if z is None else dy.double() * slope64(act, z.double())
    sums = {"dx": (dz, w.double().t()), "dw": (dz.t(), x.double().t())}
    for name, (a, b) in sums.items():
        exact = a @ b.t()
        same_pattern(got[name], exact, (name, case))
        finite_part(got[name], exact, product_tol(tame(a), tame(b), torch.float32) + 2.0 ** -21 * (tame(a).abs() @ tame(b).abs().t()), (name, case))
    same_pattern(got["db"], dz.sum(0, keepdim=True), ("db", case))


@pytest.mark.parametrize("case", [c for c in GATED_BACKWARD if c[1] * c[2] * c[3] < 5e9 and c[0] == "f32"], ids=str)
def test_gated_backward_tiles_with_infinities_and_nans(case):
    """Two sources (deltaX), stacked results with rows between them that belong to neither (deltaWg, deltaWu)."""
    kind, n, ic, oc, *want = case
    must_take(kind, "gated_backward", n, ic, oc, *want)
    x, wg, wu = matrix(n, ic, torch.float32, 1, pad=3), matrix(oc, ic, torch.float32, 2, 0.1, pad=1), matrix(oc, ic, torch.float32, 3, 0.1, pad=1)
    dh, g, u = (matrix(n, oc, torch.float32, 4 + i, pad=5) for i in range(3))
    spoil(dh, DY_PLACES)
    spoil(x, {(1, 5): 0.0, (3, 8): INF, (-1, -1): 0.0, (29, 6): -INF})
    spoil(wg, {(7, 2): 0.0, (12, 4): -INF, (30, 3): 0.0})
    spoil(wu, {(7, 6): 0.0, (-1, -1): INF})
    u[33, 30] = 0.0
    got = run_gated_backward(kind, dh, g, u, D.ACT_LEAKY_RELU, x, wg, wu, ("dx", "dwg", "dwu", "dbg", "dbu"))
    dg, du = dh.double() * u.double() * slope64(D.ACT_LEAKY_RELU, g.double()), dh.double() * act64(D.ACT_LEAKY_RELU, g.double())
    sums = {"dx": (torch.cat([dg, du], 1), torch.cat([wg, wu]).double().t()), "dwg": (dg.t(), x.double().t()), "dwu": (du.t(), x.double().t())}
    for name, (a, b) in sums.items():
        exact = a @ b.t()
        same_pattern(got[name], exact, (name, case))
        finite_part(got[name], exact, product_tol(tame(a), tame(b), torch.float32) + 2.0 ** -21 * (tame(a).abs() @ tame(b).abs().t()), (name, case))
    for name, d in (("dbg", dg), ("dbu", du)):
        same_pattern(got[name], d.sum(0, keepdim=True), (name, case))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,ic,oc", [(1, 40, 56), (5, 9, 33), (70, 137, 73), (300, 33, 9), (2, 5, 4099), (4416, 33, 35), (2319, 2465, 521)])
@pytest.mark.parametrize("act", [D.ACT_NONE, D.ACT_LEAKY_RELU])
def test_backward_of_any_form_with_infinities_and_nans(kind, n, ic, oc, act):
    """Small products straight from memory, long sums cut over workgroups, bf16 tiles."""
    dtype = TYPES[kind][1]
    x, w, dy = matrix(n, ic, dtype, 1, pad=3), matrix(oc, ic, dtype, 2, 0.1, pad=1), matrix(n, oc, dtype, 3, pad=5)
    z = matrix(n, oc, dtype, 4) if act != D.ACT_NONE else None
    dy[n // 2, oc // 3], dy[n - 1, oc - 1], dy[n // 3, 0] = INF, -INF, NAN
    x[n // 2, ic // 2], x[n - 1, ic - 1] = 0.0, INF
    w[oc // 3, ic // 3], w[oc // 2, 0], w[oc - 1, ic - 1] = 0.0, -INF, INF
    got = run_backward(kind, dy, z, act, x, w)
    dz = dy.double() if z is None else dy.double() * slope64(act, z.double())
    same_pattern(got["dx"], dz @ w.double(), "dx")
    same_pattern(got["dw"], dz.t() @ x.double(), "dw")
    same_pattern(got["db"], dz.sum(0, keepdim=True), "db")


def _us(call):
    times = []
    for _ in range(5):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        call()
        end.record()
        torch.cuda.synchronize()
        times.append(1000 * begin.elapsed_time(end))
    return sorted(times)[2]


def test_infinities_cost_a_bounded_factor():
    """What is not finite is computed again, by all wavefronts side by side: one infinite sample, or nothing but NaN, costs a small
    multiple of the call (an element at a time by one lane it would be hundreds)."""
    n, ic, oc = 12544, 256, 1024
    x, w, dy = matrix(n, ic, torch.float32, 1), matrix(oc, ic, torch.float32, 2, 0.1), matrix(n, oc, torch.float32, 3)
    y, dx, dw = torch.empty(n, oc, device="cuda"), torch.empty(n, ic, device="cuda"), torch.empty(oc, ic, device="cuda")
    size = max(D.matMul_fused_workspace(D.F32, n, ic, oc), D.dmatMul_fused_workspace(D.F32, n, ic, oc))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    s = [int(torch.cuda.current_stream().cuda_stream)]

    def forward():
        D.matMul_fused(s, 1, D.F32, x.data_ptr(), ic, w.data_ptr(), ic, 0, 0, 0.0, 0, 0, 0, 0, y.data_ptr(), oc, n, ic, oc, ws.data_ptr(), size)

    def backward():
        D.dmatMul_fused(s, 1, D.F32, dy.data_ptr(), oc, 0, 0, 0, 0.0, x.data_ptr(), ic, w.data_ptr(), ic, dx.data_ptr(), ic, dw.data_ptr(), ic, 0, n, ic, oc,
                        ws.data_ptr(), size)
    for call in (forward, backward):
        call()
        usual = _us(call)
        keep = dy[5, 9].item(), x[5, 9].item()
        dy[5, 9], x[5, 9] = INF, INF
        one = _us(call)
        dy[5, 9], x[5, 9] = keep
        x0, dy0 = x.clone(), dy.clone()
        x.fill_(INF)
        dy.fill_(INF)
        every = _us(call)
        x.copy_(x0)
        dy.copy_(dy0)
        print("%s: %.0f us, one infinity %.0f, all infinite %.0f" % (call.__name__, usual, one, every), flush=True)
        assert one <= 12 * usual and every <= 12 * usual
