"""GPU: the tile kernels of the dense operators, by sizes that provably take them (captured.py), against the formulas in 64 bits
with the tolerances that test_gpu_dense.py derives: every storage of the operands and every tile shape, whole and cut, with
reductions that end inside a step, padded and offset rows, and rows beyond 32 bits."""
import re

import pytest
import torch

from captured import kernels_of
from test_gpu_dense import (D, TYPES, check_backward, check_forward, check_gated, check_gated_backward, close, matrix, product_tol, run_backward,
                            run_forward)

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
    ("f32", 245, 1497, 625, ("st", 128, 128, True)), ("f32", 133, 301, 4483, ("tt", 128, 128, False)), ("f32", 2489, 71, 1797, ("tt", 128, 128, True)),
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


@pytest.mark.parametrize("n,ic,oc,tile", [(1500, 777, 777, ("ss", 128, 128, True)), (4100, 517, 517, ("ss", 128, 128, False)), (4097, 1003, 1003, ("ss", 256, 128, True))])
def test_fp32_tile_products_with_an_identity_are_exact(n, ic, oc, tile):
    """X I = X bit for bit: all 24 bits of an operand pass the split, also at the ends of the range."""
    taken_by = taken("f32", "forward", n, ic, oc)
    assert any(t[0] == "ss" for t in taken_by), taken_by
    x = matrix(n, ic, torch.float32, 9)
    x[0, :8] = torch.tensor([3.4e38, -3.4028234e38, 3.39e38, 1e-30, -1.1754944e-38, 0.0, 1 + 2.0 ** -23, 2.0 ** 100 * (1 + 2.0 ** -20)])
    y, _ = run_forward("f32", x, torch.eye(ic, device="cuda"), None, 0, None, False)
    assert torch.equal(y, x)


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
