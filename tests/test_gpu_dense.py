"""GPU: the dense operators (include/alpha_dense.h) against their formulas in 64 bits.

Tolerances, per element, from the arithmetic:
* the output's rounding: eps / 2 relative (bf16 2^-8, fp32 2^-24);
* a sum of K products with terms of rms t: S = sqrt(sum of squares of the terms). Roundings of the fp32 partial sums are
  independent, at most 2^-24 (nearest) or 2^-23 (cut off) of a partial sum of a few S; 16 sqrt(K + 64) 2^-23 S covers six
  sigmas of them. fp32 products leave out parts below 2^-23 of a product each: 8 * 2^-23 S;
* bf16 backward: deltaZ rounded to bf16 before its products, 2^-8 relative per term, independent: six sigmas of a uniform
  error, 6 / sqrt(3) 2^-8 S;
* activations: exponentials and erf good to a few units of 2^-24, so 2^-20 of max(1, |z|) absolute; the product's own error
  passes with a slope <= 1.2. Their derivatives are sums of terms of at most max(1, |z|) that may cancel (SiLU's
  s (1 + z (1 - s)) at z = -1.28), so what they are off by is absolute as well: 2^-21 max(1, |z|), times the factors beside
  them, and as much as that of every term of a sum over deltaZ;
A wrong part, tap, tail or index is orders above these (half the terms of a sum missing is an error of S)."""
import math

import numpy as np
import pytest
import torch

from util import load_package

pytestmark = pytest.mark.gpu
pkg = load_package()
D = pkg.Cuda_dense
TYPES = {"f32": (D.F32, torch.float32), "bf16": (D.BF16, torch.bfloat16)}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SLOPE = 0.1
GUARD = 4096


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    torch.cuda.set_device(0)


def stream():
    return [int(torch.cuda.current_stream().cuda_stream)]


def matrix(rows, cols, dtype, seed, std=1.0, pad=0, offset=0):
    """[rows, cols] whose rows are cols + pad apart and whose first element is `offset` elements behind an aligned address;
    the gaps hold NaN, which no result may show."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    stride = max(1, cols + pad)
    flat = torch.full((offset + rows * stride + 8,), float("nan"), dtype=dtype, device="cuda")
    view = flat[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    view.copy_(torch.randn(rows, cols, generator=g, device="cuda") * std)
    return view


class Out:
    """An output [rows, cols] with a row stride, filled with NaN, between guard bands; `get` checks bands and gaps."""

    def __init__(self, rows, cols, dtype, pad=0, offset=0):
        self.rows, self.cols, self.stride = rows, cols, max(1, cols + pad)
        n = rows * self.stride
        self.flat = torch.full((GUARD + offset + n + GUARD,), 7.0, dtype=dtype, device="cuda")
        self.view = self.flat[GUARD + offset:GUARD + offset + n].view(rows, self.stride)[:, :cols]
        self.view.fill_(float("nan"))

    def ptr(self):
        return self.view.data_ptr()

    def get(self):
        torch.cuda.synchronize()
        got = self.view.clone()
        self.view.fill_(7.0)
        assert bool((self.flat == 7.0).all()), "written outside the output"
        self.view.copy_(got)
        return got


def workspace(query, *args):
    n = query(*args)
    return torch.full((max(n, 256),), 0xA5, dtype=torch.uint8, device="cuda"), n


def act64(act, z):
    if act == D.ACT_NONE:
        return z
    if act == D.ACT_LEAKY_RELU:
        return torch.where(z > 0, z, z * SLOPE)
    if act == D.ACT_GELU:
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    return z * torch.sigmoid(z) if act == D.ACT_SILU else torch.sigmoid(z)


def slope64(act, z):
    if act == D.ACT_NONE:
        return torch.ones_like(z)
    if act == D.ACT_LEAKY_RELU:
        return torch.where(z > 0, 1.0, SLOPE).to(z.dtype)
    if act == D.ACT_GELU:
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * torch.sigmoid(-z)) if act == D.ACT_SILU else s * torch.sigmoid(-z)


def product_tol(a, b, dtype, extra=0.0):
    """Allowed error of a @ b^T (fp64 operands) before the output's rounding."""
    S = (a.square() @ b.square().t()).sqrt()
    k = 16 * math.sqrt(a.shape[1] + 64) * 2.0 ** -23 + extra
    if dtype == torch.float32:
        k += 8 * 2.0 ** -23
    return S * k


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    allowed = tol + HALF[got.dtype] * want.abs() * 1.01 + 1e-37
    bad = ~(err <= allowed)
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d off, first at %s: got %r, want %r, allowed %.3g" % (
            what, int(bad.sum()), bad.numel(), i, float(got[i]), float(want[i]), float(allowed[i])))


def run_forward(kind, x, w, bias, act, r, save, ypad=0, yoffset=0, in_place=False, ws=None):
    code, dtype = TYPES[kind]
    (n, ic), oc = x.shape, w.shape[0]
    y, z = Out(n, oc, dtype, ypad, yoffset), Out(n, oc, dtype, ypad) if save else None
    if in_place:
        y.view.copy_(r)
        r = y.view
    ws, size = ws or workspace(D.matMul_fused_workspace, code, n, ic, oc)
    D.matMul_fused(stream(), 1, code, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), 0 if bias is None else bias.data_ptr(), act, SLOPE,
                   0 if r is None else r.data_ptr(), 0 if r is None else r.stride(0), z.ptr() if save else 0, z.stride if save else 0,
                   y.ptr(), y.stride, n, ic, oc, ws.data_ptr(), size)
    return y.get(), z.get() if save else None


def check_forward(kind, n, ic, oc, act=0, bias=True, residual=False, save=False, pad=0, offset=0, in_place=False, seed=1):
    dtype = TYPES[kind][1]
    x, w = matrix(n, ic, dtype, seed, pad=pad, offset=offset), matrix(oc, ic, dtype, seed + 1, max(1, ic) ** -0.5, pad=pad, offset=offset)
    b = matrix(1, oc, dtype, seed + 2)[0] if bias else None
    r = matrix(n, oc, dtype, seed + 3, pad=pad) if residual else None
    r64 = r.double().clone() if residual else None
    y, z = run_forward(kind, x, w, b, act, r, save, pad, offset, in_place)
    z64 = x.double() @ w.double().t()
    tol = product_tol(x.double(), w.double(), dtype)
    if bias:
        z64 = z64 + b.double()
    tol = tol + 2.0 ** -23 * z64.abs()
    if save:
        close(z, z64, tol, "Z %s" % ((kind, n, ic, oc),))
    y64 = act64(act, z64)
    tol = 1.2 * tol + 2.0 ** -20 * z64.abs().clamp(min=1.0)
    if residual:
        y64 = y64 + r64
        tol = tol + 2.0 ** -23 * y64.abs()
    close(y, y64, tol, "Y %s" % ((kind, n, ic, oc, act),))


# rows, reduced features, produced features: one of everything, odd sizes, tails of every tile edge (16, 64, 128, 256), few rows
SIZES = [(1, 1, 1), (1, 64, 64), (2, 33, 17), (3, 8, 1000), (5, 200, 7), (16, 256, 96), (17, 130, 100), (33, 72, 200), (64, 512, 1000),
         (65, 64, 65), (127, 65, 129), (129, 257, 300), (200, 1000, 131), (255, 128, 257), (257, 1, 255), (300, 63, 520), (512, 2048, 136)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_forward_sizes(kind, size):
    check_forward(kind, *size, bias=True, save=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(1, 100, 40), (30, 136, 72), (300, 136, 264)])
@pytest.mark.parametrize("act", range(5))
def test_forward_epilogues(kind, size, act):
    check_forward(kind, *size, act=act, bias=True, residual=True, save=True)
    check_forward(kind, *size, act=act, bias=False, residual=False, save=False, seed=20)
    check_forward(kind, *size, act=act, bias=False, residual=True, in_place=True, seed=30)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(1, 96, 64), (20, 96, 64), (140, 96, 136)])
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 8), (40, 2)])
def test_forward_strides_and_alignments(kind, size, pad, offset):
    check_forward(kind, *size, act=D.ACT_SILU, bias=True, residual=True, save=True, pad=pad, offset=offset)


# both tile shapes and cut reductions, beyond one round of workgroups
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(2048, 1024, 2048), (4100, 192, 2056), (130, 8192, 136), (1030, 4096, 260), (24, 8200, 512)])
def test_forward_large(kind, size):
    check_forward(kind, *size, act=D.ACT_GELU, bias=True, residual=True, save=True)


def test_forward_row_offsets_beyond_32_bits():
    """Rows far apart: row 1100 of X begins 2^32 bytes (and more) behind row 0."""
    n, ic, oc, far = 1100, 64, 72, 1 << 21
    flat = torch.zeros((n - 1) * far + ic, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((n, ic), (far, 1))
    x.copy_(matrix(n, ic, torch.bfloat16, 5))
    w = matrix(oc, ic, torch.bfloat16, 6, 0.125)
    y, _ = run_forward("bf16", x, w, None, 0, None, False)
    x64 = x.double()
    close(y, x64 @ w.double().t(), product_tol(x64, w.double(), torch.bfloat16), "far rows")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("ic", [0])
def test_forward_of_an_empty_sum_is_the_bias(kind, ic):
    for n, oc in ((1, 8), (70, 130)):
        check_forward(kind, n, ic, oc, act=D.ACT_GELU, bias=True, residual=True, save=True)


@pytest.mark.parametrize("n", [3, 100, 600])
def test_fp32_products_with_an_identity_are_exact(n):
    """X I = X and I W^T = W^T bit for bit: all 24 bits of an operand pass, also at the ends of the range."""
    x = matrix(n, 96, torch.float32, 9)
    x[0, :8] = torch.tensor([3.4e38, -3.4028234e38, 3.39e38, 1e-30, -1.1754944e-38, 0.0, 1 + 2.0 ** -23, 2.0 ** 100 * (1 + 2.0 ** -20)])
    eye = torch.eye(96, device="cuda")
    y, _ = run_forward("f32", x, eye, None, 0, None, False)
    assert torch.equal(y, x)
    y, _ = run_forward("f32", eye, x, None, 0, None, False)
    assert torch.equal(y, x.t())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,ic,oc", [(4, 64, 64), (40, 200, 136), (300, 4096, 264)])
def test_forward_infinities_and_nans(kind, n, ic, oc):
    """As in plain arithmetic: inf * finite = inf of the product's sign, inf * 0 and inf - inf = NaN, NaN anywhere = NaN -
    in the rows and columns concerned and nowhere else."""
    dtype = TYPES[kind][1]
    x, w = matrix(n, ic, dtype, 1), matrix(oc, ic, dtype, 2)
    x[1, 7] = float("inf")
    w[3, 7] = 0.0
    w[5, 9] = float("-inf")
    x[2, 11] = float("nan")
    x[3, 12], x[3, 13] = float("inf"), float("inf")
    y, _ = run_forward(kind, x, w, None, 0, None, False)
    want = x.double() @ w.double().t()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isposinf(y), torch.isposinf(want)) and torch.equal(torch.isneginf(y), torch.isneginf(want))
    fine = torch.isfinite(want)
    z = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double(), torch.where(torch.isfinite(w), w, torch.zeros_like(w)).double()
    tol = product_tol(z[0], z[1], dtype)
    close(torch.where(fine, y, torch.zeros_like(y)), torch.where(fine, want, torch.zeros_like(want)), tol, "finite part")


# ---- backward --------------------------------------------------------------------------------------------------------

def run_backward(kind, dy, z, act, x, w, want=("dx", "dw", "db"), pad=0):
    code, dtype = TYPES[kind]
    (n, oc), ic = dy.shape, x.shape[1]
    out = {"dx": Out(n, ic, dtype, pad), "dw": Out(oc, ic, dtype, pad), "db": Out(1, oc, dtype)}
    ws, size = workspace(D.dmatMul_fused_workspace, code, n, ic, oc)

    def p(k):
        return out[k].ptr() if k in want else 0
    D.dmatMul_fused(stream(), 1, code, dy.data_ptr(), dy.stride(0), 0 if z is None else z.data_ptr(), 0 if z is None else z.stride(0), act, SLOPE,
                    x.data_ptr() if "dw" in want else 0, x.stride(0), w.data_ptr() if "dx" in want else 0, w.stride(0),
                    p("dx"), out["dx"].stride, p("dw"), out["dw"].stride, p("db"), n, ic, oc, ws.data_ptr(), size)
    return {k: out[k].get() for k in want}


def delta_error(act, factor, z):
    """What deltaZ = factor * act'(z) may be off by, in fp32 arithmetic (fp64 tensors): the derivative's and two roundings."""
    if act == D.ACT_NONE:
        return torch.zeros_like(factor)
    return factor.abs() * 2.0 ** -21 * z.abs().clamp(min=1.0)


ROUNDED = {"f32": 0.0, "bf16": 6 / math.sqrt(3) * 2.0 ** -8}      # deltaZ's rounding before its products


def check_sums(got, kind, name_w, name_b, dz, edz, x, what):
    """deltaW and deltaB of one pre-activation's gradient dz (fp64, unrounded), itself off by at most edz."""
    dtype = TYPES[kind][1]
    if name_w in got:
        close(got[name_w], dz.t() @ x, product_tol(dz.t(), x.t(), dtype, ROUNDED[kind]) + edz.t() @ x.abs(), what + name_w)
    if name_b in got:
        S = dz.square().sum(0, keepdim=True).sqrt()
        close(got[name_b], dz.sum(0, keepdim=True), S * (16 * math.sqrt(dz.shape[0] + 64) * 2.0 ** -23) + edz.sum(0, keepdim=True), what + name_b)


def check_backward(kind, n, ic, oc, act, want=("dx", "dw", "db"), pad=0, offset=0, seed=1):
    dtype = TYPES[kind][1]
    x, w = matrix(n, ic, dtype, seed, pad=pad, offset=offset), matrix(oc, ic, dtype, seed + 1, max(1, oc) ** -0.5, pad=pad, offset=offset)
    dy = matrix(n, oc, dtype, seed + 2, pad=pad, offset=offset)
    z = matrix(n, oc, dtype, seed + 3, pad=pad, offset=offset) if act != D.ACT_NONE else None
    got = run_backward(kind, dy, z, act, x, w, want, pad)
    dy64, z64, w64 = dy.double(), None if z is None else z.double(), w.double()
    dz = dy64 if z is None else dy64 * slope64(act, z64)
    edz = delta_error(act, dy64, z64)
    what = "%s " % ((kind, n, ic, oc, act),)
    check_sums(got, kind, "dw", "db", dz, edz, x.double(), what)
    if "dx" in want:
        close(got["dx"], dz @ w64, product_tol(dz, w64.t(), dtype, ROUNDED[kind]) + edz @ w64.abs(), what + "dx")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES + [(4100, 192, 264), (1024, 1024, 2048), (12544, 64, 72)])
def test_backward_sizes(kind, size):
    check_backward(kind, *size, act=D.ACT_GELU)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(1, 40, 56), (70, 136, 72)])
@pytest.mark.parametrize("act", range(5))
def test_backward_activations_and_wanted_outputs(kind, size, act):
    for want in (("dx", "dw", "db"), ("dx",), ("dw",), ("db",), ("dx", "db"), ("dw", "db")):
        check_backward(kind, *size, act=act, want=want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("act", [D.ACT_NONE, D.ACT_SILU])
def test_backward_strides_and_alignments(kind, pad, offset, act):
    check_backward(kind, 150, 104, 88, act=act, pad=pad, offset=offset)
    check_backward(kind, 9, 104, 88, act=act, pad=pad, offset=offset)


@pytest.mark.parametrize("kind", TYPES)
def test_backward_of_empty_batches_and_layers(kind):
    code, dtype = TYPES[kind]
    got = run_backward(kind, matrix(0, 24, dtype, 1), matrix(0, 24, dtype, 2), D.ACT_GELU, matrix(0, 40, dtype, 3), matrix(24, 40, dtype, 4))
    assert float(got["dw"].abs().sum()) == 0.0 and float(got["db"].abs().sum()) == 0.0
    got = run_backward(kind, matrix(24, 0, dtype, 1), matrix(24, 0, dtype, 2), D.ACT_GELU, matrix(24, 40, dtype, 3), matrix(0, 40, dtype, 4), want=("dx",))
    assert float(got["dx"].abs().sum()) == 0.0


# ---- gated pair ------------------------------------------------------------------------------------------------------

def run_gated(kind, x, wg, wu, bg, bu, act, save, pad=0):
    code, dtype = TYPES[kind]
    (n, ic), oc = x.shape, wg.shape[0]
    h = Out(n, oc, dtype, pad)
    g, u = (Out(n, oc, dtype, pad) if "g" in save else None), (Out(n, oc, dtype, pad) if "u" in save else None)
    ws, size = workspace(D.gatedMatMul_workspace, code, n, ic, oc)
    D.gatedMatMul(stream(), 1, code, x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), 0 if bg is None else bg.data_ptr(),
                  wu.data_ptr(), wu.stride(0), 0 if bu is None else bu.data_ptr(), act, SLOPE, g.ptr() if g else 0, g.stride if g else 0,
                  u.ptr() if u else 0, u.stride if u else 0, h.ptr(), h.stride, n, ic, oc, ws.data_ptr(), size)
    return h.get(), g.get() if g else None, u.get() if u else None


def check_gated(kind, n, ic, oc, act=D.ACT_SILU, bias=True, save="gu", pad=0, offset=0, wu_pad=None, seed=1):
    dtype = TYPES[kind][1]
    x = matrix(n, ic, dtype, seed, pad=pad, offset=offset)
    wg, wu = (matrix(oc, ic, dtype, seed + 1, max(1, ic) ** -0.5, pad=pad, offset=offset),
              matrix(oc, ic, dtype, seed + 2, max(1, ic) ** -0.5, pad=pad if wu_pad is None else wu_pad, offset=offset))
    bg, bu = (matrix(1, oc, dtype, seed + 3)[0], matrix(1, oc, dtype, seed + 4)[0]) if bias else (None, None)
    h, g, u = run_gated(kind, x, wg, wu, bg, bu, act, save, pad)
    x64 = x.double()
    g64, u64 = x64 @ wg.double().t(), x64 @ wu.double().t()
    tg, tu = product_tol(x64, wg.double(), dtype), product_tol(x64, wu.double(), dtype)
    if bias:
        g64, u64 = g64 + bg.double(), u64 + bu.double()
    tg, tu = tg + 2.0 ** -23 * g64.abs(), tu + 2.0 ** -23 * u64.abs()
    what = "%s " % ((kind, n, ic, oc, act),)
    if "g" in save:
        close(g, g64, tg, what + "G")
    if "u" in save:
        close(u, u64, tu, what + "U")
    a64 = act64(act, g64)
    ta = 1.2 * tg + 2.0 ** -20 * g64.abs().clamp(min=1.0)
    close(h, a64 * u64, ta * u64.abs() + a64.abs() * tu + ta * tu + 2.0 ** -23 * (a64 * u64).abs(), what + "H")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES + [(4100, 192, 1032), (1030, 2048, 520)])
def test_gated_sizes(kind, size):
    check_gated(kind, *size)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(1, 72, 40), (21, 72, 40), (140, 136, 200)])
@pytest.mark.parametrize("act", range(5))
def test_gated_activations_and_kept_tensors(kind, size, act):
    for bias, save in ((True, "gu"), (False, ""), (False, "g"), (True, "u")):
        check_gated(kind, *size, act=act, bias=bias, save=save)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(1, 96, 64), (20, 96, 64), (140, 96, 136)])
@pytest.mark.parametrize("pad,offset,wu_pad", [(0, 1, 0), (1, 0, 1), (3, 5, 3), (8, 8, 8), (8, 0, 16), (0, 0, 3)])
def test_gated_strides_and_alignments(kind, size, pad, offset, wu_pad):
    check_gated(kind, *size, pad=pad, offset=offset, wu_pad=wu_pad)


def test_gated_infinities_fp32():
    for n, ic, oc in ((2, 64, 40), (40, 200, 136), (200, 4096, 72)):
        x, wg, wu = matrix(n, ic, torch.float32, 1), matrix(oc, ic, torch.float32, 2, 0.1), matrix(oc, ic, torch.float32, 3, 0.1)
        x[1, 5] = float("inf")
        wu[2, 5] = 0.0
        h, g, u = run_gated("f32", x, wg, wu, None, None, D.ACT_LEAKY_RELU, "gu")
        g64, u64 = x.double() @ wg.double().t(), x.double() @ wu.double().t()
        for got, want in ((g, g64), (u, u64), (h, act64(D.ACT_LEAKY_RELU, g64) * u64)):
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want))


def run_gated_backward(kind, dh, g, u, act, x, wg, wu, want, pad=0):
    code, dtype = TYPES[kind]
    (n, oc), ic = dh.shape, x.shape[1]
    out = {"dx": Out(n, ic, dtype, pad), "dwg": Out(oc, ic, dtype, pad), "dwu": Out(oc, ic, dtype, pad), "dbg": Out(1, oc, dtype), "dbu": Out(1, oc, dtype)}
    ws, size = workspace(D.dgatedMatMul_workspace, code, n, ic, oc)

    def p(k):
        return out[k].ptr() if k in want else 0
    D.dgatedMatMul(stream(), 1, code, dh.data_ptr(), dh.stride(0), g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0), act, SLOPE,
                   x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), p("dx"), out["dx"].stride,
                   p("dwg"), out["dwg"].stride, p("dwu"), out["dwu"].stride, p("dbg"), p("dbu"), n, ic, oc, ws.data_ptr(), size)
    return {k: out[k].get() for k in want}


ALL_GATED = ("dx", "dwg", "dwu", "dbg", "dbu")


def check_gated_backward(kind, n, ic, oc, act=D.ACT_SILU, want=ALL_GATED, pad=0, offset=0, wu_pad=None, seed=1):
    dtype = TYPES[kind][1]
    x = matrix(n, ic, dtype, seed, pad=pad, offset=offset)
    wg, wu = (matrix(oc, ic, dtype, seed + 1, max(1, oc) ** -0.5, pad=pad, offset=offset),
              matrix(oc, ic, dtype, seed + 2, max(1, oc) ** -0.5, pad=pad if wu_pad is None else wu_pad, offset=offset))
    dh, g, u = (matrix(n, oc, dtype, seed + 3 + i, pad=pad, offset=offset) for i in range(3))
    got = run_gated_backward(kind, dh, g, u, act, x, wg, wu, want, pad)
    dh64, g64, u64, x64 = dh.double(), g.double(), u.double(), x.double()
    dg, du = dh64 * u64 * slope64(act, g64), dh64 * act64(act, g64)
    what = "%s " % ((kind, n, ic, oc, act),)
    edg = delta_error(act, dh64 * u64, g64)
    edu = dh64.abs() * 2.0 ** -20 * g64.abs().clamp(min=1.0)          # act(g)'s own error
    check_sums(got, kind, "dwg", "dbg", dg, edg, x64, what)
    check_sums(got, kind, "dwu", "dbu", du, edu, x64, what)
    if "dx" in want:
        tol = product_tol(torch.cat([dg, du], 1), torch.cat([wg.double(), wu.double()], 0).t(), dtype, ROUNDED[kind])
        tol = tol + edg @ wg.double().abs() + edu @ wu.double().abs()
        close(got["dx"], dg @ wg.double() + du @ wu.double(), tol, what + "dx")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES + [(4100, 192, 264), (1024, 512, 1032)])
def test_gated_backward_sizes(kind, size):
    check_gated_backward(kind, *size)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("act", range(5))
def test_gated_backward_activations_and_wanted_outputs(kind, act):
    for want in (ALL_GATED, ("dx",), ("dwg",), ("dwu",), ("dbu",), ("dwu", "dbg"), ("dwg", "dwu")):
        check_gated_backward(kind, 70, 136, 76, act=act, want=want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pad,offset,wu_pad", [(0, 1, 0), (3, 5, 3), (8, 8, 8), (8, 0, 16)])
def test_gated_backward_strides_and_alignments(kind, pad, offset, wu_pad):
    check_gated_backward(kind, 150, 104, 88, pad=pad, offset=offset, wu_pad=wu_pad)


# ---- gradients against differences -----------------------------------------------------------------------------------

@pytest.mark.parametrize("act", range(5))
def test_backward_agrees_with_differences_of_the_forward(act):
    """<dX, V> against (f(X + hV) - f(X - hV)) / 2h of f = <Y, deltaY> (the forward's fp32 results summed in 64 bits). A
    direction V of unit length, h = 1/16: the difference's own error is h^2/6 f''' <~ 1e-3 of |dX| for the smooth ones and
    the forward's rounding 2^-24 |Y| sqrt(N OC) / h: 2e-4; the leaky ReLU's kinks move few elements by O(h)."""
    n, ic, oc, h = 24, 40, 56, 1 / 16
    x, w, dy = matrix(n, ic, torch.float32, 1), matrix(oc, ic, torch.float32, 2, 0.2), matrix(n, oc, torch.float32, 3)
    v = matrix(n, ic, torch.float32, 4)
    v = v / v.norm()
    _, z = run_forward("f32", x, w, None, act, None, True)
    dx = run_backward("f32", dy, z, act, x, w)["dx"]

    def f(t):
        return float((run_forward("f32", t, w, None, act, None, False)[0].double() * dy.double()).sum())
    slope = (f((x + h * v).contiguous()) - f((x - h * v).contiguous())) / (2 * h)
    want = float((dx.double() * v.double()).sum())
    allowed = (0.02 if act == D.ACT_LEAKY_RELU else 2e-3) * float(dx.norm())
    assert abs(slope - want) <= allowed, (slope, want, allowed)


# ---- clipping --------------------------------------------------------------------------------------------------------

def run_clip(tensors, max_norm, eps=1e-6, in_place=False, norm_only=False, dst_offset=0):
    kinds = [D.F32 if t.dtype == torch.float32 else D.BF16 for t in tensors]
    lengths = [t.numel() for t in tensors]
    out = tensors if in_place else [torch.full((t.numel() + dst_offset,), float("nan"), dtype=t.dtype, device="cuda")[dst_offset:] for t in tensors]
    norm_c = torch.full((2,), float("nan"), device="cuda")
    n = D.gradClip_workspace(len(tensors), lengths)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device="cuda")
    D.gradClip(stream(), 1, len(tensors), kinds, lengths, [t.data_ptr() if t.numel() else 0 for t in tensors],
               None if norm_only else [t.data_ptr() if t.numel() else 0 for t in out], max_norm, eps, norm_c.data_ptr(), ws.data_ptr(), n)
    torch.cuda.synchronize()
    return norm_c.double().cpu(), out


def check_clip(tensors, max_norm, **kw):
    before = [t.clone() for t in tensors]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in before))
    c = min(1.0, max_norm / (norm + 1e-6))
    got, out = run_clip(tensors, max_norm, **kw)
    assert abs(float(got[0]) - norm) <= 2.0 ** -23 * norm and abs(float(got[1]) - c) <= 2.0 ** -23 * c
    for t, o in zip(before, out):
        # c rounded to fp32 and the product rounded once more before a bf16 output's own rounding
        close(o.view(1, -1), (t.double() * c).view(1, -1), t.double().abs().view(1, -1) * c * 2.0 ** -22, "clipped")


@pytest.mark.parametrize("lengths", [[1], [0, 5, 0], [16384], [16385, 1, 7], [100000, 3, 64, 65537], list(range(1, 120)), [1 << 22] * 3])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip(lengths, max_norm):
    tensors = [matrix(1, n, torch.float32 if i % 3 else torch.bfloat16, i)[0] for i, n in enumerate(lengths)]
    check_clip(tensors, max_norm)
    check_clip(tensors, max_norm, dst_offset=1)
    check_clip(tensors, max_norm, in_place=True)


def test_clip_of_views_at_any_element():
    flat32, flat16 = matrix(1, 70000, torch.float32, 1)[0], matrix(1, 70000, torch.bfloat16, 2)[0]
    check_clip([flat32[1:20000], flat32[20001:20003], flat16[1:30001], flat16[30003:65000], flat16[65007:65008]], 1.0)


def test_clip_keeps_elements_beside_the_views():
    flat = torch.ones(50000, device="cuda")
    run_clip([flat[3:20001], flat[20003:49999]], 1.0, in_place=True)
    assert float(flat[:3].sum()) == 3.0 and float(flat[20001:20003].sum()) == 2.0 and float(flat[49999:].sum()) == 1.0


def test_clip_of_nothing():
    got, _ = run_clip([], 1.0)
    assert got.tolist() == [0.0, 1.0]
    got, _ = run_clip([torch.zeros(10, device="cuda")], 1.0)
    assert got.tolist() == [0.0, 1.0]


def test_clip_outside_fp32_squares():
    for v in (1e-30, 3e38):
        t = torch.full((1000,), v, device="cuda")
        norm = float(t[0].double()) * math.sqrt(1000)
        got, out = run_clip([t], 1.0, eps=0.0)
        want_norm = norm if norm <= 3.4e38 else float("inf")
        assert float(got[0]) == pytest.approx(want_norm, rel=2.0 ** -22)
        c = min(1.0, 1.0 / norm)
        assert float(got[1]) == pytest.approx(c, rel=2.0 ** -22 if c > 1.2e-38 else 1.0, abs=1.5e-45)


def test_clip_nonfinite():
    t = torch.ones(100, device="cuda")
    t[7] = float("nan")
    got, out = run_clip([t, torch.ones(5, device="cuda")], 1.0)
    assert math.isnan(float(got[0])) and math.isnan(float(got[1])) and all(bool(torch.isnan(o).all()) for o in out)
    t[7] = float("inf")
    got, out = run_clip([t], 1.0)
    assert float(got[0]) == float("inf") and float(got[1]) == 0.0
    assert math.isnan(float(out[0][7])) and float(out[0][8]) == 0.0


def test_norm_only_leaves_the_tensors():
    t = matrix(1, 5000, torch.float32, 3)[0]
    before = t.clone()
    got, _ = run_clip([t], 0.1, norm_only=True)
    assert torch.equal(t, before) and float(got[0]) == pytest.approx(float(t.double().norm()), rel=2.0 ** -22)


# ---- together --------------------------------------------------------------------------------------------------------

class Block:
    """A gated feed-forward block with its down-projection and residual, and one training step of it with clipping, on
    buffers of its own: what a program would capture."""

    def __init__(self, kind, n, c, f):
        self.kind, (self.code, self.dtype), self.n, self.c, self.f = kind, TYPES[kind], n, c, f

        def new(*s):
            return torch.zeros(s, dtype=self.dtype, device="cuda")
        self.x, self.dy = new(n, c), new(n, c)
        self.wg, self.wu, self.wd, self.bd = new(f, c), new(f, c), new(c, f), new(c)
        self.g, self.u, self.h, self.y = new(n, f), new(n, f), new(n, f), new(n, c)
        self.dh, self.dx = new(n, f), new(n, c)
        self.grads = [new(f, c), new(f, c), new(c, f), new(c)]
        self.norm = torch.zeros(2, device="cuda")
        sizes = [D.gatedMatMul_workspace(self.code, n, c, f), D.matMul_fused_workspace(self.code, n, f, c), D.dmatMul_fused_workspace(self.code, n, f, c),
                 D.dgatedMatMul_workspace(self.code, n, c, f), D.gradClip_workspace(4, [t.numel() for t in self.grads])]
        self.bytes = max(sizes)
        self.ws = torch.empty(self.bytes, dtype=torch.uint8, device="cuda")

    def fresh(self, seed):
        for i, (t, std) in enumerate(((self.x, 1.0), (self.dy, 1.0), (self.wg, self.c ** -0.5), (self.wu, self.c ** -0.5), (self.wd, self.f ** -0.5), (self.bd, 1.0))):
            t.copy_(matrix(1, t.numel(), self.dtype, seed + i, std)[0].view_as(t))
        for t in (self.g, self.u, self.h, self.y, self.dh, self.dx, *self.grads):
            t.fill_(float("nan"))

    def step(self, s):
        n, c, f, code, ws, size = self.n, self.c, self.f, self.code, self.ws.data_ptr(), self.bytes
        D.gatedMatMul(s, 1, code, self.x.data_ptr(), c, self.wg.data_ptr(), c, 0, self.wu.data_ptr(), c, 0, D.ACT_SILU, 0.0,
                      self.g.data_ptr(), f, self.u.data_ptr(), f, self.h.data_ptr(), f, n, c, f, ws, size)
        D.matMul_fused(s, 1, code, self.h.data_ptr(), f, self.wd.data_ptr(), f, self.bd.data_ptr(), D.ACT_NONE, 0.0, self.x.data_ptr(), c, 0, 0,
                       self.y.data_ptr(), c, n, f, c, ws, size)
        D.dmatMul_fused(s, 1, code, self.dy.data_ptr(), c, 0, 0, D.ACT_NONE, 0.0, self.h.data_ptr(), f, self.wd.data_ptr(), f,
                        self.dh.data_ptr(), f, self.grads[2].data_ptr(), f, self.grads[3].data_ptr(), n, f, c, ws, size)
        D.dgatedMatMul(s, 1, code, self.dh.data_ptr(), f, self.g.data_ptr(), f, self.u.data_ptr(), f, D.ACT_SILU, 0.0, self.x.data_ptr(), c,
                       self.wg.data_ptr(), c, self.wu.data_ptr(), c, self.dx.data_ptr(), c, self.grads[0].data_ptr(), c, self.grads[1].data_ptr(), c,
                       0, 0, n, c, f, ws, size)
        p = [t.data_ptr() for t in self.grads]
        D.gradClip(s, 1, 4, [code] * 4, [t.numel() for t in self.grads], p, p, 1.0, 1e-6, self.norm.data_ptr(), ws, size)

    def outputs(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.g, self.u, self.h, self.y, self.dh, self.dx, *self.grads, self.norm)]

    def verify(self):
        """Every stage against its formula in 64 bits on the stage's own inputs."""
        g, u, h, y, dh, dx, dwg, dwu, dwd, dbd, norm = self.outputs()
        d = [t.double() for t in (self.x, self.wg, self.wu, self.wd, self.bd, self.dy)]
        x, wg, wu, wd, bd, dy = d
        close(y, h.double() @ wd.t() + bd + x, product_tol(h.double(), wd, self.dtype) + 2.0 ** -22 * (bd.abs() + x.abs() + 4), "y")
        extra = ROUNDED[self.kind]
        close(dh, dy @ wd, product_tol(dy, wd.t(), self.dtype), "dh")
        dg, du = dh.double() * u.double() * slope64(D.ACT_SILU, g.double()), dh.double() * act64(D.ACT_SILU, g.double())
        edg, edu = delta_error(D.ACT_SILU, dh.double() * u.double(), g.double()), dh.double().abs() * 2.0 ** -20 * g.double().abs().clamp(min=1.0)
        tol = product_tol(torch.cat([dg, du], 1), torch.cat([wg, wu]).t(), self.dtype, extra) + edg @ wg.abs() + edu @ wu.abs()
        close(dx, dg @ wg + du @ wu, tol, "dx")
        full = [dg.t() @ x, du.t() @ x, dy.t() @ h.double(), dy.sum(0)]
        total = math.sqrt(sum(float(t.square().sum()) for t in full))
        # the norm of the gradients as they were stored (rounded) is within their rounding of the exact ones'
        assert float(norm[0]) == pytest.approx(total, rel=2.0 ** -7 if self.kind == "bf16" else 1e-5)
        c = float(norm[1])
        assert c == pytest.approx(min(1.0, 1.0 / (float(norm[0]) + 1e-6)), rel=2.0 ** -22)
        tols = [product_tol(dg.t(), x.t(), self.dtype, extra) + edg.t() @ x.abs(), product_tol(du.t(), x.t(), self.dtype, extra) + edu.t() @ x.abs(), product_tol(dy.t(), h.double().t(), self.dtype),
                dy.square().sum(0).sqrt() * 16 * math.sqrt(self.n + 64) * 2.0 ** -23]
        for got, want, tol in zip((dwg, dwu, dwd, dbd), full, tols):
            # two roundings: the gradient's and the clipped one's
            close(got, want * c, tol * c + (HALF[self.dtype] + 2.0 ** -22) * want.abs() * c, "clipped gradient")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,f", [(1, 64, 176), (50, 64, 176), (392, 256, 520)])
def test_training_step_of_a_gated_block_eager_and_replayed(kind, n, c, f):
    """Eager, then captured and replayed three times with fresh inputs and eager work between the replays; every replay
    is checked against the formulas and equals the eager step on the same inputs bit for bit."""
    b = Block(kind, n, c, f)
    side = torch.cuda.Stream()
    b.fresh(100)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b.step([int(side.cuda_stream)])
    b.verify()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        b.step([int(torch.cuda.current_stream().cuda_stream)])
    for rep in range(3):
        b.fresh(200 + 50 * rep)
        torch.cuda.synchronize()
        graph.replay()
        b.verify()
        replayed = b.outputs()
        b.fresh(200 + 50 * rep)
        b.step(stream())
        for got, want in zip(replayed, b.outputs()):
            assert torch.equal(got, want)


def test_two_streams_with_a_workspace_each():
    a, b = Block("bf16", 392, 256, 520), Block("f32", 100, 128, 200)
    a.fresh(1)
    b.fresh(2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        a.step([int(s1.cuda_stream)])
        b.step([int(s2.cuda_stream)])
    a.verify()
    b.verify()


def test_results_are_bit_identical_from_run_to_run():
    for kind, size in (("bf16", (300, 4096, 264)), ("f32", (300, 1000, 136)), ("bf16", (7, 4096, 520))):
        dtype = TYPES[kind][1]
        x, w = matrix(size[0], size[1], dtype, 1), matrix(size[2], size[1], dtype, 2)
        first, _ = run_forward(kind, x, w, None, D.ACT_GELU, None, False)
        for _ in range(3):
            again, _ = run_forward(kind, x, w, None, D.ACT_GELU, None, False)
            assert torch.equal(first, again)


def test_workspace_bytes_are_enough_and_nothing_is_written_behind_them():
    for kind, size in (("bf16", (300, 4099, 264)), ("f32", (300, 1000, 136)), ("f32", (3, 65, 33))):
        code, dtype = TYPES[kind]
        n, ic, oc = size
        need = D.matMul_fused_workspace(code, n, ic, oc)
        ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        x, w = matrix(n, ic, dtype, 1), matrix(oc, ic, dtype, 2)
        run_forward(kind, x, w, None, 0, None, False, ws=(ws, need))
        assert bool((ws[need:] == 0xA5).all())
        need = D.dmatMul_fused_workspace(code, n, ic, oc)
        ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        dy, dx, dw = matrix(n, oc, dtype, 3), Out(n, ic, dtype), Out(oc, ic, dtype)
        D.dmatMul_fused(stream(), 1, code, dy.data_ptr(), oc, dy.data_ptr(), oc, D.ACT_GELU, 0.0, x.data_ptr(), ic, w.data_ptr(), ic,
                        dx.ptr(), ic, dw.ptr(), ic, 0, n, ic, oc, ws.data_ptr(), need)
        dx.get(), dw.get()
        assert bool((ws[need:] == 0xA5).all())


def test_in_place_residual_and_numpy_oracle():
    """One small case end to end against numpy."""
    x, w, r = matrix(5, 12, torch.float32, 1), matrix(6, 12, torch.float32, 2), matrix(5, 6, torch.float32, 3)
    want = np.maximum(x.cpu().numpy().astype(np.float64) @ w.cpu().numpy().astype(np.float64).T, 0) + r.cpu().numpy()
    y = r.clone()
    ws, n = workspace(D.matMul_fused_workspace, D.F32, 5, 12, 6)
    D.matMul_fused(stream(), 1, D.F32, x.data_ptr(), 12, w.data_ptr(), 12, 0, D.ACT_LEAKY_RELU, 0.0, y.data_ptr(), 6, 0, 0, y.data_ptr(), 6,
                   5, 12, 6, ws.data_ptr(), n)
    torch.cuda.synchronize()
    assert np.allclose(y.cpu().numpy(), want, rtol=1e-5, atol=1e-5)


# ---- reductions and edges of the forms that read their operands straight from memory --------------------------------
DIRECT = [(100, 2001, 70), (40, 1023, 33), (384, 9, 200), (384, 33, 777), (130, 96, 1000), (700, 41, 130), (2000, 129, 70), (257, 255, 65), (90, 15, 500)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", DIRECT)
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 0), (0, 1), (3, 2), (2, 3)])
def test_forward_of_short_reductions_and_odd_rows(kind, size, pad, offset):
    check_forward(kind, *size, act=D.ACT_LEAKY_RELU, residual=True, save=True, pad=pad, offset=offset)
    check_gated(kind, *size, pad=pad, offset=offset)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [2, 4, 5, 16])
@pytest.mark.parametrize("ic,oc", [(7, 9), (8, 64), (9, 130), (2049, 61), (4097, 5000), (1000, 4100)])
def test_few_rows_of_odd_lengths(kind, n, ic, oc):
    check_forward(kind, n, ic, oc, act=D.ACT_SILU, residual=True, save=True, pad=1)
    check_gated(kind, n, ic, oc)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(16, 36, 40), (200, 32, 760), (64, 70, 33), (1457, 64, 723), (33, 300, 9), (9, 5, 1500), (640, 333, 47)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 1), (3, 2)])
def test_backward_of_small_products(kind, size, pad, offset):
    check_backward(kind, *size, D.ACT_SILU, pad=pad, offset=offset)
    check_backward(kind, *size, D.ACT_NONE, want=("dx", "dw"), pad=pad, offset=offset)
    check_gated_backward(kind, *size, pad=pad, offset=offset)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 7])
@pytest.mark.parametrize("ic,oc", [(4, 8), (5, 2), (64, 1728), (1217, 895), (784, 176)])
def test_backward_of_few_rows(kind, n, ic, oc):
    check_backward(kind, n, ic, oc, D.ACT_LEAKY_RELU, pad=1)
    check_gated_backward(kind, n, ic, oc, pad=3)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,ic,oc", [(64, 320, 3136), (4416, 32, 34), (4416, 33, 35), (60, 100, 5001), (2, 5, 4099), (30000, 4, 6)])
@pytest.mark.parametrize("pad", [0, 3])
def test_backward_of_long_sums_of_few_results(kind, n, ic, oc, pad):
    check_backward(kind, n, ic, oc, D.ACT_SIGMOID, pad=pad)
    check_gated_backward(kind, n, ic, oc, pad=pad)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,ic,oc", [(64, 320, 3136), (4416, 33, 35), (2, 5, 4099), (200, 64, 4400), (1100, 96, 1030), (129, 2049, 513), (2000, 1500, 700)])
def test_nothing_is_written_behind_a_workspace_of_any_form(kind, n, ic, oc):
    code, dtype = TYPES[kind]
    x, w, u = matrix(n, ic, dtype, 1), matrix(oc, ic, dtype, 2), matrix(oc, ic, dtype, 3)
    dy, z = matrix(n, oc, dtype, 4), matrix(n, oc, dtype, 5)
    dx, dw, du, db = Out(n, ic, dtype), Out(oc, ic, dtype), Out(oc, ic, dtype), Out(1, oc, dtype)
    y = Out(n, oc, dtype)
    p = lambda t: t.data_ptr()
    calls = [
        (D.matMul_fused_workspace, lambda ws: D.matMul_fused(stream(), 1, code, p(x), ic, p(w), ic, 0, D.ACT_SILU, 0.0, 0, 0, 0, 0, y.ptr(), oc, n, ic, oc, *ws), (y,)),
        (D.gatedMatMul_workspace, lambda ws: D.gatedMatMul(stream(), 1, code, p(x), ic, p(w), ic, 0, p(u), ic, 0, D.ACT_SILU, 0.0, 0, 0, 0, 0, y.ptr(), oc, n, ic, oc, *ws), (y,)),
        (D.dmatMul_fused_workspace, lambda ws: D.dmatMul_fused(stream(), 1, code, p(dy), oc, p(z), oc, D.ACT_SILU, 0.0, p(x), ic, p(w), ic, dx.ptr(), ic, dw.ptr(), ic,
                                                               db.ptr(), n, ic, oc, *ws), (dx, dw, db)),
        (D.dgatedMatMul_workspace, lambda ws: D.dgatedMatMul(stream(), 1, code, p(dy), oc, p(z), oc, p(dy), oc, D.ACT_SILU, 0.0, p(x), ic, p(w), ic, p(u), ic, dx.ptr(), ic,
                                                             dw.ptr(), ic, du.ptr(), ic, db.ptr(), 0, n, ic, oc, *ws), (dx, dw, du, db)),
    ]
    for query, call, outputs in calls:
        need = query(code, n, ic, oc)
        got = []
        for poison in (0xA5, 0x5A):     # whatever lay there before
            ws = torch.full((need + 65536,), poison, dtype=torch.uint8, device="cuda")
            call((ws.data_ptr(), need))
            got.append([o.get() for o in outputs])
            assert bool((ws[need:] == poison).all()), query
        for a, b in zip(*got):
            assert bool((a == b).all()) and not bool(a.isnan().any()), query


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,ic,oc", [(64, 320, 3136), (384, 96, 1100), (20, 2001, 300), (5, 1217, 895)])
def test_calls_replayed_from_a_graph_between_eager_ones(kind, n, ic, oc):
    code, dtype = TYPES[kind]
    x, w, dy = matrix(n, ic, dtype, 1), matrix(oc, ic, dtype, 2, ic ** -0.5), matrix(n, oc, dtype, 3)
    b = matrix(1, oc, dtype, 4)[0]
    z, y = torch.empty(n, oc, dtype=dtype, device="cuda"), torch.empty(n, oc, dtype=dtype, device="cuda")
    dx, dw, db = torch.empty(n, ic, dtype=dtype, device="cuda"), torch.empty(oc, ic, dtype=dtype, device="cuda"), torch.empty(oc, dtype=dtype, device="cuda")
    wf, nf = workspace(D.matMul_fused_workspace, code, n, ic, oc)
    wb, nb = workspace(D.dmatMul_fused_workspace, code, n, ic, oc)

    def step():
        D.matMul_fused(stream(), 1, code, x.data_ptr(), ic, w.data_ptr(), ic, b.data_ptr(), D.ACT_GELU, 0.0, 0, 0, z.data_ptr(), oc, y.data_ptr(), oc, n, ic, oc, wf.data_ptr(), nf)
        D.dmatMul_fused(stream(), 1, code, dy.data_ptr(), oc, z.data_ptr(), oc, D.ACT_GELU, 0.0, x.data_ptr(), ic, w.data_ptr(), ic, dx.data_ptr(), ic, dw.data_ptr(), ic,
                        db.data_ptr(), n, ic, oc, wb.data_ptr(), nb)

    outputs = (z, y, dx, dw, db)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        x.copy_(matrix(n, ic, dtype, 10 + turn))
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in outputs]
        for t in outputs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == e).all()) for t, e in zip(outputs, want)), turn


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [(4096, 512, 4096), (4100, 256, 4104), (8000, 96, 2052)])
@pytest.mark.parametrize("in_place", [False, True])
def test_residual_of_large_tiles(kind, size, in_place):
    check_forward(kind, *size, act=D.ACT_SILU, residual=True, in_place=in_place)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [5, 16, 33, 107])
@pytest.mark.parametrize("ic,oc", [(8192, 100), (6001, 65), (3100, 1001), (2048, 3)])
@pytest.mark.parametrize("pad", [0, 3])
def test_long_sums_of_few_rows(kind, n, ic, oc, pad):
    check_forward(kind, n, ic, oc, act=D.ACT_GELU, residual=True, save=True, pad=pad, in_place=pad == 0)
    check_gated(kind, n, ic, oc, pad=pad)
