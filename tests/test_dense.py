"""The dense operators' boundary without a GPU: every function of include/alpha_dense.h is exported and bound, workspace
queries answer for every served size, and bad calls are refused before anything is enqueued."""
import ctypes
import os
import re
import subprocess

import pytest

from util import ROOT, load_package

pkg = load_package()
D = pkg.Cuda_dense
P = 1 << 20          # never dereferenced
BIG = 1 << 40


def test_every_declared_symbol_is_exported_and_bound():
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "alpha_dense.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(alpha_\w+)\s*\(", hdr)))
    out = subprocess.check_output(["nm", "-D", "--defined-only", pkg.lib_path()], text=True)
    exported = {l.split()[-1] for l in out.splitlines() if " T " in l}
    assert not [f for f in declared if f not in exported]
    assert pkg.dense.exported_symbols() == declared


@pytest.mark.parametrize("query", [D.matMul_fused_workspace, D.dmatMul_fused_workspace, D.gatedMatMul_workspace, D.dgatedMatMul_workspace])
def test_workspace_queries(query):
    for kind in (D.F32, D.BF16):
        for sizes in ((0, 0, 0), (1, 1, 1), (1, 4096, 4096), (777, 1001, 515), (0, 64, 64), (64, 0, 64), (64, 64, 0), (8192, 8192, 4096)):
            assert query(kind, *sizes) >= 0
            assert query(kind, *sizes) % 256 == 0
    for bad in ((2, 8, 8, 8), (-1, 8, 8, 8), (0, -1, 8, 8), (0, 8, -1, 8), (0, 8, 8, (1 << 22) + 1), (0, (1 << 31) - 1, 4096, 8)):
        with pytest.raises(pkg.AlphaConvError):
            query(*bad)


def forward(**kw):
    a = dict(streams=[0], length=1, type=D.BF16, X=P, xs=64, W=2 * P, ws=64, B=3 * P, act=D.ACT_GELU, k=0.0, R=4 * P, rs=32, Z=5 * P, zs=32,
             Y=6 * P, ys=32, N=5000, IC=64, OC=32, work=7 * P, bytes=BIG)
    a.update(kw)
    D.matMul_fused(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(streams=[], length=0), "stream"), (dict(type=2), "type"), (dict(act=5), "activation"), (dict(act=-1), "activation"),
    (dict(act=D.ACT_LEAKY_RELU, k=float("nan")), "slope"), (dict(X=0), "X is null"), (dict(W=0), "W is null"), (dict(Y=0), "Y is null"),
    (dict(X=P + 1), "aligned"), (dict(B=3 * P + 1), "aligned"), (dict(Y=6 * P + 1), "aligned"), (dict(type=D.F32, R=4 * P + 2), "aligned"),
    (dict(xs=63), "X_stride"), (dict(ys=31), "Y_stride"), (dict(ws=(1 << 22) + 8), "W_stride"), (dict(zs=-32), "Z_stride"),
    (dict(work=0), "workspace"), (dict(work=7 * P + 128), "workspace"), (dict(bytes=0), "workspace"), (dict(bytes=-1), "workspace"),
    (dict(N=-1), "size"), (dict(Y=P), "shares"), (dict(Z=6 * P), "share"), (dict(Z=4 * P), "shares"), (dict(R=6 * P, rs=40), "stride"),
])
def test_matMul_refusals(change, message):
    with pytest.raises(pkg.AlphaConvError, match=message):
        forward(**change)


def test_empty_outputs_need_nothing():
    forward(N=0, X=0, R=0, Z=0, Y=0)
    forward(OC=0, W=0, B=0, R=0, Z=0, Y=0)


@pytest.mark.parametrize("change,message", [
    (dict(type=7), "type"), (dict(dY=0), "deltaY"), (dict(Z=0), "Z is null"), (dict(X=0), "X is null"), (dict(W=0), "W is null"),
    (dict(dX=P), "shares"), (dict(dW=5 * P), "share"), (dict(dys=31), "deltaY_stride"), (dict(dxs=63), "deltaX_stride"), (dict(bytes=255), "workspace"),
])
def test_dmatMul_refusals(change, message):
    a = dict(streams=[0], length=1, type=D.BF16, dY=P, dys=32, Z=2 * P, zs=32, act=D.ACT_SILU, k=0.0, X=3 * P, xs=64, W=4 * P, ws=64,
             dX=5 * P, dxs=64, dW=6 * P, dws=64, dB=8 * P, N=16, IC=64, OC=32, work=7 * P, bytes=BIG)
    a.update(change)
    with pytest.raises(pkg.AlphaConvError, match=message):
        D.dmatMul_fused(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(act=9), "activation"), (dict(X=0), "X is null"), (dict(Wg=0), "Wg is null"), (dict(Wu=0), "Wu is null"), (dict(H=0), "H is null"),
    (dict(G=9 * P), "share"), (dict(U=P), "shares"), (dict(wus=8), "Wu_stride"), (dict(hs=1), "H_stride"), (dict(work=1), "workspace"),
])
def test_gatedMatMul_refusals(change, message):
    a = dict(streams=[0], length=1, type=D.F32, X=P, xs=64, Wg=2 * P, wgs=64, Bg=0, Wu=3 * P, wus=64, Bu=0, act=D.ACT_SILU, k=0.0,
             G=4 * P, gs=32, U=5 * P, us=32, H=9 * P, hs=32, N=5000, IC=64, OC=32, work=7 * P, bytes=BIG)
    a.update(change)
    with pytest.raises(pkg.AlphaConvError, match=message):
        D.gatedMatMul(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dH=0), "deltaH"), (dict(G=0), "G is null"), (dict(U=0), "U is null"), (dict(X=0), "X is null"), (dict(Wg=0), "Wg is null"),
    (dict(dWg=11 * P), "share"), (dict(dBg=13 * P), "share"), (dict(dX=P), "shares"), (dict(dwus=1), "deltaWu_stride"),
])
def test_dgatedMatMul_refusals(change, message):
    a = dict(streams=[0], length=1, type=D.F32, dH=P, dhs=32, G=2 * P, gs=32, U=3 * P, us=32, act=D.ACT_SILU, k=0.0, X=4 * P, xs=64,
             Wg=5 * P, wgs=64, Wu=6 * P, wus=64, dX=8 * P, dxs=64, dWg=10 * P, dwgs=64, dWu=11 * P, dwus=64, dBg=12 * P, dBu=13 * P,
             N=16, IC=64, OC=32, work=7 * P, bytes=BIG)
    a.update(change)
    with pytest.raises(pkg.AlphaConvError, match=message):
        D.dgatedMatMul(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(streams=[], length=0), "stream"), (dict(count=-1), "list"), (dict(types=[0, 3]), "type"), (dict(lengths=[4, -1]), "length"),
    (dict(src=[P, 0]), "src"), (dict(src=[P, 2 * P + 2]), "src"), (dict(dst=[P, 0]), "dst"), (dict(dst=[P + 1, 2 * P]), "dst"),
    (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("inf")), "max_norm"), (dict(eps=float("nan")), "eps"), (dict(max_norm=0.0, eps=0.0), "both"),
    (dict(norm_c=0), "norm_c"), (dict(norm_c=P + 2), "norm_c"), (dict(work=0), "workspace"), (dict(bytes=8), "workspace"),
])
def test_gradClip_refusals(change, message):
    a = dict(streams=[0], length=1, count=2, types=[D.F32, D.F32], lengths=[4, 5], src=[P, 2 * P], dst=[P, 2 * P], max_norm=1.0, eps=1e-6,
             norm_c=3 * P, work=7 * P, bytes=BIG)
    a.update(change)
    with pytest.raises(pkg.AlphaConvError, match=message):
        D.gradClip(*a.values())


def test_gradClip_workspace():
    assert D.gradClip_workspace(0, None) == 0
    assert D.gradClip_workspace(3, [0, 1, 1 << 20]) >= 8 * 2
    with pytest.raises(pkg.AlphaConvError):
        D.gradClip_workspace(1, [-1])
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_a_pair_of_filters_has_half_the_columns():
    # their deltaZ lie side by side in one row, whose length has the limit of a stride
    for code in (D.F32, D.BF16):
        assert D.gatedMatMul_workspace(code, 8, 8, 1 << 21) >= 0 and D.dgatedMatMul_workspace(code, 8, 8, 1 << 21) > 0
        assert D.matMul_fused_workspace(code, 8, 8, 1 << 22) >= 0 and D.dmatMul_fused_workspace(code, 8, 8, 1 << 22) > 0
        for query in (D.gatedMatMul_workspace, D.dgatedMatMul_workspace):
            with pytest.raises(pkg.AlphaConvError):
                query(code, 8, 8, (1 << 21) + 1)


def test_rows_have_a_limit():
    for query in (D.matMul_fused_workspace, D.dmatMul_fused_workspace, D.gatedMatMul_workspace, D.dgatedMatMul_workspace):
        for code in (D.F32, D.BF16):
            assert query(code, (1 << 30) - 1, 4, 2) >= 0
            with pytest.raises(pkg.AlphaConvError):
                query(code, 1 << 30, 4, 2)
