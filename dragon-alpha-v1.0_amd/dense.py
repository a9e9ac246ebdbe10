"""ctypes mirror of the dense operators of include/alpha_dense.h: the fused matrix product, the gated pair of projections,
their backward and clipping by the global gradient norm. Argument order is the C ABI's; addresses are plain integers
(device pointers / hipStream_t handles, 0 = absent) and a non-zero status raises AlphaConvError, as in native.py."""
import ctypes

from . import native

_I, _L, _P, _F = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
_functions = {}          # bound entries by name, once the library is loaded
_ONE = _L * 1

# S = stream array, i = int, l = int64, f = float, p = device pointer; n, q, t = host arrays of int, int64, addresses
_SIGS = {
    "alpha_matMul_fused": "Sii" + "pl" * 2 + "pif" + "pl" * 3 + "iiipl",
    "alpha_dmatMul_fused": "Sii" + "pl" * 2 + "if" + "pl" * 4 + "piiipl",
    "alpha_gatedMatMul": "Sii" + "pl" * 2 + "ppl" + "pif" + "pl" * 3 + "iiipl",
    "alpha_dgatedMatMul": "Sii" + "pl" * 3 + "if" + "pl" * 6 + "ppiiipl",
    "alpha_gradClip": "Siinqttffppl",
}
_SIZES = ("alpha_matMul_fused_workspace", "alpha_dmatMul_fused_workspace", "alpha_gatedMatMul_workspace", "alpha_dgatedMatMul_workspace")
_CT = {"S": ctypes.POINTER(_L), "i": _I, "l": _L, "f": _F, "p": _P, "n": ctypes.POINTER(_I), "q": ctypes.POINTER(_L), "t": ctypes.POINTER(_P)}


def exported_symbols():
    """Names the library must export (every function include/alpha_dense.h declares)."""
    return sorted(list(_SIGS) + list(_SIZES) + ["alpha_gradClip_workspace", "alpha_dense_last_error"])


def _bind():
    L = native.lib()
    for name, sig in _SIGS.items():
        getattr(L, name).argtypes = [_CT[c] for c in sig]
        getattr(L, name).restype = _I
    for name in _SIZES:
        getattr(L, name).argtypes = [_I] * 4
        getattr(L, name).restype = _L
    L.alpha_gradClip_workspace.argtypes = [_I, ctypes.POINTER(_L)]
    L.alpha_gradClip_workspace.restype = _L
    L.alpha_dense_last_error.restype = ctypes.c_char_p
    _functions.update({name: getattr(L, name) for name in exported_symbols()})
    return _functions


def _array(kind, values, count=0):
    """A host array for the C side, which reads `count` entries."""
    if values is None:
        return None
    if len(values) < count:
        raise native.AlphaConvError("a list of %d entries is shorter than the count %d" % (len(values), count))
    return (kind * max(1, len(values)))(*values)


def _call(name, streams, length, *args):
    """`args` as ctypes takes them for the signature: integers, floats, arrays."""
    if len(streams) < length:
        raise native.AlphaConvError("%s: %d streams given, length %d" % (name, len(streams), length))
    rc = (_functions or _bind())[name](_ONE(streams[0]) if len(streams) == 1 else (_L * max(1, len(streams)))(*streams), length, *args)
    if rc != 0:
        raise native.AlphaConvError("%s failed (%d): %s" % (name, rc, _functions["alpha_dense_last_error"]().decode()))


def _workspace(name, *args):
    n = (_functions or _bind())[name](*args)
    if n < 0:
        raise native.AlphaConvError("%s: size out of range %s" % (name, args))
    return n


class Cuda_dense:
    """Dense operators around the convolutions (no Java counterpart: the reference's are natives of other classes and
    come without epilogues). X[N,IC], W[OC,IC], Y[N,OC]; *_stride in elements; types F32 and BF16."""

    F32, BF16 = 0, 1
    ACT_NONE, ACT_LEAKY_RELU, ACT_GELU, ACT_SILU, ACT_SIGMOID = range(5)

    @staticmethod
    def matMul_fused_workspace(type, N, IC, OC):
        return _workspace("alpha_matMul_fused_workspace", type, N, IC, OC)

    @staticmethod
    def matMul_fused(streamArray, length, type, X, X_stride, W, W_stride, Bias, act, k, R, R_stride, Z, Z_stride, Y, Y_stride, N, IC, OC,
                     workspace, workspace_bytes):
        """Z = X W^T + Bias, Y = act(Z) + R; Bias, R and Z may be 0."""
        _call("alpha_matMul_fused", streamArray, length, type, X, X_stride, W, W_stride, Bias, act, k, R, R_stride, Z, Z_stride, Y, Y_stride,
              N, IC, OC, workspace, workspace_bytes)

    @staticmethod
    def dmatMul_fused_workspace(type, N, IC, OC):
        return _workspace("alpha_dmatMul_fused_workspace", type, N, IC, OC)

    @staticmethod
    def dmatMul_fused(streamArray, length, type, deltaY, deltaY_stride, Z, Z_stride, act, k, X, X_stride, W, W_stride, deltaX, deltaX_stride,
                      deltaW, deltaW_stride, deltaB, N, IC, OC, workspace, workspace_bytes):
        """deltaZ = deltaY * act'(Z); deltaX = deltaZ W, deltaW = deltaZ^T X, deltaB = column sums; outputs that are 0 are left out."""
        _call("alpha_dmatMul_fused", streamArray, length, type, deltaY, deltaY_stride, Z, Z_stride, act, k, X, X_stride, W, W_stride,
              deltaX, deltaX_stride, deltaW, deltaW_stride, deltaB, N, IC, OC, workspace, workspace_bytes)

    @staticmethod
    def gatedMatMul_workspace(type, N, IC, OC):
        return _workspace("alpha_gatedMatMul_workspace", type, N, IC, OC)

    @staticmethod
    def gatedMatMul(streamArray, length, type, X, X_stride, Wg, Wg_stride, Bg, Wu, Wu_stride, Bu, act, k, G, G_stride, U, U_stride, H, H_stride,
                    N, IC, OC, workspace, workspace_bytes):
        """G = X Wg^T + Bg, U = X Wu^T + Bu, H = act(G) * U; Bg, Bu, G and U may be 0."""
        _call("alpha_gatedMatMul", streamArray, length, type, X, X_stride, Wg, Wg_stride, Bg, Wu, Wu_stride, Bu, act, k, G, G_stride, U, U_stride,
              H, H_stride, N, IC, OC, workspace, workspace_bytes)

    @staticmethod
    def dgatedMatMul_workspace(type, N, IC, OC):
        return _workspace("alpha_dgatedMatMul_workspace", type, N, IC, OC)

    @staticmethod
    def dgatedMatMul(streamArray, length, type, deltaH, deltaH_stride, G, G_stride, U, U_stride, act, k, X, X_stride, Wg, Wg_stride, Wu, Wu_stride,
                     deltaX, deltaX_stride, deltaWg, deltaWg_stride, deltaWu, deltaWu_stride, deltaBg, deltaBu, N, IC, OC, workspace,
                     workspace_bytes):
        """deltaG = deltaH * U * act'(G), deltaU = deltaH * act(G) and their products; outputs that are 0 are left out."""
        _call("alpha_dgatedMatMul", streamArray, length, type, deltaH, deltaH_stride, G, G_stride, U, U_stride, act, k, X, X_stride,
              Wg, Wg_stride, Wu, Wu_stride, deltaX, deltaX_stride, deltaWg, deltaWg_stride, deltaWu, deltaWu_stride, deltaBg, deltaBu,
              N, IC, OC, workspace, workspace_bytes)

    @staticmethod
    def gradClip_workspace(count, lengths):
        return _workspace("alpha_gradClip_workspace", count, _array(_L, lengths, count))

    @staticmethod
    def gradClip(streamArray, length, count, types, lengths, src, dst, max_norm, eps, norm_c, workspace, workspace_bytes):
        """norm_c = {norm, c} with c = min(1, max_norm / (norm + eps)); dst = src * c (dst None: only the norm)."""
        _call("alpha_gradClip", streamArray, length, count, _array(_I, types, count), _array(_L, lengths, count), _array(_P, src, count),
              _array(_P, dst, count), max_norm, eps, norm_c, workspace, workspace_bytes)
