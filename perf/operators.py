"""Measured cases of the dense operators of include/alpha_dense.h: the fused matrix product and its backward, the gated
projection pair of a feed-forward block and its backward, and clipping by the global gradient norm.

    Z = X W^T + Bias,  Y = act(Z) + R                                  X[N,IC], W[OC,IC], Y[N,OC]
    deltaZ = deltaY * act'(Z),  deltaX = deltaZ W,  deltaW = deltaZ^T X,  deltaB = column sums of deltaZ
    G = X Wg^T + Bg,  U = X Wu^T + Bu,  H = act(G) * U                 Wg, Wu[OC,IC]
    deltaG = deltaH * U * act'(G),  deltaU = deltaH * act(G),  deltaX = deltaG Wg + deltaU Wu,  deltaWg = deltaG^T X, ...
    norm = sqrt(sum over all tensors and elements of g^2),  g' = g * min(1, max_norm / (norm + eps))

`own` chooses between the plain torch form and the library's calls.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = {"none": 0, "leaky_relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
SLOPE = 0.01   # of the leaky ReLU


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the classifier behind a ResNet-18 body: 64 pooled images, 512 features, 1000 classes (stored as such, no padding)
        dict(name="classifier", op="matmul", type="f32", N=64, IC=512, OC=1000, act="none", bias=True, residual=False, save=False, pad=0),
        # one token through an output projection with its residual: latency of a single row while weights stream from memory
        dict(name="token", op="matmul", type="bf16", N=1, IC=4096, OC=4096, act="none", bias=True, residual=True, save=False, pad=0),
        # training forward at an ordinary batch: up-projection, pre-activation kept for the backward
        dict(name="forward_f32", op="matmul", type="f32", N=4096, IC=1024, OC=4096, act="gelu", bias=True, residual=False, save=True, pad=0),
        # the largest forward: 8192 rows, residual added in the epilogue
        dict(name="forward_bf16", op="matmul", type="bf16", N=8192, IC=8192, OC=4096, act="silu", bias=True, residual=True, save=False, pad=0),
        # ragged everywhere: odd rows, odd features, rows that begin on two-byte boundaries
        dict(name="ragged", op="matmul", type="bf16", N=777, IC=1001, OC=515, act="leaky_relu", bias=True, residual=True, save=True, pad=3),
        # channel layer of a network body in fp32 (14x14 maps of 64 images as rows): all gradients
        dict(name="backward_f32", op="matmul_backward", type="f32", N=12544, IC=256, OC=1024, act="gelu", bias=True, pad=0),
        # the same of a large layer in bf16
        dict(name="backward_bf16", op="matmul_backward", type="bf16", N=8192, IC=4096, OC=4096, act="silu", bias=True, pad=0),
        # gated block: one token
        dict(name="gated_token", op="gated", type="bf16", N=1, IC=2048, OC=8192, act="silu", bias=False, save=False, pad=0),
        # gated block in training: both pre-activations kept
        dict(name="gated_forward", op="gated", type="bf16", N=4096, IC=4096, OC=5632, act="silu", bias=False, save=True, pad=0),
        dict(name="gated_backward", op="gated_backward", type="bf16", N=4096, IC=2048, OC=5632, act="gelu", bias=True, pad=0),
        # the gradients of a residual network's filters, biases and normalisation vectors, clipping active
        dict(name="clip_network", op="clip", type="f32", kind="network", tensors=0, largest=0, spread=0, max_norm=1.0, scale=0.01),
        # few large tensors of a wide model in bf16
        dict(name="clip_large", op="clip", type="bf16", kind="spread", tensors=48, largest=1 << 24, spread=1, max_norm=1.0, scale=0.001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A size over the logarithm of its range: a multiple of 64, a multiple of 8, or any number."""
    v = _log(rng, lo, hi)
    unit = rng.choice([64, 64, 8, 1])
    return max(lo, min(hi, max(1, v // unit) * unit))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "matmul_backward", "matmul_backward", "gated", "gated_backward", "clip"])
    kind = rng.choice(["f32", "bf16"])
    if op == "clip":
        return dict(op=op, type=kind, kind="spread", tensors=_log(rng, 1, 300), largest=_log(rng, 64, 1 << 21), spread=rng.randrange(1 << 30),
                    max_norm=rng.choice([0.5, 1.0, 1000.0]), scale=rng.choice([0.001, 0.01]))
    most = 5.0e10 if kind == "f32" else 2.5e11
    while True:
        n = rng.choice([_log(rng, 1, 16), _dim(rng, 17, 8192), _dim(rng, 17, 8192)])
        ic, oc = _dim(rng, 32, 8192), _dim(rng, 32, 8192)
        products = {"matmul": 1, "matmul_backward": 2, "gated": 2, "gated_backward": 4}[op]
        if 2.0 * products * n * ic * oc <= most:
            break
    case = dict(op=op, type=kind, N=n, IC=ic, OC=oc, act=rng.choice(list(ACTS) if op.startswith("matmul") else ["gelu", "silu", "sigmoid", "leaky_relu"]),
                bias=rng.random() < 0.6, pad=rng.choice([0, 0, 0, 8, 3]))
    if not op.endswith("backward"):
        case["save"] = rng.random() < 0.5
    if op == "matmul":
        case["residual"] = rng.random() < 0.5
    return case


def _clip_sizes(case):
    if case["kind"] == "network":
        sizes = [64 * 7 * 7 * 4, 64, 64, 64]
        inside = 64
        for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for b in range(blocks):
                sizes += [inside * width, width, width, width * 9 * width, width, width, width * 4 * width, 4 * width, 4 * width]
                if b == 0:
                    sizes += [inside * 4 * width, 4 * width, 4 * width]
                inside = 4 * width
        return sizes + [1000 * inside, 1000]
    g = torch.Generator().manual_seed(case["spread"])
    u = torch.rand(case["tensors"], generator=g, dtype=torch.float64)
    lo = max(1, case["largest"] // 64)
    return [case["largest"]] + [max(1, int(lo * (case["largest"] / lo) ** float(x))) for x in u[1:]]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "clip":
        n = sum(_clip_sizes(case))
        return {"bytes": 2 * size * n, "flops": 3 * n}
    n, ic, oc, bias = case["N"], case["IC"], case["OC"], int(case["bias"])
    if case["op"] == "matmul":
        return {"bytes": size * (n * ic + ic * oc + bias * oc + n * oc * (1 + int(case["residual"]) + int(case["save"]))), "flops": 2 * n * ic * oc}
    if case["op"] == "matmul_backward":
        return {"bytes": size * (n * oc * (1 if case["act"] == "none" else 2) + 2 * n * ic + 2 * ic * oc + bias * oc), "flops": 4 * n * ic * oc}
    if case["op"] == "gated":
        return {"bytes": size * (n * ic + 2 * ic * oc + 2 * bias * oc + n * oc * (1 + 2 * int(case["save"]))), "flops": 4 * n * ic * oc}
    return {"bytes": size * (3 * n * oc + 2 * n * ic + 4 * ic * oc + 2 * bias * oc), "flops": 8 * n * ic * oc}


# ---- inputs --------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case, made on the GPU from the seed alone; rows are `pad` elements apart from dense."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def rows(n, c, std):
        return (torch.randn(n, c + case["pad"], generator=g, device="cuda") * std).to(dtype)[:, :c]

    def vector(c):
        return (torch.randn(c, generator=g, device="cuda") * 0.1).to(dtype)

    if case["op"] == "clip":
        sizes = _clip_sizes(case)
        flat = (torch.randn(sum(sizes), generator=g, device="cuda") * case["scale"]).to(dtype)
        return {"grads": [t.clone() for t in flat.split(sizes)]}
    n, ic, oc, bias = case["N"], case["IC"], case["OC"], case["bias"]
    t = {"x": rows(n, ic, 1.0)}
    if case["op"].startswith("matmul"):
        t["w"] = rows(oc, ic, ic ** -0.5)
        if case["op"] == "matmul":
            t["bias"] = vector(oc) if bias else None
            t["r"] = rows(n, oc, 1.0) if case["residual"] else None
        else:
            t["z"] = rows(n, oc, 1.0) if case["act"] != "none" else None
            t["dy"] = rows(n, oc, 0.1)
    else:
        t["wg"], t["wu"] = rows(oc, ic, ic ** -0.5), rows(oc, ic, ic ** -0.5)
        if case["op"] == "gated":
            t["bg"], t["bu"] = (vector(oc), vector(oc)) if bias else (None, None)
        else:
            t["g"], t["u"], t["dh"] = rows(n, oc, 1.0), rows(n, oc, 1.0), rows(n, oc, 0.1)
    return t


def prepare(case, seed):
    """A program's tensors, and the output tensors it keeps from step to step."""
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "clip":
        # the clipped gradients go to one buffer, every tensor at a multiple of 64 elements, as an optimiser's bucket holds them
        starts = [0]
        for t in s["grads"]:
            starts.append(starts[-1] + (t.numel() + 63) // 64 * 64)
        s["bucket"] = torch.zeros(starts[-1], dtype=TYPES[case["type"]], device="cuda")
        s["out"] = [s["bucket"][a:a + t.numel()] for a, t in zip(starts, s["grads"])]
        s["norm"] = torch.empty(2, dtype=torch.float32, device="cuda")
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------

def _act(act, z):
    if act == "none":
        return z
    if act == "leaky_relu":
        return torch.where(z > 0, z, z * SLOPE)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    s = 1 / (1 + torch.exp(-z))
    return s if act == "sigmoid" else z * s


def _act_derivative(act, z):
    if act == "none":
        return torch.ones_like(z)
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, SLOPE)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if act == "sigmoid" else s * (1 + z * (1 - s))


def _plain_matmul(s, case, dtype):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(case["act"], z)
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(dtype), "z": z.to(dtype)} if case["save"] else {"y": y.to(dtype)}


def _plain_matmul_backward(s, case, dtype):
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_derivative(case["act"], s["z"].float())
    out = {"dx": (dz @ s["w"].float()).to(dtype), "dw": (dz.t() @ s["x"].float()).to(dtype)}
    if case["bias"]:
        out["db"] = dz.sum(0).to(dtype)
    return out


def _plain_gated(s, case, dtype):
    x = s["x"].float()
    g, u = x @ s["wg"].float().t(), x @ s["wu"].float().t()
    if case["bias"]:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    out = {"h": (_act(case["act"], g) * u).to(dtype)}
    if case["save"]:
        out["g"], out["u"] = g.to(dtype), u.to(dtype)
    return out


def _plain_gated_backward(s, case, dtype):
    g, u, dh, x = s["g"].float(), s["u"].float(), s["dh"].float(), s["x"].float()
    dg, du = dh * u * _act_derivative(case["act"], g), dh * _act(case["act"], g)
    out = {"dx": (dg @ s["wg"].float() + du @ s["wu"].float()).to(dtype), "dwg": (dg.t() @ x).to(dtype), "dwu": (du.t() @ x).to(dtype)}
    if case["bias"]:
        out["dbg"], out["dbu"] = dg.sum(0).to(dtype), du.sum(0).to(dtype)
    return out


def _plain_clip(s, case, dtype):
    squares = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]])
    norm = squares.sum().sqrt()
    coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
    c = coef.float()
    [out.copy_(t.float() * c) for out, t in zip(s["out"], s["grads"])]
    return {"norm": torch.stack([norm, coef]).float(), "bucket": s["bucket"]}


# ---- the library's calls -------------------------------------------------------------------------------------------

def _package():
    """The repository's package, whose folder's name is no Python identifier."""
    if "dragon_alpha_amd" not in sys.modules:
        import importlib.util
        folder = os.path.join(os.getcwd(), "dragon-alpha-v1.0_amd")
        spec = importlib.util.spec_from_file_location("dragon_alpha_amd", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules["dragon_alpha_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["dragon_alpha_amd"])
    return sys.modules["dragon_alpha_amd"]


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _step(t):
    return 0 if t is None else t.stride(0)


def _kept(s, key, make):
    """A workspace that the program makes once and keeps beside its tensors."""
    if key not in s:
        s[key] = make()
    return s[key]


def _own_run(s, case, dtype):
    dense = _package().Cuda_dense
    streams = [int(torch.cuda.current_stream().cuda_stream)]
    kind = dense.F32 if case["type"] == "f32" else dense.BF16
    if case["op"] == "clip":
        def plan():
            lengths = [t.numel() for t in s["grads"]]
            ws = torch.empty(dense.gradClip_workspace(len(lengths), lengths), dtype=torch.uint8, device="cuda")
            return [kind] * len(lengths), lengths, [t.data_ptr() for t in s["grads"]], [t.data_ptr() for t in s["out"]], ws
        types, lengths, src, dst, ws = _kept(s, "plan", plan)
        dense.gradClip(streams, 1, len(lengths), types, lengths, src, dst, case["max_norm"], 1e-6, s["norm"].data_ptr(), ws.data_ptr(), ws.numel())
        return {"norm": s["norm"], "bucket": s["bucket"]}
    n, ic, oc, act = case["N"], case["IC"], case["OC"], ACTS[case["act"]]

    def new(*shape):
        return torch.empty(shape, dtype=dtype, device="cuda")

    x = s["x"]
    if case["op"] == "matmul":
        ws = _kept(s, "ws", lambda: torch.empty(dense.matMul_fused_workspace(kind, n, ic, oc), dtype=torch.uint8, device="cuda"))
        y, z = new(n, oc), new(n, oc) if case["save"] else None
        dense.matMul_fused(streams, 1, kind, x.data_ptr(), _step(x), s["w"].data_ptr(), _step(s["w"]), _ptr(s["bias"]), act, SLOPE,
                           _ptr(s["r"]), _step(s["r"]), _ptr(z), _step(z), y.data_ptr(), oc, n, ic, oc, ws.data_ptr(), ws.numel())
        return {"y": y, "z": z} if case["save"] else {"y": y}
    if case["op"] == "matmul_backward":
        ws = _kept(s, "ws", lambda: torch.empty(dense.dmatMul_fused_workspace(kind, n, ic, oc), dtype=torch.uint8, device="cuda"))
        out = {"dx": new(n, ic), "dw": new(oc, ic)}
        if case["bias"]:
            out["db"] = new(oc)
        dense.dmatMul_fused(streams, 1, kind, s["dy"].data_ptr(), _step(s["dy"]), _ptr(s["z"]), _step(s["z"]), act, SLOPE,
                            x.data_ptr(), _step(x), s["w"].data_ptr(), _step(s["w"]), out["dx"].data_ptr(), ic, out["dw"].data_ptr(), ic,
                            _ptr(out.get("db")), n, ic, oc, ws.data_ptr(), ws.numel())
        return out
    if case["op"] == "gated":
        ws = _kept(s, "ws", lambda: torch.empty(dense.gatedMatMul_workspace(kind, n, ic, oc), dtype=torch.uint8, device="cuda"))
        h, g, u = new(n, oc), new(n, oc) if case["save"] else None, new(n, oc) if case["save"] else None
        dense.gatedMatMul(streams, 1, kind, x.data_ptr(), _step(x), s["wg"].data_ptr(), _step(s["wg"]), _ptr(s["bg"]),
                          s["wu"].data_ptr(), _step(s["wu"]), _ptr(s["bu"]), act, SLOPE, _ptr(g), _step(g), _ptr(u), _step(u),
                          h.data_ptr(), oc, n, ic, oc, ws.data_ptr(), ws.numel())
        return {"h": h, "g": g, "u": u} if case["save"] else {"h": h}
    ws = _kept(s, "ws", lambda: torch.empty(dense.dgatedMatMul_workspace(kind, n, ic, oc), dtype=torch.uint8, device="cuda"))
    out = {"dx": new(n, ic), "dwg": new(oc, ic), "dwu": new(oc, ic)}
    if case["bias"]:
        out["dbg"], out["dbu"] = new(oc), new(oc)
    dense.dgatedMatMul(streams, 1, kind, s["dh"].data_ptr(), _step(s["dh"]), s["g"].data_ptr(), _step(s["g"]), s["u"].data_ptr(), _step(s["u"]),
                       act, SLOPE, x.data_ptr(), _step(x), s["wg"].data_ptr(), _step(s["wg"]), s["wu"].data_ptr(), _step(s["wu"]),
                       out["dx"].data_ptr(), ic, out["dwg"].data_ptr(), ic, out["dwu"].data_ptr(), ic, _ptr(out.get("dbg")), _ptr(out.get("dbu")),
                       n, ic, oc, ws.data_ptr(), ws.numel())
    return out


def run(state):
    case = state["case"]
    dtype = TYPES[case["type"]]
    if own:
        return _own_run(state, case, dtype)
    plain = {"matmul": _plain_matmul, "matmul_backward": _plain_matmul_backward, "gated": _plain_gated, "gated_backward": _plain_gated_backward,
             "clip": _plain_clip}
    return plain[case["op"]](state, case, dtype)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    t = {k: (None if v is None else [a.double() for a in v] if isinstance(v, list) else v.double()) for k, v in _inputs(case, seed).items()}
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(a) for a in t["grads"]]))
        coef = torch.minimum(torch.ones_like(norm), case["max_norm"] / (norm + 1e-6))
        return {"norm": torch.stack([norm, coef]), "bucket": torch.cat([torch.nn.functional.pad(a * coef, (0, -a.numel() % 64)) for a in t["grads"]])}

    def value_and_slope(z):
        """act(z) and its derivative."""
        if case["act"] == "none":
            return z, None
        if case["act"] == "leaky_relu":
            slope = torch.full_like(z, SLOPE).masked_fill_(z > 0, 1.0)
            return z * slope, slope
        if case["act"] == "gelu":
            below = torch.special.ndtr(z)
            return z * below, below + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        s = torch.sigmoid(z)
        return (s, s * torch.sigmoid(-z)) if case["act"] == "sigmoid" else (z * s, s + z * s * torch.sigmoid(-z))

    def linear(x, w, bias):
        z = torch.mm(x, w.mT)
        return z if bias is None else z.add_(bias)

    if case["op"] == "matmul":
        z = linear(t["x"], t["w"], t["bias"])
        y = value_and_slope(z)[0]
        y = y if t["r"] is None else y + t["r"]
        return {"y": y, "z": z} if case["save"] else {"y": y}
    if case["op"] == "gated":
        g, u = linear(t["x"], t["wg"], t["bg"]), linear(t["x"], t["wu"], t["bu"])
        h = value_and_slope(g)[0] * u
        return {"h": h, "g": g, "u": u} if case["save"] else {"h": h}
    if case["op"] == "matmul_backward":
        dz = t["dy"] if t["z"] is None else t["dy"] * value_and_slope(t["z"])[1]
        out = {"dx": torch.mm(dz, t["w"]), "dw": torch.mm(dz.mT, t["x"])}
        return {**out, "db": dz.sum(0)} if case["bias"] else out
    value, slope = value_and_slope(t["g"])
    dg, du = t["dh"] * t["u"] * slope, t["dh"] * value
    out = {"dx": torch.mm(dg, t["wg"]) + torch.mm(du, t["wu"]), "dwg": torch.mm(dg.mT, t["x"]), "dwu": torch.mm(du.mT, t["x"])}
    return {**out, "dbg": dg.sum(0), "dbu": du.sum(0)} if case["bias"] else out
