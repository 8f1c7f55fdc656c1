"""The layer norm and the Muon update on their own: cases, inputs, plain forms and exact values.

Three operators, reached through the C ABI as a binding reaches it (pointers from aeth_malloc, outputs in buffers that the
program keeps):

  norm_fwd   aeth_ln_fwd_f32 / aeth_ln_fwd_twin_f32: layer norm over the last axis, with the row statistics that the
             backward pass needs (`saves`) or without them, with a bfloat16 copy of the output (`twin`) or without
  norm_bwd   aeth_ln_bwd_f32 / aeth_ln_bwd_twin_f32: its gradients (input, gamma, beta)
  muon       aeth_muon_multi_f32: one Muon step over a list of matrices: momentum, Newton-Schulz orthogonalisation of the
             update, step on the weights (`pass` "update"); aeth_newton_schulz_f32: the orthogonalisation alone ("ortho")

With `own` false, `run` works the same results out with elementary torch operations in float32.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5
NS = (3.4445, -4.7750, 2.0315)          # quintic of the Newton-Schulz step
LR, MOMENTUM, DECAY, STEPS = 0.02, 0.95, 0.01, 5

# the matrices of a training step of the three-convolution network (filters as [fH fW C, D], the dense layer behind them)
CNN3 = "27x32 288x64 576x128 2048x256"


def listed():
    return [
        # one sample through a network that serves requests: 256 features, no statistics kept; launch latency
        {"name": "norm fwd 1x256 serving", "op": "norm_fwd", "rows": 1, "cols": 256, "saves": False, "twin": False},
        # the hidden layer of a dense network in training, batch 128 (the benchmark's batch and width), both directions
        {"name": "norm bwd 128x256", "op": "norm_bwd", "rows": 128, "cols": 256, "twin": False},
        # every pixel of a 256x56x56x64 activation normalised over its channels, a bf16 convolution behind it
        {"name": "norm fwd 56x56 pixels x64 twin", "op": "norm_fwd", "rows": 256 * 56 * 56, "cols": 64, "saves": True, "twin": True},
        {"name": "norm bwd 56x56 pixels x64 twin", "op": "norm_bwd", "rows": 256 * 56 * 56, "cols": 64, "twin": True},
        # ragged: a row length that no vector width divides
        {"name": "norm bwd 5003x1537", "op": "norm_bwd", "rows": 5003, "cols": 1537, "twin": False},
        # long rows, many of them
        {"name": "norm fwd 16384x8192", "op": "norm_fwd", "rows": 16384, "cols": 8192, "saves": True, "twin": False},
        {"name": "norm bwd 16384x4096", "op": "norm_bwd", "rows": 16384, "cols": 4096, "twin": False},
        # one 3x3x64 filter bank of 64 filters (the headline convolution's)
        {"name": "muon 576x64", "op": "muon", "pass": "update", "shapes": "576x64", "nesterov": True},
        # a whole training step's matrices in one call
        {"name": "muon cnn3", "op": "muon", "pass": "update", "shapes": CNN3, "nesterov": True},
        # a ragged matrix, orthogonalised alone (as a test or another optimiser would)
        {"name": "ortho 1000x1537", "op": "muon", "pass": "ortho", "shapes": "1000x1537", "nesterov": False},
        # a wide layer alone, and the update of the largest square one
        {"name": "ortho 1024x4096", "op": "muon", "pass": "ortho", "shapes": "1024x4096", "nesterov": False},
        {"name": "muon 4096x4096", "op": "muon", "pass": "update", "shapes": "4096x4096", "nesterov": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "muon"])
    if op == "muon":
        if rng.random() < 0.4:          # a few layers of a small network at once
            shapes = ["%dx%d" % (_spread(rng, 16, 2048), _spread(rng, 10, 300)) for _ in range(rng.randint(2, 6))]
            return {"op": op, "pass": "update", "shapes": " ".join(shapes), "nesterov": rng.random() < 0.7}
        while True:
            r, c = _spread(rng, 24, 6000), _spread(rng, 24, 6000)
            if min(r, c) * r * c <= 4096 ** 3:
                break
        return {"op": op, "pass": rng.choice(["update", "ortho"]), "shapes": "%dx%d" % (r, c), "nesterov": rng.random() < 0.7}
    while True:
        cols = _spread(rng, 8, 20000)
        if rng.random() < 0.5:
            cols = -(-cols // 8) * 8
        rows = _spread(rng, 1, 400000)
        if rows * cols <= 1 << 26:
            break
    case = {"op": op, "rows": rows, "cols": cols, "twin": rng.random() < 0.3}
    if op == "norm_fwd":
        case["saves"] = rng.random() < 0.6
    return case


def _shapes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()]


def work(case):
    if case["op"] == "muon":
        size = flops = 0
        for r, c in _shapes(case):
            m, n = min(r, c), max(r, c)
            size += m * n
            # X X^T and the square of it are symmetric: half of their products; then the product with X
            flops += STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)
        # ortho: reads the matrix, writes the result; update: reads weights, gradient, momentum, writes weights, momentum
        return {"bytes": size * (8 if case["pass"] == "ortho" else 20), "flops": flops + 8 * size}
    rows, cols = case["rows"], case["cols"]
    n, twin = rows * cols, 2 if case["twin"] else 0
    if case["op"] == "norm_fwd":
        return {"bytes": n * (8 + twin) + 8 * cols + (8 * rows if case["saves"] else 0), "flops": 8 * n}
    return {"bytes": n * (12 + twin) + 8 * rows + 12 * cols, "flops": 14 * n}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _norm_inputs(case, seed):
    """Activations with a mean and a spread of each column's own (as behind a dense layer), gains around one, offsets
    around zero; for the backward pass the upstream gradient and the statistics that the forward pass saved."""
    g = _generator(seed)
    rows, cols = case["rows"], case["cols"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x = normal(rows, cols)
    x.mul_(0.5 + torch.rand(cols, generator=g, device="cuda")).add_(0.5 * normal(cols))
    t = {"x": x, "gamma": 1 + 0.1 * normal(cols), "beta": 0.1 * normal(cols)}
    if case["op"] == "norm_bwd":
        t["dy"] = normal(rows, cols).mul_(1e-2)
        mean = x.double().mean(1) if rows * cols <= 1 << 24 else x.mean(1)
        t["mean"] = mean.float()
        t["invstd"] = torch.rsqrt((x - t["mean"][:, None]).square_().mean(1) + EPS)
    return t


def _muon_inputs(case, seed):
    """Gradients as training gives them: a few strong directions over a floor of noise; the momentum has seen the like."""
    g = _generator(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    out = []
    for r, c in _shapes(case):
        k = max(1, min(r, c, 8))
        lean = normal(r, k) * torch.exp2(-torch.arange(k, device="cuda") / 2.0)
        strong = lean @ normal(k, c)
        grad = (strong + normal(r, c)).mul_(1e-3)
        mom = (3 * strong + normal(r, c)).mul_(1e-3)
        theta = normal(r, c).mul_(1 / math.sqrt(r))
        out.append({"theta": theta, "grad": grad, "mom": mom})
    return out


class _Span:
    """An array on the device as torch reads it (the interface that GPU array libraries share)."""

    def __init__(self, tensor, kind):
        self.tensor = tensor             # keeps the memory
        self.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": kind, "data": (tensor.ptr, False), "version": 2}


def _aether():
    at = os.path.join(os.getcwd(), "aether-ml_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import aether
    from aether import _lib
    return aether, _lib


def _buffer(shape, bf16=False):
    """(the framework's tensor, the same memory as torch sees it)"""
    aether, _ = _aether()
    t = aether.DeviceTensor(shape, np.uint16 if bf16 else np.float32)
    seen = torch.as_tensor(_Span(t, "<i2" if bf16 else "<f4"), device="cuda")
    return t, seen.view(torch.bfloat16) if bf16 else seen


def _filled(value):
    t, seen = _buffer(tuple(value.shape))
    seen.copy_(value)
    return t, seen


def prepare(case, seed):
    if case["op"] == "muon":
        t = _muon_inputs(case, seed)
        return _muon_state(case, t) if own else {"case": case, "t": t}
    t = _norm_inputs(case, seed)
    return _norm_state(case, t) if own else {"case": case, "t": t}


def _norm_state(case, t):
    """What a program keeps for the framework's calls: every tensor in the framework's memory, outputs included."""
    _, _lib = _aether()
    lib = _lib.lib()
    rows, cols = case["rows"], case["cols"]
    p = {k: _filled(v) for k, v in t.items()}
    outs = [("y" if case["op"] == "norm_fwd" else "dx", (rows, cols), False)]
    if case["twin"]:
        outs.append((outs[0][0] + "16", (rows, cols), True))
    if case["op"] == "norm_bwd":
        outs += [("dgamma", (cols,), False), ("dbeta", (cols,), False)]
    elif case["saves"]:
        outs += [("mean", (rows,), False), ("invstd", (rows,), False)]
    p.update({name: _buffer(shape, bf16) for name, shape, bf16 in outs})
    at = lambda *names: [p[k][0].ptr if k in p else None for k in names]  # noqa: E731
    if case["op"] == "norm_fwd":
        args = at("x", "gamma", "beta", "mean", "invstd", "y") + (at("y16") if case["twin"] else []) + [rows, cols, EPS]
        call = lib.aeth_ln_fwd_twin_f32 if case["twin"] else lib.aeth_ln_fwd_f32
    else:
        args = at("x", "dy", "gamma", "mean", "invstd", "dx") + (at("dx16") if case["twin"] else []) + at("dgamma", "dbeta") + [rows, cols]
        call = lib.aeth_ln_bwd_twin_f32 if case["twin"] else lib.aeth_ln_bwd_f32
    return {"case": case, "call": call, "args": args, "check": _lib.check, "keep": p, "out": {name: p[name][1] for name, _, _ in outs}}


def _muon_state(case, t):
    import ctypes as C
    _, _lib = _aether()
    lib = _lib.lib()
    p = [{k: _filled(v) for k, v in m.items()} for m in t]
    if case["pass"] == "ortho":
        (r, c), = _shapes(case)
        o = _buffer((r, c))
        return {"case": case, "call": lib.aeth_newton_schulz_f32, "args": [p[0]["grad"][0].ptr, o[0].ptr, r, c, STEPS],
                "check": _lib.check, "keep": (p, o), "out": {"o": o[1]}}
    n = len(p)
    table = [(C.c_void_p * n)(*[m[k][0].ptr for m in p]) for k in ("theta", "grad", "mom")]
    sizes = [(C.c_int * n)(*[s[k] for s in _shapes(case)]) for k in (0, 1)]
    args = [n] + table + sizes + [LR, MOMENTUM, int(case["nesterov"]), DECAY, STEPS]
    return {"case": case, "call": lib.aeth_muon_multi_f32, "args": args, "check": _lib.check, "keep": p,
            "out": [{"theta": m["theta"][1], "mom": m["mom"][1]} for m in p]}


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _norm_fwd(t, saves, twin):
    x = t["x"]
    mean = x.sum(1, keepdim=True) / x.shape[1]
    d = x - mean
    invstd = 1 / torch.sqrt((d * d).sum(1, keepdim=True) / x.shape[1] + EPS)
    y = d * invstd * t["gamma"] + t["beta"]
    out = {"y": y}
    if twin:
        out["y16"] = y.to(torch.bfloat16)
    if saves:
        out.update(mean=mean.reshape(-1), invstd=invstd.reshape(-1))
    return out


def _norm_bwd(t, twin):
    x, dy, invstd = t["x"], t["dy"], t["invstd"][:, None]
    xhat = (x - t["mean"][:, None]) * invstd
    dg = dy * t["gamma"]
    c1 = dg.sum(1, keepdim=True) / x.shape[1]
    c2 = (dg * xhat).sum(1, keepdim=True) / x.shape[1]
    dx = invstd * (dg - c1 - xhat * c2)
    out = {"dx": dx, "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if twin:
        out["dx16"] = dx.to(torch.bfloat16)
    return out


def _orthogonal(u):
    a, b, c = NS
    tall = u.shape[0] > u.shape[1]
    x = u.t() if tall else u
    norm = torch.sqrt((x * x).sum())
    x = x / torch.where(norm > 0, norm, torch.ones_like(norm))
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t().contiguous() if tall else x


def _muon(m, nesterov):
    theta, grad, mom = m["theta"], m["grad"], m["mom"]
    mom.mul_(MOMENTUM).add_(grad)
    o = _orthogonal(grad + MOMENTUM * mom if nesterov else mom)
    theta.mul_(1 - LR * DECAY).sub_(LR * math.sqrt(max(1.0, theta.shape[1] / theta.shape[0])) * o)
    return {"theta": theta, "mom": mom}


def run(state):
    case = state["case"]
    if own:
        state["check"](state["call"](*state["args"]))
        return state["out"]
    t = state["t"]
    if case["op"] == "norm_fwd":
        return _norm_fwd(t, case["saves"], case["twin"])
    if case["op"] == "norm_bwd":
        return _norm_bwd(t, case["twin"])
    if case["pass"] == "ortho":
        return {"o": _orthogonal(t[0]["grad"])}
    return [_muon(m, case["nesterov"]) for m in t]


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------


def _exact_norm(case, seed):
    t = _norm_inputs(case, seed)
    gamma, beta = t["gamma"].double(), t["beta"].double()
    cols, rows = case["cols"], case["rows"]
    step = max(1, (1 << 26) // cols)
    parts, dgamma, dbeta = [], torch.zeros_like(gamma), torch.zeros_like(gamma)
    for at in range(0, rows, step):
        x = t["x"][at:at + step].double()
        if case["op"] == "norm_fwd":
            var, mean = torch.var_mean(x, 1, correction=0)
            inv = (var + EPS) ** -0.5
            parts.append(((x - mean[:, None]) * inv[:, None] * gamma + beta, mean, inv))
        else:
            dy, inv = t["dy"][at:at + step].double(), t["invstd"][at:at + step].double()[:, None]
            xhat = (x - t["mean"][at:at + step].double()[:, None]) * inv
            back = dy * gamma
            # the Jacobian of a row: project the constant and xhat out, divide by the spread
            parts.append((inv * (back - back.mean(1, keepdim=True) - xhat * torch.mean(back * xhat, 1, keepdim=True)),))
            dgamma += torch.einsum("rc,rc->c", dy, xhat)
            dbeta += dy.sum(0)
    whole = [torch.cat(p) for p in zip(*parts)]
    name = "y" if case["op"] == "norm_fwd" else "dx"
    out = {name: whole[0]}
    if case["twin"]:
        out[name + "16"] = whole[0]
    if case["op"] == "norm_bwd":
        out.update(dgamma=dgamma, dbeta=dbeta)
    elif case["saves"]:
        out.update(mean=whole[1], invstd=whole[2])
    return out


def _exact_orthogonal(u):
    """The matrix with every singular value s replaced by p(p(...p(s))), p(s) = a s + b s^3 + c s^5, by products that act
    on the longer side through the Gram matrix of the shorter one."""
    a, b, c = NS
    u = u.double()
    x = u / torch.linalg.matrix_norm(u)
    wide = x.shape[1] >= x.shape[0]
    eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.mm(x, x.T) if wide else torch.mm(x.T, x)
        q = a * eye + torch.mm(gram, b * eye + c * gram)
        x = torch.mm(q, x) if wide else torch.mm(x, q)
    return x


def exact(case, seed):
    if case["op"] != "muon":
        return _exact_norm(case, seed)
    out = []
    for m in _muon_inputs(case, seed):
        if case["pass"] == "ortho":
            return {"o": _exact_orthogonal(m["grad"])}
        grad, theta = m["grad"].double(), m["theta"].double()
        mom = MOMENTUM * m["mom"].double() + grad
        o = _exact_orthogonal(MOMENTUM * mom + grad if case["nesterov"] else mom)
        gain = math.sqrt(max(1.0, theta.shape[1] / theta.shape[0]))
        out.append({"theta": theta - LR * DECAY * theta - LR * gain * o, "mom": mom})
    return out
