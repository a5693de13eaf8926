"""The operators of a residual policy torso as measured cases: layer norm, the linear map with bias,
activation and residual, and the gated projection, each forward and backward.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded once
at the end) or, with `own` set, through t8b.ops. `exact` restates the definitions in 64 bits.
Sizes: 512 is the policy network's hidden width, 151 its observation, 33 its outputs (32 query
features and the value), 32,768 the fights of one GPU's rollout, 65,536 a PPO minibatch and 96 an
evaluation's fights; 1,408 is 8/3 of 512 rounded up to a tile. The others are generic.
"""
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # one evaluation of 96 fights: a norm whose time is its launch
        dict(name="norm fwd 96x512", op="norm", way="fwd", rows=96, n=512, type="bf16", out="bf16", param="f32",
             slack=0),
        # a rollout decision: the fp32 residual stream normalised into the matrix products' type
        dict(name="norm fwd 32768x512", op="norm", way="fwd", rows=32768, n=512, type="f32", out="bf16", param="f32",
             slack=0),
        # raw observations, whose 151 features leave every other row off a 16-byte boundary
        dict(name="norm bwd 65536x151", op="norm", way="bwd", rows=65536, n=151, type="f32", out="f32", param="f32",
             residual=False, slack=0),
        # several minibatches' gradient through a block's norm, joined with the residual branch's gradient
        dict(name="norm bwd 262144x512", op="norm", way="bwd", rows=262144, n=512, type="bf16", out="bf16",
             param="f32", residual=True, slack=0),
        # one fight against a person: a single row through a hidden layer
        dict(name="linear fwd 1x512x512", op="linear", way="fwd", rows=1, n=512, m=512, type="bf16", out="bf16",
             bias="f32", act="tanh", residual=False, save=False, slack=0),
        # the output heads over a rollout decision: 33 fp32 columns
        dict(name="linear fwd 32768x512x33", op="linear", way="fwd", rows=32768, n=512, m=33, type="bf16", out="f32",
             bias="f32", act="none", residual=False, save=False, slack=0),
        # a gated block's way back to the residual stream, over a rollout decision
        dict(name="linear fwd 32768x1408x512", op="linear", way="fwd", rows=32768, n=1408, m=512, type="bf16",
             out="bf16", bias="bf16", act="none", residual=True, save=False, slack=0),
        # a hidden layer's gradients over a minibatch
        dict(name="linear bwd 65536x512x512", op="linear", way="bwd", rows=65536, n=512, m=512, type="bf16",
             bias="f32", act="gelu", slack=0),
        # one fight: a single row through both projections
        dict(name="gated fwd 1x512x1408", op="gated", way="fwd", rows=1, n=512, m=1408, type="bf16", bias="none",
             act="silu", save=False, slack=0),
        # a minibatch's forward pass, which keeps what its gradient needs
        dict(name="gated fwd 65536x512x1408", op="gated", way="fwd", rows=65536, n=512, m=1408, type="bf16",
             bias="none", act="silu", save=True, slack=0),
        # the same minibatch's gradients: the largest case
        dict(name="gated bwd 65536x512x1408", op="gated", way="bwd", rows=65536, n=512, m=1408, type="bf16",
             bias="none", act="silu", slack=0),
        # a ragged batch in half precision, its input a column range of a wider buffer
        dict(name="gated bwd 2051x1001x1333", op="gated", way="bwd", rows=2051, n=1001, m=1333, type="f16",
             bias="f32", act="gelu", slack=6),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Any operator and direction; rows from one to a minibatch, widths from 33 to 2,048 (norms to
    8,192), one in two off a multiple of 8; inputs packed or inside a wider buffer."""
    op, way = rng.choice(["norm", "linear", "gated"]), rng.choice(["fwd", "bwd"])
    slack = rng.choice([0, 0, 8, 3])

    def width(high):
        w = _log(rng, 33, high)
        return w if rng.random() < 0.5 else -(-w // 8) * 8

    if op == "norm":
        case = dict(op=op, way=way, rows=_log(rng, 1, 262144), n=width(8192), type=rng.choice(list(TYPES)),
                    param="f32", slack=slack)
        case["out"] = rng.choice([case["type"], "bf16"])
        if case["type"] != "f32":
            case["param"] = rng.choice(["f32", case["type"]])
        if way == "bwd":
            case["residual"] = rng.random() < 0.5
        case["rows"] = max(1, min(case["rows"], 262144 * 512 // (2 * case["n"])))
        return case
    case = dict(op=op, way=way, rows=_log(rng, 1, 65536), n=width(2048), m=width(2048), type=rng.choice(["bf16", "f16"]),
                bias=rng.choice(["none", "f32", "own"]), slack=slack,
                act=rng.choice(["none", "relu", "gelu", "silu", "tanh"] if op == "linear" else ["gelu", "silu", "relu", "tanh"]))
    case["bias"] = case["type"] if case["bias"] == "own" else case["bias"]
    if way == "fwd":
        case["save"] = rng.random() < 0.5
        if op == "linear":
            case["residual"] = rng.random() < 0.5
            case["out"] = rng.choice([case["type"], case["type"], "f32"])
    most = 65536 * 512 * 1408 // 2
    case["rows"] = max(1, min(case["rows"], most // (case["n"] * case["m"])))
    return case


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def matrix(values, dtype):
        """`values` as a user holds them: packed, or a column range of a wider buffer."""
        if not case["slack"]:
            return values.to(dtype)
        wide = torch.zeros(values.shape[0], values.shape[1] + case["slack"], device="cuda", dtype=dtype)
        wide[:, : values.shape[1]] = values
        return wide[:, : values.shape[1]]

    rows, n, t = case["rows"], case["n"], TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "norm":
        p = TYPES[case["param"]]
        # a residual stream: features of different scale and offset, rows of different size
        x = normal(rows, n) * (0.25 + normal(n).abs()) + 0.5 * normal(n)
        s["x"] = matrix(x * (0.5 + torch.rand(rows, 1, device="cuda", generator=g)), t)
        s["weight"] = (1 + 0.2 * normal(n)).to(p)
        s["bias"] = (0.1 * normal(n)).to(p)
        if case["way"] == "bwd":
            x32 = s["x"].float()
            s["mean"] = x32.mean(1)
            s["rstd"] = torch.rsqrt((x32 - s["mean"][:, None]).square().mean(1) + EPS)
            s["dy"] = (normal(rows, n) / 64).to(TYPES[case["out"]])
            s["residual"] = (normal(rows, n) / 64).to(t) if case["residual"] else None
        return s
    columns = case["m"] * (2 if case["op"] == "gated" else 1)
    s["x"] = matrix(normal(rows, n), t)
    s["weight"] = (normal(columns, n) / math.sqrt(n)).to(t)
    s["bias"] = None if case["bias"] == "none" else (0.1 * normal(columns)).to(TYPES[case["bias"]])
    if case["way"] == "fwd":
        if case.get("residual"):
            s["residual"] = normal(rows, case["m"]).to(TYPES[case["out"]])
        else:
            s["residual"] = None
    else:
        s["dy"] = (normal(rows, case["m"]) / 64).to(t)
        s["pre"] = None
        if case["act"] != "none" or case["op"] == "gated":  # as the forward pass left it
            pre = s["x"].float() @ s["weight"].float().t()
            s["pre"] = (pre if s["bias"] is None else pre + s["bias"].float()).to(t)
    return s


# ------------------------------------------------------------------ plain form
def _activation(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "tanh":
        return 1 - torch.tanh(z).square()
    if name == "silu":
        sigma = 1 / (1 + torch.exp(-z))
        return sigma * (1 + z * (1 - sigma))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _plain(s):
    case, x = s["case"], s["x"].float()
    t = s["x"].dtype
    if case["op"] == "norm":
        w = s["weight"].float()
        if case["way"] == "fwd":
            mean = x.mean(1)
            centred = x - mean[:, None]
            rstd = torch.rsqrt(centred.square().mean(1) + EPS)
            y = centred * rstd[:, None] * w + s["bias"].float()
            return {"y": y.to(TYPES[case["out"]]), "mean": mean, "rstd": rstd}
        dy = s["dy"].float()
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * w
        dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["residual"].float()
        return {"dx": dx.to(t), "dweight": (dy * xhat).sum(0).to(s["weight"].dtype),
                "dbias": dy.sum(0).to(s["bias"].dtype)}
    w, b = s["weight"].float(), s["bias"]
    if case["way"] == "fwd":
        z = x @ w.t()
        if b is not None:
            z = z + b.float()
        if case["op"] == "linear":
            y = _activation(z, case["act"])
            if s["residual"] is not None:
                y = y + s["residual"].float()
            y = y.to(TYPES[case["out"]])
        else:
            gate, up = z[:, : case["m"]], z[:, case["m"]:]
            y = (_activation(gate, case["act"]) * up).to(t)
        return {"y": y, "pre": z.to(t)} if case["save"] else {"y": y}
    dy = s["dy"].float()
    if case["op"] == "linear":
        dz = dy if s["pre"] is None else dy * _slope(s["pre"].float(), case["act"])
    else:
        gate, up = s["pre"].float().split(case["m"], 1)
        dz = torch.cat([dy * up * _slope(gate, case["act"]), dy * _activation(gate, case["act"])], 1)
    out = {"dx": (dz @ w).to(t), "dweight": (dz.t() @ x).to(t)}
    if b is not None:
        out["dbias"] = dz.sum(0).to(b.dtype)
    return out


# ------------------------------------------------------------------ the framework's operators
def _ops():
    at = str(Path(__file__).resolve().parent.parent / "tekken8-agent_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from t8b import ops
    return ops


def _own(s):
    ops, case = _ops(), s["case"]
    if case["op"] == "norm":
        if case["way"] == "fwd":
            y, mean, rstd = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=TYPES[case["out"]],
                                           save=True)
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dweight, dbias = ops.layer_norm_backward(s["dy"], s["x"], s["weight"], s["bias"], s["mean"], s["rstd"],
                                                     residual_gradient=s["residual"])
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    forward, backward = (ops.linear, ops.linear_backward) if case["op"] == "linear" else (ops.gated, ops.gated_backward)
    if case["way"] == "fwd":
        more = dict(residual=s["residual"], out_dtype=TYPES[case["out"]]) if case["op"] == "linear" else {}
        y = forward(s["x"], s["weight"], s["bias"], activation=case["act"], save=case["save"], **more)
        return {"y": y[0], "pre": y[1]} if case["save"] else {"y": y}
    dx, dweight, dbias = backward(s["dy"], s["x"], s["weight"], s["bias"], s["pre"], activation=case["act"])
    out = {"dx": dx, "dweight": dweight}
    if dbias is not None:
        out["dbias"] = dbias
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the least a pass has to do
def work(case):
    rows, n = case["rows"], case["n"]
    size = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
    e = size[case["type"]]
    if case["op"] == "norm":
        p, o = size[case["param"]], size[case["out"]]
        if case["way"] == "fwd":
            return {"bytes": rows * n * (e + o) + 8 * rows + 2 * n * p, "flops": 8 * rows * n}
        return {"bytes": rows * n * (2 * e + o + (e if case["residual"] else 0)) + 8 * rows + 3 * n * p,
                "flops": 14 * rows * n}
    m = case["m"]
    columns = m * (2 if case["op"] == "gated" else 1)
    b = size[case["bias"]] * columns
    if case["way"] == "fwd":
        o = size[case.get("out", case["type"])]
        moved = e * (rows * n + columns * n) + b + o * rows * m * (2 if case.get("residual") else 1)
        return {"bytes": moved + (e * rows * columns if case["save"] else 0), "flops": 2 * rows * n * columns}
    kept = 0 if case["act"] == "none" and case["op"] == "linear" else e * rows * columns
    return {"bytes": e * (rows * m + 2 * rows * n + 2 * columns * n) + kept + b, "flops": 4 * rows * n * columns}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and k in ("weight", "bias")}
    rows, step = case["rows"], max(1, (1 << 25) // max(case["n"], 2 * case.get("m", 1)))
    parts, sums = [], None

    def sigmoid(v):
        return torch.sigmoid(v)

    def phi(v):
        return 0.5 * torch.erfc(-v / math.sqrt(2.0))

    act = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "tanh": lambda v: v.tanh(),
           "silu": lambda v: v * sigmoid(v), "gelu": lambda v: v * phi(v)}
    slope = {"none": lambda v: torch.ones_like(v), "relu": lambda v: (v > 0).double(), "tanh": lambda v: v.cosh().pow(-2),
             "silu": lambda v: sigmoid(v) + v * sigmoid(v) * sigmoid(-v),
             "gelu": lambda v: phi(v) + v * (-v.square() / 2).exp() / math.sqrt(2 * math.pi)}
    for at in range(0, rows, step):
        part = {k: s[k][at:at + step].double() for k in ("x", "dy", "pre", "residual", "mean", "rstd")
                if isinstance(s.get(k), torch.Tensor)}
        x = part["x"]
        if case["op"] == "norm" and case["way"] == "fwd":
            var, mean = torch.var_mean(x, 1, unbiased=False)
            rstd = (var + EPS).pow(-0.5)
            parts.append({"y": torch.addcmul(d["bias"], (x - mean[:, None]) * rstd[:, None], d["weight"]),
                          "mean": mean, "rstd": rstd})
            continue
        if case["op"] == "norm":
            r, dy, n = part["rstd"][:, None], part["dy"], case["n"]
            h, g = (x - part["mean"][:, None]) * r, part["dy"] * d["weight"]
            dx = r / n * (n * g - g.sum(1)[:, None] - h * torch.einsum("ij,ij->i", g, h)[:, None])
            parts.append({"dx": dx + part.get("residual", 0)})
            total = {"dweight": torch.einsum("ij,ij->j", dy, h), "dbias": dy.sum(0)}
        else:
            f, df, m = act[case["act"]], slope[case["act"]], case["m"]
            if case["way"] == "fwd":
                z = torch.einsum("ik,jk->ij", x, d["weight"]) + d.get("bias", 0)
                y = f(z) + part.get("residual", 0) if case["op"] == "linear" else f(z[:, :m]) * z[:, m:]
                parts.append({"y": y, "pre": z} if case["save"] else {"y": y})
                continue
            dy, z = part["dy"], part.get("pre")
            if case["op"] == "gated":
                dz = torch.hstack([df(z[:, :m]) * z[:, m:] * dy, f(z[:, :m]) * dy])
            else:
                dz = dy if z is None else dy * df(z)
            parts.append({"dx": torch.einsum("ij,jk->ik", dz, d["weight"])})
            total = {"dweight": torch.einsum("ij,ik->jk", dz, x)}
            if "bias" in d:
                total["dbias"] = dz.sum(0)
        sums = total if sums is None else {k: sums[k] + v for k, v in total.items()}
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out.update(sums or {})
    return out
