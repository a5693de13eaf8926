"""The torso operators (t8b.ops) against their formulas in 64 bits on the same inputs.

Bounds, derived from how each value is computed (u = half the output type's spacing: 2^-8 for bf16's
8-bit significand, 2^-11 for f16, 2^-24 for fp32, relative; half f16's smallest spacing absolute):
  - a product sum of k terms in fp32: (k + 16) 2^-23 sum|terms|, whatever the order;
  - what a matrix product reads rounded to the operands' type: u sum|terms|;
  - an activation or its slope in fp32 through exp and erf: 2^-19 (1 + |z|);
  - a norm's sums over at most 16 registers, 32 lanes and 16 warps (80 additions): 2^-17.
"""
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = 1e-5


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}


def unit(t):
    return next(UNIT[k] for k, v in types().items() if v is t)


def tiny(t):
    return next(TINY[k] for k, v in types().items() if v is t)


def close(got, want, bound, name=""):
    """|got - want| <= bound + the output's own rounding, element by element."""
    import torch
    assert got.shape == want.shape, (name, got.shape, want.shape)
    limit = bound + unit(got.dtype) * (1 + 2 ** -8) * want.abs() + tiny(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (name, int(bad.sum()), float((off / limit).max()), torch.nonzero(bad)[:4].tolist())


def matrix(g, rows, columns, dtype, slack=0, shift=0, scale=1.0):
    """Normal values as a column range of a wider buffer: `slack` columns wider, from column `shift`."""
    import torch
    wide = torch.full((rows, columns + slack), float("nan"), device="cuda", dtype=dtype)
    view = wide[:, shift:shift + columns]
    view.copy_(torch.randn(rows, columns, device="cuda", generator=g) * scale)
    return view


def act64(z, name):
    import torch
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "tanh":
        return z.tanh(), 1 - z.tanh() ** 2
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * phi, phi + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5
    return z, torch.ones_like(z)


# ------------------------------------------------------------------ layer norm
NORM_SIZES = [(1, 1), (1, 512), (3, 7), (5, 33), (96, 512), (300, 151), (40, 256), (11, 513), (7, 1000), (33, 2048),
              (3, 8192), (3, 8193), (2, 20001), (5000, 130)]
NORM_TYPES = [("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("bf16", "bf16", "f32"), ("bf16", "f32", "bf16"),
              ("f16", "f16", "f16"), ("f16", "bf16", "f32")]


def norm64(x, w, b):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = (x.var(-1, unbiased=False, keepdim=True) + EPS) ** -0.5
    xhat = (x - mean) * rstd
    # what the statistics and xhat may be off by, relative to 2^-17
    slip = xhat.abs() + rstd * x.abs().mean(-1, keepdim=True)
    w = 1.0 if w is None else w.double()
    return xhat * w + (0.0 if b is None else b.double()), mean, rstd, xhat, slip, w


@pytest.mark.parametrize("rows,n", NORM_SIZES)
@pytest.mark.parametrize("xt,yt,pt", NORM_TYPES)
def test_layer_norm(cuda, rows, n, xt, yt, pt):
    import torch
    from t8b import ops
    T = types()
    g = torch.Generator(device="cuda").manual_seed(rows * 31 + n)
    for slack, shift in ((0, 0), (5, 3), (8, 0)):
        x = matrix(g, rows, n, T[xt], slack, shift, 3.0)
        x += torch.randn(rows, 1, device="cuda", generator=g).to(T[xt])
        w = (1 + 0.3 * torch.randn(n, device="cuda", generator=g)).to(T[pt])
        b = torch.randn(n, device="cuda", generator=g).to(T[pt])
        for weight, bias in ((w, b), (None, None), (w, None), (None, b)):
            y, mean, rstd = ops.layer_norm(x, weight, bias, EPS, out_dtype=T[yt], save=True)
            want, m, r, xhat, slip, w64 = norm64(x, weight, bias)
            assert y.dtype is T[yt]
            close(mean, m[:, 0], 2 ** -17 * x.double().abs().mean(-1))
            close(rstd, r[:, 0], 2 ** -17 * r[:, 0] * (1 + (r * x.double().abs().mean(-1, keepdim=True))[:, 0]))
            size = 2 ** -17 * slip * (w64.abs() if weight is not None else 1.0)
            close(y, want, size + 2 ** -22 * (bias.double().abs() if bias is not None else 0.0))
            assert torch.equal(y, ops.layer_norm(x, weight, bias, EPS, out_dtype=T[yt]))


@pytest.mark.parametrize("rows,n", NORM_SIZES)
@pytest.mark.parametrize("xt,yt,pt", NORM_TYPES)
def test_layer_norm_backward(cuda, rows, n, xt, yt, pt):
    import torch
    from t8b import ops
    T = types()
    g = torch.Generator(device="cuda").manual_seed(rows * 37 + n)
    for slack, shift, residual, affine in ((0, 0, True, True), (5, 3, False, True), (8, 0, True, False)):
        x = matrix(g, rows, n, T[xt], slack, shift, 2.0)
        dy = matrix(g, rows, n, T[yt], slack, shift)
        res = matrix(g, rows, n, T[xt], slack, shift) if residual else None
        w = (1 + 0.3 * torch.randn(n, device="cuda", generator=g)).to(T[pt]) if affine else None
        b = torch.zeros(n, device="cuda", dtype=T[pt]) if affine else None
        _, m, r, xhat, slip, w64 = norm64(x, w, b)
        mean, rstd = m[:, 0].float(), r[:, 0].float()
        got = ops.layer_norm_backward(dy, x, w, b, mean, rstd, residual_gradient=res)
        d = dy.double()
        gw = d * w64
        dx = r * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
        mags = gw.abs() + gw.abs().mean(-1, keepdim=True) + (xhat.abs() + slip) * (gw * slip).abs().mean(-1, keepdim=True)
        bound = 2 ** -17 * r * mags
        if residual:
            dx = dx + res.double()
            bound = bound + 2 ** -23 * res.double().abs()
        close(got[0], dx, bound, "dx")
        if not affine:
            assert got[1] is None and got[2] is None
            continue
        close(got[1], (d * xhat).sum(0), 2 ** -17 * (d.abs() * slip).sum(0), "dweight")
        close(got[2], d.sum(0), 2 ** -17 * d.abs().sum(0), "dbias")
        again = ops.layer_norm_backward(dy, x, w, b, mean, rstd, residual_gradient=res)
        assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("rows,n", [(13, 9), (41, 125), (29, 126), (19, 250), (23, 509), (9, 510), (2500, 515), (11, 4099),
                                    (9, 8185), (9, 8190), (3000, 1)])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_layer_norm_rows_that_start_off_a_vectors_boundary(cuda, rows, n, xt, yt):
    """Odd rows whose neighbours are NaN: packs shared between rows are read and written in part."""
    import torch
    from t8b import ops
    T = types()
    g = torch.Generator(device="cuda").manual_seed(rows * 41 + n)
    x, dy = matrix(g, rows, n, T[xt], 8, 0, 2.0), matrix(g, rows, n, T[yt], 16, 0)
    w, b = 1 + 0.3 * torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g)
    for at in (x, x.contiguous()):
        y, mean, rstd = ops.layer_norm(at, w, b, EPS, out_dtype=T[yt], save=True)
        want, m, r, xhat, slip, w64 = norm64(x, w, b)
        close(y, want, 2 ** -17 * slip * w64.abs() + 2 ** -22 * b.double().abs(), "y")
        close(mean, m[:, 0], 2 ** -17 * x.double().abs().mean(-1), "mean")
        dx, dw, db = ops.layer_norm_backward(dy, at, w, b, mean, rstd, residual_gradient=at)
        d = dy.double()
        gw = d * w64
        ref = r * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
        mags = gw.abs() + gw.abs().mean(-1, keepdim=True) + (xhat.abs() + slip) * (gw * slip).abs().mean(-1, keepdim=True)
        close(dx, ref + x.double(), 2 ** -16 * r * mags + 2 ** -22 * x.double().abs(), "dx")
        close(dw, (d * xhat).sum(0), 2 ** -16 * (d.abs() * slip).sum(0), "dweight")
        close(db, d.sum(0), 2 ** -17 * d.abs().sum(0), "dbias")


def test_layer_norm_rows_that_are_not_finite_and_constant_rows(cuda):
    """A row with an infinity or NaN is NaN as the formula says and touches no other row; a constant
    row gives the bias; rows whose mean is far above their spread keep their variance."""
    import torch
    from t8b import ops
    x = torch.randn(64, 512, device="cuda")
    clean = ops.layer_norm(x)
    x[3, 5] = float("inf")
    x[7, 511] = float("nan")
    x[9] = 2.5
    y = ops.layer_norm(x)
    for row in (3, 7):
        assert torch.isnan(y[row]).all()
    assert torch.equal(y[9], torch.zeros(512, device="cuda"))
    keep = [i for i in range(64) if i not in (3, 7, 9)]
    assert torch.equal(y[keep], clean[keep])
    far = 4096.0 + torch.randn(16, 512, device="cuda")
    want, *_, slip, _ = norm64(far, None, None)
    close(ops.layer_norm(far), want, 2 ** -17 * slip)


# ------------------------------------------------------------------ linear and gated
LINEAR_SIZES = [(1, 1, 1), (1, 512, 512), (2, 3, 5), (3, 64, 32), (17, 151, 33), (33, 40, 200), (128, 64, 256),
                (129, 512, 513), (257, 1001, 77), (300, 129, 1030), (1024, 640, 384), (8, 2048, 2048)]
ACTS = ["none", "relu", "gelu", "silu", "tanh"]


def linear64(x, w, b):
    z = x.double() @ w.double().T
    size = x.double().abs() @ w.double().abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, (x.shape[1] + 16) * 2.0 ** -23 * size


def bias_of(g, kind, columns, E):
    import torch
    if kind == "none":
        return None
    return (0.5 * torch.randn(columns, device="cuda", generator=g)).to(torch.float32 if kind == "f32" else E)


@pytest.mark.parametrize("rows,n,m", LINEAR_SIZES + [(40000, 192, 512)])
@pytest.mark.parametrize("et", ["bf16", "f16"])
def test_linear(cuda, rows, n, m, et):
    import torch
    from t8b import ops
    E = types()[et]
    g = torch.Generator(device="cuda").manual_seed(rows + 3 * n + 5 * m)
    for k, (act, bias, residual, out, save, slack) in enumerate([
            ("none", "none", False, E, False, 0), ("tanh", "f32", False, E, False, 0), ("gelu", "own", True, E, True, 0),
            ("silu", "f32", True, torch.float32, False, 8), ("relu", "none", True, torch.float32, True, 3),
            ("none", "f32", False, torch.float32, False, 0), ("tanh", "own", True, E, False, 5),
            ("gelu", "f32", False, E, True, 0)]):
        x = matrix(g, rows, n, E, slack, slack // 2 if slack != 8 else 0)
        w = matrix(g, m, n, E, slack, 0, n ** -0.5)
        b = bias_of(g, bias, m, E)
        r = matrix(g, rows, m, out, slack, 0) if residual else None
        got = ops.linear(x, w, b, activation=act, residual=r, out_dtype=out, save=save)
        y, pre = got if save else (got, None)
        z, slip = linear64(x, w, b)
        a, _ = act64(z, act)
        bound = 1.2 * slip + 2.0 ** -19 * (1 + z.abs()) * (act != "none")
        if residual:
            a, bound = a + r.double(), bound + 2 ** -23 * (a.abs() + r.double().abs())
        assert y.dtype is out
        close(y, a, bound, f"y {k}")
        if save:
            close(pre, z, slip, f"pre {k}")


@pytest.mark.parametrize("rows,n,m", LINEAR_SIZES + [(20000, 192, 704)])
@pytest.mark.parametrize("et", ["bf16", "f16"])
def test_gated(cuda, rows, n, m, et):
    import torch
    from t8b import ops
    E = types()[et]
    g = torch.Generator(device="cuda").manual_seed(rows + 3 * n + 7 * m)
    for k, (act, bias, save, slack) in enumerate([("silu", "none", False, 0), ("gelu", "f32", True, 0),
                                                  ("silu", "own", True, 3), ("relu", "f32", False, 8),
                                                  ("tanh", "none", True, 0), ("none", "f32", False, 0)]):
        x = matrix(g, rows, n, E, slack, 0)
        w = matrix(g, 2 * m, n, E, slack, 0, n ** -0.5)
        b = bias_of(g, bias, 2 * m, E)
        got = ops.gated(x, w, b, activation=act, save=save)
        h, pre = got if save else (got, None)
        z, slip = linear64(x, w, b)
        a, _ = act64(z[:, :m], act)
        off = 1.2 * slip[:, :m] + 2.0 ** -19 * (1 + z[:, :m].abs())
        close(h, a * z[:, m:], off * (z[:, m:].abs() + slip[:, m:]) + a.abs() * slip[:, m:], f"h {k}")
        if save:
            close(pre, z, slip, f"pre {k}")


def backward64(dy, x, w, pre, act, gated):
    d = dy.double()
    if gated:
        m = dy.shape[1]
        z, u = pre.double()[:, :m], pre.double()[:, m:]
        a, s = act64(z, act)
        import torch
        dz = torch.cat([d * u * s, d * a], 1)
        slip = 2.0 ** -19 * torch.cat([d.abs() * u.abs() * (1 + z.abs()), d.abs() * (1 + z.abs())], 1)
    elif act == "none":
        dz, slip = d, 0 * d
    else:
        _, s = act64(pre.double(), act)
        dz = d * s
        slip = 2.0 ** -19 * d.abs() * (1 + pre.double().abs())
    return dz, slip


BACKWARD = [("none", "none", 0), ("tanh", "f32", 0), ("gelu", "own", 0), ("silu", "f32", 8), ("relu", "f32", 3),
            ("none", "own", 5)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n,m", LINEAR_SIZES + [(20000, 192, 320), (4099, 72, 40)])
@pytest.mark.parametrize("et", ["bf16", "f16"])
def test_linear_and_gated_backward(cuda, rows, n, m, et, gated):
    import torch
    from t8b import ops
    E = types()[et]
    u = unit(E) * (1 + 2 ** -8)
    g = torch.Generator(device="cuda").manual_seed(rows + 3 * n + 11 * m)
    columns = 2 * m if gated else m
    for k, (act, bias, slack) in enumerate(BACKWARD):
        x = matrix(g, rows, n, E, slack, 0)
        w = matrix(g, columns, n, E, slack, 0, n ** -0.5)
        b = bias_of(g, bias, columns, E)
        dy = matrix(g, rows, m, E, slack, 0, 0.125)
        pre = matrix(g, rows, columns, E, slack, 0, 1.5) if gated or act != "none" else None
        fn = ops.gated_backward if gated else ops.linear_backward
        dx, dw, db = fn(dy, x, w, b, pre, activation=act)
        dz, slip = backward64(dy, x, w, pre, act, gated)
        rounded = slip + (u * dz.abs() + tiny(E) if act != "none" or gated else 0)
        w64, x64 = w.double(), x.double()
        close(dx, dz @ w64, rounded @ w64.abs() + (columns + 16) * 2.0 ** -23 * (dz.abs() @ w64.abs()), f"dx {k}")
        close(dw, dz.T @ x64, rounded.T @ x64.abs() + (rows + 16) * 2.0 ** -23 * (dz.abs().T @ x64.abs()), f"dw {k}")
        if b is not None:
            assert db.dtype is b.dtype
            close(db, dz.sum(0), slip.sum(0) + (rows + 16) * 2.0 ** -24 * dz.abs().sum(0), f"db {k}")
        else:
            assert db is None
        again = fn(dy, x, w, b, pre, activation=act)
        assert all(p is q or torch.equal(p, q) for p, q in zip((dx, dw, db), again))
        alone = fn(dy, x, w, None, pre, activation=act, input_gradient=False)
        assert alone[0] is None and alone[2] is None and torch.equal(alone[1], dw)
    ops.status()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n,m", [(1, 65, 2816), (17, 512, 1408), (40, 96, 4096), (300, 151, 5001), (1025, 33, 3001)])
@pytest.mark.parametrize("et", ["bf16", "f16"])
def test_gradients_of_few_rows_and_many_columns(cuda, rows, n, m, et, gated):
    """Long sums over the columns for few tiles of the input's gradient: its parts are joined in fp32."""
    import torch
    from t8b import ops
    E = types()[et]
    u = unit(E) * (1 + 2 ** -8)
    g = torch.Generator(device="cuda").manual_seed(rows + 3 * n + 11 * m)
    columns = 2 * m if gated else m
    fn = ops.gated_backward if gated else ops.linear_backward
    for slack in (0, 3):
        x, dy = matrix(g, rows, n, E, slack, 0), matrix(g, rows, m, E, slack, 0, 0.125)
        w, pre = matrix(g, columns, n, E, slack, 0, n ** -0.5), matrix(g, rows, columns, E, slack, 0, 1.5)
        b = bias_of(g, "f32", columns, E)
        dz, slip = backward64(dy, x, w, pre, "silu", gated)
        rounded = slip + u * dz.abs() + tiny(E)
        w64, x64 = w.double(), x.double()
        first = fn(dy, x, w, b, pre, activation="silu")
        close(first[0], dz @ w64, rounded @ w64.abs() + (columns + 16) * 2.0 ** -23 * (dz.abs() @ w64.abs()), f"dx {slack}")
        close(first[1], dz.T @ x64, rounded.T @ x64.abs() + (rows + 16) * 2.0 ** -23 * (dz.abs().T @ x64.abs()), f"dw {slack}")
        close(first[2], dz.sum(0), slip.sum(0) + (rows + 16) * 2.0 ** -24 * dz.abs().sum(0), f"db {slack}")
        dx, dw, db = fn(dy, x, w, None, pre, activation="silu")  # no bias: the joins alone in the last pass
        assert db is None and torch.equal(dx, first[0]) and torch.equal(dw, first[1])
    ops.status()


@pytest.mark.parametrize("name", ["norm", "linear", "gated"])
def test_gradients_against_differences(cuda, name):
    """The gradient along a random direction equals the loss's central difference along it, taken
    with the formulas in 64 bits at the values the operator saw."""
    import torch
    from t8b import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, n, m = 37, 96, 56
    E = torch.bfloat16
    x = matrix(g, rows, n, E)
    parts = {"norm": 0, "linear": 1, "gated": 2}[name]
    columns = max(1, parts) * m
    w = torch.rand(n, device="cuda", generator=g) + 0.5 if name == "norm" else matrix(g, columns, n, E, 0, 0, n ** -0.5)
    b = 0.3 * torch.randn(n if name == "norm" else columns, device="cuda", generator=g)
    dy = matrix(g, rows, n if name == "norm" else m, E)
    if name == "norm":
        _, mean, rstd = ops.layer_norm(x, w, b, save=True)
        grads = ops.layer_norm_backward(dy, x, w, b, mean, rstd)
    elif name == "linear":
        _, pre = ops.linear(x, w, b, activation="gelu", save=True)
        grads = ops.linear_backward(dy, x, w, b, pre, activation="gelu")
    else:
        _, pre = ops.gated(x, w, b, save=True)
        grads = ops.gated_backward(dy, x, w, b, pre)

    def loss(x, w, b):
        if name == "norm":
            y = (x - x.mean(1, keepdim=True)) * (x.var(1, unbiased=False, keepdim=True) + EPS) ** -0.5 * w + b
        else:
            z = x @ w.T + b
            y = act64(z, "gelu")[0] if name == "linear" else act64(z[:, :m], "silu")[0] * z[:, m:]
        return float((y * dy.double()).sum())

    at = [v.double() for v in (x, w, b)]
    for i, got in enumerate(grads):
        way = torch.randn(at[i].shape, device="cuda", generator=g, dtype=torch.float64)
        h = 1e-5
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * way, at[i] - h * way
        want = (loss(*plus) - loss(*minus)) / (2 * h)
        # each gradient element and each dz is rounded to bf16 (pre too): 4 roundings of 2^-8
        assert abs(float((got.double() * way).sum()) - want) <= 4 * 2 ** -8 * float((got.double() * way).abs().sum())


def tail64(t, rows):
    return t[-rows:].double()


def test_offsets_past_32_bits(cuda):
    """Matrices of more than 2^31 elements: their last rows against the formulas."""
    import torch
    from t8b import ops
    E, k = torch.bfloat16, 5
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(rows, n, scale=1.0):
        t = torch.empty(rows, n, device="cuda", dtype=E)
        t.normal_(0.0, scale, generator=g)
        return t

    x = normal(4_300_001, 512)
    y, mean, rstd = ops.layer_norm(x, save=True)
    want, m, r, xhat, slip, _ = norm64(x[-k:], None, None)
    close(y[-k:], want, 2 ** -17 * slip)
    dy = normal(4_300_001, 512)
    dx, _, _ = ops.layer_norm_backward(dy, x, None, None, mean, rstd)
    d = tail64(dy, k)
    ref = r * (d - d.mean(-1, keepdim=True) - xhat * (d * xhat).mean(-1, keepdim=True))
    close(dx[-k:], ref, 2 ** -16 * r * (d.abs() + d.abs().mean(-1, keepdim=True) + slip * (d * slip).abs().mean(-1, keepdim=True)))
    del y, dx, dy
    w = normal(40, 512, 512 ** -0.5)
    close(ops.linear(x, w)[-k:], *linear64(x[-k:], w, None))
    del x
    x, w = normal(1_200_003, 64), normal(2048, 64, 0.125)
    y, pre = ops.gated(x, w, activation="relu", save=True)
    z, slip = linear64(x[-k:], w, None)
    close(pre[-k:], z, slip, "pre")
    dh = normal(1_200_003, 1024, 0.125)
    dx, dw, _ = ops.gated_backward(dh, x, w, None, pre, activation="relu")
    dz, _ = backward64(dh[-k:], x[-k:], w, pre[-k:], "relu", True)
    mags = dz.abs() @ w.double().abs()
    close(dx[-k:], dz @ w.double(), (unit(E) * (1 + 2 ** -8) + (2048 + 16) * 2.0 ** -23) * mags, "dx")
    total = torch.zeros(2048, 64, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    for at in range(0, x.shape[0], 100_000):
        rows = slice(at, at + 100_000)
        part, _ = backward64(dh[rows], x[rows], w, pre[rows], "relu", True)
        total += part.T @ x[rows].double()
        size += part.abs().T @ x[rows].double().abs()
    close(dw, total, (unit(E) * (1 + 2 ** -8) + (x.shape[0] + 16) * 2.0 ** -23) * size, "dweight")
    del y, pre, dh, dx, x
    x, w = normal(1, 32768), normal(70_001, 32768, 32768 ** -0.5)
    z, slip = linear64(x, w[-k:], None)
    close(ops.linear(x, w)[:, -k:], z, slip)
    ops.status()


@pytest.mark.parametrize("n", [130, 512, 515, 1001])
def test_layer_norm_in_place(cuda, n):
    """y may be x itself, rows that share packs included."""
    import torch
    from t8b import _lib, ops
    x = torch.randn(3000, n, device="cuda").bfloat16()
    want = ops.layer_norm(x)
    status = _lib.lib().t8b_layer_norm_forward(x.data_ptr(), 1, n, 0, 0, 0, 1e-5, 3000, n, x.data_ptr(), 1, n, 0, 0, None)
    assert status == 0 and torch.equal(x, want)


def test_infinities_and_nan_stay_in_their_rows(cuda):
    import torch
    from t8b import ops
    x = torch.randn(300, 130, device="cuda").bfloat16()
    w = torch.randn(72, 130, device="cuda").bfloat16()
    clean = ops.linear(x, w, activation="tanh")
    x[5, 3] = float("inf")
    x[257, 129] = float("nan")
    y = ops.linear(x, w, activation="tanh")
    keep = [i for i in range(300) if i not in (5, 257)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[257]).all()
    assert torch.equal(y[5].float(), torch.sign(w[:, 3].float()))
    # an overflow is an infinity of the output's type
    big = torch.full((2, 64), 200.0, device="cuda", dtype=torch.float16)
    assert torch.isinf(ops.linear(big, big)).all()
    assert torch.equal(ops.linear(big, big, out_dtype=torch.float32), torch.full((2, 2), 64 * 40000.0, device="cuda"))


def test_zero_rows(cuda):
    import torch
    from t8b import ops
    E = torch.bfloat16
    x, w = torch.empty(0, 48, device="cuda", dtype=E), torch.randn(32, 48, device="cuda").to(E)
    b = torch.randn(32, device="cuda")
    y, pre = ops.linear(x, w, b, activation="tanh", save=True)
    assert y.shape == (0, 32) and pre.shape == (0, 32)
    dx, dw, db = ops.linear_backward(y, x, w, b, pre, activation="tanh")
    assert dx.shape == (0, 48) and not dw.any() and dw.shape == (32, 48) and not db.any()
    h, pre = ops.gated(x, w, b, save=True)
    assert h.shape == (0, 16)
    dx, dw, db = ops.gated_backward(h, x, w, b, pre)
    assert not dw.any() and not db.any() and db.shape == (32,)
    weight = torch.ones(48, device="cuda")
    y, mean, rstd = ops.layer_norm(x, weight, weight, save=True)
    dx, dw, db = ops.layer_norm_backward(y, x, weight, weight, mean, rstd)
    assert dx.shape == (0, 48) and not dw.any() and not db.any()


def test_leading_axes_and_other_streams(cuda):
    """Rows spread over leading axes; a call on a side stream with inputs made there; a captured
    call replayed on new values."""
    import torch
    from t8b import ops
    E = torch.bfloat16
    x = torch.randn(6, 5, 64, device="cuda").to(E)
    w = torch.randn(96, 64, device="cuda").to(E)
    flat = ops.linear(x.view(30, 64), w, activation="silu")
    assert torch.equal(ops.linear(x, w, activation="silu"), flat.view(6, 5, 96))
    # the same rows packed: equal bits (another number of rows may go through another kernel)
    assert torch.equal(ops.linear(x[:, 2], w, activation="silu"), ops.linear(x[:, 2].contiguous(), w, activation="silu"))
    assert torch.equal(ops.linear(x[2, 3], w, activation="silu"), ops.linear(x[2, 3:4], w, activation="silu")[0])
    norm = ops.layer_norm(x)
    assert torch.equal(ops.layer_norm(x[1:, 4]), norm[1:, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            z = x * 2
        y = ops.gated(z, w, stream=side)
        with torch.cuda.stream(side):
            again = ops.gated(z, w)
    side.synchronize()
    assert torch.equal(y, again) and torch.equal(y, ops.gated(x * 2, w))
    graph = torch.cuda.CUDAGraph()
    static = x.view(30, 64).clone()
    with torch.cuda.graph(graph):
        n = ops.layer_norm(static)
        y, pre = ops.gated(n, w, save=True)
        grads = ops.gated_backward(y, n, w, None, pre)
    static.copy_(torch.randn(30, 64, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    n2 = ops.layer_norm(static)
    y2, pre2 = ops.gated(n2, w, save=True)
    assert torch.equal(y, y2) and torch.equal(grads[1], ops.gated_backward(y2, n2, w, None, pre2)[1])


def test_calls_between_other_work(cuda):
    """An operator's kernels may start before the work ahead of them has ended; they see it all the
    same: behind copies, other kernels, events of other streams, themselves, and so in a captured
    graph. Integer-valued data make every sum exact, so equality is of bits."""
    import torch
    from t8b import ops
    E = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(9)
    rows, n = 4096, 256
    w = torch.randint(-1, 2, (n, n), device="cuda", generator=g).to(E)
    w2 = torch.randint(-1, 2, (2 * n, n), device="cuda", generator=g).to(E)
    side = torch.cuda.Stream()
    inputs = [torch.randint(-2, 3, (rows, n), device="cuda", generator=g).to(E) for _ in range(6)]

    def chain(x):
        """Every way in: a copy, a kernel of torch's, a wait for another stream, memory cleared."""
        at = torch.empty_like(x)
        at.copy_(x)
        y = ops.linear(at, w, activation="relu")                       # behind a copy
        y = (y * 0.0625).round()                                        # behind an operator
        fork = torch.cuda.current_stream()
        side.wait_stream(fork)
        with torch.cuda.stream(side):
            z = ops.gated(y.clamp(-4, 4), w2, activation="relu")
            z = (z * 2.0 ** -12).round()
        fork.wait_stream(side)
        zero = torch.zeros_like(z)                                      # a memset
        few = ops.linear((z + zero)[:3].clamp(-4, 4), w)
        dx, dw, _ = ops.linear_backward(y.clamp(-4, 4), at, w)          # behind a wait
        h = ops.layer_norm(dx, out_dtype=torch.float32)
        return y, z, few, dx, dw, h, ops.layer_norm(h)                  # behind itself

    torch.cuda.synchronize()
    want = []
    for x in inputs:
        out = chain(x)
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    x64 = inputs[0].double()
    assert torch.equal(want[0][0].double(), ((x64 @ w.double().T).clamp(min=0) .to(E).double() * 0.0625).to(E).double().round())
    for _ in range(3):  # nothing waited for between the calls
        got = [chain(x) for x in inputs]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    static = inputs[0].clone()
    with torch.cuda.graph(graph):
        out = chain(static)
    for x, b in zip(inputs, want):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, b))
    first = torch.cuda.CUDAGraph()  # an operator as a graph's first node
    with torch.cuda.graph(first):
        y = ops.layer_norm(static)
    static.copy_(inputs[3])
    first.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.layer_norm(inputs[3]))
    ops.status()


def test_operators_refuse_what_they_cannot_take(cuda):
    import torch
    from t8b import ops
    E = torch.bfloat16
    x, w = torch.zeros(4, 16, device="cuda", dtype=E), torch.zeros(8, 16, device="cuda", dtype=E)
    y = torch.zeros(4, 8, device="cuda", dtype=E)
    refused = [
        lambda: ops.linear(x.float(), w.float()),
        lambda: ops.linear(x, w.half()),
        lambda: ops.linear(x, w[:, :8]),
        lambda: ops.linear(x.t(), w),
        lambda: ops.linear(x.cpu(), w),
        lambda: ops.linear(x, w.cpu()),
        lambda: ops.linear(x, w, torch.zeros(7, device="cuda")),
        lambda: ops.linear(x, w, torch.zeros(8, device="cuda", dtype=torch.float16)),
        lambda: ops.linear(x, w, activation="swish"),
        lambda: ops.linear(x, w, residual=y.float()),
        lambda: ops.linear(x, w, residual=y[:3]),
        lambda: ops.linear(x, w, out_dtype=torch.float16),
        lambda: ops.linear(x[:1].expand(4, 16), w),
        lambda: ops.gated(x, w[:7]),
        lambda: ops.linear_backward(y, x, w, activation="tanh"),
        lambda: ops.linear_backward(y[:, :7], x, w),
        lambda: ops.linear_backward(y, x, w, pre=y[:3], activation="tanh"),
        lambda: ops.gated_backward(y, x, w, pre=y),
        lambda: ops.layer_norm(x.double()),
        lambda: ops.layer_norm(x, torch.ones(15, device="cuda")),
        lambda: ops.layer_norm(x, torch.ones(16, device="cuda"), torch.ones(16, device="cuda", dtype=E)),
        lambda: ops.layer_norm(x, eps=float("nan")),
        lambda: ops.layer_norm(x, eps=-1.0),
        lambda: ops.layer_norm(torch.zeros(4, 0, device="cuda")),
        lambda: ops.layer_norm_backward(x[:3], x, None, None, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")),
        lambda: ops.layer_norm_backward(x, x, None, None, torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")),
    ]
    for k, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {k} was taken")


def test_c_entries_refuse_what_they_cannot_take(cuda):
    import torch
    from t8b import _lib
    lib = _lib.lib()
    E = torch.bfloat16
    x, w = torch.zeros(64, 64, device="cuda", dtype=E), torch.zeros(64, 64, device="cuda", dtype=E)
    y = torch.zeros(64, 64, device="cuda", dtype=E)
    px, pw, py = x.data_ptr(), w.data_ptr(), y.data_ptr()
    odd = px + 2

    def linear(**k):
        a = dict(type=1, x=px, xs=64, w=pw, ws=64, b=0, bt=0, act=0, r=0, rs=64, rows=32, n=32, m=32, y=py, yt=1, ys=64,
                 p=0, ps=64, work=0, size=0)
        a.update(k)
        return lib.t8b_linear_forward(*a.values(), None)

    assert linear() == 0
    for bad in (dict(type=0), dict(type=3), dict(act=5), dict(act=-1), dict(rows=-1), dict(n=0), dict(m=0), dict(m=1 << 23),
                dict(x=0), dict(w=0), dict(y=0), dict(xs=31), dict(ys=8), dict(yt=2), dict(b=pw + 6000, bt=2), dict(y=px),
                dict(y=pw), dict(p=py), dict(r=py + 128), dict(x=odd), dict(xs=63), dict(x=odd, work=py, size=64)):
        assert linear(**bad) == _lib.T8B_EINVAL, bad
        assert lib.t8b_last_error()
    assert linear(rows=0, x=0, y=0) == 0
    assert linear(r=py) == 0  # in place on the residual
    need = lib.t8b_linear_workspace(32, 32, 32, 1)  # packed rows, no activation: no copies, no dz
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros(64, 64, device="cuda", dtype=E)

    def backward(**k):
        a = dict(type=1, dy=py, dys=64, x=px, xs=64, w=pw, ws=64, p=0, ps=64, bt=0, act=0, rows=32, n=32, m=32,
                 dx=out.data_ptr(), dxs=64, dw=0, dws=64, db=0, work=work.data_ptr(), size=need)
        a.update(k)
        return lib.t8b_linear_backward(*a.values(), None)

    assert backward() == 0
    assert lib.t8b_linear_workspace(32, 32, 32, 15) > need
    for bad in (dict(size=need - 1), dict(work=0), dict(x=px + 2, dw=out.data_ptr(), dx=0), dict(act=4, p=pw), dict(work=work.data_ptr() + 16), dict(dx=px, dw=out.data_ptr()),
                dict(dx=py), dict(act=4), dict(dw=out.data_ptr()), dict(dxs=3), dict(type=0)):
        assert backward(**bad) == _lib.T8B_EINVAL, bad
    mean = torch.zeros(64, device="cuda")

    def norm(**k):
        a = dict(x=px, xt=1, xs=64, w=0, b=0, pt=0, eps=1e-5, rows=32, n=32, y=py, yt=1, ys=64, mean=mean.data_ptr(), rstd=0)
        a.update(k)
        return lib.t8b_layer_norm_forward(*a.values(), None)

    assert norm() == 0 and norm(y=px) == 0
    for bad in (dict(xt=3), dict(yt=-1), dict(pt=9), dict(rows=-1), dict(n=0), dict(x=0), dict(y=0), dict(xs=31), dict(y=px + 2),
                dict(eps=float("inf"))):
        assert norm(**bad) == _lib.T8B_EINVAL, bad
    torch.cuda.synchronize()
    assert lib.t8b_operators_status(None) == 0
