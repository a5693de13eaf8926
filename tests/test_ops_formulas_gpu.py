"""The torso operators against formulas that the other tests do not use: automatic differentiation in 64
bits, differences of the forward formula along the gradient, activations on a grid, and the norm's types
and strides that are left. Each gradient check is also made with planted mistakes, and has to reject them.

Bounds (u: half the output type's spacing, as in test_ops_gpu.py):
  - activations in fp32: Phi within 7e-8 (Abramowitz and Stegun 7.1.26) plus the roundings of a fifth-degree
    Horner sum of partial sums below 1.5, of 2^x and of 1/x: 2^-20 in all, so gelu within |z| 2^-20 and its
    slope, which adds 0.4 |z| exp(-z^2 / 2), within 2^-20; in gelu's lower tail the series' relative error
    counts, in 64 bits 3.6e-3 at -6: 2^-8 there with fp32's roundings;
  - sigmoid: relative 2^-21 + |z| 2^-23 (2^x of a rounded product, 1/x), and so silu; its slope s (1 + z (1 - s))
    within 2^-20 (1 + |z|);
  - tanh: relative 2^-21 in the series, within 2^-20 elsewhere; its slope 1 - v^2 within 2^-19;
  - a norm's sums: at most 16 packed additions, one, 5 over lanes and 8 over warps (n to 8,192), or n / 512
    and 21 (beyond): fewer than 128 for every n here, so 2^-17 of the summed magnitudes.
"""
import math

import pytest

from test_ops_gpu import EPS, close, matrix, norm64, tiny, types, unit

pytestmark = pytest.mark.gpu


def formula(z, name):
    import torch
    return {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu}[name](z)


def rejects(check, got, name):
    """The check fails for a gradient that is 10 % too large or has the wrong sign, and for one of other rows."""
    for wrong in (got * 1.1, -got, got.roll(1, 0)):
        with pytest.raises(AssertionError):
            check(wrong.to(got.dtype))
            pytest.fail(f"{name}: a wrong gradient was taken")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "tanh"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n,m", [(37, 96, 56), (130, 33, 40), (3, 200, 24)])
@pytest.mark.parametrize("type_name", ["bf16", "f16"])
def test_gradients_against_automatic_differentiation(cuda, rows, n, m, type_name, gated, act):
    """Element by element; dz, differentiated at the saved pre, is rounded once to the operands' type."""
    import torch
    from t8b import ops
    E = types()[type_name]
    g = torch.Generator(device="cuda").manual_seed(rows + n + m)
    columns = 2 * m if gated else m
    x, w = matrix(g, rows, n, E), matrix(g, columns, n, E, 0, 0, n ** -0.5)
    b = 0.3 * torch.randn(columns, device="cuda", generator=g)
    dy = matrix(g, rows, m, E)
    if gated:
        _, pre = ops.gated(x, w, b, activation=act, save=True)
        got = ops.gated_backward(dy, x, w, b, pre, activation=act)
    else:
        _, pre = ops.linear(x, w, b, activation=act, save=True)
        got = ops.linear_backward(dy, x, w, b, pre, activation=act)
    # y = f(z) with z = x w^T + b held at the saved values, so that only the operator's own roundings are left
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    z = leaves[0] @ leaves[1].T + leaves[2]
    z = z + (pre.double() - z).detach()
    z.retain_grad()
    y = formula(z[:, :m], act) * z[:, m:] if gated else formula(z, act)
    y.backward(dy.double())
    dz = z.grad
    size = dy.double().abs().repeat(1, columns // m) * (1 + pre.double().abs())
    if gated:
        size = size * torch.cat([1 + pre.double()[:, m:].abs(), torch.ones_like(dy, dtype=torch.float64)], 1)
    slip = 2.0 ** -19 * size * (act != "none" or gated)
    rounded = slip + (unit(E) * (1 + 2 ** -8) * dz.abs() + tiny(E)) * (act != "none" or gated)
    x64, w64 = x.double().abs(), w.double().abs()
    bounds = (rounded @ w64 + (columns + 16) * 2.0 ** -23 * (dz.abs() @ w64),
              rounded.T @ x64 + (rows + 16) * 2.0 ** -23 * (dz.abs().T @ x64),
              slip.sum(0) + (rows + 16) * 2.0 ** -23 * dz.abs().sum(0))
    for name, value, leaf, bound in zip(("dx", "dweight", "dbias"), got, leaves, bounds):
        check = lambda v: close(v, leaf.grad, bound, name)  # noqa: B023,E731
        check(value)
        rejects(check, value, name)


@pytest.mark.parametrize("name", ["norm", "linear", "gated"])
def test_gradients_against_differences_along_them(cuda, name):
    """The loss's central difference along the gradient itself, where its elements add up. Every rounding of
    an operand (the output's, dz's and pre's) is its own, so they add as squares: 8 u of the root of the
    sum of squares of what each is multiplied with."""
    import torch
    from t8b import ops
    E, u = torch.bfloat16, 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(6)
    rows, n, m = 64, 96, 56
    x = matrix(g, rows, n, E)
    gated = name == "gated"
    columns = 2 * m if gated else m
    if name == "norm":
        w, b = torch.rand(n, device="cuda", generator=g) + 0.5, 0.3 * torch.randn(n, device="cuda", generator=g)
        dy = matrix(g, rows, n, E)
        _, mean, rstd = ops.layer_norm(x, w, b, save=True)
        grads = ops.layer_norm_backward(dy, x, w, b, mean, rstd)
    else:
        w, b = matrix(g, columns, n, E, 0, 0, n ** -0.5), 0.3 * torch.randn(columns, device="cuda", generator=g)
        dy = matrix(g, rows, m, E)
        forward, backward = (ops.gated, ops.gated_backward) if gated else (ops.linear, ops.linear_backward)
        _, pre = forward(x, w, b, activation="gelu", save=True)
        grads = backward(dy, x, w, b, pre, activation="gelu")

    def loss(x, w, b):
        if name == "norm":
            y = (x - x.mean(1, keepdim=True)) * (x.var(1, unbiased=False, keepdim=True) + EPS) ** -0.5 * w + b
        else:
            z = x @ w.T + b
            y = formula(z[:, :m], "gelu") * z[:, m:] if gated else formula(z, "gelu")
        return float((y * dy.double()).sum())

    at = [v.double() for v in (x, w, b)]
    if name != "norm":  # what one rounding of a dz, or of the pre behind it, moves: |f'|, |f''| are at most 1.13
        size = dy.double().abs().repeat(1, columns // m) * (1 + pre.double().abs())
        if gated:
            size = size * torch.cat([1 + pre.double()[:, m:].abs(), torch.ones_like(dy, dtype=torch.float64)], 1)
    for i, got in enumerate(grads):
        way = got.double() / got.double().norm()
        h = 1e-4
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * way, at[i] - h * way
        want = (loss(*plus) - loss(*minus)) / (2 * h)
        squares = (got.double() * way).square().sum()
        if name != "norm":
            # d(this sum) / d(dz)
            through = way @ at[1].T if i == 0 else at[0] @ way.T if i == 1 else way.expand(rows, columns)
            squares = squares + (2 * size * through).square().sum()
        limit = 8 * u * float(squares.sqrt()) + 1e-6 * abs(want)

        def check(v):
            assert abs(float((v.double() * way).sum()) - want) <= limit, (i, want, limit)  # noqa: B023

        check(got)
        for wrong in (got * 1.1, got * 0.9, -got, got * 0):
            with pytest.raises(AssertionError):
                check(wrong)
                pytest.fail(f"{name} {i}: a wrong gradient was taken")


@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "tanh"])
def test_activations_and_slopes_on_a_grid(cuda, act):
    """fp32 outputs of y = f(z) (one feature, weight 1), and f and f' as the bias gradients of one row."""
    import torch
    from t8b import ops
    for E in (torch.bfloat16, torch.float16):
        z = torch.linspace(-9, 9, 4801, device="cuda").to(E).unique()
        z = torch.cat([z, torch.tensor([0.0, 1e-4, -1e-4, 0.19, 0.2, 0.21, -0.2, 30.0, -30.0], device="cuda").to(E)])
        z64 = z.double().requires_grad_()
        value = formula(z64, act)
        if act == "gelu":  # in the lower tail torch's own form loses digits in 64 bits too
            value = z64 * 0.5 * torch.erfc(-z64 / math.sqrt(2.0))
        value.sum().backward()
        slope, value, size = z64.grad, value.detach(), z.double().abs()
        of_value, of_slope = {
            "relu": (0 * size, 0 * size),
            "gelu": (size * 2 ** -20, 0 * size + 2 ** -20),
            "silu": (value.abs() * (2 ** -21 + size * 2 ** -23), 2 ** -20 * (1 + size)),
            "tanh": (torch.where(size < 0.2, size * 2 ** -21, 0 * size + 2 ** -20), 0 * size + 2 ** -19),
        }[act]
        one = torch.ones(1, 1, device="cuda", dtype=E)
        close(ops.linear(z[:, None], one, activation=act, out_dtype=torch.float32)[:, 0], value, of_value, "value by tiles")
        few = ops.linear(z[:4, None], one, activation=act, out_dtype=torch.float32)[:, 0]
        close(few, value[:4], of_value[:4], "value by rows")
        if act == "gelu":
            tail = (z >= -6) & (z <= -2)
            y = ops.linear(z[tail][:, None], one, activation=act, out_dtype=torch.float32)[:, 0].double()
            assert bool(((y - value[tail]).abs() <= 2 ** -8 * value[tail].abs()).all())
        m = z.numel()
        w, row = torch.zeros(m, 1, device="cuda", dtype=E), torch.ones(1, m, device="cuda", dtype=E)
        _, _, db = ops.linear_backward(row, one, w, torch.zeros(m, device="cuda"), z[None], activation=act)
        keep = z != 0 if act == "relu" else torch.ones_like(z, dtype=torch.bool)  # relu has no slope at 0
        close(db[keep], slope[keep], of_slope[keep], "slope")
        both = torch.cat([z, torch.full_like(z, 3.0)])[None]
        _, _, db = ops.gated_backward(row, one, torch.zeros(2 * m, 1, device="cuda", dtype=E), torch.zeros(2 * m, device="cuda"),
                                      both, activation=act)
        close(db[:m][keep], 3 * slope[keep], 3 * of_slope[keep] + 2 ** -24 * 3 * slope[keep].abs(), "gate's slope")
        close(db[m:], value, of_value, "gate's value")


@pytest.mark.parametrize("rows,n", [(5, 33), (40, 256), (300, 151), (11, 513), (700, 515), (33, 2048), (12, 4099), (3, 9001)])
@pytest.mark.parametrize("xt,yt", [("f32", "f16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("strides", ["packed", "unlike", "wide"])
def test_layer_norm_types_and_strides(cuda, rows, n, xt, yt, strides):
    """The type pairs and the strides that test_ops_gpu.py leaves: rows off a boundary in f16, and matrices
    whose strides differ from one another modulo a vector while each starts on one."""
    import torch
    from t8b import ops
    T = types()
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    slack = {"packed": (0, 0, 0), "unlike": (0, 8 - n % 8, 3), "wide": (8, 16, 24)}[strides]
    x = matrix(g, rows, n, T[xt], slack[0], 0, 2.0)
    dy = matrix(g, rows, n, T[yt], slack[1], 0)
    res = matrix(g, rows, n, T[xt], slack[2], 0)
    w, b = 1 + 0.3 * torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g)
    y, mean, rstd = ops.layer_norm(x, w, b, EPS, out_dtype=T[yt], save=True)
    want, m, r, xhat, slip, w64 = norm64(x, w, b)
    close(y, want, 2 ** -17 * slip * w64.abs() + 2 ** -22 * b.double().abs(), "y")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, b, mean, rstd, residual_gradient=res)
    leaf, weight = x.double().requires_grad_(), w.double().requires_grad_()
    out = torch.nn.functional.layer_norm(leaf, (n,), weight, b.double(), EPS)
    out.backward(dy.double())
    d = dy.double()
    gw = d * w64
    mags = gw.abs() + gw.abs().mean(-1, keepdim=True) + (xhat.abs() + slip) * (gw * slip).abs().mean(-1, keepdim=True)
    close(dx, leaf.grad + res.double(), 2 ** -16 * r * mags + 2 ** -22 * res.double().abs(), "dx")
    close(dw, weight.grad, 2 ** -16 * (d.abs() * slip).sum(0), "dweight")
    close(db, d.sum(0), 2 ** -17 * d.abs().sum(0), "dbias")
    rejects(lambda v: close(v, weight.grad, 2 ** -16 * (d.abs() * slip).sum(0), "dweight"), dw, "dweight")
