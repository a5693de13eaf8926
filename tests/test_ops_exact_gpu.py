"""The torso operators' gradients on data whose sums are exact in fp32 (small integers), so that the only
rounding left is the output's own and equality is of bits: nothing that a sum leaves out, doubles or
takes from elsewhere fits under it. The first and last rows are 32 times as large as the others, so they
show in every sum; each check is also made against sums that lack the last row, and has to fail there."""
import pytest

pytestmark = pytest.mark.gpu


def integers(g, low, high, shape, dtype):
    import torch
    return torch.randint(low, high + 1, shape, device="cuda", generator=g).to(dtype)


def product(a, b):
    """a^T b in 64 bits, a block of rows at a time."""
    import torch
    total = torch.zeros(a.shape[1], b.shape[1], device="cuda", dtype=torch.float64)
    for at in range(0, a.shape[0], 1 << 17):
        total += a[at:at + (1 << 17)].double().T @ b[at:at + (1 << 17)].double()
    return total


def gradient_of(dy, pre, gated):
    """dz of a relu, exact in the operands' type."""
    import torch
    if not gated:
        return dy * (pre > 0)
    gate, up = pre.chunk(2, 1)
    return torch.cat([dy * up * (gate > 0), dy * gate.clamp(min=0)], 1)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [1, 31, 63, 64, 65, 127, 96 * 64 + 1, 96 * 64 + 32, 96 * 64 + 63, 20000, 20033, 65537])
@pytest.mark.parametrize("n,m,type_name,slack", [(72, 40, "bfloat16", 0), (192, 320, "bfloat16", 0), (151, 33, "float16", 3),
                                                 (512, 96, "bfloat16", 5)])
def test_gradients_are_exact_sums(cuda, rows, n, m, type_name, slack, gated):
    import torch
    from t8b import ops
    E = getattr(torch, type_name)
    g = torch.Generator(device="cuda").manual_seed(rows + 3 * n + 7 * m)
    columns = 2 * m if gated else m

    def matrix(low, high, height, width):
        wide = torch.full((height, width + slack), float("nan"), device="cuda", dtype=E)
        wide[:, :width] = integers(g, low, high, (height, width), E)
        return wide[:, :width]

    x, w = matrix(-1, 1, rows, n), matrix(-1, 1, columns, n)
    dy, pre = matrix(-1, 1, rows, m), matrix(-2, 2, rows, columns)
    for edge in {0, rows - 1}:
        x[edge] = 32.0
        dy[edge] = 1.0
        pre[edge] = 1.0
    b = torch.zeros(columns, device="cuda")
    fn = ops.gated_backward if gated else ops.linear_backward
    dx, dw, db = fn(dy, x, w, b, pre, activation="relu")
    dz = gradient_of(dy, pre, gated)
    assert torch.equal(dx, (dz.double() @ w.double()).to(E))
    want = product(dz, x)
    assert float(want.abs().max()) < 2 ** 16 and torch.equal(dw, want.to(E))
    assert torch.equal(db.double(), dz.double().sum(0))
    short = want - dz[-1:].double().T @ x[-1:].double()
    assert not bool((dw == short.to(E)).any())  # the last row shows in every element
    ops.status()


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 2367, 2368, 2369, 40001])
@pytest.mark.parametrize("n", [64, 128, 256, 512, 1024, 4096, 16384])
def test_layer_norm_gradients_are_exact_sums(cuda, rows, n):
    """x of +-1 with mean 0 and rstd 1 as given makes xhat = x; every mean is a multiple of 1 / n with n a
    power of two."""
    import torch
    from t8b import ops
    E = torch.bfloat16
    rows = min(rows, (1 << 26) // n)
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = 2 * integers(g, 0, 1, (rows, n), E) - 1
    dy = integers(g, -2, 2, (rows, n), E)
    dy[0] += 32
    dy[-1] += 32
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    w, b = torch.full((n,), 2.0, device="cuda"), torch.zeros(n, device="cuda")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, b, mean, rstd)
    dw_want, db_want = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
    step = max(1, (1 << 24) // n)
    for at in range(0, rows, step):
        d, x64 = dy[at:at + step].double(), x[at:at + step].double()
        dw_want += (d * x64).sum(0)
        db_want += d.sum(0)
        k = 2 * d
        want = k - k.mean(1, keepdim=True) - x64 * (k * x64).mean(1, keepdim=True)
        assert torch.equal(dx[at:at + step], want.to(E))
    assert torch.equal(dw.double(), dw_want) and torch.equal(db.double(), db_want)
    assert not bool((db.double() == db_want - dy[-1].double()).any())


def test_sums_over_more_than_2_31_elements_are_exact(cuda):
    import torch
    from t8b import ops
    E = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = 1_200_003
    x, w = integers(g, -1, 1, (rows, 64), E), integers(g, -1, 1, (2048, 64), E)
    dh, pre = integers(g, -1, 1, (rows, 1024), E), integers(g, -2, 2, (rows, 2048), E)
    x[-1], dh[-1], pre[-1] = 1024.0, 1.0, 1.0
    b = torch.zeros(2048, device="cuda")
    dx, dw, db = ops.gated_backward(dh, x, w, b, pre, activation="relu")
    want = torch.zeros(2048, 64, device="cuda", dtype=torch.float64)
    total = torch.zeros(2048, device="cuda", dtype=torch.float64)
    for at in range(0, rows, 100_000):
        part = slice(at, at + 100_000)
        dz = gradient_of(dh[part], pre[part], True).double()
        want += dz.T @ x[part].double()
        total += dz.sum(0)
        assert torch.equal(dx[part], (dz @ w.double()).to(E)), at
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(dw, want.to(E)) and torch.equal(db.double(), total)
    last = gradient_of(dh[-1:], pre[-1:], True).double().T @ x[-1:].double()
    assert float((dw == (want - last).to(E)).double().mean()) < 0.2  # rounded to 8 bits, some may agree
    del x, w, dh, pre, dx, dw, dz
    rows, n = 4_300_001, 512
    x = 2 * integers(g, 0, 1, (rows, n), E) - 1
    dy = torch.ones(rows, n, device="cuda", dtype=E)
    dy[-1] = 9.0
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dx, dw, db = ops.layer_norm_backward(dy, x, torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"), mean, rstd)
    assert torch.equal(db.double(), torch.full((n,), rows + 8.0, device="cuda", dtype=torch.float64))
    want = torch.zeros(n, device="cuda", dtype=torch.float64)
    for at in range(0, rows, 200_000):
        x64 = x[at:at + 200_000].double()
        d = dy[at:at + 200_000].double()
        want += (d * x64).sum(0)
        ref = d - d.mean(1, keepdim=True) - x64 * (d * x64).mean(1, keepdim=True)
        assert torch.equal(dx[at:at + 200_000], ref.to(E)), at
    assert torch.equal(dw.double(), want)
    ops.status()


def test_gradients_between_other_work(cuda):
    """Backward passes with an activation and with operands that have to be packed, one behind the other
    with nothing waited for, behind copies and torch's kernels, and captured: each kernel of a pass may
    start before the ones ahead of it have ended, and has to see what they wrote."""
    import torch
    from t8b import ops
    E = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(4)
    rows, n, m = 3000, 136, 200

    def odd(height, width):
        return torch.empty(height, width + 3, device="cuda", dtype=E)[:, :width]  # rows off 16-byte boundaries

    inputs = [(integers(g, -1, 1, (rows, n), E), integers(g, -1, 1, (2 * m, n), E), integers(g, -1, 1, (rows, m), E),
               integers(g, -2, 2, (rows, 2 * m), E)) for _ in range(5)]

    def passes(x, w, dh, pre):
        out = []
        for height in (rows, 70, 1500):  # the input's gradient split over its sum, and not
            for copy in (torch.empty, odd):
                at = [copy(*t.shape) if copy is odd else torch.empty_like(t) for t in (x[:height], w, dh[:height], pre[:height])]
                for to, t in zip(at, (x[:height], w, dh[:height], pre[:height])):
                    to.copy_(t)
                bias = torch.zeros(2 * m, device="cuda")
                dx, dw, db = ops.gated_backward(at[2], at[0], at[1], bias, at[3], activation="relu")
                back = ops.linear_backward(at[2], dx.clamp(-3, 3), at[1][:m], bias[:m], at[3][:, m:], activation="relu")
                out += [dx, dw, db, *back]
                for t in at:  # what the passes read is overwritten as soon as they are queued
                    t.fill_(float("nan"))
        return out

    want = []
    for values in inputs:
        out = passes(*values)
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
        x, w, dh, pre = values
        dz = gradient_of(dh, pre, True)
        for k in (0, 6):
            assert torch.equal(out[k], (dz.double() @ w.double()).to(E))
            assert torch.equal(out[k + 1], product(dz, x).to(E))
            assert torch.equal(out[k + 2].double(), dz.double().sum(0))
            dz1, x1 = gradient_of(dh, pre[:, m:], False), out[k].clamp(-3, 3)
            assert torch.equal(out[k + 3], (dz1.double() @ w[:m].double()).to(E))
            assert torch.equal(out[k + 4], product(dz1, x1).to(E))
            assert torch.equal(out[k + 5].double(), dz1.double().sum(0))
    for _ in range(4):
        got = [passes(*values) for values in inputs]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes(*static)
    for values, b in zip(inputs, want):
        for to, t in zip(static, values):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, b))
    ops.status()
