"""Edges of the torso operators: values, arguments and streams at which they could go wrong."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 100, 151, 320, 515, 700, 1500, 2049, 8185])
@pytest.mark.parametrize("type_name", ["float32", "bfloat16"])
def test_layer_norm_backward_of_constant_rows_of_large_values(cuda, n, type_name):
    """xhat of a constant row is 0, so dx = rstd (g - mean(g)) + residual and dweight's term is 0, however
    large mean * rstd is: what a thread holds beyond the row must not enter. Small integers in dy make
    n * mean(g) exact; dx is off by the roundings of mean(g), the difference and two products, each
    2^-24 of rstd times (|g| + |mean(g)|) at most, and by its own rounding."""
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    rows, eps = 37, 1e-5
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.full((rows, n), 2.0 ** 121, device="cuda", dtype=T)  # 2^121 / sqrt(1e-5) > 2^128
    x[1::2] = -1.0
    dy = torch.randint(-3, 4, (rows, n), device="cuda", generator=g).to(T)
    w, b = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    mean = x[:, 0].float().contiguous()
    rstd = torch.full((rows,), eps ** -0.5, device="cuda")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, b, mean, rstd)
    d, r = dy.double(), rstd.double()[:, None]
    average = d.mean(1, keepdim=True)
    want = r * (d - average)
    unit = 2.0 ** -24 if T is torch.float32 else 2.0 ** -8
    limit = 8 * 2.0 ** -24 * r * (d.abs() + average.abs()) + unit * want.abs()
    assert bool(((dx.double() - want).abs() <= limit).all())
    assert not dw.any()
    assert torch.equal(db.double(), d.sum(0))


def test_each_stall_is_reported_once(cuda):
    """A wait that ran out on one stream is reported whichever stream is asked, once, and not lost where
    other threads ask meanwhile."""
    import threading
    import time
    import torch
    from t8b import _lib, ops
    side, other = torch.cuda.Stream(), torch.cuda.Stream()

    def stall():
        _lib.call("t8b_debug_operators_stall", 64, side.cuda_stream)
        side.synchronize()

    ops.status()
    stall()
    with pytest.raises(_lib.T8bError, match="ran out"):
        ops.status(other)
    ops.status(side)
    stall()
    stall()
    with pytest.raises(_lib.T8bError, match="ran out"):
        ops.status()
    ops.status()

    reports, done = [], threading.Event()

    def poll(stream):
        while not done.is_set():
            try:
                ops.status(stream)
            except _lib.T8bError:
                reports.append(stream)

    threads = [threading.Thread(target=poll, args=(s,)) for s in (other, torch.cuda.Stream())]
    for t in threads:
        t.start()
    try:
        for i in range(300):
            stall()
            until = time.monotonic() + 10
            while len(reports) <= i and time.monotonic() < until:
                time.sleep(0)
            assert len(reports) == i + 1
    finally:
        done.set()
        for t in threads:
            t.join()
    ops.status()
    assert len(reports) == 300


def test_an_option_without_a_truth_value_raises_its_own_error(cuda):
    import torch
    from t8b import ops

    class Neither:
        def __bool__(self):
            raise KeyError("neither")

    x, w = torch.zeros(4, 16, device="cuda").bfloat16(), torch.zeros(8, 16, device="cuda").bfloat16()
    y = torch.zeros(4, 8, device="cuda").bfloat16()
    for call in (lambda: ops.layer_norm(x, save=Neither()), lambda: ops.linear(x, w, save=Neither()),
                 lambda: ops.gated(x, w, save=Neither()), lambda: ops.linear_backward(y, x, w, input_gradient=Neither()),
                 lambda: ops.gated_backward(y[:, :4], x, w, pre=y, input_gradient=Neither())):
        with pytest.raises(KeyError, match="neither"):
            call()


@pytest.mark.parametrize("gated,rows,n,m,label", [
    (False, 4, 512, 8192, "k_few_rows"), (False, 5, 512, 8192, "k_linear"), (False, 8, 512, 2816, "k_few_rows"),
    (False, 9, 512, 2816, "k_linear"), (False, 16, 512, 1408, "k_few_rows"), (False, 16, 512, 1409, "k_linear"),
    (False, 16, 513, 64, "k_linear"), (False, 17, 64, 64, "k_linear"), (True, 8, 512, 1408, "k_few_rows"),
    (True, 9, 512, 1408, "k_gated"), (True, 16, 512, 704, "k_few_rows"), (True, 16, 151, 1409, "k_gated"), (True, 16, 256, 1408, "k_few_rows"),
    (True, 16, 512, 705, "k_gated"),
])
def test_forward_passes_of_few_rows_take_the_form_that_measured_faster(cuda, gated, rows, n, m, label):
    """Small integers: every sum is exact in fp32, so the outputs are equal whichever form computes them."""
    import torch
    from t8b import ops, profile
    E = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(rows + n + m)
    columns = 2 * m if gated else m
    x = torch.randint(-2, 3, (rows, n), device="cuda", generator=g).to(E)
    w = torch.randint(-1, 2, (columns, n), device="cuda", generator=g).to(E)
    b = torch.randint(-3, 4, (columns,), device="cuda", generator=g).float()
    profile.enable()
    try:
        got = ops.gated(x, w, b, activation="relu") if gated else ops.linear(x, w, b, out_dtype=torch.float32)
        launched = profile.report()
    finally:
        profile.enable(False)
    assert set(launched) - {"k_pack"} == {label}
    z = x.double() @ w.double().T + b.double()
    if gated:
        z = z[:, :m].clamp(min=0) * z[:, m:]
        assert torch.equal(got.double(), z.to(E).double())
    else:
        assert torch.equal(got.double(), z)
