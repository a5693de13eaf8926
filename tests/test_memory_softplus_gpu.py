"""The scan's softplus by itself: one step of one state without a start, y = c (0 + size u b) = size for u = b = c = 1.

Each value is within 2^-21: 2^x good to 2^-22, the polynomial to 2^-24, its evaluation, the sum with max(v, 0) and the
products by ones a few 2^-24. Over a million values roundings cancel (1e-7 / 1,000), so that the mean shows what is common to
all: less than 2^-25, where the polynomial's error is below 2^-30 in the mean and the correction of 2^x within 2.6e-8
of its bias (which over x in -0.25 ... 0 is at most that)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low,high", [(-16.0, -8.0), (-8.0, -2.0), (-2.0, -0.25), (-0.25, 0.25), (0.25, 4.0)])
def test_softplus_has_no_bias(cuda, low, high):
    import torch
    from t8b import ops
    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(7)
    v = low + (high - low) * torch.rand(1, 1, n, device="cuda", generator=g)
    one, shared, a = torch.ones(1, 1, n, device="cuda"), torch.ones(1, 1, 1, device="cuda"), torch.full((n, 1), -1.0, device="cuda")
    want = torch.nn.functional.softplus(v.double(), threshold=50.0)
    for y in (ops.selective_scan(one, v, a, shared, shared),
              ops.selective_scan_step(one[0], v[0], a, shared[0], shared[0], torch.zeros(1, n, 1, device="cuda"))[None]):
        off = (y.double() - want) / want
        assert float(off.abs().max()) < 2 ** -21
        assert abs(float(off.mean())) < 2 ** -25
