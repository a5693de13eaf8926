"""The selective scan over sequences that are cut into chunks, where the chunks' ends are joined by the decay of a whole
chunk: growth and decay beyond fp32's range, slow states, pieces, and what a reset keeps apart.

Bounds as derived in test_memory_gpu.py: relative to the sum of the terms' magnitudes 2^-20 ((steps + 8) (2 + max |size a|)
+ 1), twice that and the sums' own roundings for gradients."""
import pytest

import memory64 as m
from test_memory_gpu import close

pytestmark = pytest.mark.gpu

NAMES = ("du", "ddelta", "da", "db", "dc", "dstate")


class Problem:
    """A scan in fp32 without softplus, gate and skip: one group, one sequence."""

    def __init__(self, seed, t, n, states, rate):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
        self.u, self.delta, self.dy = self.normal(1, t, n), self.normal(1, t, n).abs() * 0.3, self.normal(1, t, n)
        self.b, self.c = self.normal(1, t, states), self.normal(1, t, states)
        low, high = rate
        self.a = -(low + (high - low) * torch.rand(n, states, device="cuda", generator=g))
        self.state, self.reset, self.dfinal = None, None, None

    def run(self, copies=1, backward=True):
        """The operator's outputs for `copies` of the sequence (the first one's; sums over sequences of all), and what it
        launched."""
        from t8b import ops, profile

        def many(v):
            return None if v is None else v.expand(copies, *v.shape[1:]).contiguous()

        u, delta, b, c, dy = map(many, (self.u, self.delta, self.b, self.c, self.dy))
        more = dict(softplus=False, state=many(self.state), reset=many(self.reset))
        profile.enable()
        try:
            y, final, saved = ops.selective_scan(u, delta, self.a, b, c, final=True, save=True, **more)
            out = {"y": y, "final": final}
            if backward:
                du, ddelta, da, db, dc, _, _, _, dstate = ops.selective_scan_backward(dy, u, delta, self.a, b, c, saved, dfinal=many(self.dfinal), **more)
                out.update(du=du, ddelta=ddelta, da=da, db=db, dc=dc, dstate=dstate)
            launched = profile.report()
        finally:
            profile.enable(False)
        return {k: v if v is None or k == "da" else v[:1] for k, v in out.items()}, launched

    def defined(self, backward=True):
        """The definition's values, and bounds."""
        import torch
        t, n = self.u.shape[1:]
        size = self.delta.double()
        b, c = self.b[:, :, None], self.c[:, :, None]
        values = m.scan64(size, self.u, self.a, b, c, None, self.state, self.reset)
        state = None if self.state is None else self.state.abs()
        sizes = m.scan64(size.abs(), self.u.abs(), self.a, b.abs(), c.abs(), None, state, self.reset, None, values[4])
        off = 2 ** -20 * ((t + 8) * (2 + float((size[..., None] * self.a.double()).abs().max())) + 1)
        want = {"y": values[0], "final": values[3]}
        bound = {"y": off * sizes[0], "final": off * sizes[3]}
        if backward:
            absolute = torch.abs
            both = []
            for f, v in ((lambda w: w, values), (absolute, sizes)):
                dfinal = None if self.dfinal is None else f(self.dfinal)
                du, dsize, da, db, dc, _, dstate = m.scan_grad64(f(self.dy), f(size), f(self.u), f(self.a), f(b), f(c), None, v[1], v[2],
                                                                values[4], self.reset, None, dfinal)
                both.append(dict(zip(NAMES, (du, dsize, da, db[:, :, 0], dc[:, :, 0], dstate))))
            for name in NAMES:
                more = {"da": t, "db": n, "dc": n}.get(name, 0) * 2 ** -24
                want[name], bound[name] = both[0][name], (2 * off + more) * both[1][name]
        return want, bound


def check(got, want, bound):
    for name, v in want.items():
        if got[name] is not None:
            close(got[name], v, bound[name], name)


def test_a_chunk_that_grows_over_nothing(cuda):
    """Negative sizes over an empty state: whole chunks grow by 2^138 and more, and what they grow is 0. One sequence,
    which is cut, and the same among 320 (forward) or 590, which are not, give the definition's values."""
    x = Problem(3, 600, 40, 16, (0.8, 1.2))
    x.u[:, :160] = 0
    x.delta[:, :160] = -3
    want, bound = x.defined(backward=False)
    for copies, cut in ((1, True), (320, False)):
        got, launched = x.run(copies, backward=False)
        assert ("k_scan_ends" in launched) == cut
        check(got, want, bound)
    # and behind a reset, where the gradient is 0 as well
    import torch
    x = Problem(4, 600, 40, 16, (0.8, 1.2))
    x.reset = torch.zeros(1, 600, dtype=torch.bool, device="cuda")
    x.reset[:, 440] = True
    x.u[:, 440:] = 0
    x.dy[:, 440:] = 0
    x.delta[:, 440:] = -3
    want, bound = x.defined()
    for copies, cut in ((1, True), (590, False)):
        got, launched = x.run(copies)
        assert ("k_scan_back_ends" in launched) == cut
        got["da"] = got["da"] / copies
        check(got, want, bound)


@pytest.mark.parametrize("size,start", [(-2.3, 1e-35), (-5.0, 0.0), (2.3, 1e33), (5.0, 1e38)])
def test_decays_of_a_chunk_beyond_the_range(cuda, size, start):
    """A first chunk of 40 steps whose decay alone is outside of fp32's range (2^133, 2^289 and their inverses), and whose
    product with the state it starts from is not."""
    import torch
    x = Problem(5, 600, 40, 16, (0.98, 1.02))
    x.delta[:, :40] = size
    x.u[:, :60] = 0  # for some steps nothing else is there
    x.state = torch.full((1, 40, 16), start, device="cuda") * (1 + x.normal(1, 40, 16).abs()).clamp(max=3)
    want, bound = x.defined(backward=False)
    for copies, cut in ((1, True), (320, False)):
        got, launched = x.run(copies, backward=False)
        assert ("k_scan_ends" in launched) == cut
        assert bool(want["y"].float().isfinite().all())
        check(got, want, bound)


def near(got, want, limit, name):
    off, size = float((got.double() - want.double()).norm()), float(want.double().norm())
    assert off <= limit * size, (name, off, size, limit)  # (a state behind a reset may be 0)


@pytest.mark.parametrize("s,t,n,groups,states", [(1, 1000, 40, 1, 16), (2, 777, 24, 2, 24), (1, 600, 12, 1, 64)])
@pytest.mark.parametrize("cuts", [False, True])
def test_slow_states_carry_over(cuda, s, t, n, groups, states, cuts):
    """Sizes of some 0.02 under rates of 0.2 to 1: a state lasts for hundreds of steps, and what a chunk takes over is most of
    what it gives. In the norm, against the definition and against the same sequence in three pieces that hand their
    states on (the last two as gradients too): a decay is off by 2^-25 in the mean (all in one direction, at worst: t of
    them) and by 2^-22 each way (t^0.5 of them); sums, products and one chunk's decay for all of its steps 2^-19.
    A carry that is 0.1 % off is beyond that."""
    import torch
    from t8b import ops, profile
    g = torch.Generator(device="cuda").manual_seed(t)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    u, dy, z, b, c = normal(s, t, n), normal(s, t, n), normal(s, t, n), normal(s, t, groups, states), normal(s, t, groups, states)
    delta, bias = 0.3 * normal(s, t, n), torch.full((n,), -4.0, device="cuda")
    a = -(0.2 + 0.8 * torch.rand(n, states, device="cuda", generator=g))
    state, dfinal, d = normal(s, n, states), normal(s, n, states), normal(n)
    reset = lengths = None
    if cuts:
        reset = torch.rand(s, t, device="cuda", generator=g) < 1 / 300
        lengths = torch.tensor([t - 77] + [t] * (s - 1), device="cuda", dtype=torch.int32)

    def run(steps, state, dfinal):
        rows = [v[:, steps] for v in (u, delta, b, c)]
        more = dict(d=d, z=z[:, steps], delta_bias=bias, state=state, reset=None if reset is None else reset[:, steps],
                    lengths=None if lengths is None else (lengths - steps.start).clamp(0, steps.stop - steps.start).int())
        y, final, saved = ops.selective_scan(rows[0], rows[1], a, rows[2], rows[3], final=True, save=True, **more)
        back = lambda dfinal: ops.selective_scan_backward(dy[:, steps], rows[0], rows[1], a, rows[2], rows[3], saved, dfinal=dfinal, **more)  # noqa: E731
        return y, final, back

    profile.enable()
    try:
        y, final, back = run(slice(0, t), state, None)
        got = back(dfinal)
        launched = profile.report()
    finally:
        profile.enable(False)
    assert "k_scan_ends" in launched and "k_scan_back_ends" in launched

    live = m.live_of(lengths, s, t, u.device)[:, :, None]
    v = delta.double() + bias.double()
    size = torch.nn.functional.softplus(v)
    gate, slope = m.act64(z.double(), "silu")
    out, states64, befores, end, decays = m.scan64(size, u, a, b, c, d, state, reset, lengths)
    gs = torch.where(live, dy.double() * gate, torch.zeros_like(v))
    du, dsize, da, db, dc, dd, dstate = m.scan_grad64(gs, size, u, a, b, c, d, states64, befores, decays, reset, lengths, dfinal)
    dv = dsize * torch.sigmoid(v)
    dz = torch.where(live, dy.double() * out * slope, torch.zeros_like(v))
    limit = t * 2 ** -25 + t ** 0.5 * 2 ** -22 + 2 ** -19
    names = ("du", "ddelta", "da", "db", "dc", "dd", "dz", "ddelta_bias", "dstate")
    near(y, out * gate, limit, "y")
    near(final, end, limit, "final")
    for name, v, w in zip(names, got, (du, dv, da, db, dc, dd, dz, dv.sum((0, 1)), dstate)):
        near(v, w, 2 * limit, name)

    parts = [slice(0, t // 3), slice(t // 3, t // 2), slice(t // 2, t)]
    held, runs = state, []
    for part in parts:
        piece, held, back = run(part, held, None)
        runs.append((piece, back))
    near(torch.cat([r[0] for r in runs], 1), y, limit, "y of pieces")
    near(held, final, limit, "final of pieces")
    carry, sums = dfinal, {k: 0 for k in ("da", "dd", "ddelta_bias")}
    rows = {k: [] for k in ("du", "ddelta", "db", "dc", "dz")}
    for _, back in reversed(runs):
        grads = dict(zip(names, back(carry)))
        carry = grads["dstate"]
        for k in rows:
            rows[k].insert(0, grads[k])
        for k in sums:
            sums[k] = sums[k] + grads[k]
    for k, w in zip(names, got):
        near(carry if k == "dstate" else sums[k] if k in sums else torch.cat(rows[k], 1), w, 2 * limit, k + " of pieces")


def test_nothing_of_a_round_reaches_the_ones_before_it(cuda):
    """In a sequence that is cut into chunks: NaN at a reset, bit for bit nothing of it in front."""
    import torch
    from t8b import ops, profile
    g = torch.Generator(device="cuda").manual_seed(3)
    s, t, n, states = 3, 600, 40, 16
    u, delta, z, dy = (torch.randn(s, t, n, device="cuda", generator=g) for _ in range(4))
    b, c = (torch.randn(s, t, states, device="cuda", generator=g) for _ in range(2))
    a, d = -torch.exp(torch.randn(n, states, device="cuda", generator=g)), torch.ones(n, device="cuda")
    state, at = torch.randn(s, n, states, device="cuda", generator=g), 303
    reset = torch.zeros(s, t, dtype=torch.bool, device="cuda")
    reset[:, at] = True

    def run(u, delta, b, c, dy):
        more = dict(d=d, z=z, delta_bias=d, state=state, reset=reset)
        y, saved = ops.selective_scan(u, delta, a, b, c, save=True, **more)
        return y, ops.selective_scan_backward(dy, u, delta, a, b, c, saved, **more)

    profile.enable()
    try:
        y, want = run(u, delta, b, c, dy)
        launched = profile.report()
    finally:
        profile.enable(False)
    assert "k_scan_ends" in launched and "k_scan_back_ends" in launched
    late = [v.clone() for v in (u, delta, b, c, dy)]
    for v in late:
        v[:, at:at + 2] = float("nan")
        v[:, -1] = float("inf")
    y2, got = run(*late)
    assert torch.equal(y[:, :at], y2[:, :at]) and bool(y2[:, at].isnan().all())
    for k in (0, 1, 3, 4, 6):
        assert torch.equal(got[k][:, :at], want[k][:, :at]), k
    assert torch.equal(got[8], want[8])
