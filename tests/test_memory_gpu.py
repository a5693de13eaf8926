"""The memory operators (t8b.ops: causal_conv, selective_scan, policy_loss) against their definitions in 64
bits on the same inputs.

Bounds, derived from how each value is computed (u = half the output type's spacing, relative):
  - a sum of k products in fp32: k 2^-23 sum|terms|, whatever the order;
  - an activation, its slope: 2^-19 (1 + |z|), and what its argument is off by (slopes are at most 1.2);
  - 2^x 2^-22, its argument's two roundings 2^-23 |argument|; softplus of |v| < 8: 2^-20, most of it from
    v's own rounding; silu relative to itself: 2^-20 (1 + |z|);
  - a path through k decays gathers k of their errors: relative to the sum of the terms' magnitudes a scan's
    outputs and gradients are off by at most 2^-20 ((steps + 8) (2 + max |size a|) + 1 + max |z|).
"""
import pytest

import memory64 as m

pytestmark = pytest.mark.gpu

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -25}
TYPES = ["float32", "bfloat16", "float16"]


def close(got, want, bound, name=""):
    """|got - want| <= bound + the output's own rounding, element by element."""
    import torch
    assert got.shape == want.shape, (name, got.shape, want.shape)
    t = str(got.dtype).split(".")[1]
    limit = bound + UNIT[t] * (1 + 2 ** -7) * want.abs() + TINY[t]
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (name, int(bad.sum()), float((off / limit).nan_to_num(1e30).max()), torch.nonzero(bad)[:4].tolist())


class Maker:
    """Normal values from a seed, as tensors [s][t][...] in either order, or column ranges of wider buffers whose
    rest is NaN."""

    def __init__(self, seed, dtype, order="sequence", slack=0, shift=0):
        import torch
        self.torch, self.dtype, self.order, self.slack, self.shift = torch, dtype, order, slack, shift
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=None, scale=1.0):
        return (self.torch.randn(*shape, device="cuda", generator=self.g) * scale).to(dtype or self.torch.float32)

    def track(self, s, t, *row, scale=1.0):
        width = 1
        for r in row:
            width *= r
        first = (s, t) if self.order == "sequence" else (t, s)
        wide = self.torch.full((*first, width + self.slack), float("nan"), device="cuda", dtype=self.dtype)
        view = wide[..., self.shift:self.shift + width]
        view.copy_(self.torch.randn(*first, width, device="cuda", generator=self.g) * scale)
        if self.order != "sequence":
            view = view.transpose(0, 1)
        return view.unflatten(-1, row)

    def rounds(self, s, t, reset, lengths, share=0.15):
        r = n = None
        if reset:
            r = self.torch.rand(t, s, device="cuda", generator=self.g).t() < share
        if lengths:
            n = self.torch.randint(0, t + 1, (s,), device="cuda", generator=self.g, dtype=self.torch.int32)
            n[0] = t
            if s > 1:
                n[1] = 0
        return r, n


# ------------------------------------------------------------------ causal convolution
CONV = [
    # sequences, steps, channels, order, slack, shift
    (1, 1, 1, "sequence", 0, 0), (2, 3, 8, "sequence", 0, 0), (3, 2, 7, "time", 0, 0), (5, 33, 24, "time", 8, 0),
    (4, 64, 12, "sequence", 3, 1), (3, 100, 264, "sequence", 0, 0), (2, 31, 1032, "time", 1032, 1032), (70, 5, 40, "time", 0, 0),
    (1, 257, 33, "sequence", 0, 0),
]


def conv_error(x, w, b, state, reset, lengths):
    """What the pre-activations are off by."""
    ab = None if b is None else b.abs()
    size, _ = m.conv64(x.abs(), w.abs(), ab, None if state is None else state.abs(), reset, lengths)
    return (w.shape[1] + 2) * 2 ** -23 * size


@pytest.mark.parametrize("s,t,n,order,slack,shift", CONV)
@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
def test_conv(cuda, s, t, n, order, slack, shift, type_name, width):
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    k = Maker(s * 1000 + t * 10 + n + width, T, order, slack, shift)
    x = k.track(s, t, n)
    for act, params, held, reset, lengths in (("silu", torch.float32, True, True, False), ("none", T, False, False, True),
                                              ("gelu", torch.float32, True, True, True), ("tanh", T, True, False, False),
                                              ("relu", torch.float32, False, False, False)):
        w, b = k.normal(n, width, dtype=params), k.normal(n, dtype=params) if act != "none" else None
        state = k.normal(s, width - 1, n, dtype=T) if held else None
        reset, lengths = k.rounds(s, t, reset, lengths)
        y, final = ops.causal_conv(x, w, b, activation=act, state=state, reset=reset, lengths=lengths, final=True)
        p, end = m.conv64(x, w, b, state, reset, lengths)
        live = m.live_of(lengths, s, t, x.device)[:, :, None]
        want = torch.where(live, m.act64(p, act)[0], torch.zeros_like(p))
        off = conv_error(x, w, b, state, reset, lengths)
        close(y, want, 1.2 * off + (2 ** -19 * (1 + p.abs()) if act not in ("none", "relu") else 0), act)
        assert torch.equal(final.double(), end) and final.dtype is T
        if s > 1 and t > 1:
            assert (y.stride(0) < y.stride(1)) == (order == "time")
        if slack and order == "sequence":
            packed = ops.causal_conv(x.contiguous(), w, b, activation=act, state=state, reset=reset, lengths=lengths)
            assert torch.equal(y, packed)  # other packs, the same sums
        assert torch.equal(y, ops.causal_conv(x, w, b, activation=act, state=state, reset=reset, lengths=lengths))


@pytest.mark.parametrize("s,t,n,order,slack,shift", CONV)
@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
def test_conv_backward(cuda, s, t, n, order, slack, shift, type_name, width):
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    k = Maker(s * 1000 + t * 10 + n + width + 1, T, order, slack, shift)
    x, dy = k.track(s, t, n), k.track(s, t, n)
    for act, params, held, reset, lengths, tail in (("silu", torch.float32, True, True, False, True), ("none", T, False, False, True, False),
                                                    ("gelu", torch.float32, True, True, True, False), ("tanh", T, True, False, True, True)):
        w, b = k.normal(n, width, dtype=params), k.normal(n, dtype=params) if act != "none" else None
        state = k.normal(s, width - 1, n, dtype=T) if held else None
        dfinal = k.normal(s, width - 1, n, dtype=T) if tail else None
        reset, lengths = k.rounds(s, t, reset, lengths)
        dx, dw, db, dstate = ops.causal_conv_backward(dy, x, w, b, activation=act, state=state, reset=reset, lengths=lengths, dfinal=dfinal)
        assert (db is None) == (b is None) and (dstate is None) == (state is None)
        assert dw.dtype is params and dx.dtype is T
        p, _ = m.conv64(x, w, b, state, reset, lengths)
        live = m.live_of(lengths, s, t, x.device)[:, :, None]
        d = torch.where(live, dy.double(), torch.zeros_like(p))
        dp = d * m.act64(p, act)[1]
        off = d.abs() * (conv_error(x, w, b, state, reset, lengths) + (2 ** -19 * (1 + p.abs()) if act != "none" else 0))
        want = m.conv_grad64(dp, x, w, state, reset, lengths, dfinal)
        absolute = (x.abs(), w.abs(), None if state is None else state.abs(), reset, lengths)
        slip = m.conv_grad64(off, *absolute, None)
        size = m.conv_grad64(dp.abs(), *absolute, None if dfinal is None else dfinal.abs())
        close(dx, want[0], slip[0] + (width + 3) * 2 ** -23 * size[0], "dx " + act)
        close(dw, want[1], slip[1] + (s * t + 64) * 2 ** -23 * size[1], "dweight " + act)
        if b is not None:
            close(db, want[2], slip[2] + (s * t + 64) * 2 ** -23 * size[2], "dbias " + act)
        if state is not None:
            close(dstate, want[3], slip[3] + (width + 3) * 2 ** -23 * size[3], "dstate " + act)
        again = ops.causal_conv_backward(dy, x, w, b, activation=act, state=state, reset=reset, lengths=lengths, dfinal=dfinal)
        assert all(u is v or torch.equal(u, v) for u, v in zip((dx, dw, db, dstate), again))


def test_conv_of_integers_is_exact(cuda):
    """Small integers and relu: every product and sum is exact, forward and backward, in any order; over many
    runs of steps and workers, remainders among them."""
    import torch
    from t8b import ops
    for s, t, n, width in ((3, 300, 20, 4), (700, 7, 9, 3), (1, 1000, 516, 2)):
        g = torch.Generator(device="cuda").manual_seed(t)

        def whole(*shape):
            return torch.randint(-3, 4, shape, device="cuda", generator=g).float()

        x, dy, w, b, state = whole(s, t, n), whole(s, t, n), whole(n, width), whole(n) + 0.5, whole(s, width - 1, n)
        reset = torch.rand(s, t, device="cuda", generator=g) < 0.1
        y = ops.causal_conv(x, w, b, activation="relu", state=state, reset=reset)
        p, _ = m.conv64(x, w, b, state, reset)
        assert torch.equal(y.double(), p.clamp(min=0))
        got = ops.causal_conv_backward(dy, x, w, b, activation="relu", state=state, reset=reset)
        want = m.conv_grad64(dy.double() * (p > 0), x, w, state, reset)
        for u, v in zip(got, want):
            assert torch.equal(u.double(), v)


@pytest.mark.parametrize("s,n,slack", [(1, 1, 0), (3, 8, 0), (96, 1032, 0), (7, 33, 5), (130, 24, 8)])
@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
def test_conv_steps_are_the_sequence(cuda, s, n, slack, type_name, width):
    """Step by step on the state, bit for bit what a sequence gives at once, the final state too."""
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    k = Maker(s + n + width, T, "time", slack, slack)
    x = k.track(s, 9, n)
    w, b, state = k.normal(n, width), k.normal(n), k.normal(s, width - 1, n, dtype=T)
    reset, _ = k.rounds(s, 9, True, False)
    y, final = ops.causal_conv(x, w, b, activation="silu", state=state, reset=reset, final=True)
    held = state.clone()
    for t in range(9):
        one = ops.causal_conv_step(x[:, t], w, b, held, activation="silu", reset=reset[:, t])
        assert torch.equal(one, y[:, t]), t
    assert torch.equal(held, final)


# ------------------------------------------------------------------ selective scan
SCAN = [
    # sequences, steps, channels, groups, states, order, slack, shift
    (1, 1, 1, 1, 1, "sequence", 0, 0), (2, 7, 6, 1, 16, "sequence", 0, 0), (3, 8, 64, 1, 4, "time", 0, 0),
    (2, 9, 65, 1, 11, "sequence", 3, 1), (3, 40, 132, 2, 16, "time", 8, 0), (2, 23, 30, 3, 24, "sequence", 0, 0),
    (2, 17, 40, 2, 64, "time", 5, 5), (9, 16, 130, 1, 33, "sequence", 0, 0), (40, 5, 8, 1, 2, "time", 0, 0),
]


class Scanning:
    """A scan's inputs, its definition and its bound."""

    def __init__(self, k, s, t, n, groups, states, gate, skip, biased, softplus, held, reset, lengths):
        torch = k.torch
        self.u, self.delta = k.track(s, t, n), k.track(s, t, n)
        self.b, self.c = k.track(s, t, groups, states), k.track(s, t, groups, states)
        self.a = -torch.exp(k.normal(n, states))
        self.z = k.track(s, t, n) if gate else None
        self.d = k.normal(n) if skip else None
        self.delta_bias = k.normal(n) - 1.5 if biased else None
        self.softplus = softplus
        self.state = k.normal(s, n, states) if held else None
        self.reset, self.lengths = k.rounds(s, t, reset, lengths)
        live = m.live_of(self.lengths, s, t, self.u.device)[:, :, None]
        self.live = live

        def read(v):
            return torch.where(live, v.double(), torch.zeros((), dtype=torch.float64, device="cuda"))

        v = read(self.delta) + (0 if self.delta_bias is None else (self.delta_bias.double()))
        v = torch.where(live, v, torch.zeros_like(v))
        if softplus:
            self.size, self.slope = torch.nn.functional.softplus(v, threshold=50.0), torch.sigmoid(v)
        else:
            self.size, self.slope = v, torch.ones_like(v)
        self.u64 = read(self.u)
        self.b64, self.c64 = (torch.where(live[:, :, :, None], w.double(), torch.zeros((), dtype=torch.float64, device="cuda")) for w in (self.b, self.c))
        self.gate, self.gate_slope, most = torch.ones_like(v), torch.zeros_like(v), 0.0
        if gate:
            z = read(self.z)
            self.gate, self.gate_slope = m.act64(z, "silu")
            self.z64, most = z, float(z.abs().max())
        rate = float((self.size[..., None] * self.a.double()).abs().max())
        self.off = 2 ** -20 * ((t + 8) * (2 + rate) + 1 + most)
        d = None if self.d is None else self.d.double()
        state = None if self.state is None else self.state.double()
        self.out, self.states, self.befores, self.final, self.decays = m.scan64(self.size, self.u64, self.a, self.b64, self.c64, d, state,
                                                                                self.reset, self.lengths)
        absolute = lambda v: None if v is None else v.abs()
        self.sizes = m.scan64(self.size.abs(), self.u64.abs(), self.a, self.b64.abs(), self.c64.abs(), absolute(d), absolute(state),
                              self.reset, self.lengths, self.decays)

    def operands(self):
        return self.u, self.delta, self.a, self.b, self.c

    def common(self, lengths=True):
        return dict(d=self.d, z=self.z, delta_bias=self.delta_bias, softplus=self.softplus, state=self.state, reset=self.reset,
                    lengths=self.lengths)

    def gradients(self, dy, dfinal):
        """(values, magnitudes) of du, ddelta, da, db, dc, dd, dz, ddelta_bias, dstate."""
        import torch
        dy = torch.where(self.live, dy.double(), torch.zeros_like(self.size))
        d = None if self.d is None else self.d.double()
        both = []
        for absolute in (False, True):
            f = torch.abs if absolute else (lambda v: v)
            states, befores = (self.sizes[1], self.sizes[2]) if absolute else (self.states, self.befores)
            gs = f(dy * self.gate)
            du, dsize, da, db, dc, dd, dstate = m.scan_grad64(gs, f(self.size), f(self.u64), f(self.a), f(self.b64), f(self.c64),
                                                              None if d is None else f(d), states, befores, self.decays, self.reset,
                                                              self.lengths, None if dfinal is None else f(dfinal))
            dv = dsize * self.slope
            out = self.sizes[0] if absolute else self.out
            # the slope's own error is not relative to itself
            dz = f(dy) * out * ((self.gate_slope.abs() + 2 ** -1 * (1 + getattr(self, "z64", out).abs()) / 8) if absolute else self.gate_slope)
            both.append([du, dv, da, db, dc, dd, dz, dv.sum((0, 1)), dstate])
        return both


VARIANTS = [
    # gate, skip, biased, softplus, held, reset, lengths
    (True, True, True, True, True, True, False), (False, False, False, True, False, False, True),
    (True, False, True, True, True, True, True), (False, True, False, False, True, False, False),
]


def scanning(k, s, t, n, groups, states, variant):
    x = Scanning.__new__(Scanning)
    if not variant[3]:  # sizes as they come: kept positive, or h grows without bound
        original = k.track

        def positive(*shape, **more):
            v = original(*shape, **more)
            v.copy_(v.abs() * 0.3) if len(shape) == 3 else None
            return v

        k.track = positive
        x.__init__(k, s, t, n, groups, states, *variant)
        k.track = original
    else:
        x.__init__(k, s, t, n, groups, states, *variant)
    return x


@pytest.mark.parametrize("s,t,n,groups,states,order,slack,shift", SCAN)
@pytest.mark.parametrize("type_name", TYPES)
def test_scan(cuda, s, t, n, groups, states, order, slack, shift, type_name):
    import torch
    from t8b import ops
    for i, variant in enumerate(VARIANTS):
        k = Maker(s * 1000 + t * 10 + n + i, getattr(torch, type_name), order, slack, shift)
        x = scanning(k, s, t, n, groups, states, variant)
        y, final, saved = ops.selective_scan(*x.operands(), **x.common(), final=True, save=True)
        close(y, x.out * x.gate, x.off * x.sizes[0] * x.gate.abs(), f"y {variant}")
        close(final, x.final, x.off * x.sizes[3], f"final {variant}")
        assert y.dtype is x.u.dtype and final.dtype is torch.float32
        if s > 1 and t > 1:
            assert (y.stride(0) < y.stride(1)) == (order == "time")
        assert torch.equal(y, ops.selective_scan(*x.operands(), **x.common()))
        if groups == 1:
            assert torch.equal(y, ops.selective_scan(x.u, x.delta, x.a, x.b[:, :, 0], x.c[:, :, 0], **x.common()))


@pytest.mark.parametrize("s,t,n,groups,states,order,slack,shift", SCAN)
@pytest.mark.parametrize("type_name", TYPES)
def test_scan_backward(cuda, s, t, n, groups, states, order, slack, shift, type_name):
    import torch
    from t8b import ops
    names = ("du", "ddelta", "da", "db", "dc", "dd", "dz", "ddelta_bias", "dstate")
    for i, variant in enumerate(VARIANTS):
        k = Maker(s * 1000 + t * 10 + n + i, getattr(torch, type_name), order, slack, shift)
        x = scanning(k, s, t, n, groups, states, variant)
        dy = k.track(s, t, n)
        dfinal = k.normal(s, n, states) if i % 2 == 0 else None
        _, saved = ops.selective_scan(*x.operands(), **x.common(), save=True)
        got = ops.selective_scan_backward(dy, *x.operands(), saved, **x.common(), dfinal=dfinal)
        want, sizes = x.gradients(dy, dfinal)
        given = dict(dd=x.d, dz=x.z, ddelta_bias=x.delta_bias, dstate=x.state)
        for name, g, w, size in zip(names, got, want, sizes):
            if name in given and given[name] is None:
                assert g is None
                continue
            more = s * t * 2 ** -24 if name in ("da", "dd", "ddelta_bias") else n * 2 ** -24 if name in ("db", "dc") else 0
            close(g, w, (2 * x.off + more) * size, f"{name} {variant}")
        again = ops.selective_scan_backward(dy, *x.operands(), saved, **x.common(), dfinal=dfinal)
        assert all(u is v or torch.equal(u, v) for u, v in zip(got, again))


@pytest.mark.parametrize("s,n,groups,states", [(1, 1, 1, 1), (1, 40, 1, 16), (3, 6, 2, 7), (9, 33, 1, 64), (130, 10, 1, 12), (5, 8, 1, 50)])
@pytest.mark.parametrize("type_name", TYPES)
def test_scan_steps(cuda, s, n, groups, states, type_name):
    """Steps on a state in place against the definition over all of them (bounds as for a sequence)."""
    import torch
    from t8b import ops
    t = 6
    for i, variant in enumerate(VARIANTS[:1] + VARIANTS[3:]):
        k = Maker(s + n + states + i, getattr(torch, type_name), "time", 3 * i, i)
        x = scanning(k, s, t, n, groups, states, variant)
        state = x.state.clone()
        for at in range(t):
            z = None if x.z is None else x.z[:, at]
            y = ops.selective_scan_step(x.u[:, at], x.delta[:, at], x.a, x.b[:, at], x.c[:, at], state, d=x.d, z=z,
                                        delta_bias=x.delta_bias, softplus=x.softplus, reset=None if x.reset is None else x.reset[:, at])
            close(y, (x.out * x.gate)[:, at], x.off * (x.sizes[0] * x.gate.abs())[:, at], f"y {at}")
        close(state, x.final, x.off * x.sizes[3], "state")


@pytest.mark.parametrize("s,t,n,groups,states", [(1, 700, 40, 1, 16), (2, 1001, 20, 2, 5), (1, 515, 12, 1, 40)])
def test_scan_in_chunks(cuda, s, t, n, groups, states):
    """Few and long sequences, which are cut into chunks: as above, with resets and lengths that end in any chunk."""
    import torch
    from t8b import ops, profile
    for variant in ((True, True, True, True, True, False, False), (False, True, True, True, True, True, True)):
        k = Maker(t + n, torch.float32)
        x = scanning(k, s, t, n, groups, states, variant)
        if x.reset is not None:
            x.reset &= torch.rand(s, t, device="cuda", generator=k.g) < 0.05  # most chunks have none
            x = _again(x, k)
        dy, dfinal = k.track(s, t, n), k.normal(s, n, states)
        profile.enable()
        try:
            y, final, saved = ops.selective_scan(*x.operands(), **x.common(), final=True, save=True)
            got = ops.selective_scan_backward(dy, *x.operands(), saved, **x.common(), dfinal=dfinal)
            launched = profile.report()
        finally:
            profile.enable(False)
        assert "k_scan_ends" in launched and "k_scan_back_ends" in launched
        close(y, x.out * x.gate, x.off * x.sizes[0] * x.gate.abs(), "y")
        close(final, x.final, x.off * x.sizes[3], "final")
        want, sizes = x.gradients(dy, dfinal)
        for name, g, w, size in zip(("du", "ddelta", "da", "db", "dc", "dd", "dz", "ddelta_bias", "dstate"), got, want, sizes):
            if g is not None:
                close(g, w, (2 * x.off + s * t * 2 ** -24) * size, name)


def _again(x, k):
    """The definition once more, for resets that changed."""
    d, state = x.d.double(), x.state.double()
    x.out, x.states, x.befores, x.final, x.decays = m.scan64(x.size, x.u64, x.a, x.b64, x.c64, d, state, x.reset, x.lengths)
    x.sizes = m.scan64(x.size.abs(), x.u64.abs(), x.a, x.b64.abs(), x.c64.abs(), d.abs(), state.abs(), x.reset, x.lengths, x.decays)
    return x


# ------------------------------------------------------------------ policy loss
LOSS = [(1, 1, 0), (3, 5, 0), (40, 33, 0), (96, 368, 0), (17, 368, 5), (9, 1000, 0), (7, 1024, 8), (5, 1025, 0), (4, 4099, 0), (3, 4096, 0),
        (2, 50257, 0), (3, 20008, 3), (300, 64, 0)]


def packed_bits(legal):
    import torch
    rows, n = legal.shape
    words = -(-n // 32)
    padded = torch.zeros(rows, words * 32, dtype=torch.bool, device=legal.device)
    padded[:, :n] = legal
    v = (padded.view(rows, words, 32).long() << torch.arange(32, device=legal.device)).sum(2)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).int()


@pytest.mark.parametrize("rows,n,slack", LOSS)
@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("mask", ["none", "bits", "bytes"])
def test_policy_loss(cuda, rows, n, slack, type_name, mask):
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    g = torch.Generator(device="cuda").manual_seed(rows * n + slack)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def held(v):
        wide = torch.full((rows, n + slack), float("nan"), device="cuda", dtype=T)
        wide[:, :n] = v
        return wide[:, :n]

    z = held(3 * normal(rows, n))
    actions = torch.randint(n, (rows,), device="cuda", generator=g)
    legal = None
    if mask != "none":
        legal = torch.rand(rows, n, device="cuda", generator=g) < torch.rand(rows, 1, device="cuda", generator=g)
        if rows > 2:
            legal[torch.arange(rows - 1), actions[:-1]] = True
            legal[0] = False  # a row that its mask leaves empty
            z[1] = torch.where(legal[1], z[1], float("nan"))  # what is not legal may be anything
    if rows > 4:
        actions[3], actions[4] = -1, n
    lp = m.loss64(z, actions, torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), legal)["log_probabilities"]
    drift = 0.2 * normal(rows).double()
    for border in (0.8, 1.3):  # the loss's slope jumps where the ratio is clipped
        drift = torch.where((drift.exp() - border).abs() < 1e-3, drift + 0.01, drift)
    old, advantages, weights = (lp - drift).float(), normal(rows), torch.rand(rows, device="cuda", generator=g)
    frozen, sampled = held(3 * normal(rows, n)), (lp + 0.3 * normal(rows).double()).float()
    given = None if mask == "none" else packed_bits(legal) if mask == "bits" else legal if rows % 2 else legal.to(torch.uint8)
    for reference, kl, entropy, weighted in ((None, 0.0, 0.0, False), (None, 0.0, 0.05, True), (frozen, 0.3, 0.02, True), (sampled, 0.2, 0.0, True)):
        out = ops.policy_loss(z, actions, old, advantages, mask=given, reference=reference, weights=weights if weighted else None, clip=0.2,
                              clip_high=0.3, kl=kl, entropy=entropy)
        got = dict(zip(("loss", "log_probabilities", "entropies", "divergences", "dlogits"), out))
        exact = reference is frozen
        want = m.loss64(z, actions, old, advantages, legal, reference=frozen if exact else None, sampled=sampled if reference is sampled else None,
                        weights=weights if weighted else None, low=0.2, high=0.3, kl=kl, entropy=entropy)
        p, logp = want["p"], want["logp"]
        spread = (p * logp.abs()).sum(1)
        d_lp = 2 ** -20 * (1 + spread) + 2 ** -23 * want["log_probabilities"].abs()
        d_h = 2 ** -18 * (1 + spread)
        r = want["ratio"].where(want["counts"], torch.zeros_like(lp))
        d_k, far = torch.zeros_like(lp), torch.zeros_like(p)
        slope = want["slope"].where(want["counts"], torch.zeros_like(lp)).abs()
        d_slope = r * advantages.double().abs() * (d_lp + 2 ** -21)
        if exact:
            # z - q and the two sums' logarithms, which the divergence is a difference of
            far = torch.where(p > 0, (z.double() - frozen.double()).abs(), torch.zeros_like(p))
            shift = (torch.where(p > 0, z.double() - frozen.double(), torch.zeros_like(p)) - want["apart"]).abs().amax(1)
            d_k = 2 ** -18 * (1 + (p * far).sum(1) + shift)
            far = far + shift[:, None]
        elif reference is sampled:
            e = (sampled.double() - want["log_probabilities"]).where(want["counts"], torch.zeros_like(lp))
            grown = torch.expm1(e)
            d_k = grown.abs() * d_lp + 2 ** -20 * (grown.abs() + e.abs()) * e.abs() + 2 ** -22 * want["divergences"]
            d_slope = d_slope + kl * (grown + 1) * (d_lp + 2 ** -21)
        close(got["log_probabilities"], want["log_probabilities"], d_lp, "log-probabilities")
        close(got["entropies"], want["entropies"], d_h, "entropies")
        close(got["divergences"], want["divergences"], d_k, "divergences")
        close(got["loss"], want["loss"], d_slope + r * advantages.double().abs() * 2 ** -22 + kl * (d_k + 2 ** -22 * want["divergences"]) +
              entropy * (d_h + 2 ** -22 * want["entropies"]) + 2 ** -22 * want["loss"].abs(), "loss")
        inner = slope[:, None] + kl * (far + want["divergences"].abs()[:, None]) + entropy * (logp.abs() + want["entropies"].abs()[:, None])
        d_inner = d_slope[:, None] + kl * (2 ** -20 * far + d_k[:, None]) + entropy * (2 ** -20 * logp.abs() + d_h[:, None]) + 2 ** -21 * inner
        w = want["weight"].abs()[:, None]
        off = w * p * (d_inner + inner * (d_lp[:, None] + 2 ** -20 * (1 + logp.abs())))
        off = off + torch.where(torch.arange(n, device="cuda") == actions[:, None], w * (d_slope + 2 ** -22 * slope)[:, None], torch.zeros_like(off))
        close(got["dlogits"], want["dlogits"], torch.where(want["counts"][:, None], off, torch.zeros_like(off)), "dlogits")
        if legal is not None:
            assert not got["dlogits"][~legal].any()
        assert got["dlogits"].dtype is T and got["dlogits"].stride(0) * got["dlogits"].element_size() % 16 == 0
        alone = ops.policy_loss(z, actions, old, advantages, mask=given, reference=reference, weights=weights if weighted else None, clip=0.2,
                                clip_high=0.3, kl=kl, entropy=entropy, gradient=False)
        assert len(alone) == 4 and all(torch.equal(u, v) for u, v in zip(alone, out))
        again = ops.policy_loss(z, actions, old, advantages, mask=given, reference=reference, weights=weights if weighted else None, clip=0.2,
                                clip_high=0.3, kl=kl, entropy=entropy)
        assert torch.equal(again[4], out[4])
