"""Edges of the memory operators: values, arguments, streams and sizes at which they could go wrong."""
import pytest

import memory64 as m

pytestmark = pytest.mark.gpu


def scan_inputs(s, t, n, states, seed=1, dtype=None, groups=1):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = dtype or torch.float32

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    return dict(u=normal(s, t, n), delta=normal(s, t, n), a=-torch.exp(torch.randn(n, states, device="cuda", generator=g)),
                b=normal(s, t, groups, states), c=normal(s, t, groups, states)), normal


def run_scan(x, dy, **more):
    from t8b import ops
    y, final, saved = ops.selective_scan(**x, final=True, save=True, **more)
    return (y, final) + ops.selective_scan_backward(dy, **x, saved=saved, **more)


def same(got, want):
    import torch
    for k, (u, v) in enumerate(zip(got, want)):
        assert u is v or torch.equal(u, v), k


@pytest.mark.parametrize("t,chunked", [(40, False), (600, True)])
def test_what_a_reset_or_a_length_cuts_off_may_be_anything(cuda, t, chunked):
    """NaN and infinities in a round leave the rounds after it bit for bit as they were, outputs and gradients
    alike, and what lies past a sequence's length is not read."""
    import torch
    from t8b import ops
    s, n, states = 3, 40, 16
    x, normal = scan_inputs(s, t, n, states)
    z, dy, state = normal(s, t, n), normal(s, t, n), torch.randn(s, n, states, device="cuda")
    reset = torch.zeros(s, t, dtype=torch.bool, device="cuda")
    at = t // 2 + 3
    reset[:, at] = True
    lengths = torch.tensor([t, t - 5, at + 9], device="cuda", dtype=torch.int32)
    d, bias = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    more = dict(d=d, z=z, delta_bias=bias, state=state, reset=reset, lengths=lengths)
    want = run_scan(x, dy, **more)
    bad = {k: v.clone() for k, v in x.items()}
    dirty_z, dirty_dy, dirty_state = z.clone(), dy.clone(), torch.full_like(state, float("inf"))
    for value, k in ((float("nan"), 0), (float("inf"), 1), (-float("inf"), 2)):
        for v in (bad["u"], bad["delta"], bad["b"], bad["c"], dirty_z):
            v[k, at - 4:at - 1] = value
            v[k, int(lengths[k]):] = float("nan")
        dirty_dy[k, int(lengths[k]):] = float("nan")
    got = run_scan(bad, dirty_dy, d=d, z=dirty_z, delta_bias=bias, state=dirty_state, reset=reset, lengths=lengths)
    y, final, du, ddelta, da, db, dc, dd, dz, dbias, dstate = range(11)
    for k in (y, du, ddelta, db, dc, dz):
        assert torch.equal(got[k][:, at:], want[k][:, at:]), k
        for q in range(s):
            assert not got[k][q, int(lengths[q]):].any(), k
    assert torch.equal(got[final], want[final])
    if not chunked:
        # and nothing of a round reaches the ones before it
        late = {k: v.clone() for k, v in x.items()}
        for v in (late["u"], late["delta"], late["b"], late["c"]):
            v[:, at] = float("nan")
        got = run_scan(late, dy, **more)
        for k in (y, du, ddelta, db, dc, dz):
            assert torch.equal(got[k][:, :at], want[k][:, :at]), k
        assert torch.equal(got[dstate], want[dstate])
    # the convolution
    w, b = torch.randn(n, 4, device="cuda"), torch.randn(n, device="cuda")
    window = torch.randn(s, 3, n, device="cuda")
    more = dict(activation="silu", state=window, reset=reset, lengths=lengths)
    want = ops.causal_conv(x["u"], w, b, final=True, **more) + ops.causal_conv_backward(dy, x["u"], w, b, **more)
    got = ops.causal_conv(bad["u"], w, b, final=True, **more) + ops.causal_conv_backward(dirty_dy, bad["u"], w, b, **more)
    assert torch.equal(got[0][:, at:], want[0][:, at:]) and torch.equal(got[1], want[1]) and torch.equal(got[2][:, at:], want[2][:, at:])


def test_steps_after_a_reset_forget_anything(cuda):
    import torch
    from t8b import ops
    x, normal = scan_inputs(5, 1, 24, 16, dtype=torch.bfloat16)
    one = {k: v if k == "a" else v[:, 0] for k, v in x.items()}
    state, reset = torch.randn(5, 24, 16, device="cuda"), torch.tensor([0, 1, 0, 1, 1], device="cuda", dtype=torch.uint8)
    clean = torch.where(reset.bool()[:, None, None], torch.zeros_like(state), state)
    dirty = torch.where(reset.bool()[:, None, None], torch.full_like(state, float("nan")), state)
    want = ops.selective_scan_step(**one, state=clean)
    got = ops.selective_scan_step(**one, state=dirty, reset=reset)
    assert torch.equal(got, want) and torch.equal(clean, dirty)
    window = torch.randn(5, 3, 24, device="cuda").bfloat16()
    clean = torch.where(reset.bool()[:, None, None], torch.zeros_like(window), window)
    dirty = torch.where(reset.bool()[:, None, None], torch.full_like(window, float("inf")), window)
    w = torch.randn(24, 4, device="cuda")
    assert torch.equal(ops.causal_conv_step(one["u"], w, None, dirty, reset=reset), ops.causal_conv_step(one["u"], w, None, clean))
    assert torch.equal(clean, dirty)


def test_no_sequences_and_no_steps(cuda):
    import torch
    from t8b import ops
    for s, t in ((0, 5), (3, 0), (0, 0)):
        x, normal = scan_inputs(s, t, 24, 16)
        state, window = torch.randn(s, 24, 16, device="cuda"), torch.randn(s, 3, 24, device="cuda")
        z, d = normal(s, t, 24), torch.ones(24, device="cuda")
        dfinal = torch.randn(s, 24, 16, device="cuda")
        y, final, saved = ops.selective_scan(**x, z=z, d=d, delta_bias=d, state=state, final=True, save=True)
        assert y.shape == (s, t, 24) and torch.equal(final, state)
        grads = ops.selective_scan_backward(normal(s, t, 24), **x, saved=saved, z=z, d=d, delta_bias=d, state=state, dfinal=dfinal)
        assert not any(grads[k].any() for k in (2, 5, 7)) and torch.equal(grads[8], dfinal)
        w = torch.randn(24, 4, device="cuda")
        y, final = ops.causal_conv(x["u"], w, d, state=window, final=True)
        assert y.shape == (s, t, 24) and torch.equal(final, window)
        dx, dw, db, dstate = ops.causal_conv_backward(normal(s, t, 24), x["u"], w, d, state=window, dfinal=window)
        assert not dw.any() and not db.any() and torch.equal(dstate, window)
    x, _ = scan_inputs(0, 1, 24, 16)
    one = {k: v if k == "a" else v[:, 0] for k, v in x.items()}
    assert ops.selective_scan_step(**one, state=torch.zeros(0, 24, 16, device="cuda")).shape == (0, 24)
    assert ops.causal_conv_step(one["u"], torch.zeros(24, 2, device="cuda"), None, torch.zeros(0, 1, 24, device="cuda")).shape == (0, 24)
    out = ops.policy_loss(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda").long(), torch.zeros(0, device="cuda"),
                          torch.zeros(0, device="cuda"))
    assert [v.shape for v in out] == [(0,)] * 4 + [(0, 9)]


@pytest.mark.parametrize("n", [40, 2000])
def test_loss_of_rows_at_their_limits(cuda, n):
    """The type's lowest and highest values, -inf and NaN, at legal and at other places, against the definition in 64
    bits: equal where it is finite (bounds of 2^-17 of the largest term), not finite where it is not."""
    import torch
    from t8b import ops
    for T in (torch.float32, torch.bfloat16, torch.float16):
        low, high = torch.finfo(T).min, torch.finfo(T).max
        z = torch.randn(12, n, device="cuda").to(T)
        legal = torch.ones(12, n, dtype=torch.bool, device="cuda")
        actions = torch.arange(12, device="cuda")
        z[0] = low                       # masked by the lowest value everywhere: uniform
        z[1, 5:] = low                   # and but for a few
        z[2] = high
        z[3, 7:] = -float("inf")
        z[4, 4] = float("nan")           # the action's own logit
        legal[5, 30:] = False
        z[5, 30:] = float("nan")         # what is not legal may be anything
        legal[6, 20:] = False
        z[6, 20:] = float("inf")
        legal[7] = False                 # a row that its mask leaves empty
        legal[8, 8] = False              # an action that is not legal
        actions[9], actions[10] = -1, n
        z[11, 11] = -float("inf")        # an action of probability 0
        old, advantages = torch.full((12,), -3.0, device="cuda"), torch.randn(12, device="cuda")
        want = m.loss64(z, actions, old, advantages, legal, entropy=0.1, weights=torch.ones(12, device="cuda"))
        loss, lp, h, k, grad = ops.policy_loss(z, actions, old, advantages, mask=legal, entropy=0.1, weights=torch.ones(12, device="cuda"))
        for row in (0, 1, 2, 3, 5, 6, 7, 8, 9, 10, 11):
            for got, w in ((loss, want["loss"]), (lp, want["log_probabilities"]), (h, want["entropies"])):
                if torch.isfinite(w[row]):
                    assert abs(float(got[row]) - float(w[row])) <= 2 ** -17 * (10 + abs(float(w[row]))), (row, T)
                else:
                    assert float(got[row]) == float(w[row])
            unit = torch.finfo(T).eps
            assert torch.allclose(grad[row].double(), want["dlogits"][row], rtol=unit, atol=2 ** -17 * float(want["dlogits"][row].abs().max()) + 1e-7), (row, T)
        assert loss[4].isnan() and lp[4].isnan()
        assert not torch.stack([v[7:11] for v in (loss, lp, h, k)]).any() and not grad[7:11].any()


def test_loss_with_an_impossible_reference(cuda):
    """The divergence is infinite where the reference gives 0 to a legal action of the policy, finite where neither
    gives any."""
    import torch
    from t8b import ops
    for n in (40, 2000):
        z, q = torch.randn(2, 3, n, device="cuda").unbind(0)
        q[0, 6] = -float("inf")
        z[1, 6] = q[1, 6] = -float("inf")
        q[2, 6] = float("nan")
        legal = torch.ones(3, n, dtype=torch.bool, device="cuda")
        legal[2, 6] = False
        args = (z, torch.zeros(3, device="cuda").long(), torch.full((3,), -3.0, device="cuda"), torch.ones(3, device="cuda"))
        k, grad = ops.policy_loss(*args, mask=legal, reference=q, kl=0.5)[3:]
        want = m.loss64(*args, legal, reference=q, kl=0.5)
        assert float(k[0]) == float("inf")
        assert torch.allclose(k[1:].double(), want["divergences"][1:], rtol=1e-4, atol=1e-6)
        assert torch.allclose(grad[1:].double(), want["dlogits"][1:], rtol=1e-4, atol=1e-7)


def test_offsets_beyond_32_bits(cuda):
    """Rows that lie more than 2^31 elements apart, of every operand."""
    import torch
    from t8b import ops
    wide = torch.zeros((1 << 31) + (1 << 22), device="cuda", dtype=torch.bfloat16)
    far = 1 << 30
    g = torch.Generator(device="cuda").manual_seed(3)

    def spread(shape, strides, offset):
        view = wide.as_strided(shape, strides, offset)
        view.copy_(torch.randn(shape, device="cuda", generator=g))
        return view

    s, t, n, states = 2, 3, 24, 16
    tracks = [spread((s, t, n), (far // 2, far // 2 + 4096, 1), 64 * i) for i in range(4)]  # u, delta, z, dy
    b, c = (spread((s, t, 1, states), (far // 2, far // 2 + 4096, states, 1), 512 + 64 * i) for i in range(2))
    assert (s - 1) * (far // 2) + (t - 1) * (far // 2 + 4096) > (1 << 30)
    a = -torch.exp(torch.randn(n, states, device="cuda", generator=g))
    near = lambda v: v.contiguous().clone()  # noqa: E731

    def scan(u, delta, z, dy, b, c):
        y, final, saved = ops.selective_scan(u, delta, a, b, c, z=z, final=True, save=True)
        return (y, final) + ops.selective_scan_backward(dy, u, delta, a, b, c, saved, z=z)

    same(scan(*tracks, b, c), scan(*map(near, tracks), near(b), near(c)))
    w = torch.randn(n, 4, device="cuda", generator=g)
    x, dy = tracks[0], tracks[3]
    assert torch.equal(ops.causal_conv(x, w, activation="silu"), ops.causal_conv(near(x), w, activation="silu"))
    same(ops.causal_conv_backward(dy, x, w), ops.causal_conv_backward(near(dy), near(x), w))
    for n in (368, 2000):
        z = spread((3, n), (far, 1), 1 << 20)
        rows = (torch.tensor([1, 2, 3], device="cuda"), torch.full((3,), -5.0, device="cuda"), torch.ones(3, device="cuda"))
        same(ops.policy_loss(z, *rows, entropy=0.1), ops.policy_loss(near(z), *rows, entropy=0.1))


def test_streams_and_graphs(cuda):
    """On another stream, and captured twice into graphs that run in turn on new inputs: the same outputs."""
    import torch
    from t8b import ops
    s, t, n, states = 2, 300, 40, 16
    x, normal = scan_inputs(s, t, n, states, dtype=torch.bfloat16)
    z, dy = normal(s, t, n), normal(s, t, n)
    w = torch.randn(n, 4, device="cuda")
    logits, actions, old, advantages = (torch.randn(50, 368, device="cuda"), torch.randint(368, (50,), device="cuda"),
                                        torch.full((50,), -6.0, device="cuda"), torch.randn(50, device="cuda"))
    state, window = torch.zeros(s, n, states, device="cuda"), torch.zeros(s, 3, n, device="cuda").bfloat16()
    one = {k: v if k == "a" else v[:, 0] for k, v in x.items()}

    def everything(stream=None):
        u = ops.causal_conv(x["u"], w, activation="silu", stream=stream)
        y, saved = ops.selective_scan(**dict(x, u=u), z=z, save=True, stream=stream)
        out = [u, y, *ops.selective_scan_backward(dy, **dict(x, u=u), saved=saved, z=z, stream=stream)]
        out += ops.causal_conv_backward(dy, x["u"], w, activation="silu", stream=stream)
        out += ops.policy_loss(logits, actions, old, advantages, entropy=0.1, stream=stream)
        out += [ops.causal_conv_step(one["u"], w, None, window, stream=stream), ops.selective_scan_step(**one, state=state, stream=stream)]
        return [v for v in out if v is not None]

    def fresh():
        state.zero_()
        window.zero_()

    want = everything()
    fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = everything(side)
    side.synchronize()
    same(got, want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = everything()
        graphs.append((graph, outputs))
    for seed in (5, 6):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for v in (x["u"], x["delta"], dy, logits):
            v.copy_(torch.randn(v.shape, device="cuda", generator=g))
        fresh()
        want = everything()
        for graph, outputs in graphs:
            fresh()
            graph.replay()
            torch.cuda.synchronize()
            same(outputs, want)
    with pytest.raises(ValueError, match="stream"):
        ops.causal_conv(torch.zeros(2, 3, 8), w, stream=side)


def test_two_calls_at_once(cuda):
    """Calls on two streams share nothing: each gives what it gives alone."""
    import torch
    sides = [torch.cuda.Stream() for _ in range(2)]
    problems = [scan_inputs(4, 500, 64, 16, seed=k) for k in range(2)]
    dys = [normal(4, 500, 64) for _, normal in problems]
    want = [run_scan(x, dy) for (x, _), dy in zip(problems, dys)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for side, (x, _), dy in zip(sides, problems, dys):
            with torch.cuda.stream(side):
                got.append(run_scan(x, dy))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            same(g, w)


def test_a_broadcast_input_is_read_as_its_copies(cuda):
    import torch
    from t8b import ops
    x, normal = scan_inputs(3, 20, 32, 16)
    shared = {k: v if k == "a" else v[:1].expand_as(v) for k, v in x.items()}
    copies = {k: v.contiguous() for k, v in shared.items()}
    dy = normal(3, 20, 32)
    same(run_scan(shared, dy), run_scan(copies, dy))
    w = torch.randn(32, 3, device="cuda")
    assert torch.equal(ops.causal_conv(shared["u"], w), ops.causal_conv(copies["u"], w))


def test_wrong_arguments_raise_before_anything_is_queued(cuda):
    import torch
    from t8b import ops, profile
    x, normal = scan_inputs(3, 8, 24, 16)
    u, delta, a, b, c = (x[k] for k in ("u", "delta", "a", "b", "c"))
    w, z = torch.randn(24, 4, device="cuda"), normal(3, 8, 24)
    state, window = torch.zeros(3, 24, 16, device="cuda"), torch.zeros(3, 3, 24, device="cuda")
    reset = torch.zeros(3, 8, dtype=torch.bool, device="cuda")
    saved = torch.zeros(3 * 16 * 24, device="cuda")
    rows, actions = torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda").long()
    logits = torch.zeros(6, 40, device="cuda")
    before = profile.launch_count()
    bad = [
        lambda: ops.causal_conv(u[0], w), lambda: ops.causal_conv(u, w[:23]), lambda: ops.causal_conv(u, torch.zeros(24, 5, device="cuda")),
        lambda: ops.causal_conv(u, w[:, :1].contiguous()), lambda: ops.causal_conv(u, w.bfloat16()), lambda: ops.causal_conv(u, w.t().contiguous().t()),
        lambda: ops.causal_conv(u.double(), w), lambda: ops.causal_conv(u[..., ::2], w[:12]), lambda: ops.causal_conv(u, w, w[0]),
        lambda: ops.causal_conv(u, w, state=window[:, :2]), lambda: ops.causal_conv(u, w, state=window.half()),
        lambda: ops.causal_conv(u, w, reset=reset[:, :7]), lambda: ops.causal_conv(u, w, reset=reset.float()),
        lambda: ops.causal_conv(u, w, lengths=torch.zeros(3, device="cuda").long()), lambda: ops.causal_conv(u, w, lengths=torch.zeros(2, device="cuda").int()),
        lambda: ops.causal_conv(u, w, activation="softmax"), lambda: ops.causal_conv(u, w.cpu()), lambda: ops.causal_conv(u, w, reset=reset.cpu()),
        lambda: ops.causal_conv_backward(u[:, :7], u, w), lambda: ops.causal_conv_backward(u.half(), u, w),
        lambda: ops.causal_conv_backward(u, u, w, dfinal=window[:2]), lambda: ops.causal_conv_step(u, w, None, window),
        lambda: ops.causal_conv_step(u[:, 0], w, None, window.transpose(0, 1)), lambda: ops.causal_conv_step(u[:, 0], w, None, window[:, :, :23]),
        lambda: ops.causal_conv_step(u[:, 0], w, None, window, reset=reset),
        lambda: ops.selective_scan(u, delta[:, :7], a, b, c), lambda: ops.selective_scan(u, delta.half(), a, b, c),
        lambda: ops.selective_scan(u, delta, a.half(), b, c), lambda: ops.selective_scan(u, delta, a[:23], b, c),
        lambda: ops.selective_scan(u, delta, torch.zeros(24, 65, device="cuda"), b, c), lambda: ops.selective_scan(u, delta, a, b[..., :15], c),
        lambda: ops.selective_scan(u, delta, a, b, c[:, :, 0]), lambda: ops.selective_scan(u, delta, a, b.expand(3, 8, 5, 16), c.expand(3, 8, 5, 16)),
        lambda: ops.selective_scan(u, delta, a, b, c, d=rows), lambda: ops.selective_scan(u, delta, a, b, c, z=z[:2]),
        lambda: ops.selective_scan(u, delta, a, b, c, delta_bias=a[:, 0]), lambda: ops.selective_scan(u, delta, a, b, c, state=state.half()),
        lambda: ops.selective_scan(u, delta, a, b, c, state=state[:, :, :15]), lambda: ops.selective_scan(u.cpu(), delta, a, b, c),
        lambda: ops.selective_scan_backward(z, u, delta, a, b, c, saved[:-1]), lambda: ops.selective_scan_backward(z, u, delta, a, b, c, None),
        lambda: ops.selective_scan_backward(z[:, :7], u, delta, a, b, c, saved), lambda: ops.selective_scan_backward(z, u, delta, a, b, c, saved.half()),
        lambda: ops.selective_scan_step(u[:, 0], delta[:, 0], a, b[:, 0], c[:, 0], state[:2]),
        lambda: ops.selective_scan_step(u[:, 0], delta[:, 0], a, b[:, 0], c[:, 0], None),
        lambda: ops.policy_loss(logits, actions.int(), rows, rows), lambda: ops.policy_loss(logits, actions[:5], rows, rows),
        lambda: ops.policy_loss(logits, actions, rows.half(), rows), lambda: ops.policy_loss(logits, actions, rows, rows[:5]),
        lambda: ops.policy_loss(logits.double(), actions, rows, rows), lambda: ops.policy_loss(logits, actions, rows, rows, mask=logits),
        lambda: ops.policy_loss(logits, actions, rows, rows, mask=torch.zeros(6, 1, device="cuda").int()),
        lambda: ops.policy_loss(logits, actions, rows, rows, mask=torch.zeros(5, 40, device="cuda").bool()),
        lambda: ops.policy_loss(logits, actions, rows, rows, reference=logits.half()), lambda: ops.policy_loss(logits, actions, rows, rows, reference=logits[:, :39]),
        lambda: ops.policy_loss(logits, actions, rows, rows, reference=rows.half()), lambda: ops.policy_loss(logits, actions, rows, rows, weights=rows[:5]),
        lambda: ops.policy_loss(logits, actions, rows, rows, clip=-0.1), lambda: ops.policy_loss(logits, actions, rows, rows, kl=float("nan")),
        lambda: ops.policy_loss(logits[:1].expand(6, 40), actions, rows, rows),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted", k)
    with pytest.raises(TypeError):
        ops.policy_loss(logits, actions, rows, rows, clip="0.2")

    class Neither:
        def __bool__(self):
            raise KeyError("neither")

    with pytest.raises(KeyError, match="neither"):
        ops.selective_scan(u, delta, a, b, c, save=Neither())
    assert profile.launch_count() == before
