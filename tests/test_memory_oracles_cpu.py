"""The 64-bit definitions that the memory operators' tests compare with, against automatic differentiation
and against differences along the gradient."""
import pytest
import torch

import memory64 as m


def cases(seed, s, t):
    g = torch.Generator().manual_seed(seed)
    reset = torch.rand(s, t, generator=g) < 0.2
    lengths = torch.randint(0, t + 1, (s,), generator=g, dtype=torch.int32)
    lengths[0] = t
    return g, [(None, None), (reset, None), (None, lengths), (reset, lengths)]


def against(function, leaves, weigh, grads):
    """`grads` against automatic differentiation of sum(weigh * function()), and against a difference along a
    random direction (central, of step 1e-5: an error of about 1e-9 of the third derivative)."""
    outs = function()
    total = sum((o * w).sum() for o, w in zip(outs, weigh))
    want = torch.autograd.grad(total, leaves, allow_unused=True)
    g = torch.Generator().manual_seed(5)
    moves = [torch.randn(v.shape, generator=g, dtype=torch.float64) for v in leaves]

    def at(step):
        with torch.no_grad():
            for v, d in zip(leaves, moves):
                v += step * d
            value = sum((o * w).sum() for o, w in zip(function(), weigh))
            for v, d in zip(leaves, moves):
                v -= step * d
        return float(value)

    slope = (at(1e-5) - at(-1e-5)) / 2e-5
    along = sum(float((d * v).sum()) for d, v in zip(moves, grads))
    assert slope == pytest.approx(along, rel=1e-6, abs=1e-6)
    for v, w in zip(grads, want):
        w = torch.zeros_like(v) if w is None else w
        assert torch.allclose(v, w, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("steps", [1, 2, 7])
def test_conv(width, steps):
    g, variants = cases(width * 10 + steps, 3, steps)
    for reset, lengths in variants:
        x, w, b, state = (torch.randn(*v, generator=g, dtype=torch.float64).requires_grad_()
                          for v in ((3, steps, 5), (5, width), (5,), (3, width - 1, 5)))
        dy, dfinal = torch.randn(3, steps, 5, generator=g).double(), torch.randn(3, width - 1, 5, generator=g).double()

        def run():
            p, final = m.conv64(x, w, b, state, reset, lengths)
            live = m.live_of(lengths, 3, steps, x.device)[:, :, None]
            return torch.where(live, m.act64(p, "silu")[0], torch.zeros_like(p)), final

        with torch.no_grad():
            p, _ = m.conv64(x, w, b, state, reset, lengths)
            grads = m.conv_grad64(dy * m.act64(p, "silu")[1], x, w, state, reset, lengths, dfinal)
        against(run, (x, w, b, state), (dy, dfinal), grads)


@pytest.mark.parametrize("steps,groups", [(1, 1), (6, 1), (9, 2)])
def test_scan(steps, groups):
    g, variants = cases(steps + groups, 3, steps)
    for reset, lengths in variants:
        size, u, a, b, c, d, state = (torch.randn(*v, generator=g, dtype=torch.float64)
                                      for v in ((3, steps, 6), (3, steps, 6), (6, 4), (3, steps, groups, 4), (3, steps, groups, 4),
                                                (6,), (3, 6, 4)))
        size, a = size.abs() * 0.3, -a.abs()
        leaves = [v.requires_grad_() for v in (u, size, a, b, c, d, state)]
        gs, dfinal = torch.randn(3, steps, 6, generator=g).double(), torch.randn(3, 6, 4, generator=g).double()

        def run():
            y, _, _, final, _ = m.scan64(size, u, a, b, c, d, state, reset, lengths)
            return y, final

        with torch.no_grad():
            _, states, befores, _, decays = m.scan64(size, u, a, b, c, d, state, reset, lengths)
            grads = m.scan_grad64(gs, size, u, a, b, c, d, states, befores, decays, reset, lengths, dfinal)
        against(run, leaves, (gs, dfinal), grads)


@pytest.mark.parametrize("kind", ["none", "logits", "sampled"])
@pytest.mark.parametrize("masked", [False, True])
def test_loss(kind, masked):
    g = torch.Generator().manual_seed(7)
    z = torch.randn(40, 9, generator=g, dtype=torch.float64).requires_grad_()
    actions = torch.randint(9, (40,), generator=g)
    legal = torch.rand(40, 9, generator=g) < 0.6
    legal[torch.arange(40), actions] = True
    legal[3] = False  # a row without legal actions
    actions[5], actions[6] = -1, 9
    legal = legal if masked else None
    old, advantages = torch.randn(40, generator=g) * 0.2 - 2, torch.randn(40, generator=g)
    more = dict(reference=torch.randn(40, 9, generator=g) if kind == "logits" else None,
                sampled=old + 0.1 * torch.randn(40, generator=g) if kind == "sampled" else None,
                weights=torch.rand(40, generator=g), low=0.2, high=0.3, kl=0.1, entropy=0.02)
    weights = more["weights"].double()

    def run():
        return m.loss64(z, actions, old, advantages, legal, **more)["loss"],

    # a row of -inf has no derivative that automatic differentiation finds: differences alone decide there
    with torch.no_grad():
        grad = m.loss64(z, actions, old, advantages, legal, **more)["dlogits"]
        base = z.clone()
        for row, column in [(r, c) for r in range(0, 40, 3) for c in range(9)]:
            values = []
            for step in (1e-5, -1e-5):
                z.copy_(base)
                z[row, column] += step
                values.append(float((run()[0] * weights).sum()))
            z.copy_(base)
            assert (values[0] - values[1]) / 2e-5 == pytest.approx(float(grad[row, column]), rel=1e-5, abs=1e-8)
    assert not grad[5].any() and not grad[6].any()
    if masked:
        assert not grad[3].any() and not grad[~legal].any()
