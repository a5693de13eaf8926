"""A reset's step takes nothing over, however large its own decay is: exp(size a) beyond fp32 times a state that is 0
gives 0, in sequences (whole and ragged tiles, cut into chunks or not), in single steps and in the gradients."""
import pytest

import memory64 as m
from test_memory_gpu import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("s,t,states,channels", [(3, 16, 16, 32), (2, 13, 5, 7), (2, 600, 16, 24), (1, 700, 40, 8)])
@pytest.mark.parametrize("type_name", ["float32", "bfloat16"])
def test_a_growing_step_at_a_reset(cuda, s, t, states, channels, type_name):
    """Sizes of -40 under rates of -3 (e^120) at the resets alone. At a reset y = c b size u exactly as without a state:
    four roundings and the sum over the states; elsewhere the bounds of test_memory_gpu.py for sizes up to 1."""
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    g = torch.Generator(device="cuda").manual_seed(t + states)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    u, b, c, dy = (v.to(T) for v in (normal(s, t, channels), normal(s, t, 1, states), normal(s, t, 1, states), normal(s, t, channels)))
    delta = (torch.rand(s, t, channels, device="cuda", generator=g) * 0.3).to(T)
    a = -(2.9 + 0.2 * torch.rand(channels, states, device="cuda", generator=g))
    state = normal(s, channels, states)
    reset = torch.zeros(s, t, dtype=torch.bool, device="cuda")
    for at in (0, 3, 8, 12, t // 2, t - 1):
        reset[:, at] = True
    delta[reset] = -40
    size = delta.double()
    # a reset's decay meets nothing: its value does not matter to the definition, as long as it is finite
    out, states64, befores, final, decays = m.scan64(size, u, a, b, c, None, state, reset)
    sizes = m.scan64(size.abs(), u.abs(), a, b.abs(), c.abs(), None, state.abs(), reset, None, decays)
    off = 2 ** -20 * ((t + 8) * (2 + 0.3 * 3.1) + 1)
    y, end, saved = ops.selective_scan(u, delta, a, b, c, softplus=False, state=state, reset=reset, final=True, save=True)
    close(y, out, off * sizes[0], "y")
    close(end, final, off * sizes[3], "final")
    got = ops.selective_scan_backward(dy, u, delta, a, b, c, saved, softplus=False, state=state, reset=reset)
    want, size_of = ([*m.scan_grad64(f(dy.double()), f(size), f(u.double()), f(a.double()), f(b.double()), f(c.double()), None, v[1], v[2],
                                     decays, reset)] for f, v in ((lambda w: w, (out, states64, befores)), (torch.abs, sizes)))
    for name, k, q in (("du", 0, 0), ("ddelta", 1, 1), ("da", 2, 2), ("db", 3, 3), ("dc", 4, 4), ("dstate", 8, 6)):
        close(got[k], want[q], (2 * off + max(s * t, channels) * 2 ** -24) * size_of[q], name)
    held = state.clone()
    for at in range(min(t, 20)):
        one = ops.selective_scan_step(u[:, at], delta[:, at], a, b[:, at], c[:, at], held, softplus=False, reset=reset[:, at])
        close(one, out[:, at], off * sizes[0][:, at], f"step {at}")


def test_a_rate_of_minus_infinity_forgets_at_once(cuda):
    """a = -inf (exp of a large logarithm): every step starts from 0, at resets and elsewhere."""
    import torch
    from t8b import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    s, t, n, states = 2, 21, 16, 16
    u, b, c = (torch.randn(s, t, w, device="cuda", generator=g) for w in (n, states, states))
    delta = torch.rand(s, t, n, device="cuda", generator=g) + 0.1
    reset = torch.rand(s, t, device="cuda", generator=g) < 0.3
    a = torch.full((n, states), -float("inf"), device="cuda")
    y = ops.selective_scan(u, delta, a, b, c, softplus=False, reset=reset)
    want = delta.double() * u.double() * (b.double() * c.double()).sum(2, keepdim=True)
    size = (delta * u).double().abs() * (b.double() * c.double()).abs().sum(2, keepdim=True)
    close(y, want, (states + 3) * 2 ** -23 * size, "y")
