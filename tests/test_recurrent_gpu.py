"""The policy with memory (t8b.recurrent): a rollout against the same decisions one at a time, its gradients
against the network in 64 bits with the roundings that the operators make between one another, and the
command that fits one to a rollout."""
import pytest

import memory64 as m

pytestmark = pytest.mark.gpu


def network(policy, p, x, reset):
    """Each operator's output is rounded to bf16 on the way forward, and its gradient on the way back."""
    import torch

    class Stored(torch.autograd.Function):
        @staticmethod
        def forward(_, v):
            return v.to(torch.bfloat16).double()

        @staticmethod
        def backward(_, d):
            return d.to(torch.bfloat16).double()

    stored = Stored.apply

    def norm(name, v):
        c = v - v.mean(-1, keepdim=True)
        return stored(c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * p[name + ".weight"] + p[name + ".bias"])

    rounds = None if reset is None else reset.t()
    x = stored(norm("observation", x) @ p["input"].T + p["input.bias"])
    for i in range(policy.blocks):
        v, z = stored(norm(f"{i}.norm", x) @ p[f"{i}.in"].T).chunk(2, -1)
        pre, _ = m.conv64(v.transpose(0, 1), p[f"{i}.taps"], p[f"{i}.taps.bias"], None, rounds)
        u = stored(pre * torch.sigmoid(pre))
        mixed = stored(u @ p[f"{i}.mix"].T)
        size = stored(mixed[..., :policy.rank] @ p[f"{i}.size"].T)
        b, c = mixed[..., policy.rank:].split(policy.states, -1)
        size = torch.nn.functional.softplus(size + p[f"{i}.size.bias"], threshold=50.0)
        y, _, _, _, _ = m.scan64(size, u, -torch.exp(p[f"{i}.rate"]), b[:, :, None], c[:, :, None], p[f"{i}.skip"], None, rounds)
        z = z.transpose(0, 1)
        y = stored(y * z * torch.sigmoid(z)).transpose(0, 1)
        x = stored(x + y @ p[f"{i}.out"].T)
    out = norm("final", x) @ p["head"].T + p["head.bias"]
    return out[..., :policy.outputs], out[..., policy.outputs]


def problem(steps, fights, seed, **sizes):
    import torch
    from t8b.recurrent import MemoryPolicy
    g = torch.Generator(device="cuda").manual_seed(seed)
    policy = MemoryPolicy(151, 33, seed=3, **sizes)
    for p in policy.parameters.values():  # biases and norms away from their initial 0 and 1
        if p.dim() == 1:
            p += 0.1 * torch.randn(p.shape, device="cuda", generator=g)
    x = torch.rand(steps, fights, 151, device="cuda", generator=g)
    reset = torch.rand(steps, fights, device="cuda", generator=g) < 0.1
    return g, policy, x, reset


@pytest.mark.parametrize("steps,fights,sizes", [
    (13, 7, dict(hidden=64, inner=96, states=16, rank=8, blocks=2)), (40, 3, dict(hidden=128, inner=200, states=5, rank=16, blocks=1)),
    (9, 33, dict(hidden=512, inner=1024, blocks=1)),
])
def test_gradients_against_the_network_with_its_roundings(cuda, steps, fights, sizes):
    """What the reference does not round: the state's products' order, gs and the sums inside an operator, and dz of
    a product (each an independent relative error below 2^-9, 2^-9 / sqrt 3 in the mean); values near a tie
    round the other way, and a decay passes a sequence's error on to its next steps (a memory of some ten). At
    most 24 such errors lie behind a gradient: 24^0.5 2^-9 / 3^0.5 = 0.55 % of its norm, held to 2 %, which a
    gradient that is 5 % off does not meet."""
    import torch
    g, policy, x, reset = problem(steps, fights, steps, **sizes)
    dlogits = (torch.randn(steps, fights, 33, device="cuda", generator=g) / x[..., 0].numel()).bfloat16().float()
    dvalues = (torch.randn(steps, fights, device="cuda", generator=g) / x[..., 0].numel()).bfloat16().float()
    logits, values, kept = policy.forward(x, reset)
    grads = policy.backward(dlogits, dvalues, kept)
    p = {k: (policy._weights[k] if k in policy._weights else v).detach().double().requires_grad_() for k, v in policy.parameters.items()}
    want, want_values = network(policy, p, x.double(), reset)
    ((want * dlogits.double()).sum() + (want_values * dvalues.double()).sum()).backward()
    for got, w in ((logits, want.detach()), (values, want_values.detach())):
        assert float((got.double() - w).norm() / w.norm()) < 0.02
    assert set(grads) == set(p)
    for name, v in grads.items():
        assert v.shape == p[name].shape
        norm = float(p[name].grad.norm())
        off = [float((scale * v.double() - p[name].grad).norm()) / norm for scale in (1.0, 1.05, -1.0)]
        assert off[0] < 0.02 < off[1] and off[2] > 1, (name, off)
    from t8b import ops
    ops.status()


def test_steps_are_the_rollout(cuda):
    """One decision at a time gives what the whole rollout gives: the operators' sums have another order (a product of
    few rows), so that values near a tie round the other way, 2^-8 of some 20 roundings each."""
    import torch
    g, policy, x, reset = problem(11, 40, 5, hidden=64, inner=96, states=16, rank=8, blocks=2)
    logits, values, _ = policy.forward(x, reset)
    memory = policy.memory(40)
    for t in range(11):
        one, value = policy.step(x[t], memory, reset[t])
        for got, want in ((one, logits[t]), (value, values[t])):
            assert float((got - want).norm() / want.norm()) < 0.02, t


def test_a_round_does_not_reach_the_next(cuda):
    """Observations before a reset, NaN among them, change nothing behind it, nor any gradient's terms there."""
    import torch
    g, policy, x, reset = problem(20, 4, 6, hidden=64, inner=96, rank=8, blocks=2)
    reset[:] = False
    reset[9] = True
    logits, values, _ = policy.forward(x, reset)
    other = x.clone()
    other[:9] = torch.rand(9, 4, 151, device="cuda", generator=g)
    other[3] = float("nan")
    again, values2, _ = policy.forward(other, reset)
    assert torch.equal(logits[9:], again[9:]) and torch.equal(values[9:], values2[9:])
    assert bool(again[3:9].isnan().all())


def test_command_fits_a_rollout(cuda, capsys):
    import math
    from t8b import recurrent
    last = recurrent.main(["--environments", "256", "--horizon", "32", "--steps", "4", "--fights", "64", "--hidden", "128", "--inner", "256"])
    assert "ms a step" in capsys.readouterr().out
    assert all(math.isfinite(v) for v in last)
