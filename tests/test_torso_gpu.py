"""The residual torso (t8b.torso): its gradients against automatic differentiation of the same
network in 64 bits, and the command that fits one to a rollout's returns."""
import pytest

pytestmark = pytest.mark.gpu


def network64(torso, p, x):
    import torch

    def norm(name, v):
        c = v - v.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * p[name + ".weight"] + p[name + ".bias"]

    x = norm("observation", x) @ p["input"].T + p["input.bias"]
    for i in range(torso.blocks):
        gate, up = (norm(f"{i}.norm", x) @ p[f"{i}.gated"].T).chunk(2, -1)
        x = x + (gate * torch.sigmoid(gate) * up) @ p[f"{i}.out"].T
    return norm("final", x) @ p["head"].T + p["head.bias"]


def test_torso_gradients_match_automatic_differentiation(cuda):
    """Every activation and gradient between operators is rounded to bf16 (2^-8 each): outputs
    within 3 % of their norm, gradients within 5 % of theirs."""
    import torch
    from t8b.torso import ResidualTorso
    torch.manual_seed(0)
    torso = ResidualTorso(151, 33, hidden=128, features=200, blocks=2, seed=3)
    x = torch.rand(700, 151, device="cuda")
    d = torch.randn(700, 33, device="cuda") / 700
    y, kept = torso.forward(x)
    grads = torso.backward(d, kept)
    p = {k: (torso._weights[k] if k in torso._weights else v).double().requires_grad_() for k, v in torso.parameters.items()}
    want = network64(torso, p, x.double())
    want.backward(d.double())
    want = want.detach()
    assert float((y.double() - want).norm() / want.norm()) < 0.03
    assert set(grads) == set(p)
    for name, g in grads.items():
        assert g.shape == p[name].shape
        off = float((g.double() - p[name].grad).norm() / p[name].grad.norm())
        assert off < 0.05, (name, off)


def test_fit_lowers_the_loss(cuda):
    import torch
    from t8b.torso import ResidualTorso, fit
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(4096, 40, device="cuda", generator=g)
    target = torch.sin(4 * x[:, :1]) * x[:, 1:2] + x[:, 2:3]
    target = (target - target.mean()) / target.std()
    torso = ResidualTorso(40, 1, hidden=64, features=96, blocks=2)
    losses = fit(torso, x, target, 150, batch=1024)
    assert float(losses[0]) > 0.5 and float(torch.stack(losses[-10:]).mean()) < 0.1


def test_command_fits_a_rollouts_returns(cuda, capsys):
    from t8b import torso
    last = torso.main(["--environments", "256", "--horizon", "16", "--steps", "60", "--blocks", "1", "--hidden", "128",
                       "--features", "192"])
    assert "ms a step" in capsys.readouterr().out
    assert last < 0.95
