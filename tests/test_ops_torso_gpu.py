"""The residual torso's forward and backward against the same network in 64 bits with the roundings that
the operators make between one another, so that what is left is small."""
import pytest

pytestmark = pytest.mark.gpu


def network(torso, p, x):
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

    x = stored(norm("observation", x) @ p["input"].T + p["input.bias"])
    for i in range(torso.blocks):
        gate, up = stored(norm(f"{i}.norm", x) @ p[f"{i}.gated"].T).chunk(2, -1)
        x = stored(x + stored(gate * torch.sigmoid(gate) * up) @ p[f"{i}.out"].T)
    return norm("final", x) @ p["head"].T + p["head.bias"]


@pytest.mark.parametrize("rows,outputs,hidden,features,blocks", [(700, 33, 128, 200, 2), (5, 1, 64, 96, 1), (4099, 33, 512, 1408, 2)])
def test_torso_against_the_network_with_its_roundings(cuda, rows, outputs, hidden, features, blocks):
    """What the reference does not round: h from gate and up before they are stored, and dz (twice a block and
    once in the head's place of it), each an independent relative error below 2^-9, 2^-9 / sqrt 3 in the mean;
    values near a tie round the other way. At most 12 such errors lie behind a gradient: 12^0.5 2^-9 / 3^0.5 =
    0.4 % of its norm, held to 1 %, which a gradient that is 5 % off does not meet."""
    import torch
    from t8b.torso import ResidualTorso
    g = torch.Generator(device="cuda").manual_seed(rows)
    torso = ResidualTorso(151, outputs, hidden, features, blocks, seed=3)
    for name, p in torso.parameters.items():  # biases and norms away from their initial 0 and 1
        if p.dim() == 1:
            p += 0.1 * torch.randn(p.shape, device="cuda", generator=g)
    x = torch.rand(rows, 151, device="cuda", generator=g)
    d = (torch.randn(rows, outputs, device="cuda", generator=g) / rows).bfloat16()
    y, kept = torso.forward(x)
    grads = torso.backward(d.float(), kept)
    p = {k: (torso._weights[k] if k in torso._weights else v).detach().double().requires_grad_()
         for k, v in torso.parameters.items()}
    want = network(torso, p, x.double())
    want.backward(d.double())
    want = want.detach()
    assert float((y.double() - want).norm() / want.norm()) < 0.01
    assert set(grads) == set(p)
    for name, v in grads.items():
        norm = float(p[name].grad.norm())
        off = [float((scale * v.double() - p[name].grad).norm()) / norm for scale in (1.0, 1.05, -1.0)]
        assert off[0] < 0.01 < off[1] and off[2] > 1, (name, off)
    from t8b import ops
    ops.status()
