"""A pre-norm residual torso over the operators of t8b.ops, and a command that fits one to returns.

    x = linear(layer_norm(observation))
    x = x + linear(gated(layer_norm(x)))        for each block
    outputs = linear(layer_norm(x))             in fp32

`python -m t8b.torso` (with tekken8-agent_b200 on the path) plays one self-play iteration, takes its
rollout's observations and returns, and fits the torso's single output to the returns.
"""
from __future__ import annotations

import argparse
import time
from pathlib import Path

import torch

from . import ops


class ResidualTorso:
    """Parameters are fp32 (`parameters`, a dict of tensors that an optimizer steps); the matrix
    products read bf16 copies that `refresh` makes after a step."""

    def __init__(self, observation_size: int, outputs: int, hidden: int = 512, features: int = 1408, blocks: int = 2,
                 activation: str = "silu", seed: int = 1, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.blocks, self.activation = blocks, activation
        self.parameters: dict[str, torch.Tensor] = {}
        self._weights: dict[str, torch.Tensor] = {}

        def norm(name, n):
            self.parameters[name + ".weight"] = torch.ones(n, device=device)
            self.parameters[name + ".bias"] = torch.zeros(n, device=device)

        def matrix(name, out, n, gain=1.0, bias=True):
            self.parameters[name] = gain * n ** -0.5 * torch.randn(out, n, device=device, generator=g)
            if bias:
                self.parameters[name + ".bias"] = torch.zeros(out, device=device)

        norm("observation", observation_size)
        matrix("input", hidden, observation_size)
        for i in range(blocks):
            norm(f"{i}.norm", hidden)
            matrix(f"{i}.gated", 2 * features, hidden, bias=False)
            matrix(f"{i}.out", hidden, features, (2 * blocks) ** -0.5, bias=False)
        norm("final", hidden)
        matrix("head", outputs, hidden, 0.1)
        self.refresh()

    def refresh(self):
        """bf16 copies of the matrices, for the products."""
        for name, p in self.parameters.items():
            if p.dim() == 2:
                if name not in self._weights:
                    self._weights[name] = torch.empty_like(p, dtype=torch.bfloat16)
                self._weights[name].copy_(p)

    def _norm(self, name, x, kept):
        p = self.parameters
        y, mean, rstd = ops.layer_norm(x, p[name + ".weight"], p[name + ".bias"], out_dtype=torch.bfloat16, save=True)
        kept[name] = (x, mean, rstd)
        return y

    def forward(self, observations: torch.Tensor):
        """The fp32 outputs of fp32 observations, and what `backward` needs."""
        p, w, kept = self.parameters, self._weights, {}
        n = self._norm("observation", observations, kept)
        x = ops.linear(n, w["input"], p["input.bias"])
        kept["input"] = n
        for i in range(self.blocks):
            n = self._norm(f"{i}.norm", x, kept)
            h, pre = ops.gated(n, w[f"{i}.gated"], activation=self.activation, save=True)
            kept[f"{i}.gated"], kept[f"{i}.out"] = (n, pre), h
            x = ops.linear(h, w[f"{i}.out"], residual=x)
        n = self._norm("final", x, kept)
        kept["head"] = n
        return ops.linear(n, w["head"], p["head.bias"], out_dtype=torch.float32), kept

    def backward(self, gradient: torch.Tensor, kept: dict) -> dict[str, torch.Tensor]:
        """The parameters' gradients from the outputs' (fp32)."""
        p, w, grads = self.parameters, self._weights, {}

        def linear(name, dy, x, bias):
            dx, grads[name], db = ops.linear_backward(dy, x, w[name], p[name + ".bias"] if bias else None)
            if bias:
                grads[name + ".bias"] = db
            return dx

        def norm(name, dy, residual=None):
            x, mean, rstd = kept[name]
            dx, grads[name + ".weight"], grads[name + ".bias"] = ops.layer_norm_backward(
                dy, x, p[name + ".weight"], p[name + ".bias"], mean, rstd, residual_gradient=residual)
            return dx

        dx = norm("final", linear("head", gradient.to(torch.bfloat16), kept["head"], True))
        for i in reversed(range(self.blocks)):
            dh = linear(f"{i}.out", dx, kept[f"{i}.out"], False)
            n, pre = kept[f"{i}.gated"]
            dn, grads[f"{i}.gated"], _ = ops.gated_backward(dh, n, w[f"{i}.gated"], None, pre,
                                                            activation=self.activation)
            dx = norm(f"{i}.norm", dn, residual=dx)
        norm("observation", linear("input", dx, kept["input"], True))
        return grads


def fit(torso: ResidualTorso, observations: torch.Tensor, targets: torch.Tensor, steps: int, batch: int = 65536,
        learning_rate: float = 1e-3, seed: int = 1) -> list[torch.Tensor]:
    """Adam on the mean squared error over random minibatches; the losses, on the device."""
    g = torch.Generator(device=observations.device).manual_seed(seed)
    names = list(torso.parameters)
    optimizer = torch.optim.Adam(list(torso.parameters.values()), lr=learning_rate)
    losses = []
    for _ in range(steps):
        rows = torch.randint(observations.shape[0], (min(batch, observations.shape[0]),), device=observations.device,
                             generator=g)
        y, kept = torso.forward(observations[rows])
        off = y - targets[rows]
        losses.append(off.square().mean())
        grads = torso.backward(off * (2.0 / off.numel()), kept)
        for name in names:
            torso.parameters[name].grad = grads[name].to(torch.float32)
        optimizer.step()
        torso.refresh()
    ops.status(device=observations.device)
    return losses


def main(arguments=None) -> float:
    from . import roster as roster_module
    from .train import SelfPlayTrainer
    root = Path(__file__).resolve().parent.parent.parent
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--roster", default=str(root / "tests" / "golden" / "roster41.bin.xz"))
    parser.add_argument("--environments", type=int, default=8192)
    parser.add_argument("--horizon", type=int, default=32)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--blocks", type=int, default=2)
    parser.add_argument("--hidden", type=int, default=512)
    parser.add_argument("--features", type=int, default=1408)
    a = parser.parse_args(arguments)
    trainer = SelfPlayTrainer(roster_module.load(a.roster), a.environments, a.horizon, epochs=1, minibatches=4)
    trainer.iterate()
    observations = trainer.rollout.tensor("observations").flatten(0, 1)
    returns = trainer.rollout.tensor("returns").reshape(-1, 1)
    targets = (returns - returns.mean()) / returns.std().clamp(min=1e-6)
    torso = ResidualTorso(observations.shape[1], 1, a.hidden, a.features, a.blocks)
    losses = fit(torso, observations, targets, 1)  # the first step's one-time costs stay out of the time
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = torch.stack(losses + fit(torso, observations, targets, a.steps, seed=2))
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    last = float(losses[-max(1, a.steps // 10):].mean())
    print(f"samples {observations.shape[0]}  steps {a.steps}  {1e3 * seconds / a.steps:.2f} ms a step  "
          f"loss {float(losses[0]):.4f} -> {last:.4f}")
    return last


if __name__ == "__main__":
    main()
