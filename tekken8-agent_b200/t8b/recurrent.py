"""A policy with memory over the operators of t8b.ops, and a command that fits one to a rollout.

    x = linear(layer_norm(observation))
    for each block:
        v, z = linear(layer_norm(x))
        u = silu(causal_conv(v))
        size, b, c = linear(u), the sizes through a second, narrower linear map
        x = x + linear(selective_scan(u, size, a, b, c, d, z))
    logits, value = linear(layer_norm(x))       in fp32

Rounds end inside a rollout: `reset` marks the decisions at which a new one begins, and nothing before it
reaches what comes after. `forward` takes whole rollouts, [step][fight] as the rollout buffer holds them;
`step` takes one decision of every fight and moves its memory on.

`python -m t8b.recurrent` (with tekken8-agent_b200 on the path) plays one self-play iteration and fits the
policy to it: the clipped policy loss over the recorded decisions, held near the policy that played.
"""
from __future__ import annotations

import argparse
import math
import time
from pathlib import Path

import torch

from . import ops


class MemoryPolicy:
    """Parameters are fp32 (`parameters`, a dict of tensors that an optimizer steps); the matrix products
    read bf16 copies that `refresh` makes after a step. `outputs` counts the actions; the value comes beside
    them. `inner` and `rank` are 8's multiples."""

    def __init__(self, observation_size: int, outputs: int, hidden: int = 512, inner: int = 1024, states: int = 16,
                 rank: int = 32, width: int = 4, blocks: int = 1, seed: int = 1, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.blocks, self.inner, self.states, self.rank, self.width = blocks, inner, states, rank, width
        self.outputs = outputs
        self.parameters: dict[str, torch.Tensor] = {}
        self._weights: dict[str, torch.Tensor] = {}

        def normal(*shape, scale=1.0):
            return scale * torch.randn(*shape, device=device, generator=g)

        def norm(name, n):
            self.parameters[name + ".weight"] = torch.ones(n, device=device)
            self.parameters[name + ".bias"] = torch.zeros(n, device=device)

        def matrix(name, out, n, gain=1.0):
            self.parameters[name] = normal(out, n, scale=gain * n ** -0.5)

        norm("observation", observation_size)
        matrix("input", hidden, observation_size)
        self.parameters["input.bias"] = torch.zeros(hidden, device=device)
        for i in range(blocks):
            norm(f"{i}.norm", hidden)
            matrix(f"{i}.in", 2 * inner, hidden)
            self.parameters[f"{i}.taps"] = normal(inner, width, scale=width ** -0.5)
            self.parameters[f"{i}.taps.bias"] = torch.zeros(inner, device=device)
            matrix(f"{i}.mix", rank + 2 * states, inner)
            matrix(f"{i}.size", inner, rank)
            # softplus(bias) from 0.001 to 0.1: memories of some ten to some thousand decisions
            size = torch.exp(torch.rand(inner, device=device, generator=g) * math.log(100) + math.log(1e-3))
            self.parameters[f"{i}.size.bias"] = size + torch.log(-torch.expm1(-size))
            self.parameters[f"{i}.rate"] = torch.log(torch.arange(1, states + 1, device=device).float()).repeat(inner, 1)
            self.parameters[f"{i}.skip"] = torch.ones(inner, device=device)
            matrix(f"{i}.out", hidden, inner, (2 * blocks) ** -0.5)
        norm("final", hidden)
        # the actions, the value, and rows that nothing reads: the outputs' rows start on 16 bytes
        matrix("head", -(-(outputs + 1) // 8) * 8, hidden, 0.1)
        self.parameters["head.bias"] = torch.zeros(self.parameters["head"].shape[0], device=device)
        self.refresh()

    _products = ("input", "in", "mix", "size", "out", "head")

    def refresh(self):
        """bf16 copies of the matrices, for the products."""
        for name, p in self.parameters.items():
            if name.rsplit(".", 1)[-1] in self._products:
                if name not in self._weights:
                    self._weights[name] = torch.empty_like(p, dtype=torch.bfloat16)
                self._weights[name].copy_(p)

    def memory(self, fights: int):
        """The memory of `fights` fights that have seen nothing, for `step`."""
        device = self.parameters["head"].device
        return [(torch.zeros(fights, self.width - 1, self.inner, device=device, dtype=torch.bfloat16),
                 torch.zeros(fights, self.inner, self.states, device=device)) for _ in range(self.blocks)]

    def _norm(self, name, x, kept):
        p = self.parameters
        y, mean, rstd = ops.layer_norm(x, p[name + ".weight"], p[name + ".bias"], out_dtype=torch.bfloat16, save=True)
        kept[name] = (x, mean, rstd)
        return y

    def _mix(self, i, u):
        """(sizes before the bias, b, c) of u [...][inner]."""
        mixed = ops.linear(u, self._weights[f"{i}.mix"])
        size = ops.linear(mixed[..., :self.rank], self._weights[f"{i}.size"])
        b, c = mixed[..., self.rank:].split(self.states, -1)
        return mixed, size, b, c

    def step(self, observations: torch.Tensor, memory, reset=None):
        """(logits, values) fp32 of one decision of every fight; `memory` (of `memory`) is moved on in place,
        from nothing for the fights whose `reset` (bool) is set."""
        p, w = self.parameters, self._weights

        def norm(name, x):
            return ops.layer_norm(x, p[name + ".weight"], p[name + ".bias"], out_dtype=torch.bfloat16)

        x = ops.linear(norm("observation", observations), w["input"], p["input.bias"])
        for i, (window, state) in enumerate(memory):
            v, z = ops.linear(norm(f"{i}.norm", x), w[f"{i}.in"]).split(self.inner, -1)
            u = ops.causal_conv_step(v, p[f"{i}.taps"], p[f"{i}.taps.bias"], window, activation="silu", reset=reset)
            _, size, b, c = self._mix(i, u)
            y = ops.selective_scan_step(u, size, -torch.exp(p[f"{i}.rate"]), b, c, state, d=p[f"{i}.skip"], z=z,
                                        delta_bias=p[f"{i}.size.bias"], reset=reset)
            x = ops.linear(y, w[f"{i}.out"], residual=x)
        out = ops.linear(norm("final", x), w["head"], p["head.bias"], out_dtype=torch.float32)
        return out[..., :self.outputs], out[..., self.outputs]

    def forward(self, observations: torch.Tensor, reset=None):
        """(logits, values) fp32 of observations [step][fight][...], from an empty memory, and what `backward`
        needs. reset: bool [step][fight]."""
        p, w, kept = self.parameters, self._weights, {}
        rounds = None if reset is None else reset.t()
        kept["rounds"] = rounds
        n = self._norm("observation", observations, kept)
        x = ops.linear(n, w["input"], p["input.bias"])
        kept["input"] = n
        for i in range(self.blocks):
            n = self._norm(f"{i}.norm", x, kept)
            both = ops.linear(n, w[f"{i}.in"])
            v, z = both.split(self.inner, -1)
            u = ops.causal_conv(v.transpose(0, 1), p[f"{i}.taps"], p[f"{i}.taps.bias"], activation="silu",
                                reset=rounds).transpose(0, 1)
            mixed, size, b, c = self._mix(i, u)
            a = -torch.exp(p[f"{i}.rate"])
            operands = [t.transpose(0, 1) for t in (u, size)] + [a] + [t.transpose(0, 1) for t in (b, c)]
            y, saved = ops.selective_scan(*operands, d=p[f"{i}.skip"], z=z.transpose(0, 1),
                                          delta_bias=p[f"{i}.size.bias"], reset=rounds, save=True)
            kept[i] = (n, v, z, u, mixed, operands, saved, y)
            x = ops.linear(y.transpose(0, 1), w[f"{i}.out"], residual=x)
        n = self._norm("final", x, kept)
        kept["head"] = n
        out = ops.linear(n, w["head"], p["head.bias"], out_dtype=torch.float32)
        return out[..., :self.outputs], out[..., self.outputs], kept

    def backward(self, dlogits: torch.Tensor, dvalues: torch.Tensor, kept: dict) -> dict[str, torch.Tensor]:
        """The parameters' gradients from the outputs'."""
        p, w, grads, rounds = self.parameters, self._weights, {}, kept["rounds"]

        def linear(name, dy, x, bias=False):
            dx, grads[name], db = ops.linear_backward(dy, x, w[name], p[name + ".bias"] if bias else None)
            if bias:
                grads[name + ".bias"] = db
            return dx

        def norm(name, dy, residual=None):
            x, mean, rstd = kept[name]
            dx, grads[name + ".weight"], grads[name + ".bias"] = ops.layer_norm_backward(
                dy, x, p[name + ".weight"], p[name + ".bias"], mean, rstd, residual_gradient=residual)
            return dx

        out = torch.zeros(*dvalues.shape, p["head"].shape[0], device=dvalues.device, dtype=torch.bfloat16)
        out[..., :self.outputs] = dlogits
        out[..., self.outputs] = dvalues
        dx = norm("final", linear("head", out, kept["head"], True))
        for i in reversed(range(self.blocks)):
            n, v, z, u, mixed, operands, saved, y = kept[i]
            dy = linear(f"{i}.out", dx, y.transpose(0, 1))
            du, dsize, da, db, dc, grads[f"{i}.skip"], dz, grads[f"{i}.size.bias"], _ = ops.selective_scan_backward(
                dy.transpose(0, 1), *operands, saved, d=p[f"{i}.skip"], z=z.transpose(0, 1),
                delta_bias=p[f"{i}.size.bias"], reset=rounds)
            grads[f"{i}.rate"] = da * operands[2]  # a = -exp(rate) is its own slope
            dmixed = torch.cat([linear(f"{i}.size", dsize.transpose(0, 1), mixed[..., :self.rank])] +
                               [t.transpose(0, 1) for t in (db, dc)], -1)
            du = du.transpose(0, 1) + linear(f"{i}.mix", dmixed, u)
            dv, grads[f"{i}.taps"], grads[f"{i}.taps.bias"], _ = ops.causal_conv_backward(
                du.transpose(0, 1), v.transpose(0, 1), p[f"{i}.taps"], p[f"{i}.taps.bias"], activation="silu",
                reset=rounds)
            both = torch.cat([t.transpose(0, 1) for t in (dv, dz)], -1)
            dx = norm(f"{i}.norm", linear(f"{i}.in", both, n), residual=dx)
        norm("observation", linear("input", dx, kept["input"], True))
        return grads


def fit(policy: MemoryPolicy, rollout: dict, steps: int, fights: int = 512, learning_rate: float = 5e-4, clip: float = 0.2,
        kl: float = 1.0, entropy: float = 0.01, seed: int = 1) -> list[torch.Tensor]:
    """Adam on the policy loss plus half the values' squared error over random fights of a rollout: a dict of
    [step][fight] tensors observations, masks (int32 bits), actions, old_log_probabilities, advantages,
    returns, resets, and reference (the frozen policy's logits; None: no divergence). The losses, on the
    device: policy, divergence and value of each step."""
    observations = rollout["observations"]
    g = torch.Generator(device=observations.device).manual_seed(seed)
    names = list(policy.parameters)
    optimizer = torch.optim.Adam(list(policy.parameters.values()), lr=learning_rate)
    losses = []
    for _ in range(steps):
        columns = torch.randperm(observations.shape[1], device=observations.device, generator=g)[:fights]
        batch = {k: None if v is None else v[:, columns] for k, v in rollout.items()}
        logits, values, kept = policy.forward(batch["observations"], batch["resets"])
        loss, _, _, divergence, dlogits = ops.policy_loss(
            logits, batch["actions"], batch["old_log_probabilities"], batch["advantages"], mask=batch["masks"],
            reference=batch["reference"], clip=clip, kl=kl if batch["reference"] is not None else 0.0, entropy=entropy)
        off = values - batch["returns"]
        losses.append(torch.stack([loss.mean(), divergence.mean(), off.square().mean()]))
        grads = policy.backward(dlogits, off / off.numel(), kept)
        for name in names:
            policy.parameters[name].grad = grads[name].to(torch.float32)
        optimizer.step()
        policy.refresh()
    ops.status(device=observations.device)
    return losses


def rollout_of(trainer, reference: bool = True) -> dict:
    """The trainer's last rollout as `fit` takes it. `reference`: the logits that its policy has for the
    recorded observations now (after an update: the updated policy's)."""
    rollout, policy = trainer.rollout, trainer.policy
    out = {name: rollout.tensor(tensor) for name, tensor in (
        ("observations", "observations"), ("masks", "action_mask_bits"), ("actions", "actions"),
        ("old_log_probabilities", "old_log_probabilities"), ("advantages", "advantages"), ("returns", "returns"))}
    ended = rollout.tensor("terminated")
    out["resets"] = torch.zeros_like(ended, dtype=torch.bool)
    out["resets"][1:] = ended[:-1] != 0
    out["reference"] = None
    if reference:
        steps, fights = out["actions"].shape
        out["reference"] = torch.empty(steps, fights, policy.config.action_count, device=out["actions"].device)
        tables = rollout.tensor("feature_tables")
        for t in range(steps):
            given = policy.forward(out["observations"][t], None, fights, 1, t, True, None, tables[t],
                                   mask_bits=out["masks"][t], want_logits=True)
            out["reference"][t].copy_(given["logits"])
    return out


def main(arguments=None) -> list[float]:
    from . import roster as roster_module
    from .train import SelfPlayTrainer
    root = Path(__file__).resolve().parent.parent.parent
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--roster", default=str(root / "tests" / "golden" / "roster41.bin.xz"))
    parser.add_argument("--environments", type=int, default=4096)
    parser.add_argument("--horizon", type=int, default=128)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--fights", type=int, default=512)
    parser.add_argument("--blocks", type=int, default=1)
    parser.add_argument("--hidden", type=int, default=512)
    parser.add_argument("--inner", type=int, default=1024)
    parser.add_argument("--states", type=int, default=16)
    a = parser.parse_args(arguments)
    trainer = SelfPlayTrainer(roster_module.load(a.roster), a.environments, a.horizon, epochs=1, minibatches=4)
    trainer.iterate()
    data = rollout_of(trainer)
    scale = data["returns"].std().clamp(min=1e-6)
    data["returns"] = (data["returns"] - data["returns"].mean()) / scale
    policy = MemoryPolicy(data["observations"].shape[2], trainer.policy.config.action_count, a.hidden, a.inner, a.states,
                          blocks=a.blocks)
    losses = fit(policy, data, 1, a.fights)  # the first step's one-time costs stay out of the time
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = torch.stack(losses + fit(policy, data, a.steps, a.fights, seed=2))
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    last = losses[-max(1, a.steps // 10):].mean(0).tolist()
    print(f"fights {a.environments}  steps {a.steps}  {1e3 * seconds / a.steps:.2f} ms a step  policy {float(losses[0, 0]):.4f} -> "
          f"{last[0]:.4f}  divergence {float(losses[0, 1]):.4f} -> {last[1]:.4f}  value {float(losses[0, 2]):.4f} -> {last[2]:.4f}")
    return last


if __name__ == "__main__":
    main()
