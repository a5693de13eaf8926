"""The operators of a policy with memory as measured cases: the short causal convolution and the
selective state space scan (prompts, training steps, single steps), and the clipped policy loss over
masked logits with its gradient.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, with `own` set, through t8b.ops. `exact` restates the definitions in 64 bits.
Sizes: 1,024 is twice the policy network's hidden width of 512 (a memory block's inner width), 128 the
horizon of a rollout and 512 x 128 = 65,536 steps a PPO minibatch of whole fights, 32,768 the fights of
one GPU's rollout, 96 an evaluation's fights, 368 the action candidates. 16 states a channel and 4 taps
are generic, as are the other sizes.
"""
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # an evaluation's 96 fights, one decision: a call whose time is its launch
        dict(name="conv step 96x1024", op="conv", way="step", sequences=96, n=1024, width=4, type="bf16", act="silu",
             reset=True, slack=0),
        # a minibatch of whole fights, [step][fight] as the rollout lies, rounds ending inside it
        dict(name="conv fwd 512x128x1024", op="conv", way="fwd", sequences=512, steps=128, n=1024, width=4,
             type="bf16", act="silu", order="time", reset=True, lengths=False, slack=1024),
        # its gradients
        dict(name="conv bwd 512x128x1024", op="conv", way="bwd", sequences=512, steps=128, n=1024, width=4,
             type="bf16", act="silu", order="time", reset=True, lengths=False, slack=1024),
        # one fight against a person: a single step of a single sequence
        dict(name="scan step 1x1024x16", op="scan", way="step", sequences=1, n=1024, states=16, groups=1, type="bf16",
             gate=True, reset=False, slack=32),
        # a rollout's decision: every fight's state read and written, 1.07 GB
        dict(name="scan step 32768x512x16", op="scan", way="step", sequences=32768, n=512, states=16, groups=1,
             type="bf16", gate=True, reset=True, slack=32),
        # the forward pass over a minibatch of whole fights
        dict(name="scan fwd 512x128x1024x16", op="scan", way="fwd", sequences=512, steps=128, n=1024, states=16,
             groups=1, type="bf16", gate=True, order="time", reset=True, lengths=False, slack=32),
        # one long record, first to last: parallel work only along its length
        dict(name="scan fwd 1x8192x1024x16", op="scan", way="fwd", sequences=1, steps=8192, n=1024, states=16,
             groups=1, type="bf16", gate=True, order="sequence", reset=False, lengths=False, slack=32),
        # a training step over the minibatch: forward pass and gradients, the largest case
        dict(name="scan train 512x128x1024x16", op="scan", way="train", sequences=512, steps=128, n=1024, states=16,
             groups=1, type="bf16", gate=True, order="time", reset=True, lengths=False, slack=32),
        # a ragged batch of records of different lengths in half precision, two groups, odd sizes and strides
        dict(name="scan train 7x1501x650x24", op="scan", way="train", sequences=7, steps=1501, n=650, states=24,
             groups=2, type="f16", gate=False, order="sequence", reset=False, lengths=True, slack=5),
        # an evaluation's decision: losses of 96 rows
        dict(name="loss 96x368", op="loss", way="fwd", rows=96, n=368, type="f32", mask="bits", reference="none",
             slack=0),
        # a minibatch of decisions with its gradient, held near the frozen policy that it started from
        dict(name="loss grad 65536x368", op="loss", way="grad", rows=65536, n=368, type="f32", mask="bits",
             reference="logits", slack=0),
        # a large vocabulary of an odd size, its estimate of the divergence from the sampled log-probabilities
        dict(name="loss grad 4096x50257", op="loss", way="grad", rows=4096, n=50257, type="bf16", mask="none",
             reference="sampled", slack=47),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Any operator and direction: 1 to 1,024 sequences of 1 to 4,096 steps (single steps: of up to 32,768
    sequences), 8 to 2,048 channels, 2 to 64 states, 1 to 65,536 rows of 5 to 65,536 logits, no more in all
    than the largest listed case; one width in two off a multiple of 8; inputs packed or inside wider buffers."""
    op = rng.choice(["conv", "scan", "loss"])
    case = dict(op=op, type=rng.choice(list(TYPES)))

    def width(low, high):
        w = _log(rng, low, high)
        return w if rng.random() < 0.5 else -(-w // 8) * 8

    if op == "loss":
        case.update(way=rng.choice(["fwd", "grad", "grad"]), n=width(5, 65536), mask=rng.choice(["none", "bits", "bytes"]),
                    reference=rng.choice(["none", "logits", "sampled"]), slack=rng.choice([0, 0, 8, 3]))
        case["rows"] = min(_log(rng, 1, 65536), max(1, (1 << 27) // case["n"]))
        return case
    case.update(way=rng.choice(["step", "fwd", "bwd" if op == "conv" else "train"]), n=width(8, 2048),
                slack=rng.choice([0, 0, 8, 3]))
    if op == "conv":
        case.update(width=rng.choice([2, 3, 4, 4]), act=rng.choice(["none", "silu", "silu"]))
        states = 4
    else:
        states = case["states"] = rng.choice([16, 16, _log(rng, 2, 64)])
        case.update(groups=rng.choice([1, 1, 2]), gate=rng.random() < 0.6)
        case["n"] += case["n"] % case["groups"]
    case["reset"] = rng.random() < 0.5
    if case["way"] == "step":
        case["sequences"] = min(_log(rng, 1, 32768), max(1, (1 << 28) // (case["n"] * states)))
        return case
    case.update(steps=_log(rng, 1, 4096), order=rng.choice(["time", "sequence"]), lengths=rng.random() < 0.4)
    case["sequences"] = min(_log(rng, 1, 1024), max(1, (1 << 29) // (case["n"] * states * case["steps"])))
    return case


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)
    t, n = TYPES[case["type"]], case["n"]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def held(values, dtype=t):
        """`values` as a user holds them: packed, or a column range of a wider buffer."""
        if not case["slack"]:
            return values.to(dtype)
        wide = torch.zeros(*values.shape[:-1], values.shape[-1] + case["slack"], device="cuda", dtype=dtype)
        wide[..., : values.shape[-1]] = values
        return wide[..., : values.shape[-1]]

    if case["op"] == "loss":
        rows = case["rows"]
        logits = 2.0 * normal(rows, n)
        s["logits"] = held(logits)
        legal = None
        if case["mask"] != "none":
            legal = uniform(rows, n) < 0.05 + 0.9 * uniform(rows, 1)  # few legal actions, or nearly all
            legal[torch.arange(rows, device="cuda"), torch.randint(n, (rows,), device="cuda", generator=g)] = True
        z = s["logits"].double() if legal is None else s["logits"].double().masked_fill(~legal, -math.inf)
        # sampled by the policy that played: the logits a little off
        noise = -torch.log(-torch.log(uniform(rows, n).clamp(1e-7, 1 - 1e-7)))
        s["actions"] = (z.float() + noise).argmax(1)
        del noise
        lp = torch.log_softmax(z, 1).gather(1, s["actions"][:, None])[:, 0]
        del z
        # the ratio's logarithm: a few updates' drift; none within 1e-4 of a border, where the last bits of the
        # log-probability would decide which side of it a row is on
        drift = 0.15 * normal(rows).double()
        for border in (math.log(1 - 0.2), math.log(1 + 0.2)):
            drift = torch.where((drift - border).abs() < 1e-4, drift + 3e-4, drift)
        s["old"] = (lp - drift).float()
        s["advantages"] = normal(rows)
        s["weights"] = (uniform(rows) < 0.9).float() / rows  # some steps count for nothing: padding
        s["mask"] = legal
        if case["mask"] == "bits":
            words = -(-n // 32)
            padded = torch.zeros(rows, 32 * words, dtype=torch.bool, device="cuda")
            padded[:, :n] = legal
            value = padded.view(rows, words, 32).long() << torch.arange(32, device="cuda")
            value = value.sum(2)
            s["bits"] = torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32)
        if case["reference"] == "logits":
            s["reference"] = held(logits + 0.3 * normal(rows, n))
        elif case["reference"] == "sampled":
            s["reference"] = (lp + 0.2 * normal(rows).double()).float()
        return s

    sequences, steps = case["sequences"], case.get("steps", 1)

    def sequence(*shape, make=normal, dtype=t, hold=True):
        """[sequences][steps][...] in the case's order, or [sequences][...] for single steps."""
        if case["way"] == "step":
            v = make(sequences, *shape)
            return held(v, dtype) if hold else v
        if case["order"] == "time":
            v = make(steps, sequences, *shape)
            return (held(v, dtype) if hold else v).transpose(0, 1)
        v = make(sequences, steps, *shape)
        return held(v, dtype) if hold else v

    if case["reset"]:  # rounds of some forty decisions
        s["reset"] = sequence(hold=False, make=lambda *shape: uniform(*shape) < 0.025)
    if case.get("lengths"):
        s["lengths"] = (steps * (0.1 + 0.9 * uniform(sequences))).ceil().to(torch.int32)
    if case["op"] == "conv":
        k = case["width"]
        s["x"] = sequence(n)
        s["weight"] = (normal(n, k) / math.sqrt(k)).contiguous()
        s["bias"] = 0.1 * normal(n)
        s["state"] = normal(sequences, k - 1, n).to(t)
        if case["way"] == "bwd":
            s["dy"] = sequence(n, make=lambda *shape: normal(*shape) / 64, hold=False).to(t)
        return s
    m, groups = case["states"], case["groups"]
    s["u"] = sequence(n)
    s["delta"] = sequence(n, make=lambda *shape: 0.5 * normal(*shape))
    # B and C as they come from one projection: column ranges of it
    both = sequence(groups * 2 * m)
    both = both.unflatten(-1, (2, groups, m))
    s["b"], s["c"] = both.select(-3, 0), both.select(-3, 1)
    s["a"] = -torch.exp(torch.log(torch.arange(1, m + 1, device="cuda").float()) + 0.2 * normal(n, m))
    s["d"] = 1 + 0.2 * normal(n)
    step = torch.exp(uniform(n) * math.log(100) + math.log(1e-3))  # steps from 0.001 to 0.1
    s["delta_bias"] = step + torch.log(-torch.expm1(-step))
    s["z"] = sequence(n) if case["gate"] else None
    s["state"] = 0.3 * normal(sequences, n, m)
    if case["way"] == "train":
        s["dy"] = sequence(n, make=lambda *shape: normal(*shape) / 64, hold=False).to(t)
    return s


# ------------------------------------------------------------------ plain form
def _silu(z):
    sigma = 1 / (1 + torch.exp(-z))
    return z * sigma, sigma * (1 + z * (1 - sigma))


def _live(s, t):
    """Which sequences have a step t, as a column; None where all have."""
    return None if "lengths" not in s else (s["lengths"] > t)[:, None]


def _like(values, x):
    """`values` in x's type and in the order of its axes."""
    values = values.to(x.dtype)
    if x.dim() == 3 and x.stride(0) < x.stride(1):
        return values.transpose(0, 1).contiguous().transpose(0, 1)
    return values


def _plain_conv(s):
    case, x, w, b = s["case"], s["x"], s["weight"].float(), s["bias"].float()
    k = case["width"]
    if case["way"] == "step":
        window = s["state"].float()
        if case["reset"]:
            window = torch.where(s["reset"][:, None, None], torch.zeros_like(window), window)
        window = torch.cat([window, x.float()[:, None]], 1)
        p = b + (window * w.t()).sum(1)
        s["state"].copy_(window[:, 1:])
        return {"y": (_silu(p)[0] if case["act"] == "silu" else p).to(x.dtype), "state": s["state"]}
    steps = case["steps"]
    rows = torch.cat([s["state"].float(), x.float()], 1)  # [sequences][width - 1 + steps][n]
    # whether the tap j steps back belongs to the same round and record
    since = torch.full((case["sequences"], steps), k, device=x.device)
    if case["reset"]:
        count = since.new_full((case["sequences"],), k)
        for t in range(steps):
            count = torch.where(s["reset"][:, t], torch.zeros_like(count), count + 1)
            since[:, t] = count
    live = torch.ones(case["sequences"], steps, 1, dtype=torch.bool, device=x.device)
    if "lengths" in s:
        live = (torch.arange(steps, device=x.device) < s["lengths"][:, None])[:, :, None]
    taps = [torch.where((since >= j)[:, :, None], rows[:, k - 1 - j:k - 1 - j + steps], torch.zeros((), device=x.device))
            for j in range(k)]
    p = b + sum(tap * w[:, k - 1 - j] for j, tap in enumerate(taps))
    if case["way"] == "fwd":
        y = torch.where(live, _silu(p)[0] if case["act"] == "silu" else p, torch.zeros_like(p))
        last = s["lengths"].long() if "lengths" in s else torch.full((case["sequences"],), steps, device=x.device)
        at = last[:, None] + torch.arange(k - 1, device=x.device)  # the last width - 1 rows
        final = rows.gather(1, at[:, :, None].expand(-1, -1, x.shape[2]))
        if case["reset"]:
            count = torch.where(last > 0, since.gather(1, (last - 1).clamp(min=0)[:, None])[:, 0], torch.full_like(last, k))
            keep = torch.arange(k - 1, device=x.device) >= k - 2 - count[:, None]
            final = torch.where(keep[:, :, None], final, torch.zeros_like(final))
        return {"y": _like(y, x), "state": final.to(x.dtype)}
    dp = torch.where(live, s["dy"].float() * (_silu(p)[1] if case["act"] == "silu" else torch.ones_like(p)), torch.zeros_like(p))
    drows = torch.zeros_like(rows)
    dw = torch.zeros_like(w)
    for j, tap in enumerate(taps):
        drows[:, k - 1 - j:k - 1 - j + steps] += torch.where((since >= j)[:, :, None], dp * w[:, k - 1 - j], torch.zeros_like(dp))
        dw[:, k - 1 - j] = (dp * tap).sum((0, 1))
    return {"dx": _like(drows[:, k - 1:], x), "dweight": dw, "dbias": dp.sum((0, 1)), "dstate": drows[:, :k - 1].to(x.dtype)}


def _plain_scan(s):
    case, a, d = s["case"], s["a"], s["d"]
    u = s["u"].float()
    v = s["delta"].float() + s["delta_bias"]
    size = torch.where(v > 20, v, torch.log1p(torch.exp(v)))  # softplus
    per = case["n"] // case["groups"]
    h = s["state"]
    if case["way"] == "step":
        if case["reset"]:
            h = torch.where(s["reset"][:, None, None], torch.zeros_like(h), h)
        b, c = (s[k].float().repeat_interleave(per, 1) for k in "bc")
        h = torch.exp(size[:, :, None] * a) * h + (size * u)[:, :, None] * b
        y = (h * c).sum(2) + d * u
        if s["z"] is not None:
            y = y * _silu(s["z"].float())[0]
        s["state"].copy_(h)
        return {"y": y.to(s["u"].dtype), "state": s["state"]}
    steps, keep = case["steps"], case["way"] == "train"
    y, kept = torch.zeros_like(u), []
    b, c = s["b"].float(), s["c"].float()
    zero = torch.zeros((), device=u.device)

    def shared(v, t):
        v = v[:, t]
        return v.repeat_interleave(per, 1) if case["groups"] > 1 else v  # [sequences][n or 1][states]

    for t in range(steps):
        if case["reset"]:
            h = torch.where(s["reset"][:, t, None, None], zero, h)
        before = h
        step = size[:, t]
        h = torch.exp(step[:, :, None] * a) * h + (step * u[:, t])[:, :, None] * shared(b, t)
        out = (h * shared(c, t)).sum(2) + d * u[:, t]
        live = _live(s, t)
        if live is not None:
            h = torch.where(live[:, :, None], h, before)
            out = torch.where(live, out, zero)
        y[:, t] = out
        if keep:
            kept.append((before, h))
    final = h
    gate = slope = None
    if s["z"] is not None:
        gate, slope = _silu(s["z"].float())
    if not keep:
        return {"y": _like(y if gate is None else y * gate, s["u"]), "state": final}
    dy = s["dy"].float()
    out = {"y": _like(y if gate is None else y * gate, s["u"])}
    if gate is not None:
        out["dz"] = _like(dy * y * slope, s["z"])
        dy = dy * gate
    du, dsize = torch.zeros_like(u), torch.zeros_like(u)
    db, dc, da, dd = torch.zeros_like(b), torch.zeros_like(c), torch.zeros_like(a), torch.zeros_like(d)
    carry = torch.zeros_like(final)
    for t in reversed(range(steps)):
        before, h = kept[t]
        kept[t] = None
        step, live = size[:, t], _live(s, t)
        given = dy[:, t] if live is None else torch.where(live, dy[:, t], zero)
        decay = torch.exp(step[:, :, None] * a)
        g = carry + given[:, :, None] * shared(c, t)
        if live is not None:
            g = torch.where(live[:, :, None], g, zero)
        dc[:, t] = (given[:, :, None] * h).unflatten(1, (case["groups"], per)).sum(2)
        db[:, t] = ((step * u[:, t])[:, :, None] * g).unflatten(1, (case["groups"], per)).sum(2)
        gb = (g * shared(b, t)).sum(2)
        through = g * decay * before
        du[:, t] = d * given + step * gb
        dsize[:, t] = u[:, t] * gb + (through * a).sum(2)
        da += (through * step[:, :, None]).sum(0)
        dd += (given * u[:, t]).sum(0)
        g = g * decay
        if live is not None:
            g = torch.where(live[:, :, None], g, carry)
        carry = torch.where(s["reset"][:, t, None, None], zero, g) if case["reset"] else g
    dv = dsize * torch.where(v > 20, torch.ones_like(v), 1 / (1 + torch.exp(-v)))
    out.update(du=_like(du, s["u"]), ddelta=_like(dv, s["u"]), db=_like_shared(db, s), dc=_like_shared(dc, s), da=da, dd=dd,
               ddelta_bias=dv.sum((0, 1)), dstate=carry)
    return out


def _like_shared(values, s):
    return values.to(s["b"].dtype)


def _plain_loss(s):
    case, z = s["case"], s["logits"].float()
    rows = torch.arange(case["rows"], device=z.device)
    zero = torch.zeros((), device=z.device)
    legal = s["mask"]
    if legal is not None:
        z = torch.where(legal, z, torch.full_like(zero, -math.inf))
    off = z - z.amax(1, keepdim=True)
    e = torch.exp(off)
    # in 64 bits from here: the ratio against the border of the clipped range
    total = e.sum(1, dtype=torch.float64)
    p = e / total.float()[:, None]
    logp = off - torch.log(total).float()[:, None]
    lp = off[rows, s["actions"]].double() - torch.log(total)
    entropy = -torch.where(p > 0, p * logp, zero).sum(1)
    ratio = torch.exp(lp - s["old"].double())
    advantage = s["advantages"].double()
    free, held = ratio * advantage, ratio.clamp(1 - 0.2, 1 + 0.2) * advantage
    loss = -torch.minimum(free, held) - 0.01 * entropy.double()
    slope = torch.where(free <= held, -free, torch.zeros_like(free))  # of the loss in the log-probability
    divergence = torch.zeros_like(entropy)
    apart = None
    if case["reference"] == "sampled":
        gap = s["reference"].double() - lp
        divergence = (torch.exp(gap) - gap - 1).float()
        slope = slope + 0.1 * (1 - torch.exp(gap))
    elif case["reference"] == "logits":
        q = s["reference"].float()
        if legal is not None:
            q = torch.where(legal, q, torch.full_like(zero, -math.inf))
        q = q - q.amax(1, keepdim=True)
        apart = logp - (q - torch.log(torch.exp(q).sum(1, keepdim=True)))
        apart = torch.where(p > 0, apart, zero)
        divergence = (p * apart).sum(1)
    out = {"loss": (loss + 0.1 * divergence.double()).float(), "log_probabilities": lp.float(), "entropies": entropy,
           "divergences": divergence}
    if case["way"] == "fwd":
        return out
    grad = -p * slope.float()[:, None] + 0.01 * torch.where(p > 0, p * (logp + entropy[:, None]), zero)
    if apart is not None:
        grad += 0.1 * p * (apart - divergence[:, None])
    grad[rows, s["actions"]] += slope.float()
    out["dlogits"] = (grad * s["weights"][:, None]).to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------ the framework's operators
def _ops():
    at = str(Path(__file__).resolve().parent.parent / "tekken8-agent_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from t8b import ops
    return ops


def _own(s):
    ops, case = _ops(), s["case"]
    if case["op"] == "loss":
        mask = s["bits"] if case["mask"] == "bits" else s["mask"]
        out = ops.policy_loss(s["logits"], s["actions"], s["old"], s["advantages"], mask=mask,
                              reference=s.get("reference"), weights=s["weights"], clip=0.2, kl=0.1, entropy=0.01,
                              gradient=case["way"] == "grad")
        return dict(zip(("loss", "log_probabilities", "entropies", "divergences", "dlogits"), out))
    reset, lengths = s.get("reset"), s.get("lengths")
    if case["op"] == "conv":
        common = dict(activation=case["act"], reset=reset)
        if case["way"] == "step":
            y = ops.causal_conv_step(s["x"], s["weight"], s["bias"], s["state"], **common)
            return {"y": y, "state": s["state"]}
        common.update(state=s["state"], lengths=lengths)
        if case["way"] == "fwd":
            y, state = ops.causal_conv(s["x"], s["weight"], s["bias"], final=True, **common)
            return {"y": y, "state": state}
        dx, dw, db, dstate = ops.causal_conv_backward(s["dy"], s["x"], s["weight"], s["bias"], **common)
        return {"dx": dx, "dweight": dw, "dbias": db, "dstate": dstate}
    operands = (s["u"], s["delta"], s["a"], s["b"], s["c"])
    common = dict(d=s["d"], z=s["z"], delta_bias=s["delta_bias"], softplus=True, reset=reset)
    if case["way"] == "step":
        y = ops.selective_scan_step(*operands, s["state"], **common)
        return {"y": y, "state": s["state"]}
    common.update(state=s["state"], lengths=lengths)
    if case["way"] == "fwd":
        y, state = ops.selective_scan(*operands, final=True, **common)
        if reset is not None and lengths is not None:
            # a round that begins behind a record's end leaves it nothing, by the definition here: the operator does
            # not look behind the end
            behind = torch.arange(case["steps"], device=state.device) >= lengths[:, None]
            state = torch.where((reset & behind).any(1)[:, None, None], torch.zeros_like(state), state)
        return {"y": y, "state": state}
    y, saved = ops.selective_scan(*operands, save=True, **common)
    du, ddelta, da, db, dc, dd, dz, dbias, dstate = ops.selective_scan_backward(s["dy"], *operands, saved, **common)
    out = {"y": y}
    if dz is not None:
        out["dz"] = dz
    out.update(du=du, ddelta=ddelta, db=db, dc=dc, da=da, dd=dd, ddelta_bias=dbias, dstate=dstate)
    return out


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "scan": _plain_scan, "loss": _plain_loss}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the least a pass has to do
def work(case):
    e, n = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]], case["n"]
    if case["op"] == "loss":
        rows = case["rows"]
        mask = {"none": 0, "bits": 4 * -(-n // 32), "bytes": n}[case["mask"]]
        reference = {"none": 0, "sampled": 4, "logits": e * n}[case["reference"]]
        if case["way"] == "fwd":
            return {"bytes": rows * (e * n + mask + reference + 32), "flops": 6 * rows * n}
        return {"bytes": rows * (2 * e * n + mask + reference + 36), "flops": 14 * rows * n}
    sequences, tokens = case["sequences"], case["sequences"] * case.get("steps", 1)
    flags = tokens if case["reset"] else 0
    if case["op"] == "conv":
        k = case["width"]
        window = e * sequences * (k - 1) * n
        if case["way"] in ("step", "fwd"):
            return {"bytes": 2 * e * tokens * n + 2 * window + flags + 4 * n * (k + 1), "flops": 2 * tokens * n * (k + 2)}
        return {"bytes": 3 * e * tokens * n + 2 * window + flags + 8 * n * (k + 1), "flops": 2 * tokens * n * (3 * k + 4)}
    m, groups = case["states"], case["groups"]
    shared = 2 * e * tokens * groups * m
    streams = 4 if case["gate"] else 3
    state = 4 * sequences * n * m
    if case["way"] in ("step", "fwd"):
        return {"bytes": streams * e * tokens * n + shared + 2 * state + flags + 4 * n * (m + 2), "flops": 7 * tokens * n * m}
    # forward and backward: u, delta, z and dy once, y, du, ddelta and dz once
    return {"bytes": 2 * streams * e * tokens * n + 2 * shared + 2 * state + flags + 8 * n * (m + 2),
            "flops": 24 * tokens * n * m}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The definitions in 64 bits; gradients by automatic differentiation of them."""
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "loss": _exact_loss}[case["op"]](case, s)


def _exact_loss(case, s):
    parts = []
    for at in range(0, case["rows"], max(1, (1 << 25) // case["n"])):
        rows = slice(at, at + max(1, (1 << 25) // case["n"]))
        z = s["logits"][rows].double().requires_grad_(case["way"] == "grad")
        legal = torch.ones_like(z, dtype=torch.bool) if s["mask"] is None else s["mask"][rows]
        log_all = z - torch.logsumexp(z.masked_fill(~legal, -1e300), 1)[:, None]
        p = log_all.exp() * legal
        lp = torch.take_along_dim(log_all, s["actions"][rows][:, None], 1).squeeze(1)
        advantage = s["advantages"][rows].double()
        ratio = (lp - s["old"][rows].double()).exp()
        within = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 0.8)), torch.full_like(ratio, 1.2))
        entropy = -(p * log_all).sum(1)
        if case["reference"] == "none":
            divergence = torch.zeros_like(lp)
        elif case["reference"] == "sampled":
            back = s["reference"][rows].double() - lp
            divergence = torch.expm1(back) - back
        else:
            q = s["reference"][rows].double()
            q = q - torch.logsumexp(q.masked_fill(~legal, -1e300), 1)[:, None]
            divergence = (p * (log_all - q)).sum(1)
        loss = torch.maximum(-ratio * advantage, -within * advantage) + 0.1 * divergence - 0.01 * entropy
        part = {"loss": loss, "log_probabilities": lp, "entropies": entropy, "divergences": divergence}
        if case["way"] == "grad":
            part["dlogits"], = torch.autograd.grad((loss * s["weights"][rows].double()).sum(), z)
        parts.append({k: v.detach() for k, v in part.items()})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_conv(case, s):
    k, step = case["width"], case["way"] == "step"
    x = s["x"][:, None] if step else s["x"]
    leaves = {key: v.double().requires_grad_(case["way"] == "bwd") for key, v in
              (("x", x), ("weight", s["weight"]), ("bias", s["bias"]), ("state", s["state"]))}
    window = [leaves["state"][:, j] for j in range(k - 1)]
    steps, ys, ended = x.shape[1], [], None
    reset = s["reset"][:, None] if step and case["reset"] else s.get("reset")
    lengths = s.get("lengths")
    finals = [torch.zeros_like(w) for w in window]
    for t in range(steps + 1):
        if lengths is not None:  # the windows of the records that end here
            finals = [torch.where((lengths == t)[:, None], w, f) for w, f in zip(window, finals)]
        if t == steps:
            break
        if reset is not None:
            window = [w * (~reset[:, t, None]).double() for w in window]
        window = window + [leaves["x"][:, t]]
        p = leaves["bias"] + torch.einsum("jsc,cj->sc", torch.stack(window), leaves["weight"])
        y = p * torch.sigmoid(p) if case["act"] == "silu" else p
        ys.append(y if lengths is None else y * (lengths > t)[:, None])
        window = window[1:]
    y = torch.stack(ys, 1)
    if case["way"] != "bwd":
        state = torch.stack(window if lengths is None else finals, 1)
        return {"y": y[:, 0] if step else y, "state": state}
    grads = torch.autograd.grad((y * s["dy"].double()).sum(), [leaves[key] for key in ("x", "weight", "bias", "state")])
    return dict(zip(("dx", "dweight", "dbias", "dstate"), grads))


def _exact_scan(case, s):
    step, train = case["way"] == "step", case["way"] == "train"
    expand = (lambda v: None if v is None else v[:, None]) if step else (lambda v: v)
    steps, n, m, groups = case.get("steps", 1), case["n"], case["states"], case["groups"]
    per = n // groups
    block = max(1, (3 << 28) // (steps * n * m)) if train else case["sequences"]
    parts, sums = [], None
    for at in range(0, case["sequences"], block):
        cut = slice(at, at + block)
        one = {k: expand(s[k][cut]).double() for k in ("u", "delta", "b", "c", "z") if s[k] is not None}
        one.update({k: s[k].double() for k in ("a", "d", "delta_bias")}, state=s["state"][cut].double())
        if train:
            for v in one.values():
                v.requires_grad_()
        reset = expand(s["reset"][cut]) if case["reset"] else None
        lengths = s["lengths"][cut] if "lengths" in s else None
        size = torch.nn.functional.softplus(one["delta"] + one["delta_bias"], threshold=40.0)
        h = one["state"].unflatten(1, (groups, per))  # [sequences][groups][channels][states]
        a = one["a"].unflatten(0, (groups, per))
        ys = []
        for t in range(steps):
            if reset is not None:
                h = h * (~reset[:, t])[:, None, None, None]
            x = one["u"][:, t].unflatten(1, (groups, per))
            dt = size[:, t].unflatten(1, (groups, per))
            new = (dt[..., None] * a).exp() * h + torch.einsum("sgc,sgn->sgcn", dt * x, one["b"][:, t])
            out = torch.einsum("sgcn,sgn->sgc", new, one["c"][:, t]).flatten(1) + one["d"] * one["u"][:, t]
            if lengths is not None:
                alive = lengths > t
                new = torch.where(alive[:, None, None, None], new, h)
                out = out * alive[:, None]
            h = new
            ys.append(out)
        y = torch.stack(ys, 1)
        if "z" in one:
            y = y * one["z"] * torch.sigmoid(one["z"])
        if not train:
            return {"y": y[:, 0] if step else y, "state": h.flatten(1, 2)}
        names = [k for k in ("z", "u", "delta", "b", "c", "a", "d", "delta_bias", "state") if k in one]
        grads = dict(zip(names, torch.autograd.grad((y * s["dy"][cut].double()).sum(), [one[k] for k in names])))
        total = {k: grads.pop(k) for k in ("a", "d", "delta_bias")}
        parts.append({"y": y.detach(), **{"d" + k: v for k, v in grads.items()}})
        sums = total if sums is None else {k: sums[k] + v for k, v in total.items()}
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out.update({"d" + k: v for k, v in sums.items()})
    order = ("y", "dz", "du", "ddelta", "db", "dc", "da", "dd", "ddelta_bias", "dstate")
    return {k: out[k] for k in order if k in out}
