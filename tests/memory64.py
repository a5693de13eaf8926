"""The memory operators' definitions and gradients in 64 bits, step by step, on any device.

Every function also runs on magnitudes: given the absolute values of its inputs (and the true decays,
ratios or probabilities), each of its sums becomes the sum of its terms' absolute values, which is what a
bound on rounding errors is a multiple of."""
import torch


def live_of(lengths, sequences, steps, device):
    if lengths is None:
        return torch.ones(sequences, steps, dtype=torch.bool, device=device)
    return torch.arange(steps, device=device) < lengths.clamp(0, steps)[:, None]


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "tanh":
        return z.tanh(), 1 - z.tanh() ** 2
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * phi, phi + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    return z, torch.ones_like(z)


# ------------------------------------------------------------------ causal convolution
def conv64(x, w, b, state, reset=None, lengths=None):
    """(pre-activations [s][t][c], the final state)."""
    s, steps, n = x.shape
    k = w.shape[1]
    x, w = x.double(), w.double()
    window = torch.zeros(s, k - 1, n, dtype=torch.float64, device=x.device) if state is None else state.double()
    live = live_of(lengths, s, steps, x.device)
    out = torch.zeros(s, steps, n, dtype=torch.float64, device=x.device)
    for t in range(steps):
        begun = window
        if reset is not None:
            begun = torch.where(reset[:, t, None, None] != 0, torch.zeros_like(begun), begun)
        row = torch.where(live[:, t, None], x[:, t], torch.zeros_like(x[:, t]))
        full = torch.cat([begun, row[:, None]], 1)
        p = (full * w.t()).sum(1)
        if b is not None:
            p = p + b.double()
        out[:, t] = torch.where(live[:, t, None], p, torch.zeros_like(p))
        window = torch.where(live[:, t, None, None], full[:, 1:], window)
    return out, window


def conv_grad64(dp, x, w, state, reset=None, lengths=None, dfinal=None):
    """(dx, dweight, dbias, dstate) from the pre-activations' gradient."""
    s, steps, n = x.shape
    k = w.shape[1]
    x, w = x.double(), w.double()
    live = live_of(lengths, s, steps, x.device)
    window = torch.zeros(s, k - 1, n, dtype=torch.float64, device=x.device) if state is None else state.double()
    windows = []
    for t in range(steps):
        begun = window
        if reset is not None:
            begun = torch.where(reset[:, t, None, None] != 0, torch.zeros_like(begun), begun)
        row = torch.where(live[:, t, None], x[:, t], torch.zeros_like(x[:, t]))
        full = torch.cat([begun, row[:, None]], 1)
        windows.append(full)
        window = torch.where(live[:, t, None, None], full[:, 1:], window)
    dwindow = torch.zeros_like(window) if dfinal is None else dfinal.double()
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros(n, dtype=torch.float64, device=x.device)
    for t in reversed(range(steps)):
        on = live[:, t, None]
        d = torch.where(on, dp[:, t].double(), torch.zeros_like(x[:, t]))
        dfull = d[:, None] * w.t()
        dw += (d[:, None] * windows[t]).sum(0).t()
        db += d.sum(0)
        dfull[:, 1:] += torch.where(on[:, None], dwindow, torch.zeros_like(dwindow))
        dx[:, t] = torch.where(on, dfull[:, k - 1], torch.zeros_like(dfull[:, k - 1]))
        back = dfull[:, :k - 1]
        if reset is not None:
            back = torch.where(reset[:, t, None, None] != 0, torch.zeros_like(back), back)
        dwindow = torch.where(on[:, None], back, dwindow)
    return dx, dw, db, dwindow


# ------------------------------------------------------------------ selective scan
def spread64(v, per):
    """[s][t][groups][states] -> [s][t][channels][states]"""
    return v.double().repeat_interleave(per, 2)


def scan64(size, u, a, b, c, d, state, reset=None, lengths=None, decays=None):
    """(outputs before the gate, every step's state [s][t][c][n], the state before each step, the final state, the
    decays) of sizes and inputs [s][t][c], b and c [s][t][g][n]."""
    s, steps, n = u.shape
    per = n // b.shape[2]
    size, u, a = size.double(), u.double(), a.double()
    b, c = spread64(b, per), spread64(c, per)
    live = live_of(lengths, s, steps, u.device)
    h = torch.zeros(s, n, a.shape[1], dtype=torch.float64, device=u.device) if state is None else state.double()
    outs, states, befores, rates = [], [], [], []
    zero = torch.zeros((), dtype=torch.float64, device=u.device)
    for t in range(steps):
        before = h
        if reset is not None:
            before = torch.where(reset[:, t, None, None] != 0, zero, h)
        e = torch.exp(size[:, t, :, None] * a) if decays is None else decays[t]
        on = live[:, t, None, None]
        new = torch.where(on, e * before + (size[:, t] * u[:, t])[:, :, None] * b[:, t], h)
        out = (new * c[:, t]).sum(2)
        if d is not None:
            out = out + d.double() * u[:, t]
        outs.append(torch.where(on[:, :, 0], out, zero))
        states.append(new)
        befores.append(before)
        rates.append(e)
        h = new
    return torch.stack(outs, 1) if steps else torch.zeros_like(u), states, befores, h, rates


def scan_grad64(gs, size, u, a, b, c, d, states, befores, decays, reset=None, lengths=None, dfinal=None):
    """(du, dsize, da, db, dc, dd, dstate) from the gradient of the outputs before the gate."""
    s, steps, n = u.shape
    groups = b.shape[2]
    per = n // groups
    gs, size, u, a = gs.double(), size.double(), u.double(), a.double()
    wide_b, wide_c = spread64(b, per), spread64(c, per)
    live = live_of(lengths, s, steps, u.device)
    zero = torch.zeros((), dtype=torch.float64, device=u.device)
    carry = torch.zeros(s, n, a.shape[1], dtype=torch.float64, device=u.device) if dfinal is None else dfinal.double()
    du, dsize = torch.zeros_like(u), torch.zeros_like(u)
    db, dc = torch.zeros(b.shape, dtype=torch.float64, device=u.device), torch.zeros(b.shape, dtype=torch.float64, device=u.device)
    da, dd = torch.zeros_like(a), torch.zeros(n, dtype=torch.float64, device=u.device)
    for t in reversed(range(steps)):
        on = live[:, t, None, None]
        given = torch.where(on[:, :, 0], gs[:, t], zero)
        g = torch.where(on, carry + given[:, :, None] * wide_c[:, t], zero)
        dc[:, t] = (given[:, :, None] * torch.where(on, states[t], zero)).unflatten(1, (groups, per)).sum(2)
        db[:, t] = ((size[:, t] * u[:, t])[:, :, None] * g).unflatten(1, (groups, per)).sum(2)
        gb = (g * wide_b[:, t]).sum(2)
        through = g * decays[t] * befores[t]
        du[:, t] = size[:, t] * gb + (0 if d is None else d.double() * given)
        dsize[:, t] = u[:, t] * gb + (through * a).sum(2)
        da += (through * size[:, t, :, None]).sum(0)
        dd += (given * u[:, t]).sum(0)
        back = g * decays[t]
        if reset is not None:
            back = torch.where(reset[:, t, None, None] != 0, zero, back)
        carry = torch.where(on, back, carry)
    du = torch.where(live[:, :, None], du, zero)
    dsize = torch.where(live[:, :, None], dsize, zero)
    return du, dsize, da, db, dc, dd, carry


# ------------------------------------------------------------------ policy loss
def loss64(logits, actions, old, advantages, legal=None, reference=None, sampled=None, weights=None, low=0.2, high=0.2,
           kl=0.0, entropy=0.0):
    """A dict of the loss, log-probabilities, entropies, divergences and dlogits, and of the terms that bounds
    are built of. A row whose action is not legal is 0 everywhere."""
    z = logits.double()
    rows, n = z.shape
    if legal is None:
        legal = torch.ones(rows, n, dtype=torch.bool, device=z.device)
    inside = (actions >= 0) & (actions < n)
    at = actions.clamp(0, n - 1)[:, None]
    counts = inside & legal.gather(1, at)[:, 0]
    zero, never = torch.zeros((), dtype=torch.float64, device=z.device), torch.tensor(-float("inf"), dtype=torch.float64, device=z.device)
    zm = torch.where(legal, z, never)


    def log_softmax(v):  # from the largest: beside one of 1e38 the logarithm of a sum is lost even in 64 bits
        v = v - v.amax(1, keepdim=True)
        return v - torch.log(torch.exp(v).sum(1, keepdim=True))

    logp = log_softmax(zm)
    p = torch.where(legal, logp.exp(), zero)
    some = p > 0
    lp = logp.gather(1, at)[:, 0]
    h = -torch.where(some, p * logp, zero).sum(1)
    ratio = torch.exp(lp - old.double())
    adv = advantages.double()
    free, held = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    slope = torch.where(free <= held, -free, zero)
    k = torch.zeros_like(lp)
    apart = torch.zeros_like(p)
    if reference is not None:
        q = torch.where(legal, reference.double(), never)
        apart = torch.where(some, logp - log_softmax(q), zero)
        k = torch.where(some, p * apart, zero).sum(1)
    if sampled is not None:
        e = sampled.double() - lp
        k = torch.expm1(e) - e
        slope = slope - kl * torch.expm1(e)
    w = torch.full((rows,), 1.0 / rows, dtype=torch.float64, device=z.device) if weights is None else weights.double()
    inner = torch.where(some, -slope[:, None] + kl * (apart - (k[:, None] if reference is not None else 0)) + entropy * (logp + h[:, None]), zero)
    grad = torch.where(some, p * inner, zero)
    grad = grad + torch.where(torch.arange(n, device=z.device) == at, slope[:, None], zero)
    mask = counts[:, None]
    out = {"loss": -torch.minimum(free, held) + kl * k - entropy * h, "log_probabilities": lp, "entropies": h, "divergences": k}
    out = {key: torch.where(counts, v, zero) for key, v in out.items()}
    out["dlogits"] = torch.where(mask, grad * w[:, None], zero)
    out.update(p=p, logp=torch.where(some, logp, zero), apart=apart, ratio=ratio, slope=slope, weight=w, counts=counts)
    return out
