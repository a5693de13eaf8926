"""Operands and outputs of the memory operators that lie more than 2^31 elements apart."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

FAR = 1 << 31
SEQUENCE, STEP = 4096, (1 << 30) + 8192  # of two sequences of three steps (an output's axes have to nest)
SPAN = SEQUENCE + 2 * STEP + (1 << 16)
assert 2 * STEP > FAR


class Buffer:
    """Rows of a bf16 buffer of SPAN elements."""

    def __init__(self, seed):
        import torch
        self.wide = torch.empty(SPAN, device="cuda", dtype=torch.bfloat16)
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.at = 0

    def rows(self, *row, filled=True):
        import torch
        width = 1
        for r in row:
            width *= r
        inner = [1] * len(row)
        for k in reversed(range(len(row) - 1)):
            inner[k] = inner[k + 1] * row[k + 1]
        view = self.wide.as_strided((2, 3, *row), (SEQUENCE, STEP, *inner), self.at)
        self.at += -(-width // 64) * 64
        if filled:
            view.copy_(torch.randn(view.shape, device="cuda", generator=self.g))
        else:
            view.fill_(float("nan"))
        return view


def track(v):
    from t8b import _lib
    return _lib.Track(v.data_ptr(), v.stride(0), v.stride(1))


def fine(status):
    from t8b import _lib
    assert status == 0, _lib.lib().t8b_last_error()


def test_sequences_far_apart(cuda):
    """Inputs and outputs, through the C entries, bit for bit as through t8b.ops with everything close together."""
    import torch
    from t8b import _lib, ops
    lib = _lib.lib()
    n, states, groups = 24, 16, 2
    buffer = Buffer(3)
    u, delta, z, dy = (buffer.rows(n) for _ in range(4))
    b, c = (buffer.rows(groups, states) for _ in range(2))
    near = [v.contiguous().clone() for v in (u, delta, z, dy, b, c)]
    a = -torch.exp(torch.randn(n, states, device="cuda", generator=buffer.g))
    # a buffer each: outputs may not lie between one another's rows
    y, du, ddelta, dz = (Buffer(4).rows(n, filled=False) for _ in range(4))
    db, dc = (Buffer(4).rows(groups, states, filled=False) for _ in range(2))
    q = _lib.Sequences(sequences=2, steps=3, channels=n)
    scan = _lib.Scan(type=1, softplus=1, groups=groups, states=states, u=track(u), delta=track(delta), z=track(z), b=track(b), c=track(c),
                     b_group=states, c_group=states, a=a.data_ptr())
    saved = torch.empty(lib.t8b_selective_scan_saved(C.byref(q), groups, states), device="cuda")
    final, da = torch.empty(2, n, states, device="cuda"), torch.empty(n, states, device="cuda")
    size = lib.t8b_selective_scan_workspace(C.byref(q), groups, states, 1)
    workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    fine(lib.t8b_selective_scan_forward(C.byref(q), C.byref(scan), track(y), final.data_ptr(), saved.data_ptr(), None, 0, stream))
    gradients = _lib.ScanGradients(du=track(du), ddelta=track(ddelta), dz=track(dz), db=track(db), dc=track(dc), db_group=states, dc_group=states,
                                   da=da.data_ptr())
    fine(lib.t8b_selective_scan_backward(C.byref(q), C.byref(scan), track(dy), saved.data_ptr(), None, C.byref(gradients), workspace.data_ptr(),
                                         size, stream))
    want_y, want_final, kept = ops.selective_scan(near[0], near[1], a, near[4], near[5], z=near[2], final=True, save=True)
    want = ops.selective_scan_backward(near[3], near[0], near[1], a, near[4], near[5], kept, z=near[2])
    assert torch.equal(y, want_y) and torch.equal(final, want_final) and torch.equal(saved, kept)
    for got, k in ((du, 0), (ddelta, 1), (da, 2), (db, 3), (dc, 4), (dz, 6)):
        assert torch.equal(got, want[k]), k
    again = ops.selective_scan_backward(dy, u, delta, a, b, c, saved, z=z)
    assert all(v is w or torch.equal(v, w) for v, w in zip(again, want))

    w = torch.randn(n, 4, device="cuda", generator=buffer.g)
    dw = torch.empty_like(w)
    y.fill_(float("nan"))
    du.fill_(float("nan"))
    size = lib.t8b_causal_conv_workspace(C.byref(q), 4)
    silu = ops.ACTIVATIONS.index("silu")
    fine(lib.t8b_causal_conv_forward(C.byref(q), 1, track(u), w.data_ptr(), None, 0, 4, silu, None, track(y), None, stream))
    workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
    fine(lib.t8b_causal_conv_backward(C.byref(q), 1, track(dy), track(u), w.data_ptr(), None, 0, 4, silu, None, None, track(du), dw.data_ptr(), None,
                                      None, workspace.data_ptr(), size, stream))
    assert torch.equal(y, ops.causal_conv(near[0], w, activation="silu"))
    dx, dweight, _, _ = ops.causal_conv_backward(near[3], near[0], w, activation="silu")
    assert torch.equal(du, dx) and torch.equal(dw, dweight)
    # single steps of three sequences that far apart
    state, other = torch.zeros(3, n, states, device="cuda"), torch.zeros(3, n, states, device="cuda")
    one = ops.selective_scan_step(u[1], delta[1], a, b[1], c[1], state, z=z[1])
    assert torch.equal(one, ops.selective_scan_step(near[0][1], near[1][1], a, near[4][1], near[5][1], other, z=near[2][1]))
    assert torch.equal(state, other)
    window, other = torch.ones(3, 3, n, device="cuda", dtype=torch.bfloat16), torch.ones(3, 3, n, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(ops.causal_conv_step(u[1], w, None, window), ops.causal_conv_step(near[0][1], w, None, other))
    assert torch.equal(window, other)


@pytest.mark.parametrize("n", [368, 2000, 2001])
def test_loss_rows_far_apart(cuda, n):
    """Logits, a reference, a mask and the gradient: three rows each, 2^30 and more apart."""
    import torch
    from t8b import _lib, ops
    lib = _lib.lib()
    far = (1 << 30) + 4096
    g = torch.Generator(device="cuda").manual_seed(n)

    def spread(dtype, offset=0):
        wide = torch.empty(2 * far + (1 << 16), device="cuda", dtype=dtype)
        return wide.as_strided((3, n), (far, 1), offset)

    z, q, grad, mask = spread(torch.bfloat16), spread(torch.bfloat16), spread(torch.bfloat16), spread(torch.uint8)
    assert 2 * z.stride(0) > FAR
    for v in (z, q):
        v.copy_(torch.randn(3, n, device="cuda", generator=g))
    mask.copy_(torch.rand(3, n, device="cuda", generator=g) < 0.7)
    actions = mask.int().argmax(1)
    old, advantages = torch.full((3,), -5.0, device="cuda"), torch.tensor([1.0, -1.0, 2.0], device="cuda")
    loss = torch.empty(3, device="cuda")
    call = _lib.PolicyLoss(type=1, mask_kind=2, reference_kind=1, clip_low=0.2, clip_high=0.2, kl=0.3, entropy=0.1, rows=3, n=n,
                           logits=z.data_ptr(), logits_stride=far, actions=actions.data_ptr(), old_log_probabilities=old.data_ptr(),
                           advantages=advantages.data_ptr(), mask=mask.data_ptr(), mask_stride=far, reference=q.data_ptr(), reference_stride=far)
    grad.fill_(float("nan"))
    fine(lib.t8b_policy_loss(C.byref(call), loss.data_ptr(), None, None, None, grad.data_ptr(), far, torch.cuda.current_stream().cuda_stream))
    out = ops.policy_loss(z, actions, old, advantages, mask=mask, reference=q, kl=0.3, entropy=0.1)
    # (rows that start alike, so that the same kernel takes them)
    pad = -(-n // 8) * 8
    close = [torch.zeros(3, pad, device="cuda", dtype=torch.bfloat16)[:, :n].copy_(v) for v in (z, q)]
    want = ops.policy_loss(close[0], actions, old, advantages, mask=mask.contiguous(), reference=close[1], kl=0.3, entropy=0.1)
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[4])
    assert all(torch.equal(v, w) for v, w in zip(out, want))


def test_kept_states_beyond_32_bits(cuda):
    """More than 2^31 kept floats, as many partial sums in the workspace: the last sequences as alone."""
    import torch
    from t8b import ops
    s, t, n, states, some = 32768 + 64, 8, 1024, 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.bfloat16)

    u, delta, dy, b, c = normal(s, t, n), normal(s, t, n), normal(s, t, n), normal(s, t, states), normal(s, t, states)
    a = -torch.exp(torch.randn(n, states, device="cuda", generator=g))

    def run(rows):
        y, saved = ops.selective_scan(u[rows], delta[rows], a, b[rows], c[rows], save=True)
        got = ops.selective_scan_backward(dy[rows], u[rows], delta[rows], a, b[rows], c[rows], saved)
        return saved.numel(), [y, got[0], got[1], got[3], got[4]]

    count, got = run(slice(0, s))
    assert count > FAR
    for rows in (slice(0, some), slice(s - some, s)):
        for v, w in zip(got, run(rows)[1]):
            assert torch.equal(v[rows], w)
