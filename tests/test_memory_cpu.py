"""Memory operator checks that need no GPU: the module refuses what is not a CUDA tensor, the C entries refuse
bad arguments before they queue anything, and the queries answer."""
import ctypes as C

import pytest


def test_module_refuses_without_a_gpu():
    import torch
    from t8b import ops
    x, w = torch.zeros(2, 3, 8), torch.zeros(8, 4)
    a, b, row = torch.zeros(8, 4), torch.zeros(2, 3, 4), torch.zeros(2)
    for call in (lambda: ops.causal_conv(x, w), lambda: ops.causal_conv_backward(x, x, w), lambda: ops.causal_conv(x, None),
                 lambda: ops.causal_conv_step(x[:, 0], w, None, x), lambda: ops.causal_conv(x, w, activation="softmax"),
                 lambda: ops.selective_scan(x, x, a, b, b), lambda: ops.selective_scan(x, 1, a, b, b),
                 lambda: ops.selective_scan_backward(x, x, x, a, b, b, row), lambda: ops.selective_scan_step(x[:, 0], x[:, 0], a, b[:, 0], b[:, 0], x),
                 lambda: ops.policy_loss(x[0, :2], row.long(), row, row), lambda: ops.policy_loss(None, row.long(), row, row)):
        with pytest.raises(ValueError):
            call()


def sequences(**more):
    from t8b import _lib
    q = dict(sequences=4, steps=6, channels=8)
    q.update(more)
    return _lib.Sequences(**q)


def track(data=4096, sequence=48, step=8):
    from t8b import _lib
    return _lib.Track(data, sequence, step)


def refused(status, words):
    from t8b import _lib
    assert status == _lib.T8B_EINVAL
    message = _lib.lib().t8b_last_error().decode()
    assert words in message, message


def test_conv_refuses():
    from t8b import _lib
    lib = _lib.lib()

    def forward(q=None, kind=1, x=None, weight=4096, bias=None, parameter=0, width=4, act=3, state=None, y=None, final=None):
        q = sequences() if q is None else q
        return lib.t8b_causal_conv_forward(C.byref(q), kind, track() if x is None else x, weight, bias, parameter, width, act, state,
                                           track(1 << 20) if y is None else y, final, None)

    refused(lib.t8b_causal_conv_forward(None, 1, track(), 4096, None, 0, 4, 3, None, track(1 << 20), None, None), "null")
    refused(forward(q=sequences(sequences=-1)), "sequences")
    refused(forward(q=sequences(steps=-1)), "steps")
    refused(forward(q=sequences(channels=0)), "channels")
    refused(forward(q=sequences(reset=1, reset_sequence=-1)), "reset")
    refused(forward(q=sequences(lengths=2)), "aligned")
    refused(forward(kind=7), "type")
    refused(forward(kind=1, parameter=2), "fp32 or of x's type")
    for width in (0, 1, 5):
        refused(forward(width=width), "width")
    refused(forward(act=9), "activation")
    refused(forward(weight=None), "weight is null")
    refused(forward(weight=4098), "aligned")
    refused(forward(x=track(None)), "null")
    refused(forward(x=track(4097)), "aligned")
    refused(forward(x=track(4096, -8, 8)), "stride")
    refused(forward(x=track(4096, 1 << 61, 8)), "stride")
    refused(forward(y=track(1 << 20, 48, 7)), "overlap")
    refused(forward(y=track(1 << 20, 8, 8)), "overlap")
    refused(forward(y=track(4096)), "overlaps")
    refused(forward(final=4096), "overlaps")
    refused(lib.t8b_causal_conv_backward(C.byref(sequences()), 1, track(1 << 20), track(), 4096, None, 0, 4, 3, None, None, track(1 << 21),
                                         1 << 22, None, None, None, 0, None), "workspace")
    refused(lib.t8b_causal_conv_step(C.byref(sequences()), 1, track(), 4096, None, 0, 4, 3, None, track(1 << 20), None), "state is null")


def scan(**more):
    from t8b import _lib
    given = dict(type=1, softplus=1, groups=1, states=4, u=track(), delta=track(1 << 16), b=track(1 << 17, 24, 4), c=track(1 << 18, 24, 4),
                 b_group=4, c_group=4, a=1 << 19)
    given.update(more)
    return _lib.Scan(**given)


def test_scan_refuses():
    from t8b import _lib
    lib = _lib.lib()

    def forward(q=None, s=None, y=None, final=None, saved=None):
        q, s = sequences() if q is None else q, scan() if s is None else s
        return lib.t8b_selective_scan_forward(C.byref(q), C.byref(s), track(1 << 20) if y is None else y, final, saved, None, 0, None)

    refused(lib.t8b_selective_scan_forward(C.byref(sequences()), None, track(1 << 20), None, None, None, 0, None), "null")
    refused(forward(s=scan(type=4)), "type")
    for states in (0, 65):
        refused(forward(s=scan(states=states)), "states")
    for groups in (0, 3):
        refused(forward(s=scan(groups=groups)), "groups")
    refused(forward(s=scan(a=None)), "a is null")
    refused(forward(s=scan(a=(1 << 19) + 2)), "aligned")
    refused(forward(s=scan(delta=track(None))), "null")
    refused(forward(s=scan(b=track(1 << 17, -4, 4))), "stride")
    refused(forward(s=scan(groups=2, c_group=-1)), "group stride")
    refused(forward(y=track(1 << 16)), "overlaps")
    refused(forward(final=4096), "overlaps")
    long = sequences(sequences=1, steps=4096)
    refused(forward(q=long), "workspace")
    g = _lib.ScanGradients(du=track(1 << 21), ddelta=track(1 << 22), db=track(1 << 23, 24, 4), dc=track(1 << 24, 24, 4), db_group=4, dc_group=4,
                           da=1 << 25)
    back = lambda saved, g, workspace=None, size=0: lib.t8b_selective_scan_backward(  # noqa: E731
        C.byref(sequences()), C.byref(scan()), track(1 << 20), saved, None, C.byref(g) if g else None, workspace, size, None)
    refused(back(1 << 26, None), "gradients are null")
    refused(back(None, g), "saved is null")
    refused(back(1 << 26, g), "workspace")
    g.dz = track(1 << 27)
    refused(back(1 << 26, g), "dz without z")
    refused(lib.t8b_selective_scan_step(C.byref(sequences()), C.byref(scan()), None, track(1 << 20), None), "state is null")


def test_loss_refuses():
    from t8b import _lib
    lib = _lib.lib()

    def loss(dlogits=None, **more):
        given = dict(type=0, rows=4, n=8, logits=4096, logits_stride=8, actions=1 << 13, old_log_probabilities=1 << 14, advantages=1 << 15,
                     clip_low=0.2, clip_high=0.2)
        given.update(more)
        return lib.t8b_policy_loss(C.byref(_lib.PolicyLoss(**given)), 1 << 16, None, None, None, dlogits, 8, None)

    refused(lib.t8b_policy_loss(None, None, None, None, None, None, 8, None), "null")
    refused(loss(type=3), "type")
    refused(loss(rows=-1), "rows")
    for n in (0, (1 << 24) + 1):
        refused(loss(n=n), "logits a row")
    refused(loss(logits=None), "null")
    refused(loss(logits=4098), "aligned")
    refused(loss(logits_stride=7), "stride")
    refused(loss(mask_kind=3), "mask")
    refused(loss(mask_kind=1), "mask is null")
    refused(loss(reference_kind=3), "reference")
    refused(loss(reference_kind=1), "reference is null")
    refused(loss(reference_kind=2), "reference is null")
    refused(loss(actions=None), "actions")
    refused(loss(clip_low=-0.1), "clipped range")
    refused(loss(clip_high=float("nan")), "clipped range")
    refused(loss(kl=float("inf")), "coefficients")
    refused(loss(entropy=float("nan")), "coefficients")
    refused(loss(dlogits=4096), "overlaps")


def test_queries():
    from t8b import _lib
    lib = _lib.lib()
    for s, t, n, states in ((1, 1, 1, 1), (3, 40, 65, 16), (512, 128, 1024, 16), (1, 8192, 1024, 64)):
        q = sequences(sequences=s, steps=t, channels=n)
        assert lib.t8b_selective_scan_saved(C.byref(q), 1, states) == s * -(-t // 8) * states * n
        assert lib.t8b_selective_scan_workspace(C.byref(q), 1, states, 1) >= 4 * (s * t * 2 * states + n * (states + 2))
        assert lib.t8b_causal_conv_workspace(C.byref(q), 4) >= 4 * 5 * n
    assert lib.t8b_selective_scan_workspace(C.byref(sequences(sequences=512, steps=128, channels=1024)), 1, 16, 0) == 0  # enough sequences
    assert lib.t8b_selective_scan_workspace(C.byref(sequences(sequences=1, steps=8192, channels=1024)), 1, 16, 0) > 0  # one, cut into chunks
    for bad in (sequences(sequences=0), sequences(steps=0)):
        assert lib.t8b_selective_scan_saved(C.byref(bad), 1, 4) == lib.t8b_selective_scan_workspace(C.byref(bad), 1, 4, 1) == 0
    assert lib.t8b_selective_scan_saved(C.byref(sequences()), 3, 4) == 0  # groups that do not divide the channels


def test_structs_match_the_c_compiler(tmp_path):
    import subprocess
    from conftest import ROOT
    from t8b import _lib
    names = {"t8b_track_t": _lib.Track, "t8b_sequences_t": _lib.Sequences, "t8b_scan_t": _lib.Scan,
             "t8b_scan_gradients_t": _lib.ScanGradients, "t8b_policy_loss_t": _lib.PolicyLoss}
    lines = []
    for name, cls in names.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    source = tmp_path / "layout.c"
    source.write_text(f'#include "t8b.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void){{{"".join(lines)}return 0;}}\n')
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "layout")]).split()]
    want = []
    for cls in names.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, field).offset for field, _ in cls._fields_]
    assert got == want
