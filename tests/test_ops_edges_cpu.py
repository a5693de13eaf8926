"""Refusals of the torso operators' C entries that need no GPU: each comes back before anything is queued."""
import pytest

BASE, STEP = 1 << 40, 1 << 30  # addresses that no refused call touches


def call(entry, names, **changed):
    from t8b import _lib
    values = dict(names)
    assert set(changed) <= set(values)
    values.update(changed)
    return getattr(_lib.lib(), entry)(*values.values(), None)


def at(i):
    return BASE + i * STEP


LINEAR = dict(type=1, x=at(0), xs=64, w=at(1), ws=64, b=at(2), bt=0, act=1, r=at(3), rs=64, rows=40, n=64, m=64, y=at(4), yt=0,
              ys=64, p=at(5), ps=64, work=0, size=0)
GATED = dict(type=1, x=at(0), xs=64, w=at(1), ws=64, b=at(2), bt=0, act=1, rows=40, n=64, m=64, y=at(4), ys=64, p=at(5), ps=128,
             work=0, size=0)
BACKWARD = dict(type=1, dy=at(0), dys=64, x=at(1), xs=64, w=at(2), ws=64, p=at(3), ps=128, bt=0, act=1, rows=40, n=64, m=64,
                dx=at(4), dxs=64, dw=at(5), dws=64, db=at(6), work=at(7), size=1 << 29)
NORM = dict(x=at(0), xt=0, xs=64, w=at(1), b=at(2), pt=0, eps=1e-5, rows=40, n=64, y=at(3), yt=1, ys=64, mean=at(4), rstd=at(5))
NORM_BACKWARD = dict(dy=at(0), yt=1, dys=64, x=at(1), xt=0, xs=64, w=at(2), pt=0, mean=at(3), rstd=at(4), r=at(5), rs=64, rows=40,
                     n=64, dx=at(6), dxs=64, dw=at(7), db=at(8), work=at(9), size=1 << 29)


@pytest.mark.parametrize("entry,names,elements", [
    ("t8b_linear_forward", LINEAR, dict(x=2, w=2, b=4, r=4, y=4, p=2)),
    ("t8b_gated_forward", GATED, dict(x=2, w=2, b=4, y=2, p=2)),
    ("t8b_linear_backward", BACKWARD, dict(dy=2, x=2, w=2, p=2, dx=2, dw=2, db=4)),
    ("t8b_gated_backward", BACKWARD, dict(dy=2, x=2, w=2, p=2, dx=2, dw=2, db=4)),
    ("t8b_layer_norm_forward", NORM, dict(x=4, w=4, b=4, y=2, mean=4, rstd=4)),
    ("t8b_layer_norm_backward", NORM_BACKWARD, dict(dy=2, x=4, w=4, mean=4, rstd=4, r=4, dx=4, dw=4, db=4)),
])
def test_pointers_off_their_elements_are_refused(entry, names, elements):
    from t8b import _lib
    for name, size in elements.items():
        for off in {1, size // 2}:
            assert call(entry, names, **{name: names[name] + off}) == _lib.T8B_EINVAL, (name, off)
            assert b"aligned to its elements" in _lib.lib().t8b_last_error(), (name, off)


class FakeDevice:
    """torch.cuda.device, as far as it says which device is current."""
    current = 0

    def __init__(self, device):
        import torch
        self.index = FakeDevice.current if device is None else torch.device(device).index

    def __enter__(self):
        self.before, FakeDevice.current = FakeDevice.current, self.index

    def __exit__(self, *error):
        FakeDevice.current = self.before


class FakeStream:
    def __init__(self, index):
        import torch
        self.device, self.cuda_stream = torch.device("cuda", index), 1000 + index


def test_status_reads_the_record_of_the_streams_device(monkeypatch):
    """The library answers for the current device: each stream's own has to be current."""
    import torch
    from t8b import _lib, ops
    asked = []

    class Library:
        @staticmethod
        def t8b_operators_status(raw):
            asked.append((FakeDevice.current, raw))
            return _lib.T8B_OK if FakeDevice.current != 2 else _lib.T8B_ECUDA

        @staticmethod
        def t8b_last_error():
            return b"a wait ran out"

    monkeypatch.setattr(torch.cuda, "device", FakeDevice)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: FakeStream(FakeDevice.current))
    monkeypatch.setattr(ops._lib, "lib", lambda: Library)
    ops.status()
    ops.status(FakeStream(1))
    ops.status(device=torch.device("cuda", 3))
    with pytest.raises(_lib.T8bError):
        ops.status(FakeStream(2))
    assert asked == [(0, 1000), (1, 1001), (3, 1003), (2, 1002)]
    assert FakeDevice.current == 0


def test_a_stream_of_another_device_is_refused():
    """A call runs where its tensors are; a stream elsewhere could not order it."""
    import torch
    from t8b import ops
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    at = FakeStream(1)
    for refused in (lambda: ops.linear(x, w, stream=at), lambda: ops.linear_backward(x, x, w, stream=at),
                    lambda: ops.gated(x, w, stream=at), lambda: ops.gated_backward(x, x, w, stream=at),
                    lambda: ops.layer_norm(x, stream=at),
                    lambda: ops.layer_norm_backward(x, x, None, None, x, x, stream=at)):
        with pytest.raises(ValueError, match="the stream is on cuda:1, x on cpu"):
            refused()
