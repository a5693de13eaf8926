"""Torso operator checks that need no GPU: the module loads and binds, refuses what is not a CUDA
tensor, and the workspace queries answer."""
import pytest


def test_module_refuses_without_a_gpu():
    import torch
    from t8b import ops
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.linear(x, w), lambda: ops.gated(x, w), lambda: ops.layer_norm(x),
                 lambda: ops.linear_backward(x, x, w), lambda: ops.gated_backward(x, x, w),
                 lambda: ops.layer_norm_backward(x, x, None, None, x, x), lambda: ops.linear(x, None),
                 lambda: ops.linear(1, w), lambda: ops.linear(x, w, activation="softmax"),
                 lambda: ops.linear(x, w, activation=None), lambda: ops.layer_norm(x, out_dtype="bf16"),
                 lambda: ops.layer_norm(x, out_dtype=torch.int32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.layer_norm(x, eps="small")


def test_entries_refuse_without_queueing():
    from t8b import _lib
    lib = _lib.lib()
    assert lib.t8b_linear_forward(0, 0, 8, 0, 8, 0, 0, 0, 0, 8, 4, 8, 8, 0, 0, 8, 0, 8, 0, 0, None) == _lib.T8B_EINVAL
    assert b"bf16 or f16" in lib.t8b_last_error()
    assert lib.t8b_layer_norm_forward(0, 0, 8, 0, 0, 0, 1e-5, 4, 8, 0, 0, 8, 0, 0, None) == _lib.T8B_EINVAL
    assert b"null" in lib.t8b_last_error()


def test_workspace_queries():
    from t8b import _lib
    lib = _lib.lib()
    for rows, n, m in ((1, 1, 1), (7, 151, 33), (65536, 512, 1408), (2051, 1001, 1333)):
        forward, backward = lib.t8b_linear_workspace(rows, n, m, 6), lib.t8b_linear_workspace(rows, n, m, 15)
        assert forward >= 2 * (rows * n + m * n) and backward >= forward + 2 * rows * m
        assert lib.t8b_gated_workspace(rows, n, m, 15) >= backward
        assert lib.t8b_linear_workspace(rows, n, m, 0) == 0
        parts = [lib.t8b_linear_workspace(rows, n, m, what) for what in (1, 9, 11, 15)]
        assert parts == sorted(parts) and parts[1] - parts[0] >= 2 * rows * m
        assert lib.t8b_layer_norm_workspace(rows, n) >= 8 * n
    for bad in ((0, 8, 8), (-1, 8, 8), (8, 0, 8), (8, 8, 1 << 30)):
        assert lib.t8b_linear_workspace(*bad, 15) == 0
