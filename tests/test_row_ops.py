"""The row operators' refusals (no kernel is launched: every call is turned down before it reaches the GPU) and the host's
view of strided rows."""
import ctypes

import pytest
import torch

from compression_amd import _lib, ops
from compression_amd._lib import MpcError


def test_rows_of_views():
    t = torch.zeros(4, 6, 8)
    assert ops._rows(t, "t") == (24, 8)
    assert ops._rows(t[:, :, :5], "t") == (24, 8)                       # a slice of wider rows
    assert ops._rows(t[::2, 0], "t") == (2, 96)
    assert ops._rows(t[:, :1, 1:4], "t") == (4, 48)                     # (the axis of one row has no say)
    assert ops._rows(t[0, 0], "t") == (1, 8)
    assert ops._rows(torch.zeros(8).expand(5, 8), "t") == (5, 0)        # a broadcast row
    assert ops._rows(torch.zeros(3, 7)[:, :1], "t") == (3, 7)
    assert ops._rows(torch.zeros(0, 7), "t") == (0, 7)
    for bad in (t[:, :4], t.transpose(0, 1)[..., :5]):
        with pytest.raises(MpcError, match="evenly spaced"):
            ops._rows(bad, "t")
    with pytest.raises(MpcError, match="consecutive"):
        ops._rows(t[..., ::2], "t")
    for bad in (torch.zeros(3, 0), torch.zeros(())):
        with pytest.raises(MpcError, match="at least one value"):
            ops._rows(bad, "t")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.rms_norm(x), lambda: ops.linear(x.half(), x.half()), lambda: ops.prior_balance(x),
                 lambda: ops.prior_balance_grad(x, x, x)):
        with pytest.raises(MpcError, match="no CPU path"):
            call()


def test_linear_workspace_of_a_bad_description_is_zero():
    lib = _lib.load()
    d = _lib.LinearDesc(_lib.MPC_TYPE_F32, _lib.MPC_TYPE_F32, 0, 4, 4, 4, 4, 4, 0, 4)
    assert lib.mpc_linear_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.mpc_linear_workspace_bytes(None) == 0
    assert lib.mpc_prior_balance_workspace_bytes(-1, 64) == 0
    assert lib.mpc_prior_balance_workspace_bytes(16, 0) == 0
    assert lib.mpc_prior_balance_workspace_bytes(16, 1025) == 0
    assert lib.mpc_prior_balance_workspace_bytes(0, 64) > 0


def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    d = _lib.LinearDesc(_lib.MPC_TYPE_F16, _lib.MPC_TYPE_F16, 0, 4, 4, 4, 4, 4, 0, 4)
    assert lib.mpc_linear_forward(None, ctypes.byref(d), None, None, None, None, None, None, None, 0, None) == -1
    assert lib.mpc_rms_norm(None, None, 0, None, 0, None, 1, 1, 0.0, 0, None, None, 0, None) == -1
    assert lib.mpc_prior_balance(None, None, 0, 1, 1, 1, 1, 1.0, 1, None, None, 0, None, None, None) == -1
    assert lib.mpc_prior_balance_grad(None, None, 0, 1, 1, 1, 1, 1.0, 1, None, None, None, None, None, 1, 1) == -1
