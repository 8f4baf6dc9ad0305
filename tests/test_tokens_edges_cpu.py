"""CPU: the operators on rows of channels where a call's arguments, not its numbers, decide what happens.  No kernel runs
here."""
import ctypes as C
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd

from super_resolution_amd import _lib, tokens
from super_resolution_amd._lib import FfnArgs


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


P = 4096   # an address that nothing reads


def ffn(**kw):
    a = FfnArgs()
    a.rows, a.channels, a.hidden = 70, 264, 520
    for k, v in kw.items():
        setattr(a, k, v)
    a.x_ld = a.dy_ld = a.channels
    for k in ("x_dev", "w_gate_dev", "w_up_dev", "w_down_dev", "y_dev", "dy_dev", "dx_dev", "workspace_dev", "saved_dev"):
        if not getattr(a, k):
            setattr(a, k, P)
    return C.byref(a)


@pytest.mark.parametrize("dtype,channels", [(_lib.DTYPE_BF16, 264), (_lib.DTYPE_F16, 1000), (_lib.DTYPE_BF16, 2056), (_lib.DTYPE_F32, 20),
                                            (_lib.DTYPE_F32, 100), (_lib.DTYPE_F32, 132)])
@pytest.mark.parametrize("rows", [1, 33, 70, 300])
@pytest.mark.parametrize("backward", [0, 1])
def test_gate_and_up_weights_are_padded_together(L, dtype, channels, rows, backward):
    """The kernels read both with one row stride, and a padded copy's rows are longer at these widths: where one of the two has to
    be copied, both are."""
    size = lambda **kw: L.sr355_gated_ffn_workspace_bytes(ffn(dtype=dtype, channels=channels, rows=rows, **kw), backward)
    odd = P + 4
    both = size(w_gate_dev=odd, w_up_dev=odd)
    assert both > size()
    assert size(w_gate_dev=odd) == both and size(w_up_dev=odd) == both


def test_forward_mode_derivatives_are_refused():
    """(They would be zero: the kernels compute no tangent.)"""
    x, w, wd = torch.ones(4, 8), torch.ones(16, 8), torch.ones(8, 16)
    rng = torch.zeros(2, dtype=torch.int64)
    for call in (tokens.layer_norm, lambda t: tokens.gated_ffn(t, w, w, wd), lambda t: tokens.dropout(t, 0.5, rng),
                 lambda t: torch.ops.sr355.layer_norm_fwd(t, None, None, 1e-5, False)):
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fwd.make_dual(x, torch.ones_like(x)))


def test_the_binding_is_built_for_the_running_interpreter(monkeypatch):
    """Its headers, its libraries and its C++ ABI are those of the PyTorch that will load it, whatever python3 is on PATH."""
    asked = []
    monkeypatch.setattr(_lib.subprocess, "run", lambda cmd, **kw: asked.append(cmd) or subprocess.CompletedProcess(cmd, 0, ""))
    _lib.build()
    _lib.build(again=True)
    assert len(asked) == 2 and all(f"PYTHON={sys.executable}" in cmd for cmd in asked)


def test_layer_norm_counts_channels_without_overflow(L):
    """A thread steps 256 channels at a time behind the last one, in an int."""
    last = 2 ** 31 - 1
    for c in (last, last - 254):
        assert L.sr355_layer_norm_fwd(P, 1, c, c, 0, None, None, 0, 1e-5, P, None, None, None) == -1
        assert L.sr355_layer_norm_bwd(P, c, P, c, 1, c, 0, None, 0, P, P, P, None, None, None, 0, None) == -1
        assert b"channels" in L.sr355_last_error()
        assert L.sr355_layer_norm_bwd_workspace_bytes(c) == 0
    assert L.sr355_layer_norm_bwd_workspace_bytes(last - 255) > 0


@pytest.mark.parametrize("dtype,rows,hidden", [(_lib.DTYPE_F32, 1 << 30, 72), (_lib.DTYPE_BF16, 0x7fffff00, 264), (_lib.DTYPE_F16, 1 << 30, 1 << 20)])
def test_gated_ffn_refuses_more_tiles_than_a_grid_has(L, dtype, rows, hidden):
    """A launch of 2^32 threads or more would leave out what is beyond."""
    call = lambda: ffn(dtype=dtype, rows=rows, channels=8, hidden=hidden, workspace_bytes=1 << 62, saved_bytes=1 << 62, dw_up_dev=P)
    for entry in (L.sr355_gated_ffn_fwd, L.sr355_gated_ffn_bwd):
        assert entry(call(), None) == -1
        assert b"too many tiles" in L.sr355_last_error()
