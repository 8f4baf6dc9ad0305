"""CPU: the operators on rows of channels where PyTorch traces them: with fake tensors, in make_fx, export and compile.  Only shapes
are computed here."""
import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.fx.experimental.symbolic_shapes import ShapeEnv

from super_resolution_amd import _lib, token_ops, tokens
from super_resolution_amd._lib import FfnArgs

CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def inputs(dtype=torch.bfloat16, rows=(3, 5), c=24, f=40):
    e = lambda *s: torch.empty(*s, dtype=dtype, device="cuda", requires_grad=True)
    return e(*rows, c), [e(f, c), e(f, c), e(c, f)], [e(f), e(f), e(c)], torch.empty(2, dtype=torch.int64, device="cuda")


def calls(x, ws, bs, rng):
    v = torch.empty(x.shape[-1], device="cuda", requires_grad=True)
    return (lambda: tokens.layer_norm(x), lambda: tokens.layer_norm(x, v, v), lambda: tokens.layer_norm(x, None, v),
            lambda: tokens.dropout(x, 0.5, rng), lambda: tokens.dropout(x, 0.5, rng, 3, x), lambda: tokens.gated_ffn(x, *ws),
            lambda: tokens.gated_ffn(x, *ws, *bs, activation="gelu"), lambda: tokens.gated_ffn(x, *ws, None, bs[1]))


@pytest.mark.parametrize("dtype", list(CODES))
def test_fake_tensors_pass_through_the_public_functions(dtype):
    with FakeTensorMode():
        args = inputs(dtype)
        x = args[0]
        for call in calls(*args):
            y = call()
            assert y.shape == x.shape and y.dtype == dtype and y.device == x.device and y.requires_grad
            with torch.no_grad():
                assert not call().requires_grad
        with torch.device("cuda"):
            block = tokens.FeedForwardBlock(24, 40, dropout=0.1)
        y = block(x)
        assert y.shape == x.shape and y.requires_grad


def test_the_saved_bytes_of_the_fake_are_those_of_the_library():
    L = _lib.lib()
    for dtype, code in CODES.items():
        for rows in (0, 1, 7, 300, 70001):
            for hidden in (1, 8, 31, 33, 127, 128, 129, 255, 256, 257, 264, 1333, 8192):
                a = FfnArgs()
                a.dtype, a.rows, a.channels, a.hidden, a.x_ld = code, rows, 16, hidden, 16
                assert token_ops.saved_bytes(rows, hidden, dtype) == L.sr355_gated_ffn_saved_bytes(C.byref(a)), (dtype, rows, hidden)


def step(x, wg, wu, wd, rng, w):
    h = tokens.gated_ffn(tokens.layer_norm(x, w), wg, wu, wd)
    return tokens.dropout(h, 0.25, rng, 2, x)


def names(graph):
    return [n.target.name().split("::")[1] for n in graph.nodes if n.op == "call_function" and "sr355" in str(n.target)]


@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_a_trace_holds_the_operators(mode):
    with FakeTensorMode(shape_env=ShapeEnv() if mode == "symbolic" else None):
        x, ws, _, rng = inputs()
        args = [t.detach() for t in (x, *ws, rng, torch.empty(24, device="cuda"))]
    graph = make_fx(step, tracing_mode=mode)(*args).graph
    assert names(graph) == ["layer_norm_fwd", "gated_ffn_fwd", "dropout"]


def test_a_module_is_exported_in_one_graph():
    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = tokens.FeedForwardBlock(24, 40, dropout=0.1)

        def forward(self, x):
            return self.block(x) * 2

    with FakeTensorMode():
        with torch.device("cuda"):
            net = Net()
        x = torch.empty(6, 24, device="cuda")
        program = torch.export.export(net, (x,), dynamic_shapes=({0: torch.export.Dim("rows", min=2, max=4096)},))
    assert names(program.graph) == ["layer_norm_fwd", "gated_ffn_fwd", "dropout"]
