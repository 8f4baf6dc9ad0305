"""``torch.library`` custom ops (namespace ``sr355``) on rows of channels: layer normalisation, the gated feed-forward block
and dropout onto a skip (csrc/layer_norm.hip, gated_ffn.hip, dropout.hip behind the C ABI of libsr355.so).

Argument checks, memory, streams and autograd are in ``_torch_tokens.so`` (csrc/torch_tokens.cpp), built beside the library;
the functions that a program calls are in ``tokens``.  They go to the binding's own autograd nodes, and to these ops where
PyTorch has to see an operator: in ``torch.compile`` and ``torch.export``, with fake tensors and under dispatch modes."""
from __future__ import annotations

import ctypes as C
import importlib.util
import os
from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from ._lib import Sr355Error

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}     # SR355_ACT_* of include/sr355.h
BINDING_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_tokens.so")

_binding = None


def binding():
    """The C++ module, connected to the library that the package uses."""
    global _binding
    if _binding is None:
        if not os.path.exists(BINDING_PATH):
            raise Sr355Error(f"{BINDING_PATH} is missing: build it with `make -C {_lib.CSRC_DIR}` (or "
                             "`python -c 'import __graft_entry__ as g; g.build()'`). There is no fallback.")
        L = _lib.lib()
        spec = importlib.util.spec_from_file_location("super_resolution_amd._torch_tokens", BINDING_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.connect({n: C.cast(getattr(L, n), C.c_void_p).value for n in _lib.EXPORTS if
                        n == "sr355_last_error" or n.startswith(("sr355_layer_norm", "sr355_dropout", "sr355_gated_ffn"))})
        _binding = module
    return _binding


def _whole(t: Optional[Tensor], like: Tensor, dtype: torch.dtype) -> Tensor:
    """An op returns tensors: an empty one for what was not asked for."""
    return like.new_empty((0,), dtype=dtype) if t is None else t


@torch.library.custom_op("sr355::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                   want_stats: bool) -> Tuple[Tensor, Tensor]:
    """Layer normalisation over the last dimension, and the rows' mean and 1 / sqrt(var + eps) as fp32 ``[2, rows]`` where
    ``want_stats`` (else an empty tensor)."""
    return binding().layer_norm_fwd(x, weight, bias, eps, want_stats)


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps, want_stats):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape), x.new_empty((2, rows) if want_stats else (0,), dtype=torch.float32))


def _norm_context(ctx, inputs, output):
    x, weight, bias, eps, want_stats = inputs
    ctx.save_for_backward(x, weight, output[1] if want_stats else None)
    ctx.eps = eps
    ctx.param_dtype = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)


def _norm_backward(ctx, dy, _):
    x, weight, stats = ctx.saved_tensors
    if stats is None:                     # (a caller of the op who did not ask for them)
        stats = torch.ops.sr355.layer_norm_fwd(x, weight, None, ctx.eps, True)[1]
    need = list(ctx.needs_input_grad[:3])
    grads = torch.ops.sr355.layer_norm_bwd(dy, x, weight, stats, ctx.param_dtype, need)
    return (*(g if n else None for g, n in zip(grads, need)), None, None)


layer_norm_fwd.register_autograd(_norm_backward, setup_context=_norm_context)


@torch.library.custom_op("sr355::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy: Tensor, x: Tensor, weight: Optional[Tensor], stats: Tensor, param_dtype: torch.dtype,
                   need: List[bool]) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients of ``layer_norm_fwd`` with respect to (x, weight, bias); an empty tensor where ``need`` says no."""
    dx, dw, db = binding().layer_norm_bwd(dy, x, weight, stats, param_dtype, need)
    return _whole(dx, x, x.dtype), _whole(dw, x, param_dtype), _whole(db, x, param_dtype)


@layer_norm_bwd.register_fake
def _(dy, x, weight, stats, param_dtype, need):
    c = x.shape[-1]
    return (x.new_empty(x.shape if need[0] else (0,)), x.new_empty((c,) if need[1] else (0,), dtype=param_dtype),
            x.new_empty((c,) if need[2] else (0,), dtype=param_dtype))


@torch.library.custom_op("sr355::dropout", mutates_args=())
def dropout(x: Tensor, skip: Optional[Tensor], p: float, rng: Tensor, site: int) -> Tensor:
    """``(keep ? x / (1 - p) : 0) + skip``: see ``tokens.dropout``."""
    return binding().dropout_fwd(x, skip, p, rng, site)


@dropout.register_fake
def _(x, skip, p, rng, site):
    return x.new_empty(x.shape)


def _dropout_context(ctx, inputs, output):
    _, _, ctx.p, rng, ctx.site = inputs
    ctx.save_for_backward(rng)


def _dropout_backward(ctx, dy):
    dx = torch.ops.sr355.dropout(dy, None, ctx.p, ctx.saved_tensors[0], ctx.site) if ctx.needs_input_grad[0] else None
    return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


dropout.register_autograd(_dropout_backward, setup_context=_dropout_context)


@torch.library.custom_op("sr355::gated_ffn_fwd", mutates_args=())
def gated_ffn_fwd(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, b_gate: Optional[Tensor],
                  b_up: Optional[Tensor], b_down: Optional[Tensor], activation: int,
                  want_saved: bool) -> Tuple[Tensor, Tensor]:
    """``(act(x w_gate' + b_gate) * (x w_up' + b_up)) w_down' + b_down``, and the bytes that the backward pass reads where
    ``want_saved`` (else an empty tensor)."""
    return binding().gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, want_saved)


@gated_ffn_fwd.register_fake
def _(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, want_saved):
    size = saved_bytes(x.numel() // x.shape[-1], w_gate.shape[0], x.dtype) if want_saved else 0
    return x.new_empty(x.shape), x.new_empty((size,), dtype=torch.uint8)


def saved_bytes(rows, hidden: int, dtype: torch.dtype):
    """``sr355_gated_ffn_saved_bytes``, for a number of rows that may be symbolic."""
    e = dtype.itemsize
    line = 128 // e
    step = line if hidden >= 4 * line else 8
    n = rows * ((hidden + step - 1) // step * step)
    whole = lambda b: (b + 255) // 256 * 256
    return 3 * whole(n * e) + (2 * whole(n) if e == 2 else 0) + 256


def _ffn_context(ctx, inputs, output):
    x, w_gate, w_up, w_down, b_gate, b_up, b_down, ctx.activation, want_saved = inputs
    ctx.save_for_backward(x, w_gate, w_up, w_down, b_gate, b_up, output[1] if want_saved else None)


def _ffn_backward(ctx, dy, _):
    x, w_gate, w_up, w_down, b_gate, b_up, saved = ctx.saved_tensors
    if saved is None:                     # (a caller of the op who did not ask for it)
        saved = torch.ops.sr355.gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, None, ctx.activation, True)[1]
    need = list(ctx.needs_input_grad[:7])
    grads = torch.ops.sr355.gated_ffn_bwd(dy, x, w_gate, w_up, w_down, saved, ctx.activation, need)
    return (*(g if n else None for g, n in zip(grads, need)), None, None)


gated_ffn_fwd.register_autograd(_ffn_backward, setup_context=_ffn_context)


@torch.library.custom_op("sr355::gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, saved: Tensor, activation: int,
                  need: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients of ``gated_ffn_fwd`` with respect to (x, w_gate, w_up, w_down, b_gate, b_up, b_down); an empty tensor
    where ``need`` says no."""
    return tuple(_whole(g, x, x.dtype) for g in binding().gated_ffn_bwd(dy, x, w_gate, w_up, w_down, saved, activation, need))


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, saved, activation, need):
    f, c = w_gate.shape
    shapes = (x.shape, (f, c), (f, c), (c, f), (f,), (f,), (c,))
    return tuple(x.new_empty(s if n else (0,)) for s, n in zip(shapes, need))
