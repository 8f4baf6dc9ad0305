"""``torch.library`` custom ops (namespace ``sr355``) on rows of channels over the C ABI of libsr355.so: layer
normalisation, the gated feed-forward block and dropout onto a skip (csrc/layer_norm.hip, gated_ffn.hip, dropout.hip).

Tensors are ``[..., C]``; a tensor whose rows do not lie at one stride with their channels contiguous is copied first.
The autograd functions and the module on top are in ``tokens``."""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from ._lib import DTYPE_BF16, DTYPE_F16, DTYPE_F32, FfnArgs, check
from .ops import _on, _ptr, _stream, now

CODES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16, torch.float32: DTYPE_F32}
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}     # SR355_ACT_* of include/sr355.h


def check_rows(who: str, x: Tensor, *others: Optional[Tensor]) -> None:
    """``x`` is a tensor of rows in one of the types, and what comes with it lies on its device."""
    if not x.is_cuda:
        raise RuntimeError(f"{who}: runs on ROCm devices only (got a tensor on {x.device}); there is no CPU fallback")
    if x.dtype not in CODES:
        raise RuntimeError(f"{who}: expected bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"{who}: expected rows of at least one channel, got shape {tuple(x.shape)}")
    for t in others:
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{who}: tensors on {x.device} and {t.device}")


def as_rows(x: Tensor) -> Tuple[Tensor, int]:
    """``x`` as ``[rows, C]`` with contiguous channels, and its row stride in elements."""
    c = x.shape[-1]
    if x.is_contiguous():
        return x, c
    r = x.reshape(-1, c)
    if r.shape[0] > 1 and r.stride(0) < c or c > 1 and r.stride(1) != 1:
        r = r.contiguous()
    return r, (r.stride(0) if r.shape[0] > 1 else c)


def _vector(who: str, name: str, v: Optional[Tensor], n: int, dtypes) -> Optional[Tensor]:
    if v is None:
        return None
    if v.shape != (n,) or v.dtype not in dtypes:
        raise RuntimeError(f"{who}: {name} must have shape ({n},) and type {' or '.join(map(str, dtypes))}, got "
                           f"{tuple(v.shape)} of {v.dtype}")
    return v.contiguous()


# ------------------------------------------------------------------------------------
def _norm_params(who: str, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor]):
    dtypes = (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32)
    w = _vector(who, "weight", weight, x.shape[-1], dtypes)
    b = _vector(who, "bias", bias, x.shape[-1], dtypes)
    if w is not None and b is not None and w.dtype != b.dtype:
        raise RuntimeError(f"{who}: weight and bias are of types {w.dtype} and {b.dtype}")
    return w, b, (w.dtype if w is not None else b.dtype if b is not None else torch.float32)


@torch.library.custom_op("sr355::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                   want_stats: bool) -> Tuple[Tensor, Tensor]:
    """Layer normalisation over the last dimension, and the rows' mean and 1 / sqrt(var + eps) as fp32 ``[2, rows]`` where
    ``want_stats`` (else an empty tensor)."""
    check_rows("layer_norm", x, weight, bias)
    w, b, wt = _norm_params("layer_norm", x, weight, bias)
    if not eps >= 0.0:
        raise RuntimeError(f"layer_norm: eps must not be negative, got {eps}")
    r, ld = as_rows(x)
    c = x.shape[-1]
    rows = x.numel() // c
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows) if want_stats else (0,), dtype=torch.float32, device=x.device)
    at = stats.data_ptr() if want_stats else None
    with _on(x.device):
        check(_lib.lib().sr355_layer_norm_fwd(r.data_ptr(), rows, c, ld, CODES[x.dtype], _ptr(w), _ptr(b), CODES[wt], eps,
                                              y.data_ptr(), at, at + 4 * rows if at else at, _stream()),
              "sr355_layer_norm_fwd")
    return y, stats


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps, want_stats):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape), x.new_empty((2, rows) if want_stats else (0,), dtype=torch.float32))


@torch.library.custom_op("sr355::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy: Tensor, x: Tensor, weight: Optional[Tensor], stats: Tensor, param_dtype: torch.dtype,
                   need: List[bool]) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients of ``layer_norm_fwd`` with respect to (x, weight, bias); an empty tensor where ``need`` says no."""
    check_rows("layer_norm backward", x, dy, weight, stats)
    c = x.shape[-1]
    rows = x.numel() // c
    if dy.shape != x.shape or dy.dtype != x.dtype or stats.shape != (2, rows) or stats.dtype != torch.float32:
        raise RuntimeError("layer_norm backward: the gradient must have x's shape and type, the statistics be fp32 [2, rows]")
    r, ld = as_rows(x)
    g, g_ld = as_rows(dy)
    w = _vector("layer_norm backward", "weight", weight, c, (param_dtype,))
    stats = stats.contiguous()
    dx = torch.empty(x.shape if need[0] else (0,), dtype=x.dtype, device=x.device)
    dw = torch.empty((c,) if need[1] else (0,), dtype=param_dtype, device=x.device)
    db = torch.empty((c,) if need[2] else (0,), dtype=param_dtype, device=x.device)
    L = _lib.lib()
    size = L.sr355_layer_norm_bwd_workspace_bytes(c) if need[1] or need[2] else 0
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    at = stats.data_ptr() if rows else None
    with _on(x.device):
        check(L.sr355_layer_norm_bwd(g.data_ptr(), g_ld, r.data_ptr(), ld, rows, c, CODES[x.dtype], _ptr(w),
                                     CODES[param_dtype], at, at + 4 * rows if at else at,
                                     dx.data_ptr() if need[0] else None, dw.data_ptr() if need[1] else None,
                                     db.data_ptr() if need[2] else None, ws.data_ptr(), size, _stream()),
              "sr355_layer_norm_bwd")
    return dx, dw, db


@layer_norm_bwd.register_fake
def _(dy, x, weight, stats, param_dtype, need):
    c = x.shape[-1]
    return (x.new_empty(x.shape if need[0] else (0,)), x.new_empty((c,) if need[1] else (0,), dtype=param_dtype),
            x.new_empty((c,) if need[2] else (0,), dtype=param_dtype))


# ------------------------------------------------------------------------------------
@torch.library.custom_op("sr355::dropout", mutates_args=())
def dropout(x: Tensor, skip: Optional[Tensor], p: float, rng: Tensor, site: int) -> Tensor:
    """``(keep ? x / (1 - p) : 0) + skip``: see ``tokens.dropout``."""
    check_rows("dropout", x, skip, rng)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout: the probability must lie in [0, 1], got {p}")
    if rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
        raise RuntimeError("dropout: the generator's state is a contiguous int64 tensor of two words (seed, step)")
    if not 0 <= site < 1 << 32:
        raise RuntimeError(f"dropout: the site must lie in [0, 2^32), got {site}")
    if skip is not None and (skip.shape != x.shape or skip.dtype != x.dtype):
        raise RuntimeError(f"dropout: the skip must have x's shape and type, got {tuple(skip.shape)} of {skip.dtype}")
    x = x.contiguous()
    skip = None if skip is None else skip.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on(x.device):
        check(_lib.lib().sr355_dropout(x.data_ptr(), _ptr(skip), x.numel(), CODES[x.dtype], p, rng.data_ptr(), site,
                                       y.data_ptr(), _stream()), "sr355_dropout")
    return y


@dropout.register_fake
def _(x, skip, p, rng, site):
    return x.new_empty(x.shape)


# ------------------------------------------------------------------------------------
def _ffn_args(who: str, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: int) -> Tuple[FfnArgs, List]:
    """The common fields of an ``sr355_ffn_args`` record, and the tensors that have to outlive the call."""
    check_rows(who, x, w_gate, w_up, w_down)
    c = x.shape[-1]
    f = w_gate.shape[0] if w_gate.dim() == 2 else 0
    for name, w, shape in (("w_gate", w_gate, (f, c)), ("w_up", w_up, (f, c)), ("w_down", w_down, (c, f))):
        if w.dtype != x.dtype or w.shape != shape or f < 1:
            raise RuntimeError(f"{who}: {name} must have shape {shape} (at least one hidden channel) and x's type {x.dtype}, "
                               f"got {tuple(w.shape)} of {w.dtype}")
    if not 0 <= activation < len(ACTIVATIONS):
        raise RuntimeError(f"{who}: unknown activation {activation}")
    r, ld = as_rows(x)
    keep = [r, w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()]
    a = FfnArgs()
    a.dtype, a.activation, a.rows, a.channels, a.hidden = CODES[x.dtype], activation, x.numel() // c, c, f
    a.x_dev, a.x_ld = r.data_ptr(), ld
    a.w_gate_dev, a.w_up_dev, a.w_down_dev = keep[1].data_ptr(), keep[2].data_ptr(), keep[3].data_ptr()
    return a, keep


def _scratch(size: int, a: FfnArgs, who: str, device) -> Tensor:
    if size == 0:
        check(-1, who)
    return torch.empty(size, dtype=torch.uint8, device=device)


@torch.library.custom_op("sr355::gated_ffn_fwd", mutates_args=())
def gated_ffn_fwd(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, b_gate: Optional[Tensor],
                  b_up: Optional[Tensor], b_down: Optional[Tensor], activation: int,
                  want_saved: bool) -> Tuple[Tensor, Tensor]:
    """``(act(x w_gate' + b_gate) * (x w_up' + b_up)) w_down' + b_down``, and the bytes that the backward pass reads where
    ``want_saved`` (else an empty tensor)."""
    a, keep = _ffn_args("gated_ffn", x, w_gate, w_up, w_down, activation)
    check_rows("gated_ffn", x, b_gate, b_up, b_down)
    for name, b, n in (("b_gate", b_gate, a.hidden), ("b_up", b_up, a.hidden), ("b_down", b_down, a.channels)):
        if b is not None:
            keep.append(_vector("gated_ffn", name, b, n, (x.dtype,)))
            setattr(a, name + "_dev", keep[-1].data_ptr())
    L = _lib.lib()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    saved = torch.empty(L.sr355_gated_ffn_saved_bytes(C.byref(a)) if want_saved else 0, dtype=torch.uint8, device=x.device)
    a.y_dev = y.data_ptr()
    if want_saved:
        a.saved_dev, a.saved_bytes = saved.data_ptr(), saved.numel()
    ws = _scratch(L.sr355_gated_ffn_workspace_bytes(C.byref(a), 0), a, "sr355_gated_ffn_workspace_bytes", x.device)
    a.workspace_dev, a.workspace_bytes = ws.data_ptr(), ws.numel()
    with _on(x.device):
        check(L.sr355_gated_ffn_fwd(C.byref(a), _stream()), "sr355_gated_ffn_fwd")
    return y, saved


@gated_ffn_fwd.register_fake
def _(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, want_saved):
    a = FfnArgs()
    a.dtype, a.activation, a.rows, a.channels, a.hidden = CODES[x.dtype], activation, x.numel() // x.shape[-1], x.shape[-1], w_gate.shape[0]
    a.x_ld = a.channels
    size = _lib.lib().sr355_gated_ffn_saved_bytes(C.byref(a)) if want_saved else 0
    return x.new_empty(x.shape), x.new_empty((size,), dtype=torch.uint8)


@torch.library.custom_op("sr355::gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, saved: Tensor, activation: int,
                  need: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients of ``gated_ffn_fwd`` with respect to (x, w_gate, w_up, w_down, b_gate, b_up, b_down); an empty tensor
    where ``need`` says no."""
    a, keep = _ffn_args("gated_ffn backward", x, w_gate, w_up, w_down, activation)
    check_rows("gated_ffn backward", x, dy, saved)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise RuntimeError("gated_ffn backward: the gradient must have x's shape and type")
    g, ld = as_rows(dy)
    keep.append(g)
    a.dy_dev, a.dy_ld = g.data_ptr(), ld
    a.saved_dev, a.saved_bytes = (saved.data_ptr() if a.rows else None), saved.numel()
    shapes = (x.shape, w_gate.shape, w_up.shape, w_down.shape, (a.hidden,), (a.hidden,), (a.channels,))
    out = tuple(torch.empty(s if n else (0,), dtype=x.dtype, device=x.device) for s, n in zip(shapes, need))
    for name, t, n in zip(("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), out, need):
        if n and t.numel():
            setattr(a, name + "_dev", t.data_ptr())
    L = _lib.lib()
    ws = _scratch(L.sr355_gated_ffn_workspace_bytes(C.byref(a), 1), a, "sr355_gated_ffn_workspace_bytes", x.device)
    a.workspace_dev, a.workspace_bytes = ws.data_ptr(), ws.numel()
    with _on(x.device):
        check(L.sr355_gated_ffn_bwd(C.byref(a), _stream()), "sr355_gated_ffn_bwd")
    return out


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, saved, activation, need):
    f, c = w_gate.shape
    shapes = (x.shape, (f, c), (f, c), (c, f), (f,), (f,), (c,))
    return tuple(x.new_empty(s if n else (0,)) for s, n in zip(shapes, need))


layer_norm_fwd_now = now(layer_norm_fwd)
layer_norm_bwd_now = now(layer_norm_bwd)
dropout_now = now(dropout)
gated_ffn_fwd_now = now(gated_ffn_fwd)
gated_ffn_bwd_now = now(gated_ffn_bwd)
