"""Operators on rows of channels ("tokens"): tensors ``[..., C]``, where the rows are an image's pixels or a sequence.

``layer_norm``, ``gated_ffn`` and ``dropout`` are HIP kernels, forward and backward, in bfloat16, float16 and float32, with
fp32 sums of a fixed order; ``FeedForwardBlock`` composes them into the channel-mixing half of a residual block,
``x + dropout(gated_ffn(layer_norm(x)))``.  They stand beside the conv core's 3x3 convs, BatchNorm and residual adds:
``rows_from_blocked`` and ``blocked_from_rows`` go between its blocked activations and rows.

Any sizes, leading dimensions and strides are taken; what is not laid out as rows of contiguous channels is copied first.
Widths that are multiples of 16 bytes are the fast ones.  All calls run on the current stream of their tensors' device, can
be captured into a graph, and keep nothing between calls.  A training call that is captured refuses leaves, its own and those
that its inputs were made from, that a live autograd graph of the default stream still holds: PyTorch would add their gradients
up there."""
from __future__ import annotations

import copy
from typing import Optional

import torch
import torch.distributed as dist
from torch import Tensor, nn
from torch.compiler import is_dynamo_compiling

from . import token_ops as ops


def _recorded(*tensors: Optional[Tensor]) -> bool:
    """Whether autograd records a call with these inputs."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# Each function asks the binding, which answers with nothing where PyTorch has to see an operator (a compiler that traces this code
# is told apart here): then the registered op is called.
def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x``.  ``weight`` and ``bias``, ``[C]``,
    are of x's type or float32 (both of one type), and so are their gradients.  A row of one channel or of equal channels
    gives ``bias`` (for ``eps`` > 0).  Statistics and sums are float32; the backward pass takes each row's mean rounded to it, so
    the gradients of float32 rows whose mean is some 10^4 times their deviation or more lose bits that ``y`` keeps."""
    if not is_dynamo_compiling():
        y = (ops._binding or ops.binding()).layer_norm(x, weight, bias, eps)
        if y is not None:
            return y
    return torch.ops.sr355.layer_norm_fwd(x, weight, bias, eps, _recorded(x, weight, bias))[0]


def dropout(x: Tensor, p: float, rng: Tensor, site: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """``x`` with each element dropped with probability ``p`` and the others divided by ``1 - p``, plus ``residual`` (x's
    shape and type) where one is given.  No mask is stored: which elements stay is a function of the element's index in
    ``x`` (row-major), the generator's state ``rng`` and ``site``, and the backward pass computes it again.

    ``rng`` is an int64 tensor of two words on x's device, a seed and a step (modulo 2^32).  Calls that share both take
    different ``site`` numbers or drop the same elements; a training loop advances the step.  The kernel reads ``rng`` when
    it runs, so a captured graph's replays drop what the words say then; changing them in place between a call and its
    backward pass is an error that autograd reports.  ``p`` counts in steps of 2^-16 and the scale is that of the nearest
    step; a dropped infinity or NaN is dropped."""
    if not is_dynamo_compiling():
        y = (ops._binding or ops.binding()).dropout(x, p, rng, site, residual)
        if y is not None:
            return y
    return torch.ops.sr355.dropout(x, residual, p, rng, site)


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, b_gate: Optional[Tensor] = None,
              b_up: Optional[Tensor] = None, b_down: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`` for rows ``x`` ``[..., C]``, ``w_gate`` and
    ``w_up`` ``[F, C]`` and ``w_down`` ``[C, F]`` (``nn.Linear`` weights), all of x's type.  ``activation``: "silu", "gelu"
    (by the error function), "relu" or "sigmoid".  A call that autograd records keeps eight bytes (float32: twelve) per
    hidden channel of every row of x.

    Products accumulate in fp32.  bfloat16 and float16 are rounded at these places beside the results: the hidden channels,
    once, between the two products (y is off by some 1.4 of one rounding); the gradients of the two projections, as operands of the
    products behind them (their bias gradients are summed before); act and the up projection times act', which the backward pass
    reads, are cut to 24 bits.  Calls of up to 64 rows whose rows * C * F is at most 2^19 hold the hidden channels with twice their
    bits, so y is rounded once there, and the same row may come out a step apart in a larger call; w_down's gradient takes them
    rounded in either case."""
    if activation not in ops.ACTIVATIONS:
        raise RuntimeError(f"gated_ffn: activation must be one of {', '.join(ops.ACTIVATIONS)}, got {activation!r}")
    if not is_dynamo_compiling():
        y = (ops._binding or ops.binding()).gated_ffn(x, w_gate, w_up, w_down, b_gate, b_up, b_down, ops.ACTIVATIONS[activation])
        if y is not None:
            return y
    return torch.ops.sr355.gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, ops.ACTIVATIONS[activation],
                                         _recorded(x, w_gate, w_up, w_down, b_gate, b_up, b_down))[0]


def rows_from_blocked(x: Tensor, channels: int) -> Tensor:
    """The conv core's blocked activations ``[N, H, units, W, c]`` as rows ``[N, H, W, channels]`` (a copy)."""
    if x.dim() != 5 or not 0 < channels <= x.shape[2] * x.shape[4]:
        raise RuntimeError(f"rows_from_blocked: expected blocked activations of at least {channels} channels, got {tuple(x.shape)}")
    N, H, U, W, c = x.shape
    return x.permute(0, 1, 3, 2, 4).reshape(N, H, W, U * c)[..., :channels]


def blocked_from_rows(x: Tensor) -> Tensor:
    """bfloat16 rows ``[N, H, W, C]`` as the conv core's blocked activations ``[N, H, units, W, 8]``, zeros behind C."""
    if x.dim() != 4 or x.dtype != torch.bfloat16:
        raise RuntimeError(f"blocked_from_rows: expected bfloat16 rows [N, H, W, C], got {tuple(x.shape)} of {x.dtype}")
    from .conv_core import units_for
    N, H, W, c = x.shape
    units = units_for(c)
    if units * 8 != c:
        x = nn.functional.pad(x, (0, units * 8 - c))
    return x.reshape(N, H, W, units, 8).permute(0, 1, 3, 2, 4).contiguous()


def _rank() -> int:
    return dist.get_rank() if dist.is_available() and dist.is_initialized() else 0


class FeedForwardBlock(nn.Module):
    """``x + dropout(gated_ffn(layer_norm(x)))`` on rows ``[..., channels]``: the channel-mixing half of a residual block.

    Parameters are float32; where x is bfloat16 or float16 the projections' are rounded to its type for the call (their
    gradients come back as float32) and the normalisation's are used as they are.  In training mode with ``dropout > 0``
    every call takes the seed and step of ``rng_state`` (a buffer that checkpoints carry; ``seed()`` sets it) and advances
    the step, on the device, so that replays of a captured graph do too.  A forward pass that is run again for its gradients
    (activation checkpointing) would take the next step and drop other elements: set ``rng_state`` back for it.

    Every block starts with a seed of its own, drawn from PyTorch's default generator (``torch.manual_seed`` makes it
    repeatable), and so does a ``deepcopy``, so stacked blocks drop different elements; blocks that are given one seed by
    ``seed()`` or one ``state_dict`` drop the same.  The rank in ``torch.distributed``'s default group is dropout's ``site``:
    replicas with equal seeds (DistributedDataParallel makes their buffers equal) drop different elements."""

    def __init__(self, channels: int, hidden: int, dropout: float = 0.0, activation: str = "silu", bias: bool = True,
                 eps: float = 1e-5):
        super().__init__()
        if channels < 1 or hidden < 1 or not 0.0 <= dropout <= 1.0 or activation not in ops.ACTIVATIONS:
            raise ValueError(f"FeedForwardBlock: channels={channels}, hidden={hidden}, dropout={dropout}, activation={activation!r}")
        self.channels, self.hidden, self.dropout, self.activation = channels, hidden, dropout, activation
        self.norm = nn.LayerNorm(channels, eps=eps)
        self.gate = nn.Linear(channels, hidden, bias=bias)
        self.up = nn.Linear(channels, hidden, bias=bias)
        self.down = nn.Linear(hidden, channels, bias=bias)
        self.register_buffer("rng_state", torch.zeros(2, dtype=torch.int64))
        self._draw_seed()

    def _draw_seed(self) -> None:
        with torch.no_grad():
            self.rng_state[:1].random_(-(1 << 62), 1 << 62)
            self.rng_state[1:].zero_()

    def __deepcopy__(self, memo):
        block = self.__class__.__new__(self.__class__)
        memo[id(self)] = block
        block.__dict__.update({k: copy.deepcopy(v, memo) for k, v in self.__dict__.items()})
        block._draw_seed()
        return block

    def seed(self, seed: int) -> None:
        """Start the dropout's generator at step 0 of ``seed``."""
        with torch.no_grad():
            self.rng_state.copy_(torch.tensor([seed, 0], dtype=torch.int64))

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() < 1 or x.shape[-1] != self.channels:
            raise RuntimeError(f"FeedForwardBlock: expected rows of {self.channels} channels, got {tuple(x.shape)}")

        def typed(t: Optional[Tensor]) -> Optional[Tensor]:
            return None if t is None else t.to(x.dtype)

        h = layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps)
        h = gated_ffn(h, typed(self.gate.weight), typed(self.up.weight), typed(self.down.weight), typed(self.gate.bias),
                      typed(self.up.bias), typed(self.down.bias), self.activation)
        if not self.training or self.dropout == 0.0:
            return x + h
        rng = self.rng_state.clone()          # what this call's backward pass reads, while the buffer moves on
        self.rng_state[1].add_(1)
        return dropout(h, self.dropout, rng, _rank(), x)
