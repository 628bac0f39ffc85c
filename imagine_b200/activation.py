"""Activations that keep their input in 8 bits for the backward pass.

``act_checkpoint_int8`` computes the activation and the checkpoint of its input
(int8 codes, one fp32 scale for every 128 elements of a row), ``act_backward_int8`` the
gradient from the checkpoint; ``checkpointed_activation`` is the two as one
differentiable operator.  The numeric steps run in libw8a8 (include/w8a8.h); there
is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _native as N
from .adapters import _on, _raw_stream, _rows, _same
from .linear import _code, _cuda

ACTIVATIONS = {"gelu_tanh": N.CKPT_GELU_TANH, "swiglu": N.CKPT_SWIGLU, "silu": N.CKPT_SILU}


def _act(act: str) -> tuple:
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}; one of {', '.join(sorted(ACTIVATIONS))}")
    return ACTIVATIONS[act], 2 if act == "swiglu" else 1


def _groups(k: int) -> int:
    return -(-k // N.CKPT_GROUP)


def act_checkpoint_int8(x: torch.Tensor, act: str = "gelu_tanh"):
    """``act(x)`` and the 8-bit checkpoint of x: ``(y [..., K], q int8, scale fp32)``.

    ``gelu_tanh`` and ``silu`` take x [..., K]; ``swiglu`` takes [..., 2K] rows
    ``[gate | up]`` and gives ``silu(gate) * up``.  Each half of a row is cut into
    groups of 128 (the last may be shorter): ``scale = max(amax / 127, 1e-30)``, ``q =
    round(x / scale)`` (half to even).  q has x's shape, scale [..., halves *
    ceil(K / 128)].  A group that holds an infinity or a NaN keeps NaN as its scale, and so
    gives NaN gradients."""
    code, halves = _act(act)
    dev = _cuda("x", x).device
    width = x.shape[-1]
    if width % halves:
        raise ValueError(f"swiglu rows are [gate | up]: {width} features do not halve")
    k = width // halves
    x2, ldx = _rows(x)
    lead, dtype = x.shape[:-1], x.dtype
    code_t = _code(dtype)
    whole = x2 is x  # contiguous: the results may be made like it
    y = torch.empty_like(x) if whole and halves == 1 else x.new_empty((*lead, k))
    q = torch.empty_like(x, dtype=torch.int8) if whole else x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty((*lead, halves * _groups(k)), dtype=torch.float32)
    with _on(dev):
        N.check(N.LIB.w8a8_act_checkpoint(x2.data_ptr(), code_t, ldx, math.prod(lead), k, code, y.data_ptr(),
                                          q.data_ptr(), scale.data_ptr(), _raw_stream(dev.index)))
    return y, q, scale


def act_backward_int8(dy: torch.Tensor, q: torch.Tensor, scale: torch.Tensor,
                      act: str = "gelu_tanh") -> torch.Tensor:
    """Gradient of ``act_checkpoint_int8``'s input from its checkpoint: ``dy *
    act'(q * scale)`` in dy's dtype, of q's shape."""
    code, halves = _act(act)
    dev = _cuda("dy", dy).device
    _same("q", q, dev)
    _same("scale", scale, dev)
    lead, k, dtype = dy.shape[:-1], dy.shape[-1], dy.dtype
    if q.dtype != torch.int8 or q.shape != (*lead, halves * k):
        raise ValueError(f"q must be int8 {(*lead, halves * k)}, got {tuple(q.shape)} of {q.dtype}")
    if scale.dtype != torch.float32 or scale.shape != (*lead, halves * _groups(k)):
        raise ValueError(f"scale must be fp32 {(*lead, halves * _groups(k))}, got "
                         f"{tuple(scale.shape)} of {scale.dtype}")
    code_t = _code(dtype)
    dy2, lddy = _rows(dy)
    if not q.is_contiguous():
        q = q.contiguous()
    if not scale.is_contiguous():
        scale = scale.contiguous()
    dx = torch.empty_like(q, dtype=dtype)
    with _on(dev):
        N.check(N.LIB.w8a8_act_backward(dy2.data_ptr(), code_t, lddy, math.prod(lead), k, code, q.data_ptr(),
                                        scale.data_ptr(), dx.data_ptr(), _raw_stream(dev.index)))
    return dx


class _Checkpointed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, act):
        y, q, scale = act_checkpoint_int8(x, act)
        ctx.act = act
        ctx.save_for_backward(q, scale)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return act_backward_int8(dy, *ctx.saved_tensors, ctx.act), None


def checkpointed_activation(x: torch.Tensor, act: str = "gelu_tanh") -> torch.Tensor:
    """``act(x)``, differentiable, keeping x for the backward pass as its 8-bit
    checkpoint (half of a bf16 input's bytes, and 1/32 of the codes' more for the scales).  A training
    step that is captured into a CUDA graph is captured whole, with no eager graph of the same
    leaves alive, as with any differentiable operator."""
    return _Checkpointed.apply(x, act)
