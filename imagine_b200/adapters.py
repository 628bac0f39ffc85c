"""Low-rank adapters beside the W8A8 linears, and what training them needs.

``lora_add`` adds the adapters of many requests to one shared projection's
output; ``lora_backward`` gives their gradients, from the projection's input or
from the int8 codes the W8A8 linear made of it; ``int8_linear_backward`` is the
frozen linear's input gradient; ``int8_linear_lora`` puts the three together as
one differentiable operator.  The numeric steps run in libw8a8 through the C ABI
(include/w8a8.h), as in ``imagine_b200.linear``: there is no CPU path.

``lora_add``, ``lora_backward`` and ``int8_linear_backward`` do not record
themselves for autograd; ``int8_linear_lora`` does.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _native as N
from . import linear as L
from .linear import _code, _cuda, _vp


_NO_SWITCH = contextlib.nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on(dev: torch.device):
    """The device made current for the launch, where it is not already."""
    return _NO_SWITCH if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _same(name: str, t, dev: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.get_device() != dev.index:
        _cuda(name, t, dev)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> tuple:
    """``t`` as rows of its last dimension, unit stride, that do not overlap (itself
    or a view where its strides allow, else a copy), and the row stride."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, max(width, 1)
    m = math.prod(t.shape[:-1])
    t2 = t if t.dim() == 2 else t.reshape(m, width)
    if (t2.stride(1) != 1 and width > 1) or (m > 1 and t2.stride(0) < width):
        t2 = t2.contiguous()
    return t2, (t2.stride(0) if m > 1 else max(width, 1))


def _out_rows(name: str, t: torch.Tensor, shape, dtype, dev) -> int:
    """The row stride of an output, which has to be written in place."""
    _same(name, t, dev)
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
        raise ValueError(f"{name} must be {tuple(shape)} of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    if t.is_contiguous():
        return max(t.shape[-1], 1)
    m, width = math.prod(t.shape[:-1]), t.shape[-1]
    try:
        t2 = t.view(m, width)
    except RuntimeError as e:
        raise ValueError(f"{name} must have rows one stride apart") from e
    if (t2.stride(1) != 1 and width > 1) or (m > 1 and t2.stride(0) < width):
        raise ValueError(f"{name} must have unit-stride rows that do not overlap")
    return t2.stride(0) if m > 1 else max(width, 1)


def _adapters(a, b, k: int, n: int, dtype, dev) -> tuple:
    """The stacked adapters, checked: (a, its slot stride, b, its slot stride, S, R)."""
    _same("a", a, dev)
    _same("b", b, dev)
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("a must be [adapters, rank, K] and b [adapters, N, rank]")
    s, r, ka = a.shape
    if ka != k or b.shape != (s, n, r):
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit inputs of {k} and "
                         f"outputs of {n} features")
    if a.dtype != dtype or b.dtype != dtype:
        raise ValueError(f"a and b must be {dtype}, got {a.dtype} and {b.dtype}")
    if s < 1:
        raise ValueError("at least one adapter is needed")
    if not 1 <= r <= 128:
        raise ValueError(f"rank must be 1 to 128, got {r}")
    slot_a, slot_b = r * k, n * r
    # a slice of a larger stack is taken as it lies
    if not a.is_contiguous():
        if a.stride(2) == 1 and a.stride(1) == k and a.stride(0) >= slot_a:
            slot_a = a.stride(0)
        else:
            a = a.contiguous()
    if not b.is_contiguous():
        if b.stride(2) == 1 and b.stride(1) == r and b.stride(0) >= slot_b:
            slot_b = b.stride(0)
        else:
            b = b.contiguous()
    return a, slot_a, b, slot_b, s, r


def _index(adapter, lead, m: int, dev) -> tuple:
    """(index tensor or None, 1 for int64, rows per index).  ``adapter`` has the
    leading dimensions of the rows it covers: [B, S] for each token, [B] for each sample."""
    if adapter is None:
        return None, 0, 1
    _same("adapter", adapter, dev)
    if adapter.dtype != torch.int32 and adapter.dtype != torch.int64:
        raise ValueError(f"adapter must be int32 or int64, got {adapter.dtype}")
    if adapter.shape != lead[:adapter.dim()]:
        raise ValueError(f"adapter {tuple(adapter.shape)} must have the leading dimensions of {tuple(lead)}")
    if not adapter.is_contiguous():
        adapter = adapter.contiguous()
    return adapter, int(adapter.dtype == torch.int64), max(1, m // max(adapter.numel(), 1))


def _scaling(scaling, s: int, dev):
    if scaling is None:
        return None
    if isinstance(scaling, (int, float)):
        return torch.full((s,), float(scaling), dtype=torch.float32, device=dev)
    _same("scaling", scaling, dev)
    if scaling.numel() != s or scaling.dtype != torch.float32:
        raise ValueError(f"scaling must be fp32 with one value for each of {s} adapters, got "
                         f"{tuple(scaling.shape)} of {scaling.dtype}")
    return scaling if scaling.is_contiguous() else scaling.contiguous()


# Workspace sizes: functions of the shape and the device alone (current when they are asked for).
@functools.lru_cache(maxsize=4096)
def _lora_bytes(device: int, m: int, n: int, k: int, s: int, r: int, backward: int) -> int:
    nbytes = N.LIB.w8a8_lora_workspace_bytes(m, n, k, s, r, backward)
    N.check(nbytes if nbytes < 0 else 0)
    return nbytes


@functools.lru_cache(maxsize=4096)
def _input_grad_bytes(device: int, m: int, n: int, k: int, code: int) -> int:
    nbytes = N.LIB.w8a8_input_grad_workspace_bytes(m, n, k, code)
    N.check(nbytes if nbytes < 0 else 0)
    return nbytes


def _workspace(nbytes: int, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
             adapter: Optional[torch.Tensor] = None, scaling=None, *,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The low-rank adapters of a batch's requests, added to the output of the
    projection they share: ``out = y + scaling[s] * (x a[s]^T) b[s]^T``.

    ``y`` [..., N] is the projection's output for ``x`` [..., K], ``a`` [S, R, K]
    and ``b`` [S, N, R] the stacked adapters (R 1 to 128; smaller ones padded
    with zeros), all of one dtype (bf16, f16 or fp32).  ``adapter`` (int32 or int64)
    is each row's adapter and has x's leading dimensions or the first of them
    ([B] for [B, S, K]: one for each sample); an index outside [0, S), such as
    -1, means no adapter and returns y's row.  None: adapter 0 everywhere.
    ``scaling``: fp32 [S], or one number.  ``out`` may be ``y``, to add in place, and
    is no operand's memory otherwise.

    The contraction over K and the rank are summed in fp32 and the result is
    rounded once; the same call gives the same bits.  NaN and infinity stay in the rows (and
    adapters) that hold them, where an infinity gives an infinity or a NaN."""
    dev = _cuda("x", x).device
    _same("y", y, dev)
    shape, dtype = x.shape, x.dtype
    lead, k, n = shape[:-1], shape[-1], y.shape[-1]
    if y.shape[:-1] != lead:
        raise ValueError(f"x {tuple(shape)} and y {tuple(y.shape)} must have the same rows")
    if y.dtype != dtype:
        raise ValueError(f"x is {dtype} but y {y.dtype}")
    code = _code(dtype)
    a, slot_a, b, slot_b, s, r = _adapters(a, b, k, n, dtype, dev)
    y2, ldy = _rows(y)
    x2, ldx = _rows(x)
    m = math.prod(lead)
    idx, idx64, per = _index(adapter, lead, m, dev)
    c = _scaling(scaling, s, dev)
    given = out is not None
    if not given:
        out, ldo = (torch.empty_like(y) if y2 is y else y.new_empty(y.shape)), max(n, 1)
    else:
        ldo = _out_rows("out", out, y.shape, dtype, dev)
    with _on(dev):
        nbytes = _lora_bytes(dev.index, m, n, k, s, r, 0)
        ws = _workspace(nbytes, dev)
        N.check(N.LIB.w8a8_lora_add(
            y2.data_ptr(), ldy, x2.data_ptr(), ldx, code, a.data_ptr(), slot_a, b.data_ptr(), slot_b,
            _ptr(idx), idx64, per, _ptr(c), out.data_ptr(), ldo, m, n, k, s, r, _ptr(ws), nbytes,
            _raw_stream(dev.index)))
    if given:
        increment_version(out)  # a graph that saved it says so
    return out


def lora_backward(dy: torch.Tensor, x: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor,
                  adapter: Optional[torch.Tensor] = None, scaling=None, *,
                  x_scale: Optional[torch.Tensor] = None, dx: Optional[torch.Tensor] = None,
                  need_dx: bool = True, need_weights: bool = True):
    """Gradients of ``lora_add`` for ``dy`` [..., N]: ``(dx, da, db)``.

    ``dx = scaling[s] * (dy b[s]) a[s]`` (zero in rows without an adapter),
    ``da[s]`` and ``db[s]`` the sums over the rows of adapter s (zero without
    rows), all in dy's dtype.  ``x`` is the forward input, or with ``x_scale`` the
    int8 codes of ``quantize_int8_rowwise`` (its 8-bit checkpoint; one fp32 scale a
    row).  A given ``dx`` (the base linear's input gradient; no operand's memory) is added
    to, in place.
    ``need_dx`` / ``need_weights`` False: None in their place (x may then be None)."""
    dev = _cuda("dy", dy).device
    lead, n, k, dtype = dy.shape[:-1], dy.shape[-1], a.shape[-1], dy.dtype
    code = _code(dtype)
    a, slot_a, b, slot_b, s, r = _adapters(a, b, k, n, dtype, dev)
    dy2, lddy = _rows(dy)
    m = math.prod(lead)
    x2, ldx, xs = None, k, None
    if need_weights:
        _same("x", x, dev)
        if x.shape != (*lead, k):
            raise ValueError(f"x {tuple(x.shape)} does not fit dy {tuple(dy.shape)} and inputs of {k} features")
        if x.dtype != (dtype if x_scale is None else torch.int8):
            raise ValueError(f"x is {x.dtype}: int8 codes come with x_scale, anything else is dy's {dtype}")
        if x_scale is not None:
            _same("x_scale", x_scale, dev)
            if x_scale.dtype != torch.float32 or x_scale.numel() != m:
                raise ValueError(f"x_scale must be fp32 with one value for each of {m} rows")
            xs = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
        x2, ldx = _rows(x)
    idx, idx64, per = _index(adapter, lead, m, dev)
    c = _scaling(scaling, s, dev)
    lddx, accumulate = k, 0
    if not need_dx:
        dx = None
    elif dx is None:
        dx = dy.new_empty((*lead, k))
    else:
        lddx, accumulate = _out_rows("dx", dx, (*lead, k), dtype, dev), 1
    da = db = None
    if need_weights:
        da = torch.empty_like(a) if slot_a == r * k else dy.new_empty((s, r, k))
        db = torch.empty_like(b) if slot_b == n * r else dy.new_empty((s, n, r))
    with _on(dev):
        nbytes = _lora_bytes(dev.index, m, n, k, s, r, 1 if need_weights else 2)
        ws = _workspace(nbytes, dev)
        N.check(N.LIB.w8a8_lora_backward(
            dy2.data_ptr(), lddy, _ptr(x2), ldx, _ptr(xs), code, a.data_ptr(), slot_a, b.data_ptr(),
            slot_b, _ptr(idx), idx64, per, _ptr(c), _ptr(dx), lddx, accumulate, _ptr(da), _ptr(db), m,
            n, k, s, r, _ptr(ws), nbytes, _raw_stream(dev.index)))
    if accumulate:
        increment_version(dx)
    return dx, da, db


def int8_linear_backward(dy: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                         out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Input gradient of ``int8_linear``: ``dx = dy (weight_scale * weight)`` for
    ``dy`` [..., N] and the int8 ``weight`` [N, K] with its scales (N or 1), dx
    [..., K] in dy's dtype.  The quantisation of the input passes the gradient through
    unchanged (the straight-through estimate).

    Products are summed in fp32 and the result is rounded once.  fp32 and f16 keep their
    own precision in between; bf16 takes the weight as dequantised to bf16 (off by 2^-8 of itself
    at most), or, where one scale serves the whole weight, as its exact codes."""
    dev = _cuda("dy", dy).device
    _same("weight", weight, dev)
    if weight.dim() != 2 or weight.dtype != torch.int8:
        raise ValueError("weight must be a 2-D int8 tensor [N, K]")
    if out_dtype not in (None, dy.dtype):
        raise ValueError(f"the gradient of {dy.dtype} is {dy.dtype}, not {out_dtype}")
    n, k = weight.shape
    if dy.shape[-1] != n:
        raise ValueError(f"dy has {dy.shape[-1]} features, the weight {n} outputs")
    ws = weight_scale
    if ws.get_device() != dev.index or ws.dtype != torch.float32 or not ws.is_contiguous():
        ws = ws.to(device=dev, dtype=torch.float32).contiguous()
    if ws.numel() != n and ws.numel() != 1:
        raise ValueError(f"INT8 weight scale must be scalar or per-output-channel, got "
                         f"{tuple(weight_scale.shape)} for weight shape {tuple(weight.shape)}")
    code = _code(dy.dtype)
    dy2, lddy = _rows(dy)
    w2, ldw = _rows(weight)
    lead = dy.shape[:-1]
    m = math.prod(lead)
    dx = dy.new_empty((*lead, k))
    with _on(dev):
        nbytes = _input_grad_bytes(dev.index, m, n, k, code)
        work = _workspace(nbytes, dev)
        N.check(N.LIB.w8a8_input_grad(
            dy2.data_ptr(), lddy, w2.data_ptr(), ldw, ws.data_ptr(), ws.numel(), code, dx.data_ptr(),
            max(k, 1), m, n, k, _ptr(work), nbytes, _raw_stream(dev.index)))
    return dx


class _Int8LinearLora(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, weight_scale, bias, a, b, adapter, scaling, keep_input):
        dev = x.device
        n, k = weight.shape
        ws = weight_scale.to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
        m = math.prod(x.shape[:-1])
        x2 = _rows(x)[0].reshape(m, k)
        w = weight if weight.is_contiguous() else weight.contiguous()
        q, xs = L.quantize_int8_rowwise(x2)
        bias = None if bias is None else bias.to(device=dev, dtype=x.dtype).reshape(-1).contiguous()
        if bias is not None and bias.numel() != n:
            raise ValueError(f"bias has {bias.numel()} elements for {n} outputs")
        y = torch.empty((m, n), dtype=x.dtype, device=dev)
        ep = L._epilogue(ws, bias, None, None, "eager", None, n, n)
        stream = L._stream(dev)
        if 1 <= m <= 2:
            N.check(N.LIB.w8a8_gemv_dequant(_vp(q), _vp(w), _vp(xs), ctypes.byref(ep), _vp(y),
                                            _code(x.dtype), m, n, k, stream))
        elif m > 0:
            # the linear's split-K scratch belongs to a stream, and a graph may be replayed
            # on any: captured, tiles run whole (the same bits)
            split = 1 if torch.cuda.is_current_stream_capturing() else None
            L._gemm_dequant(q, w, xs.reshape(-1), ep, y, x.dtype, m, n, k, None, split, stream)
        y = y.reshape(*x.shape[:-1], n)
        lora_add(y, x, a, b, adapter, scaling, out=y)
        kept = (x, None) if keep_input else (q.reshape(x.shape), xs)
        ctx.save_for_backward(*kept, w, ws, a, b, adapter, scaling)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, xs, w, ws, a, b, adapter, scaling = ctx.saved_tensors
        need_x, need_a, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[4], ctx.needs_input_grad[5]
        with _on(dy.device):
            dx = int8_linear_backward(dy, w, ws) if need_x else None
            da = db = None
            if need_x or need_a or need_b:
                dx, da, db = lora_backward(dy, x, a, b, adapter, scaling, x_scale=xs, dx=dx,
                                           need_dx=need_x, need_weights=need_a or need_b)
        return (dx, None, None, None, da if need_a else None, db if need_b else None, None, None, None)


def int8_linear_lora(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                     bias: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor,
                     adapter: Optional[torch.Tensor] = None, scaling=None, *,
                     keep_input: bool = False) -> torch.Tensor:
    """``lora_add(int8_linear(x, weight, weight_scale, bias), x, a, b, adapter,
    scaling)`` with gradients for x, a and b (the int8 weight, its scales and the
    bias are frozen).  The linear is the plain one, [N, K] codes with N scales or one: no ConvRot
    weight, input or output activation, or residual.

    For the backward pass it keeps the int8 codes that the linear made of x
    (half of a bf16 input's bytes), from which da and db are taken; with ``keep_input`` it
    keeps x itself instead.  Operands as in the two operators.  A training step that is
    captured into a CUDA graph is captured whole, with no eager graph of the same leaves
    alive (autograd's accumulation would run on the eager graph's stream)."""
    dev = _cuda("x", x).device
    with _on(dev):
        _cuda("weight", weight, dev)
        if weight.dim() != 2 or weight.dtype != torch.int8:
            raise ValueError("weight must be a 2-D int8 tensor [N, K]")
        n, k = weight.shape
        if x.shape[-1] != k:
            raise ValueError(f"Input and weight inner dimensions must match, got {x.shape[-1]} and {k}")
        if k == 0:
            raise ValueError("int8_linear_lora needs K > 0")
        if weight_scale.numel() not in (1, n):
            raise ValueError(f"INT8 weight scale must be scalar or per-output-channel, got "
                             f"{tuple(weight_scale.shape)} for weight shape {tuple(weight.shape)}")
        _code(x.dtype)
        for name, t in (("weight_scale", weight_scale), ("bias", bias), ("scaling", scaling)):
            if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"{name} is frozen in int8_linear_lora: detach it")
        _adapters(a, b, k, n, x.dtype, dev)
        scaling = _scaling(scaling, a.shape[0], dev)
        return _Int8LinearLora.apply(x, weight, weight_scale, bias, a, b, adapter, scaling, keep_input)
