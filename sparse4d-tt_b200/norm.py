"""LayerNorm with gradients (``s4d_norm_forward`` / ``s4d_norm_backward``), for training the decoder
layers around the DFA: the forward-only ``ops.layer_norm`` stays the decoder's inference kernel.

* ``decoder_norm(x, weight, bias, eps)`` -- differentiable, like ``F.layer_norm`` over the last
  dimension.
* ``decoder_norm_forward`` / ``decoder_norm_backward`` -- the two passes by themselves, for
  programs that keep their own buffers (no autograd; capturable in a CUDA graph).

fp32, bf16 or fp16 rows of 1 to 16384 features; ``weight`` and ``bias`` in fp32 or in the rows' type.
Statistics and arithmetic are fp32.  There is no CPU path: CPU tensors are rejected.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib_decoder as D

Tensor = torch.Tensor

MAX_WIDTH = 16384


def _rows(t: Tensor, width: int) -> Tuple[Tensor, int]:
    """``t [..., width]`` and the stride of its rows: ``t`` itself or a view where the strides allow it (rows
    may be strided, or one row broadcast), a contiguous copy otherwise."""
    t = D.in_memory(t)
    if t.is_contiguous():
        return t, width
    v = t if t.dim() == 2 else t.reshape(-1, width)
    if (v.stride(1) != 1 and width != 1) or v.stride(0) < 0:
        v = v.contiguous()
    return v, (v.stride(0) if v.shape[0] > 1 else width)


def _param(name: str, what: str, t: Tensor, dtype: torch.dtype, width: int) -> torch.dtype:
    if t.shape != (width,) or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be a contiguous [{width}] tensor, got {list(t.shape)}")
    if t.dtype != torch.float32 and t.dtype != dtype:
        raise TypeError(f"{name}: {what} must be torch.float32 or {dtype}, got {t.dtype}")
    return t.dtype


def _width(name: str, x: Tensor) -> int:
    if x.dtype not in D.DTYPES:
        raise TypeError(f"{name}: x must be one of {list(D.DTYPES)}, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{name}: the last dimension must be 1 to {MAX_WIDTH}, got {list(x.shape)}")
    return x.shape[-1]


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def decoder_norm_forward(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                         eps: float = 1e-5, out: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(y, mean, rstd)``: ``y = (x - mean) * rstd * weight + bias`` over the last dimension of
    ``x [..., width]``, ``mean`` and ``rstd`` (fp32, ``[...]``) as ``decoder_norm_backward`` takes
    them.  ``out``: a contiguous tensor like ``x`` to write ``y`` into (it may be ``x`` itself)."""
    name = "decoder_norm_forward"
    if out is None:
        done = D.calls().norm_forward(x, weight, bias, eps)
        if done is not None:
            return done
    index = D.same_device(name, x, weight, bias, out)
    weight, bias = D.in_memory(weight), D.in_memory(bias)
    width, dtype = _width(name, x), x.dtype
    pt = torch.float32 if weight is None else _param(name, "weight", weight, dtype, width)
    if bias is not None:
        bt = _param(name, "bias", bias, dtype, width)
        if weight is not None and bt != pt:
            raise TypeError(f"{name}: weight and bias must share one type")
        pt = bt
    shape = x.shape
    if out is None:
        out = x.new_empty(shape)
    elif out.dtype != dtype:
        raise TypeError(f"{name}: out must be {dtype}, got {out.dtype}")
    elif out.shape != shape or not out.is_contiguous() or out.is_neg():
        raise ValueError(f"{name}: out must be a contiguous {list(shape)} tensor")
    elif (D.overlap(out, x) and (out.data_ptr() != x.data_ptr() or not x.is_contiguous())) or any(
            t is not None and D.overlap(out, t) for t in (weight, bias)):
        raise ValueError(f"{name}: out must be x itself or share no memory with the arguments")
    v, ld = _rows(x, width)
    stats = shape[:-1]
    mean, rstd = x.new_empty(stats, dtype=torch.float32), x.new_empty(stats, dtype=torch.float32)
    with D.on_device(index):
        st = D.lib().s4d_norm_forward(v.data_ptr(), ld, D.DTYPES[dtype], _ptr(weight), _ptr(bias), D.DTYPES[pt],
                                      out.data_ptr(), width, mean.data_ptr(), rstd.data_ptr(), x.numel() // width,
                                      width, eps, D.stream_ptr(index))
    if st:
        D.check(name, st)
    return out, mean, rstd


def decoder_norm_backward(dout: Tensor, x: Tensor, weight: Optional[Tensor], mean: Tensor, rstd: Tensor,
                          need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True,
                          param_dtype: Optional[torch.dtype] = None
                          ) -> Tuple[Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """``(dx, dweight, dbias)`` of ``decoder_norm_forward`` from its output's gradient ``dout`` (like
    ``x``), its input, weight, ``mean`` and ``rstd``; None for each that is not needed.  ``dweight``
    and ``dbias`` are ``[width]`` in ``param_dtype`` (the weight's type, or fp32 without a weight),
    summed over all rows in fp32 in an order that depends on the sizes alone."""
    name = "decoder_norm_backward"
    if param_dtype is None or (weight is not None and param_dtype == weight.dtype):
        done = D.calls().norm_backward(dout, x, weight, mean, rstd, need_dx, need_dweight, need_dbias)
        if done is not None:
            return done
    index = D.same_device(name, x, dout, weight, mean, rstd)
    weight, mean, rstd = D.in_memory(weight), D.in_memory(mean), D.in_memory(rstd)
    width, dtype, shape = _width(name, x), x.dtype, x.shape
    if dout.dtype != dtype:
        raise TypeError(f"{name}: dout must be {dtype}, got {dout.dtype}")
    if dout.shape != shape:
        raise ValueError(f"{name}: dout must be {list(shape)}, got {list(dout.shape)}")
    pt = torch.float32 if weight is None else _param(name, "weight", weight, dtype, width)
    if param_dtype is not None:
        if param_dtype not in (torch.float32, dtype) or (weight is not None and param_dtype != pt):
            raise ValueError(f"{name}: param_dtype must be the weight's type, torch.float32 or {dtype}")
        pt = param_dtype
    if mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise TypeError(f"{name}: mean and rstd must be torch.float32")
    stats = shape[:-1]
    if mean.shape != stats or rstd.shape != stats or not mean.is_contiguous() or not rstd.is_contiguous():
        raise ValueError(f"{name}: mean and rstd must be contiguous {list(stats)} tensors")
    (v, ld), (g, gld) = _rows(x, width), _rows(dout, width)
    rows = x.numel() // width
    dx = x.new_empty(shape) if need_dx else None
    dw = x.new_empty(width, dtype=pt) if need_dweight else None
    db = x.new_empty(width, dtype=pt) if need_dbias else None
    lib = D.lib()
    with D.on_device(index):
        need = lib.s4d_norm_backward_workspace_bytes(rows, width) if need_dweight or need_dbias else 0
        ws = x.new_empty(need // 4, dtype=torch.float32) if need else None
        st = lib.s4d_norm_backward(g.data_ptr(), gld, v.data_ptr(), ld, D.DTYPES[dtype], _ptr(weight), D.DTYPES[pt],
                                   mean.data_ptr(), rstd.data_ptr(), _ptr(dx), width, _ptr(dw), _ptr(db), rows, width,
                                   _ptr(ws), need, D.stream_ptr(index))
    if st:
        D.check(name, st)
    return dx, dw, db


class _DecoderNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = decoder_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.param_dtype = next((t.dtype for t in (weight, bias) if t is not None), None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*decoder_norm_backward(dout, x, weight, mean, rstd, need[0], need[1], need[2], ctx.param_dtype), None)


def decoder_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                 eps: float = 1e-5) -> Tensor:
    """Differentiable LayerNorm over the last dimension of ``x [..., width]``
    (``F.layer_norm(x, (width,), weight, bias, eps)``), first derivatives only."""
    return _DecoderNorm.apply(x, weight, bias, eps)
