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
from .ops import _check_dtype, _ptr, _require, _require_cuda, _stream_ptr

Tensor = torch.Tensor

MAX_WIDTH = 16384
_TYPES = tuple(D.DTYPES)


def _rows(t: Tensor, width: int) -> Tensor:
    """``t [..., width]`` as ``[rows, width]`` with unit column stride: a view where the strides allow
    one (rows may be strided, or one row broadcast), a contiguous copy otherwise."""
    v = t if t.dim() == 2 else t.reshape(-1, width)
    return v if (v.stride(1) == 1 or width == 1) and v.stride(0) >= 0 else v.contiguous()


def _params(name: str, dtype: torch.dtype, width: int, **ps: Optional[Tensor]) -> torch.dtype:
    """The one type of the given ``[width]`` parameters (fp32 when there are none)."""
    found = None
    for k, t in ps.items():
        if t is None:
            continue
        _require(tuple(t.shape) == (width,), lambda: f"{name}: {k} must be [{width}], got {list(t.shape)}")
        _require(t.is_contiguous(), lambda: f"{name}: {k} must be contiguous")
        _check_dtype(name, t, (torch.float32, dtype), k)
        if found is not None and t.dtype != found:
            raise TypeError(f"{name}: the parameters must share one type")
        found = t.dtype
    return torch.float32 if found is None else found


def _width(name: str, x: Tensor) -> int:
    _require(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_WIDTH,
             lambda: f"{name}: the last dimension must be 1 to {MAX_WIDTH}, got {list(x.shape)}")
    return int(x.shape[-1])


def decoder_norm_forward(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                         eps: float = 1e-5, out: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(y, mean, rstd)``: ``y = (x - mean) * rstd * weight + bias`` over the last dimension of
    ``x [..., width]``, ``mean`` and ``rstd`` (fp32, ``[...]``) as ``decoder_norm_backward`` takes
    them.  ``out``: a contiguous tensor like ``x`` to write ``y`` into (it may be ``x`` itself)."""
    name = "decoder_norm_forward"
    dev = _require_cuda(name, x, weight, bias, out)
    _check_dtype(name, x, _TYPES, "x")
    width = _width(name, x)
    pt = _params(name, x.dtype, width, weight=weight, bias=bias)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    else:
        _check_dtype(name, out, (x.dtype,), "out")
        _require(out.shape == x.shape and out.is_contiguous(),
                 lambda: f"{name}: out must be a contiguous {list(x.shape)} tensor")
    v = _rows(x, width)
    rows = int(v.shape[0])
    stats = torch.empty((2,) + tuple(x.shape[:-1]), dtype=torch.float32, device=dev)
    mean, rstd = stats[0], stats[1]
    with D.on_device(dev):
        st = D.lib().s4d_norm_forward(v.data_ptr(), v.stride(0) if rows > 1 else width, D.DTYPES[x.dtype],
                                      _ptr(weight), _ptr(bias), D.DTYPES[pt], out.data_ptr(), width, mean.data_ptr(),
                                      rstd.data_ptr(), rows, width, float(eps), _stream_ptr(dev))
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
    dev = _require_cuda(name, dout, x, weight, mean, rstd)
    _check_dtype(name, x, _TYPES, "x")
    _check_dtype(name, dout, (x.dtype,), "dout")
    width = _width(name, x)
    _require(dout.shape == x.shape, lambda: f"{name}: dout must be {list(x.shape)}, got {list(dout.shape)}")
    pt = _params(name, x.dtype, width, weight=weight)
    if param_dtype is not None:
        _require(param_dtype in (torch.float32, x.dtype) and (weight is None or param_dtype == weight.dtype),
                 lambda: f"{name}: param_dtype must be the weight's type, torch.float32 or {x.dtype}")
        pt = param_dtype
    for k, t in (("mean", mean), ("rstd", rstd)):
        _check_dtype(name, t, (torch.float32,), k)
        _require(t.shape == x.shape[:-1] and t.is_contiguous(),
                 lambda: f"{name}: {k} must be a contiguous {list(x.shape[:-1])} tensor")
    v, g = _rows(x, width), _rows(dout, width)
    rows = int(v.shape[0])
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_dx else None
    dw = torch.empty(width, dtype=pt, device=dev) if need_dweight else None
    db = torch.empty(width, dtype=pt, device=dev) if need_dbias else None
    lib = D.lib()
    with D.on_device(dev):
        need = lib.s4d_norm_backward_workspace_bytes(rows, width) if need_dweight or need_dbias else 0
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        st = lib.s4d_norm_backward(g.data_ptr(), g.stride(0) if rows > 1 else width, v.data_ptr(),
                                   v.stride(0) if rows > 1 else width, D.DTYPES[x.dtype], _ptr(weight), D.DTYPES[pt],
                                   mean.data_ptr(), rstd.data_ptr(), _ptr(dx), width, _ptr(dw), _ptr(db), rows, width,
                                   _ptr(ws), need, _stream_ptr(dev))
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
