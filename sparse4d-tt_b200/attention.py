"""Attention of the decoder's instances with capped, biased and masked scores (``s4d_attention_*`` of
``include/s4d_decoder.h``), on the tensor cores.

For head h, query i and key j::

    x = scale q_i.k_j                     scale = dim ** -0.5 unless given
    z = softcap tanh(x / softcap)         (x when softcap is 0)
    s = z - slopes_h |q_pos_i - k_pos_j|  positions in 1 or 2 coordinates; slopes per head, or per
                                          query and head
    seen: j < k_len[b]  and  q_segment_i == k_segment_j >= 0
    out_i = sum over the seen keys of softmax(s)_j v_j; 0 for a query that sees none

The distance bias is the decoder's ground-plane distance between instances (or the distance along a
sequence), the segments its denoising groups (or packed documents; a negative id is padding), and
``k_len`` the frames' own numbers of valid cached instances.  bf16 or fp16, 8 to 128 features a
head, ``kv_heads`` that divide ``heads``, any number of queries from one to many: few queries over
many keys are split along the keys.

* ``decoder_attention`` -- differentiable in q, k, v and the slopes (bf16).
* ``decoder_attention_forward`` / ``decoder_attention_backward`` -- the two passes by themselves, for
  programs that keep their own buffers (no autograd; capturable in a CUDA graph).

There is no CPU path: CPU tensors are rejected.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib as L
from . import _lib_decoder as D
from .ops import _check_dtype, _ptr, _require, _require_cuda, _stream_ptr

Tensor = torch.Tensor

_TYPES = (torch.bfloat16, torch.float16)


def _operand(t: Tensor) -> Tensor:
    """``t [B, N, heads, dim]`` with strides the kernels read in place (unit stride along dim, the others
    positive multiples of 8, 16-byte aligned); a contiguous copy otherwise (an expanded tensor, for
    one)."""
    s = t.stride()
    if s[3] == 1 and t.data_ptr() % 16 == 0:
        for i in (0, 1, 2):
            if t.shape[i] > 1 and (s[i] <= 0 or s[i] % 8):
                break
        else:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _fill(name: str, q: Tensor, k: Tensor, v: Tensor, scale: Optional[float], softcap: float,
          slopes: Optional[Tensor], q_pos: Optional[Tensor], k_pos: Optional[Tensor], q_segment: Optional[Tensor],
          k_segment: Optional[Tensor], k_len: Optional[Tensor], error_flag: Optional[Tensor]):
    """The checked arguments of a call: ``(device, AttentionArgs)``; the tensors they point to are kept
    in the struct's ``keep``."""
    dev = _require_cuda(name, q, k, v, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    for what, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype not in _TYPES or t.dtype != q.dtype:
            raise TypeError(f"{name}: q, k and v must share one of {list(_TYPES)}, {what} is {t.dtype}")
        if t.dim() != 4:
            raise ValueError(f"{name}: {what} must be [batch, rows, heads, dim], got {list(t.shape)}")
    B, nq, H, dim = q.shape
    nk, G = int(k.shape[1]), int(k.shape[2])
    if k.shape != (B, nk, G, dim) or v.shape != k.shape:
        raise ValueError(f"{name}: k and v must be [{B}, keys, kv_heads, {dim}], got {list(k.shape)} and "
                         f"{list(v.shape)}")
    if G == 0 or H % G:
        raise ValueError(f"{name}: the {H} heads must be a multiple of the {G} kv_heads")
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"{name}: dim must be a multiple of 8 from 8 to 128, got {dim}")
    a = D.AttentionArgs()
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim = B, nq, nk, H, G, dim
    a.dtype = D.DTYPES[q.dtype]
    q, k, v = _operand(q), _operand(k), _operand(v)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    a.scale = dim ** -0.5 if scale is None else float(scale)
    a.softcap = float(softcap)
    keep = [q, k, v]
    if (slopes is None) != (q_pos is None) or (q_pos is None) != (k_pos is None):
        raise ValueError(f"{name}: slopes, q_pos and k_pos go together")
    if slopes is not None:
        _check_dtype(name, slopes, (torch.float32,), "slopes")
        _check_dtype(name, q_pos, (torch.float32,), "q_pos")
        _check_dtype(name, k_pos, (torch.float32,), "k_pos")
        pos = int(q_pos.shape[-1]) if q_pos.dim() == 3 else 0
        _require(pos in (1, 2) and tuple(q_pos.shape) == (B, nq, pos) and tuple(k_pos.shape) == (B, nk, pos),
                 lambda: f"{name}: q_pos and k_pos must be [{B}, {nq} / {nk}, 1 or 2], got {list(q_pos.shape)} and "
                         f"{list(k_pos.shape)}")
        if tuple(slopes.shape) == (H,):
            a.slope_stride[:] = (0, 0, slopes.stride(0))
        else:
            _require(tuple(slopes.shape) == (B, nq, H),
                     lambda: f"{name}: slopes must be [{H}] or [{B}, {nq}, {H}], got {list(slopes.shape)}")
            a.slope_stride[:] = slopes.stride()
        q_pos, k_pos = q_pos.contiguous(), k_pos.contiguous()
        a.pos_dim, a.slopes, a.q_pos, a.k_pos = pos, slopes.data_ptr(), q_pos.data_ptr(), k_pos.data_ptr()
        keep += [slopes, q_pos, k_pos]
    if (q_segment is None) != (k_segment is None):
        raise ValueError(f"{name}: q_segment and k_segment go together")
    if q_segment is not None:
        _check_dtype(name, q_segment, (torch.int32,), "q_segment")
        _check_dtype(name, k_segment, (torch.int32,), "k_segment")
        _require(tuple(q_segment.shape) == (B, nq) and tuple(k_segment.shape) == (B, nk),
                 lambda: f"{name}: q_segment and k_segment must be [{B}, {nq}] and [{B}, {nk}]")
        q_segment, k_segment = q_segment.contiguous(), k_segment.contiguous()
        a.q_segment, a.k_segment = q_segment.data_ptr(), k_segment.data_ptr()
        keep += [q_segment, k_segment]
    if k_len is not None:
        _check_dtype(name, k_len, (torch.int32,), "k_len")
        _require(tuple(k_len.shape) == (B,), lambda: f"{name}: k_len must be [{B}], got {list(k_len.shape)}")
        k_len = k_len.contiguous()
        a.k_len = k_len.data_ptr()
        keep.append(k_len)
    if error_flag is not None:
        _check_dtype(name, error_flag, (torch.int32,), "error_flag")
        a.error_flag = error_flag.data_ptr()
    a.keep = keep
    return dev, a


def decoder_attention_forward(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None, softcap: float = 0.0,
                              slopes: Optional[Tensor] = None, q_pos: Optional[Tensor] = None,
                              k_pos: Optional[Tensor] = None, q_segment: Optional[Tensor] = None,
                              k_segment: Optional[Tensor] = None, k_len: Optional[Tensor] = None,
                              out: Optional[Tensor] = None, error_flag: Optional[Tensor] = None
                              ) -> Tuple[Tensor, Tensor]:
    """``(out, lse)`` of ``q [B, Nq, H, dim]`` over ``k``, ``v`` ``[B, Nk, G, dim]``: ``out`` like ``q``
    (contiguous), ``lse [B, H, Nq]`` fp32, the log-sum-exp of each row's seen scores (-inf without any),
    which ``decoder_attention_backward`` takes.

    ``slopes [H]`` or ``[B, Nq, H]`` fp32 with ``q_pos [B, Nq, 1 or 2]`` and ``k_pos [B, Nk, 1 or 2]``
    fp32 give the distance bias; ``q_segment [B, Nq]`` and ``k_segment [B, Nk]`` int32 the document
    mask; ``k_len [B]`` int32 the valid keys of each batch entry (read on the device, clamped to
    0 .. Nk).  ``out``: a contiguous tensor like ``q`` to write into."""
    name = "decoder_attention_forward"
    dev, a = _fill(name, q, k, v, scale, softcap, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _require_cuda(name, q, out)
        _check_dtype(name, out, (q.dtype,), "out")
        _require(out.shape == q.shape and out.is_contiguous() and out.data_ptr() % 16 == 0,
                 lambda: f"{name}: out must be a contiguous, 16-byte aligned {list(q.shape)} tensor")
    lse = torch.empty(a.batch, a.heads, a.queries, dtype=torch.float32, device=dev)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    lib = D.lib()
    with D.on_device(dev):
        need = lib.s4d_attention_forward_workspace_bytes(C.byref(a))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a.workspace, a.workspace_bytes = _ptr(ws), need
        st = lib.s4d_attention_forward(C.byref(a), _stream_ptr(dev))
    D.check(name, st)
    return out, lse


def decoder_attention_backward(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor,
                               scale: Optional[float] = None, softcap: float = 0.0, slopes: Optional[Tensor] = None,
                               q_pos: Optional[Tensor] = None, k_pos: Optional[Tensor] = None,
                               q_segment: Optional[Tensor] = None, k_segment: Optional[Tensor] = None,
                               k_len: Optional[Tensor] = None, need_dkv: bool = True, need_dslopes: bool = True,
                               error_flag: Optional[Tensor] = None
                               ) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """``(dq, dk, dv, dslopes)`` of ``decoder_attention_forward`` from its output's gradient ``dout`` (like
    ``q``), its arguments and its results, in bf16 (``dslopes`` fp32, like ``slopes``; None without them).
    ``need_dkv`` / ``need_dslopes`` False leave those out (None).  Positions have no gradient.  No
    atomics: equal calls give equal bits."""
    name = "decoder_attention_backward"
    dev, a = _fill(name, q, k, v, scale, softcap, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    _require_cuda(name, q, dout, out, lse)
    _check_dtype(name, q, (torch.bfloat16,), "q")
    for what, t in (("dout", dout), ("out", out)):
        _check_dtype(name, t, (q.dtype,), what)
        _require(t.shape == q.shape, lambda: f"{name}: {what} must be {list(q.shape)}, got {list(t.shape)}")
    _require(out.is_contiguous() and out.data_ptr() % 16 == 0, lambda: f"{name}: out must be contiguous")
    _check_dtype(name, lse, (torch.float32,), "lse")
    _require(tuple(lse.shape) == (a.batch, a.heads, a.queries) and lse.is_contiguous(),
             lambda: f"{name}: lse must be a contiguous [{a.batch}, {a.heads}, {a.queries}] tensor")
    dout = _operand(dout)
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
    dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=dev) if need_dkv else None for _ in range(2))
    ds = torch.empty(slopes.shape, dtype=torch.float32, device=dev) if slopes is not None and need_dslopes else None
    a.out, a.lse, a.dout, a.dq, a.dk, a.dv, a.dslopes = (out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(),
                                                         _ptr(dk), _ptr(dv), _ptr(ds))
    a.dout_stride[:] = dout.stride()[:3]
    a.dslopes_per_row = int(ds is not None and ds.dim() == 3)
    if a.batch == 0:
        if ds is not None:
            ds.zero_()
        return dq, dk, dv, ds
    lib = D.lib()
    with D.on_device(dev):
        need = lib.s4d_attention_backward_workspace_bytes(C.byref(a))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a.workspace, a.workspace_bytes = _ptr(ws), need
        st = lib.s4d_attention_backward(C.byref(a), _stream_ptr(dev))
    D.check(name, st)
    return dq, dk, dv, ds


class _DecoderAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, scale, softcap, q_pos, k_pos, q_segment, k_segment, k_len):
        rest = (q_pos, k_pos, q_segment, k_segment, k_len)
        out, lse = decoder_attention_forward(q, k, v, scale, softcap, slopes, *rest)
        ctx.save_for_backward(q, k, v, out, lse, slopes, *rest)
        ctx.scale, ctx.softcap = scale, softcap
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, slopes, *rest = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, ds = decoder_attention_backward(dout, q, k, v, out, lse, ctx.scale, ctx.softcap, slopes, *rest,
                                                    need_dkv=need[1] or need[2], need_dslopes=need[3])
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, ds, *([None] * 7))


def decoder_attention(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None, softcap: float = 0.0,
                      slopes: Optional[Tensor] = None, q_pos: Optional[Tensor] = None, k_pos: Optional[Tensor] = None,
                      q_segment: Optional[Tensor] = None, k_segment: Optional[Tensor] = None,
                      k_len: Optional[Tensor] = None) -> Tensor:
    """``out`` of ``decoder_attention_forward``, differentiable (first derivatives) in ``q``, ``k``, ``v`` and
    ``slopes``.  Gradients are for bf16: fp16 inputs that require one are rejected (dS of a long row lies
    in fp16's subnormal range), and so are positions that require one."""
    name = "decoder_attention"
    if torch.is_grad_enabled():
        for what, t in (("q_pos", q_pos), ("k_pos", k_pos)):
            _require(t is None or not t.requires_grad, lambda: f"{name}: {what} has no gradient; detach it")
        if q.dtype != torch.bfloat16 and any(t is not None and t.requires_grad for t in (q, k, v, slopes)):
            raise TypeError(f"{name}: gradients are implemented for torch.bfloat16, got {q.dtype}")
    return _DecoderAttention.apply(q, k, v, slopes, scale, softcap, q_pos, k_pos, q_segment, k_segment, k_len)
