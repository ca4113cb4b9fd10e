"""Attention of the decoder's instances with capped, biased and masked scores (``s4d_attention_*`` of
``include/s4d_decoder.h``), on the tensor cores.

For head h, query i and key j::

    x = scale q_i.k_j                     scale = dim ** -0.5 unless given
    z = softcap tanh(x / softcap)         (x when softcap is 0; at most 1024)
    s = z - slopes_h |q_pos_i - k_pos_j|  positions in 1 or 2 coordinates (with 2, differences below 2^63);
                                          slopes per head, or per query and head
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
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib_decoder as D

Tensor = torch.Tensor

_ZERO3 = (0, 0, 0)


def _operand(t: Tensor) -> Tuple[Tensor, Tuple[int, ...]]:
    """``t [B, N, heads, dim]`` and its strides, such that the kernels can read it in place (unit stride along
    dim, the others positive multiples of 8, 16-byte aligned); a contiguous copy where ``t`` is not
    (an expanded tensor, for one)."""
    t = D.in_memory(t)
    sb, sn, sh, sd = t.stride()
    b, n, h, _ = t.shape
    if (sd == 1 and t.data_ptr() % 16 == 0 and (b <= 1 or (sb > 0 and sb % 8 == 0))
            and (n <= 1 or (sn > 0 and sn % 8 == 0)) and (h <= 1 or (sh > 0 and sh % 8 == 0))):
        return t, (sb, sn, sh)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()[:3]


class _Args(NamedTuple):
    """The checked arguments of a call, in the order of ``s4d_attention_args``."""

    index: int        # CUDA device
    sizes: tuple      # batch, queries, keys, heads, kv_heads, dim, pos_dim
    operands: tuple   # q, k, v pointers and strides
    slopes: tuple     # pointer, strides
    optional: tuple   # q_pos, k_pos, q_segment, k_segment, k_len
    error_flag: int
    scalars: tuple    # scale, softcap, dtype
    keep: tuple       # the tensors pointed to that are copies


def _checked(name: str, q: Tensor, k: Tensor, v: Tensor, scale: Optional[float], softcap: float,
             slopes: Optional[Tensor], q_pos: Optional[Tensor], k_pos: Optional[Tensor], q_segment: Optional[Tensor],
             k_segment: Optional[Tensor], k_len: Optional[Tensor], error_flag: Optional[Tensor]) -> _Args:
    index = D.same_device(name, q, k, v, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    dtype = q.dtype
    if dtype not in (torch.bfloat16, torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"{name}: q, k and v must share one of [torch.bfloat16, torch.float16], got {dtype}, {k.dtype} "
                        f"and {v.dtype}")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{name}: q, k and v must be [batch, rows, heads, dim], got {list(q.shape)}, {list(k.shape)} "
                         f"and {list(v.shape)}")
    B, nq, H, dim = q.shape
    kb, nk, G, kd = k.shape
    if kb != B or kd != dim or v.shape != k.shape:
        raise ValueError(f"{name}: k and v must be [{B}, keys, kv_heads, {dim}], got {list(k.shape)} and "
                         f"{list(v.shape)}")
    if G == 0 or H % G:
        raise ValueError(f"{name}: the {H} heads must be a multiple of the {G} kv_heads")
    if softcap and C.c_float(softcap).value == 0.0:
        raise ValueError(f"{name}: softcap {softcap} is 0 in fp32, which would be no cap")
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"{name}: dim must be a multiple of 8 from 8 to 128, got {dim}")
    (q, qs), (k, ks), (v, vs) = _operand(q), _operand(k), _operand(v)
    slopes, q_pos, k_pos = D.in_memory(slopes), D.in_memory(q_pos), D.in_memory(k_pos)
    keep = (q, k, v, slopes, q_pos, k_pos)
    pos, slope, qp, kp = 0, (0, 0, 0, 0), 0, 0
    if slopes is not None:
        if q_pos is None or k_pos is None:
            raise ValueError(f"{name}: slopes, q_pos and k_pos go together")
        if slopes.dtype != torch.float32 or q_pos.dtype != torch.float32 or k_pos.dtype != torch.float32:
            raise TypeError(f"{name}: slopes, q_pos and k_pos must be torch.float32")
        pos = q_pos.shape[-1] if q_pos.dim() == 3 else 0
        if pos not in (1, 2) or q_pos.shape != (B, nq, pos) or k_pos.shape != (B, nk, pos):
            raise ValueError(f"{name}: q_pos and k_pos must be [{B}, {nq} / {nk}, 1 or 2], got {list(q_pos.shape)} and "
                             f"{list(k_pos.shape)}")
        if slopes.shape == (H,):
            slope = (slopes.data_ptr(), 0, 0, slopes.stride(0))
        elif slopes.shape == (B, nq, H):
            slope = (slopes.data_ptr(), *slopes.stride())
        else:
            raise ValueError(f"{name}: slopes must be [{H}] or [{B}, {nq}, {H}], got {list(slopes.shape)}")
        if not (q_pos.is_contiguous() and k_pos.is_contiguous()):
            q_pos, k_pos = q_pos.contiguous(), k_pos.contiguous()
            keep += (q_pos, k_pos)
        qp, kp = q_pos.data_ptr(), k_pos.data_ptr()
    elif q_pos is not None or k_pos is not None:
        raise ValueError(f"{name}: slopes, q_pos and k_pos go together")
    qseg = kseg = 0
    if q_segment is not None and k_segment is not None:
        if q_segment.dtype != torch.int32 or k_segment.dtype != torch.int32:
            raise TypeError(f"{name}: q_segment and k_segment must be torch.int32")
        if q_segment.shape != (B, nq) or k_segment.shape != (B, nk):
            raise ValueError(f"{name}: q_segment and k_segment must be [{B}, {nq}] and [{B}, {nk}]")
        if not (q_segment.is_contiguous() and k_segment.is_contiguous()):
            q_segment, k_segment = q_segment.contiguous(), k_segment.contiguous()
            keep += (q_segment, k_segment)
        qseg, kseg = q_segment.data_ptr(), k_segment.data_ptr()
    elif q_segment is not None or k_segment is not None:
        raise ValueError(f"{name}: q_segment and k_segment go together")
    klen = 0
    if k_len is not None:
        if k_len.dtype != torch.int32:
            raise TypeError(f"{name}: k_len must be torch.int32")
        if k_len.shape != (B,):
            raise ValueError(f"{name}: k_len must be [{B}], got {list(k_len.shape)}")
        if not k_len.is_contiguous():
            k_len = k_len.contiguous()
            keep += (k_len,)
        klen = k_len.data_ptr()
    flag = 0
    if error_flag is not None:
        if error_flag.dtype != torch.int32:
            raise TypeError(f"{name}: error_flag must be torch.int32")
        flag = error_flag.data_ptr()
    return _Args(index, (B, nq, nk, H, G, dim, pos), (q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs), slope,
                 (qp, kp, qseg, kseg, klen), flag, (dim ** -0.5 if scale is None else scale, softcap, D.DTYPES[dtype]),
                 keep)


def _pack(a: _Args, out: int, lse: int, workspace: int = 0, workspace_bytes: int = 0, per_row: int = 0, dout: int = 0,
          dout_stride=_ZERO3, dq: int = 0, dk: int = 0, dv: int = 0, dslopes: int = 0) -> bytes:
    try:
        return D.ATTENTION_ARGS.pack(*a.sizes, *a.operands, out, lse, *a.slopes, *a.optional, workspace, workspace_bytes,
                                     a.error_flag, *a.scalars, per_row, dout, *dout_stride, dq, dk, dv, dslopes)
    except OverflowError:
        raise ValueError(f"scale and softcap must fit in fp32, got {a.scalars[:2]}") from None


def _address(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


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
    0 .. Nk).  ``out``: a contiguous tensor like ``q`` to write into (not one of the arguments).  ``error_flag`` (int32) gets
    ``S4D_FLAG_WAIT_TIMEOUT`` should a kernel give up waiting; the rows concerned are then NaN."""
    name = "decoder_attention_forward"
    if out is None and error_flag is None:
        done = D.calls().attention_forward(q, k, v, scale, softcap, slopes, q_pos, k_pos, q_segment, k_segment, k_len)
        if done is not None:
            return done
    a = _checked(name, q, k, v, scale, softcap, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    if out is None:
        out = q.new_empty(q.shape)
    else:
        D.same_device(name, q, out)
        if out.dtype != q.dtype:
            raise TypeError(f"{name}: out must be {q.dtype}, got {out.dtype}")
        if out.shape != q.shape or not out.is_contiguous() or out.is_neg() or out.data_ptr() % 16:
            raise ValueError(f"{name}: out must be a contiguous, 16-byte aligned {list(q.shape)} tensor")
        if any(t is not None and D.overlap(out, t) for t in (q, k, v, slopes, q_pos, k_pos, q_segment, k_segment, k_len)):
            raise ValueError(f"{name}: out must not share memory with the arguments")
    B, nq, _, H = a.sizes[:4]
    lse = q.new_empty((B, H, nq), dtype=torch.float32)
    lib = D.lib()
    args = _pack(a, out.data_ptr(), lse.data_ptr())
    with D.on_device(a.index):
        need = lib.s4d_attention_forward_workspace_bytes(args)
        if need:
            ws = q.new_empty(need // 4, dtype=torch.float32)
            args = _pack(a, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need)
        st = lib.s4d_attention_forward(args, D.stream_ptr(a.index))
    if st:
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
    if error_flag is None:
        done = D.calls().attention_backward(dout, q, k, v, out, lse, scale, softcap, slopes, q_pos, k_pos, q_segment,
                                            k_segment, k_len, need_dkv, need_dslopes)
        if done is not None:
            return done
    a = _checked(name, q, k, v, scale, softcap, slopes, q_pos, k_pos, q_segment, k_segment, k_len, error_flag)
    D.same_device(name, q, dout, out, lse)
    out, lse = D.in_memory(out), D.in_memory(lse)
    B, nq, _, H = a.sizes[:4]
    if q.dtype != torch.bfloat16 or dout.dtype != torch.bfloat16 or out.dtype != torch.bfloat16:
        raise TypeError(f"{name}: q, dout and out must be torch.bfloat16, got {q.dtype}, {dout.dtype} and {out.dtype}")
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"{name}: dout and out must be {list(q.shape)}, got {list(dout.shape)} and {list(out.shape)}")
    if not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"{name}: out must be contiguous and 16-byte aligned")
    if lse.dtype != torch.float32:
        raise TypeError(f"{name}: lse must be torch.float32")
    if lse.shape != (B, H, nq) or not lse.is_contiguous():
        raise ValueError(f"{name}: lse must be a contiguous [{B}, {H}, {nq}] tensor")
    dout, dstride = _operand(dout)
    dq = q.new_empty(q.shape)
    dk, dv = (k.new_empty(k.shape), k.new_empty(k.shape)) if need_dkv else (None, None)
    ds = slopes.new_empty(slopes.shape) if slopes is not None and need_dslopes else None
    if B == 0:
        return dq, dk, dv, None if ds is None else ds.zero_()
    rest = (int(ds is not None and ds.dim() == 3), dout.data_ptr(), dstride, dq.data_ptr(), _address(dk), _address(dv),
            _address(ds))
    lib = D.lib()
    args = _pack(a, out.data_ptr(), lse.data_ptr(), 0, 0, *rest)
    with D.on_device(a.index):
        need = lib.s4d_attention_backward_workspace_bytes(args)
        if need:
            ws = q.new_empty(need // 4, dtype=torch.float32)
            args = _pack(a, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need, *rest)
        st = lib.s4d_attention_backward(args, D.stream_ptr(a.index))
    if st:
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
            if t is not None and t.requires_grad:
                raise ValueError(f"{name}: {what} has no gradient; detach it")
        if q.dtype != torch.bfloat16 and any(t is not None and t.requires_grad for t in (q, k, v, slopes)):
            raise TypeError(f"{name}: gradients are implemented for torch.bfloat16, got {q.dtype}")
    return _DecoderAttention.apply(q, k, v, slopes, scale, softcap, q_pos, k_pos, q_segment, k_segment, k_len)
