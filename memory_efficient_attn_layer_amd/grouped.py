"""Attention of packed prompts with grouped heads, given q, k and v:
``grouped_attn_varlen``, forward and backward.

The block's attention has one key/value head per query head and lives between
its projections; this is the operator alone, for layers that make their own q, k
and v: ``Hq`` query heads share ``Hkv`` key/value heads (head h reads head
h // (Hq // Hkv)), sequences lie back to back as in ``fused_attn_varlen``, and
attention is causal inside each. Runs in libmea.so on the current stream, in
bfloat16 and float16 (gradients: bfloat16); there is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .attention import check_offsets

SUPPORTED_WIDTHS = (32, 64, 128, 256)
MAX_TOKEN_STRIDE = 1 << 24  # elements


def _check_scale(scale, N: int) -> float:
    scale = 1.0 / math.sqrt(N) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError(f"scale={scale} must be in [2^-100, 2^100]")
    return scale


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` dense, at a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` (.., tokens, heads, N) as the library reads it, with any strides that
    are multiples of 8 elements; a dense copy of anything else."""
    *outer, last = t.stride()
    bits = t.data_ptr() >> 1
    for s in outer:
        bits |= s
    return t if last == 1 and bits & 7 == 0 else _aligned(t)


def _tokens(t: torch.Tensor) -> torch.Tensor:
    """The same for (tokens, heads, N), whose token stride has a limit."""
    return _rows(t) if t.stride(0) <= MAX_TOKEN_STRIDE else _aligned(t)


def _validate(q, k, v) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise ValueError(f"{name} must be a (total_tokens, heads, N) tensor")
    if q.dtype not in _lib.MEA_DTYPES:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    total, Hq, N = q.shape
    if total < 1 or Hq < 1:
        raise ValueError(f"empty input: q.shape={tuple(q.shape)}")
    if N not in SUPPORTED_WIDTHS:
        raise ValueError(f"head width N={N} not supported (supported: {SUPPORTED_WIDTHS})")
    if k.shape != v.shape or k.shape[0] != total or k.shape[2] != N or k.shape[1] < 1:
        raise ValueError(f"k and v must be ({total}, Hkv, {N}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if Hq % k.shape[1] != 0:
        raise ValueError(f"{Hq} query heads are no multiple of {k.shape[1]} key/value heads")
    for name, t in (("k", k), ("v", v)):
        if t.dtype != q.dtype:
            raise TypeError(f"{name} is {t.dtype}, q is {q.dtype}")
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q is on {q.device}")
    if not q.is_cuda:
        raise RuntimeError("grouped_attn_varlen runs only on a ROCm GPU device (there is no CPU path)")


def _plan(q, k, v, nseq: int, scale: float) -> tuple[_lib.MeaGrouped, int]:
    """The call's descriptor and the workspace bytes of its backward."""
    total, Hq, N = q.shape
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    return _lib.grouped_plan(total, nseq, Hq, k.shape[1], N, sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], scale,
                             _lib.MEA_DTYPES[q.dtype])


def _forward(q, k, v, cu_seqlens, scale, save):
    """(o, o_rest, lse), the last two None without ``save``; q, k, v as _tokens leaves them."""
    dev = q.device
    d, _ = _plan(q, k, v, cu_seqlens.shape[0] - 1, scale)
    total, Hq, N = q.shape
    o = torch.empty((total, Hq, N), device=dev, dtype=q.dtype)
    rest = torch.empty_like(o) if save else None
    lse = torch.empty((Hq, total), device=dev, dtype=torch.float32) if save else None
    with _lib.on_device(dev):
        rc = _lib.load().mea_grouped_fwd(d, cu_seqlens.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                         _lib.ptr(rest), _lib.ptr(lse), _lib.stream_of(dev))
    if rc != 0:
        _lib.check(rc, "mea_grouped_fwd")
    return o, rest, lse


class GroupedAttentionFunction(torch.autograd.Function):
    """Autograd op behind ``grouped_attn_varlen`` where a gradient is wanted:
    saves q, k, v, the output, what rounding it to 16 bits left and its
    log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        q, k, v = _tokens(q), _tokens(k), _tokens(v)
        o, rest, lse = _forward(q, k, v, cu_seqlens, scale, True)
        ctx.save_for_backward(q, k, v, cu_seqlens, o, rest, lse)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, grad_output):
        if torch.is_grad_enabled():  # create_graph
            raise RuntimeError("grouped_attn_varlen has no second derivative")
        q, k, v, cu, o, rest, lse = ctx.saved_tensors
        dev = q.device
        dout = _aligned(grad_output)
        d, ws_bytes = _plan(q, k, v, cu.shape[0] - 1, ctx.scale)
        dq, dk, dv = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k, v))
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        with _lib.on_device(dev):
            rc = _lib.load().mea_grouped_bwd(d, cu.data_ptr(), dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                             o.data_ptr(), rest.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                             dv.data_ptr(), ws.data_ptr(), ws_bytes, _lib.stream_of(dev))
        if rc != 0:
            _lib.check(rc, "mea_grouped_bwd")
        return dq, dk, dv, None, None


def grouped_attn_varlen(q, k, v, cu_seqlens, scale=None):
    """Causal attention of packed sequences: q (total, Hq, N), k and v
    (total, Hkv, N), Hq a multiple of Hkv, N in 32, 64, 128, 256; returns
    (total, Hq, N). ``cu_seqlens``: the nseq + 1 offsets of the sequences, as in
    ``fused_attn_varlen`` (a list or CPU tensor is checked; an int32 device tensor
    is trusted, and tokens it gives to no sequence get zeros). ``scale`` defaults
    to 1 / sqrt(N). Rows of q, k and v may have strides of their own (a slice of
    a joint projection is read in place)."""
    _validate(q, k, v)
    scale = _check_scale(scale, q.shape[2])
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.device.type == "cpu":
        host = [int(x) for x in (cu_seqlens.tolist() if isinstance(cu_seqlens, torch.Tensor) else cu_seqlens)]
        check_offsets(host, q.shape[0])
        cu_seqlens = torch.tensor(host, dtype=torch.int32, device=q.device)
    elif cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.device != q.device:
        raise ValueError("cu_seqlens must be a 1-D int32 tensor of nseq + 1 offsets on the device of q")
    cu_seqlens = cu_seqlens.contiguous()
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return _forward(_tokens(q), _tokens(k), _tokens(v), cu_seqlens, scale, False)[0]
    if q.dtype != torch.bfloat16:
        raise TypeError(f"gradients are taken in bfloat16 only, got {q.dtype}")
    return GroupedAttentionFunction.apply(q, k, v, cu_seqlens, scale)


__all__ = ["GroupedAttentionFunction", "grouped_attn_varlen", "SUPPORTED_WIDTHS"]
