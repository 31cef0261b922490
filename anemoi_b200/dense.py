"""Dense attention with a gradient, beside the sparse mixed-precision call: what a model is tuned with, and what its
dense-first layers compute.

    out = softmax(scale * q k^T) v

``dense_attention`` is differentiable: its backward pass recomputes the probabilities from the rows' log-sum-exps, so that
nothing of the size of queries x keys is kept.  ``dense_attention_backward`` is the same gradient as a plain call.  Both run
as tcgen05 kernels of this library (``anemoi_sm100_dense_attention``); there is no eager fallback.

``q``: ``[B, Sq, Hq, D]``, ``k`` and ``v``: ``[B, Sk, Hk, D]``, fp16 or bf16, D = 64 or 128, Hq a multiple of Hk (query head h
reads key head ``h // (Hq // Hk)``); strided views with a contiguous last dimension and every head on 16 bytes are fine.
``query_lengths`` / ``key_lengths``: int32 ``[B]`` on the device, how many leading tokens of each sample count (values are
clamped to the tensors' lengths).  What stands behind them is not used, be it NaN; the outputs' rows there are zeros, and so
are those of queries that see no key.  ``causal``: query i of a sample sees the keys up to ``i + keys - queries`` of it.
"""

from __future__ import annotations

import math

import torch

from . import native
from .executor import _status_word


def _tensor(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> torch.Tensor:
    if not t.is_cuda or t.ndim != 4 or t.dtype not in (torch.float16, torch.bfloat16) or t.shape[-1] not in (64, 128):
        raise ValueError(f"{name} must be [B, tokens, heads, 64 or 128] in fp16 or bf16, on a CUDA device")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0]
                             or t.shape[-1] != like.shape[-1]):
        raise ValueError(f"{name} must have q's dtype, device, batch and head dimension")
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16
                      or any(t.size(i) > 1 and (t.stride(i) <= 0 or t.stride(i) % 8) for i in range(3))):
        raise ValueError(f"the heads of {name} must be contiguous and start on 16 bytes")
    return t


def _lengths(t: torch.Tensor | None, name: str, q: torch.Tensor) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != (q.shape[0],) or t.dtype != torch.int32 or t.device != q.device:
        raise ValueError(f"{name} must be int32 [B] on q's device")
    return t.contiguous()


def _check(q, k, v, scale, causal, query_lengths, key_lengths):
    _tensor(q, "q")
    _tensor(k, "k", q)
    _tensor(v, "v", q)
    if k.shape != v.shape:
        raise ValueError("k and v must share [B, tokens, heads, D]")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError("q's heads must be a multiple of k's")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("scale must be positive")
    shape = native.DenseShape(
        batch=q.shape[0], q_heads=q.shape[2], k_heads=k.shape[2], q_tokens=q.shape[1], k_tokens=k.shape[1],
        head_dim=q.shape[3], causal=int(bool(causal)), is_bf16=int(q.dtype == torch.bfloat16), scale=scale)
    return shape, _lengths(query_lengths, "query_lengths", q), _lengths(key_lengths, "key_lengths", q)


def _strides(*tensors):
    return [s for t in tensors for s in t.stride()[:3]]


def _forward(q, k, v, scale, causal, query_lengths, key_lengths):
    shape, q_lengths, k_lengths = _check(q, k, v, scale, causal, query_lengths, key_lengths)
    if q.numel() == 0 or k.numel() == 0:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, dtype=torch.float32, device=q.device)
        return out, lse
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
    native.dense_attention(shape, q, k, v, q_lengths, k_lengths, _strides(q, k, v, out), out, lse, _status_word(q.device))
    return out, lse


def dense_attention_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, *, scale: float | None = None, causal: bool = False,
                             query_lengths: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None):
    """``(dq, dk, dv)`` from the gradient of ``out``; ``out`` and ``lse`` are what ``dense_attention`` gave for the same
    arguments.  Equal calls give equal bits."""
    shape, q_lengths, k_lengths = _check(q, k, v, scale, causal, query_lengths, key_lengths)
    for name, t in (("grad_out", grad_out), ("out", out)):
        if t.shape != q.shape:
            raise ValueError(f"{name} must have q's shape")
        _tensor(t, name, q)
    if (lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32 or lse.device != q.device
            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous fp32 [B, heads, queries] on q's device")
    make = torch.zeros if q.numel() == 0 or k.numel() == 0 else torch.empty
    dq, dk, dv = (make(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if make is torch.empty:
        native.dense_attention_backward(shape, grad_out, q, k, v, out, lse, q_lengths, k_lengths,
                                        _strides(grad_out, q, k, v, out, dq, dk, dv), dq, dk, dv, _status_word(q.device))
    return dq, dk, dv


class _DenseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, query_lengths, key_lengths, scale, causal):
        out, lse = _forward(q, k, v, scale, causal, query_lengths, key_lengths)
        ctx.save_for_backward(q, k, v, out, lse, query_lengths, key_lengths)
        ctx.options = dict(scale=scale, causal=causal)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, _):
        q, k, v, out, lse, query_lengths, key_lengths = ctx.saved_tensors
        # autograd hands gradients over in any layout (expanded, transposed)
        if not grad_out.is_contiguous() or grad_out.data_ptr() % 16:
            grad_out = grad_out.clone(memory_format=torch.contiguous_format)
        grads = dense_attention_backward(grad_out, q, k, v, out, lse, query_lengths=query_lengths, key_lengths=key_lengths,
                                         **ctx.options)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, causal: bool = False,
                    query_lengths: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None,
                    return_lse: bool = False):
    """``out`` ``[B, Sq, Hq, D]`` (with ``return_lse`` also the rows' log-sum-exps ``[B, Hq, Sq]``, fp32, without a gradient
    of their own).  ``scale``: D ** -0.5 by default."""
    out, lse = _DenseAttention.apply(q, k, v, query_lengths, key_lengths, scale, causal)
    return (out, lse) if return_lse else out


__all__ = ["dense_attention", "dense_attention_backward"]
