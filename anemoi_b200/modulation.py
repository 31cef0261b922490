"""The gated residual behind a block, the norm and the modulation in front of the next one, in one pass, with gradients.

    x_out = x + gate * post(y)                                post(y): y, or its norm times ``post_weight``
    h     = norm(x_out) * weight * (1 + scale) + shift

The reference fuses the same steps of its blocks in Triton
(anemoi/models/minimax_h3/solengine/models/minimax_h3/optimized/fusions.py:1-23, RMS norm, forward only).  Here the norm
may be an RMS norm or a layer norm, and every function is differentiable: autograd records it, and
``fused_gate_norm_modulate_backward`` is the same gradient as a plain call.  Each runs as kernels of this library
(``anemoi_sm100_gate_norm_modulate``); there is no eager fallback.

Rows: ``x`` and ``y`` are ``[..., C]`` in fp16 or bf16, the last dimension contiguous, the others one row stride apart (a
slice of a wider tensor is fine), C a multiple of 8 up to 8,192.  Modulation (gate, scale, shift), in the rows' type or fp32:
``[C]``, ``[..., C]`` without the token dimension (one per sample), or ``[..., F, C]`` with F dividing the tokens (one per
frame; F = tokens: one per token).  Weights: ``[C]`` in the rows' type.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import native

_NORMS = {None: 0, "rms": 1, "layer": 2}


class GateNormGradients(NamedTuple):
    """Gradients of ``fused_gate_norm_modulate``'s arguments (None where there was no such argument)."""

    x: torch.Tensor
    y: torch.Tensor | None
    gate: torch.Tensor | None
    scale: torch.Tensor | None
    shift: torch.Tensor | None
    weight: torch.Tensor | None
    post_weight: torch.Tensor | None


def _rows(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> torch.Tensor:
    """``t`` as rows ``[R, C]`` that the kernel can read, without a copy."""
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the shape, dtype and device of x")
    if t.ndim < 1 or t.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name} must be [..., C] in fp16 or bf16")
    width = t.shape[-1]
    if width == 0 or width % 8 or width > 8192:
        raise ValueError(f"the channels of {name} must be a multiple of 8, at most 8192, got {width}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its channels")
    if t.numel() == 0:
        return t.reshape(-1, width)
    try:
        flat = t.view(-1, width)
    except RuntimeError:
        raise ValueError(f"the rows of {name} must be one stride apart") from None
    if flat.stride(0) % 8 or flat.data_ptr() % 16:
        raise ValueError(f"the rows of {name} must start on 16 bytes")
    return flat


def _modulation(t: torch.Tensor, name: str, x: torch.Tensor) -> torch.Tensor:
    """``t`` as ``[G, C]``, G dividing the rows of ``x``: consecutive rows share one."""
    if t.dtype not in (x.dtype, torch.float32) or t.device != x.device or t.ndim < 1 or t.shape[-1] != x.shape[-1]:
        raise ValueError(f"{name} must be [..., C] on x's device, in x's dtype or fp32")
    lead = x.shape[:-1]
    if t.ndim == 1:
        fits = True
    elif t.ndim == x.ndim - 1:
        fits = t.shape[:-1] == lead[:-1]
    elif t.ndim == x.ndim:
        # the token dimension may be cut into frames
        fits = t.shape[:-2] == lead[:-1] and t.shape[-2] > 0 and lead[-1] % t.shape[-2] == 0
    else:
        fits = False
    if not fits:
        raise ValueError(f"{name} must be [C], x's shape without its tokens, or x's shape with its tokens cut into frames; "
                         f"got {tuple(t.shape)} for x {tuple(x.shape)}")
    step = 16 // t.element_size()
    flat = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_zeros((1, x.shape[-1]))
    if flat.stride(-1) != 1 or flat.stride(0) % step or flat.data_ptr() % 16:
        flat = flat.contiguous() if flat.stride(-1) != 1 or flat.stride(0) % step else flat.clone()
    return flat


def _weight(t: torch.Tensor | None, name: str, x: torch.Tensor) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != x.shape[-1:] or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must be [C] of x's dtype, on its device")
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _Call:
    """One call's arguments, checked and laid out as the kernels read them."""

    def __init__(self, x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm):
        if norm not in ("rms", "layer") or post_norm not in _NORMS:
            raise ValueError("norm must be 'rms' or 'layer', post_norm None, 'rms' or 'layer'")
        if not (eps >= 0.0):
            raise ValueError("eps must not be negative")
        if (y is None) != (gate is None):
            raise ValueError("y and gate go together")
        if y is None and post_norm is not None:
            raise ValueError("post_norm normalises y")
        if post_weight is not None and post_norm is None:
            raise ValueError("post_weight weighs the norm of y: it needs post_norm")
        if not x.is_cuda:
            raise ValueError("x must be on a CUDA device")
        self.x = _rows(x, "x")
        self.y = None if y is None else _rows(y, "y", x)
        mods = {name: _modulation(t, name, x)
                for name, t in (("gate", gate), ("scale", scale), ("shift", shift)) if t is not None}
        if len({t.dtype for t in mods.values()}) > 1:
            raise ValueError("gate, scale and shift must have one dtype")
        groups = max((t.size(0) for t in mods.values()), default=1)
        for name, t in mods.items():
            if t.size(0) not in (1, groups):
                raise ValueError("gate, scale and shift must be given for the same tokens")
        self.mods = mods
        self.groups = groups
        # one row for all groups: a stride of zero
        self.strides = {name: 0 if t.size(0) < groups else t.stride(0) for name, t in mods.items()}
        self.weight = _weight(weight, "weight", x)
        self.post_weight = _weight(post_weight, "post_weight", x)
        self.native = native.Rows(
            rows=self.x.size(0), groups=groups, width=x.shape[-1], norm=_NORMS[norm], post=_NORMS[post_norm],
            is_bf16=int(x.dtype == torch.bfloat16),
            mod_is_fp32=int(any(t.dtype == torch.float32 for t in mods.values())), eps=float(eps))

    def row_stride(self, t):
        return 0 if t is None else t.stride(0)


def _forward(x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm, with_norm=True):
    c = _Call(x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm)
    x_out = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if with_norm else None
    if x.numel():
        native.gate_norm_modulate(
            c.native, c.x, c.y, c.mods.get("gate"), c.mods.get("scale"), c.mods.get("shift"), c.weight, c.post_weight,
            (c.row_stride(c.x), c.row_stride(c.y), *(c.strides.get(k, 0) for k in ("gate", "scale", "shift"))), x_out, h)
    return x_out, h


def _like_modulation(t: torch.Tensor, sums: torch.Tensor, groups: int) -> torch.Tensor:
    """Sums of ``groups`` groups in the shape of the argument (which may have been one row for all of them)."""
    if t.numel() // t.shape[-1] == groups:
        return sums.view(t.shape)
    return sums.float().sum(0).to(t.dtype).view(t.shape)


def _backward(dx_out, dh, x_out, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm) -> GateNormGradients:
    c = _Call(x_out, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm)
    if dx_out is None and dh is None:
        raise ValueError("one of the outputs' gradients is needed")
    given = [None if t is None else _rows(t, name, x_out) for name, t in (("dx_out", dx_out), ("dh", dh))]
    dx = torch.empty(x_out.shape, dtype=x_out.dtype, device=x_out.device)
    dy = None if y is None else torch.empty_like(dx)
    rows = x_out.numel() // x_out.shape[-1] if x_out.numel() else 0
    make = torch.empty if rows else torch.zeros

    def sums(name, wanted=True):
        if name not in c.mods or not wanted:
            return None
        return make((c.groups, x_out.shape[-1]), dtype=c.mods[name].dtype, device=x_out.device)

    def weight_sums(t, wanted=True):
        return None if t is None or not wanted else make(t.shape, dtype=t.dtype, device=t.device)

    norm_wanted = dh is not None
    dgate, dscale, dshift = sums("gate"), sums("scale", norm_wanted), sums("shift", norm_wanted)
    dweight, dpost = weight_sums(c.weight, norm_wanted), weight_sums(c.post_weight)
    if rows:
        native.gate_norm_modulate_backward(
            c.native, *given, c.x, c.y, c.mods.get("gate"), c.mods.get("scale"), c.weight, c.post_weight,
            (c.row_stride(given[0]), c.row_stride(given[1]), c.row_stride(c.x), c.row_stride(c.y),
             c.strides.get("gate", 0), c.strides.get("scale", 0)), dx, dy, dgate, dscale, dshift, dweight, dpost)
    like = {name: t for name, t in (("gate", gate), ("scale", scale), ("shift", shift)) if t is not None}
    shaped = {name: None if s is None else _like_modulation(like[name], s, c.groups)
              for name, s in (("gate", dgate), ("scale", dscale), ("shift", dshift))}
    return GateNormGradients(dx, dy, shaped["gate"], shaped["scale"], shaped["shift"], dweight, dpost)


def _readable(t: torch.Tensor | None) -> torch.Tensor | None:
    """A gradient as autograd hands it over (expanded, transposed, ...) in a form that the kernels read."""
    if t is None or t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _GateNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm, with_norm):
        x_out, h = _forward(x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm, with_norm)
        ctx.save_for_backward(x if x_out is None else x_out, y, gate, scale, shift, weight, post_weight)
        ctx.options = (eps, norm, post_norm)
        ctx.outputs = (x_out is not None, h is not None)
        ctx.set_materialize_grads(False)
        return tuple(t for t in (x_out, h) if t is not None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        given = iter(grads)
        dx_out, dh = (_readable(next(given)) if there else None for there in ctx.outputs)
        if dx_out is None and dh is None:
            return (None,) * 11
        out = _backward(dx_out, dh, *ctx.saved_tensors, *ctx.options)
        return (*(g if need else None for g, need in zip(out, ctx.needs_input_grad)), None, None, None, None)


def fused_gate_norm_modulate(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, scale: torch.Tensor | None = None,
                             shift: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                             post_weight: torch.Tensor | None = None, *, eps: float = 1e-6, norm: str = "rms",
                             post_norm: str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x_out, h)``: the residual stream behind a block and the modulated input of the next one.

    ``h`` is the norm of the unrounded sum.  ``post_norm`` normalises ``y`` before the gate, ``post_weight`` then weighs it."""
    return _GateNorm.apply(x, y, gate, scale, shift, weight, post_weight, eps, norm, post_norm, True)


def fused_norm_modulate(x: torch.Tensor, scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                        weight: torch.Tensor | None = None, *, eps: float = 1e-6, norm: str = "rms") -> torch.Tensor:
    """``norm(x) * weight * (1 + scale) + shift``: the input of a stack's first block."""
    return _GateNorm.apply(x, None, None, scale, shift, weight, None, eps, norm, None, True)[0]


def fused_gate_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, post_weight: torch.Tensor | None = None, *,
                        eps: float = 1e-6, post_norm: str | None = None) -> torch.Tensor:
    """``x + gate * post(y)``: the residual stream behind a stack's last block."""
    return _GateNorm.apply(x, y, gate, None, None, None, post_weight, eps, "rms", post_norm, False)[0]


def fused_gate_norm_modulate_backward(dx_out: torch.Tensor | None, dh: torch.Tensor | None, x_out: torch.Tensor,
                                      y: torch.Tensor, gate: torch.Tensor, scale: torch.Tensor | None = None,
                                      weight: torch.Tensor | None = None, post_weight: torch.Tensor | None = None, *,
                                      eps: float = 1e-6, norm: str = "rms",
                                      post_norm: str | None = None) -> GateNormGradients:
    """The gradients of ``fused_gate_norm_modulate`` from those of its outputs (None: that output was not used).

    ``x_out`` is the residual stream that it returned.  ``x`` of the result is the gradient of the stream before the block,
    which is also that of ``x_out``; ``shift``'s has the shape of ``scale`` (None without ``scale``)."""
    # (shift's values are not needed, its shape is scale's)
    return _backward(dx_out, dh, x_out, y, gate, scale, scale, weight, post_weight, eps, norm, post_norm)


__all__ = ["GateNormGradients", "fused_gate_norm_modulate", "fused_gate_norm_modulate_backward", "fused_gate_residual",
           "fused_norm_modulate"]
