"""Gated feature decoder on the sm_100a tensor-core kernels.

Compositing cost grows with the number of feature channels, so a semantic
scene carries few (16 to 128) and a small gated block per pixel turns them
into class logits, or other values of a 2D network, 256 at most.  An addition to the reference,
whose feature rendering (src/mlx3d/splatting/render.py:164-220) ends at the
composited channels.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat

__all__ = ["FeatureDecoder", "decode_features"]


def _workspace(x, dy, f, c, weights):
    size = nat.load().gs_decode_workspace_bytes(nat.ptr(x), nat.ptr(dy), x.shape[0], x.shape[1], f, c, int(weights))
    return torch.empty((size,), device=x.device, dtype=torch.uint8) if size else None


def _prepare(w_gate, w_up, w_down):
    (f, d), c = w_gate.shape, w_down.shape[0]
    image = torch.empty((nat.load().gs_decode_image_bytes(d, f, c),), device=w_gate.device, dtype=torch.uint8)
    nat.call_on(w_gate.device, "gs_decode_prepare", nat.ptr(w_gate), nat.ptr(w_up), nat.ptr(w_down),
                nat.DTYPES[w_gate.dtype], d, f, c, nat.ptr(image), image.numel())
    return image


def _forward(x, w_gate, w_up, w_down, act):
    """y, and the weights' image (None where few rows were decoded without one)."""
    n, d = x.shape
    f, c = w_gate.shape[0], w_down.shape[0]
    y = torch.empty((n, c), device=x.device, dtype=x.dtype)
    if nat.load().gs_decode_is_few(n, d, f, c):
        nat.call_on(x.device, "gs_decode_forward_few", nat.ptr(x), nat.ptr(w_gate), nat.ptr(w_up), nat.ptr(w_down),
                    nat.DTYPES[x.dtype], n, d, f, c, act, nat.ptr(y))
        return y, None
    image = _prepare(w_gate, w_up, w_down)
    ws = _workspace(x, None, f, c, False)
    nat.call_on(x.device, "gs_decode_forward", nat.ptr(x), nat.DTYPES[x.dtype], n, d, f, c, act, nat.ptr(image),
                image.numel(), nat.ptr(y), nat.ptr(ws), 0 if ws is None else ws.numel())
    return y, image


class _Decode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        y, image = _forward(x, w_gate, w_up, w_down, act)
        ctx.save_for_backward(x, w_gate, w_up, w_down, image)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, image = ctx.saved_tensors
        n, d = x.shape
        f, c = w_gate.shape[0], w_down.shape[0]
        dev = x.device
        dy = dy.contiguous()
        if image is None:
            image = _prepare(w_gate, w_up, w_down)
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        weights = any(ctx.needs_input_grad[1:4])
        grads = tuple(torch.empty_like(w) for w in (w_gate, w_up, w_down)) if weights else (None, None, None)
        ws = _workspace(x, dy, f, c, weights)
        nat.call_on(dev, "gs_decode_backward", nat.ptr(x), nat.ptr(dy), nat.DTYPES[x.dtype], n, d, f, c, ctx.act,
                    nat.ptr(image), image.numel(), nat.ptr(dx), *(nat.ptr(g) for g in grads), nat.ptr(ws),
                    0 if ws is None else ws.numel())
        return (dx, *(g if need else None for g, need in zip(grads, ctx.needs_input_grad[1:4])), None)


def decode_features(features: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                    activation: str = "silu") -> torch.Tensor:
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T`` per pixel; differentiable (reverse mode) in all four tensors.

    ``features`` (..., D) with D <= 128, ``w_gate`` and ``w_up`` (F, D), ``w_down`` (C, F) with C <= 256; the
    weights are all float16 or all bfloat16 and set the type of the computation: features of another floating
    type are rounded to it.  ``activation`` is "silu" or "gelu" (the error-function form).  Returns (..., C) in
    the weights' type.

    Products are summed in 32 bits.  The hidden values, and their gradients in the backward pass, are rounded to
    the weights' type as operands of the next products (the forward of at most 64 rows of a small block keeps them
    in 32 bits); they stay on chip.  In float16 a hidden value above 65504 becomes infinite and a hidden gradient
    below 2^-25 zero: scale ``features`` and the loss accordingly, or take bfloat16."""
    act = nat.GS_GATES.get(activation)
    if act is None:
        raise ValueError("activation must be 'silu' or 'gelu'.")
    for name, w in (("features", features), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not w.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor (got {w.dtype})")
    if features.ndim < 1 or w_gate.ndim != 2 or w_down.ndim != 2:
        raise ValueError("features must have shape (..., D), w_gate and w_up (F, D), w_down (C, F).")
    lead, d = features.shape[:-1], features.shape[-1]
    f, c = w_gate.shape[0], w_down.shape[0]
    if w_gate.shape != (f, d) or w_up.shape != (f, d) or w_down.shape != (c, f):
        raise ValueError("features (..., D), w_gate (F, D), w_up (F, D) and w_down (C, F) must agree.")
    if not 1 <= d <= nat.GS_DECODE_MAX_D:
        raise ValueError(f"features must have 1 to {nat.GS_DECODE_MAX_D} channels (got {d}).")
    if not 1 <= c <= nat.GS_DECODE_MAX_C:
        raise ValueError(f"the decoder must have 1 to {nat.GS_DECODE_MAX_C} outputs (got {c}).")
    if not 1 <= f <= nat.GS_DECODE_MAX_F:
        raise ValueError(f"the decoder must have 1 to {nat.GS_DECODE_MAX_F} hidden units (got {f}).")
    ty = w_gate.dtype
    if ty not in (torch.float16, torch.bfloat16) or w_up.dtype != ty or w_down.dtype != ty:
        raise TypeError("w_gate, w_up and w_down must all be float16 or all bfloat16.")
    x = nat.require_cuda("features", features, ty)
    w_gate = nat.require_cuda("w_gate", w_gate, ty)
    w_up = nat.require_cuda("w_up", w_up, ty)
    w_down = nat.require_cuda("w_down", w_down, ty)
    nat.same_device(x.device, w_gate=w_gate, w_up=w_up, w_down=w_down)
    if x.numel() // d > nat.GS_DECODE_MAX_N:
        raise ValueError(f"features must have at most {nat.GS_DECODE_MAX_N} rows.")
    flat = len(lead) == 1
    if not flat:
        x = x.reshape(-1, d)
    if nat.differentiated(x, w_gate, w_up, w_down):
        y = _Decode.apply(x, w_gate, w_up, w_down, act)
    else:
        y = _forward(x, w_gate, w_up, w_down, act)[0]
    return y if flat else y.reshape(*lead, c)


class FeatureDecoder:
    """The weights of a gated decoder as float32 leaves ``params`` ("w_gate", "w_up", "w_down"), computed in
    ``dtype``: ``decoder(features)`` rounds them and calls :func:`decode_features`."""

    def __init__(self, params: dict[str, torch.Tensor], activation: str = "silu", dtype=torch.bfloat16):
        if set(params) != {"w_gate", "w_up", "w_down"}:
            raise ValueError("params must hold w_gate, w_up and w_down.")
        if activation not in nat.GS_GATES:
            raise ValueError("activation must be 'silu' or 'gelu'.")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("dtype must be torch.float16 or torch.bfloat16.")
        self.params, self.activation, self.dtype = params, activation, dtype

    @classmethod
    def create(cls, channels: int, hidden: int, outputs: int, activation: str = "silu", dtype=torch.bfloat16,
               device="cuda", generator: torch.Generator | None = None) -> "FeatureDecoder":
        """Normal weights of variance 1 / fan-in, as trainable leaves."""
        def w(rows, cols):
            return (torch.randn((rows, cols), device=device, generator=generator) / cols ** 0.5).requires_grad_(True)

        return cls({"w_gate": w(hidden, channels), "w_up": w(hidden, channels), "w_down": w(outputs, hidden)},
                   activation, dtype)

    def __call__(self, features: torch.Tensor) -> torch.Tensor:
        p = self.params
        return decode_features(features, p["w_gate"].to(self.dtype), p["w_up"].to(self.dtype),
                               p["w_down"].to(self.dtype), self.activation)
