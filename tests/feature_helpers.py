"""Plain 64-bit forms of the feature-field operators, on the CPU or the GPU."""

from __future__ import annotations

import math

import torch

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype) -> float:
    """The largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def distill64(logits, values, index, t=1.0, weight=None):
    """Row losses and rows' gradients from the definition."""
    s = logits.double()
    v, i = values.double(), index.long()
    c = s.shape[-1]
    gone = (i < 0) | (i >= c) | (v == -math.inf)
    i = i.masked_fill(gone, 0)
    empty = gone.all(-1, keepdim=True)
    v = v.masked_fill(gone, -math.inf)
    v = v - v.amax(-1, keepdim=True).masked_fill(empty, 0.0)  # huge equal values: log p must not cancel
    logp = (v / t).masked_fill(gone, -math.inf)
    logp = logp - torch.logsumexp(logp.masked_fill(empty, 0.0), -1, keepdim=True)
    p = torch.exp(logp).masked_fill(gone, 0.0)
    logq = s / t - torch.logsumexp(s / t, -1, keepdim=True)
    term = (p * (logp.masked_fill(gone, 0.0) - logq.gather(-1, i))).masked_fill(p == 0, 0.0)
    w = torch.ones(s.shape[:-1], dtype=torch.float64, device=s.device) if weight is None else weight.double()
    loss = w * t * t * term.sum(-1)
    grad = torch.exp(logq).scatter_add(-1, i, -p) * (w * t)[..., None]
    return loss.masked_fill(empty[..., 0], 0.0), grad.masked_fill(empty, 0.0)


def distill_tolerance(logits, values, t, k):
    """(absolute error of a row loss / (weight T^2), relative error of a q or p), per row.

    The exponents (s - max) / T carry three roundings (difference, 1 / T, product), relative 3 * 2^-24 each; exp and
    log are within 2 ulp (2^-22); a lane sums C / 32 terms, the warp five more, one rounding each."""
    fin = lambda x: torch.where(torch.isfinite(x), x, torch.zeros_like(x))  # noqa: E731
    s, v = fin(logits.double()), fin(values.double())
    far = (s.amax(-1) - s.amin(-1)).clamp(max=700.0 * t) / t + (v.amax(-1) - v.amin(-1)).clamp(max=700.0 * t) / t
    rel = 2.0 ** -24 * (3 * far + logits.shape[-1] / 32 + k / 32 + 10 + 24)
    return rel * (1 + far), rel


def write64(logits, k, bits):
    """Offsets, scales (64-bit quotients), indices and codes of cache rows."""
    ty = logits.dtype
    z = logits.double().cpu()
    n, c = z.shape
    z = z.masked_fill(~torch.isfinite(z) | (z <= torch.finfo(ty).min), -math.inf)
    v, i = z.sort(dim=1, descending=True, stable=True)
    m = min(k, c)
    values = torch.full((n, k), -math.inf, dtype=torch.float64)
    index = torch.full((n, k), -1, dtype=torch.int32)
    values[:, :m], index[:, :m] = v[:, :m], i[:, :m].int()
    gone = values == -math.inf
    index[gone] = -1
    first = values[:, :1].masked_fill(gone[:, :1], 0.0)
    last = values.masked_fill(gone, math.inf).amin(1, keepdim=True)
    span = (first - last).masked_fill(gone[:, :1], 0.0)
    levels = 2.0 ** bits - 1
    code = torch.round((first - values).masked_fill(gone, 0.0) * levels / span).masked_fill((span == 0) | gone, 0.0)
    return first, span / levels, index, code


def read64(first, scale, index, code):
    """What the records stand for: the stored (float32) offset and step, one rounding at the end."""
    value = first - code * scale.float().double()
    return value.float().masked_fill(index < 0, -math.inf)
