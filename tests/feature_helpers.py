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


def decode64(x, w_gate, w_up, w_down, act, dy=None):
    """y, and with dy the gradients (dx, d w_gate, d w_up, d w_down), from the definition."""
    x, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    g, u = x @ wg.T, x @ wu.T
    if act == "silu":
        gate = torch.sigmoid(g)
        slope = gate * (1 + g * (1 - gate))
    else:
        gate = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        slope = gate + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    a = g * gate
    y = (a * u) @ wd.T
    if dy is None:
        return y
    dy = dy.double()
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    return y, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (a * u)


def decode_tolerances(x, w_gate, w_up, w_down, act, dy=None):
    """Absolute bounds of decode64's outputs, element by element.

    Each second product sums terms of which one factor was rounded to 16 bits (half a step e), plus 32-bit
    accumulation: an instruction sums 16 products and the accumulator, each sum off by at most 2^-23 of the
    magnitudes (truncation).  First products g, u, dh: their 32-bit errors, carried through the activation
    (|slope| <= 1.13, |slope'| <= 1), change h, dg, du by at most 4 * 2^-23 * (terms) of the magnitudes' products;
    the hardware exponential and reciprocal add 2^-20.  All of it is below eps32 = 2^-17 (K + 16) / 16 relative to the
    products of magnitudes; the final rounding adds half a step of the value."""
    e = half_step(x.dtype)
    ax, ag, au, ad = (t.double().abs() for t in (x, w_gate, w_up, w_down))
    k1 = (x.shape[1] + 16) / 16
    eps = 2.0 ** -17 * k1
    mg, mu = ax @ ag.T, ax @ au.T  # magnitudes of the sums that give g and u
    x64, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    g, u = x64 @ wg.T, x64 @ wu.T
    gate = torch.sigmoid(g) if act == "silu" else 0.5 * torch.erfc(-g / math.sqrt(2.0))
    a = (g * gate).abs()
    # errors of a and u from the first products, of h = a u
    ea, eu = 1.13 * eps * mg + 2.0 ** -20 * a, eps * mu
    eh = (e + 2.0 ** -22) * a * u.abs() + ea * u.abs() + eu * a + ea * eu
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a subnormal step of a rounded operand
    y = decode64(x, w_gate, w_up, w_down, act)
    acc = 2.0 ** -23 * (w_gate.shape[0] / 16 + 16)
    out = [(eh + sub) @ ad.T + acc * ((a * u.abs()) @ ad.T) + e * y.abs() + sub]
    if dy is None:
        return out[0]
    ady = dy.double().abs()
    mdh = ady @ ad
    _, dx, dwg, dwu, dwd = decode64(x, w_gate, w_up, w_down, act, dy)
    edh = 2.0 ** -17 * (w_down.shape[0] + 16) / 16 * mdh
    dh = (dy.double() @ wd).abs()
    edg = 1.13 * ((e + 2.0 ** -19) * dh * u.abs() + edh * (u.abs() + eu) + dh * eu) + dh * u.abs() * eps * mg + sub
    edu = (e + 2.0 ** -22) * dh * a + edh * (a + ea) + dh * ea + sub
    mdg, mdu = 1.13 * mdh * mu, mdh * (1.13 * mg)
    acc_f = 2.0 ** -23 * (2 * w_gate.shape[0] / 16 + 16)
    acc_n = 2.0 ** -23 * (x.shape[0] / 16 + 160)
    out.append(edg @ ag + edu @ au + acc_f * (mdg @ ag + mdu @ au) + e * dx.abs() + sub)
    out.append(edg.T @ ax + acc_n * (mdg.T @ ax) + e * dwg.abs() + sub)
    out.append(edu.T @ ax + acc_n * (mdu.T @ ax) + e * dwu.abs() + sub)
    out.append(ady.T @ (eh + sub) + acc_n * (ady.T @ (a * u.abs())) + e * dwd.abs() + sub)
    return out


def decode_norm_bound(dtype) -> float:
    """Bound of |error| / |value| (Frobenius norms) of y and of each gradient, for rows of random signs.

    Every term of a sum has one factor rounded to 16 bits, by at most half a step e of itself, e / sqrt(3) in the root
    mean square, independently; so has every sum at the end.  Terms of random signs add up like their errors: the
    ratio of the norms is at most e sqrt(2 / 3), with what float32 accumulators lose (2.1e-4 of a stretch of like
    signs, far less here) below e.  Twice that is allowed.  A walk that loses one tile of 128 rows out of n is off by
    sqrt(128 / n)."""
    return 2 * half_step(dtype)


def norm_off(got, want) -> float:
    return float((got.double() - want.double()).norm() / want.double().norm())
