"""What is timed of the feature-field operators, and their plain forms.

Semantic feature fields: a scene's rendered feature channels are decoded to
class logits by a small gated block (``splatting.decode_features``), compared
with a 2D teacher's largest logits (``losses.distill_loss``), which are kept
quantised on the device (``staging.TeacherCache``).  ``own`` chooses between
the plain forms (elementary torch operations) and the framework's kernels.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LEVELS = {8: 255.0, 4: 15.0}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # One picked point's features decoded on a click: latency.
        dict(name="decode_point", kind="decode", rows=1, d=32, f=64, c=20, type="bf16", act="silu"),
        # A 1280x720 view of 32 feature channels, decoded for display.
        dict(name="decode_view", kind="decode", rows=1280 * 720, d=32, f=128, c=150, type="fp16", act="silu"),
        # A 4K view of 64 channels: the largest frame the render benchmark has.
        dict(name="decode_4k", kind="decode", rows=3840 * 2160, d=64, f=256, c=150, type="bf16", act="silu"),
        # A small batch of sampled pixels with ragged sizes, forward and backward.
        dict(name="decode_train_odd", kind="decode_train", rows=4099, d=47, f=171, c=133, type="fp16", act="gelu"),
        # One 1600x1060 training view, forward and backward.
        dict(name="decode_train_view", kind="decode_train", rows=1600 * 1060, d=64, f=256, c=150, type="bf16",
             act="silu"),
        # Per-pixel agreement with the teacher on a 1280x720 test view, few classes rendered directly.
        dict(name="distill_eval_view", kind="distill_eval", rows=1280 * 720, c=20, k=5, type="fp32", t=1.0),
        # The loss and its gradient on a 1920x1080 view of composited (fp32) logits.
        dict(name="distill_train_view", kind="distill_train", rows=1920 * 1080, c=150, k=8, type="fp32", t=2.0,
             reduction="mean"),
        # An open vocabulary: few sampled rows, very many classes.
        dict(name="distill_train_open", kind="distill_train", rows=1031, c=32001, k=32, type="bf16", t=1.0,
             reduction="mean"),
        # A training step on pixels sampled from all views, teacher read from the cache.
        dict(name="distill_train_cached", kind="distill_cached", rows=262147, c=133, k=8, type="fp16", t=2.0, bits=8,
             held=1280 * 720 * 2, reduction="sum"),
        # The teacher's 1920x1080 output written to the cache once it has run, and read back.
        dict(name="cache_write_view", kind="cache_write", rows=1920 * 1080, c=150, k=8, type="bf16", bits=8),
        # A coarse patch grid of an open-vocabulary teacher, many entries a row, 4 bits.
        dict(name="cache_write_open", kind="cache_write", rows=16383, c=1201, k=32, type="fp32", bits=4),
        # Targets of pixels sampled from five 1280x720 views.
        dict(name="cache_read_rows", kind="cache_read", rows=1000003, c=150, k=8, bits=8, held=1280 * 720 * 5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _reduction(rng, ty):
    # the mean's gradients (1 / rows) fall below fp16's range: there a program takes the sum
    return "sum" if ty == "fp16" else rng.choice(["sum", "mean"])


def draw(rng):
    kind = rng.choice(["decode", "decode_train", "decode_train", "distill_eval", "distill_train", "distill_train",
                       "distill_cached", "cache_write", "cache_write", "cache_read"])
    if kind in ("decode", "decode_train"):
        # x, hidden and logits of the largest draw stay below the largest listed case
        return dict(kind=kind, rows=_log_int(rng, 1, 1_500_000), d=_log_int(rng, 3, 128), f=_log_int(rng, 8, 256),
                    c=_log_int(rng, 2, 150), type=rng.choice(["bf16", "fp16"]),
                    act=rng.choice(["silu", "gelu"]))
    if kind in ("distill_eval", "distill_train"):
        c = _log_int(rng, 2, 32768)
        rows = _log_int(rng, 1, max(1, min(2_000_000, 150_000_000 // c)))
        ty = rng.choice(list(_TYPES))
        return dict(kind=kind, rows=rows, c=c, k=_log_int(rng, 1, 64), type=ty, t=rng.choice([0.5, 1.0, 2.0, 4.0]),
                    reduction=_reduction(rng, ty))
    if kind == "distill_cached":
        c = _log_int(rng, 2, 2048)
        rows = _log_int(rng, 1, min(500_000, 100_000_000 // c))
        ty = rng.choice(list(_TYPES))
        return dict(kind=kind, rows=rows, c=c, k=_log_int(rng, 1, 32), type=ty, t=rng.choice([0.5, 1.0, 2.0]),
                    bits=rng.choice([4, 8]), held=_log_int(rng, 1, 2_000_000), reduction=_reduction(rng, ty))
    if kind == "cache_write":
        c = _log_int(rng, 2, 32767)
        rows = _log_int(rng, 1, max(1, min(1_000_000, 100_000_000 // c)))
        return dict(kind=kind, rows=rows, c=c, k=_log_int(rng, 1, 32), type=rng.choice(list(_TYPES)),
                    bits=rng.choice([4, 8]))
    return dict(kind=kind, rows=_log_int(rng, 1, 1_000_000), c=_log_int(rng, 2, 32767), k=_log_int(rng, 1, 32),
                bits=rng.choice([4, 8]), held=_log_int(rng, 1, 4_000_000))


# -------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _record_bytes(k, bits):
    return (8 + 2 * k + (k * bits + 7) // 8 + 15) // 16 * 16


def _records(g, rows, k, c, bits):
    """A cache as it was saved: random records (offset, scale, indices, codes); some entries and rows absent."""
    code_bytes = (k * bits + 7) // 8
    off = torch.randn((rows, 1), device="cuda", generator=g) * 3.0 + 6.0
    scale = torch.rand((rows, 1), device="cuda", generator=g) * (8.0 / _LEVELS[bits])
    first = torch.randint(0, c, (rows, 1), device="cuda", generator=g)
    index = (first + torch.arange(k, device="cuda") * 7) % c
    count = torch.randint(0, 4 * k + 1, (rows, 1), device="cuda", generator=g)  # most rows are full
    index = torch.where(torch.arange(k, device="cuda") < count, index, torch.full_like(index, -1)).to(torch.int16)
    codes = torch.randint(0, 256, (rows, code_bytes), device="cuda", generator=g, dtype=torch.uint8)
    if bits == 4 and k % 2:
        codes[:, -1] &= 15
    rec = torch.zeros((rows, _record_bytes(k, bits)), device="cuda", dtype=torch.uint8)
    rec[:, 0:4] = off.view(torch.uint8)
    rec[:, 4:8] = scale.view(torch.uint8)
    rec[:, 8:8 + 2 * k] = index.contiguous().view(torch.uint8)
    rec[:, 8 + 2 * k:8 + 2 * k + code_bytes] = codes
    return rec


def _cache(case, records):
    from mlx3d_b200.staging import TeacherCache

    cache = TeacherCache(records.shape[0], case["k"], case["c"], bits=case["bits"], device="cuda")
    cache.load_state_dict({"records": records})
    return cache


def prepare(case, seed):
    g = _gen(seed)
    kind, rows, c = case["kind"], case["rows"], case["c"]
    s = {"case": case}
    if kind in ("decode", "decode_train"):
        d, f, ty = case["d"], case["f"], _TYPES[case["type"]]
        x = torch.randn((rows, d), device="cuda", generator=g)
        x *= torch.rand((rows, 1), device="cuda", generator=g) > 0.1  # pixels that no Gaussian covers are zero
        s["x"] = x.to(ty)
        s["w_gate"] = (torch.randn((f, d), device="cuda", generator=g) / math.sqrt(d)).to(ty)
        s["w_up"] = (torch.randn((f, d), device="cuda", generator=g) / math.sqrt(d)).to(ty)
        s["w_down"] = (torch.randn((c, f), device="cuda", generator=g) * (2.0 / math.sqrt(f))).to(ty)
        if kind == "decode_train":
            s["dy"] = (torch.randn((rows, c), device="cuda", generator=g) * 0.05).to(ty)
            for n in ("x", "w_gate", "w_up", "w_down"):
                s[n].requires_grad_(True)
        return s
    if kind in ("distill_eval", "distill_train", "distill_cached"):
        s["logits"] = (torch.randn((rows, c), device="cuda", generator=g) * 2.0).to(_TYPES[case["type"]])
        s["weight"] = torch.rand((rows,), device="cuda", generator=g)  # e.g. the view's alpha
        if kind == "distill_cached":
            s["records"] = _records(g, case["held"], case["k"], c, case["bits"])
            s["pick"] = torch.randint(0, case["held"], (rows,), device="cuda", generator=g)
            if own:
                s["cache"] = _cache(case, s["records"])
            return s
        k = case["k"]
        s["values"] = (torch.randn((rows, k), device="cuda", generator=g) * 2.0 + 6.0).half().sort(
            dim=1, descending=True).values
        first = torch.randint(0, c, (rows, 1), device="cuda", generator=g)
        index = ((first + torch.arange(k, device="cuda") * 7) % c).to(torch.int32)
        absent = torch.rand((rows, 1), device="cuda", generator=g) < 0.05  # pixels without a label
        absent = absent | (torch.rand((rows, k), device="cuda", generator=g) < 0.02)
        s["index"] = index.masked_fill(absent, -1)
        return s
    if kind == "cache_write":
        z = torch.randn((rows, c), device="cuda", generator=g) * 3.0
        z += torch.randn((c,), device="cuda", generator=g) * 2.0  # common and rare classes
        ty = _TYPES[case["type"]]
        z = z.to(ty)
        if c > 4:  # classes that this view's prompt leaves out, masked in both usual ways
            z[:, 1] = -math.inf
            z[:, c // 2] = torch.finfo(ty).min
        s["logits"] = z
        s["start"] = 5
        held = rows + 11
        if own:
            from mlx3d_b200.staging import TeacherCache

            s["cache"] = TeacherCache(held, case["k"], c, bits=case["bits"], device="cuda")
        return s
    s["records"] = _records(g, case["held"], case["k"], c, case["bits"])
    s["pick"] = torch.randint(0, case["held"], (rows,), device="cuda", generator=g)
    if own:
        s["cache"] = _cache(case, s["records"])
    return s


# --------------------------------------------------------------- plain forms
def _gate(g, name):
    """act(g) / g: the logistic function, or the normal distribution function."""
    if name == "silu":
        return 1.0 / (1.0 + torch.exp(-g))
    return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))


def _slope(g, gate, name):
    """act'(g)."""
    if name == "silu":
        return gate * (1.0 + g * (1.0 - gate))
    return gate + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)


def _plain_decode(s):
    case = s["case"]
    ty = s["x"].dtype
    wg, wu, wd = (s[n].detach().float() for n in ("w_gate", "w_up", "w_down"))
    x = s["x"].detach().float()
    g, u = x @ wg.T, x @ wu.T
    gate = _gate(g, case["act"])
    a = g * gate
    h = a * u
    y = (h @ wd.T).to(ty)
    if case["kind"] == "decode":
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dwd = dy.T @ h
    dg, du = dh * u * _slope(g, gate, case["act"]), dh * a
    dx = dg @ wg + du @ wu
    return [y] + [t.to(ty) for t in (dx, dg.T @ x, du.T @ x, dwd)]


def _plain_distill(s, values, index):
    """Row losses, or their sum or mean with its gradient."""
    case = s["case"]
    t = case["t"]
    z = s["logits"].float()
    rows, c = z.shape
    here = (index >= 0) & (index < c) & (values != -math.inf)
    at = torch.where(here, index, torch.zeros_like(index)).long()
    v = torch.where(here, values.float() / t, torch.full_like(values, -math.inf, dtype=torch.float32))
    some = here.any(dim=1)
    top = torch.where(some, v.amax(dim=1), torch.zeros_like(v[:, 0]))
    e = torch.exp(v - top[:, None])
    total = torch.where(some, e.sum(dim=1), torch.ones_like(top))
    p = e / total[:, None]
    z = z / t
    m = z.amax(dim=1, keepdim=True)
    z = z - m
    lse = torch.log(torch.exp(z).sum(dim=1))
    logp = v - top[:, None] - torch.log(total)[:, None]
    term = torch.where(p > 0, p * (logp - (z.gather(1, at) - lse[:, None])), torch.zeros_like(p))
    loss = term.sum(dim=1) * (t * t) * s["weight"]
    if case["kind"] == "distill_eval":
        return loss
    n = rows if case["reduction"] == "mean" else 1
    scale = (s["weight"] * (t / n) * some)[:, None]
    grad = torch.exp(z - lse[:, None])
    grad.scatter_add_(1, at, -p)
    grad *= scale
    return [(loss.double().sum() / n).float(), grad.to(s["logits"].dtype)]


def _plain_unpack(records, k, bits):
    """Values (fp32) and indices of saved records."""
    off = records[:, 0:4].contiguous().view(torch.float32)
    scale = records[:, 4:8].contiguous().view(torch.float32)
    index = records[:, 8:8 + 2 * k].contiguous().view(torch.int16).to(torch.int32)
    codes = records[:, 8 + 2 * k:8 + 2 * k + (k * bits + 7) // 8]
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1)[:, :k]
    values = off - codes.float() * scale
    return values.masked_fill(index < 0, -math.inf), index


def _plain_write(s):
    case = s["case"]
    k, c = case["k"], case["c"]
    z = s["logits"].float()
    usable = (z > torch.finfo(s["logits"].dtype).min) & (z < math.inf)
    order = torch.sort(torch.where(usable, z, torch.full_like(z, -math.inf)), dim=1, descending=True, stable=True)
    v, index = order.values[:, :k], order.indices[:, :k].to(torch.int32)
    if k > c:
        v = torch.nn.functional.pad(v, (0, k - c), value=-math.inf)
        index = torch.nn.functional.pad(index, (0, k - c), value=-1)
    here = v > -math.inf
    index = torch.where(here, index, torch.full_like(index, -1))
    # In 64 bits: with few mantissa bits in the logits, many quotients lie exactly between two codes.
    v = v.double()
    first = torch.where(here[:, :1], v[:, :1], torch.zeros_like(v[:, :1]))
    last = torch.where(here, v, first).amin(dim=1, keepdim=True)
    levels = _LEVELS[case["bits"]]
    span = first - last
    code = torch.where(here & (span > 0), torch.round((first - v) * levels / span), torch.zeros_like(v))
    value = first.float() - code.float() * (span / levels).float()
    return [value.masked_fill(~here, -math.inf), index]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind in ("decode", "decode_train"):
            return _plain_decode(state)
        if kind in ("distill_eval", "distill_train"):
            return _plain_distill(state, state["values"], state["index"])
        if kind == "distill_cached":
            values, index = _plain_unpack(state["records"][state["pick"]], case["k"], case["bits"])
            return _plain_distill(state, values, index)
        if kind == "cache_write":
            return _plain_write(state)
        return list(_plain_unpack(state["records"][state["pick"]], case["k"], case["bits"]))

    from mlx3d_b200.losses import distill_loss, distill_loss_and_grad
    from mlx3d_b200.splatting import decode_features

    if kind in ("decode", "decode_train"):
        leaves = [state[n] for n in ("x", "w_gate", "w_up", "w_down")]
        y = decode_features(*leaves, activation=case["act"])
        if kind == "decode":
            return y
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    if kind == "distill_eval":
        return distill_loss(state["logits"], (state["values"], state["index"]), temperature=case["t"],
                            weight=state["weight"], reduction="none")
    if kind in ("distill_train", "distill_cached"):
        teacher = state["cache"].at(state["pick"]) if kind == "distill_cached" else (state["values"], state["index"])
        return list(distill_loss_and_grad(state["logits"], teacher, temperature=case["t"], weight=state["weight"],
                                          reduction=case["reduction"]))
    if kind == "cache_write":
        cache, start = state["cache"], state["start"]
        cache.write(start, state["logits"])
        return list(cache.read(slice(start, start + case["rows"])))
    return list(state["cache"].read(state["pick"]))


# ---------------------------------------------------------------------- work
def work(case):
    kind, p, c = case["kind"], case["rows"], case["c"]
    if kind in ("decode", "decode_train"):
        d, f = case["d"], case["f"]
        weights = 2 * (2 * f * d + c * f)
        flops = 2 * p * (2 * d * f + f * c)
        if kind == "decode":
            return {"bytes": 2 * p * (d + c) + weights, "flops": flops}
        return {"bytes": 2 * p * (2 * d + 2 * c) + 2 * weights, "flops": 3 * flops}
    k = case["k"]
    if kind.startswith("distill"):
        size = 4 if case["type"] == "fp32" else 2
        teacher = _record_bytes(k, case["bits"]) + 8 if kind == "distill_cached" else 6 * k
        if kind == "distill_eval":
            return {"bytes": p * (c * size + teacher + 8), "flops": 4 * p * c}
        return {"bytes": p * (2 * c * size + teacher + 4), "flops": 6 * p * c}
    if kind == "cache_write":  # the logits, the records (written and read back), values and indices
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": p * (c * size + 2 * _record_bytes(k, case["bits"]) + 8 * k), "flops": p * c}
    return {"bytes": p * (_record_bytes(k, case["bits"]) + 8 + 8 * k), "flops": 2 * p * k}


# --------------------------------------------------------------- 64-bit forms
def _exact_decode(case, s):
    ty = torch.float64
    wg, wu, wd = (s[n].detach().to(ty) for n in ("w_gate", "w_up", "w_down"))
    ys, dxs = [], []
    sums = [torch.zeros_like(w) for w in (wg, wu, wd)]
    for lo in range(0, case["rows"], 1 << 18):
        x = s["x"].detach()[lo:lo + (1 << 18)].to(ty)
        g, u = torch.einsum("pd,fd->pf", x, wg), torch.einsum("pd,fd->pf", x, wu)
        if case["act"] == "silu":
            half = 0.5 * (1.0 + torch.tanh(0.5 * g))  # the logistic function
            a, slope = g * half, half + g * half * (1.0 - half)
        else:
            phi = 0.5 * torch.erfc(-g / 2.0 ** 0.5)
            a, slope = g * phi, phi + g * torch.exp(-(g ** 2) / 2.0) / (2.0 * math.pi) ** 0.5
        ys.append(torch.einsum("pf,cf->pc", a * u, wd))
        if case["kind"] == "decode":
            continue
        dy = s["dy"][lo:lo + (1 << 18)].to(ty)
        dh = torch.einsum("pc,cf->pf", dy, wd)
        sums[2] += torch.einsum("pc,pf->cf", dy, a * u)
        dg, du = dh * u * slope, dh * a
        sums[0] += torch.einsum("pf,pd->fd", dg, x)
        sums[1] += torch.einsum("pf,pd->fd", du, x)
        dxs.append(torch.einsum("pf,fd->pd", dg, wg) + torch.einsum("pf,fd->pd", du, wu))
    return torch.cat(ys) if case["kind"] == "decode" else [torch.cat(ys), torch.cat(dxs), *sums]


def _exact_records(rec, k, bits):
    head = rec[:, :8].contiguous().view(torch.float32).double()
    index = rec[:, 8:8 + 2 * k].contiguous().view(torch.int16).int()
    raw = rec[:, 8 + 2 * k:].int()
    col = torch.arange(k, device="cuda")
    code = raw[:, col] if bits == 8 else (raw[:, col // 2] >> (4 * (col % 2))) & 15
    values = head[:, :1] - code.double() * head[:, 1:]
    return torch.where(index >= 0, values, -math.inf), index


def _exact_distill(case, s):
    t, c, p = case["t"], case["c"], case["rows"]
    losses, grads = [], []
    n = p if case.get("reduction") == "mean" else 1
    step = max(1, (1 << 27) // c)
    for lo in range(0, p, step):
        z = s["logits"][lo:lo + step].double() / t
        w = s["weight"][lo:lo + step].double()
        if case["kind"] == "distill_cached":
            v, i = _exact_records(s["records"][s["pick"][lo:lo + step]], case["k"], case["bits"])
        else:
            v, i = s["values"][lo:lo + step].double(), s["index"][lo:lo + step]
        i = i.long()
        gone = (i < 0) | (i >= c) | (v == -math.inf)
        i = i.masked_fill(gone, 0)
        empty = gone.all(dim=1, keepdim=True)
        logp = (v / t).masked_fill(gone, -math.inf)
        logp = logp - torch.logsumexp(logp.masked_fill(empty, 0.0), dim=1, keepdim=True)
        prob = torch.exp(logp).masked_fill(gone, 0.0)
        logq = z - torch.logsumexp(z, dim=1, keepdim=True)
        part = (prob * (logp.masked_fill(gone, 0.0) - logq.gather(1, i))).masked_fill(prob == 0, 0.0)
        losses.append(w * t * t * part.sum(dim=1))
        if case["kind"] != "distill_eval":
            q = torch.exp(logq).scatter_add(1, i, -prob).masked_fill(empty, 0.0)
            grads.append(q * (w[:, None] * t / n))
    loss = torch.cat(losses)
    return loss if case["kind"] == "distill_eval" else [loss.sum() / n, torch.cat(grads)]


def _exact_write(case, s):
    k, c = case["k"], case["c"]
    levels = 2.0 ** case["bits"] - 1.0
    lowest = torch.finfo(s["logits"].dtype).min
    values, indices = [], []
    step = max(1, (1 << 27) // c)
    for lo in range(0, case["rows"], step):
        z = s["logits"][lo:lo + step].double()
        z = z.masked_fill((z <= lowest) | ~torch.isfinite(z), -math.inf)
        v, i = z.sort(dim=1, descending=True, stable=True)
        n = z.shape[0]
        full = torch.full((n, k), -math.inf, dtype=torch.float64, device="cuda")
        index = torch.full((n, k), -1, dtype=torch.int32, device="cuda")
        m = min(k, c)
        full[:, :m], index[:, :m] = v[:, :m], i[:, :m].int()
        gone = full == -math.inf
        index[gone] = -1
        high = full[:, :1].masked_fill(gone[:, :1], 0.0)
        low = full.masked_fill(gone, math.inf).amin(dim=1, keepdim=True)
        span = (high - low).masked_fill(gone[:, :1], 0.0)
        place = ((high - full).masked_fill(gone, 0.0) * levels).div(span).masked_fill(span == 0, 0.0)
        code = place.floor()  # to the nearest, halves to the even code
        rest = place - code
        code = torch.where((rest > 0.5) | ((rest == 0.5) & (code % 2 == 1)), code + 1.0, code)
        values.append((high - code * span / levels).masked_fill(gone, -math.inf))
        indices.append(index)
    return [torch.cat(values), torch.cat(indices)]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("decode", "decode_train"):
        return _exact_decode(case, s)
    if kind.startswith("distill"):
        return _exact_distill(case, s)
    if kind == "cache_write":
        return _exact_write(case, s)
    return list(_exact_records(s["records"][s["pick"]], case["k"], case["bits"]))
