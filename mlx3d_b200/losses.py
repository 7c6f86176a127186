"""Image losses of the 3DGS training recipe (src/mlx3d/losses/image_metrics.py).

``ssim`` and ``l1_dssim_loss`` run on the fused sm_100a kernels behind
``gs_l1_ssim_forward`` / ``gs_l1_ssim_backward``: one forward kernel for the
five windowed statistics, the SSIM and L1 sums, one backward kernel for the
gradient of both terms.  ``l1_loss`` runs on ``gs_l1_forward`` /
``gs_l1_backward``; ``psnr`` is a one-line reduction.

``distill_loss`` (an addition to the reference's losses) trains rendered or
decoded class logits against a 2D teacher's largest logits, given as arrays
or kept in a :class:`~mlx3d_b200.staging.TeacherCache`, on ``gs_distill``.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .staging import TeacherRows

__all__ = ["ssim", "l1_loss", "psnr", "l1_dssim_loss", "distill_loss", "distill_loss_and_grad"]


def _prep(pred, target):
    if pred.shape != target.shape:
        raise ValueError("pred and target must have the same shape.")
    if pred.ndim == 4:
        if pred.shape[0] != 1:
            raise ValueError("batched SSIM supports a batch of one image (N=1).")
        pred, target = pred[0], target[0]
    if pred.ndim != 3:
        raise ValueError("images must have shape (H, W, C) or (1, H, W, C).")
    return nat.require_cuda("pred", pred), nat.require_cuda("target", target.detach())


class _L1DSSIM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target, lam, max_val, window_size, sigma):
        H, W, C = pred.shape
        lib = nat.load()
        ws = torch.empty((lib.gs_l1_ssim_workspace_bytes(H, W, C),), device=pred.device, dtype=torch.uint8)
        loss = torch.empty((3,), device=pred.device, dtype=torch.float32)
        nat.call("gs_l1_ssim_forward", nat.ptr(pred), nat.ptr(target), H, W, C, lam, max_val, window_size, sigma,
                 nat.ptr(ws), ws.numel(), nat.ptr(loss), nat.stream())
        ctx.save_for_backward(pred, target, ws)
        ctx.args = (lam, max_val, window_size, sigma)
        return loss[0], loss[1], loss[2]

    @staticmethod
    def backward(ctx, g_loss, g_l1, g_ssim):
        pred, target, ws = ctx.saved_tensors
        lam, max_val, window_size, sigma = ctx.args
        H, W, C = pred.shape
        grad = torch.empty_like(pred)
        # d total = g_loss * d loss + g_l1 * d l1 + g_ssim * d ssim, each term linear in the
        # kernel's (l1 weight, ssim weight) = (1 - lam, -lam): one launch per needed term, the
        # cotangent read on the device, the later terms accumulated into the first.
        terms = []
        if g_loss is not None:
            terms.append((g_loss, 1.0, lam))
        if g_l1 is not None:
            terms.append((g_l1, 1.0, 0.0))
        if g_ssim is not None:
            terms.append((g_ssim, -1.0, 1.0))
        if not terms:
            return torch.zeros_like(pred), None, None, None, None, None
        for k, (g, sign, lam_k) in enumerate(terms):
            g = g.detach().to(torch.float32).contiguous()
            nat.call("gs_l1_ssim_backward_dev", nat.ptr(pred), nat.ptr(target), H, W, C, lam_k, window_size,
                     sigma, nat.ptr(ws), ws.numel(), nat.ptr(g), sign, int(k > 0), nat.ptr(grad), nat.stream())
        return grad, None, None, None, None, None


class _L1(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target):
        lib = nat.load()
        n = pred.numel()
        ws = torch.empty((lib.gs_l1_workspace_bytes(n),), device=pred.device, dtype=torch.uint8)
        loss = torch.empty((1,), device=pred.device, dtype=torch.float32)
        nat.call("gs_l1_forward", nat.ptr(pred), nat.ptr(target), n, nat.ptr(ws), ws.numel(), nat.ptr(loss),
                 nat.stream())
        ctx.save_for_backward(pred, target)
        return loss[0]

    @staticmethod
    def backward(ctx, g):
        pred, target = ctx.saved_tensors
        grad = torch.empty_like(pred)
        g = g.detach().to(torch.float32).contiguous()
        nat.call("gs_l1_backward", nat.ptr(pred), nat.ptr(target), pred.numel(), nat.ptr(g), nat.ptr(grad),
                 nat.stream())
        return grad, None


def l1_dssim_loss(pred: torch.Tensor, target: torch.Tensor, lambda_dssim: float = 0.2, max_val: float = 1.0,
                  window_size: int = 11, sigma: float = 1.5):
    """``(1 - lambda) * mean|pred - target| + lambda * (1 - ssim(pred, target))``
    (trainer.py:300-305); returns ``(loss, l1, ssim)`` scalar tensors."""
    pred, target = _prep(pred, target)
    return _L1DSSIM.apply(pred, target, float(lambda_dssim), float(max_val), int(window_size), float(sigma))


def ssim(pred: torch.Tensor, target: torch.Tensor, max_val: float = 1.0, window_size: int = 11,
         sigma: float = 1.5) -> torch.Tensor:
    """Mean SSIM with a Gaussian window (image_metrics.py:66-85); differentiable in pred."""
    return l1_dssim_loss(pred, target, 1.0, max_val, window_size, sigma)[2]


def l1_loss(pred: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """mean |pred - target| on the fused sm_100a kernels (deterministic sum);
    differentiable in pred."""
    if pred.shape != target.shape:
        raise ValueError("pred and target must have the same shape.")
    pred = nat.require_cuda("pred", pred)
    target = nat.require_cuda("target", target.detach())
    return _L1.apply(pred.contiguous(), target.contiguous())


def psnr(pred: torch.Tensor, target: torch.Tensor, max_val: float = 1.0) -> torch.Tensor:
    mse = ((pred - target) ** 2).mean()
    return 10.0 * torch.log10((max_val * max_val) / torch.clamp(mse, min=1e-12))


def _plain(t: torch.Tensor) -> torch.Tensor:
    return t.detach() if t.requires_grad else t


class _DistillArgs:
    """Checked arguments of one distillation call; keeps the tensors alive."""

    def __init__(self, logits, teacher, temperature, weight, reduction):
        if reduction not in ("mean", "sum", "none"):
            raise ValueError("reduction must be 'mean', 'sum' or 'none'.")
        temperature = float(temperature)
        if not nat.GS_DISTILL_MIN_TEMPERATURE <= temperature <= nat.GS_DISTILL_MAX_TEMPERATURE:
            raise ValueError(f"temperature must be in [{nat.GS_DISTILL_MIN_TEMPERATURE:g}, "
                             f"{nat.GS_DISTILL_MAX_TEMPERATURE:g}].")
        if not isinstance(logits, torch.Tensor) or logits.ndim < 1 or logits.shape[-1] < 1:
            raise ValueError("logits must have shape (..., C) with C >= 1.")
        lead = logits.shape[:-1]
        self.rows = math.prod(lead)
        if reduction == "mean" and self.rows == 0:
            raise ValueError("reduction='mean' needs at least one row of logits.")
        self.records = self.row_ids = self.values = self.index = None
        if isinstance(teacher, TeacherRows):
            if teacher.count != self.rows:
                raise ValueError(f"teacher has {teacher.count} rows, logits {self.rows}.")
            if teacher.cache.num_classes != logits.shape[-1]:
                raise ValueError(f"the teacher cache holds {teacher.cache.num_classes} classes, "
                                 f"logits have {logits.shape[-1]}.")
        elif isinstance(teacher, (tuple, list)) and len(teacher) == 2:
            values, index = teacher
            if not isinstance(values, torch.Tensor) or not isinstance(index, torch.Tensor):
                raise TypeError("teacher must be (values, index) tensors or TeacherCache.at(rows).")
            if values.ndim != logits.ndim or values.shape[:-1] != lead or values.shape != index.shape:
                raise ValueError("teacher values and index must both have shape (..., K) with the logits' rows.")
            if not 1 <= values.shape[-1] <= nat.GS_TEACHER_MAX_K:
                raise ValueError(f"the teacher must have 1 to {nat.GS_TEACHER_MAX_K} entries a row.")
            if index.dtype not in (torch.int32, torch.int64, torch.int16):
                raise TypeError("teacher index must be int16, int32 or int64.")
        else:
            raise TypeError("teacher must be (values, index) tensors or TeacherCache.at(rows).")
        if weight is not None and (not isinstance(weight, torch.Tensor) or weight.shape != lead):
            raise ValueError("weight must have the shape of the logits' rows.")
        logits = nat.require_float("logits", logits)
        dev = logits.device
        if isinstance(teacher, TeacherRows):
            cache = teacher.cache
            self.records, self.row_ids = cache.records, teacher.rows
            self.native = nat.GsTeacher(None, None, cache.records.data_ptr(), nat.ptr(teacher.rows), teacher.first,
                                        cache.num_rows, 0, cache.k, cache.bits)
        else:
            self.values = nat.require_float("teacher values", _plain(teacher[0]))
            index = teacher[1]
            if index.dtype == torch.int64:  # out of int32's range is out of the classes' range
                index = index.clamp(-1, 2**31 - 1)
            self.index = nat.require_cuda("teacher index", index, torch.int32)
            self.native = nat.GsTeacher(self.values.data_ptr(), self.index.data_ptr(), None, None, 0, 0,
                                        nat.DTYPES[self.values.dtype], self.values.shape[-1], 0)
        self.weight = None if weight is None else nat.require_cuda("weight", _plain(weight))
        if self.records is None:
            nat.same_device(dev, teacher_values=self.values, teacher_index=self.index, weight=self.weight)
        else:
            nat.same_device(dev, teacher=self.records, weight=self.weight)
        self.logits = logits
        self.lead = lead
        self.temperature = temperature
        self.reduction = reduction
        self.scale = 1.0 / self.rows if reduction == "mean" else 1.0

    def run(self, logits, want_loss=True, grad=None, cotangent=None):
        """One launch: the loss (row losses for 'none') and / or the gradient into ``grad``."""
        dev = logits.device
        row_loss = loss = ws = None
        if want_loss:
            if self.reduction == "none":
                row_loss = torch.empty(self.lead, device=dev, dtype=torch.float32)
            else:
                loss = torch.empty((), device=dev, dtype=torch.float32)
                ws = torch.empty((nat.distill_workspace_bytes(),), device=dev, dtype=torch.uint8)
        nat.call_on(dev, "gs_distill", nat.ptr(logits), nat.DTYPES[logits.dtype], self.rows, logits.shape[-1],
                    ctypes.byref(self.native), self.temperature, nat.ptr(self.weight), self.scale,
                    nat.ptr(cotangent), int(self.reduction == "none"), nat.ptr(row_loss), nat.ptr(loss),
                    nat.ptr(grad), nat.ptr(ws), 0 if ws is None else ws.numel())
        return row_loss if self.reduction == "none" else loss


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):
        ctx.args = args
        ctx.save_for_backward(logits, args.records, args.row_ids, args.values, args.index, args.weight)
        args.logits = None  # saved above
        return args.run(logits)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits = ctx.saved_tensors[0]
        grad = torch.empty_like(logits)
        ctx.args.run(logits, want_loss=False, grad=grad, cotangent=g.to(torch.float32).contiguous())
        return grad, None


def distill_loss(logits: torch.Tensor, teacher, temperature: float = 1.0, weight: torch.Tensor | None = None,
                 reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's largest logits; differentiable (reverse mode) in ``logits``.

    ``logits`` (..., C), float32, float16 or bfloat16: class logits of rendered pixels (for instance
    ``render_features(...)["logits"]``).  ``teacher`` is ``(values, index)``, both (..., K) with K <= 256, or
    ``TeacherCache.at(rows)``.  Per row, with p the softmax of the teacher's values / T over its entries and q
    the softmax of logits / T over all C classes::

        L = weight * T^2 * sum_k p_k (log p_k - log q[index_k])

    with 1e-18 <= T <= 1e18 (T^2 is a 32-bit factor).  An entry whose index is outside [0, C) or whose value is
    -inf is absent; a row without entries (an unlabelled pixel) has loss and gradient 0.  Entries of one class add up.  ``reduction`` is "mean" (over all rows), "sum"
    or "none" (a float32 loss per row).  With float16 logits take "sum": a mean's gradients, of the order of
    1 / rows, fall below float16's range.  No gradient flows to the teacher or to ``weight``."""
    args = _DistillArgs(logits, teacher, temperature, weight, reduction)
    if nat.differentiated(args.logits):
        return _Distill.apply(args.logits, args)
    return args.run(args.logits)


def distill_loss_and_grad(logits: torch.Tensor, teacher, temperature: float = 1.0,
                          weight: torch.Tensor | None = None,
                          reduction: str = "mean") -> tuple[torch.Tensor, torch.Tensor]:
    """``distill_loss`` and its gradient with respect to ``logits`` (their shape and type) in one pass over the
    logits, outside autograd: hand the gradient on with ``logits.backward(grad)``.  With ``reduction="none"``
    each row's gradient is its own loss's."""
    args = _DistillArgs(_plain(logits) if isinstance(logits, torch.Tensor) else logits, teacher, temperature, weight,
                        reduction)
    grad = torch.empty_like(args.logits)
    loss = args.run(args.logits, grad=grad)
    return loss, grad
