"""Per-step inputs: host-to-device staging, and teacher targets kept on the device.

Double-buffered host-to-device staging of per-step inputs.

The reference trains from host-resident arrays (MLX unified memory); on a
discrete GPU each step's inputs must cross PCIe.  ``HostStager`` keeps two
device copies of a set of tensors and fills one on a dedicated copy stream
while the compute stream works on the other, so the copy of step k+1 runs
under the kernels of step k.  Every step still copies all of its inputs:
nothing is cached across steps.

Ordering is carried by CUDA events only (no host synchronisation):
  * the compute stream waits for the copy that filled the slot it acquires;
  * a copy into a slot waits for the compute work that last read that slot
    (recorded by :meth:`release`).

``TeacherCache`` keeps a 2D network's largest logits of every training pixel
on the device, quantised as they are written (an addition; the reference has
no per-pixel teacher targets).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native as nat

__all__ = ["HostStager", "TeacherCache", "TeacherRows"]


class HostStager:
    def __init__(self, like: dict[str, torch.Tensor], device, requires_grad: tuple[str, ...] = ()):
        """``like`` gives the names, shapes and dtypes of the staged tensors;
        names in ``requires_grad`` are made autograd leaves on the device."""
        self.device = torch.device(device)
        self.copy_stream = torch.cuda.Stream(device=self.device)
        self.slots = []
        for _ in range(2):
            slot = {k: torch.empty(v.shape, dtype=v.dtype, device=self.device) for k, v in like.items()}
            for k in requires_grad:
                slot[k].requires_grad_(True)
            self.slots.append(slot)
        self._filled = [None, None]
        self._released = [None, None]
        self._next = 0
        self._pending: list[int] = []

    def h2d_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.slots[0].values())

    def prefetch(self, host: dict[str, torch.Tensor]) -> None:
        """Queue the copy of ``host`` (pinned tensors) into the next free slot."""
        if len(self._pending) >= 2:
            raise RuntimeError("HostStager: both slots are already filled; acquire() one first")
        for k, dst in self.slots[0].items():
            if not host[k].is_pinned():
                raise ValueError(f"HostStager: host tensor {k!r} must be in pinned memory")
        i = self._next
        self._next ^= 1
        with torch.cuda.stream(self.copy_stream):
            if self._released[i] is not None:
                self.copy_stream.wait_event(self._released[i])
            with torch.no_grad():
                for k, dst in self.slots[i].items():
                    dst.copy_(host[k], non_blocking=True)
            ev = torch.cuda.Event()
            ev.record(self.copy_stream)
        self._filled[i] = ev
        self._pending.append(i)

    def acquire(self) -> tuple[int, dict[str, torch.Tensor]]:
        """The oldest filled slot, ordered after its copy on the current stream."""
        if not self._pending:
            raise RuntimeError("HostStager: nothing prefetched")
        i = self._pending.pop(0)
        torch.cuda.current_stream(self.device).wait_event(self._filled[i])
        return i, self.slots[i]

    def release(self, i: int) -> None:
        """Mark the current stream's work on slot ``i`` as the point after which
        the next copy into it may start."""
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(self.device))
        self._released[i] = ev


@dataclass(frozen=True)
class TeacherRows:
    """Rows of a :class:`TeacherCache`, as ``distill_loss`` takes them."""

    cache: "TeacherCache"
    rows: torch.Tensor | None  # int64 row numbers, or None for [first, first + count)
    first: int
    count: int


class TeacherCache:
    """A teacher's ``k`` largest logits per row (pixel), in ``bits`` (8 or 4) bits.

    The teacher runs once per view; its full logits do not fit for hundreds of views, its largest ones do.
    Each row is one record of :attr:`record_bytes` bytes in :attr:`records`: the largest logit and a step
    (float32), k class indices (int16) and k codes, ``value = largest - code * step``.  Rows that were never
    written hold no entries.  Reads and writes run on the current stream of the cache's device; a program that
    uses several streams orders them itself.
    """

    def __init__(self, rows: int, k: int, num_classes: int, bits: int = 8, device="cuda"):
        rows, k, num_classes = int(rows), int(k), int(num_classes)
        if rows < 0:
            raise ValueError("rows must not be negative.")
        if not 1 <= k <= nat.GS_CACHE_MAX_K:
            raise ValueError(f"k must be in [1, {nat.GS_CACHE_MAX_K}].")
        if not 1 <= num_classes <= nat.GS_CACHE_MAX_CLASSES:
            raise ValueError(f"num_classes must be in [1, {nat.GS_CACHE_MAX_CLASSES}].")
        if bits not in (4, 8):
            raise ValueError("bits must be 8 or 4.")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"device must be a CUDA device (got {device}); mlx3d_b200 has no CPU path")
        self.num_rows, self.k, self.num_classes, self.bits = rows, k, num_classes, int(bits)
        self.record_bytes = int(nat.load().gs_teacher_record_bytes(k, self.bits))
        # An ordinary tensor even where the cache is made beside a teacher that runs in inference mode: losses save
        # it for their backward.
        with torch.inference_mode(False):
            self.records = torch.zeros((rows, self.record_bytes), dtype=torch.uint8, device=device)
            self.records[:, 8:8 + 2 * k] = 255  # index -1: absent
        self.device = self.records.device

    def __len__(self) -> int:
        return self.num_rows

    def at(self, rows) -> TeacherRows:
        """The rows of one call: a ``slice`` (step 1, within the cache) or an int64 / int32 tensor of row
        numbers on the cache's device, any shape; numbers outside [0, len(cache)) stand for rows without
        entries."""
        if isinstance(rows, slice):
            if rows.step not in (None, 1):
                raise ValueError("a slice of the teacher cache must have step 1.")
            first = 0 if rows.start is None else int(rows.start)
            stop = self.num_rows if rows.stop is None else int(rows.stop)
            if not 0 <= first <= stop <= self.num_rows:
                raise ValueError(f"rows [{first}, {stop}) are outside the cache of {self.num_rows} rows.")
            return TeacherRows(self, None, first, stop - first)
        if not isinstance(rows, torch.Tensor) or rows.dtype not in (torch.int64, torch.int32):
            raise TypeError("rows must be a slice or an int64 / int32 tensor.")
        rows = nat.require_cuda("rows", rows, torch.int64)
        nat.same_device(self.device, rows=rows)
        return TeacherRows(self, rows, 0, rows.numel())

    def write(self, start: int, logits: torch.Tensor) -> None:
        """Rows [start, start + n) from the teacher's full logits (..., num_classes), n rows in all: the k
        largest, largest first, equal ones by lowest index.  Infinities, NaN and the type's lowest value (a
        masked class) are never taken; a row with fewer than k usable classes leaves its last entries absent."""
        if not isinstance(logits, torch.Tensor) or logits.ndim < 1 or logits.shape[-1] != self.num_classes:
            raise ValueError(f"logits must have shape (..., {self.num_classes}).")
        n = logits.numel() // self.num_classes
        start = int(start)
        if start < 0 or start + n > self.num_rows:
            raise ValueError(f"rows [{start}, {start + n}) are outside the cache of {self.num_rows} rows.")
        logits = nat.require_float("logits", logits.detach() if logits.requires_grad else logits)
        nat.same_device(self.device, logits=logits)
        nat.call_on(self.device, "gs_teacher_write", nat.ptr(logits), nat.DTYPES[logits.dtype], n, self.num_classes,
                    nat.ptr(self.records), self.num_rows, start, self.k, self.bits)
        # a loss that was computed from the old rows must not run its backward on the new ones
        torch.autograd.graph.increment_version(self.records)

    def read(self, rows) -> tuple[torch.Tensor, torch.Tensor]:
        """``(values, index)`` of :meth:`at`'s rows, (..., k): float32 values (-inf where absent) and int32
        class indices (-1 where absent)."""
        at = self.at(rows)
        shape = ((at.count,) if at.rows is None else tuple(at.rows.shape)) + (self.k,)
        values = torch.empty(shape, dtype=torch.float32, device=self.device)
        index = torch.empty(shape, dtype=torch.int32, device=self.device)
        nat.call_on(self.device, "gs_teacher_read", nat.ptr(self.records), self.num_rows, nat.ptr(at.rows), at.first,
                    at.count, self.k, self.bits, nat.ptr(values), nat.ptr(index))
        return values, index

    def state_dict(self) -> dict:
        return {"records": self.records.clone(), "k": self.k, "num_classes": self.num_classes, "bits": self.bits}

    def load_state_dict(self, state: dict) -> None:
        """Copy saved records into this cache (same rows, k, num_classes and bits)."""
        for name in ("k", "num_classes", "bits"):
            if name in state and int(state[name]) != getattr(self, name):
                raise ValueError(f"the saved cache has {name} = {state[name]}, this one {getattr(self, name)}.")
        rec = state["records"]
        if rec.dtype != torch.uint8 or tuple(rec.shape) != tuple(self.records.shape):
            raise ValueError(f"records must be uint8 of shape {tuple(self.records.shape)}.")
        self.records.copy_(rec)
