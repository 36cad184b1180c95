"""The global norm over many gradient tensors and clipping by it (``sm_grad_norm`` / ``sm_grad_clip``; csrc/gradnorm.hip):
``Trainer(gradient_clip_val=...)`` of the reference's pytorch_lightning (requirements.txt:76), i.e.
``torch.nn.utils.clip_grad_norm_``, as two launches per 120 tensors with no host synchronisation.

    norm = sqrt(sum of all squares) or max |g|;   out = g * min(1, max_norm / (norm + 1e-6))

float32 / bfloat16 / float16 tensors may be mixed. Sums are held in 64 bits; the norm has the same bits every time. A norm
that is not finite is not an error (finding out would synchronise): the coefficient follows the formula, infinity clips to 0
(and infinity * 0 = NaN), a NaN makes every gradient NaN.
"""
from __future__ import annotations

import math
from array import array
from operator import attrgetter

import numpy as np
import torch

from . import hip, ops

_TYPE_ID = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}           # SM_TYPE_*
_SIZE = (4, 2, 2)
_T = torch.Tensor
_dtype = attrgetter("dtype")


def _dense(t) -> bool:
    """One element per address of a range: a permutation of a contiguous tensor."""
    want = 1
    for st, sz in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if st != want:
            return False
        want *= sz
    return True


class _Table:
    """Pointers, element counts and types of a list of tensors as the library reads them. A list is walked once per attribute
    with C-level maps: a model's few hundred tensors are handed over anew every step, and at a microsecond a tensor the walk
    would be the operator's time."""

    def __init__(self, tensors, what):
        kinds = set(map(_dtype, tensors))
        if not kinds <= _TYPE_ID.keys():
            raise ValueError(f"{what}: {[str(d) for d in kinds - _TYPE_ID.keys()]} (float32, bfloat16 or float16)")
        if len(kinds) == 1:
            self.types = array("i", [_TYPE_ID[kinds.pop()]]) * len(tensors)
        else:
            self.types = array("i", [_TYPE_ID[d] for d in map(_dtype, tensors)])
        devices = set(map(_T.get_device, tensors))
        if -1 in devices:
            raise ValueError(f"{what}: device tensors only (there is no CPU form)")
        if devices and devices != {torch.cuda.current_device()}:
            raise ValueError(f"{what}: tensors on devices {sorted(devices)}, the current device is cuda:{torch.cuda.current_device()}")
        self.contiguous = list(map(_T.is_contiguous, tensors))
        if not all(self.contiguous):
            for t, ok in zip(tensors, self.contiguous):
                if not ok and not _dense(t):
                    raise ValueError(f"{what}: strides {t.stride()} of {tuple(t.shape)} leave gaps or overlap")
        self.ptrs = array("Q", map(_T.data_ptr, tensors))
        self.numel = array("Q", map(_T.numel, tensors))
        self.n = len(tensors)

    def spans(self):
        start = np.frombuffer(self.ptrs, dtype=np.uint64)
        size = np.asarray(_SIZE, dtype=np.uint64)[np.frombuffer(self.types, dtype=np.int32)]
        return start, start + np.frombuffer(self.numel, dtype=np.uint64) * size


def _address(a) -> int | None:
    return a.buffer_info()[0] if len(a) else None


def _norm_kind(norm_type) -> int:
    n = float(norm_type)
    if n == 2.0:
        return 0
    if n == math.inf:
        return 1
    raise ValueError(f"norm_type={norm_type!r}: 2 or inf")


def _max_norm(v) -> float:
    v = float(v)
    if not v >= 0.0:
        raise ValueError(f"max_norm={v}: a number >= 0")
    return v


def _refuse_overlap(g: _Table, o: _Table):
    """What is written must be written once: an output that overlaps another output, or a gradient other than its own
    (the same tensor listed twice, for one), has no defined result."""
    if g.n == 0:
        return
    os_, oe = o.spans()
    live = np.nonzero(oe > os_)[0]
    if live.size == 0:
        return
    order = live[np.argsort(os_[live], kind="stable")]
    ss, ee = os_[order], oe[order]
    if (ee[:-1] > ss[1:]).any():
        raise ValueError("two of the tensors to be written overlap (a gradient listed twice?)")
    if o is g:
        return
    gs, ge = g.spans()
    lo, hi = np.searchsorted(ee, gs, "right"), np.searchsorted(ss, ge, "left")      # outputs that gradient i touches
    for i in np.nonzero((hi > lo) & (ge > gs))[0]:
        if hi[i] - lo[i] > 1 or order[lo[i]] != i or os_[i] != gs[i]:
            raise ValueError("an output overlaps a gradient that is not its own")


class GradClip:
    """The call's tables for gradients that stay where they are (an arena's views, ``zero_grad(set_to_none=False)``): checked
    and laid out once, used every step. Keeps the tensors alive; ``grads`` may hold None (a parameter without a gradient).
    ``out``: one tensor per gradient that receives the clipped values, of any of the three types (both contiguous with as
    many elements, or the same shape and strides); None: the gradients themselves are scaled in place (where nothing is clipped the second pass ends at once).
    Calls on two streams need the caller's ordering only where both write the same outputs: each has scratch of its own."""

    def __init__(self, grads, out=None):
        grads = list(grads)
        if out is not None:
            out = list(out)
            if len(out) != len(grads):
                raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")
        if type(None) in set(map(type, grads)):
            out = None if out is None else [o for o, g in zip(out, grads) if g is not None]
            grads = [g for g in grads if g is not None]
        self.grads, self.out = grads, grads if out is None else out
        g = self._g = _Table(grads, "grads")
        if out is None or not grads:
            o = self._o = g
        else:
            if type(None) in set(map(type, out)):
                raise ValueError("an output is missing for a gradient that is there")
            o = self._o = _Table(out, "out")
            if g.numel != o.numel:
                raise ValueError("an output has not as many elements as its gradient")
            if not (all(g.contiguous) and all(o.contiguous)):
                for a, b, ca, cb in zip(grads, out, g.contiguous, o.contiguous):
                    if not (ca and cb) and (a.shape != b.shape or a.stride() != b.stride()):
                        raise ValueError(f"out {tuple(b.shape)} / {b.stride()} does not match its gradient {tuple(a.shape)} / {a.stride()}")
            same = np.frombuffer(g.ptrs, dtype=np.uint64) == np.frombuffer(o.ptrs, dtype=np.uint64)
            if (same & (np.frombuffer(g.numel, dtype=np.uint64) > 0) & (np.frombuffer(g.types, np.int32) != np.frombuffer(o.types, np.int32))).any():
                raise ValueError("an output that is its gradient must have its type")
        _refuse_overlap(g, o)
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._args = (_address(g.ptrs), _address(o.ptrs), _address(g.numel), _address(g.types), _address(o.types), g.n)
        self._ws_bytes = ops.lib.sm_grad_norm_ws_bytes(g.n)

    def _result(self):
        """(norm, scratch) of one call: two streams, or two captured graphs, of one plan share nothing"""
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the plan's tensors live on {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        return (torch.empty((), dtype=torch.float32, device=self.device),
                torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device))

    def norm(self, norm_type=2.0) -> torch.Tensor:
        """The global norm as a float32 device scalar."""
        kind = _norm_kind(norm_type)
        out, ws = self._result()
        gp, _, numel, types, _, n = self._args
        hip.check(ops.lib.sm_grad_norm(gp, numel, types, n, kind, ws.data_ptr(), self._ws_bytes, out.data_ptr(), hip.stream()), "sm_grad_norm")
        return out

    def clip(self, max_norm, norm_type=2.0) -> torch.Tensor:
        """Clips, and returns the norm BEFORE clipping (float32 device scalar)."""
        kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
        out, ws = self._result()
        hip.check(ops.lib.sm_grad_clip(*self._args, kind, max_norm, ws.data_ptr(), self._ws_bytes, out.data_ptr(), hip.stream()), "sm_grad_clip")
        return out


def grad_norm(grads, norm_type=2.0) -> torch.Tensor:
    """The global norm of a list of gradients (``GradClip.norm`` for a list that changes from call to call; None entries are
    skipped; the same tensor listed twice counts twice)."""
    kind = _norm_kind(norm_type)
    t = _Table([g for g in grads if g is not None], "grads")
    ws = torch.empty(ops.lib.sm_grad_norm_ws_bytes(t.n), dtype=torch.uint8, device="cuda")
    out = torch.empty((), dtype=torch.float32, device="cuda")
    hip.check(ops.lib.sm_grad_norm(_address(t.ptrs), _address(t.numel), _address(t.types), t.n, kind, ws.data_ptr(), ws.numel(),
                                   out.data_ptr(), hip.stream()), "sm_grad_norm")
    return out


def clip_grad_norm(grads, max_norm, norm_type=2.0, out=None) -> torch.Tensor:
    """``GradClip(grads, out).clip(max_norm, norm_type)`` for a list that changes from call to call: scales the gradients in
    place (or into ``out``) and returns the norm before clipping."""
    _norm_kind(norm_type), _max_norm(max_norm)
    return GradClip(grads, out).clip(max_norm, norm_type)
