"""The global norm over many gradient tensors and clipping by it (``sm_grad_norm`` / ``sm_grad_clip``; csrc/gradnorm.hip):
``Trainer(gradient_clip_val=...)`` of the reference's pytorch_lightning (requirements.txt:76), i.e.
``torch.nn.utils.clip_grad_norm_``, as two launches per 120 tensors with no host synchronisation.

    norm = sqrt(sum of all squares) or max |g|;   out = g * min(1, max_norm / (norm + 1e-6))

float32 / bfloat16 / float16 tensors may be mixed. Sums are held in 64 bits; the norm has the same bits every time. A norm
that is not finite is not an error (finding out would synchronise): the coefficient follows the formula, infinity clips to 0
(and infinity * 0 = NaN), a NaN makes every gradient NaN.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import hip, ops

_TYPE_ID = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}           # SM_TYPE_*


def _dense(t) -> bool:
    """One element per address of a range: contiguous, or a permutation of a contiguous tensor."""
    if t.is_contiguous():
        return True
    want = 1
    for st, sz in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if st != want:
            return False
        want *= sz
    return True


def _check(tensors, what):
    for t in tensors:
        if t.dtype not in _TYPE_ID:
            raise ValueError(f"{what}: {t.dtype} tensor (float32, bfloat16 or float16)")
        if not t.is_cuda:
            raise ValueError(f"{what}: device tensors only (there is no CPU form)")
        if t.device.index != torch.cuda.current_device():
            raise ValueError(f"{what}: a tensor lives on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
        if not _dense(t):
            raise ValueError(f"{what}: strides {t.stride()} of {tuple(t.shape)} leave gaps or overlap")


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


class GradClip:
    """The call's tables for gradients that stay where they are (an arena's views, ``zero_grad(set_to_none=False)``): checked
    and laid out once, used every step. Keeps the tensors alive; ``grads`` may hold None (a parameter without a gradient).
    ``out``: one tensor per gradient (same shape and element order) that receives the clipped values, of any of the three
    types; None: the gradients themselves are scaled in place (where nothing is clipped the second pass ends at once).
    Concurrent use of ONE plan on two streams is not allowed (its scratch is its own); two plans over the same gradients are
    independent."""

    def __init__(self, grads, out=None):
        grads = list(grads)
        if out is not None:
            out = list(out)
            if len(out) != len(grads):
                raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")
        pairs = [(g, g if out is None else out[i]) for i, g in enumerate(grads) if g is not None]
        self.grads, self.out = [g for g, _ in pairs], [o for _, o in pairs]
        _check(self.grads, "grads")
        self.device = torch.device("cuda", torch.cuda.current_device())
        if out is not None:
            if any(o is None for o in self.out):
                raise ValueError("an output is missing for a gradient that is there")
            _check(self.out, "out")
            for g, o in pairs:
                if o.shape != g.shape or (o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous())):
                    raise ValueError(f"out {tuple(o.shape)} / {o.stride()} does not match its gradient {tuple(g.shape)} / {g.stride()}")
                if o.data_ptr() == g.data_ptr() and o.dtype != g.dtype and g.numel():
                    raise ValueError("an output that is its gradient must have its type")
        self._refuse_overlap(pairs)
        n = len(pairs)
        self._n = n
        self._in = (C.c_void_p * n)(*[g.data_ptr() for g in self.grads])
        self._outp = (C.c_void_p * n)(*[o.data_ptr() for o in self.out])
        self._numel = (C.c_size_t * n)(*[g.numel() for g in self.grads])
        self._types = (C.c_int * n)(*[_TYPE_ID[g.dtype] for g in self.grads])
        self._out_types = (C.c_int * n)(*[_TYPE_ID[o.dtype] for o in self.out])
        self._ws = torch.empty(ops.lib.sm_grad_norm_ws_bytes(n), dtype=torch.uint8, device=self.device)

    @staticmethod
    def _refuse_overlap(pairs):
        """What is written must be written once: an output that overlaps another output, or a gradient other than its own
        (the same tensor listed twice, for one), has no defined result."""
        span = lambda t: (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
        outs = sorted(span(o) + (i,) for i, (_, o) in enumerate(pairs) if o.numel())
        for (_, e0, _), (s1, _, _) in zip(outs, outs[1:]):
            if s1 < e0:
                raise ValueError("two of the tensors to be written overlap (a gradient listed twice?)")
        ins = sorted(span(g) + (i,) for i, (g, _) in enumerate(pairs) if g.numel())
        k = 0
        for s, e, i in outs:
            while k < len(ins) and ins[k][1] <= s and ins[k][0] < s:
                k += 1
            j = k
            while j < len(ins) and ins[j][0] < e:
                if ins[j][1] > s and (ins[j][2] != i or ins[j][0] != s):
                    raise ValueError("an output overlaps a gradient that is not its own")
                j += 1

    def _current(self):
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the plan's tensors live on {self.device}, the current device is cuda:{torch.cuda.current_device()}")

    def norm(self, norm_type=2.0) -> torch.Tensor:
        """The global norm as a float32 device scalar."""
        kind = _norm_kind(norm_type)
        self._current()
        out = torch.empty((), dtype=torch.float32, device=self.device)
        hip.check(ops.lib.sm_grad_norm(self._in, self._numel, self._types, self._n, kind, self._ws.data_ptr(), self._ws.numel(),
                                       out.data_ptr(), hip.stream()), "sm_grad_norm")
        return out

    def clip(self, max_norm, norm_type=2.0) -> torch.Tensor:
        """Clips, and returns the norm BEFORE clipping (float32 device scalar)."""
        kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
        self._current()
        out = torch.empty((), dtype=torch.float32, device=self.device)
        hip.check(ops.lib.sm_grad_clip(self._in, self._outp, self._numel, self._types, self._out_types, self._n, kind, max_norm,
                                       self._ws.data_ptr(), self._ws.numel(), out.data_ptr(), hip.stream()), "sm_grad_clip")
        return out


def grad_norm(grads, norm_type=2.0) -> torch.Tensor:
    """The global norm of a list of gradients (``GradClip.norm`` for a list that changes from call to call; None entries are
    skipped; the same tensor listed twice counts twice)."""
    kind = _norm_kind(norm_type)
    grads = [g for g in grads if g is not None]
    _check(grads, "grads")
    n = len(grads)
    ws = torch.empty(ops.lib.sm_grad_norm_ws_bytes(n), dtype=torch.uint8, device="cuda")
    out = torch.empty((), dtype=torch.float32, device="cuda")
    hip.check(ops.lib.sm_grad_norm((C.c_void_p * n)(*[g.data_ptr() for g in grads]), (C.c_size_t * n)(*[g.numel() for g in grads]),
                                   (C.c_int * n)(*[_TYPE_ID[g.dtype] for g in grads]), n, kind, ws.data_ptr(), ws.numel(),
                                   out.data_ptr(), hip.stream()), "sm_grad_norm")
    return out


def clip_grad_norm(grads, max_norm, norm_type=2.0, out=None) -> torch.Tensor:
    """``GradClip(grads, out).clip(max_norm, norm_type)`` for a list that changes from call to call: scales the gradients in
    place (or into ``out``) and returns the norm before clipping."""
    _norm_kind(norm_type), _max_norm(max_norm)
    return GradClip(grads, out).clip(max_norm, norm_type)
