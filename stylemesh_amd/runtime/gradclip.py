"""The global norm over many gradient tensors and clipping by it (``sm_grad_norm`` / ``sm_grad_clip``; csrc/gradnorm.hip):
``Trainer(gradient_clip_val=...)`` of the reference's pytorch_lightning (requirements.txt:76), i.e.
``torch.nn.utils.clip_grad_norm_``, as two launches per 200 tensors with no host synchronisation.

    norm = sqrt(sum of all squares) or max |g|;   out = g * min(1, max_norm / (norm + 1e-6))

float32 / bfloat16 / float16 tensors may be mixed. Sums are held in 64 bits; the norm has the same bits every time. A norm
that is not finite is not an error (finding out would synchronise): the coefficient follows the formula, infinity clips to 0
(and infinity * 0 = NaN), a NaN makes every gradient NaN.
"""
from __future__ import annotations

import math

import torch

from . import hip, ops

try:
    from .. import _tensor_list
except ImportError as e:
    raise ImportError("stylemesh_amd/_tensor_list.so is missing or does not fit this torch: build it with "
                      "`python -c 'import __graft_entry__ as g; g.build()'` or stylemesh_amd/csrc/build.sh") from e


def _dense(t) -> bool:
    """One element per address of a range: a permutation of a contiguous tensor."""
    want = 1
    for st, sz in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if st != want:
            return False
        want *= sz
    return True


class _Table:
    """Pointers, element counts and types of a list of tensors as the library reads them (csrc/tensor_list.cpp: one walk in
    native code). Keeps the tensors: the table holds only their addresses, and what a caller made on the way in (an iterator of
    converted gradients) has no other owner until the launch."""

    def __init__(self, tensors, what):
        self.tensors = tensors
        self.packed, at, odd, device, self.contiguous = _tensor_list.pack(tensors)
        if odd >= 0:
            t = tensors[odd]
            raise ValueError(f"{what}: entry {odd} is {t.dtype}, {t.layout} (strided float32, bfloat16 or float16)")
        self.n = n = len(tensors)
        if n:
            if device == -1:
                raise ValueError(f"{what}: device tensors only (there is no CPU form)")
            if device != torch.cuda.current_device():
                raise ValueError(f"{what}: tensors on {sorted(set(str(t.device) for t in tensors))}, the current device is "
                                 f"cuda:{torch.cuda.current_device()}")
        self.ptrs, self.numel, self.types = (at, at + 8 * n, at + 16 * n) if n else (None, None, None)
        if not self.contiguous:
            for t in tensors:
                if not t.is_contiguous() and not _dense(t):
                    raise ValueError(f"{what}: strides {t.stride()} of {tuple(t.shape)} leave gaps or overlap")

    def holds(self) -> bool:
        return _tensor_list.pack(self.tensors)[0] == self.packed


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


# What is written must be written once: an output that overlaps another output, or a gradient other than its own (the same
# tensor listed twice, for one), has no defined result.
_WRONG = (None, "an output has not as many elements as its gradient", "an output that is its gradient must have its type",
          "two of the tensors to be written overlap (a gradient listed twice?)", "an output overlaps a gradient that is not its own")


class GradClip:
    """The call's tables for gradients that stay where they are (an arena's views, ``zero_grad(set_to_none=False)``): checked
    and laid out once, used every step. Keeps the tensors alive, and refuses them where their memory was exchanged since (``module.to``, ``t.data = ...``); ``grads``
    may hold None (a parameter without a gradient).
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
            if not (g.contiguous and o.contiguous):
                for a, b in zip(grads, out):
                    if not (a.is_contiguous() and b.is_contiguous()) and (a.shape != b.shape or a.stride() != b.stride()):
                        raise ValueError(f"out {tuple(b.shape)} / {b.stride()} does not match its gradient {tuple(a.shape)} / {a.stride()}")
        wrong = _tensor_list.check_outputs(g.packed, o.packed)
        if wrong:
            raise ValueError(_WRONG[wrong])
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._args = (g.ptrs, o.ptrs, g.numel, g.types, o.types, g.n)
        self._ws_bytes = ops.lib.sm_grad_norm_ws_bytes(g.n)

    def __reduce__(self):      # (a copy's tables are those of ITS tensors)
        return GradClip, (self.grads, None if self.out is self.grads else self.out)

    def _result(self):
        """(norm, scratch) of one call: two streams, or two captured graphs, of one plan share nothing"""
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the plan's tensors live on {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        return (torch.empty((), dtype=torch.float32, device=self.device),
                torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device))

    def _check(self):
        """Refuses tensors whose memory was exchanged or given up since the plan was made (``module.to``, ``t.data = ...``,
        ``storage.resize_``): the tables hold addresses."""
        for table, what in ((self._g, "gradient"),) if self._o is self._g else ((self._g, "gradient"), (self._o, "output")):
            if not table.holds():
                raise ValueError(f"a {what}'s memory was exchanged since the plan was made: make a new GradClip")

    def norm(self, norm_type=2.0) -> torch.Tensor:
        """The global norm as a float32 device scalar."""
        kind = _norm_kind(norm_type)
        self._check()
        out, ws = self._result()
        gp, _, numel, types, _, n = self._args
        hip.check(ops.lib.sm_grad_norm(gp, numel, types, n, kind, ws.data_ptr(), self._ws_bytes, out.data_ptr(), ops.eager_stream()), "sm_grad_norm")
        return out

    def clip(self, max_norm, norm_type=2.0) -> torch.Tensor:
        """Clips, and returns the norm BEFORE clipping (float32 device scalar)."""
        kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
        self._check()
        return self._clip(kind, max_norm)

    def _clip(self, kind, max_norm):
        out, ws = self._result()
        hip.check(ops.lib.sm_grad_clip(*self._args, kind, max_norm, ws.data_ptr(), self._ws_bytes, out.data_ptr(), ops.eager_stream()), "sm_grad_clip")
        _tensor_list.written(self.out)      # (autograd refuses a graph that saved one of them before)
        return out


def grad_norm(grads, norm_type=2.0) -> torch.Tensor:
    """The global norm of a list of gradients (``GradClip.norm`` for a list that changes from call to call; None entries are
    skipped; the same tensor listed twice counts twice)."""
    kind = _norm_kind(norm_type)
    t = _Table([g for g in grads if g is not None], "grads")
    ws = torch.empty(ops.lib.sm_grad_norm_ws_bytes(t.n), dtype=torch.uint8, device="cuda")
    out = torch.empty((), dtype=torch.float32, device="cuda")
    hip.check(ops.lib.sm_grad_norm(t.ptrs, t.numel, t.types, t.n, kind, ws.data_ptr(), ws.numel(),
                                   out.data_ptr(), ops.eager_stream()), "sm_grad_norm")
    return out


def clip_grad_norm(grads, max_norm, norm_type=2.0, out=None) -> torch.Tensor:
    """``GradClip(grads, out).clip(max_norm, norm_type)`` for a list that changes from call to call: scales the gradients in
    place (or into ``out``) and returns the norm before clipping."""
    kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
    return GradClip(grads, out)._clip(kind, max_norm)
