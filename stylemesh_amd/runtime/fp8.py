"""Matrices in 8-bit floating point with one scale per block of 128, their products and a layer's forward / backward pass
over them (``sm_fp8_*``; csrc/fp8.hip). The rung below the library's fp16x2 arithmetic for products that tolerate 8 bits:
feature maps against filters, activations against a resident weight, and the gradient products of a training step.

Every call is asynchronous on torch's current stream, allocates its results (and, for a product that splits its depth, its
scratch) from torch's allocator and synchronises nothing. There is no autograd node: ``linear_fp8_fwd`` /
``linear_fp8_bwd`` are the two halves of a step, as the sampler's and the losses' are (``ops.tex_sample_fwd`` / ``_bwd``), for a
``torch.autograd.Function`` or a loop of one's own. Where autograd records, a tensor that requires a gradient is refused by them (and
as ``out`` / ``dw``): the result would silently have none. A quantised copy never has one, whatever it is made from.
"""
from __future__ import annotations

import torch

from . import ops

try:
    from .. import _fp8_host
except ImportError as e:
    raise ImportError("stylemesh_amd/_fp8_host.so is missing or does not fit this torch: build it with "
                      "`python -c 'import __graft_entry__ as g; g.build()'` or stylemesh_amd/csrc/build.sh") from e

BLOCK = 128
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FMT_ID = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}                      # SM_FP8_*
_TYPE_ID = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}           # SM_TYPE_*
_MAX_DIM = 65535 * 128       # rows / columns of a matrix (the quantiser's grid)
_NO_MATRIX = (None, None, 0, 0)      # codes, scales, tiles?, pitch


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _check_device(*devices):
    """Launches go to the CURRENT device's current stream: tensors of another device (or of the host) are refused."""
    cur = None
    for d in devices:
        if d is None:
            continue
        if d < 0:
            raise ValueError("device tensors only (there is no CPU form)")
        if cur is None:
            cur = torch.cuda.current_device()
        if d != cur:
            raise ValueError(f"a tensor lives on cuda:{d}, the current device is cuda:{cur}")


class Fp8Matrix:
    """[rows, cols] as 8-bit codes and block scales: value = code * scale of its block.

    ``data``: float8_e4m3fn / float8_e5m2 [rows, cols rounded up to 128], contiguous; the codes behind column ``cols`` must be
    ZERO (the product runs over whole blocks; ``from_parts`` pads). ``block``: "rows" - a scale per row and 128 columns - or
    "tiles" - per 128 x 128 tile. ``scale``: uint8 power-of-two scales [ceil(KB / 4), S, 4], byte s = 2^(s - 127), the byte of
    (row, block kb) at [kb / 4, row, kb % 4], KB = ceil(cols / 128), S = rows or ceil(rows / 128) - or float32 scales [KB, S].
    The tensors are used as they are, no copy is taken - but for codes laid out column by column (quantising ``x.t()`` in plain
    torch leaves them so), which are copied once, here."""

    __slots__ = ("_data", "_scale", "_rows", "_cols", "_tiles", "_fmt", "_f32", "_pitch", "_device")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int, block: str = "rows"):
        if block not in ("rows", "tiles"):
            raise ValueError(f"block={block!r}: 'rows' or 'tiles'")
        if data.dtype not in _FMT_ID:
            raise ValueError(f"codes of type {data.dtype}: float8_e4m3fn or float8_e5m2")
        if data.dim() != 2 or cols < 0 or data.shape[1] != _blocks(cols) * BLOCK or not (data.is_contiguous() or data.t().is_contiguous()):
            raise ValueError(f"codes must be dense [rows, {_blocks(max(cols, 0)) * BLOCK}] for {cols} columns, got "
                             f"{tuple(data.shape)}, strides {data.stride()}; from_parts takes any strides and widths")
        if not data.is_contiguous():
            data = data.contiguous()
        if data.data_ptr() % 16:
            raise ValueError("codes must start on a 16-byte boundary")
        kb, s = _blocks(cols), data.shape[0] if block == "rows" else _blocks(data.shape[0])
        want = {torch.uint8: (-(-kb // 4), s, 4), torch.float32: (kb, s)}.get(scale.dtype)
        if want is None or tuple(scale.shape) != want or not scale.is_contiguous():
            raise ValueError(f"scales must be contiguous uint8 {(-(-kb // 4), s, 4)} or float32 {(kb, s)}, got {scale.dtype} "
                             f"{tuple(scale.shape)}")
        if scale.data_ptr() % 4:
            raise ValueError("scales must start on a 4-byte boundary")
        if scale.device != data.device:
            raise ValueError(f"codes on {data.device}, scales on {scale.device}")
        self._set(data, scale, data.shape[0], int(cols), int(block == "tiles"), _FMT_ID[data.dtype], int(scale.dtype == torch.float32),
                  data.get_device())

    def _set(self, data, scale, rows, cols, tiles, fmt, f32, device):
        # what every call hands on, of the tensors this object keeps (and never exchanges: the properties are read-only);
        # device -1: host
        self._data, self._scale, self._rows, self._cols, self._tiles, self._fmt, self._f32 = data, scale, rows, cols, tiles, fmt, f32
        self._pitch, self._device = -(-cols // BLOCK) * BLOCK, device

    def __reduce__(self):      # (torch pickles bytes, but no 8-bit floats)
        return _rebuild, (self._data.view(torch.uint8), self._data.dtype, self._scale, self._cols, self.block)

    data = property(lambda self: self._data)
    scale = property(lambda self: self._scale)
    _ptrs = property(lambda self: (self._data.data_ptr(), self._scale.data_ptr()))
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    block = property(lambda self: "tiles" if self._tiles else "rows")

    @property
    def shape(self):
        return (self._rows, self._cols)

    @property
    def device(self):
        return self.data.device

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scale: torch.Tensor, block: str = "rows") -> "Fp8Matrix":
        """From codes [rows, cols] of any strides and scales [S, KB] as checkpoints hold them - int32 / uint8 exponent
        bytes (2^(s - 127)) or float32 - in this class's layout (copies: once per weight, not per call)."""
        if codes.dim() != 2:
            raise ValueError(f"codes must be a matrix, got {tuple(codes.shape)}")
        rows, cols = codes.shape
        kb, s = _blocks(cols), rows if block == "rows" else _blocks(rows)
        if tuple(scale.shape) != (s, kb):
            raise ValueError(f"scales must be {(s, kb)} for {block} of {(rows, cols)}, got {tuple(scale.shape)}")
        data = torch.zeros(rows, kb * BLOCK, dtype=torch.uint8, device=codes.device)
        data[:, :cols] = codes.contiguous().view(torch.uint8)
        if scale.dtype == torch.float32:
            packed = scale.t().contiguous()
        elif scale.dtype in (torch.uint8, torch.int32):
            if scale.dtype == torch.int32 and scale.numel() and not 0 <= int(scale.min()) <= int(scale.max()) <= 255:
                raise ValueError("exponent bytes lie in 0 ... 255")
            packed = pack_scale_bytes(scale)
        else:
            raise ValueError(f"scales of type {scale.dtype}: float32, or exponent bytes as uint8 / int32")
        return cls(data.view(codes.dtype), packed, cols, block)

    def scales(self) -> torch.Tensor:
        """The scales as float32 [S, KB]."""
        if self.scale.dtype == torch.float32:
            return self.scale.t()
        e = self.scale.permute(1, 0, 2).reshape(self.scale.shape[1], -1)[:, :_blocks(self.cols)].int()
        # 2^(e - 127) from the bits; byte 0 is 2^-127 (a subnormal fp32), 255 is NaN
        bits = torch.where(e == 255, 0x7fc00000, torch.where(e == 0, 0x00400000, e << 23))
        return bits.view(torch.float32)

    def dequantize(self) -> torch.Tensor:
        """float32 [rows, cols] (torch operations: for reports and tests)."""
        s = self.scales().repeat_interleave(BLOCK, dim=1)
        if self.block == "tiles":
            s = s.repeat_interleave(BLOCK, dim=0)[:self.rows]
        return (self.data.float() * s)[:, :self.cols]

    def transposed(self) -> "Fp8Matrix":
        """The transpose of a ``tiles`` matrix - its tiles are the transpose's tiles, the codes are the same (a copy: once per
        weight update; ``fp8_quantize_both(w, block="tiles")`` makes both from the weight in one pass). Row scales have no
        such transpose: ``ValueError``."""
        if self.block != "tiles":
            raise ValueError("only a matrix with tile scales can be transposed as it is (row blocks become column blocks)")
        rows, cols = self.shape
        data = torch.zeros(cols, _blocks(rows) * BLOCK, dtype=torch.uint8, device=self.device)
        data[:, :rows] = self.data.view(torch.uint8)[:, :cols].t()
        if self.scale.dtype == torch.float32:
            scale = self.scale.t().contiguous()
        else:
            e = self.scale.permute(1, 0, 2).reshape(self.scale.shape[1], -1)[:, :_blocks(cols)]
            scale = pack_scale_bytes(e.t())
        return Fp8Matrix(data.view(self.data.dtype), scale, rows, "tiles")


def _rebuild(codes, dtype, scale, cols, block):
    return Fp8Matrix(codes.view(dtype), scale, cols, block)


def pack_scale_bytes(e: torch.Tensor) -> torch.Tensor:
    """Exponent bytes [S, KB] -> the stored form [ceil(KB / 4), S, 4] (uint8, padded with 127 = 1.0)."""
    e = torch.nn.functional.pad(e.to(torch.uint8), (0, -e.shape[1] % 4), value=127)
    return e.view(e.shape[0], -1, 4).permute(1, 0, 2).contiguous()


def _check_matrix(x, what):
    """x: a matrix the kernels read or write"""
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPE_ID or x.dim() != 2 or x.layout != torch.strided or x.is_neg():
        raise ValueError(f"{what} must be a strided float32 / bfloat16 / float16 matrix, got "
                         f"{(x.dtype, tuple(x.shape), x.layout) if isinstance(x, torch.Tensor) else type(x)}")
    (rows, cols), (sr, sc) = x.shape, x.stride()
    # (the stride of a dimension of one element means nothing)
    if (cols > 1 and sc != 1) or (rows > 1 and sr < cols):
        raise ValueError(f"{what} must have unit column stride and rows that do not overlap, got strides {x.stride()} for "
                         f"{tuple(x.shape)}; pass .contiguous(), or transpose=True for a transposed matrix")
    if rows > _MAX_DIM or cols > _MAX_DIM:
        raise ValueError(f"{what}: {tuple(x.shape)} has a dimension above {_MAX_DIM}")
    _check_device(x.get_device())


def _check_no_graph(x, what):
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient and there is no autograd node: call under torch.no_grad(), in an autograd.Function, "
                         "or with .detach()")


def _refuse(x, what, in_graph=True):
    """The native call would not take its arguments: says why."""
    _check_matrix(x, what)
    if in_graph:
        _check_no_graph(x, what)
    raise ValueError(f"{what} cannot be used: {x.dtype} {tuple(x.shape)}, strides {x.stride()} on {x.device}")


def _check_held(*matrices):
    """The native call would not take its matrices: their tensors no longer hold what they were made of."""
    for m in matrices:
        if m is not None:
            try:
                Fp8Matrix(m._data, m._scale, m._cols, m.block)
            except (ValueError, RuntimeError) as e:
                raise ValueError(f"the tensors of an Fp8Matrix {m.shape} were exchanged since it was made: {e}") from None
            if m._data.shape[0] != m._rows or not m._data.is_contiguous() or any(t.untyped_storage().nbytes() < t.storage_offset() * t.itemsize + t.nbytes for t in (m._data, m._scale)):
                raise ValueError(f"the tensors of an Fp8Matrix {m.shape} were resized or laid out anew since it was made")


_new = Fp8Matrix.__new__


def _quantize(x, block, fmt, plain, transpose):
    if fmt not in FORMATS:
        raise ValueError(f"fmt={fmt!r}: 'e4m3' or 'e5m2'")
    if block not in ("rows", "tiles"):
        raise ValueError(f"block={block!r}: 'rows' or 'tiles'")
    fid, tiles = _FMT_ID[FORMATS[fmt]], int(block == "tiles")
    done = None
    if isinstance(x, torch.Tensor) and x.is_cuda:
        device = torch.cuda.current_device()
        done = _fp8_host.quantize(x, fid, tiles, plain, transpose, device, ops.eager_stream())
    if done is None:
        _refuse(x, "x", in_graph=False)
    rows, cols, n, t = done
    if plain:
        q, s = n
        n = _new(Fp8Matrix)
        n._set(q, s, rows, cols, tiles, fid, 0, device)
    if transpose:
        q, s = t
        t = _new(Fp8Matrix)
        t._set(q, s, cols, rows, tiles, fid, 0, device)
    return n, t


def fp8_quantize(x: torch.Tensor, block: str = "rows", fmt: str = "e4m3", transpose: bool = False) -> Fp8Matrix:
    """``x`` [rows, cols] (float32 / bfloat16 / float16, unit column stride, any row stride) - or, with ``transpose``, its
    transpose - as an ``Fp8Matrix`` with power-of-two scales: per block the smallest power of two that brings the largest
    finite magnitude into the format's range; x / scale is exact, the code is it rounded to nearest even. NaN stays NaN, an
    infinity becomes NaN (e4m3 has none) or infinity (e5m2); neither touches its neighbours' scale. (A magnitude from
    1.9375 * 2^127 on rounds up to 2^128, which fp32 does not hold: ``dequantize`` shows infinity.)"""
    n, t = _quantize(x, block, fmt, not transpose, bool(transpose))
    return t if transpose else n


def fp8_quantize_both(x: torch.Tensor, block: str = "rows", fmt: str = "e4m3"):
    """(``fp8_quantize(x)``, ``fp8_quantize(x, transpose=True)``) from one read of ``x``: what a training step needs of its
    activations and output gradients (rows) and of its weights (tiles)."""
    return _quantize(x, block, fmt, True, True)


def _check_fast(fast_accum, dtype):
    if fast_accum and dtype != torch.bfloat16:
        raise ValueError(f"fast_accum is for bfloat16 results, this one is {dtype}")
    return bool(fast_accum)


def matmul_fp8(a: Fp8Matrix, b: Fp8Matrix, out: torch.Tensor | None = None, out_dtype=None, accumulate: bool = False,
               fast_accum: bool = False) -> torch.Tensor:
    """[M, N] = A B^T for A [M, K] (``rows`` scales, e4m3 or e5m2) and B [N, K] (e4m3, ``rows`` or ``tiles`` scales), both with
    power-of-two or both with float32 scales; the codes are widened, the sums held in fp32 and rounded once to ``out_dtype``
    (float32 / bfloat16 / float16; default bfloat16). ``out``: result of that type and shape, unit column stride; ``accumulate``:
    added to it (in fp32, then rounded once). ``fast_accum`` (bfloat16 results only) permits the 8-bit matrix instruction, up to twice as
    fast on large products - its sum of eight products keeps 13 bits below the largest of them, so a result may be off by
    7 * 2^-13 of sum |a||b|, however small the result itself is (rows with outliers that cancel lose most)."""
    if not isinstance(a, Fp8Matrix) or not isinstance(b, Fp8Matrix):
        raise ValueError("matmul_fp8 takes two Fp8Matrix operands")
    if a._tiles:
        raise ValueError("the first operand needs row scales")
    if b._fmt != 0:
        raise ValueError("the second operand must be e4m3")
    M, N, K = a._rows, b._rows, a._cols
    if K != b._cols:
        raise ValueError(f"inner dimensions differ: {a.shape} x {b.shape}^T")
    if a._f32 != b._f32:
        raise ValueError(f"one operand has {a.scale.dtype} scales, the other {b.scale.dtype}")
    if max(M, N, K) > _MAX_DIM:
        raise ValueError(f"a dimension above {_MAX_DIM}")
    _check_device(a._device, b._device)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if out_dtype is None:
            out_dtype = torch.bfloat16
        if out_dtype not in _TYPE_ID:
            raise ValueError(f"out_dtype={out_dtype}: float32, bfloat16 or float16")
        dtype = _TYPE_ID[out_dtype]
        fast = _check_fast(fast_accum, out_dtype)
    else:
        _check_matrix(out, "out")
        _check_no_graph(out, "out")
        if tuple(out.shape) != (M, N) or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, the product {out_dtype or out.dtype} {(M, N)}")
        dtype = 0
        fast = _check_fast(fast_accum, out.dtype)
    done = _fp8_host.matmul(a._data, a._scale, a._fmt, a._pitch, b._data, b._scale, b._tiles, b._pitch, a._f32, M, N, K, out, dtype,
                            bool(accumulate), fast, a._device, ops.eager_stream())
    if done is None:
        _check_held(a, b)
        _refuse(out, "out")
    return done


def _weight_arg(w, what="weight"):
    if not isinstance(w, Fp8Matrix) or w._fmt != 0 or w._f32:
        raise ValueError(f"{what} must be an e4m3 Fp8Matrix with power-of-two scales")
    return w


def linear_fp8_fwd(x: torch.Tensor, weight: Fp8Matrix, out_dtype=None, keep_transposed: bool = False, fast_accum: bool = False):
    """y [M, N] = q(x) weight^T for x [M, K] and a resident weight [N, K] (``fp8_quantize(w, block="tiles")``), in ``out_dtype``
    (default: x's). ``keep_transposed``: returns (y, q(x^T)), the second for ``linear_fp8_bwd``'s weight gradient - quantised
    from the same read of x. ``fast_accum``: as ``matmul_fp8``'s."""
    _weight_arg(weight)
    if out_dtype is not None and out_dtype not in _TYPE_ID:
        raise ValueError(f"out_dtype={out_dtype}: float32, bfloat16 or float16")
    if keep_transposed:
        if isinstance(x, torch.Tensor):
            _check_no_graph(x, "x")
        n, t = _quantize(x, "rows", "e4m3", True, True)
        return matmul_fp8(n, weight, out_dtype=x.dtype if out_dtype is None else out_dtype, fast_accum=fast_accum), t
    if fast_accum:
        _check_matrix(x, "x")
        _check_fast(fast_accum, x.dtype if out_dtype is None else out_dtype)
    y = None
    if weight._device >= 0 and weight._device == torch.cuda.current_device():
        y = _fp8_host.linear(x, weight._data, weight._scale, weight._tiles, weight._pitch, weight._rows, weight._cols,
                             -1 if out_dtype is None else _TYPE_ID[out_dtype], bool(fast_accum), weight._device, ops.eager_stream())
    if y is None:
        _check_matrix(x, "x")
        _check_no_graph(x, "x")
        if x.shape[1] != weight._cols:
            raise ValueError(f"x has {x.shape[1]} columns, the weight {weight._cols}")
        _check_device(weight._device)
        _check_held(weight)
        _refuse(x, "x")
    return y


def linear_fp8_bwd(dy: torch.Tensor, x_t: Fp8Matrix | None, weight_t: Fp8Matrix | None, fmt: str = "e4m3", dx_dtype=None,
                   dw: torch.Tensor | None = None, accumulate: bool = False, fast_accum: bool = False):
    """(dx, dw) of ``linear_fp8_fwd``'s layer: dx [M, K] = q(dy) weight (in ``dx_dtype``, default dy's) from
    ``weight_t`` = the weight's transpose [K, N] (``weight.transposed()`` / ``fp8_quantize_both(w, block="tiles")[1]``), and
    dw [N, K] = q(dy^T) q(x^T)^T in float32 from ``x_t`` = [K, M] (``keep_transposed``). ``fmt``: format of the gradient's
    codes. ``dw`` / ``accumulate``: write into, or add to, an existing float32 gradient. Either of ``x_t`` / ``weight_t`` may be
    None: that gradient is not computed and None is returned in its place. ``fast_accum``: as ``matmul_fp8``'s, for dx; dw is
    always summed in fp32."""
    _check_matrix(dy, "dy")
    _check_no_graph(dy, "dy")
    M, N = dy.shape
    if x_t is None and weight_t is None:
        raise ValueError("nothing to compute: both x_t and weight_t are None")
    if fmt not in FORMATS:
        raise ValueError(f"fmt={fmt!r}: 'e4m3' or 'e5m2'")
    K = (weight_t if weight_t is not None else _weight_arg(x_t, "x_t")).rows
    dx = None
    if weight_t is not None:
        if _weight_arg(weight_t, "weight_t").cols != N:
            raise ValueError(f"dy has {N} columns, weight_t {weight_t.cols}")
        if dx_dtype is None:
            dx_dtype = dy.dtype
        elif dx_dtype not in _TYPE_ID:
            raise ValueError(f"dx_dtype={dx_dtype}: float32, bfloat16 or float16")
        _check_fast(fast_accum, dx_dtype)
    if x_t is not None:
        if _weight_arg(x_t, "x_t").cols != M or x_t.rows != K:
            raise ValueError(f"dy has {M} rows and the layer {K} inputs, x_t is {x_t.shape}")
        if dw is not None and (dw.dtype != torch.float32 or tuple(dw.shape) != (N, K)):
            raise ValueError(f"dw must be float32 {(N, K)}, got {dw.dtype} {tuple(dw.shape)}")
        if accumulate and dw is None:
            raise ValueError("accumulate needs dw")
    elif dw is not None:
        raise ValueError("dw given, but no x_t to compute it from")
    if K > _MAX_DIM:
        raise ValueError(f"a dimension above {_MAX_DIM}")
    if dw is not None:
        _check_matrix(dw, "dw")
        _check_no_graph(dw, "dw")
    _check_device(None if weight_t is None else weight_t._device, None if x_t is None else x_t._device)
    if not (M and N and K):      # a gradient without elements, or a sum without terms
        if weight_t is not None:
            dx = torch.zeros((M, K), dtype=dx_dtype, device=dy.device)
        if x_t is not None:
            if dw is None:
                dw = torch.zeros((N, K), dtype=torch.float32, device=dy.device)
            elif not accumulate:
                dw.zero_()
        return dx, dw
    wt = (weight_t._data, weight_t._scale, weight_t._tiles, weight_t._pitch) if weight_t is not None else _NO_MATRIX
    xt = (x_t._data, x_t._scale, x_t._tiles, x_t._pitch) if x_t is not None else _NO_MATRIX
    done = _fp8_host.backward(dy, _FMT_ID[FORMATS[fmt]], K, *wt, *xt, -1 if dx_dtype is None else _TYPE_ID[dx_dtype], dw, bool(accumulate),
                              bool(fast_accum and weight_t is not None), dy.get_device(), ops.eager_stream())
    if done is None:
        _check_held(weight_t, x_t)
        _refuse(dy, "dy")
    return done
