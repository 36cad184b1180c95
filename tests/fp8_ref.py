"""The 8-bit block format in 64 bits on the CPU: what ``stylemesh_amd.runtime.fp8`` computes, from the definition."""
import torch

LIMIT = {"e4m3": 448.0, "e5m2": 57344.0}
GRID = {"e4m3": (3, -6), "e5m2": (2, -14)}      # mantissa bits, exponent of the smallest normal value


def round_to(y, fmt):
    """float64 -> the format's grid (ties to even), |y| within its range; NaN / inf as the format has them."""
    bits, low = GRID[fmt]
    mant, ex = torch.frexp(y)
    q = (ex - 1).clamp_min(low).double()
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), q - bits)
    r = torch.round(y / step) * step
    bad = ~torch.isfinite(y)
    odd = torch.full_like(y, float("nan")) if fmt == "e4m3" else y
    return torch.where(bad, odd, torch.where(y == 0, y, r))


def exponent(amax, fmt):
    """smallest e in [-127, 127] with amax <= LIMIT 2^e; 0 for amax = 0"""
    if amax == 0:
        return 0
    e = -127
    while LIMIT[fmt] * 2.0 ** e < amax and e < 127:
        e += 1
    return e


def quantize(x, block, fmt):
    """(values of the codes [R, C padded to 128], exponents [S][KB]) of a matrix, float64 / int64"""
    x = x.detach().cpu().double()
    R, C = x.shape
    kb, s = -(-C // 128), R if block == "rows" else -(-R // 128)
    vals = torch.zeros(R, kb * 128, dtype=torch.float64)
    exps = torch.zeros(s, kb, dtype=torch.int64)
    step = 1 if block == "rows" else 128
    for i in range(s):
        for j in range(kb):
            part = x[i * step:(i + 1) * step, j * 128:(j + 1) * 128]
            a = part.abs()
            a = a[torch.isfinite(a)]
            e = exponent(float(a.max()) if a.numel() else 0.0, fmt)
            exps[i, j] = e
            vals[i * step:(i + 1) * step, j * 128:j * 128 + part.shape[1]] = round_to(part * 2.0 ** -e, fmt)
    return vals, exps


def values(vals, exps, block, cols):
    f = torch.pow(torch.tensor(2.0, dtype=torch.float64), exps.double()).repeat_interleave(128, dim=1)
    if block == "tiles":
        f = f.repeat_interleave(128, dim=0)[:vals.shape[0]]
    return (vals * f)[:, :cols]


def requantized(x, block="rows", fmt="e4m3"):
    """the values x stands for after quantisation, float64"""
    return values(*quantize(x, block, fmt), block, x.shape[1])


def matmul_bound(a, b, out_dtype, ref):
    """|error| of a fp32-accumulated sum of K products in any order, rounding or truncating: every one of the K additions is
    off by at most 2^-23 of the largest partial sum, which sum |a| |b| bounds; plus half a step of the result's type (its
    smallest subnormal where the result is that small)."""
    K = a.shape[1]
    mag = a.abs() @ b.abs().t()
    acc = (K + 8) * 2.0 ** -23 * mag
    half = torch.finfo(out_dtype).eps / 2
    return acc + half * (ref.abs() + acc) + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
