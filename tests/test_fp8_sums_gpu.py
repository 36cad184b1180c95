"""How many bits the sums of the 8-bit products keep, and over which scales (runtime/fp8.py), against 64 bits."""
import pytest
import torch

import fp8_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _fp8():
    require_gpu()
    from stylemesh_amd.runtime import fp8
    return fp8


def _matrix(fp8, values, dtype=E4, block="rows", scale="e8m0"):
    """values (which the format holds) with scales of 1"""
    r, c = values.shape
    kb, s = -(-c // 128), r if block == "rows" else -(-r // 128)
    data = torch.zeros(r, kb * 128, device="cuda")
    data[:, :c] = values
    codes = data.to(dtype)
    assert torch.equal(codes.float(), data)
    sc = torch.full((-(-kb // 4), s, 4), 127, dtype=torch.uint8, device="cuda") if scale == "e8m0" else torch.ones(kb, s, device="cuda")
    return fp8.Fp8Matrix(codes, sc, c, block)


def _outliers(M, N, K, fmt, seed):
    """Integers: every eighth column an outlier v that cancels in pairs, small odd and even numbers between. K / 16 v^2 + 9 K <
    2^24: every partial sum, in any order, is a whole number that fp32 holds, so a sum of fp32 is exact. An outlier's product
    is at least 2^11 (v >= 48), 13 bits below which the ones of the small products lie or end."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    fits = [v for v in (48, 64, 96, 128, 160, 176, 192, 224, 256, 320, 384, 448) if (K // 16 + 1) * v * v + 9 * K < 1 << 24]
    v = max(v for v in fits if fmt == E4 or v in (48, 64, 96, 128, 160, 192, 224, 256, 320, 384, 448))      # (e5m2: three bits)
    a = torch.randint(-3, 4, (M, K), generator=g, device="cuda").float()
    b = torch.randint(-3, 4, (N, K), generator=g, device="cuda").float()
    at = torch.arange(0, K // 16 * 16, 8, device="cuda")
    a[:, at] = v * (1.0 - 2.0 * (torch.arange(at.numel(), device="cuda") % 2))
    b[:, at] = float(v)
    return a, b


# one shape or more per form: stream (up to 16 rows, 32, long B, split), 64 x 64 (ring of four, of three, split), 128 x 128, 256-row tiles
FORMS = [(1, 200, 1024), (16, 130, 900), (20, 70, 1024), (32, 6200, 1000), (4, 100, 8192), (100, 200, 1024), (33, 70, 2304), (40, 100, 4100),
         (1500, 1540, 1024), (1800, 1930, 1000), (4000, 4000, 1024)]


@pytest.mark.parametrize("M,N,K", FORMS)
@pytest.mark.parametrize("scale,block", [("e8m0", "rows"), ("e8m0", "tiles"), ("f32", "rows"), ("f32", "tiles")])
def test_sums_keep_what_fp32_keeps(M, N, K, scale, block):
    """Outlier channels that cancel: the result is the small terms' sum, to the last bit, in every form and for every type."""
    fp8 = _fp8()
    for fmt in (E4, E5):
        a, b = _outliers(M, N, K, fmt, 5)
        ref = a.double() @ b.double().t()
        qa, qb = _matrix(fp8, a, fmt, "rows", scale), _matrix(fp8, b, E4, block, scale)
        for dt in DT.values():
            assert torch.equal(fp8.matmul_fp8(qa, qb, out_dtype=dt), ref.to(dt)), dt


@pytest.mark.parametrize("M,N,K", [(1, 200, 1024), (7, 300, 2000), (16, 70, 8192), (60, 90, 1500), (300, 200, 1024)])
def test_layer_passes_keep_what_fp32_keeps(M, N, K):
    """The layer's forward pass and its input gradient in bfloat16, on values that the quantiser leaves as they are."""
    fp8 = _fp8()
    a, b = _outliers(M, N, K, E4, 6)
    ref = (a.double() @ b.double().t()).bfloat16()
    w8 = fp8.fp8_quantize(b, "tiles")
    for x in (a, a.bfloat16(), a.half()):
        assert torch.equal(fp8.linear_fp8_fwd(x, w8, out_dtype=torch.bfloat16), ref)
        assert torch.equal(fp8.linear_fp8_fwd(x, w8, out_dtype=torch.bfloat16, keep_transposed=True)[0], ref)
    # dx = dy W with dy = a [M, K] and W^T = b [N, K]
    assert torch.equal(fp8.linear_fp8_bwd(a.bfloat16(), None, w8)[0], ref)
    assert torch.equal(fp8.linear_fp8_bwd(a, None, w8, dx_dtype=torch.bfloat16)[0], ref)


@pytest.mark.parametrize("M,N,K", FORMS)
@pytest.mark.parametrize("scale,block", [("e8m0", "rows"), ("f32", "tiles")])
def test_fast_sums_stay_within_their_bound(M, N, K, scale, block):
    """fast_accum: seven of eight products lose up to 2^-13 of the largest, fp32 sums lose (K + 8) 2^-23, both of sum |a||b|; one
    rounding to bfloat16. On the outliers it does lose: the exact sums are another arithmetic."""
    fp8 = _fp8()
    for fmt in (E4, E5):
        a, b = _outliers(M, N, K, fmt, 7)
        ref = a.double() @ b.double().t()
        qa, qb = _matrix(fp8, a, fmt, "rows", scale), _matrix(fp8, b, E4, block, scale)
        out = fp8.matmul_fp8(qa, qb, fast_accum=True)
        lost = (7 * 2.0 ** -13 + (K + 8) * 2.0 ** -23) * (a.double().abs() @ b.double().abs().t())
        assert out.dtype == torch.bfloat16
        assert ((out.double() - ref).abs() <= lost + 2.0 ** -8 * (ref.abs() + lost)).all()
        if K in (1000, 1024) and (scale == "e8m0" or M > 32):      # (few rows under fp32 scales have no such form)
            assert not torch.equal(out, ref.bfloat16())
    # values without outliers: small integers are exact under 13 bits too
    g = torch.Generator(device="cuda").manual_seed(9)
    a, b = (torch.randint(-3, 4, (r, K), generator=g, device="cuda").float() for r in (M, N))
    want = (a.double() @ b.double().t()).bfloat16()
    assert torch.equal(fp8.matmul_fp8(_matrix(fp8, a, E4, "rows", scale), _matrix(fp8, b, E4, block, scale), fast_accum=True), want)


@pytest.mark.parametrize("M,N,K", [(1, 200, 1024), (16, 70, 500), (40, 90, 1500), (300, 200, 1024)])
def test_fast_sums_of_the_layer_passes(M, N, K):
    fp8 = _fp8()
    a, b = _outliers(M, N, K, E4, 8)
    ref = a.double() @ b.double().t()
    w8, w8t = fp8.fp8_quantize_both(b, "tiles")
    lost = (7 * 2.0 ** -13 + (K + 8) * 2.0 ** -23) * (a.double().abs() @ b.double().abs().t())
    ok = lambda y: y.dtype == torch.bfloat16 and bool(((y.double() - ref).abs() <= lost + 2.0 ** -8 * (ref.abs() + lost)).all())
    for x in (a, a.bfloat16(), a.half()):
        assert ok(fp8.linear_fp8_fwd(x, w8, out_dtype=torch.bfloat16, fast_accum=True))
    assert ok(fp8.linear_fp8_fwd(a.bfloat16(), w8, keep_transposed=True, fast_accum=True)[0])
    # with both gradients: dw is the exact sum whatever is asked of dx (dw [K, N] = q(a^T) q(x^T)^T of integers)
    x = torch.randint(-3, 4, (M, N), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").float()
    dx, dw = fp8.linear_fp8_bwd(a.bfloat16(), fp8.fp8_quantize(x, transpose=True), w8, fast_accum=True)
    assert ok(dx) and torch.equal(dw.double(), a.double().t() @ x.double())


def _spread(rows, cols, fmt, g):
    """codes over the whole of a format, the largest and the smallest among them, as values"""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(fmt).float()
    codes = codes[torch.isfinite(codes)]
    return codes[torch.randint(0, codes.numel(), (rows, cols), generator=g, device="cuda")]


def _scaled(values, scale, block):
    """value64 [rows, cols] of codes' values under scales [S, KB] (float64)"""
    f = scale.repeat_interleave(128, dim=1)[:, :values.shape[1]]
    if block == "tiles":
        f = f.repeat_interleave(128, dim=0)[:values.shape[0]]
    return values.double() * f


SCALE_FORMS = [(3, 70, 600), (20, 130, 520), (7, 90, 8300), (100, 200, 640), (40, 70, 2400), (1500, 1540, 300), (1800, 1930, 260), (4000, 4000, 260)]


def _check_scaled(out, av, bv, K, fast):
    """Where the terms' magnitudes stay within fp32: the sum's own loss, roundings of the block's factor, product and addition
    (three half steps of the block's share), and what lies below the normal range, at most 2^-126 an instruction (four a block).
    Rows and columns that hold a NaN or an infinity are the caller's to look at."""
    mag = av.abs() @ bv.abs().t()
    ref = av @ bv.t()
    ok = mag < 2.0 ** 127
    lost = (K + 8) * 2.0 ** -23 * mag + (K / 32 + 4) * 2.0 ** -126
    if fast:
        lost = lost + 7 * 2.0 ** -13 * mag
    half = torch.finfo(out.dtype).eps / 2
    err = (out.double() - ref).abs()
    assert bool(((err <= lost + half * (ref.abs() + lost)) | ~ok).all())
    assert float(ok.float().mean()) > 0.3


@pytest.mark.parametrize("M,N,K", SCALE_FORMS)
@pytest.mark.parametrize("block", ["rows", "tiles"])
def test_fp32_scales_of_any_size(M, N, K, block):
    """Scales whose product leaves fp32 although their share of the sum does not: large against small sums, large against zero
    blocks (which stay zero), tiny pairs, zero scales."""
    fp8 = _fp8()
    for fmt in (E4, E5):
        g = torch.Generator(device="cuda").manual_seed(21)
        a, b = _spread(M, K, fmt, g), _spread(N, K, E4, g)
        a[0::5, 128:256] = 0
        a[1::5] *= 2.0 ** -6 if fmt == E4 else 2.0 ** -10
        a = a.to(fmt).float()
        kb, s = -(-K // 128), N if block == "rows" else -(-N // 128)
        u = lambda *shape: 1 + torch.rand(*shape, generator=g, device="cuda")
        pick = lambda n, e: torch.tensor(e, device="cuda", dtype=torch.float64)[torch.arange(n, device="cuda") % len(e)]
        two = torch.tensor(2.0, dtype=torch.float64, device="cuda")
        sa = (torch.pow(two, pick(M, [0, 66, -100, 100, -70, 40]))[:, None] * u(M, kb)).float()
        sb = (torch.pow(two, pick(s, [66, 0, -120, 20, 80] if block == "rows" else [66, -60]))[:, None] * u(s, kb)).float()
        sa[0::5, 1] = 3e38
        sa[2, 0] = 0
        qa = fp8.Fp8Matrix(_matrix(fp8, a, fmt).data, sa.t().contiguous(), K, "rows")
        qb = fp8.Fp8Matrix(_matrix(fp8, b).data, sb.t().contiguous(), K, block)
        av, bv = _scaled(a, sa.double(), "rows"), _scaled(b, sb.double(), block)
        _check_scaled(fp8.matmul_fp8(qa, qb, out_dtype=torch.float32), av, bv, K, False)
        _check_scaled(fp8.matmul_fp8(qa, qb, fast_accum=True), av, bv, K, True)
        sa[1, 0] = float("nan")
        qa = fp8.Fp8Matrix(qa.data, sa.t().contiguous(), K, "rows")
        out = fp8.matmul_fp8(qa, qb, out_dtype=torch.float32)
        assert bool(torch.isnan(out[1]).all()) and not bool(torch.isnan(out[2]).any())


@pytest.mark.parametrize("M,N,K", SCALE_FORMS)
@pytest.mark.parametrize("block", ["rows", "tiles"])
def test_scale_bytes_of_any_size(M, N, K, block):
    """Bytes from 0 (2^-127) to 254 under the largest and the smallest codes: values that bf16 or fp32 could not hold, in sums
    that fp32 does."""
    fp8 = _fp8()
    for fmt in (E4, E5):
        g = torch.Generator(device="cuda").manual_seed(22)
        a, b = _spread(M, K, fmt, g), _spread(N, K, E4, g)
        kb, s = -(-K // 128), N if block == "rows" else -(-N // 128)
        pick = lambda n, e: torch.tensor(e, device="cuda", dtype=torch.int32)[torch.arange(n, device="cuda") % len(e)]
        ea = pick(M, [0, 127, 254, 3, 200, 30, 225])[:, None] + torch.randint(0, 2, (M, kb), generator=g, device="cuda", dtype=torch.int32)
        eb = pick(s, [254, 127, 0, 60, 226] if block == "rows" else [253, 0])[:, None].expand(s, kb).contiguous()
        ea.clamp_(max=254)
        qa = fp8.Fp8Matrix.from_parts(_matrix(fp8, a, fmt).data[:, :K], ea, "rows")
        qb = fp8.Fp8Matrix.from_parts(_matrix(fp8, b).data[:, :K], eb, block)
        two = torch.tensor(2.0, dtype=torch.float64, device="cuda")
        av, bv = _scaled(a, torch.pow(two, ea.double() - 127), "rows"), _scaled(b, torch.pow(two, eb.double() - 127), block)
        _check_scaled(fp8.matmul_fp8(qa, qb, out_dtype=torch.float32), av, bv, K, False)
        _check_scaled(fp8.matmul_fp8(qa, qb, fast_accum=True), av, bv, K, True)
        ea[1, 0] = 255
        out = fp8.matmul_fp8(fp8.Fp8Matrix(qa.data, fp8.pack_scale_bytes(ea), K), qb, out_dtype=torch.float32)
        assert bool(torch.isnan(out[1]).all()) and not bool(torch.isnan(out[0]).any())


@pytest.mark.parametrize("M", [1, 16, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_passes_over_the_whole_range(M, dtype):
    """Activations and output gradients near both ends of fp32 against weights that bring them back."""
    fp8 = _fp8()
    N, K = 70, 300
    g = torch.Generator(device="cuda").manual_seed(23)
    for ex, ew in ((-125, 100), (120, -110), (-139, 120)):
        if ex < -133 and dtype == torch.bfloat16:
            continue
        x = (torch.randn(M, K, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** ex).to(dtype)
        w = (torch.randn(N, K, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** ew).float()
        w8, w8t = fp8.fp8_quantize_both(w, "tiles")
        xv, wv = R.requantized(x).cuda(), R.requantized(w, "tiles").cuda()
        for y in (fp8.linear_fp8_fwd(x, w8, out_dtype=torch.float32), fp8.linear_fp8_fwd(x, w8, out_dtype=torch.float32, keep_transposed=True)[0]):
            _check_scaled(y, xv, wv, K, False)
        dy = (torch.randn(M, N, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** ex).to(dtype)
        dx, dw = fp8.linear_fp8_bwd(dy, fp8.fp8_quantize((x.double() * 2.0 ** (ew - ex)).float(), transpose=True), w8t, dx_dtype=torch.float32)
        _check_scaled(dx, R.requantized(dy).cuda(), wv.t(), N, False)
        _check_scaled(dw, R.requantized(dy.t()).cuda(), R.requantized((x.double() * 2.0 ** (ew - ex)).float().t()).cuda(), M, False)


def test_fast_sums_into_out_and_without_terms():
    fp8 = _fp8()
    g = torch.Generator(device="cuda").manual_seed(31)
    for M, N, K in ((5, 70, 0), (5, 70, 300), (200, 70, 0), (200, 300, 2000)):
        a, b = (torch.randint(-3, 4, (r, K), generator=g, device="cuda").float() for r in (M, N))
        old = torch.randint(-8, 9, (M + 2, N + 5), generator=g, device="cuda").bfloat16()
        want = a.double() @ b.double().t()
        qa, qb = _matrix(fp8, a), _matrix(fp8, b, block="tiles")
        for accumulate in (False, True):
            big = old.clone()
            out = big[1:M + 1, 2:N + 2]
            assert fp8.matmul_fp8(qa, qb, out=out, accumulate=accumulate, fast_accum=True) is out
            assert torch.equal(out, (want + (old[1:M + 1, 2:N + 2].double() if accumulate else 0)).bfloat16())
            big[1:M + 1, 2:N + 2] = old[1:M + 1, 2:N + 2]
            assert torch.equal(big, old)
