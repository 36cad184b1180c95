"""8-bit block-scaled matrices (runtime/fp8.py) against their definition in 64 bits (fp8_ref.py)."""
import math

import pytest
import torch

import fp8_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _fp8():
    require_gpu()
    from stylemesh_amd.runtime import fp8
    return fp8


def _rand(rows, cols, seed, dtype=torch.float32, spread=4.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    return x.clamp(-6e4, 6e4).to(dtype)


def _check_matrix(q, x, block, fmt):
    """codes, scale bytes and padding of ``q`` are exactly the definition's"""
    vals, exps = R.quantize(x, block, fmt)
    got = q.data.float().double().cpu()
    assert tuple(got.shape) == tuple(vals.shape)
    torch.testing.assert_close(got, vals, rtol=0, atol=0, equal_nan=True)
    kb = exps.shape[1]
    want = torch.full((-(-kb // 4), exps.shape[0], 4), 127, dtype=torch.uint8)
    for j in range(kb):
        want[j // 4, :, j % 4] = (exps[:, j] + 127).to(torch.uint8)
    assert torch.equal(q.scale.cpu(), want)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (1, 129), (3, 127), (128, 128), (129, 640), (257, 385), (16, 4096), (1000, 5)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_is_the_definition(rows, cols, dtype, fmt):
    fp8 = _fp8()
    x = _rand(rows, cols, rows * 7 + cols, DT[dtype])
    xd = x.cuda()
    for block in ("rows", "tiles"):
        _check_matrix(fp8.fp8_quantize(xd, block, fmt), x, block, fmt)
        _check_matrix(fp8.fp8_quantize(xd, block, fmt, transpose=True), x.t(), block, fmt)
        n, t = fp8.fp8_quantize_both(xd, block, fmt)
        _check_matrix(n, x, block, fmt)
        _check_matrix(t, x.t(), block, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", ["rows", "tiles"])
def test_quantize_extreme_values(fmt, block):
    """Zeros, subnormals, the largest floats, values at the rounding borders and exactly at the format's limit, NaN and
    infinities (which must leave their block's scale alone)."""
    fp8 = _fp8()
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    rows = [[0.0, -0.0, 0.0], [tiny, -tiny, 3 * tiny], [big, -big, 1.0], [448.0, 447.9999, 1.0], [448.0001, 1.0, -2.0],
            [57344.0, 57345.0, 3.0], [1.0, 1.0625, 1.1875], [float("nan"), 2.0, 3.0], [float("inf"), 5.0, -0.25],
            [float("-inf"), float("nan"), 0.0], [2.0 ** -126, 2.0 ** -127, 2.0 ** -140], [2.0 ** 119, 2.0 ** 127 * 1.75, 1e30]]
    x = torch.zeros(128 * len(rows), 200)
    for i, r in enumerate(rows):
        x[128 * i, :3] = torch.tensor(r)
        x[128 * i + 5, 150:153] = torch.tensor(r)
    _check_matrix(fp8.fp8_quantize(x.cuda(), block, fmt), x, block, fmt)
    _check_matrix(fp8.fp8_quantize(x.cuda(), block, fmt, transpose=True), x.t(), block, fmt)


def test_quantize_every_rounding_border():
    """All codes' values and the midpoints between neighbours, shifted by one fp32 step either way."""
    fp8 = _fp8()
    for fmt, dt in fp8.FORMATS.items():
        v = torch.arange(256, dtype=torch.uint8).view(dt).float()
        v = v[torch.isfinite(v)].sort().values
        mid = (v[1:] + v[:-1]) / 2
        pts = torch.cat([v, mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)])
        x = torch.zeros(pts.numel(), 130)
        x[:, 0], x[:, 1] = pts, R.LIMIT[fmt]
        _check_matrix(fp8.fp8_quantize(x.cuda(), "rows", fmt), x, "rows", fmt)


def test_quantize_strided_offset_and_empty():
    fp8 = _fp8()
    base = _rand(50, 401, 5).cuda()
    for dt in DT.values():
        b = base.to(dt)
        for view in (b[:, 3:300], b[7:, 1:130], b[::3, 5:], b[4:5, 2:9]):
            _check_matrix(fp8.fp8_quantize(view), view.cpu(), "rows", "e4m3")
            _check_matrix(fp8.fp8_quantize(view, transpose=True), view.cpu().t(), "rows", "e4m3")
    for shape in ((0, 5), (5, 0), (0, 0)):
        q = fp8.fp8_quantize(torch.zeros(*shape, device="cuda"))
        assert q.shape == shape and q.data.shape[0] == shape[0]
        t = fp8.fp8_quantize(torch.zeros(*shape, device="cuda"), transpose=True)
        assert t.shape == shape[::-1]


def _operands(fp8, M, N, K, block, fmt, scale, seed=0):
    a, b = _rand(M, K, seed + 1, spread=1.0), _rand(N, K, seed + 2, spread=1.0)
    qa, qb = fp8.fp8_quantize(a.cuda(), "rows", fmt), fp8.fp8_quantize(b.cuda(), block)
    if scale == "f32":
        g = torch.Generator().manual_seed(seed)
        f = lambda q: fp8.Fp8Matrix(q.data, (q.scales() * (1 + torch.rand(q.scales().shape, generator=g).cuda())).t().contiguous(),
                                    q.cols, q.block)
        qa, qb = f(qa), f(qb)
    return qa, qb, _value(qa), _value(qb)


def _value(q):
    """what an Fp8Matrix stands for in 64 bits (its scales are checked against the definition elsewhere)"""
    s = q.scales().double().cpu().repeat_interleave(128, dim=1)
    if q.block == "tiles":
        s = s.repeat_interleave(128, dim=0)[:q.rows]
    return (q.data.float().double().cpu() * s)[:, :q.cols]


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 4096, 512), (2, 130, 257), (5, 33, 1000), (16, 48, 640), (17, 1, 129), (31, 300, 2304), (64, 64, 128),
          (65, 129, 131), (127, 255, 385), (128, 128, 1024), (200, 513, 1100), (300, 64, 5000), (257, 1025, 513), (1000, 260, 256), (1, 7, 20000),
          (40, 24, 9000), (700, 700, 130)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("block", ["rows", "tiles"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
def test_matmul(M, N, K, block, scale):
    fp8 = _fp8()
    for fmt in ("e4m3", "e5m2"):
        a, b, av, bv = _operands(fp8, M, N, K, block, fmt, scale)
        ref = av @ bv.t()
        for dt in (torch.float32, torch.bfloat16):
            out = fp8.matmul_fp8(a, b, out_dtype=dt)
            assert out.dtype == dt
            bound = R.matmul_bound(av, bv, dt, ref)
            assert ((out.double().cpu() - ref).abs() <= bound).all()


def test_matmul_is_exact_on_integers():
    """Small integers: every product and partial sum is exact in fp32, so the result is too - for every shape rule."""
    fp8 = _fp8()
    g = torch.Generator().manual_seed(3)
    for M, N, K in SHAPES + [(512, 512, 2048), (2048, 2048, 256), (4096, 300, 384), (260, 4100, 640)]:
        a = torch.randint(-8, 9, (M, K), generator=g).float()
        b = torch.randint(-8, 9, (N, K), generator=g).float()
        ref = (a.cuda().double() @ b.cuda().double().t())
        for block in ("rows", "tiles"):
            out = fp8.matmul_fp8(fp8.fp8_quantize(a.cuda()), fp8.fp8_quantize(b.cuda(), block), out_dtype=torch.float32)
            assert torch.equal(out.double(), ref), (M, N, K, block)
            out16 = fp8.matmul_fp8(fp8.fp8_quantize(a.cuda()), fp8.fp8_quantize(b.cuda(), block), out_dtype=torch.float16)
            assert torch.equal(out16, ref.float().half()), (M, N, K, block)


@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (19, 130, 700), (300, 200, 257), (5, 3, 20000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_matmul_into_strided_out_and_accumulate(M, N, K, dtype):
    fp8 = _fp8()
    g = torch.Generator().manual_seed(4)
    a = torch.randint(-3, 4, (M, K), generator=g).float()
    b = torch.randint(-1, 2, (N, K), generator=g).float()
    qa, qb = fp8.fp8_quantize(a.cuda()), fp8.fp8_quantize(b.cuda(), "tiles")
    big = torch.full((M + 2, N + 9), 7.0, device="cuda", dtype=DT[dtype])
    out = big[1:M + 1, 3:N + 3]
    fp8.matmul_fp8(qa, qb, out=out)
    ref = a.double() @ b.double().t()
    assert torch.equal(out.cpu(), ref.to(DT[dtype]))
    first = out.clone().double().cpu()
    fp8.matmul_fp8(qa, qb, out=out, accumulate=True)
    assert torch.equal(out.cpu(), (first + ref).to(DT[dtype]))      # |sums| < 2^24: exact in fp32, rounded once
    border = big.clone()
    border[1:M + 1, 3:N + 3] = 7.0
    assert (border == 7.0).all()


def test_matmul_empty_dimensions():
    fp8 = _fp8()
    z = lambda m, k, block="rows": fp8.fp8_quantize(torch.zeros(m, k, device="cuda"), block)
    assert fp8.matmul_fp8(z(0, 5), z(3, 5)).shape == (0, 3)
    assert fp8.matmul_fp8(z(3, 5), z(0, 5, "tiles")).shape == (3, 0)
    out = torch.full((3, 4), 2.0, device="cuda")
    assert torch.equal(fp8.matmul_fp8(z(3, 0), z(4, 0), out=out, accumulate=True), torch.full((3, 4), 2.0, device="cuda"))
    assert torch.equal(fp8.matmul_fp8(z(3, 0), z(4, 0), out=out), torch.zeros(3, 4, device="cuda"))


def test_matmul_nan_and_inf_stay_in_their_row():
    fp8 = _fp8()
    for M in (4, 300):
        a, b = _rand(M, 500, 1, spread=0.5), _rand(70, 500, 2, spread=0.5)
        a[2, 130] = float("nan")
        b[5, 3] = float("nan")
        qa, qb = fp8.fp8_quantize(a.cuda()), fp8.fp8_quantize(b.cuda())
        out = fp8.matmul_fp8(qa, qb, out_dtype=torch.float32).cpu()
        bad = torch.zeros(M, 70, dtype=torch.bool)
        bad[2], bad[:, 5] = True, True
        assert torch.equal(torch.isnan(out), bad)
        a[2, 130] = float("inf")
        out = fp8.matmul_fp8(fp8.fp8_quantize(a.cuda(), fmt="e5m2"), fp8.fp8_quantize(b.cuda()), out_dtype=torch.float32).cpu()
        assert torch.isfinite(out[[0, 1, 3]][:, [0, 4, 6]]).all() and not torch.isfinite(out[2]).any()


def test_matmul_scale_bytes_over_the_whole_range():
    """Scales far from 1 on both sides, 2^-127 (byte 0) among them, and the NaN byte 255."""
    fp8 = _fp8()
    for M in (3, 200):
        K, N = 512, 20
        codes = torch.ones(M, K).to(torch.float8_e4m3fn).cuda()
        wcodes = torch.ones(N, K).to(torch.float8_e4m3fn).cuda()
        sa = torch.full((M, 4), 127, dtype=torch.int32)
        sa[0], sa[1, 0], sa[2] = 0, 255, torch.tensor([254, 200, 100, 1])
        sb = torch.full((N, 4), 127, dtype=torch.int32)
        sb[3] = 60
        a = fp8.Fp8Matrix.from_parts(codes, sa.cuda())
        b = fp8.Fp8Matrix.from_parts(wcodes, sb.cuda())
        out = fp8.matmul_fp8(a, b, out_dtype=torch.float32).double().cpu()
        two = torch.tensor(2.0, dtype=torch.float64)
        ref = 128 * (torch.pow(two, sa.double() - 127) @ torch.pow(two, sb.double() - 127).t())
        ref[1] = float("nan")
        ref[2, :3] = float("inf") if ref[2, 0] > torch.finfo(torch.float32).max else ref[2, 0]
        ref = ref.float().double()
        ok = ~torch.isnan(ref)
        assert torch.isnan(out[1]).all()
        # a result below the normal range may be flushed: 2^-126 absolutely; else one rounding
        fin = ok & torch.isfinite(ref)
        assert ((out - ref).abs()[fin] <= 2.0 ** -23 * ref.abs()[fin] + 2.0 ** -126).all()
        assert torch.equal(torch.isinf(out)[ok], torch.isinf(ref)[ok])


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (1, 4100, 1000), (3, 130, 257), (16, 500, 2304), (37, 257, 515), (300, 140, 640)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_forward(M, N, K, dtype):
    fp8 = _fp8()
    x, w = _rand(M, K, 11, DT[dtype], spread=1.0), _rand(N, K, 12, spread=1.0) * 0.05
    w8 = fp8.fp8_quantize(w.cuda(), "tiles")
    y = fp8.linear_fp8_fwd(x.cuda(), w8)
    xv, wv = R.requantized(x), R.requantized(w, "tiles")
    ref = xv @ wv.t()
    assert y.dtype == DT[dtype]
    assert ((y.double().cpu() - ref).abs() <= R.matmul_bound(xv, wv, DT[dtype], ref)).all()
    y2, xt = fp8.linear_fp8_fwd(x.cuda(), w8, out_dtype=torch.float32, keep_transposed=True)
    assert ((y2.double().cpu() - ref).abs() <= R.matmul_bound(xv, wv, torch.float32, ref)).all()
    _check_matrix(xt, x.t(), "rows", "e4m3")


def test_linear_forward_rows_are_independent():
    """A row's result does not depend on what else is in the batch, NaN included, at every batch size around the rules' borders."""
    fp8 = _fp8()
    x, w = _rand(70, 700, 21, torch.bfloat16, spread=0.5).cuda(), _rand(200, 700, 22, spread=0.5).cuda()
    w8 = fp8.fp8_quantize(w, "tiles")
    xv, wv = R.requantized(x.cpu()), R.requantized(w.cpu(), "tiles")
    ref = xv @ wv.t()
    bound = R.matmul_bound(xv, wv, torch.bfloat16, ref)
    for m in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 70):
        y = fp8.linear_fp8_fwd(x[:m], w8)
        assert ((y.double().cpu() - ref[:m]).abs() <= bound[:m]).all(), m
        xn = x[:m].clone()
        xn[m // 2, 5] = float("nan")
        yn = fp8.linear_fp8_fwd(xn, w8)
        assert torch.isnan(yn[m // 2]).all()
        keep = [i for i in range(m) if i != m // 2]
        assert torch.equal(yn[keep], y[keep])


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (130, 70, 257), (300, 140, 640), (515, 33, 100)])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_backward(M, N, K, fmt, dtype):
    fp8 = _fp8()
    x, w, dy = _rand(M, K, 31, DT[dtype], spread=1.0), _rand(N, K, 32, spread=1.0) * 0.05, _rand(M, N, 33, DT[dtype], spread=1.0) * 1e-3
    w8, w8t = fp8.fp8_quantize_both(w.cuda(), "tiles")
    _, xt = fp8.linear_fp8_fwd(x.cuda(), w8, keep_transposed=True)
    dx, dw = fp8.linear_fp8_bwd(dy.cuda(), xt, w8t, fmt=fmt)
    gv, gtv = R.requantized(dy, "rows", fmt), R.requantized(dy.t(), "rows", fmt)
    wv, xtv = R.requantized(w, "tiles"), R.requantized(x.t())
    ref = gv @ wv
    assert dx.dtype == DT[dtype] and ((dx.double().cpu() - ref).abs() <= R.matmul_bound(gv, wv.t(), DT[dtype], ref)).all()
    ref = gtv @ xtv.t()
    assert dw.dtype == torch.float32 and ((dw.double().cpu() - ref).abs() <= R.matmul_bound(gtv, xtv, torch.float32, ref)).all()
    # the stored weight's own transpose gives the same bits; a missing operand leaves its gradient out
    dx2, none = fp8.linear_fp8_bwd(dy.cuda(), None, w8.transposed(), fmt=fmt)
    assert none is None and torch.equal(dx2, dx)
    acc = dw.clone()
    none, dw2 = fp8.linear_fp8_bwd(dy.cuda(), xt, None, fmt=fmt, dw=acc, accumulate=True)
    assert none is None and dw2 is acc and torch.equal(acc, dw + dw)


def test_linear_gradients_against_differences():
    """On values the format holds exactly the layer is linear, so finite differences ARE the gradients: integers, exact in
    fp32 throughout, compared without a tolerance."""
    fp8 = _fp8()
    g = torch.Generator().manual_seed(9)
    M, N, K = 150, 70, 200
    ints = lambda *s, lim=4: torch.randint(-lim, lim + 1, s, generator=g).float().cuda()
    x, w, dy = ints(M, K), ints(N, K), ints(M, N, lim=2)
    f = lambda xx, ww: (dy.double() * fp8.linear_fp8_fwd(xx, fp8.fp8_quantize(ww, "tiles")).double()).sum()
    _, xt = fp8.linear_fp8_fwd(x, fp8.fp8_quantize(w, "tiles"), keep_transposed=True)
    dx, dw = fp8.linear_fp8_bwd(dy, xt, fp8.fp8_quantize(w, "tiles", transpose=True))
    for _ in range(4):
        d = ints(M, K, lim=2)
        assert float(f(x + d, w) - f(x, w)) == float((dx.double() * d.double()).sum())
        d = ints(N, K, lim=2)
        assert float(f(x, w + d) - f(x, w)) == float((dw.double() * d.double()).sum())


def test_from_parts_transposed_and_dequantize():
    fp8 = _fp8()
    w = _rand(300, 257, 41, spread=1.0)
    q, qt = fp8.fp8_quantize_both(w.cuda(), "tiles")
    t = q.transposed()
    assert torch.equal(t.data.view(torch.uint8), qt.data.view(torch.uint8)) and torch.equal(t.scale, qt.scale) and t.shape == (257, 300)
    assert torch.equal(q.dequantize().double().cpu(), R.requantized(w, "tiles"))
    vals, exps = R.quantize(w, "rows", "e4m3")
    p = fp8.Fp8Matrix.from_parts(vals[:, :257].to(torch.float8_e4m3fn).cuda(), (exps + 127).int().cuda())
    n = fp8.fp8_quantize(w.cuda())
    assert torch.equal(p.data.view(torch.uint8), n.data.view(torch.uint8)) and torch.equal(p.scale, n.scale)
    f = fp8.Fp8Matrix.from_parts(q.data[:, :257], q.scales(), "tiles")       # fp32 scales
    assert torch.equal(f.dequantize(), q.dequantize()) and torch.equal(f.transposed().dequantize(), q.dequantize().t())


def test_offsets_beyond_32_bits():
    """Codes, inputs and results larger than 2^32 bytes / 2^31 elements: the last rows are right."""
    fp8 = _fp8()
    K, M = 65536, 70000                                   # 4.6 G codes, 9.2 GB of bf16
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(5)
    tail = torch.randint(-4, 5, (3, K), generator=g).float()
    x[-3:] = tail.cuda().bfloat16()
    q = fp8.fp8_quantize(x)
    assert torch.equal(q.data[-3:].float().cpu(), R.quantize(tail, "rows", "e4m3")[0].float())
    t = fp8.fp8_quantize(x, transpose=True)
    assert t.shape == (K, M)
    del x
    assert torch.equal(t.data[-200:, M - 3:M].float().cpu() * t.scales()[-200:, -1:].cpu(), tail[:, -200:].t())
    del t
    w = torch.randint(-2, 3, (24, K), generator=g).float()
    w8 = fp8.fp8_quantize(w.cuda(), "tiles")
    out = fp8.matmul_fp8(q, w8, out_dtype=torch.float32)
    assert torch.equal(out[-3:].cpu().double(), tail.double() @ w.double().t()) and not out[:-3].any()
    del out
    # as the second operand (a long list of weight rows against one activation row)
    a8 = fp8.fp8_quantize(w[:1].cuda())
    out = fp8.matmul_fp8(a8, fp8.Fp8Matrix(q.data, q.scale, K, "rows"), out_dtype=torch.float32)
    assert torch.equal(out[0, -3:].cpu().double(), tail.double() @ w[0].double()) and not out[0, :-3].any()
    del q, out
    ones = lambda n: fp8.fp8_quantize(torch.ones(n, 128, device="cuda"))
    out = fp8.matmul_fp8(ones(60000), ones(40000), out_dtype=torch.bfloat16)      # 2.4 G results
    assert bool((out[-1] == 128).all()) and bool((out[30000] == 128).all())


def test_runs_on_the_current_stream_and_in_a_graph():
    """Two captured graphs of split products (scratch of their own) replayed on two streams, against the eager results."""
    fp8 = _fp8()
    g = torch.Generator().manual_seed(6)
    mk = lambda *s: torch.randint(-4, 5, s, generator=g).float().cuda()
    xs = [mk(5, 20000), mk(5, 20000)]
    w8 = fp8.fp8_quantize(mk(64, 20000), "tiles")
    dy = mk(5, 64)
    def step(x):
        y, xt = fp8.linear_fp8_fwd(x, w8, out_dtype=torch.float32, keep_transposed=True)
        return (y,) + fp8.linear_fp8_bwd(dy, xt, wt)
    wt = w8.transposed()
    want = [step(x) for x in xs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for x, st in zip(xs, side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(x)
        st.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(step(x))
        graphs.append(gr)
    for round_ in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, side):
            with torch.cuda.stream(st):
                gr.replay()
        eager = step(xs[round_ % 2])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[round_ % 2]))


def test_training_step_of_a_layer():
    """Quantise, product, gradient products, norm and clip, update - in the order a training step runs them - against the
    same step in 64 bits."""
    fp8 = _fp8()
    from stylemesh_amd.runtime.gradclip import GradClip
    M, N, K, lr, max_norm = 200, 96, 300, 0.5, 0.25
    x, w, target = _rand(M, K, 51, spread=0.3), _rand(N, K, 52, spread=0.3) * 0.05, _rand(M, N, 53, spread=0.1)
    wd, xd, td = w.cuda(), x.cuda(), target.cuda()
    dw = torch.empty(N, K, device="cuda")
    plan = GradClip([dw])
    w64 = w.double()
    for step in range(3):
        w8, w8t = fp8.fp8_quantize_both(wd, "tiles")
        y, xt = fp8.linear_fp8_fwd(xd, w8, keep_transposed=True)
        dy = (y - td) * (2.0 / y.numel())
        _, _ = fp8.linear_fp8_bwd(dy, xt, w8t, dw=dw)
        raw = dw.clone()
        norm = plan.clip(max_norm)
        # the 64-bit step from the same weights and the same output gradient (whose codes a last bit could tip)
        ref = R.requantized(dy.cpu().t()) @ R.requantized(x.t()).t()
        bound = R.matmul_bound(R.requantized(dy.cpu().t()), R.requantized(x.t()), torch.float32, ref)
        assert ((raw.double().cpu() - ref).abs() <= bound).all()
        rn = float(raw.double().norm())
        assert abs(float(norm) - rn) <= 2.0 ** -23 * rn
        coef = min(1.0, max_norm / (rn + 1e-6))
        assert ((dw.double() - raw.double() * coef).abs() <= 2.0 ** -22 * raw.double().abs() + 1e-44).all()
        wd -= lr * dw


def test_linear_backward_without_elements():
    fp8 = _fp8()
    q = lambda m, k, block="rows": fp8.fp8_quantize(torch.zeros(m, k, device="cuda"), block)
    for M, N, K in ((0, 5, 7), (3, 0, 7), (3, 5, 0)):
        dy = torch.ones(M, N, device="cuda")
        dx, dw = fp8.linear_fp8_bwd(dy, q(K, M), q(K, N, "tiles"))
        assert dx.shape == (M, K) and dw.shape == (N, K) and not dx.any() and not dw.any()
        old = torch.full((N, K), 3.0, device="cuda")
        assert fp8.linear_fp8_bwd(dy, q(K, M), None, dw=old, accumulate=True)[1] is old and (old == 3.0).all()
        assert not fp8.linear_fp8_bwd(dy, q(K, M), None, dw=old)[1].any()


def test_products_on_a_side_stream_and_interleaved():
    """Two streams at once, each with split products, quantisers and backward passes of its own: no scratch is shared."""
    fp8 = _fp8()
    g = torch.Generator().manual_seed(8)
    mk = lambda *s: torch.randint(-4, 5, s, generator=g).float().cuda()
    x, w, dy = [mk(100, 9000) for _ in range(2)], mk(64, 9000), mk(100, 64)
    w8, w8t = fp8.fp8_quantize_both(w, "tiles")
    def work(i):
        y, xt = fp8.linear_fp8_fwd(x[i], w8, out_dtype=torch.float32, keep_transposed=True)
        return (y,) + fp8.linear_fp8_bwd(dy, xt, w8t)
    want = [work(i) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [[], []]
        for r in range(6):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(work(i))
        torch.cuda.synchronize()
        for i in range(2):
            for res in got[i]:
                assert all(torch.equal(a, b) for a, b in zip(res, want[i]))


@pytest.mark.parametrize("M", [1, 7, 16, 17, 40])
@pytest.mark.parametrize("K", [1, 129, 1100])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_forward_of_views(M, K, dtype):
    """Inputs that start at any element and whose rows lie further apart, on both sides of the fused rule's border."""
    fp8 = _fp8()
    big, w = _rand(M + 2, K + 9, 41, DT[dtype], spread=0.5), _rand(70, K, 42, spread=0.5)
    w8 = fp8.fp8_quantize(w.cuda(), "tiles")
    x = big[1:M + 1, 3:K + 3]
    xv, wv = R.requantized(x), R.requantized(w, "tiles")
    ref = xv @ wv.t()
    for out_dtype in (torch.bfloat16, torch.float32):
        y = fp8.linear_fp8_fwd(big.cuda()[1:M + 1, 3:K + 3], w8, out_dtype=out_dtype)
        assert ((y.double().cpu() - ref).abs() <= R.matmul_bound(xv, wv, out_dtype, ref)).all()


@pytest.mark.parametrize("M", [1, 16, 20, 40, 200])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_linear_forward_long_rows_with_nan_and_inf(M, bad):
    """K where a bfloat16 result takes the 8-bit instruction: a NaN or an infinity fills its own row with NaN and nothing else."""
    fp8 = _fp8()
    x, w = _rand(M, 2000, 51, torch.bfloat16, spread=0.5).cuda(), _rand(90, 2000, 52, spread=0.5).cuda()
    w8 = fp8.fp8_quantize(w, "tiles")
    y = fp8.linear_fp8_fwd(x, w8)
    assert torch.isfinite(y).all()
    x[M // 2, 1999] = float(bad)
    yb = fp8.linear_fp8_fwd(x, w8)
    keep = [i for i in range(M) if i != M // 2]
    assert torch.isnan(yb[M // 2]).all() and torch.equal(yb[keep], y[keep])


@pytest.mark.parametrize("M,N,K", [(1800, 1930, 1100), (4000, 4000, 1100), (4000, 3900, 520)])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_matmul_large_tiles(M, N, K, scale, out):
    """Sizes that take the larger tiles, both arithmetics; the reference covers rows and columns at the tiles' borders."""
    fp8 = _fp8()
    for fmt, block in (("e4m3", "rows"), ("e5m2", "tiles")):
        a, b, av, bv = _operands(fp8, M, N, K, block, fmt, scale, seed=60)
        y = fp8.matmul_fp8(a, b, out_dtype=DT[out]).double().cpu()
        rows = sorted({0, 15, 16, 63, 127, 128, 255, 256, 1000, M - 129, M - 128, M - 17, M - 2, M - 1})
        ref = av[rows] @ bv.t()
        assert ((y[rows] - ref).abs() <= R.matmul_bound(av[rows], bv, DT[out], ref)).all()
        cols = sorted({0, 15, 63, 64, 127, 128, 255, 256, 1001, N - 130, N - 3, N - 1})
        ref = av @ bv[cols].t()
        assert ((y[:, cols] - ref).abs() <= R.matmul_bound(av, bv[cols], DT[out], ref)).all()


@pytest.mark.parametrize("rows,cols", [(1500, 1500), (129, 16400), (4300, 515)])
@pytest.mark.parametrize("dtype,fmt", [("f32", "e4m3"), ("bf16", "e5m2"), ("f16", "e4m3")])
def test_quantize_large_is_the_definition(rows, cols, dtype, fmt):
    """Enough tiles for the large blocks' form; NaN, infinities, a zero row and column, and subnormal scales among them."""
    fp8 = _fp8()
    x = _rand(rows, cols, rows + cols, DT[dtype], spread=1.0)
    x[7], x[:, 130] = 0, 0
    x[100, 3], x[101, 140], x[128, cols - 1] = float("nan"), float("inf"), float("-inf")
    if dtype == "f32":
        x[:, 5] *= 2.0 ** -140
        x[20] *= 2.0 ** -140
    xd = x.cuda()
    n, t = fp8.fp8_quantize_both(xd, "rows", fmt)
    _check_matrix(n, x, "rows", fmt)
    _check_matrix(t, x.t(), "rows", fmt)
    q = fp8.fp8_quantize(xd, "rows", fmt, transpose=True)
    assert torch.equal(q.data.view(torch.uint8), t.data.view(torch.uint8)) and torch.equal(q.scale, t.scale)
    assert torch.equal(fp8.fp8_quantize(xd, "rows", fmt).data.view(torch.uint8), n.data.view(torch.uint8))
    a, b = fp8.fp8_quantize_both(xd, "tiles", fmt)
    _check_matrix(a, x, "tiles", fmt)
    _check_matrix(b, x.t(), "tiles", fmt)


def test_a_recorded_step_with_these_calls_is_not_replayed():
    """They allocate their results: a recording must not come back with this call's pointers."""
    fp8 = _fp8()
    from stylemesh_amd.runtime import gradclip, hip, ops, program
    x = torch.ones(4, 200, device="cuda")
    w8 = fp8.fp8_quantize(torch.ones(8, 200, device="cuda"), "tiles")
    q, t = fp8.fp8_quantize_both(x)
    for call in (lambda: fp8.fp8_quantize(x), lambda: fp8.matmul_fp8(q, w8), lambda: fp8.linear_fp8_fwd(x, w8),
                 lambda: fp8.linear_fp8_bwd(torch.ones(4, 8, device="cuda"), t, w8.transposed()), lambda: gradclip.clip_grad_norm([x], 1e9),
                 lambda: gradclip.grad_norm([x])):
        ops.lib = rec = program.Recorder()
        try:
            call()
        finally:
            ops.lib = hip.lib
        assert rec.problem is not None


def test_refusals_on_the_device():
    """What the native calls do not take comes back as a ValueError that names it, and nothing is written."""
    fp8 = _fp8()
    x = torch.ones(8, 256, device="cuda")
    w8 = fp8.fp8_quantize(torch.ones(16, 256, device="cuda"), "tiles")
    q = fp8.fp8_quantize(x)
    out = torch.zeros(8, 16, device="cuda")
    dy, (_, xt), wt = torch.ones(8, 16, device="cuda"), fp8.fp8_quantize_both(x), w8.transposed()
    for f in (lambda: fp8.fp8_quantize(x.t()), lambda: fp8.fp8_quantize(x[:, ::2]), lambda: fp8.fp8_quantize(x[0]), lambda: fp8.fp8_quantize(x.double()),
              lambda: fp8.fp8_quantize(x[:1].expand(8, 256)), lambda: fp8.fp8_quantize(x.to_sparse()), lambda: fp8.fp8_quantize_both(x.cpu()),
              lambda: fp8.linear_fp8_fwd(x.t(), w8), lambda: fp8.linear_fp8_fwd(x[:, :255], w8), lambda: fp8.linear_fp8_fwd(x.cpu(), w8),
              lambda: fp8.linear_fp8_fwd(x.int(), w8), lambda: fp8.linear_fp8_fwd(x, w8, out_dtype=torch.int32), lambda: fp8.linear_fp8_fwd(None, w8),
              lambda: fp8.matmul_fp8(q, w8, out=out.t()), lambda: fp8.matmul_fp8(q, w8, out=out[:7]), lambda: fp8.matmul_fp8(q, w8, out=out.cpu()),
              lambda: fp8.matmul_fp8(q, w8, out=out, out_dtype=torch.float16), lambda: fp8.matmul_fp8(q, w8, out=out[:1].expand(8, 16)),
              lambda: fp8.linear_fp8_bwd(dy.t(), xt, wt), lambda: fp8.linear_fp8_bwd(dy[:7], xt, wt), lambda: fp8.linear_fp8_bwd(dy, xt, wt, dw=out),
              lambda: fp8.linear_fp8_bwd(dy, xt, wt, dw=torch.zeros(256, 16, device="cuda").t()), lambda: fp8.linear_fp8_bwd(dy, xt, wt, dx_dtype=torch.int8)):
        with pytest.raises(ValueError):
            f()
    torch.cuda.synchronize()
    assert not out.any()


@pytest.mark.parametrize("M,N,K", [(1500, 1540, 300), (200, 12000, 1300), (1500, 1500, 1)])
@pytest.mark.parametrize("scale,block", [("e8m0", "rows"), ("f32", "rows"), ("f32", "tiles")])
def test_matmul_more_small_tiles_than_two_a_cu(M, N, K, scale, block):
    fp8 = _fp8()
    a, b, av, bv = _operands(fp8, M, N, K, block, "e4m3", scale, seed=70)
    ref = av @ bv.t()
    for dt in (torch.float32, torch.bfloat16):
        out = fp8.matmul_fp8(a, b, out_dtype=dt)
        assert ((out.double().cpu() - ref).abs() <= R.matmul_bound(av, bv, dt, ref)).all()


@pytest.mark.parametrize("M,N,K", [(1029, 517, 1283), (517, 300, 900), (300, 517, 129)])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_linear_backward_of_both_products_in_one_launch(M, N, K, fmt):
    """Either product may be the longer one; the result is the two single calls', bit for bit."""
    fp8 = _fp8()
    dy, x, w = _rand(M, N, 81, spread=0.5).cuda(), _rand(M, K, 82, spread=0.5).cuda(), _rand(N, K, 83, spread=0.5).cuda()
    xt, wt = fp8.fp8_quantize(x, transpose=True), fp8.fp8_quantize(w, "tiles", transpose=True)
    dx, dw = fp8.linear_fp8_bwd(dy, xt, wt, fmt=fmt)
    q, qt = fp8.fp8_quantize_both(dy, fmt=fmt)
    assert torch.equal(dx, fp8.matmul_fp8(q, wt, out_dtype=torch.float32)) and torch.equal(dw, fp8.matmul_fp8(qt, xt, out_dtype=torch.float32))
    base = torch.randn_like(dw)
    acc = base.clone()
    fp8.linear_fp8_bwd(dy, xt, wt, fmt=fmt, dw=acc, accumulate=True)
    assert torch.equal(acc, fp8.matmul_fp8(qt, xt, out=base, accumulate=True))


@pytest.mark.parametrize("M,N,K", [(256, 130, 300), (128, 70, 257)])
def test_linear_backward_from_codes_laid_out_by_columns(M, N, K):
    """Transposed activations quantised in plain torch: with M a multiple of 128 their codes lie column by column."""
    fp8 = _fp8()
    x, w, dy = _rand(M, K, 91, spread=0.5).cuda(), _rand(N, K, 92, spread=0.5).cuda(), _rand(M, N, 93, spread=0.5).cuda()
    want, wt = fp8.fp8_quantize(x, transpose=True), fp8.fp8_quantize(w, "tiles", transpose=True)
    codes = want.data.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    assert not codes.is_contiguous()
    xt = fp8.Fp8Matrix(codes, want.scale, M)
    for a, b in zip(fp8.linear_fp8_bwd(dy, xt, wt), fp8.linear_fp8_bwd(dy, want, wt)):
        assert torch.equal(a, b)


def test_written_tensors_versions_rise():
    """out and dw of the caller, and clipped gradients: autograd refuses a graph that saved what has been written since."""
    fp8 = _fp8()
    from stylemesh_amd.runtime.gradclip import clip_grad_norm
    x, w = torch.ones(8, 256, device="cuda"), torch.ones(16, 256, device="cuda")
    a, b = fp8.fp8_quantize(x), fp8.fp8_quantize(w, "tiles")
    out, dw, g = torch.zeros(8, 16, device="cuda"), torch.zeros(16, 256, device="cuda"), torch.ones(8, 16, device="cuda")
    for t, call in ((out, lambda: fp8.matmul_fp8(a, b, out=out)), (dw, lambda: fp8.linear_fp8_bwd(g, fp8.fp8_quantize(x, transpose=True), None, dw=dw)),
                    (g, lambda: clip_grad_norm([g], 0.5))):
        leaf = torch.ones(t.shape, device="cuda", requires_grad=True)
        y = (leaf * t).sum()
        n = t._version
        call()
        assert t._version == n + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_tensors_of_a_recording_graph_are_refused():
    """A result without a gradient must not come back silently; quantising a parameter is fine, and so are the two halves inside an
    autograd.Function, whose gradients are the halves' own."""
    fp8 = _fp8()
    w = torch.nn.Parameter(_rand(70, 300, 1, spread=0.3).cuda())
    w8, w8t = fp8.fp8_quantize_both(w, "tiles")
    assert not w8.scales().requires_grad
    for x in (torch.ones(4, 300, device="cuda", requires_grad=True), torch.ones(4, 300, device="cuda", requires_grad=True) * 2):
        q = fp8.fp8_quantize(x)
        out = torch.zeros(4, 70, device="cuda", requires_grad=True)
        dy = torch.ones(4, 70, device="cuda")
        _, xt = fp8.fp8_quantize_both(x)
        for f in (lambda: fp8.linear_fp8_fwd(x, w8), lambda: fp8.linear_fp8_fwd(x, w8, keep_transposed=True), lambda: fp8.matmul_fp8(q, w8, out=out),
                  lambda: fp8.linear_fp8_bwd(dy.clone().requires_grad_(), xt, w8t), lambda: fp8.linear_fp8_bwd(dy, xt, w8t, dw=w)):
            with pytest.raises(ValueError, match="requires a gradient"):
                f()
        with torch.no_grad():
            y = fp8.linear_fp8_fwd(x, w8)
        assert torch.equal(y, fp8.linear_fp8_fwd(x.detach(), w8)) and not out.any()

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            w8, ctx.wt = fp8.fp8_quantize_both(w, "tiles")
            y, ctx.xt = fp8.linear_fp8_fwd(x, w8, keep_transposed=True)
            return y

        @staticmethod
        def backward(ctx, dy):
            return fp8.linear_fp8_bwd(dy, ctx.xt, ctx.wt)

    x = torch.nn.Parameter(_rand(40, 300, 2, spread=0.3).cuda())
    dy = _rand(40, 70, 3, spread=0.3).cuda()
    Layer.apply(x, w).backward(dy)
    dx, dw = fp8.linear_fp8_bwd(dy, fp8.fp8_quantize(x, transpose=True), w8t)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


def test_matrices_whose_tensors_were_exchanged():
    """Addresses are read at every call: codes exchanged for others are the ones used, memory given up is refused."""
    fp8 = _fp8()
    g = torch.Generator().manual_seed(2)
    ints = lambda *s: torch.randint(-3, 4, s, generator=g).float().cuda()
    x, w, v, dy = ints(5, 300), ints(70, 300), ints(70, 300), ints(5, 70)
    q, w8, v8 = fp8.fp8_quantize(x), fp8.fp8_quantize(w, "tiles"), fp8.fp8_quantize(v, "tiles")
    assert torch.equal(w8.scale, v8.scale)
    xt, wt = fp8.fp8_quantize(x, transpose=True), w8.transposed()
    calls = lambda: (lambda: fp8.matmul_fp8(q, w8), lambda: fp8.linear_fp8_fwd(x, w8), lambda: fp8.linear_fp8_fwd(x, w8, keep_transposed=True))
    w8.data.set_(v8.data)
    want = x @ v.t()
    assert torch.equal(fp8.matmul_fp8(q, w8, out_dtype=torch.float32), want) and torch.equal(fp8.linear_fp8_fwd(x, w8), want)
    w8.data.set_(v8.data[:69])
    for f in calls():
        with pytest.raises(ValueError, match="since it was made"):
            f()
    w8 = fp8.fp8_quantize(w, "tiles")
    w8.data.untyped_storage().resize_(0)
    for f in calls():
        with pytest.raises(ValueError, match="since it was made"):
            f()
    for m in (xt, wt):
        m.scale.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match="since it was made"):
            fp8.linear_fp8_bwd(dy, xt if m is xt else None, wt if m is wt else None)
    q.data.set_(q.data.cpu().view(torch.uint8).cuda().view(torch.float8_e5m2).view(torch.uint8).view(torch.float8_e4m3fn))
    assert torch.equal(fp8.matmul_fp8(q, fp8.fp8_quantize(w, "tiles"), out_dtype=torch.float32), x @ w.t())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_subnormal_values_under_normal_scales(dtype, fmt):
    """Blocks whose largest value leaves a normal scale (2^-126 and just above) over values below the type's normal range, which the
    format holds: they keep their codes, in the rows, tiles, transposed and small forms and inside the layer's forward pass."""
    fp8 = _fp8()
    fi = torch.finfo(DT[dtype])
    low = math.log2(fi.smallest_normal)
    g = torch.Generator().manual_seed(6)
    for rows, cols in ((20, 300), (1300, 1500)):
        steps = torch.randint(-64, 65, (rows, cols), generator=g).double()
        x = steps * 2.0 ** (low - 6)                       # multiples of 1/64 of the smallest normal value: subnormal, or that value
        top = 2.0 ** (low + torch.arange(cols) % 12)
        x[torch.arange(rows) % 3 == 0] = torch.where(torch.arange(cols) % 7 == 0, top, x[torch.arange(rows) % 3 == 0])
        x = x.to(DT[dtype])
        xd = x.cuda()
        for block in ("rows", "tiles")[:1 if rows > 1000 else 2]:
            n, t = fp8.fp8_quantize_both(xd, block, fmt)
            _check_matrix(n, x, block, fmt)
            _check_matrix(t, x.t(), block, fmt)
            assert torch.equal(fp8.fp8_quantize(xd, block, fmt).data.view(torch.uint8), n.data.view(torch.uint8))
    if fmt == "e4m3":
        w = torch.eye(300)[:70] * 2.0 ** 100
        y = fp8.linear_fp8_fwd(x[:9, :300].cuda(), fp8.fp8_quantize(w.cuda(), "tiles"), out_dtype=torch.float32)
        assert torch.equal(y.double().cpu(), (R.requantized(x[:9, :300]) * 2.0 ** 100)[:, :70].float().double())
