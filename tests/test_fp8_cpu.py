"""What the 8-bit block-scaled operators refuse (no launch: runs without a GPU)."""
import pytest
import torch

import fp8_ref as R
from stylemesh_amd.runtime import fp8, hip

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def mat(rows, cols, block="rows", dtype=E4, scale="e8m0"):
    kb, s = -(-cols // 128), rows if block == "rows" else -(-rows // 128)
    sc = torch.full((-(-kb // 4), s, 4), 127, dtype=torch.uint8) if scale == "e8m0" else torch.ones(kb, s)
    return fp8.Fp8Matrix(torch.zeros(rows, kb * 128, dtype=torch.uint8).view(dtype), sc, cols, block)


def test_matrix_refusals():
    d, s = torch.zeros(4, 256, dtype=torch.uint8).view(E4), torch.full((1, 4, 4), 127, dtype=torch.uint8)
    assert fp8.Fp8Matrix(d, s, 200).shape == (4, 200)
    bad = [lambda: fp8.Fp8Matrix(d, s, 300), lambda: fp8.Fp8Matrix(d, s, 100), lambda: fp8.Fp8Matrix(d, s, -1),
           lambda: fp8.Fp8Matrix(d, s, 200, "columns"), lambda: fp8.Fp8Matrix(d.view(torch.uint8), s, 200),
           lambda: fp8.Fp8Matrix(d, s[:, :3], 200), lambda: fp8.Fp8Matrix(d, s, 200, "tiles"), lambda: fp8.Fp8Matrix(d, s.int(), 200),
           lambda: fp8.Fp8Matrix(d, torch.ones(4, 2), 200), lambda: fp8.Fp8Matrix(d[:, :128], s, 100), lambda: fp8.Fp8Matrix(d[0], s, 200),
           lambda: fp8.Fp8Matrix(torch.zeros(4 * 256 + 1, dtype=torch.uint8)[1:].view(4, 256).view(E4), s, 200),
           lambda: fp8.Fp8Matrix.from_parts(d, torch.ones(4, 3)), lambda: fp8.Fp8Matrix.from_parts(d[0], torch.ones(4, 2)),
           lambda: fp8.Fp8Matrix.from_parts(d, torch.ones(4, 2).double()), lambda: mat(4, 200).transposed()]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_quantize_refusals():
    x = torch.zeros(4, 8)
    for f in (lambda: fp8.fp8_quantize(x), lambda: fp8.fp8_quantize(x, fmt="e3m4"), lambda: fp8.fp8_quantize(x, block="cols"),
              lambda: fp8.fp8_quantize(x.double()), lambda: fp8.fp8_quantize(x[0]), lambda: fp8.fp8_quantize(x.t()),
              lambda: fp8.fp8_quantize(x[:, ::2]), lambda: fp8.fp8_quantize(x[:1].expand(4, 8)), lambda: fp8.fp8_quantize_both(x.int()),
              lambda: fp8.fp8_quantize(None), lambda: fp8.fp8_quantize(torch.zeros(1, 1).expand(1, 65535 * 128 + 1))):
        with pytest.raises(ValueError):
            f()


def test_product_refusals():
    a, b = mat(4, 200), mat(6, 200)
    x, out = torch.zeros(4, 200), torch.zeros(4, 6)
    for f in (lambda: fp8.matmul_fp8(a, b), lambda: fp8.matmul_fp8(a, mat(6, 201)), lambda: fp8.matmul_fp8(mat(4, 200, "tiles"), b),
              lambda: fp8.matmul_fp8(a, mat(6, 200, dtype=E5)), lambda: fp8.matmul_fp8(a, mat(6, 200, scale="f32")),
              lambda: fp8.matmul_fp8(a, out), lambda: fp8.matmul_fp8(a, b, accumulate=True), lambda: fp8.matmul_fp8(a, b, out=out),
              lambda: fp8.linear_fp8_fwd(x, a), lambda: fp8.linear_fp8_fwd(x, mat(6, 300)), lambda: fp8.linear_fp8_fwd(x, x),
              lambda: fp8.linear_fp8_fwd(x, mat(6, 200, scale="f32")), lambda: fp8.linear_fp8_bwd(x, None, None),
              lambda: fp8.linear_fp8_bwd(x, mat(8, 4), mat(8, 200, "tiles"), dw=torch.zeros(200, 8).half()),
              lambda: fp8.linear_fp8_bwd(x, None, mat(8, 200, "tiles"), dw=torch.zeros(200, 8))):
        with pytest.raises(ValueError):
            f()


def test_c_entry_refusals():
    """Bad arguments come back as an error code before anything is launched."""
    lib = hip.lib
    q = lambda *a: lib.sm_fp8_quantize(*a)
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr()) % 16
    assert q(p, 0, 4, 8, 8, 0, 0, None, None, None, None, None) != 0
    assert q(p, 0, 4, 8, 8, 0, 0, p, None, None, None, None) != 0
    assert q(p, 3, 4, 8, 8, 0, 0, p, p, None, None, None) != 0
    assert q(p, 0, 4, 8, 8, 2, 0, p, p, None, None, None) != 0
    assert q(p, 0, 4, 8, 7, 0, 0, p, p, None, None, None) != 0
    assert q(p, 0, -1, 8, 8, 0, 0, p, p, None, None, None) != 0
    assert q(None, 0, 4, 8, 8, 0, 0, p, p, None, None, None) != 0
    assert q(p, 0, 0, 8, 8, 0, 0, p, p, None, None, None) == 0
    ok = [p, p, 0, 256, p, p, 0, 256, 0, 4, 6, 200, p, 0, 6, 0, None, 0, None]
    m = lambda **k: lib.sm_fp8_matmul(*[k.get(f"a{i}", v) for i, v in enumerate(ok)])
    for bad in (dict(a0=None), dict(a1=None), dict(a2=2), dict(a3=128), dict(a3=250), dict(a0=p + 1), dict(a4=None), dict(a7=100), dict(a9=-1),
                dict(a12=None), dict(a13=3), dict(a14=5)):
        assert m(**bad) != 0, bad
    assert m(a9=0) == 0 and m(a10=0) == 0
    # a product that splits its depth needs its scratch
    need = lib.sm_fp8_matmul_ws_bytes(1, 16, 1 << 20)
    if need:
        assert m(a9=1, a10=16, a11=1 << 20, a3=1 << 20, a7=1 << 20, a14=16, a16=p, a17=need - 1) != 0
    assert lib.sm_fp8_matmul_ws_bytes(0, 5, 5) == 0 and lib.sm_fp8_matmul_ws_bytes(5, -1, 5) == 0


def test_reference_rounding_is_the_types_own():
    """The oracle's grid against torch's casts, over all codes and midpoints."""
    for fmt, dt in fp8.FORMATS.items():
        v = torch.arange(256, dtype=torch.uint8).view(dt).float()
        v = v[torch.isfinite(v)]
        v = torch.cat([v, (v[1:] + v[:-1]) / 2]).double()
        assert torch.equal(R.round_to(v, fmt), v.float().to(dt).double())
    assert R.exponent(448.0, "e4m3") == 0 and R.exponent(448.1, "e4m3") == 1 and R.exponent(224.0, "e4m3") == -1 and R.exponent(0.0, "e4m3") == 0


def test_scale_bytes_round_trip():
    e = torch.randint(0, 256, (5, 7), dtype=torch.int32)
    m = fp8.Fp8Matrix.from_parts(torch.zeros(5, 800, dtype=torch.uint8).view(E4), e)
    assert tuple(m.scale.shape) == (2, 5, 4) and int(m.scale[1, 2, 1]) == int(e[2, 5]) and int(m.scale[1, 2, 3]) == 127
    want = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127)
    got = m.scales().double()
    assert torch.equal(got[e < 255], want[e < 255]) and torch.isnan(got[e == 255]).all()
    t = fp8.Fp8Matrix.from_parts(torch.zeros(300, 700, dtype=torch.uint8).view(E4), e[:3, :6], "tiles").transposed()
    assert t.shape == (700, 300) and torch.equal(t.scales()[e[:3, :6].t() < 255], want[:3, :6].t()[e[:3, :6].t() < 255].float())


def test_gradient_clip_flag_and_entry_refusals():
    import ctypes as C
    from stylemesh_amd.model.optimize import build_parser
    base = ["--style_image_path", "synthetic:1:8x8"]
    assert build_parser().parse_args(base).gradient_clip_val == 0.0
    assert build_parser().parse_args(base + ["--gradient_clip_val", "0.5"]).gradient_clip_val == 0.5
    lib = hip.lib
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr()) % 16
    one = lambda t, v: (t * 1)(v)
    ptrs, n, ty = one(C.c_void_p, p), one(C.c_size_t, 16), one(C.c_int, 0)
    need = lib.sm_grad_norm_ws_bytes(1)
    bad_ty, half = one(C.c_int, 3), one(C.c_int, 1)
    other = one(C.c_void_p, p + 4096)
    assert lib.sm_grad_norm(ptrs, n, ty, -1, 0, p, need, p, None) != 0
    assert lib.sm_grad_norm(ptrs, n, bad_ty, 1, 0, p, need, p, None) != 0
    assert lib.sm_grad_norm(None, n, ty, 1, 0, p, need, p, None) != 0
    assert lib.sm_grad_norm(one(C.c_void_p, None), n, ty, 1, 0, p, need, p, None) != 0
    assert lib.sm_grad_norm(ptrs, n, ty, 1, 0, p, 0, p, None) != 0
    assert lib.sm_grad_norm(ptrs, n, ty, 1, 0, None, need, p, None) != 0
    assert lib.sm_grad_norm(ptrs, n, ty, 1, 0, p, need, None, None) != 0
    assert lib.sm_grad_norm(ptrs, one(C.c_size_t, 1 << 41), ty, 1, 0, p, need, p, None) != 0
    clip = lambda out, oty, mx, ws: lib.sm_grad_clip(ptrs, out, n, ty, oty, 1, 0, mx, p, ws, p, None)
    assert clip(other, ty, -1.0, need) != 0 and clip(other, ty, float("nan"), need) != 0 and clip(None, ty, 1.0, need) != 0
    assert clip(other, bad_ty, 1.0, need) != 0 and clip(ptrs, half, 1.0, need) != 0 and clip(other, ty, 1.0, 8 * 0) != 0
    seg, reg = one(C.c_size_t, 64), one(C.c_float, 0.0)
    g = lambda **k: lib.sm_adam_grad_clip(p, p, k.get("n", 64), seg, reg, 1, 1.0, k.get("t"), k.get("l", 0), k.get("m", 1.0), k.get("ws", p),
                                          k.get("wb", 1 << 15), k.get("out", p), None)
    for bad in (dict(n=0), dict(n=63), dict(t=p, l=1), dict(t=p, l=25), dict(m=-1.0), dict(m=float("nan")), dict(ws=None), dict(wb=8), dict(out=None)):
        assert g(**bad) != 0, bad


def test_gradient_lists_of_host_tensors_are_refused():
    from stylemesh_amd.runtime import gradclip
    t = torch.ones(4)
    for f in (lambda: gradclip.clip_grad_norm([t], 1.0), lambda: gradclip.grad_norm([t]), lambda: gradclip.GradClip([t]),
              lambda: gradclip.clip_grad_norm([t], -1.0), lambda: gradclip.clip_grad_norm([t], 1.0, 3.0), lambda: gradclip.GradClip([t], [])):
        with pytest.raises(ValueError):
            f()


def test_a_matrix_keeps_its_tensors():
    """Pointers are taken once, so the tensors cannot be exchanged; scales that are read as dwords start on one."""
    m = mat(4, 200)
    for name in ("data", "scale", "cols", "block"):
        with pytest.raises(AttributeError):
            setattr(m, name, getattr(m, name))
    d = torch.zeros(4, 256, dtype=torch.uint8).view(E4)
    with pytest.raises(ValueError):
        fp8.Fp8Matrix(d, torch.zeros(17, dtype=torch.uint8)[1:].view(1, 4, 4), 200)
    for e in (256, -1):
        with pytest.raises(ValueError):
            fp8.Fp8Matrix.from_parts(d, torch.full((4, 2), e, dtype=torch.int32))


def test_c_entry_limits():
    """Sizes, pitches and alignments whose offsets the kernels could not hold."""
    lib = hip.lib
    buf = torch.zeros(1 << 12, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr()) % 16
    q = lambda rows, cols, a=p, b=p: lib.sm_fp8_quantize(p, 0, rows, cols, 1 << 31, 0, 0, a, p, b, p, None)
    big = 65535 * 128 + 1
    assert q(big, 1) != 0 and q(1, big) != 0 and q((1 << 31) - 1, 1) != 0 and q(1, (1 << 31) - 1) != 0 and q(1, 1, a=p + 8) != 0 and q(1, 1, b=p + 4) != 0
    ok = [p, p, 0, 256, p, p, 0, 256, 0, 40, 6, 200, p, 0, 6, 0, None, 0, None]
    m = lambda **k: lib.sm_fp8_matmul(*[k.get(f"a{i}", v) for i, v in enumerate(ok)])
    for bad in (dict(a1=p + 1), dict(a5=p + 2), dict(a3=1 << 24), dict(a7=1 << 24), dict(a9=1 << 30), dict(a10=1 << 30, a14=1 << 30),
                dict(a11=(1 << 31) - 1, a3=1 << 31, a7=1 << 31)):
        assert m(**bad) != 0, bad
    ok2 = [p, 0, 200, p, p, 0, 256, 40, 6, 200, p, 0, 6, p, 1 << 30, None]
    f = lambda **k: lib.sm_fp8_linear(*[k.get(f"a{i}", v) for i, v in enumerate(ok2)])
    for bad in (dict(a13=p + 8), dict(a14=100), dict(a2=199), dict(a6=128), dict(a3=p + 8), dict(a7=4, a3=p + 8), dict(a7=4, a6=250), dict(a7=4, a8=1 << 30, a12=1 << 30)):
        assert f(**bad) != 0, bad


def test_tensor_list_walk():
    """The native walk over a list: what it reports of host tensors, odd types and non-tensors."""
    import struct
    from stylemesh_amd import _tensor_list as tl
    packed, at, odd, device, contiguous = tl.pack([torch.ones(3), torch.ones(2, 5).half(), torch.ones(4).bfloat16()])
    assert struct.unpack("3i", packed[48:]) == (0, 2, 1) and odd == -1 and device == -1 and contiguous and at
    assert tl.pack([]) [2:] == (-1, -2, True)
    assert tl.pack([torch.ones(3), torch.ones(3).double()])[2] == 1
    assert tl.pack([torch.ones(3).to_sparse()])[2] == 0
    for bad in ([1], [None], [torch.ones(1), "x"]):
        with pytest.raises(ValueError):
            tl.pack(bad)
    for f in (lambda: tl.pack((torch.ones(1),)), lambda: tl.check_outputs(b"123", b""), lambda: tl.check_outputs([], b"")):
        with pytest.raises(TypeError):
            f()


def test_outputs_of_a_list_against_every_pair():
    """Overlap of outputs with each other and with other entries' inputs, against the quadratic definition."""
    import random
    import struct
    from stylemesh_amd import _tensor_list as tl
    rng = random.Random(3)
    table = lambda e: b"".join(struct.pack(f"{len(e)}{c}", *[x[i] for x in e]) for i, c in enumerate("QQi"))
    seen = set()
    for _ in range(3000):
        n = rng.randint(0, 5)
        span = rng.choice([60, 400])
        g = [(rng.randrange(span), rng.choice([0, 1, 5, 9]), rng.randrange(3)) for _ in range(n)]
        o = [rng.choice([e, (rng.randrange(span), e[1], rng.randrange(3))]) for e in g]
        if n and rng.random() < 0.05:
            o[0] = (o[0][0], o[0][1] + 1, o[0][2])
        end = lambda e: e[0] + e[1] * (2 if e[2] else 4)
        hit = lambda a, b: a[1] and b[1] and a[0] < end(b) and b[0] < end(a)
        want = 0
        if any(a[1] != b[1] for a, b in zip(g, o)):
            want = 1
        elif any(a[1] and a[0] == b[0] and a[2] != b[2] for a, b in zip(g, o)):
            want = 2
        elif any(hit(o[i], o[j]) for i in range(n) for j in range(i)):
            want = 3
        elif any(hit(g[i], o[j]) and (i != j or g[i][0] != o[j][0]) for i in range(n) for j in range(n)):
            want = 4
        assert tl.check_outputs(table(g), table(o)) == want, (g, o)
        t = table(g)
        assert tl.check_outputs(t, t) == (3 if any(hit(g[i], g[j]) for i in range(n) for j in range(i)) else 0)
        seen.add(want)
    assert seen == {0, 1, 2, 3, 4}


def test_gradient_list_limits():
    """Sizes and addresses the packed table could not hold come back as an error."""
    import ctypes as C
    lib = hip.lib
    p = 1 << 20
    arr = lambda t, *v: (t * len(v))(*v)
    ty = arr(C.c_int, 0, 0)
    norm = lambda ptrs, n: lib.sm_grad_norm(arr(C.c_void_p, *ptrs), arr(C.c_size_t, *n), ty, 2, 0, p, 1 << 14, p, None)
    assert norm((p, 1 << 48), (4, 4)) != 0 and norm((p, p), (1 << 63, 1 << 63)) != 0 and norm((p, p), (1 << 40, 4)) != 0
    clip = lambda out: lib.sm_grad_clip(arr(C.c_void_p, p, p), arr(C.c_void_p, *out), arr(C.c_size_t, 4, 4), ty, ty, 2, 0, 1.0, p, 1 << 14, p, None)
    assert clip((p, 1 << 50)) != 0
    assert lib.sm_grad_norm(arr(C.c_void_p, p, p), arr(C.c_size_t, 4, 4), ty, 2, 0, p + 4, 1 << 14, p, None) != 0


def test_copies_have_their_own_pointers():
    """copy, deepcopy and pickle make a matrix of the new tensors, not one that still points at the old ones."""
    import copy
    import pickle
    for m in (mat(4, 200), mat(300, 200, "tiles"), mat(4, 200, scale="f32")):
        for c in (copy.copy(m), copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
            assert c._ptrs == (c.data.data_ptr(), c.scale.data_ptr()) and c.shape == m.shape and c.block == m.block and c._pitch == m._pitch
            assert torch.equal(c.data.view(torch.uint8), m.data.view(torch.uint8)) and torch.equal(c.scale, m.scale)
        assert copy.deepcopy(m)._ptrs != m._ptrs


def test_codes_laid_out_by_columns_are_copied():
    """Quantising a transposed matrix in plain torch leaves the codes column by column: the same matrix, rows at the pitch."""
    g = torch.Generator().manual_seed(4)
    codes = torch.randint(0, 120, (256, 300), generator=g, dtype=torch.uint8).t()      # [300, 256], strides (1, 300)
    sc = torch.full((1, 300, 4), 127, dtype=torch.uint8)
    for dtype in (E4, E5):
        m = fp8.Fp8Matrix(codes.view(dtype), sc, 256)
        assert m.data.is_contiguous() and m.data.dtype == dtype and torch.equal(m.data.view(torch.uint8), codes)
        assert m._ptrs == (m.data.data_ptr(), m.scale.data_ptr()) and m._pitch == 256
    row = torch.zeros(256, 1, dtype=torch.uint8).t().view(E4)                          # one row: nothing to copy
    assert fp8.Fp8Matrix(row, torch.full((1, 1, 4), 127, dtype=torch.uint8), 256).data.data_ptr() == row.data_ptr()


def test_gradients_of_an_iterator_live_until_the_launch(monkeypatch):
    """A list of temporaries has no owner but the call: their memory must not be handed out again (as this call's scratch, for
    one) before the launch that reads it."""
    import weakref
    from stylemesh_amd.runtime import gradclip, ops
    refs, alive = [], []

    def temporaries():
        for _ in range(3):
            t = torch.ones(4)
            refs.append(weakref.ref(t))
            yield t
            del t

    note = lambda result: alive.append(all(r() is not None for r in refs)) or result
    real_pack, real_empty = gradclip._tensor_list.pack, torch.empty
    monkeypatch.setattr(gradclip._tensor_list, "pack", lambda tensors: (*real_pack(tensors)[:3], 0, True))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "empty", lambda *size, dtype, device: note(real_empty(*size, dtype=dtype)))
    monkeypatch.setattr(ops, "eager_stream", lambda: 0)
    monkeypatch.setattr(ops, "lib", type("Lib", (), {"sm_grad_norm_ws_bytes": staticmethod(lambda n: 8192),
                                                     "sm_grad_norm": staticmethod(lambda *a: note(0)),
                                                     "sm_grad_clip": staticmethod(lambda *a: note(0))}))
    for call in (lambda: gradclip.grad_norm(temporaries()), lambda: gradclip.clip_grad_norm(temporaries(), 1.0)):
        refs.clear()
        alive.clear()
        call()
        assert len(alive) == 3 and all(alive)


def test_fast_sums_are_for_bfloat16_results():
    a, b, x = mat(4, 200), mat(6, 200), torch.zeros(4, 200)
    for f in (lambda: fp8.matmul_fp8(a, b, out_dtype=torch.float32, fast_accum=True), lambda: fp8.matmul_fp8(a, b, out_dtype=torch.float16, fast_accum=True),
              lambda: fp8.linear_fp8_fwd(x, b, fast_accum=True), lambda: fp8.linear_fp8_fwd(x, b, torch.float16, fast_accum=True),
              lambda: fp8.linear_fp8_bwd(torch.zeros(4, 6), None, mat(200, 6, "tiles"), fast_accum=True)):
        with pytest.raises(ValueError):
            f()
    lib = hip.lib
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr()) % 16
    ok = [p, p, 0, 256, p, p, 0, 256, 0, 4, 6, 200, p, 0, 6, 0, None, 0, None]
    m = lambda t, **k: lib.sm_fp8_matmul(*[k.get(f"a{i}", v) if i != 13 else t for i, v in enumerate(ok)])
    for t in (16, 18, 19, 32, 33, -1, -15):
        assert m(t) != 0 and m(t, a9=0) != 0, t
        assert lib.sm_fp8_linear(p, 0, 200, p, p, 0, 256, 0, 6, 200, p, t, 6, p, 1 << 15, None) != 0, t
    assert m(17, a9=0) == 0 and lib.sm_fp8_linear(p, 0, 200, p, p, 0, 256, 0, 6, 200, p, 17, 6, p, 1 << 15, None) == 0


def test_clipped_tensors_versions_rise(monkeypatch):
    """A graph that saved a tensor before it was clipped must be refused by autograd, as after torch's own in-place operations."""
    from stylemesh_amd import _tensor_list as tl
    from stylemesh_amd.runtime import gradclip, ops
    a, b, v = torch.ones(4), torch.ones(6), torch.ones(9)
    with torch.inference_mode():
        i = torch.ones(2)
    before = [t._version for t in (a, v)]
    tl.written([a, v[2:5], i])
    assert [t._version for t in (a, v)] == [n + 1 for n in before] and b._version == 0
    for bad, kind in (((a,), TypeError), ([a, None], ValueError)):
        with pytest.raises(kind):
            tl.written(bad)
    real_pack, real_empty = tl.pack, torch.empty
    monkeypatch.setattr(tl, "pack", lambda tensors: (*real_pack(tensors)[:3], 0, True))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "empty", lambda *size, dtype, device: real_empty(*size, dtype=dtype))
    monkeypatch.setattr(ops, "eager_stream", lambda: 0)
    monkeypatch.setattr(ops, "lib", type("Lib", (), {"sm_grad_norm_ws_bytes": staticmethod(lambda n: 8192), "sm_grad_norm": staticmethod(lambda *a: 0),
                                                     "sm_grad_clip": staticmethod(lambda *a: 0)}))
    w = torch.ones(4, requires_grad=True)
    y = (w * b[:4]).sum()
    gradclip.clip_grad_norm([b], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out, n = torch.ones(6), b._version
    plan = gradclip.GradClip([b], [out])
    plan.norm()
    assert (b._version, out._version) == (n, 0)
    plan.clip(1.0)
    assert (b._version, out._version) == (n, 1)


def test_tensors_of_a_recording_graph_are_refused_on_the_host_too():
    b, x = mat(6, 200), torch.zeros(4, 200, requires_grad=True)
    for f in (lambda: fp8._check_no_graph(x, "x"), lambda: fp8._check_no_graph(x * 2, "x"), lambda: fp8.linear_fp8_fwd(x, b, keep_transposed=True)):
        with pytest.raises(ValueError, match="requires a gradient"):
            f()
    with torch.no_grad():
        fp8._check_no_graph(x, "x")
    fp8._check_no_graph(x.detach(), "x")


def test_matrices_whose_tensors_were_exchanged_are_named():
    make = lambda: mat(4, 200)
    fp8._check_held(make(), None, mat(300, 200, "tiles"), mat(4, 200, scale="f32"))
    other = torch.zeros(4, 256, dtype=torch.uint8).view(E4)
    m = make()
    m.data.set_(other)                                    # as large as before: its own codes from now on
    fp8._check_held(m)
    assert m._ptrs[0] == other.data_ptr()
    for change in (lambda m: m.data.set_(other[:3]), lambda m: m.data.untyped_storage().resize_(0), lambda m: m.scale.set_(m.scale[:, :2].clone()),
                   lambda m: m.scale.untyped_storage().resize_(3), lambda m: m.data.set_(other[:, :128]),
                   lambda m: m.data.set_(torch.zeros(256, 4, dtype=torch.uint8).view(E4).t())):
        m = make()
        change(m)
        with pytest.raises(ValueError, match="since it was made"):
            fp8._check_held(m)


def test_a_plan_refuses_tensors_whose_memory_was_exchanged(monkeypatch):
    from stylemesh_amd import _tensor_list as tl
    from stylemesh_amd.runtime import gradclip, ops
    launched = []
    real_pack, real_empty = tl.pack, torch.empty

    def pack(tensors):      # (host tensors: the addresses that the walk leaves out)
        packed, at, odd, _, contiguous = real_pack(tensors)
        return b"".join(t.data_ptr().to_bytes(8, "little") for t in tensors) + packed[8 * len(tensors):], at, odd, 0, contiguous
    monkeypatch.setattr(tl, "pack", pack)
    monkeypatch.setattr(tl, "check_outputs", lambda a, b: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "empty", lambda *size, dtype, device: real_empty(*size, dtype=dtype))
    monkeypatch.setattr(ops, "eager_stream", lambda: 0)
    note = staticmethod(lambda *a: launched.append(1) and 0 or 0)
    monkeypatch.setattr(ops, "lib", type("Lib", (), {"sm_grad_norm_ws_bytes": staticmethod(lambda n: 8192), "sm_grad_norm": note, "sm_grad_clip": note}))
    for where in ("grads", "out"):
        for change in (lambda t: setattr(t, "data", t.data.clone()), lambda t: t.untyped_storage().resize_(0), lambda t: t.set_(t[:3].clone()),
                       lambda t: setattr(t, "data", t.data.half())):
            grads, out = [torch.ones(4), torch.ones(6)], [torch.ones(4), torch.ones(6)]
            plan = gradclip.GradClip(grads, out)
            plan.clip(1.0), plan.norm()
            n = len(launched)
            change(getattr(plan, where)[1])
            for f in (lambda: plan.clip(1.0), plan.norm):
                with pytest.raises(ValueError, match="exchanged"):
                    f()
            assert len(launched) == n == 2
            launched.clear()


def test_calls_that_no_step_program_may_hold_are_not_replayable():
    for name in ("sm_fp8_quantize", "sm_fp8_matmul", "sm_fp8_linear", "sm_fp8_linear_backward", "sm_grad_norm", "sm_grad_clip", "sm_adam_grad_clip",
                 "sm_adam_fused_clipped"):
        assert hip.lib.sm_call_id(name.encode()) < 0, name
    assert hip.lib.sm_call_id(b"sm_adam_fused") >= 0


def test_clip_scratch_must_be_aligned():
    import ctypes as C
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr()) % 16
    seg, reg = (C.c_size_t * 1)(64), (C.c_float * 1)(0.0)
    for off in (1, 2, 4):
        assert hip.lib.sm_adam_grad_clip(p, p, 64, seg, reg, 1, 1.0, None, 0, 1.0, p + off, 1 << 15, p, None) != 0
