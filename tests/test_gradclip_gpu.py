"""Global gradient norm and clipping (runtime/gradclip.py) against the formulas in 64 bits."""
import math

import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _mod():
    require_gpu()
    from stylemesh_amd.runtime import gradclip
    return gradclip


def _grads(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g) * scale * 10.0 ** -(i % 3)).to(DT[dtypes[i % len(dtypes)]]).cuda()
            for i, s in enumerate(sizes)]


def _norm64(grads, kind):
    vals = [t.double().cpu() for t in grads if t is not None and t.numel()]
    if not vals:
        return 0.0
    if kind == math.inf:
        return max(float(v.abs().max()) for v in vals)
    return math.sqrt(sum(float((v * v).sum()) for v in vals))


def _check(before, after, norm, max_norm, kind):
    """norm: one rounding to fp32 (plus the 64-bit sums' own error, below 2^-40 for these sizes); values: coefficient rounded
    to fp32, product in fp32, one rounding to the output's type - each at most half a step, subnormals absolutely."""
    want = _norm64(before, kind)
    assert abs(float(norm) - want) <= 2.0 ** -24 * want * (1 + 2.0 ** -10)
    coef = min(1.0, max_norm / (want + 1e-6))
    for b, a in zip(before, after):
        ref = b.double().cpu() * coef
        fi = torch.finfo(a.dtype)
        err = (a.double().cpu() - ref).abs()
        assert (err <= (fi.eps / 2 + 2.0 ** -22) * ref.abs() + fi.smallest_normal * fi.eps).all()


SIZES = [[1], [7], [1, 2, 3], [4096], [4097, 0, 4095], [100003], [64, 1728, 64, 36864, 128, (128, 64, 3, 3)], [5] * 130, [999] * 257, [2_500_000, 3, 70000]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtypes", [("f32",), ("bf16",), ("f16", "f32", "bf16")], ids="-".join)
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_norm_and_clip(sizes, dtypes, kind):
    gc = _mod()
    grads = _grads(sizes, dtypes)
    before = [g.clone() for g in grads]
    want = _norm64(before, kind)
    n = gc.grad_norm(grads, kind)
    assert n.dtype == torch.float32 and n.shape == () and abs(float(n) - want) <= 2.0 ** -24 * want * (1 + 2.0 ** -10)
    for max_norm in (0.3 * want, 10 * want + 1):
        # into other tensors, of every type
        for odt in (None, "f32", "bf16", "f16"):
            out = [torch.full_like(g, 3.0, dtype=g.dtype if odt is None else DT[odt]) for g in grads]
            norm = gc.GradClip(grads, out).clip(max_norm, kind)
            _check(before, out, norm, max_norm, kind)
            assert all(torch.equal(a, b) for a, b in zip(grads, before))
        # in place
        mine = [g.clone() for g in before]
        norm = gc.clip_grad_norm(mine, max_norm, kind)
        _check(before, mine, norm, max_norm, kind)
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(mine, before))


def test_same_bits_every_time_and_whatever_the_list_form():
    gc = _mod()
    grads = _grads([300_001, 5, 40_000] * 50, ("f32", "bf16"))
    plan = gc.GradClip(grads, [torch.empty_like(g) for g in grads])
    first = plan.clip(0.1)
    for _ in range(5):
        assert torch.equal(plan.clip(0.1), first) and torch.equal(gc.grad_norm(grads), first) and torch.equal(plan.norm(), first)


def test_values_whose_squares_leave_fp32():
    gc = _mod()
    for v in (3e30, 1e-30, 2.0 ** -140):
        g = torch.full((10_000,), v, device="cuda")
        want = _norm64([g], 2.0)
        n = gc.grad_norm([g])
        assert abs(float(n) - want) <= 2.0 ** -24 * want + 2.0 ** -150


def test_non_finite_norms_follow_the_formula():
    gc = _mod()
    for kind in (2.0, math.inf):
        for where in (0, 9_999):
            g = torch.ones(10_000, device="cuda")
            h = torch.ones(33, device="cuda")
            g[where] = float("inf")
            assert math.isinf(float(gc.clip_grad_norm([g, h], 1.0, kind)))
            assert math.isnan(float(g[where])) and float(g.nan_to_num(0.0).abs().sum()) == 0 and float(h.abs().sum()) == 0
            g = torch.ones(10_000, device="cuda")
            g[where] = float("nan")
            assert math.isnan(float(gc.clip_grad_norm([g, h], 1.0, kind)))
            assert torch.isnan(g).all() and torch.isnan(h).all()


def test_lists_with_gaps_and_empty_lists():
    gc = _mod()
    assert float(gc.grad_norm([])) == 0.0 and float(gc.grad_norm([None, torch.zeros(0, device="cuda")])) == 0.0
    assert float(gc.clip_grad_norm([], 1.0)) == 0.0
    assert float(gc.clip_grad_norm([None, torch.zeros(0, device="cuda")], 1.0)) == 0.0
    g = torch.full((4,), 2.0, device="cuda")
    assert float(gc.clip_grad_norm([None, g, torch.zeros(0, device="cuda"), None], 1.0)) == 4.0
    torch.testing.assert_close(g.cpu(), torch.full((4,), 0.5), rtol=2.0 ** -20, atol=0)
    z = torch.zeros(5, device="cuda")
    assert float(gc.clip_grad_norm([z], 0.0)) == 0.0 and not z.any()
    assert float(gc.grad_norm([g, g], 2.0)) == pytest.approx(math.sqrt(2.0), rel=1e-5)       # listed twice, counted twice


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_views_at_any_element(dtype):
    """Unaligned starts, odd lengths, permuted dense layouts; the neighbours of what is written keep their values."""
    gc = _mod()
    for off in range(0, 9):
        base = torch.randn(20_000, generator=torch.Generator().manual_seed(off)).to(DT[dtype]).cuda()
        views = [base[off:off + 4099], base[5_000 + off:5_001 + off], base[6_000:6_000 + 8 * (off + 1)]]
        outb = torch.full((20_000,), 9.0, dtype=DT[dtype], device="cuda")
        outs = [outb[3 * off:3 * off + 4099], outb[5_000:5_001], outb[7_001:7_001 + 8 * (off + 1)]]
        before = [v.clone() for v in views]
        norm = gc.GradClip(views, outs).clip(0.5)
        _check(before, outs, norm, 0.5, 2.0)
        keep = torch.ones(20_000, dtype=torch.bool, device="cuda")
        for o in outs:
            s = (o.data_ptr() - outb.data_ptr()) // outb.element_size()
            keep[s:s + o.numel()] = False
        assert (outb[keep] == 9.0).all()
        ref = base.clone()
        norm = gc.clip_grad_norm(views, 0.5)
        _check(before, views, norm, 0.5, 2.0)
        keep = torch.ones(20_000, dtype=torch.bool, device="cuda")
        for v in views:
            s = (v.data_ptr() - base.data_ptr()) // base.element_size()
            keep[s:s + v.numel()] = False
        assert torch.equal(base[keep], ref[keep])
    p = torch.randn(6, 10, 4, 3).to(DT[dtype]).cuda().permute(2, 0, 3, 1)
    before = p.clone()
    norm = gc.clip_grad_norm([p], 0.25)
    _check([before], [p], norm, 0.25, 2.0)
    cl = torch.randn(2, 8, 5, 5).to(DT[dtype]).cuda().to(memory_format=torch.channels_last)
    out = torch.empty_like(cl)
    norm = gc.GradClip([cl], [out]).clip(0.25)
    _check([cl], [out], norm, 0.25, 2.0)


def test_refusals():
    gc = _mod()
    g = torch.ones(8, 8, device="cuda")
    h = torch.ones(8, 8, device="cuda")
    bad = [lambda: gc.clip_grad_norm([g, g], 1.0), lambda: gc.clip_grad_norm([g, g[2:]], 1.0), lambda: gc.clip_grad_norm([g.flatten()[:33], g.flatten()[32:]], 1.0),
           lambda: gc.clip_grad_norm([g], -1.0), lambda: gc.clip_grad_norm([g], float("nan")), lambda: gc.clip_grad_norm([g], 1.0, 1.0),
           lambda: gc.clip_grad_norm([g[:, ::2]], 1.0), lambda: gc.clip_grad_norm([g[:, :4]], 1.0), lambda: gc.clip_grad_norm([g[:1].expand(8, 8)], 1.0),
           lambda: gc.clip_grad_norm([g.double()], 1.0), lambda: gc.clip_grad_norm([g.cpu()], 1.0), lambda: gc.grad_norm([g.int()]),
           lambda: gc.GradClip([g, h], [h, g]), lambda: gc.GradClip([g], []), lambda: gc.GradClip([g], [None]), lambda: gc.GradClip([g], [h[:4]]),
           lambda: gc.GradClip([g], [h.t()]), lambda: gc.GradClip([g, h], [torch.empty_like(g)] * 2), lambda: gc.GradClip([g, g], [g, h]),
           lambda: gc.GradClip([g[:4]], [g[2:6]])]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    assert (g == 1).all() and (h == 1).all()
    # the same gradient into two outputs is fine: it is only read
    a, b = torch.empty_like(g), torch.empty_like(g)
    assert float(gc.GradClip([g, g], [a, b]).clip(1e9)) == pytest.approx(math.sqrt(128.0)) and torch.equal(a, g) and torch.equal(b, g)


def test_in_a_graph_and_on_two_streams():
    """A captured clip replayed between eager work; two plans on two streams at once."""
    gc = _mod()
    src = _grads([70_001, 12, 5_000], ("f32", "bf16"))
    outs = [[torch.empty_like(g) for g in src] for _ in range(2)]
    plans = [gc.GradClip(src, o) for o in outs]
    want_n = plans[0].clip(0.5).clone()
    want = [o.clone() for o in outs[0]]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, norms = [], []
    for p, s in zip(plans, st):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            p.clip(0.5)
        s.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            norms.append(p.clip(0.5))
        graphs.append(gr)
    for r in range(4):
        for o in outs[0] + outs[1] + norms:
            o.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, st):
            with torch.cuda.stream(s):
                gr.replay()
        eager = gc.grad_norm(src)
        torch.cuda.synchronize()
        assert torch.equal(eager, want_n)
        for n, o in zip(norms, outs):
            assert torch.equal(n, want_n) and all(torch.equal(a, b) for a, b in zip(o, want))


def test_more_than_two_to_the_31_elements():
    gc = _mod()
    n = (1 << 31) + 4097
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-1], g[0], g[1 << 31] = 3.0, 4.0, 12.0
    assert float(gc.grad_norm([g])) == 13.0
    assert float(gc.clip_grad_norm([g], 1.0)) == 13.0
    ref = torch.tensor([4.0, 12.0, 3.0]) / 13.0
    assert ((g[[0, 1 << 31, n - 1]].float().cpu() - ref).abs() <= 2.0 ** -8 * ref).all() and float(g[1:100].abs().sum()) == 0


def test_one_plan_in_two_graphs():
    """Two captured graphs of the SAME plan on two streams at once: neither uses the other's partial sums."""
    gc = _mod()
    src = _grads([3_000_001, 12, 50_000], ("f32", "bf16"))
    plan = gc.GradClip(src)
    want = [plan.norm(), plan.norm(math.inf)]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, norms = [], []
    for kind, s in zip((2.0, math.inf), st):
        s.wait_stream(torch.cuda.current_stream())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            norms.append(plan.norm(kind))
        graphs.append(gr)
    for r in range(4):
        for n in norms:
            n.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, st):
            with torch.cuda.stream(s):
                gr.replay()
        eager = plan.norm()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(norms, want))


def test_a_copied_plan_works_on_the_copies():
    import copy
    gc = _mod()
    g = [torch.full((5000,), 2.0, device="cuda"), torch.ones(3, device="cuda")]
    for out in (None, [torch.zeros_like(t) for t in g]):
        plan = gc.GradClip(g, out)
        other = copy.deepcopy(plan)
        other.clip(1.0)
        assert float(g[0][0]) == 2.0 and (out is None or not out[0].any())
        assert all(a.data_ptr() != b.data_ptr() for a, b in zip(plan.grads, other.grads))
        assert float(torch.stack([t.norm() for t in other.out]).norm()) == pytest.approx(1.0, rel=1e-5)
        assert (other.out is other.grads) == (out is None)


def test_a_plan_refuses_tensors_whose_memory_was_exchanged():
    gc = _mod()
    for change in (lambda t: setattr(t, "data", t.data.clone()), lambda t: t.untyped_storage().resize_(0), lambda t: setattr(t, "data", t.data.half())):
        g, o = [torch.full((5000,), 2.0, device="cuda"), torch.ones(3, device="cuda")], [torch.zeros(5000, device="cuda"), torch.zeros(3, device="cuda")]
        for plan, t in ((gc.GradClip(g, o), o[0]), (gc.GradClip(g), g[0])):
            assert float(plan.clip(1e9)) == pytest.approx(math.sqrt(20003.0), rel=1e-6)
            keep = t.data
            change(t)
            for f in (lambda: plan.clip(1.0), plan.norm):
                with pytest.raises(ValueError, match="exchanged"):
                    f()
            if keep.untyped_storage().nbytes():
                t.data = keep                              # the plan's own memory again
                assert float(plan.clip(1e9)) == pytest.approx(math.sqrt(20003.0), rel=1e-6)
