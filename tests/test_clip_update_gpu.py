"""Gradient clipping inside the fused texture update: norm and coefficient of the total gradient (data term + regulariser), the
clipped update, and the paths that turn it on (engine, optimizer facade, trainer)."""
import math
import tempfile

import numpy as np
import pytest
import torch

from golden_cases import FLAGSETS
from gpu_util import require_gpu
from test_engine_gpu import make_engine
from test_model_surface_gpu import make_model, to_cuda
from test_round2_gpu import small_views

pytestmark = pytest.mark.gpu


def _state(sizes, seed, live=None):
    g = torch.Generator().manual_seed(seed)
    n = sum(sizes)
    r = lambda s: (torch.randn(n, generator=g) * s).cuda()
    p, gr, m, v = r(20.0), r(1e-3), r(1e-4), r(1e-4) ** 2
    if live is not None:
        p, gr, m, v = p * live, gr * live, m * live, v * live
    return p, gr, m, v


def _total64(p, g, seg_end, reg, gs):
    out = torch.empty(p.numel(), dtype=torch.float64, device=p.device)
    b = 0
    for e, c in zip(seg_end, reg):
        out[b:e] = np.float32(gs) * g[b:e].double() + float(np.float32(c)) * p[b:e].double()
        b = e
    return out


SIZES = [[3 * 64 * 64, 3 * 32 * 32, 3 * 16 * 16, 3 * 8 * 8], [5], [1023, 1030], [3 * 512 * 512, 7], [3 * 1000 * 1000, 3 * 500 * 500]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: str(s[0]))
@pytest.mark.parametrize("flagged", [False, True])
def test_norm_coefficient_and_clipped_update(sizes, flagged):
    """norm: fp32 elements (one rounded multiply-add each: half a step, which the 64-bit sum of squares can only carry over) and
    one rounding; m, v: the gradient's rounding, the coefficient's and the product's, then the update's own three."""
    require_gpu()
    from stylemesh_amd.runtime import ops
    seg_end = np.cumsum(sizes).tolist()
    n, reg, gs = seg_end[-1], [0.41e-4, 0.2e-4, 0.05e-4, 0.0][:len(sizes)], 0.5
    flags, log2 = None, 0
    live = None
    if flagged:
        log2 = 6
        flags = (torch.rand(-(-n // 64), generator=torch.Generator().manual_seed(1)) < 0.4).to(torch.int32).cuda()
        live = flags.bool().repeat_interleave(64)[:n]
    p, g, m, v = _state(sizes, 3, live)
    tot = _total64(p, g, seg_end, reg, gs)
    want = float(tot.norm())
    clip, ws = torch.zeros(2, device="cuda"), torch.empty(ops.adam_grad_clip_ws_bytes(), dtype=torch.uint8, device="cuda")
    for max_norm in (0.25 * want, 4.0 * want + 1.0):
        ops.adam_grad_clip(p, g, seg_end, reg, max_norm, clip, ws, grad_scale=gs, touched=flags, touched_log2=log2)
        norm, coef = clip.tolist()
        c64 = min(1.0, max_norm / (want + 1e-6))
        assert abs(norm - want) <= 2.0 ** -22 * want and abs(coef - c64) <= 2.0 ** -22 * c64
        P, G, M, V = p.clone(), g.clone(), m.clone(), v.clone()
        sq = torch.zeros(len(sizes), device="cuda")
        ops.adam_fused(P, G, M, V, seg_end, reg, 0.7, 3, grad_scale=gs, sumsq_out=sq, touched=flags, touched_log2=log2, clip=clip)
        gr = tot * c64
        m64 = m.double() + (gr - m.double()) * (1 - 0.9)
        v64 = v.double() * 0.999 + gr * gr * (1 - 0.999)
        step = (0.7 / (1 - 0.9 ** 3)) * m64 / (v64.sqrt() / math.sqrt(1 - 0.999 ** 3) + 1e-8)
        p64 = (p.double() - step).clamp(ops.CLAMP_LO, ops.CLAMP_HI)
        # (data term and regulariser may cancel: the gradient's rounding is relative to its terms)
        terms = (0.5 * g.double().abs() + max(reg) * p.double().abs()) * c64
        assert ((M.double() - m64).abs() <= 2.0 ** -21 * (m.double().abs() + terms) + 1e-44).all()
        assert ((V.double() - v64).abs() <= 2.0 ** -20 * (v.double().abs() + terms * terms) + 1e-44).all()
        assert not G.any()
        ok = gr.abs() > 1e-3 * terms        # (elsewhere the sign of a cancelled gradient decides)
        err = (P.double() - p64).abs()
        assert (err <= 2.0 ** -12 * step.abs() + 2.0 ** -22 * p.double().abs() + 1e-9)[ok].all()
        if max_norm > want:      # nothing clipped: bit for bit the plain update
            Q, H, A, B = p.clone(), g.clone(), m.clone(), v.clone()
            sq2 = torch.zeros(len(sizes), device="cuda")
            ops.adam_fused(Q, H, A, B, seg_end, reg, 0.7, 3, grad_scale=gs, sumsq_out=sq2, touched=flags, touched_log2=log2)
            assert torch.equal(P, Q) and torch.equal(M, A) and torch.equal(V, B)


def test_norm_has_the_same_bits_every_time_and_bad_norms_follow_the_formula():
    require_gpu()
    from stylemesh_amd.runtime import ops
    sizes = [3 * 300 * 300, 77]
    seg_end = np.cumsum(sizes).tolist()
    p, g, _, _ = _state(sizes, 5)
    ws = torch.empty(ops.adam_grad_clip_ws_bytes(), dtype=torch.uint8, device="cuda")
    run = lambda: (lambda c: (ops.adam_grad_clip(p, g, seg_end, [0.1, 0.0], 1.0, c, ws), c)[1])(torch.zeros(2, device="cuda"))
    first = run()
    assert all(torch.equal(run(), first) for _ in range(4))
    g[7] = float("inf")
    assert run().tolist() == [math.inf, 0.0]
    g[8] = float("nan")
    assert torch.isnan(run()).all()
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.adam_grad_clip(p, g, seg_end, [0.1, 0.0], bad, torch.zeros(2, device="cuda"), ws)


@pytest.mark.parametrize("graphs", [False, True])
def test_engine_steps_clip_the_total_gradient(graphs):
    """Engine steps over two views: in every step the moments receive the clipped gradient of that very step."""
    views = [to_cuda(v) for v in small_views((3, 4))]
    eng = make_engine(FLAGSETS["with_angle_and_depth"], None)
    eng.use_graphs = graphs
    eng.gradient_clip_val = 0.5
    a = eng.arena
    for i in range(6):
        eng.step_compute(views[i // 3])
        assert eng._adam_early_done is None                # the split update would apply a part of the gradient unclipped
        g, p, m = a.g.clone(), a.p.clone(), a.m.clone()
        eng.optimizer_step()
        tot = _total64(p, g, a.seg_end, eng.reg_coef, 1.0)
        want = float(tot.norm())
        norm, coef = eng.grad_clip.tolist()
        assert abs(norm - want) <= 2.0 ** -22 * want and want > 0.5 and coef < 1
        applied = (a.m.double() - 0.9 * m.double()) / 0.1   # m' = 0.9 m + 0.1 g
        assert abs(float(applied.norm()) - 0.5) <= 1e-4
        assert not a.g.any()


def test_clipping_switches_the_overlapped_updates_off():
    eng = make_engine(FLAGSETS["with_angle_and_depth"], None)

    class Reducer:
        owner_aware, ready, n_idx, chunk, chunk_log2 = True, True, 10 ** 9, 64, 6

        def pipelined(self, *a):
            raise AssertionError("not to be called")
    eng.pipeline_exchange = eng.deferred_exchange = True
    assert eng.use_pipelined_exchange(Reducer()) and eng.use_deferred_exchange(Reducer())
    eng.gradient_clip_val = 1.0
    assert not eng.use_pipelined_exchange(Reducer()) and not eng.use_deferred_exchange(Reducer())


def test_trainer_flag_reaches_the_update():
    from stylemesh_amd.trainer import JsonlLogger, MiniTrainer
    m = make_model(FLAGSETS["with_angle_and_depth"])

    class DM:
        def train_dataloader(self):
            return iter(small_views((3, 3, 4)))
    with tempfile.TemporaryDirectory() as tmp:
        tr = MiniTrainer(max_epochs=1, logger=JsonlLogger(tmp), progress=False, gradient_clip_val=0.25)
        tr.fit(m, DM())
    eng = m._engine
    norm, coef = eng.grad_clip.tolist()
    assert tr.global_step == 3 and eng.step_count == 3 and norm > 0.25 and abs(coef - 0.25 / (norm + 1e-6)) <= 2.0 ** -20 * coef
    # three steps of gradients of norm 0.25 from zero moments
    assert float(eng.arena.m.norm()) <= (1 - 0.9 ** 3) * 0.25 * (1 + 1e-5)


def test_trainer_clips_any_modules_gradients():
    require_gpu()
    from stylemesh_amd.trainer import JsonlLogger, MiniTrainer

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.lin = torch.nn.Linear(4, 3)
            self.unused = torch.nn.Parameter(torch.zeros(2))
            self.seen = []

        def training_step(self, batch, i):
            return {"loss": (self.lin(batch[0]) ** 2).sum() * 100}

        def configure_optimizers(self):
            opt = torch.optim.SGD(self.parameters(), lr=1e-3)
            step = opt.step

            def noting(*a, **k):
                self.seen.append(math.sqrt(sum(float(q.grad.double().square().sum()) for q in self.parameters() if q.grad is not None)))
                return step(*a, **k)
            opt.step = noting
            return [opt], []

    class DM:
        def train_dataloader(self):
            g = torch.Generator().manual_seed(2)
            return iter([(torch.randn(8, 4, generator=g),) for _ in range(3)])
    net = Net()
    with tempfile.TemporaryDirectory() as tmp:
        MiniTrainer(max_epochs=1, logger=JsonlLogger(tmp), progress=False, gradient_clip_val=0.5, device=torch.device("cuda", 0)).fit(net, DM())
    assert len(net.seen) == 3 and all(abs(s - 0.5) <= 1e-5 for s in net.seen)


def test_refused_values():
    from stylemesh_amd.runtime.engine import EngineConfig
    from stylemesh_amd.trainer import MiniTrainer
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            EngineConfig(gradient_clip_val=bad).validate()
        with pytest.raises(ValueError):
            MiniTrainer(gradient_clip_val=bad, logger=object())
    assert MiniTrainer(gradient_clip_val=None, logger=object()).gradient_clip_val == 0.0


def test_trainer_clips_double_gradients_on_the_device():
    """A type that the device operators refuse."""
    require_gpu()
    from stylemesh_amd.trainer import _clip_gradients
    g = torch.Generator().manual_seed(4)
    params = [torch.nn.Parameter(torch.zeros(3, 5, dtype=torch.float64, device="cuda")), torch.nn.Parameter(torch.zeros(7, device="cuda")),
              torch.nn.Parameter(torch.zeros(2, device="cuda"))]
    for q in params[:2]:
        q.grad = torch.randn(q.shape, generator=g).to(q) * 10
    want = [q.grad.double().clone() for q in params[:2]]
    norm = math.sqrt(sum(float(w.square().sum()) for w in want))
    _clip_gradients(params, 0.5)
    for q, w in zip(params, want):
        assert ((q.grad.double() - w * (0.5 / (norm + 1e-6))).abs() <= 2.0 ** -20 * w.abs()).all()


def test_clipping_is_not_switched_inside_a_step():
    """Small steps are replayed as a program whose update does not clip: switched on between the two halves of such a step,
    the gradient would silently be applied unclipped."""
    eng = make_engine(FLAGSETS["with_angle_and_depth"], None)
    view = to_cuda(small_views((3,))[0])
    for _ in range(6):
        eng.step_compute(view)
        eng.optimizer_step()
    for first, then in ((0.0, 0.5), (0.5, 0.0)):
        eng.gradient_clip_val = first
        eng.step_compute(view)
        eng.gradient_clip_val = then
        count = eng.step_count
        with pytest.raises(RuntimeError, match="gradient_clip_val"):
            eng.optimizer_step()
        assert eng.step_count == count
        eng.gradient_clip_val = first
        eng.optimizer_step()
    # a value may change, and a new step takes whatever holds at its start
    eng.gradient_clip_val = 0.5
    eng.step_compute(view)
    eng.gradient_clip_val = 0.25
    eng.optimizer_step()
    norm, coef = eng.grad_clip.tolist()
    assert norm > 0.5 and abs(coef - 0.25 / (norm + 1e-6)) <= 2.0 ** -20 * coef
    eng.gradient_clip_val = 0.0
    eng.step_compute(view)
    eng.optimizer_step()


@pytest.mark.parametrize("exchange", ["plain", "pipelined", "owner_aware"])
def test_two_ranks_clip_by_the_same_norm(exchange):
    """Two ranks over gloo on one device (they take turns on it), an epoch of the trainer with ``gradient_clip_val``: the norm
    is the mean gradient's - data terms of both ranks and regulariser - on both, bit for bit, whatever exchange is asked for, and
    the textures end identical."""
    require_gpu()
    import os
    from test_round2_gpu import REPO, _launch_ranks
    env = {"STYLEMESH_TEST_BACKEND": "gloo", "STYLEMESH_TEST_CLIP": "0.25"}
    env.update({"plain": {}, "pipelined": {"STYLEMESH_PIPELINE_EXCHANGE": "1"}, "owner_aware": {"STYLEMESH_DEFERRED_EXCHANGE": "1"}}[exchange])
    with tempfile.TemporaryDirectory() as tmp:
        r = _launch_ranks([os.path.join(REPO, "tests", "two_rank_clip_worker.py"), "trainer", tmp], 2, env, timeout=100)
        assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
        r0, r1 = (torch.load(os.path.join(tmp, f"rank{k}.pt")) for k in (0, 1))
        c0, c1 = (torch.load(os.path.join(tmp, f"clip{k}.pt")) for k in (0, 1))
    assert r0["steps"] == r1["steps"] == 6 and not r0["deferred"] and c0["clip"].shape == (6, 2)
    assert torch.equal(c0["clip"], c1["clip"])
    for a, b in zip(r0["layers"], r1["layers"]):
        assert torch.equal(a, b) and float(a.abs().max()) > 0
    norm, coef, want, applied = c0["clip"][:, 0].double(), c0["clip"][:, 1].double(), c0["want"], c0["applied"]
    assert ((norm - want).abs() <= 2.0 ** -22 * want).all() and (want > 0.25).all()
    assert ((coef - 0.25 / (want + 1e-6)).abs() <= 2.0 ** -20 * coef).all()
    assert ((applied - 0.25).abs() <= 1e-4).all()
