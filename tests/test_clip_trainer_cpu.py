"""``MiniTrainer(gradient_clip_val=)`` on modules whose gradients the device operators do not take: on the host, in float64."""
import math
import tempfile

import pytest
import torch

from stylemesh_amd.trainer import JsonlLogger, MiniTrainer


class Net(torch.nn.Module):
    def __init__(self, dtype):
        super().__init__()
        self.emb = torch.nn.Embedding(5, 4, dtype=dtype)
        self.lin = torch.nn.Linear(4, 3, dtype=dtype)
        self.unused = torch.nn.Parameter(torch.zeros(2, dtype=dtype))
        self.seen = []

    def training_step(self, batch, i):
        return {"loss": (self.lin(self.emb(batch[0])) ** 2).sum() * 100}

    def configure_optimizers(self):
        opt = torch.optim.SGD(self.parameters(), lr=1e-3)
        step = opt.step
        norm = lambda: math.sqrt(sum(float(q.grad.double().square().sum()) for q in self.parameters() if q.grad is not None))

        def noting(*a, **k):
            self.seen.append(norm())
            return step(*a, **k)
        opt.step = noting
        return [opt], []


class DM:
    def train_dataloader(self):
        return iter([(torch.tensor([0, 1, i, 4]),) for i in range(3)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_host_modules_are_clipped(dtype):
    torch.manual_seed(0)
    net = Net(dtype)
    before = [q.detach().clone() for q in net.parameters()]
    with tempfile.TemporaryDirectory() as tmp:
        tr = MiniTrainer(max_epochs=1, logger=JsonlLogger(tmp), progress=False, gradient_clip_val=0.5, device="cpu")
        tr.fit(net, DM())
    # each gradient: the coefficient's rounding, the product's, of values in the parameters' type
    tol = 4 * torch.finfo(dtype).eps
    assert tr.global_step == 3 and len(net.seen) == 3 and all(abs(s - 0.5) <= 0.5 * tol + 1e-6 for s in net.seen)
    moved = math.sqrt(sum(float((a.detach() - b).double().square().sum()) for a, b in zip(net.parameters(), before)))
    assert 0 < moved <= 3 * 0.5 * 1e-3 * 1.01 or dtype == torch.bfloat16


def test_a_small_gradient_is_left_alone():
    torch.manual_seed(0)
    net = Net(torch.float64)
    with tempfile.TemporaryDirectory() as tmp:
        MiniTrainer(max_epochs=1, logger=JsonlLogger(tmp), progress=False, gradient_clip_val=1e9, device="cpu").fit(net, DM())
    torch.manual_seed(0)
    other = Net(torch.float64)
    with tempfile.TemporaryDirectory() as tmp:
        MiniTrainer(max_epochs=1, logger=JsonlLogger(tmp), progress=False, device="cpu").fit(other, DM())
    assert net.seen == other.seen and all(torch.equal(a, b) for a, b in zip(net.parameters(), other.parameters()))
