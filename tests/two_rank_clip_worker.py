"""``two_rank_worker.py`` with gradient clipping (STYLEMESH_TEST_CLIP): every step's norm and coefficient, the total gradient's norm
in 64 bits and that of the gradient the moments received go to ``clip<rank>.pt``."""
import functools
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import two_rank_worker  # noqa: E402  (puts the repository on the path)
from stylemesh_amd import trainer  # noqa: E402
from stylemesh_amd.runtime.engine import StepEngine  # noqa: E402


def main():
    rank, out_dir = int(os.environ["RANK"]), sys.argv[2]
    trainer.MiniTrainer = functools.partial(trainer.MiniTrainer, gradient_clip_val=float(os.environ["STYLEMESH_TEST_CLIP"]))
    rec = {"clip": [], "want": [], "applied": []}
    plain = StepEngine.optimizer_step

    def noting(eng, world_size=1):
        a = eng.arena
        total, b = torch.empty(a.p.numel(), dtype=torch.float64, device=a.p.device), 0
        for e, c in zip(a.seg_end, eng.reg_coef):
            total[b:e] = a.g[b:e].double() / world_size + c * a.p[b:e].double()
            b = e
        m = a.m.double()
        plain(eng, world_size)
        rec["clip"].append(eng.grad_clip.cpu())
        rec["want"].append(total.norm().cpu())
        rec["applied"].append(((a.m.double() - 0.9 * m) / 0.1).norm().cpu())
    StepEngine.optimizer_step = noting
    two_rank_worker.main()
    torch.save({k: torch.stack(v) for k, v in rec.items()}, os.path.join(out_dir, f"clip{rank}.pt"))


if __name__ == "__main__":
    main()
