"""fused_clip_grad_norm_ over a group: each rank holds a part of the gradients, and all clip by the norm of the whole.

Gradients go tensor by tensor on the CPU; `--listed RANKS` gives these ranks a stand-in for the kernels' list, so that the branch around
it runs, also beside ranks that go tensor by tensor.
"""
import argparse
import math
import sys
from pathlib import Path

import torch
import torch.distributed as dist

sys.path.insert(0, str(Path(__file__).resolve().parents[2]))
from trainscale_b200.parallel import dist_utils  # noqa: E402


class Listed:
    """What ops.optim.GradList does, in fp64."""

    def __init__(self, grads):
        self.grads = grads

    @staticmethod
    def of(grads, norm_type):
        return Listed(grads)

    def norm(self, norm_type):
        return torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in self.grads]), norm_type).float()

    def clip_(self, norm, max_norm):
        for g in self.grads:
            g.mul_((max_norm / (norm + 1e-6)).clamp(max=1.0))


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--listed", default="")
    listed = [int(r) for r in p.parse_args().listed.split(",") if r]
    dist.init_process_group("gloo")
    rank, world = dist.get_rank(), dist.get_world_size()
    if rank in listed:
        dist_utils.GradList = Listed
    scales = [1.0] + ([1e25, 1e-25] if len(listed) == world else [])         # (tensor by tensor, squares are fp32 as ever)
    for scale in scales:
        for kind in (2.0, 1.0, math.inf):
            every = [[torch.randn(5, 7, generator=torch.Generator().manual_seed(10 * r + i)) * scale for i in range(2)] for r in range(world)]
            whole = torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for part in every for g in part]), kind)
            ps = [torch.nn.Parameter(torch.zeros(5, 7)) for _ in range(2)]
            for q, g in zip(ps, every[rank]):
                q.grad = g.clone()
            limit = float(whole) / 4
            norm = dist_utils.fused_clip_grad_norm_(ps, limit, group=dist.group.WORLD, norm_type=kind)
            assert norm.dtype == torch.float32 and abs(float(norm) / float(whole) - 1) < 1e-5, (scale, kind, float(norm), float(whole))
            factor = min(1.0, limit / (float(whole) + 1e-6))
            for q, g in zip(ps, every[rank]):
                torch.testing.assert_close(q.grad, g * factor, rtol=1e-5, atol=1e-37)
    dist.destroy_process_group()
    print("ok=True")


main()
