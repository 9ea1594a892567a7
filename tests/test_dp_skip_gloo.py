"""The data-parallel step with a clip (fused=False) on two CPU ranks over gloo:
the norm is the averaged gradient's, so a gradient that is not finite on one
rank makes every rank skip the step, statistics included, and the ranks stay
alike. Only the host logic runs: the library's calls are restated in torch."""
import datetime
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_dp_gloo import _free_port

N, K, STEPS = 20, 1, 4
BAD_STEP = 1  # rank 1's gradient has a NaN


class _Plan:
    """AdamW's two halves as far as the trainer calls them: clip by the norm, skip, a step of plain descent."""

    def __init__(self, st):
        self.st, self.grad_scale = st, torch.ones(())

    def clip(self):
        norm = self.st.grads[:self.st.size].double().square().sum().sqrt()
        scale = torch.where(norm < 1.0, 1.0, 1.0 / norm)
        self.grad_scale = torch.where(torch.isfinite(norm), scale, float("nan")).float()
        return self.grad_scale

    def update(self):
        if torch.isfinite(self.grad_scale):
            self.st.params -= 0.1 * self.grad_scale * self.st.grads[:self.st.size]
            self.st.adam_state[0] += 1
        else:
            self.st.adam_state[2] += 1


def _calls(st, rank, step):
    """Fakes of the library's calls; pointers are the tensors themselves."""
    gen = torch.Generator().manual_seed(10 * step + rank)

    def forward(*a):
        image, radii, valid, extras = a[-5:-1]
        image.zero_()
        extras.zero_()
        radii.copy_(torch.randint(1, 50, (N,), generator=gen).float())
        valid.copy_((torch.rand(N, generator=gen) < 0.7).to(torch.uint8))

    def backward(*a):
        g = torch.randn(st.size, generator=gen)
        if step == BAD_STEP and rank == 1:
            g[5] = float("nan")
        st.grads[:st.size] = g

    def grad2d(gmeans, means, *a):
        a[-2].copy_(gmeans.norm(dim=1) * means[:, 2].abs().clamp(min=0.01))

    def stats(g2d, radii, valid, radii_valid, mask, n, gate, accum, denom, max_radii, stream):
        if not torch.isfinite(gate):
            return
        accum += g2d
        denom += ((valid > 0) & (mask > 0)).int()
        torch.where(radii_valid > 0, torch.maximum(max_radii, radii), max_radii, out=max_radii)

    return {"gs_render_forward": forward, "gs_render_backward": backward, "gs_grad2d_magnitude": grad2d,
            "gs_accumulate_density_stats_gated": stats, "gs_l1_dssim_loss": lambda *a: None}


def _worker(rank, world, port, out):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path[:0] = [os.path.join(root, "jax-gs_b200"), root]
    from gs_b200 import _lib
    from gs_b200.training import trainer
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    st = trainer.DensityState(N, K, "cpu")
    st.params.copy_(torch.randn(st.size, generator=torch.Generator().manual_seed(1)))
    st.active_mask[:15] = True
    plan = _Plan(st)
    trainer.DensityState.adamw = lambda self, opt: plan
    trainer.workspace = lambda *a: torch.empty(0, dtype=torch.uint8)
    _lib.ptr, _lib.stream = (lambda t: t), (lambda d: 0)
    opt = trainer.AdamConfig(max_grad_norm=1.0)
    record = []
    for step in range(STEPS):
        fakes = _calls(st, rank, step)
        _lib.call = lambda fn, *a: fakes[fn](*a)
        trainer._step(st, torch.zeros(8, 8, 3), torch.eye(4), (8, 8, 10.0, 10.0, 4.0, 4.0), opt, 0,
                      dist.group.WORLD, 16, fused=False)
        record.append([t.clone() for t in (st.params, st.grad_accum, st.max_radii, st.denom, st.adam_state)])
    out[rank] = record
    dist.barrier()
    dist.destroy_process_group()


def test_a_gradient_that_is_not_finite_on_one_rank_skips_the_step_on_both():
    ctx = mp.get_context("spawn")
    out = ctx.Manager().dict()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=120)
    assert all(p.exitcode == 0 for p in procs)
    a, b = out[0], out[1]
    for step in range(STEPS):
        for x, y in zip(a[step][:3], b[step][:3]):  # parameters and shared statistics; denom is a rank's own
            assert torch.equal(x, y) and torch.isfinite(x).all(), step
    for run in (a, b):
        for x, y in zip(run[BAD_STEP][:4], run[BAD_STEP - 1][:4]):
            assert torch.equal(x, y)
        assert run[-1][4].tolist() == [STEPS - 1, 0, 1, 0]
        for step in (2, 3):
            assert not torch.equal(run[step][0], run[step - 1][0]) and run[step][3].sum() > run[step - 1][3].sum()
