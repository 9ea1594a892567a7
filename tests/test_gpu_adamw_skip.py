"""Training steps that the clip skips (a gradient that is not finite): the whole
state stays as it was, the densification statistics too."""
import numpy as np
import pytest
import torch

from tests.test_gpu_adamw_train import _state

pytestmark = pytest.mark.gpu


def _bad(view):
    target = view[0].clone()
    target[10:30, 10:30] = float("nan")
    return target, view[1]


def _stats(st):
    return [t.clone() for t in (st.grad_accum, st.denom, st.max_radii)]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_skipped_step_leaves_the_statistics(bits, captured):
    from gs_b200.training.trainer import CapturedStep, train_step
    st, opt, cam, views = _state(max_grad_norm=1.0, moment_bits=bits)
    if captured:
        step = CapturedStep(st, *views[0], cam, opt, sh_degree=3)
    else:
        step = lambda *view: train_step(st, *view, cam, opt, sh_degree=3)  # noqa: E731
        step(*views[0])
    before = _stats(st)
    assert float(before[0].abs().max()) > 0 and int(before[1].max()) == 1
    step(*_bad(views[1]))
    assert int(st.skipped) == 1
    for a, b in zip(before, _stats(st)):
        assert torch.equal(a, b)
    step(*views[2])
    assert int(st.denom.max()) == 2 and torch.isfinite(st.grad_accum).all()


def test_statistics_are_those_of_the_steps_taken():
    """A run with a skipped step in it ends with the statistics of the run without."""
    from gs_b200.training.trainer import train_step
    runs = []
    for bad in (False, True):
        st, opt, cam, views = _state(max_grad_norm=1.0)
        train_step(st, *views[0], cam, opt, sh_degree=3)
        p0 = st.params.clone()
        if bad:
            train_step(st, *_bad(views[1]), cam, opt, sh_degree=3)
            assert torch.equal(st.params, p0)
        runs.append(_stats(st))
    assert torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])
    # grad_accum: one step's gradients, whose atomics change order between runs (the gradients' own bar)
    a, b = (r[0].cpu().numpy() for r in runs)
    assert (np.abs(a - b) <= 1e-3 * (np.abs(a) + np.abs(a).max())).all()


def test_without_a_clip_nothing_is_skipped():
    """Weight decay alone skips nothing: the statistics take the gradient as it is, as plain Adam's do."""
    from gs_b200.training.trainer import train_step
    for kw in (dict(weight_decay=(0.0, 0.01, 0.0, 0.0, 0.0)), dict()):
        st, opt, cam, views = _state(**kw)
        train_step(st, *_bad(views[1]), cam, opt, sh_degree=3)
        assert not torch.isfinite(st.grad_accum).all() and int(st.denom.max()) == 1
        assert st.count == int(st.adam_state[0]) == 1


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 0.5, None])
@pytest.mark.parametrize("n", [1, 257, 1000])
def test_gated_statistics(n, bad):
    """The gated entries are the plain ones while the gate is finite or absent, and change nothing else."""
    from gs_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(n)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    gm, means, w2c = rand(n, 3), rand(n, 3), torch.eye(4, device="cuda")
    radii, valid, active = rand(n).abs() * 20, (rand(n) > 0).to(torch.uint8), (rand(n) > -0.5).to(torch.uint8)
    g2d = rand(n).abs()
    gate = None if bad is None else torch.tensor(bad, device="cuda")
    closed = bad is not None and not np.isfinite(bad)
    P, st = _lib.ptr, _lib.stream(gm.device)
    start = (rand(n).abs(), torch.arange(n, dtype=torch.int32, device="cuda"), rand(n).abs())
    view = (P(gm), P(means), P(w2c), n, 400.0, 410.0, 64, 48, P(radii), P(valid), P(active))
    pair = (P(g2d), P(radii), P(valid), None, P(active), n)
    for plain, gated, args in (("gs_density_step_stats", "gs_density_step_stats_gated", view),
                               ("gs_accumulate_density_stats", "gs_accumulate_density_stats_gated", pair)):
        one, two = [t.clone() for t in start], [t.clone() for t in start]
        tail = (None,) if plain == "gs_density_step_stats" else ()
        _lib.call(plain, *args, *(P(t) for t in one), *tail, st)
        _lib.call(gated, *args, P(gate), *(P(t) for t in two), *tail, st)
        for a, b, s in zip(one, two, start):
            assert torch.equal(b, s if closed else a)
