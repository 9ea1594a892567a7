"""The trainer's steps with weight decay, gradient clipping and 8-bit moments
(gs_adamw_step in place of the plain Adam), against the restatement of the
update on the gradients the step itself computed."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as A
from tests.helpers import random_scene, to_torch

pytestmark = pytest.mark.gpu

WD = (0.0, 0.01, 0.0, 0.05, 0.02)


def _state(n=1300, active=900, seed=3, **kw):
    from gs_b200.core.gaussians import Gaussians
    from gs_b200.training.trainer import AdamConfig, init_density_state
    sc = random_scene(seed, n, 96, 80, sh_degree=3, behind=0.05)
    t = to_torch(sc, "cuda")
    g = Gaussians(means=t["means"][:active], scales=t["scales"][:active], quaternions=t["quats"][:active],
                  opacities=t["opac"][:active], sh_coeffs=t["sh"][:active])
    opt = AdamConfig.from_extent(3.0, 100, **kw)
    st = init_density_state(g, opt, n)
    cam = (sc["W"], sc["H"], sc["fx"], sc["fy"], sc["cx"], sc["cy"])
    rng = np.random.default_rng(seed)
    views = [(torch.tensor(rng.uniform(0, 1, (80, 96, 3)).astype(np.float32), device="cuda"),
              torch.tensor(sc["w2c"], device="cuda")) for _ in range(4)]
    return st, opt, cam, views


def _moments(st):
    if st.moments8 is None:
        return [x.cpu().numpy() for x in (st.mu, st.nu)]
    return [torch.cat(st.moments8.split(x)).cpu().numpy() for x in st.moments8.values()]


@pytest.mark.parametrize("kw", [dict(weight_decay=WD), dict(max_grad_norm=1e-4), dict(moment_bits=8, moment_seed=5),
                                dict(weight_decay=WD, max_grad_norm=1e-4, moment_bits=8)],
                         ids=["decay", "clip", "8bit", "all"])
@pytest.mark.parametrize("n", [1300, 1301])
def test_train_step_updates_as_restated(kw, n):
    from gs_b200.training.trainer import train_step
    st, opt, cam, views = _state(n, **kw)
    act = st.active_mask.cpu().numpy()
    for c, (target, w2c) in enumerate(views[:3]):
        p0 = st.params.cpu().numpy()
        m0, v0 = _moments(st)
        train_step(st, target, w2c, cam, opt, sh_degree=3)
        p1 = st.params.cpu().numpy()
        m1, v1 = _moments(st)
        grads = st.grads[:st.size].cpu().numpy()
        scale = np.float32(1.0)
        if opt.max_grad_norm is not None:
            norm, want_scale = A.grad_norm([grads], opt.max_grad_norm)
            got = st._adamw[1].norm.out.cpu().numpy()
            np.testing.assert_allclose(got, [norm, want_scale], rtol=2.0 ** -23)
            assert want_scale < 1.0  # the clip is at work
            scale = got[1]
        m, v = A.moments(m0, v0, grads, scale, opt.b1, opt.b2)
        lrs = opt.lrs(c)
        for i, (a, b) in enumerate(st.segments):
            s = slice(a, b)
            rows = np.repeat(act, (b - a) // st.n)
            want, err = A.param(p0[s], m[s], v[s], c, lrs[i], opt.weight_decay[i], opt.b1, opt.b2, opt.eps, rows)
            assert (np.abs(p1[s] - want) <= err).all(), i
            if opt.moment_bits == 8:
                h = A.noise(opt.moment_seed, c, i, b - a)
                for got, x, u, signed in ((m1[s], m[s], h % 65536, True), (v1[s], v[s], h // 65536, False)):
                    np.testing.assert_array_equal(got, A.decode(*A.encode(x, u / 65536.0, signed), signed))
        if opt.moment_bits == 32:
            np.testing.assert_array_equal(m1, m)
            np.testing.assert_array_equal(v1, v)
        assert int(st.adam_state[0]) == st.count == c + 1


def test_changed_rates_are_taken_over():
    from gs_b200.training.trainer import train_step
    st, opt, cam, views = _state(weight_decay=WD)
    train_step(st, *views[0], cam, opt, sh_degree=3)
    plan = st._adamw[1]
    opt.opacities_lr = 0.0
    opt.weight_decay = (0.0, 0.0, 0.0, 0.5, 0.0)
    before = st.gaussians.opacities.clone()
    means = st.gaussians.means.clone()
    train_step(st, *views[1], cam, opt, sh_degree=3)
    assert st._adamw[1] is plan
    assert torch.equal(st.gaussians.opacities, before) and not torch.equal(st.gaussians.means, means)
    opt.b2 = 0.99
    train_step(st, *views[1], cam, opt, sh_degree=3)
    assert st._adamw[1] is not plan and int(st.adam_state[0]) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_not_finite_skips_the_step(bits):
    from gs_b200.training.trainer import train_step
    st, opt, cam, views = _state(max_grad_norm=1.0, moment_bits=bits)
    train_step(st, *views[0], cam, opt, sh_degree=3)
    p0, mom = st.params.clone(), [t.clone() for t in st.moment_buffers()]
    bad = views[1][0].clone()
    bad[10:30, 10:30] = float("nan")
    train_step(st, bad, views[1][1], cam, opt, sh_degree=3)
    assert not torch.isfinite(st.grads[:st.size]).all()
    assert torch.equal(st.params, p0)
    assert all(torch.equal(a, b) for a, b in zip(mom, st.moment_buffers()))
    assert int(st.skipped) == 1 and int(st.adam_state[0]) == 1
    train_step(st, *views[2], cam, opt, sh_degree=3)
    assert int(st.skipped) == 1 and int(st.adam_state[0]) == 2 and not torch.equal(st.params, p0)
    assert torch.isfinite(st.params).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Each replay is the restated update of the gradients it computed."""
    from gs_b200.training.trainer import CapturedStep
    st, opt, cam, views = _state(weight_decay=WD, max_grad_norm=1e-4, moment_bits=bits)
    step = CapturedStep(st, *views[0], cam, opt, sh_degree=3)
    assert int(st.adam_state[0]) == 1
    for c, view in enumerate(views[1:], 1):
        p0 = st.params.cpu().numpy()
        m0, v0 = _moments(st)
        step(*view)
        grads = st.grads[:st.size].cpu().numpy()
        scale = st._adamw[1].norm.scale.cpu().numpy()
        m, v = A.moments(m0, v0, grads, scale, opt.b1, opt.b2)
        a, b = st.segments[4]
        rows = np.repeat(st.active_mask.cpu().numpy(), (b - a) // st.n)
        want, err = A.param(p0[a:b], m[a:b], v[a:b], c, opt.sh_lr, WD[4], opt.b1, opt.b2, opt.eps, rows)
        assert (np.abs(st.params.cpu().numpy()[a:b] - want) <= err).all()
        assert int(st.adam_state[0]) == st.count == c + 1


def test_density_control_moves_8bit_moments():
    """densify_and_prune on a state with 8-bit moments: everything as on the
    same state with the values in 32 bits, the moments rounded to nearest."""
    from gs_b200.training.density import densify_and_prune
    from gs_b200.training.trainer import DensityState, train_step
    st, opt, cam, views = _state(moment_bits=8)
    for target, w2c in views:
        train_step(st, target, w2c, cam, opt, sh_degree=3)
    ref = DensityState(st.n, st.sh_k, "cuda")
    ref.params.copy_(st.params)
    for buf, x in zip((ref.mu, ref.nu), _moments(st)):
        buf.copy_(torch.tensor(x))
    for name in ("active_mask", "grad_accum", "denom", "max_radii"):
        getattr(ref, name).copy_(getattr(st, name))
    noise = torch.randn((st.n, 3), device="cuda")
    thr = float(torch.quantile(st.grad_accum / st.denom.clamp(min=1), 0.8))
    for s in (st, ref):
        densify_and_prune(s, grad_threshold=thr, noise=noise)
    assert int(st.densify_info[1] + st.densify_info[2]) > 0
    assert torch.equal(st.densify_info, ref.densify_info)
    for name in ("params", "active_mask", "grad_accum", "denom", "max_radii"):
        assert torch.equal(getattr(st, name), getattr(ref, name)), name
    got = _moments(st)
    for x, want, signed in ((got[0], ref.mu.cpu().numpy(), True), (got[1], ref.nu.cpu().numpy(), False)):
        for a, b in st.segments:
            w = want[a:b]
            np.testing.assert_array_equal(x[a:b], A.decode(*A.encode(w, np.full(b - a, 0.5), signed), signed))
    train_step(st, *views[0], cam, opt, sh_degree=3)  # and goes on
    assert torch.isfinite(st.params).all()


def test_memory_of_8bit_moments():
    from gs_b200.training.trainer import DensityState
    a, b = DensityState(1000, 16, "cuda"), DensityState(1000, 16, "cuda", moment_bits=8)
    size = lambda s: sum(t.numel() * t.element_size() for t in s.moment_buffers())  # noqa: E731
    assert size(b) < 0.27 * size(a) and b.mu is None and b.nu is None
