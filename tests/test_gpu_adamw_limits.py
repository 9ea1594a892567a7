"""Hyperparameters at their limits: what plain Adam takes, a clip does not refuse."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as A
from tests.test_gpu_adamw_train import _moments, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(max_grad_norm=1e6), dict(moment_bits=8)], ids=["plain", "clip", "8bit"])
def test_a_schedule_that_ends_at_zero(kw):
    """means_lr_end = 0: the first step has the initial rate, 0^(c / steps) = 0 from then on."""
    from gs_b200.training.trainer import train_step
    st, opt, cam, views = _state(**kw)
    opt.means_lr_end = 0.0
    m0 = st.gaussians.means.clone()
    train_step(st, *views[0], cam, opt, sh_degree=3)
    m1, s1 = st.gaussians.means.clone(), st.gaussians.scales.clone()
    assert not torch.equal(m0, m1)
    for view in views[1:3]:
        train_step(st, *view, cam, opt, sh_degree=3)
        assert torch.equal(st.gaussians.means, m1)
    assert not torch.equal(st.gaussians.scales, s1) and st.count == 3


def test_adamw_takes_a_decay_rate_of_zero():
    from gs_b200.training.optimizer import AdamW, ParamTensor
    for bits in (32, 8):
        p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
        opt = AdamW([ParamTensor(p, g, lr=0.5, lr_decay_rate=0.0, lr_transition_steps=1e6)], moment_bits=bits)
        opt.step()
        after = p.clone()
        # g / (|g| + 1e-8) = 1 to the roundings of the update's factors (56 of 2^-24, tests/adamw_ref.py)
        np.testing.assert_allclose(after.cpu().numpy(), 0.5, rtol=0, atol=0.5 * 57 * 2.0 ** -24)
        opt.step()
        assert torch.equal(p, after) and int(opt.count) == 2


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-38, 1e-60])
@pytest.mark.parametrize("bits", [32, 8])
def test_an_eps_below_the_smallest_normal_number(eps, bits):
    """It counts as that number: rows with a second moment move as with eps = 0 (|root| is at least 2^-74.5, far
    above), rows without one stay."""
    from gs_b200.training.trainer import train_step
    st, opt, cam, views = _state(max_grad_norm=1e6, moment_bits=bits)
    opt.eps = eps
    for c, view in enumerate(views[:2]):
        p0 = st.params.cpu().numpy()
        m0, v0 = _moments(st)
        train_step(st, *view, cam, opt, sh_degree=3)
        m, v = A.moments(m0, v0, st.grads[:st.size].cpu().numpy(), st._adamw[1].norm.scale.cpu().numpy(), opt.b1, opt.b2)
        p1 = st.params.cpu().numpy()
        assert np.isfinite(p1).all()
        lrs = opt.lrs(c)
        rows = st.active_mask.cpu().numpy()
        for i, (a, b) in enumerate(st.segments):
            s = slice(a, b)
            act = np.repeat(rows, (b - a) // st.n)
            seen = v[s] > 0
            want, err = A.param(p0[s], m[s], v[s], c, lrs[i], 0.0, opt.b1, opt.b2, 0.0, act)
            assert (np.abs(p1[s] - want) <= err)[seen].all(), i
            still = (v[s] == 0) & (m[s] == 0)
            assert still.any() and (p1[s][still] == p0[s][still]).all()
