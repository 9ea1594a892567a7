"""AdamW, the gradient norm and the 8-bit moments without a GPU: refusals of
the C ABI and of the Python plans, and the format's restatement."""
import ctypes
import math

import numpy as np
import pytest
import torch

from gs_b200 import _lib
from tests import adamw_ref as R

E = _lib.GS_ERR_INVALID_ARGUMENT
P = 0x10000  # never dereferenced: the calls below are rejected first


def tensor(**kw):
    t = _lib.GsAdamwTensor()
    for k, v in dict(dict(param=P, grad=P, mu=P, nu=P, mu_exp=P, nu_exp=P, count=256, width=1, lr_init=1e-3,
                          decay_rate=1.0, transition_steps=1.0, weight_decay=0.0), **kw).items():
        setattr(t, k, v)
    return t


def config(**kw):
    c = _lib.GsAdamwConfig()
    for k, v in dict(dict(b1=0.9, b2=0.999, eps=1e-8, moment_bits=32, seed=1), **kw).items():
        setattr(c, k, v)
    return c


def step(t=None, c=None, n=1, state=P, tensors=True):
    arr = (_lib.GsAdamwTensor * 1)(t or tensor())
    return _lib.lib().gs_adamw_step(arr if tensors else None, n, ctypes.byref(c or config()), None, state, None)


BAD_TENSORS = [
    dict(count=-1), dict(count=(1 << 37) + 1), dict(param=None), dict(grad=None), dict(mu=None), dict(nu=None),
    dict(param=P + 2), dict(mu=P + 1), dict(nu=P + 2), dict(grad=P + 2), dict(grad=P + 1, grad_type=1),
    dict(grad_type=3), dict(grad_type=-1), dict(copy=P, copy_type=0), dict(copy=P, copy_type=3),
    dict(copy=P + 1, copy_type=1), dict(active=P, width=0), dict(active=P, width=3), dict(active=P, width=32769, count=32769),
    dict(lr_init=math.nan), dict(lr_init=math.inf), dict(weight_decay=math.nan), dict(decay_rate=0.0),
    dict(decay_rate=math.inf), dict(transition_steps=0.0), dict(transition_steps=math.nan),
]


@pytest.mark.parametrize("kw", BAD_TENSORS, ids=[str(k) for k in BAD_TENSORS])
def test_step_refuses_tensors(kw):
    assert step(tensor(**kw)) == E


@pytest.mark.parametrize("kw", [dict(moment_bits=16), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=math.nan),
                                dict(b2=1.0 - 1e-12), dict(eps=0.0), dict(eps=1e-60), dict(eps=1e-39), dict(eps=math.inf),
                                dict(eps=math.nan)])
def test_step_refuses_hyperparameters(kw):
    assert step(c=config(**kw)) == E


def test_step_refuses_the_rest():
    lib = _lib.lib()
    assert step(n=-1) == E
    assert step(tensors=False) == E
    assert step(state=None) == E
    assert lib.gs_adamw_step((_lib.GsAdamwTensor * 1)(tensor()), 1, None, None, P, None) == E
    eight = config(moment_bits=8)
    assert step(tensor(mu_exp=None), eight) == E
    assert step(tensor(nu_exp=None), eight) == E
    many = (_lib.GsAdamwTensor * 9)(*[tensor(count=1 << 37) for _ in range(9)])
    assert lib.gs_adamw_step(many, 9, ctypes.byref(config()), None, P, None) == _lib.GS_ERR_TOO_LARGE


def test_norm_refuses():
    lib = _lib.lib()

    def norm(n=1, max_norm=1.0, out=P, ws=P, nbytes=1 << 20, tensors=True, **kw):
        t = _lib.GsGradTensor()
        for k, v in dict(dict(grad=P, count=10, type=0), **kw).items():
            setattr(t, k, v)
        return lib.gs_grad_norm((_lib.GsGradTensor * 1)(t) if tensors else None, n, max_norm, None, out, ws, nbytes,
                                None)

    for kw in (dict(n=-1), dict(tensors=False), dict(out=None), dict(max_norm=0.0), dict(max_norm=-1.0),
               dict(max_norm=math.nan), dict(count=-1), dict(type=3), dict(grad=None), dict(grad=P + 2),
               dict(grad=P + 1, type=1), dict(ws=P + 4)):
        assert norm(**kw) == E, kw
    assert norm(ws=None) == _lib.GS_ERR_WORKSPACE_TOO_SMALL
    assert norm(nbytes=lib.gs_grad_norm_workspace_bytes(1) - 1) == _lib.GS_ERR_WORKSPACE_TOO_SMALL
    assert lib.gs_grad_norm_workspace_bytes(-1) == 0
    assert lib.gs_grad_norm_workspace_bytes(5000) > lib.gs_grad_norm_workspace_bytes(5)


def test_conversions_refuse():
    lib = _lib.lib()
    good = [P, P, P, P, 10, 0, P, P]
    for i, bad in ((0, None), (1, None), (2, None), (3, None), (4, -1), (5, 2), (5, -1), (6, None), (7, None),
                   (0, P + 1), (1, P + 2), (6, P + 2), (7, P + 1)):
        args = list(good)
        args[i] = bad
        assert lib.gs_moments8_decode(*args, None) == E, (i, bad)
    good = [P, P, 10, P, P, P, P]
    for i, bad in ((0, None), (1, None), (2, -1), (3, None), (4, None), (5, None), (6, None), (0, P + 2), (3, P + 1)):
        args = list(good)
        args[i] = bad
        assert lib.gs_moments8_encode(*args, None) == E, (i, bad)
    assert lib.gs_moments8_decode(None, None, None, None, 0, 0, None, None, None) == 0  # nothing to do
    assert lib.gs_moments8_encode(None, None, 0, None, None, None, None, None) == 0


def test_plans_refuse_host_tensors():
    from gs_b200.training.optimizer import AdamW, GradNorm, Moments8, ParamTensor
    t = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        AdamW([ParamTensor(t, t, lr=1e-3)])
    with pytest.raises(ValueError, match="CUDA"):
        GradNorm([t])
    with pytest.raises(ValueError, match="no tensors"):
        AdamW([])
    with pytest.raises(ValueError, match="no gradients"):
        GradNorm([])
    with pytest.raises(ValueError, match="CUDA"):
        Moments8([4], "cpu")
    with pytest.raises(ValueError, match="device"):
        Moments8([4])


def test_shared_memory_is_found():
    from gs_b200.training.optimizer import _check_overlap
    buf = torch.zeros(100)
    _check_overlap([("a", buf[:50]), ("b", buf[50:])], [])
    _check_overlap([("a", buf[:50])], [("c", buf[50:80]), ("d", buf[60:100])])  # reads may share
    with pytest.raises(ValueError, match="a"):
        _check_overlap([("a", buf[:51]), ("b", buf[50:])], [])
    with pytest.raises(ValueError, match="same"):
        _check_overlap([("same", buf), ("same", buf)], [])
    with pytest.raises(ValueError, match="g"):
        _check_overlap([("p", buf[10:20])], [("g", buf)])
    with pytest.raises(ValueError, match="g"):
        _check_overlap([("p", buf)], [("g", buf[10:20])])


@pytest.mark.parametrize("signed", [True, False])
def test_every_code_keeps_its_value(signed):
    """Decoding and encoding again is the identity, at any noise, whatever power of two the block has."""
    codes = np.arange(256, dtype=np.uint8)
    for field in (1, 60, 127, 200, 254):
        exps = np.full(2, field, np.uint8)
        val = R.decode(codes, exps, signed)
        x = val.astype(np.float32)
        with np.errstate(over="ignore"):
            ok = np.isfinite(x).all() and (x.astype(np.float64) == val).all()
        if not ok:
            continue  # out of float32's range at this exponent
        for u in (0.0, 0.5, 0.999):
            c, e = R.encode(x, np.full(256, u), signed)
            np.testing.assert_array_equal(R.decode(c, e, signed), val)


def test_trainer_refusals():
    """The fused data-parallel update is plain Adam; a state and an optimizer
    agree on the moments' bits; 8-bit moments live on a GPU."""
    from gs_b200.training import density, trainer
    st = trainer.DensityState(4, 1, "cpu")
    cam = (16, 16, 10.0, 10.0, 8.0, 8.0)
    for kw in (dict(weight_decay=(0.0, 0.1, 0.0, 0.0, 0.0)), dict(max_grad_norm=1.0)):
        opt = trainer.AdamConfig(**kw)
        assert not opt.is_adam
        with pytest.raises(ValueError, match="fused=False"):
            trainer._step(st, None, None, cam, opt, 0, object(), None)
    with pytest.raises(ValueError, match="bits"):
        trainer._step(st, None, None, cam, trainer.AdamConfig(moment_bits=8), 0, None, None)
    assert trainer.AdamConfig().is_adam and trainer.AdamConfig.from_extent(2.0, max_grad_norm=1.0).max_grad_norm == 1.0
    with pytest.raises(ValueError, match="CUDA"):
        trainer.DensityState(4, 1, "cpu", moment_bits=8)
    with pytest.raises(ValueError, match="moment_bits"):
        trainer.DensityState(4, 1, "cpu", moment_bits=16)
    with pytest.raises(ValueError, match="five"):
        st.adamw(trainer.AdamConfig(weight_decay=(0.1,)))
    assert [t.data_ptr() for t in st.moment_buffers()] == [st.mu.data_ptr(), st.nu.data_ptr()]
    st.moments8 = object()
    with pytest.raises(ValueError, match="8-bit"):
        density.gather_moments(st, None)
