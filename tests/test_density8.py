"""gs_densify_and_prune8 without a GPU: its workspace and what it refuses."""
import pytest

from gs_b200 import _lib

E = _lib.GS_ERR_INVALID_ARGUMENT
P = 0x10000  # never dereferenced: the calls below are rejected first
GOOD = dict(params=P, mu=P, nu=P, mu_exp=P, nu_exp=P, n=1000, sh_k=16, active=P, grad_accum=P, denom=P, max_radii=P,
            noise=P, enabled=1, threshold=0.1, min_opacity=0.1, extent=1.0, screen=512.0, ws=P, ws_bytes=1 << 30,
            info=P, stream=None)


def call(**kw):
    return _lib.lib().gs_densify_and_prune8(*dict(GOOD, **kw).values())


@pytest.mark.parametrize("kw", [dict(params=None), dict(mu=None), dict(nu=None), dict(mu_exp=None), dict(nu_exp=None),
                                dict(active=None), dict(grad_accum=None), dict(denom=None), dict(max_radii=None),
                                dict(noise=None), dict(info=None), dict(n=-1), dict(sh_k=0), dict(sh_k=17),
                                dict(n=1 << 30)], ids=str)
def test_refuses(kw):
    assert call(**kw) == E


def test_workspace():
    lib = _lib.lib()
    need = lib.gs_density8_workspace_bytes(1000, 16)
    codes = sum(-(-1000 * w // 128) * 128 for w in (3, 3, 4, 1, 48))
    assert need == lib.gs_density_workspace_bytes(1000) + codes + codes // 128
    for kw in (dict(ws=None), dict(ws=P + 128), dict(ws_bytes=need - 1)):
        assert call(**kw) == _lib.GS_ERR_WORKSPACE_TOO_SMALL
    assert lib.gs_density8_workspace_bytes(-1, 16) == 0 and lib.gs_density8_workspace_bytes(10, 17) == 0
