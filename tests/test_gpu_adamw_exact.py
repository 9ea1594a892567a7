"""The update's root and quotient are rounded to nearest: with 32-bit moments, and
with 8-bit ones in the kernel for few elements. The kernel for many elements with
8-bit moments takes approximations of 2^-23 each."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _step(n, bits, g, eps, lr, align=0, grad=torch.float32):
    """The parameter after one step from 0 with b1 = b2 = 0: m' = g, v' = g^2, no bias correction (1 - 0^t = 1)."""
    from gs_b200.training.optimizer import AdamW, ParamTensor
    p = torch.zeros(n + align, device="cuda")[align:]
    gt = torch.zeros(n + align, device="cuda", dtype=grad)[align:]
    gt.copy_(torch.tensor(g, device="cuda"))
    AdamW([ParamTensor(p, gt, lr=lr)], b1=0.0, b2=0.0, eps=eps, moment_bits=bits).step()
    return p.cpu().numpy(), gt.float().cpu().numpy()


def _gradient(n, low, high, seed):
    rng = np.random.default_rng(seed)
    return (rng.choice([-1.0, 1.0], n) * 10.0 ** rng.uniform(low, high, n)).astype(np.float32)


@pytest.mark.parametrize("bits,n,align", [(32, 5000, 0), (32, 5000, 1), (32, 900_000, 0), (32, 900_000, 1),
                                          (8, 5000, 0), (8, 5000, 1)])
@pytest.mark.parametrize("eps", [1e-20, 1e-30, 1.2e-38])
def test_a_root_that_is_exact(bits, n, align, eps):
    """sqrt(g g) rounded to nearest is |g| whatever the product's rounding (no over- or underflow), and an eps far
    below its last place adds nothing: with lr a power of two the update is exactly -+ lr."""
    g = _gradient(n, -6, 3, n)
    p, _ = _step(n, bits, g, eps, 2.0 ** -7, align)
    np.testing.assert_array_equal(p, -np.sign(g) * np.float32(2.0 ** -7))


@pytest.mark.parametrize("bits,n,align", [(32, 5000, 0), (32, 900_000, 0), (32, 900_000, 1), (8, 5000, 0)])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eps", [1e-3, 1e-11])
def test_sum_and_quotient(bits, n, align, grad, eps):
    """p' = -lr g / (|g| + eps): the root is exact (above), the sum and the quotient are rounded once each and lr is
    a power of two: two roundings of 2^-24, and 2^-44 for their product (2^-48) and what a Newton step on a
    reciprocal that is off by 2^-23 leaves (2^-46). The root stays exact with a Newton step too: the product's
    rounding moves it by at most 0.71 of half a unit in |g|'s last place. (eps 1e-11 is above 2^-39, below which
    other instructions serve.)"""
    g = _gradient(n, -5, 0, n + 1) * np.float32(eps / 1e-3)
    p, g = _step(n, bits, g, eps, 2.0 ** -7, align, grad)
    g = g.astype(np.float64)
    want = -2.0 ** -7 * g / (np.abs(g) + np.float64(np.float32(eps)))
    off = np.abs(p - want) > np.abs(want) * (2 * U + 2.0 ** -44)
    assert not off.any(), (int(off.sum()), np.flatnonzero(off)[:5])


@pytest.mark.parametrize("align", [0, 1])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eps", [1e-3, 1e-8, 1e-30])
def test_many_elements_with_8bit_moments(align, grad, eps):
    """The root of a product rounded by 2^-24 (half of it), the approximate root and reciprocal (2^-23 each), the
    sum and the result (2^-24 each): 6.5 units of 2^-24, and 2^-42 for their products."""
    n = 900_000
    p, g = _step(n, 8, _gradient(n, -6, 2, 3), eps, 2.0 ** -7, align, grad)
    g = g.astype(np.float64)
    want = -2.0 ** -7 * g / (np.abs(g) + np.float64(np.float32(eps)))
    off = np.abs(p - want) > np.abs(want) * (6.5 * U + 2.0 ** -42)
    assert not off.any(), (int(off.sum()), np.flatnonzero(off)[:5])


@pytest.mark.parametrize("eps", [1e-8, 1e-30])
@pytest.mark.parametrize("n", [1000, 900_000])
def test_values_at_the_ends(n, eps):
    """32-bit moments: a second moment that overflows divides by infinity, one that is zero or subnormal leaves eps,
    NaN passes; nothing else makes a NaN."""
    from gs_b200.training.optimizer import AdamW, ParamTensor
    g = torch.zeros(n, device="cuda")
    cases = [(1e25, 0.0), (-1e25, 0.0), (0.0, 0.0), (float("nan"), None), (float("inf"), None), (1e-22, 1e-22),
             (1e-30, 1e-30)]
    for i, (x, _) in enumerate(cases):
        g[i::len(cases)] = x
    p = torch.zeros(n, device="cuda")
    AdamW([ParamTensor(p, g, lr=2.0 ** -7)], b1=0.0, b2=0.0, eps=eps).step()
    p = p.cpu().numpy().astype(np.float64)
    e = float(np.float32(eps))
    for i, (x, root_of) in enumerate(cases):
        got = p[i::len(cases)]
        if root_of is None:
            assert np.isnan(got).all(), x
        elif x == 0.0 or abs(x) > 1e20:
            assert (got == 0.0).all(), x
        else:
            # v' = x^2 in float32, subnormal (1e-44) or 0
            root = float(np.sqrt(np.float64(np.float32(x) * np.float32(x))))
            want = -2.0 ** -7 * float(np.float32(x)) / (root + e)
            np.testing.assert_allclose(got, want, rtol=5 * U, atol=0)


@pytest.mark.parametrize("bits,n,align", [(32, 5000, 0), (32, 900_000, 0), (32, 900_000, 1), (8, 5000, 0),
                                          (8, 900_000, 0), (8, 900_000, 1)])
@pytest.mark.parametrize("eps", [1e-8, 1e-15])
def test_one_rounding_of_the_parameter(bits, n, align, eps):
    """With weight decay too, p' is rounded once at its own size (2^-24 of it); the rest are roundings of the update
    and of the decay, as tests/adamw_ref.py counts them."""
    from gs_b200.training.optimizer import AdamW, ParamTensor
    rng = np.random.default_rng(bits + n)
    p0 = rng.standard_normal(n).astype(np.float32)
    p = torch.zeros(n + align, device="cuda")[align:]
    g = torch.zeros(n + align, device="cuda")[align:]
    p.copy_(torch.tensor(p0))
    g.copy_(torch.tensor(_gradient(n, -6, 0, 5)))
    lr, wd = 1e-3, 0.3
    AdamW([ParamTensor(p, g, lr=lr, weight_decay=wd)], eps=eps, moment_bits=bits).step()
    z = np.zeros(n, np.float32)
    m, v = R.moments(z, z, g.cpu().numpy(), 1.0, 0.9, 0.999)
    want, _ = R.param(p0, m, v, 0, lr, wd, 0.9, 0.999, eps)
    upd = np.abs(want - p0) + 2 * lr * wd * np.abs(p0)  # no less than the update and the decay apart
    off = np.abs(p.cpu().numpy() - want) > U * np.abs(want) + 56 * U * upd
    assert not off.any(), (int(off.sum()), np.flatnonzero(off)[:5])
