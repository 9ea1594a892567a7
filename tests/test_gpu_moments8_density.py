"""Density control on 8-bit moments: its memory, and the moments of every slot
against the rows' moves in 64 bits."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as A

pytestmark = pytest.mark.gpu


def _scene(n, k, bits, seed=0, moves=0.2):
    """A state with moments, statistics that clone and split some Gaussians and empty slots for them."""
    from gs_b200.training.trainer import DensityState
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = DensityState(n, k, "cuda", moment_bits=bits)
    st.params.copy_(torch.randn(st.size, generator=g, device="cuda"))
    st.gaussians.scales.mul_(0.8).sub_(3.5)  # around the split size
    st.gaussians.opacities.add_(2.0)
    st.active_mask.copy_(torch.rand(n, generator=g, device="cuda") < 0.6)
    st.grad_accum.copy_((torch.rand(n, generator=g, device="cuda") < moves).float())
    st.denom.fill_(1)
    mu = torch.randn(st.size, generator=g, device="cuda") * torch.exp(3 * torch.randn(st.size, generator=g, device="cuda"))
    nu = torch.exp(4 * torch.randn(st.size, generator=g, device="cuda")) * 1e-6
    if bits == 8:
        flat = [torch.zeros(st.moments8.total, device="cuda") for _ in range(2)]
        for t, x in zip(flat, (mu, nu)):
            for part, (a, b) in zip(st.moments8.split(t), st.segments):
                part.copy_(x[a:b])
        st.moments8.set_values(*flat)
    else:
        st.mu.copy_(mu)
        st.nu.copy_(nu)
    return st


def _values(st):
    return [torch.cat(st.moments8.split(x)).cpu().numpy() for x in st.moments8.values()]


@pytest.mark.parametrize("n,k", [(1, 1), (37, 4), (1000, 16), (4099, 16), (20_001, 9)])
def test_moved_moments(n, k):
    """Every slot that receives a row has the row's moments, rounded to nearest in its own block; the other
    slots' values are those of blocks that hold them exactly, or rounded in a block that changed."""
    from gs_b200.training.density import densify_and_prune
    from gs_b200.training.trainer import DensityState
    st = _scene(n, k, 8, seed=n)
    before = _values(st)
    ref = DensityState(n, k, "cuda")
    ref.params.copy_(st.params)
    for buf, x in zip((ref.mu, ref.nu), before):
        buf.copy_(torch.tensor(x))
    for name in ("active_mask", "grad_accum", "denom", "max_radii"):
        getattr(ref, name).copy_(getattr(st, name))
    noise = torch.randn((n, 3), device="cuda")
    for s in (st, ref):
        densify_and_prune(s, grad_threshold=0.5, noise=noise)
    assert torch.equal(st.densify_info, ref.densify_info)
    if n >= 1000:
        assert int(st.densify_info[1]) > 0 and int(st.densify_info[2]) > 0
    for name in ("params", "active_mask", "grad_accum", "denom", "max_radii"):
        assert torch.equal(getattr(st, name), getattr(ref, name)), name
    for x, want, signed in zip(_values(st), (ref.mu.cpu().numpy(), ref.nu.cpu().numpy()), (True, False)):
        for a, b in st.segments:
            w = want[a:b]
            np.testing.assert_array_equal(x[a:b], A.decode(*A.encode(w, np.full(b - a, 0.5), signed), signed))


@pytest.mark.parametrize("enabled", [True, False])
def test_moments_stay_where_nothing_moves(enabled):
    from gs_b200.training.density import densify_and_prune
    st = _scene(5000, 16, 8, seed=4, moves=0.0 if enabled else 0.5)
    before = [t.clone() for t in st.moment_buffers()]
    densify_and_prune(st, densify_enabled=enabled, grad_threshold=0.5)
    assert int(st.densify_info[3]) == 0
    for a, b in zip(before, st.moment_buffers()):
        assert torch.equal(a, b)


def test_a_block_that_is_not_finite_moves_as_one():
    """A row from a block that reads as NaN makes its new block NaN; the blocks of the row's other groups stay finite."""
    from gs_b200.training.density import densify_and_prune
    st = _scene(2000, 4, 8, seed=9)
    before = _values(st)
    src_block = 3
    st.moments8.mu_exp[src_block] = 255
    active0 = st.active_mask.clone()
    densify_and_prune(st, grad_threshold=0.5)
    assert int(st.densify_info[1]) > 0
    mu = _values(st)[0]
    bad = np.isnan(mu)
    assert bad[src_block * 128:(src_block + 1) * 128].all()
    assert not np.isnan(_values(st)[1]).any() and not np.isnan(before[0]).any()
    first = st.segments[0][1]
    assert not bad[first:].any()  # the block lies in the first group
    assert (bad[:first].reshape(-1)[: first // 128 * 128].reshape(-1, 128).all(1)
            == bad[:first // 128 * 128].reshape(-1, 128).any(1)).all()
    del active0


def _peak(bits, n=400_000, k=16):
    from gs_b200.training.density import densify_and_prune
    st = _scene(n, k, bits, seed=1)
    noise = torch.randn((n, 3), device="cuda")
    st._buffers.clear()
    held = sum(t.numel() * t.element_size() for t in st.moment_buffers())
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    densify_and_prune(st, grad_threshold=0.5, noise=noise)
    torch.cuda.synchronize()
    assert int(st.densify_info[1]) > 0
    return held, torch.cuda.max_memory_allocated() - base, st.size


def test_peak_memory():
    """Density control keeps what 8-bit moments save: beside the moments it needs at most one moment's codes
    (1 byte an element and the exponent bytes) more than it does with 32-bit moments, so that the peak of the
    moments and what moves them stays below half of the 32-bit moments."""
    held32, extra32, size = _peak(32)
    held8, extra8, _ = _peak(8)
    assert held32 == 8 * size
    assert extra8 - extra32 <= 1.05 * size + (1 << 20)
    assert held8 + extra8 - extra32 < 0.5 * held32
