"""Checks of AdamW's saved state that need no GPU."""
import pytest
import torch


def test_state_of_other_sizes_is_refused(monkeypatch):
    """8-bit moments of tensors in another order have buffers of the same length; their codes are not this plan's."""
    from gs_b200.training import optimizer as O
    monkeypatch.setattr(O, "_check_cuda", lambda *a, **k: None)
    monkeypatch.setattr(O, "_stream", lambda device: 0)

    def plan(sizes, bits=8):
        buf = lambda n: torch.zeros(n, dtype=torch.uint8)  # noqa: E731
        total = sum(-(-s // O.BLOCK) * O.BLOCK for s in sizes)
        m = O.Moments8(sizes, mu=buf(total), nu=buf(total), mu_exp=buf(total // O.BLOCK), nu_exp=buf(total // O.BLOCK))
        return O.AdamW([O.ParamTensor(torch.zeros(s), torch.zeros(s), lr=1e-3) for s in sizes], moments=m)

    a, b = plan([100, 200, 50]), plan([200, 100, 50])
    a.moments.mu.fill_(3)
    with pytest.raises(ValueError, match="sizes"):
        b.load_state_dict(a.state_dict())
    assert not b.moments.mu.any()
    c = plan([100, 200, 50])
    c.load_state_dict(a.state_dict())
    assert torch.equal(c.moments.mu, a.moments.mu)
    old = a.state_dict()
    del old["sizes"]  # as saved before the sizes were
    c.load_state_dict(old)
