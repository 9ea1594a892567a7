"""AdamW, the gradient norm and the conversions over so many elements that every
CTA takes several tiles and goes from one tensor to the next: rates, hash keys,
row flags, types and staged data are those of the tile's own tensor. All
elements are compared with the restatement (tests/adamw_ref.py)."""
import math

import numpy as np
import pytest
import torch

from tests import adamw_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# (gradient, copy, elements behind a 16-byte boundary, width of the mask's rows or 0, share of its rows)
KINDS = [("f32", None, 0, 0, 0.0), ("f32", None, 1, 0, 0.0), ("bf16", "bf16", 0, 0, 0.0), ("f32", None, 0, 48, 0.5),
         ("f16", "f16", 3, 0, 0.0), ("f32", "f16", 1, 7, 1.0), ("f32", None, 0, 3, 0.0), ("bf16", None, 0, 1, 0.3),
         ("f32", "bf16", 2, 4, 0.0), ("f16", None, 0, 32, 1.0)]


def _tensors(sizes, seed):
    from gs_b200.training.optimizer import ParamTensor
    rng = np.random.default_rng(seed)
    out = []
    for i, n in enumerate(sizes):
        grad, copy, off, width, share = KINDS[i % len(KINDS)]
        n = n // width * width if width else n
        p = torch.tensor((rng.standard_normal(n + off) * 0.05).astype(np.float32), device="cuda")[off:]
        g = (rng.standard_normal(n + off) * 10.0 ** rng.uniform(-6, -1)).astype(np.float32)
        active = None
        if width:
            active = torch.tensor(rng.uniform(size=n // width) < share, device="cuda")
            rows = np.repeat(active.cpu().numpy(), width)
            keep = rows | (rng.uniform(size=n) < 0.01 * (i % 2))  # some rows that are off have gradients all the same
            g[off:][~keep] = 0.0
            p = p.view(-1, width)
        g = torch.tensor(g, device="cuda").to(DT[grad])[off:]
        c = torch.zeros(n, dtype=DT[copy], device="cuda") if copy else None
        out.append(ParamTensor(p, g, lr=1e-3 * (1 + i % 7), weight_decay=0.05 * (i % 3), lr_decay_rate=0.5 ** (i % 4),
                               lr_transition_steps=10.0 + i % 5, active=active, copy=c))
    return out


def _np(t):
    return t.detach().float().cpu().numpy().reshape(-1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [
    [90_000 + 1237 * i for i in range(40)],                          # nearly every tile another tensor
    [1_900_001, 3, 1_300_000, 0, 2_000_100, 513, 700_005, 128, 64],  # several tiles in each, then the next
    [2_050_001] + [5, 1029, 300, 2047] * 80 + [2_100_000],           # hundreds of small ones between two large ones
], ids=["forty", "few", "hundreds"])
def test_tiles_of_many_tensors(bits, sizes):
    from gs_b200.training.optimizer import AdamW
    tensors = _tensors(sizes, len(sizes))
    opt = AdamW(tensors, moment_bits=bits, seed=17, count=3)
    assert sum(t.param.numel() for t in tensors) > 4_000_000
    for c in (3, 4):
        before = [(_np(t.param), m.cpu().numpy().reshape(-1), v.cpu().numpy().reshape(-1))
                  for t, (m, v) in zip(tensors, opt.moment_values())]
        opt.step()
        for i, (t, (p0, m0, v0), (m1, v1)) in enumerate(zip(tensors, before, opt.moment_values())):
            if not p0.size:
                continue
            m, v = R.moments(m0, v0, _np(t.grad), 1.0, 0.9, 0.999)
            lr = t.lr * t.lr_decay_rate ** (c / t.lr_transition_steps)
            rows = None
            if t.active is not None:
                rows = np.repeat(t.active.cpu().numpy(), p0.size // t.active.numel())
            want, err = R.param(p0, m, v, c, lr, t.weight_decay, 0.9, 0.999, 1e-8, rows)
            p1 = _np(t.param)
            off = np.abs(p1 - want) > err
            assert not off.any(), (i, np.flatnonzero(off)[:5], p1[off][:5], want[off][:5])
            m1, v1 = m1.cpu().numpy().reshape(-1), v1.cpu().numpy().reshape(-1)
            if bits == 32:
                np.testing.assert_array_equal(m1, m, err_msg=str(i))
                np.testing.assert_array_equal(v1, v, err_msg=str(i))
            else:
                h = R.noise(17, c, i, p0.size)
                for got, x, u, signed in ((m1, m, h % 65536, True), (v1, v, h // 65536, False)):
                    want8 = R.decode(*R.encode(x, u / 65536.0, signed), signed)
                    np.testing.assert_array_equal(got, want8, err_msg=str(i))
            if t.copy is not None:
                assert torch.equal(t.copy, t.param.reshape(-1).to(t.copy.dtype)), i
    assert int(opt.count) == 5


@pytest.mark.parametrize("count", [5, 9, 60, 200, 1500])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_norm_over_tiles_of_many_tensors(count, grad):
    """Magnitudes differ by orders between tensors, so that a tensor left out or taken twice shows."""
    from gs_b200.training.optimizer import GradNorm
    rng = np.random.default_rng(count)
    share = rng.dirichlet(np.ones(count))
    sizes = [int(x) for x in share * (13_000_000 if grad == "bf16" else 6_500_000)]
    grads = []
    for i, n in enumerate(sizes):
        a = torch.randn(n + i % 3, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) * 10.0 ** rng.uniform(-2, 2)
        grads.append(a.to(DT[grad])[i % 3:])
    plan = GradNorm(grads, 1.0)
    out = plan().cpu().numpy()
    np.testing.assert_allclose(out, R.grad_norm([_np(t) for t in grads], 1.0), rtol=2.0 ** -23)
    for t in grads[:: max(1, count // 5)]:
        t.zero_()
    np.testing.assert_allclose(plan().cpu().numpy(), R.grad_norm([_np(t) for t in grads], 1.0), rtol=2.0 ** -23)


def test_conversions_of_many_elements():
    """More than two rounds of the decoding grid, and five of the encoding one."""
    from gs_b200.training.optimizer import Moments8
    rng = np.random.default_rng(0)
    m8 = Moments8([5_900_003, 77, 300_001], "cuda")
    mu = (rng.standard_normal(m8.total) * 10.0 ** rng.uniform(-20, 3, m8.total)).astype(np.float32)
    nu = (10.0 ** rng.uniform(-30, 2, m8.total)).astype(np.float32)
    m8.set_values(torch.tensor(mu, device="cuda"), torch.tensor(nu, device="cuda"))
    for codes, exps, x, signed in ((m8.mu, m8.mu_exp, mu, True), (m8.nu, m8.nu_exp, nu, False)):
        c, e = R.encode(x, np.full(x.size, 0.5), signed)
        np.testing.assert_array_equal(codes.cpu().numpy(), c)
        np.testing.assert_array_equal(exps.cpu().numpy(), e)
    vm, vn = m8.values()
    np.testing.assert_array_equal(vm.cpu().numpy(), R.decode(m8.mu.cpu().numpy(), m8.mu_exp.cpu().numpy(), True))
    np.testing.assert_array_equal(vn.cpu().numpy(), R.decode(m8.nu.cpu().numpy(), m8.nu_exp.cpu().numpy(), False))
    bm, bn = m8.values(torch.bfloat16)
    assert torch.equal(bm.float(), vm) and torch.equal(bn.float(), vn)


@pytest.mark.parametrize("count", [1, 7, 8, 9, 127, 129, 1003, 2_500_005])
@pytest.mark.parametrize("codes_at,values_at", [(0, 0), (4, 0), (0, 1), (4, 2), (8, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conversions_of_any_count_and_alignment(count, codes_at, values_at, dtype):
    """The C entries on codes that are 4- but not 8-byte aligned, values off 16 bytes, counts off 8; nothing behind."""
    from gs_b200 import _lib
    rng = np.random.default_rng(count)
    blocks = -(-count // 128)
    x = [torch.tensor((rng.standard_normal(count) * 10.0 ** rng.uniform(-8, 2, count)).astype(np.float32), device="cuda")
         for _ in range(2)]
    x[1].abs_()
    codes = [torch.full((count + 16,), 77, dtype=torch.uint8, device="cuda") for _ in range(2)]
    exps = [torch.full((blocks + 1,), 77, dtype=torch.uint8, device="cuda") for _ in range(2)]
    P, st = _lib.ptr, _lib.stream(x[0].device)
    at = [t[codes_at:] for t in codes]
    _lib.call("gs_moments8_encode", P(x[0]), P(x[1]), count, P(at[0]), P(at[1]), P(exps[0]), P(exps[1]), st)
    out = [torch.full((count + 8,), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    vals = [t[values_at:] for t in out]
    _lib.call("gs_moments8_decode", P(at[0]), P(at[1]), P(exps[0]), P(exps[1]), count,
              _lib.GS_TYPE_F32 if dtype == torch.float32 else _lib.GS_TYPE_BF16, P(vals[0]), P(vals[1]), st)
    for k, signed in ((0, True), (1, False)):
        c, e = R.encode(x[k].cpu().numpy(), np.full(count, 0.5), signed)
        got = at[k].cpu().numpy()
        np.testing.assert_array_equal(got[:count], c)
        assert (got[count:] == 77).all() and (codes[k][:codes_at] == 77).all()
        assert int(exps[k][blocks]) == 77
        np.testing.assert_array_equal(exps[k][:blocks].cpu().numpy(), e)
        v = vals[k].float().cpu().numpy()
        np.testing.assert_array_equal(v[:count], R.decode(c, e, signed))
        assert (v[count:] == 7.0).all() and (out[k][:values_at].float() == 7.0).all()
