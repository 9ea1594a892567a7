"""AdamW over many tensors, the global gradient norm and the 8-bit moments on
the GPU, against the restatement in tests/adamw_ref.py: moments and codes
exactly, parameters within the roundings of their update."""
import math

import numpy as np
import pytest
import torch

from tests import adamw_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _views(rng_sizes, align, dtype, device="cuda"):
    """Views of one flat buffer: starts at multiples of `align` elements, plus `align == 1` shifted by one."""
    starts, at = [], 1 if align == 1 else 0
    for s in rng_sizes:
        starts.append(at)
        at += -(-s // align) * align
    flat = torch.full((at + 8,), 7.0, dtype=dtype, device=device)
    return flat, [flat[a:a + s] for a, s in zip(starts, rng_sizes)]


class Setup:
    """Tensors of the given sizes with their numpy doubles."""

    def __init__(self, sizes, bits, grad="f32", copy=None, active=None, align=128, seed=0, lr=2e-3, wd=0.1, **kw):
        from gs_b200.training.optimizer import AdamW, ParamTensor
        rng = np.random.default_rng(seed)
        self.sizes, self.bits, self.seed = sizes, bits, seed
        self.flat_p, self.p = _views(sizes, align, torch.float32)
        self.flat_g, self.g = _views(sizes, align, DT[grad])
        self.copies = _views(sizes, align, DT[copy])[1] if copy else [None] * len(sizes)
        self.active = active or [None] * len(sizes)
        for i, n in enumerate(sizes):
            self.p[i].copy_(torch.tensor(rng.standard_normal(n).astype(np.float32) * 0.05))
        self.set_grads(rng)
        if active:
            self.p = [p.view(a.numel(), -1) if a is not None else p for p, a in zip(self.p, self.active)]
        self.lr = [lr * (1 + i % 3) for i in range(len(sizes))]
        self.wd = [wd * (i % 2) for i in range(len(sizes))]
        self.decay, self.steps = 0.01, 1000.0
        self.b1, self.b2, self.eps = kw.get("b1", 0.9), kw.get("b2", 0.999), kw.get("eps", 1e-8)
        tensors = [ParamTensor(p, g, lr=self.lr[i], weight_decay=self.wd[i], lr_decay_rate=self.decay,
                               lr_transition_steps=self.steps, active=self.active[i], copy=self.copies[i])
                   for i, (p, g) in enumerate(zip(self.p, self.g))]
        moments = kw.pop("moments", None)
        if bits == 32 and moments is None:
            mv = [_views(sizes, align, torch.float32)[1] for _ in range(2)]
            for t in mv[0] + mv[1]:
                t.zero_()
            moments = list(zip(*mv))
        self.opt = AdamW(tensors, moment_bits=bits, moments=moments, seed=seed, **kw)

    def set_grads(self, rng, scale=1e-3):
        for g in self.g:
            n = g.numel()
            a = rng.standard_normal(n) * np.exp(2.0 * rng.standard_normal(n)) * scale
            a[rng.uniform(size=n) < 0.2] = 0.0
            g.copy_(torch.tensor(a.astype(np.float32)))

    def read(self):
        """(p, g, mu, nu) of every tensor as float32 arrays."""
        mv = self.opt.moment_values()
        return [tuple(x.detach().float().cpu().numpy().reshape(-1) for x in (p, g, m, v))
                for p, g, (m, v) in zip(self.p, self.g, mv)]

    def codes(self):
        m = self.opt.moments
        out = []
        for a, n in zip(m.starts, m.sizes):
            e = slice(a // 128, a // 128 + -(-n // 128))
            out.append(tuple(t.cpu().numpy() for t in (m.mu[a:a + n], m.nu[a:a + n], m.mu_exp[e], m.nu_exp[e])))
        return out

    def step_and_check(self, scale=1.0):
        before = self.read()
        c = int(self.opt.count)
        self.opt.step()
        after = self.read()
        codes = self.codes() if self.bits == 8 else None
        for i, ((p0, g, m0, v0), (p1, _, m1, v1)) in enumerate(zip(before, after)):
            if not p0.size:
                continue
            m, v = R.moments(m0, v0, g, scale, self.b1, self.b2)
            act = None
            if self.active[i] is not None:
                act = np.repeat(self.active[i].cpu().numpy() != 0, p0.size // self.active[i].numel())
            lr = self.lr[i] * self.decay ** (c / self.steps)
            want, err = R.param(p0, m, v, c, lr, self.wd[i], self.b1, self.b2, self.eps, act)
            off = np.abs(p1 - want) > err
            assert not off.any(), (i, np.flatnonzero(off)[:5], p1[off][:5], want[off][:5], p0[off][:5])
            if self.bits == 32:
                np.testing.assert_array_equal(m1, m)
                np.testing.assert_array_equal(v1, v)
            else:
                h = R.noise(self.seed, c, i, p0.size)
                for got, x, u, signed, exps in ((codes[i][0], m, h % 65536, True, codes[i][2]),
                                                (codes[i][1], v, h // 65536, False, codes[i][3])):
                    want_c, want_e = R.encode(x, u / 65536.0, signed)
                    np.testing.assert_array_equal(exps, want_e)
                    np.testing.assert_array_equal(got, want_c)
            if self.copies[i] is not None:
                want_copy = torch.tensor(p1).to(self.copies[i].dtype)
                assert torch.equal(self.copies[i].cpu(), want_copy)
        assert int(self.opt.count) == c + 1


SIZES = {
    "one": [1],
    "small": [1, 127, 128, 129, 0, 5, 1024, 1025, 2047],
    "middle": [4099, 100_003, 17, 33_000],
}


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("align", [128, 4, 1])
def test_step_matches_restatement(bits, sizes, align):
    s = Setup(SIZES[sizes], bits, align=align, seed=3)
    rng = np.random.default_rng(5)
    for _ in range(3):
        s.step_and_check()
        s.set_grads(rng)
    # nothing outside the tensors was written
    pad = torch.ones_like(s.flat_p, dtype=torch.bool)
    for p in s.p:
        a = (p.data_ptr() - s.flat_p.data_ptr()) // 4
        pad[a:a + p.numel()] = False
    assert (s.flat_p[pad] == 7.0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("copy", ["bf16", "f16", None])
@pytest.mark.parametrize("align", [128, 2, 1])
def test_types(bits, grad, copy, align):
    s = Setup([4096, 333, 1, 1500], bits, grad=grad, copy=copy, align=align, seed=7,
              grad_scale=torch.tensor(0.3, device="cuda"))
    for _ in range(2):
        s.step_and_check(scale=np.float32(0.3))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 40, 1001])
@pytest.mark.parametrize("align", [128, 1])
def test_active_rows(bits, n, align):
    """Rows that the mask leaves out keep their parameter (none left, some, all), their moments go on."""
    rng = np.random.default_rng(n)
    masks = [torch.tensor(rng.uniform(size=n) < f, device="cuda") for f in (0.0, 0.5, 1.0)]
    widths = [3, 1, 48, 7, 4]
    active = [masks[1], masks[0], masks[1], masks[2].to(torch.uint8), None]
    s = Setup([n * w for w in widths], bits, active=active, align=align, seed=11)
    s.p[4] = s.p[4].view(-1)
    for _ in range(2):
        s.step_and_check()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [8, 9, 256, 257, 600])
def test_many_tensors(bits, count):
    rng = np.random.default_rng(count)
    s = Setup([int(x) for x in rng.integers(0, 300, count)], bits, seed=count, grad="bf16")
    s.step_and_check()
    s.step_and_check()


@pytest.mark.parametrize("b1,b2,eps", [(0.0, 0.999, 1e-8), (0.9, 0.0, 1e-8), (0.95, 0.9999, 1e-15), (0.5, 0.9, 1e-3)])
@pytest.mark.parametrize("count", [0, 1, 100_000])
def test_hyperparameters(b1, b2, eps, count):
    for bits in (32, 8):
        s = Setup([1000, 77], bits, seed=2, b1=b1, b2=b2, eps=eps, count=count)
        s.decay, s.steps = 1.0, 1.0
        for t in s.opt.tensors:
            t.lr_decay_rate, t.lr_transition_steps = 1.0, 1.0
        s.opt.refresh()
        s.step_and_check()
        s.step_and_check()


@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(bits):
    """Subnormal to huge gradients in one block, a block of zeros, a block whose second moments underflow."""
    s = Setup([640], bits, seed=4)
    g = np.zeros(640, np.float32)
    g[:128] = np.logspace(-44, 15, 128)
    g[128:256] = -np.logspace(-12, -4, 128)
    g[384:512] = 1e-30
    g[512:] = np.float32(1e18)
    s.g[0].copy_(torch.tensor(g))
    for _ in range(3):
        s.step_and_check()


def test_values_that_are_not_finite_stay_in_their_block():
    s = Setup([512], 8, seed=1)
    s.g[0][200] = float("nan")
    s.g[0][300] = float("inf")
    s.opt.step()
    mu, nu = (x.cpu().numpy() for x in s.opt.moments.values())
    bad = np.zeros(512, bool)
    bad[128:384] = True
    np.testing.assert_array_equal(np.isnan(mu[:512]), bad)
    np.testing.assert_array_equal(np.isnan(nu[:512]), bad)
    p = s.p[0].cpu().numpy()
    np.testing.assert_array_equal(np.flatnonzero(np.isnan(p)), [200, 300])
    t = Setup([512], 32, seed=1)
    t.g[0][200] = float("nan")
    t.opt.step()
    (p, _, m, v), = t.read()
    for x in (p, m, v):
        np.testing.assert_array_equal(np.flatnonzero(np.isnan(x)), [200])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_not_finite_skips_the_step(bits, bad):
    scale = torch.tensor(bad, device="cuda")
    s = Setup([300, 2000], bits, copy="bf16", grad_scale=scale, count=5)
    before, copies = s.read(), [c.clone() for c in s.copies]
    s.opt.step()
    s.opt.step()
    for x, y in zip(before, s.read()):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(copies, s.copies))
    assert int(s.opt.count) == 5 and int(s.opt.skipped) == 2
    scale.fill_(0.5)
    s.step_and_check(scale=np.float32(0.5))
    assert int(s.opt.skipped) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(bits):
    runs = []
    for captured in (False, True):
        s = Setup([5000, 129, 40_000], bits, seed=9, max_grad_norm=0.01)
        if captured:
            s.opt.step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                s.opt.step()
            for _ in range(4):
                graph.replay()
        else:
            for _ in range(5):
                s.opt.step()
        assert int(s.opt.count) == 5
        runs.append(s.read())
    for x, y in zip(*runs):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)


def test_another_stream_and_the_version_counter():
    s = Setup([50_000], 8, seed=6)
    s.p[0].requires_grad_(False)
    version = s.p[0]._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step_and_check()
    torch.cuda.current_stream().wait_stream(side)
    assert s.p[0]._version > version
    w = torch.ones(10, device="cuda", requires_grad=True)
    from gs_b200.training.optimizer import AdamW, ParamTensor
    opt = AdamW([ParamTensor(w, torch.ones(10, device="cuda"), lr=1e-3)])
    y = (w * w).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rounding_keeps_the_mean():
    """A constant gradient, 400 steps: the mean of nu over 65536 elements follows the 32-bit one. Each step's
    rounding is unbiased with a deviation below one step (1/8) of the value; a value remembers 1000 steps, so its
    own deviation is below sqrt(400) / 8 = 2.5 of the value and the mean's below 2.5 / 256 = 1 %: four of them."""
    n = 65536
    s = Setup([n], 8, seed=12, lr=0.0)
    s.g[0].fill_(1e-3)
    for _ in range(400):
        s.opt.step()
    (_, _, m, v), = s.read()
    want_v = 1e-6 * (1 - 0.999 ** 400)
    want_m = 1e-3 * (1 - 0.9 ** 400)
    assert abs(v.mean(dtype=np.float64) / want_v - 1) < 0.04
    assert abs(m.mean(dtype=np.float64) / want_m - 1) < 0.04
    assert v.min() > 0


def test_a_moment_that_decays_never_reaches_zero():
    s = Setup([256], 8, seed=13, lr=1e-3, b2=0.5)
    s.set_grads(np.random.default_rng(0))
    s.g[0][0] = 1.0  # the block's largest value
    s.opt.step()
    nu0 = s.read()[0][3]
    s.g[0].zero_()
    s.g[0][0] = 1.0
    for _ in range(200):
        s.step_and_check()
    p, _, _, nu = s.read()[0]
    # the second block decays as a whole, by 2^-200: to 0 in float32 itself (2^-149)
    assert (nu[:128][nu0[:128] > 0] > 0).all() and (nu[128:] == 0).all() and np.isfinite(p).all()


def test_far_elements():
    """A tensor of more than 2^32 bytes of parameters and 2^31 elements: its ends against the restatement."""
    from gs_b200.training.optimizer import AdamW, ParamTensor
    n = (1 << 31) + 129
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    ends = [slice(0, 256), slice(n - 257, n)]  # the second from a block's start
    rng = np.random.default_rng(0)
    for e in ends:
        g[e] = torch.tensor(rng.standard_normal(e.stop - e.start).astype(np.float32) * 1e-3).cuda()
        p[e] = 1.0
    opt = AdamW([ParamTensor(p, g, lr=1e-2, weight_decay=0.1)], moment_bits=8, seed=5)
    opt.step()
    m8 = opt.moments
    for e in ends:
        k = e.stop - e.start
        gn = g[e].float().cpu().numpy()
        m, v = R.moments(np.zeros(k, np.float32), np.zeros(k, np.float32), gn, 1.0, 0.9, 0.999)
        want, err = R.param(np.ones(k, np.float32), m, v, 0, 1e-2, 0.1, 0.9, 0.999, 1e-8)
        assert (np.abs(p[e].cpu().numpy() - want) <= err).all()
        h = R.noise(5, 0, 0, k, start=e.start)
        cm, em = R.encode(m, (h % 65536) / 65536.0, True)
        cv, ev = R.encode(v, (h // 65536) / 65536.0, False)
        b = slice(e.start // 128, -(-e.stop // 128))
        np.testing.assert_array_equal(m8.mu[e].cpu().numpy(), cm)
        np.testing.assert_array_equal(m8.nu[e].cpu().numpy(), cv)
        np.testing.assert_array_equal(m8.mu_exp[b].cpu().numpy(), em)
        np.testing.assert_array_equal(m8.nu_exp[b].cpu().numpy(), ev)
    assert float(p[1000:1 << 20].abs().max()) == 0.0
    del p, g, opt, m8
    torch.cuda.empty_cache()


# ---- gradient norm -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [[1], [0], [0, 3, 0], [127, 4096, 2049, 1], [1_000_003]])
@pytest.mark.parametrize("align", [128, 1])
def test_norm_matches(grad, sizes, align):
    from gs_b200.training.optimizer import GradNorm
    rng = np.random.default_rng(1)
    _, g = _views(sizes, align, DT[grad])
    for t in g:
        t.copy_(torch.tensor(rng.standard_normal(t.numel()).astype(np.float32)))
    arrays = [t.float().cpu().numpy() for t in g]
    for max_norm, unscale in ((math.inf, None), (0.5, None), (0.5, 2.0 ** -10), (1e6, 0.25)):
        u = None if unscale is None else torch.tensor(unscale, device="cuda")
        plan = GradNorm(g, max_norm, u)
        want = R.grad_norm(arrays, max_norm, 1.0 if unscale is None else unscale)
        for _ in range(2):
            out = plan().cpu().numpy().astype(np.float64)
            # one rounding to float32 (2^-24); the sums are in 64 bits
            np.testing.assert_allclose(out, want, rtol=2.0 ** -23)
        assert float(plan.norm) == out[0] and float(plan.scale) == out[1]


@pytest.mark.parametrize("count", [8, 9, 1024, 1025, 2500])
def test_norm_of_many_tensors(count):
    from gs_b200.training.optimizer import GradNorm
    rng = np.random.default_rng(count)
    sizes = [int(x) for x in rng.integers(0, 200, count)]
    _, g = _views(sizes, 128, torch.float32)
    for t in g:
        t.copy_(torch.tensor(rng.standard_normal(t.numel()).astype(np.float32)))
    out = GradNorm(g, 1.0)().cpu().numpy()
    np.testing.assert_allclose(out, R.grad_norm([t.cpu().numpy() for t in g], 1.0), rtol=2.0 ** -23)


def test_norm_is_the_same_every_time():
    from gs_b200.training.optimizer import GradNorm
    g = torch.randn(3_000_001, device="cuda")
    plan = GradNorm([g])
    first = plan().clone()
    for _ in range(20):
        assert torch.equal(plan(), first)


@pytest.mark.parametrize("value,norm", [(1e30, 1e30 * 100), (1e-30, 1e-30 * 100), (math.nan, None), (math.inf, None),
                                        (3e38, None)])
def test_norm_range(value, norm):
    """No overflow or underflow of the squares; a norm that float32 does not hold is not finite."""
    from gs_b200.training.optimizer import GradNorm
    g = torch.zeros(20_000, device="cuda")
    g[7::2] = value if math.isfinite(value) else 1.0
    g[7::2][10_000 - 4:] = 0.0
    if not math.isfinite(value):
        g[12_345] = value
    n = int((g != 0).sum())
    out = GradNorm([g], 1.0)().cpu().numpy()
    if norm is None:
        assert not math.isfinite(out[0]) and math.isnan(out[1])
    else:
        want = abs(float(np.float32(value))) * math.sqrt(n)
        np.testing.assert_allclose(out, [want, min(1.0, 1.0 / want)], rtol=2.0 ** -23)


# ---- the chain, conversions and refusals -------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_steps_and_a_bad_gradient(bits):
    """Norm, clip and step as a training loop runs them; a gradient that overflowed is stepped over."""
    s = Setup([3000, 129, 50], bits, seed=8, max_grad_norm=0.02, grad="f16")
    rng = np.random.default_rng(3)
    for k in range(4):
        s.set_grads(rng, scale=10.0 ** -(k % 3))
        if k == 2:
            s.g[1][5] = float("inf")
            before = s.read()
            s.opt.step()
            for x, y in zip(before, s.read()):
                for a, b in zip((x[0], x[2], x[3]), (y[0], y[2], y[3])):
                    np.testing.assert_array_equal(a, b)
            assert int(s.opt.skipped) == 1
            continue
        norm, scale = R.grad_norm([g.float().cpu().numpy() for g in s.g], 0.02)
        s.opt.norm()
        np.testing.assert_allclose(s.opt.norm.out.cpu().numpy(), [norm, scale], rtol=2.0 ** -23)
        s.step_and_check(scale=s.opt.norm.scale.cpu().numpy())
    assert int(s.opt.count) == 3


def test_adamw_is_adam_without_decay():
    """Against the framework's own flat Adam on the same inputs: the moments to the
    rounding of their sums, the parameters to that of the update."""
    from gs_b200 import _lib
    from gs_b200.training.optimizer import AdamW, ParamTensor
    n = 10_001
    g = torch.randn(n, device="cuda") * 1e-2
    p = torch.randn(n, device="cuda")
    q, mu, nu = p.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    opt = AdamW([ParamTensor(p, g, lr=1e-3)])
    for _ in range(5):
        opt.step()
        _lib.call("gs_adam_step_flat_device", _lib.ptr(q), _lib.ptr(g), _lib.ptr(mu), _lib.ptr(nu), n, 1e-3, 0.9,
                  0.999, 1e-8, _lib.ptr(state), _lib.stream(q.device))
    (m, v), = opt.moment_values()
    # five sums of roundings of 2^-24 each (FMA in one of the two)
    torch.testing.assert_close(m, mu, rtol=20 * 2.0 ** -24, atol=1e-9)
    torch.testing.assert_close(v, nu, rtol=20 * 2.0 ** -24, atol=1e-12)
    # 1 - 0.999f^t loses 2^-24 / (1 - 0.999) = 6e-5 of itself there, half of that in the root: 5 steps of 1e-3.
    # p itself is rounded once a step on each side: 10 roundings of 2^-24 in five steps
    torch.testing.assert_close(p, q, rtol=10 * 2.0 ** -24, atol=5 * 1e-3 * 6e-5)


@pytest.mark.parametrize("sizes", [[1], [128], [1000, 0, 129, 5]])
def test_conversions(sizes):
    from gs_b200.training.optimizer import Moments8
    rng = np.random.default_rng(0)
    m8 = Moments8(sizes, "cuda")
    z = m8.values()
    assert float(z[0].abs().max()) == 0.0 and float(z[1].abs().max()) == 0.0
    mu = (rng.standard_normal(m8.total) * np.exp(3 * rng.standard_normal(m8.total))).astype(np.float32)
    nu = (np.exp(6 * rng.standard_normal(m8.total)) * 1e-6).astype(np.float32)
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
    before = [t.clone() for t in (m8.mu, m8.nu)]
    m8.set_values(vm, vn)
    after = m8.values()
    assert torch.equal(after[0], vm) and torch.equal(after[1], vn)
    del before


def test_state_dict_round_trip():
    for bits in (32, 8):
        s = Setup([500, 200], bits, seed=1)
        t = Setup([500, 200], bits, seed=1)
        s.opt.step()
        t.opt.load_state_dict(s.opt.state_dict())
        for a, b in zip(s.p, t.p):
            b.copy_(a)
        s.opt.step()
        t.opt.step()
        for x, y in zip(s.read(), t.read()):
            for a, b in zip(x, y):
                np.testing.assert_array_equal(a, b)
        assert int(t.opt.count) == 2
    with pytest.raises(ValueError, match="bits"):
        t.opt.load_state_dict(Setup([500, 200], 32).opt.state_dict())
    with pytest.raises(ValueError, match="sizes"):
        t.opt.load_state_dict(Setup([500, 300], 8).opt.state_dict())


def test_refusals():
    from gs_b200.training.optimizer import AdamW, GradNorm, Moments8, ParamTensor
    z = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")  # noqa: E731
    bad = [
        (ParamTensor(z(8, torch.float16), z(8), lr=1.0), "dtype"),
        (ParamTensor(z(8), z(8, torch.float64), lr=1.0), "dtype"),
        (ParamTensor(z(8), z(9), lr=1.0), "elements"),
        (ParamTensor(z((8, 8)).t()[1:], z(56), lr=1.0), "contiguous"),
        (ParamTensor(z(8), z(8), lr=1.0, active=z(7, torch.bool)), "flags"),
        (ParamTensor(z(8), z(8), lr=1.0, active=z(8)), "dtype"),
        (ParamTensor(z((1, 32_769)), z(32_769), lr=1.0, active=z(1, torch.bool)), "32768"),
        (ParamTensor(z(8), z(8), lr=1.0, copy=z(8)), "dtype"),
        (ParamTensor(z(8), z(8), lr=1.0, copy=z(9, torch.float16)), "elements"),
        (ParamTensor(z(8), torch.zeros(8), lr=1.0), "CUDA"),
    ]
    for t, match in bad:
        with pytest.raises(ValueError, match=match):
            AdamW([t])
    p = z(8)
    with pytest.raises(ValueError, match="shares memory"):
        AdamW([ParamTensor(p, z(8), lr=1.0), ParamTensor(p, z(8), lr=1.0)])
    with pytest.raises(ValueError, match="shares memory"):
        AdamW([ParamTensor(p, p, lr=1.0)])
    ok = [ParamTensor(z(8), z(8), lr=1.0)]
    for kw, match in ((dict(moment_bits=16), "moment_bits"), (dict(moments=[]), "pairs"),
                      (dict(moments=[(z(8), z(7))]), "elements"), (dict(moments=Moments8([9], "cuda")), "sizes"),
                      (dict(moment_bits=32, moments=Moments8([8], "cuda")), "moment_bits"), (dict(count=-1), "count"),
                      (dict(grad_scale=z(2)), "one value"), (dict(max_grad_norm=0.0), "positive")):
        with pytest.raises(ValueError, match=match):
            AdamW(ok, **kw)
    from gs_b200._lib import GsError
    for kw in (dict(b1=1.0), dict(b2=-0.5), dict(eps=0.0)):
        with pytest.raises(GsError):
            AdamW(ok, **kw).step()
    opt = AdamW([ParamTensor(z(8), z(8), lr=math.nan)])
    with pytest.raises(GsError):
        opt.step()
    with pytest.raises(ValueError, match="expected"):
        GradNorm([z(8)], unscale=z(1, torch.float64))
    with pytest.raises(ValueError, match="bytes"):
        Moments8([8], mu=z(8, torch.uint8), nu=z(128, torch.uint8), mu_exp=z(1, torch.uint8), nu_exp=z(1, torch.uint8))
    with pytest.raises(ValueError, match="dtype"):
        Moments8([8], "cuda").values(torch.float16)


# ---- the kernels for many elements (the others above run in the kernel for few) ------------------------------


BIG = [700_001, 513, 0, 4097, 2048, 130, 1]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad,copy,align", [
    ("f32", None, 128), ("f32", "bf16", 128), ("bf16", None, 128), ("bf16", "bf16", 128), ("f16", "f16", 128),
    ("f16", None, 128), ("f32", None, 1), ("f32", None, 4), ("f32", None, 2), ("f32", "f16", 1), ("bf16", None, 1),
    ("bf16", "bf16", 1), ("f16", "f16", 4), ("bf16", None, 2)])
def test_many_elements(bits, grad, copy, align):
    s = Setup(BIG, bits, grad=grad, copy=copy, align=align, seed=21, grad_scale=torch.tensor(0.7, device="cuda"))
    for _ in range(2):
        s.step_and_check(scale=np.float32(0.7))
    pad = torch.ones_like(s.flat_p, dtype=torch.bool)
    for p in s.p:
        a = (p.data_ptr() - s.flat_p.data_ptr()) // 4
        pad[a:a + p.numel()] = False
    assert (s.flat_p[pad] == 7.0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copy", [None, "bf16"])
@pytest.mark.parametrize("align", [128, 1])
def test_many_rows(bits, copy, align):
    """Masks with whole chunks on, whole chunks off and changing row by row; widths from 1 to the largest."""
    rng = np.random.default_rng(0)
    n = 20_011
    flags = rng.uniform(size=n) < 0.5
    flags[:9000] = True
    flags[11_000:] = False
    mask = torch.tensor(flags, device="cuda")
    wide = torch.tensor([True, False, True], device="cuda")
    widths = [3, 1, 4, 48, 7, 32_768]
    active = [mask] * 5 + [wide]
    s = Setup([n * w for w in widths[:5]] + [3 * widths[5]], bits, active=active, copy=copy, align=align, seed=22)
    for g, act, w in zip(s.g, active, widths):  # rows that are off have no gradient, as in a scene
        g.view(-1, w)[~act] = 0.0
    for _ in range(2):
        s.step_and_check()


def test_tensors_of_all_kinds_in_one_call():
    from gs_b200.training.optimizer import AdamW, Moments8, ParamTensor
    rng = np.random.default_rng(4)
    sizes = [300_001, 250_000, 100_000, 99_999, 5000]
    kinds = [("f32", 0, None), ("f32", 1, "bf16"), ("bf16", 0, None), ("f16", 1, "f16"), ("bf16", 3, None)]
    for bits in (32, 8):
        tensors = []
        for n, (grad, off, copy) in zip(sizes, kinds):
            p = torch.tensor(rng.standard_normal(n + off).astype(np.float32), device="cuda")[off:]
            g = torch.tensor(rng.standard_normal(n + off).astype(np.float32), device="cuda").to(DT[grad])[off:]
            c = torch.zeros(n, dtype=DT[copy], device="cuda") if copy else None
            tensors.append(ParamTensor(p, g, lr=1e-3, weight_decay=0.1, copy=c))
        opt = AdamW(tensors, moment_bits=bits, seed=3)
        p0 = [t.param.cpu().numpy() for t in tensors]
        opt.step()
        for i, (t, (mu, nu), n) in enumerate(zip(tensors, opt.moment_values(), sizes)):
            z = np.zeros(n, np.float32)
            m, v = R.moments(z, z, t.grad.float().cpu().numpy(), 1.0, 0.9, 0.999)
            want, err = R.param(p0[i], m, v, 0, 1e-3, 0.1, 0.9, 0.999, 1e-8)
            assert (np.abs(t.param.cpu().numpy() - want) <= err).all(), i
            if bits == 32:
                np.testing.assert_array_equal(mu.cpu().numpy(), m)
                np.testing.assert_array_equal(nu.cpu().numpy(), v)
            else:
                h = R.noise(3, 0, i, n)
                np.testing.assert_array_equal(mu.cpu().numpy(), R.decode(*R.encode(m, (h % 65536) / 65536.0, True), True))
                np.testing.assert_array_equal(nu.cpu().numpy(),
                                              R.decode(*R.encode(v, (h // 65536) / 65536.0, False), False))
            if t.copy is not None:
                assert torch.equal(t.copy, t.param.to(t.copy.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_subnormal_moments_of_rows_that_are_off_decay(bits):
    """Exponent byte 0 does not mean zero: a block of subnormal moments goes on, whatever the mask."""
    n = 800_000
    off = torch.zeros(n, dtype=torch.bool, device="cuda")
    s = Setup([n], bits, active=[off], seed=23)
    s.g[0].fill_(0.0)
    s.g[0].view(-1)[:300_000] = 2e-39 * torch.arange(300_000, device="cuda").remainder(7)
    s.step_and_check()
    s.g[0].fill_(0.0)
    for _ in range(2):
        s.step_and_check()
    assert float(s.opt.moment_values()[0][0].abs().max()) > 0


def test_extreme_gradients_of_many_elements():
    s = Setup([655_360], 8, seed=24)
    rng = np.random.default_rng(1)
    g = (rng.choice([-1.0, 1.0], 655_360) * 10.0 ** rng.uniform(-44, 18, 655_360)).astype(np.float32)
    g[:1024] = np.float32(1e18)
    g[4096:5000] = 0.0
    s.g[0].copy_(torch.tensor(g))
    for _ in range(2):
        s.step_and_check()
    s.g[0][10_000] = float("nan")
    s.g[0][20_000] = float("-inf")
    s.opt.step()
    mu, nu = (np.isnan(x.cpu().numpy()) for x in s.opt.moments.values())
    bad = np.zeros(655_360, bool)
    for e in (10_000, 20_000):
        bad[e // 128 * 128:e // 128 * 128 + 128] = True
    np.testing.assert_array_equal(mu, bad)
    np.testing.assert_array_equal(nu, bad)
    np.testing.assert_array_equal(np.flatnonzero(np.isnan(s.p[0].cpu().numpy())), [10_000, 20_000])


@pytest.mark.parametrize("bits", [32, 8])
def test_many_elements_skip_and_replay(bits):
    """A skipped step of the large kernels leaves everything; replays equal eager steps."""
    scale = torch.tensor(math.nan, device="cuda")
    s = Setup(BIG, bits, copy="f16", grad_scale=scale)
    before = s.read()
    s.opt.step()
    for x, y in zip(before, s.read()):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)
    assert int(s.opt.count) == 0 and int(s.opt.skipped) == 1
    scale.fill_(1.0)
    t = Setup(BIG, bits, copy="f16")
    graph = torch.cuda.CUDAGraph()
    s.opt.step()
    t.opt.step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        t.opt.step()
    for _ in range(2):
        s.opt.step()
        graph.replay()
    for x, y in zip(s.read(), t.read()):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)
    assert int(t.opt.count) == 3


def test_no_tensors_is_a_step():
    import ctypes
    from gs_b200 import _lib
    state = torch.zeros(4, dtype=torch.int32, device="cuda")
    cfg = _lib.GsAdamwConfig(b1=0.9, b2=0.999, eps=1e-8, moment_bits=8, seed=0)
    out = torch.zeros(4, device="cuda")
    ws = torch.empty(_lib.lib().gs_grad_norm_workspace_bytes(0), dtype=torch.uint8, device="cuda")
    _lib.call("gs_adamw_step", None, 0, ctypes.byref(cfg), None, _lib.ptr(state), _lib.stream(state.device))
    _lib.call("gs_grad_norm", None, 0, 1.0, None, _lib.ptr(out), _lib.ptr(ws), ws.numel(), _lib.stream(state.device))
    assert state.tolist() == [1, 0, 0, 0] and out[:2].tolist() == [0.0, 1.0]


def test_far_elements_and_rows():
    """32-bit moments, row mask and norm past 2^31 elements."""
    from gs_b200.training.optimizer import AdamW, GradNorm, ParamTensor
    w = 32_768
    rows = (1 << 31) // w + 3
    p = torch.zeros((rows, w), device="cuda")
    g = torch.zeros((rows, w), dtype=torch.bfloat16, device="cuda")
    mask = torch.ones(rows, dtype=torch.bool, device="cuda")
    mask[-2] = False
    rng = np.random.default_rng(0)
    last = torch.tensor(rng.standard_normal((3, w)).astype(np.float32)).cuda()
    g[-3:] = last
    g[0, 0] = 2.0
    arrays = [g[-3:].float().cpu().numpy(), np.float32([2.0])]
    np.testing.assert_allclose(GradNorm([g])().cpu().numpy()[0], R.grad_norm(arrays)[0], rtol=2.0 ** -23)
    opt = AdamW([ParamTensor(p, g, lr=1e-2, active=mask)])
    opt.step()
    (mu, nu), = opt.moment_values()
    z = np.zeros(3 * w, np.float32)
    m, v = R.moments(z, z, arrays[0].reshape(-1), 1.0, 0.9, 0.999)
    want, err = R.param(z, m, v, 0, 1e-2, 0.0, 0.9, 0.999, 1e-8, np.repeat([True, False, True], w))
    assert (np.abs(p[-3:].cpu().numpy().reshape(-1) - want) <= err).all()
    np.testing.assert_array_equal(mu[-3:].cpu().numpy().reshape(-1), m)
    np.testing.assert_array_equal(nu[-3:].cpu().numpy().reshape(-1), v)
    assert float(p[1:1000].abs().max()) == 0.0 and abs(float(p[0, 0]) + 1e-2) < 1e-6
    del p, g, opt, mu, nu
    torch.cuda.empty_cache()


def test_plans_on_threads_and_streams():
    """Plans of their own on two host threads and two streams, eager and as graphs, end as they do one after the other."""
    import threading

    def run(seed, steps):
        s = Setup([150_001, 700, 33], 8 if seed % 2 else 32, seed=seed, max_grad_norm=0.5)
        for _ in range(steps):
            s.opt.step()
        return s

    want = [run(seed, 40) for seed in (1, 2)]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[seed] = run(seed, 40)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 -- shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(seed,)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    both = [run(seed, 1) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in both], []
    for s in both:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            s.opt.step()
    for _ in range(39):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, (got[1], got[2]), both):
        for x, y, z in zip(a.read(), b.read(), c.read()):
            for i in range(4):
                np.testing.assert_array_equal(x[i], y[i])
                np.testing.assert_array_equal(x[i], z[i])
