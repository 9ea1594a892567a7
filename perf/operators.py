"""Cases and plain forms of the optimizer's operators: the global gradient norm with its clip factor, and the
AdamW step over many tensors with its moments in 32 bits or in 8.

A case is a set of tensors held as views of flat buffers, as the trainers hold them. Layout "scene": the five
parameter groups of N Gaussian slots with K spherical-harmonic coefficients, back to back, under an active mask.
Layout "list": tensors of ragged sizes, each starting at a multiple of 128 elements. With own = False, run()
computes with elementary torch operations; with own = True it calls gs_b200.training.optimizer.

The 8-bit moments are blocks of 128 elements from each tensor's start, with one exponent byte F a block and moment:
  F = (bits(largest magnitude) + 0xfffff) >> 23, 255 where the block is not finite (its values read as NaN)
  mu: sign bit and 7 bits (4 exponent, 3 mantissa), nu: 8 bits (5 exponent, 3 mantissa), with gradual underflow:
  code = min((bits(|x| * 2^(127 - F) * 2^-s) + noise) >> 20, largest code), s = 112 (mu) or 96 (nu); a nu > 0 is
  never stored as 0. noise holds 16 random bits, shifted left by 4, of a hash of (seed, step, tensor, block, element).
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 128
GOLDEN = 0x9E3779B9
M32 = 0xFFFFFFFF
B1, B2, EPS = 0.9, 0.999, 1e-8
MAX_NORM = 1.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "": 0}


def listed():
    return [
        # a toy scene's gradient: the launch counts
        {"name": "norm, 1k slots", "op": "norm", "layout": "scene", "n": 1000, "k": 16, "active": 1.0, "grad": "f32"},
        # many tensors of mixed sizes, gradients from a 16-bit backward pass
        {"name": "norm, 197 bf16 tensors", "op": "norm", "layout": "list", "tensors": 197, "elements": 50_000_000, "grad": "bf16"},
        # the gradient of the densification benchmark's scene (3M Gaussians in 4M slots, degree 3)
        {"name": "norm, 4M slots", "op": "norm", "layout": "scene", "n": 4_000_000, "k": 16, "active": 0.75, "grad": "f32"},
        # a small preview scene of degree 1 colours: the launch counts
        {"name": "adamw32, 1k slots", "op": "adamw32", "layout": "scene", "n": 1000, "k": 4, "active": 1.0, "grad": "f32"},
        # the flagship training benchmark: 100k Gaussians in 200k slots
        {"name": "adamw32, 200k slots", "op": "adamw32", "layout": "scene", "n": 200_000, "k": 16, "active": 0.5, "grad": "f32"},
        # the large training benchmark: 1M Gaussians at degree 3
        {"name": "adamw32, 1M slots", "op": "adamw32", "layout": "scene", "n": 1_000_000, "k": 16, "active": 1.0, "grad": "f32"},
        # an odd capacity, so the groups start off 16-byte boundaries
        {"name": "adamw32, 333331 slots", "op": "adamw32", "layout": "scene", "n": 333_331, "k": 9, "active": 0.9, "grad": "f32"},
        # many tensors: 16-bit gradients, 32-bit masters, a 16-bit copy for the next forward pass
        {"name": "adamw32, 197 tensors", "op": "adamw32", "layout": "list", "tensors": 197, "elements": 50_000_000, "grad": "bf16", "copy": "bf16"},
        # a toy scene with 8-bit moments
        {"name": "adamw8, 1k slots", "op": "adamw8", "layout": "scene", "n": 1000, "k": 16, "active": 1.0, "grad": "f32"},
        # the flagship training benchmark with 8-bit moments
        {"name": "adamw8, 200k slots", "op": "adamw8", "layout": "scene", "n": 200_000, "k": 16, "active": 0.5, "grad": "f32"},
        # many tensors with loss-scaled fp16 gradients
        {"name": "adamw8, 197 tensors", "op": "adamw8", "layout": "list", "tensors": 197, "elements": 50_000_000, "grad": "f16", "copy": "f16"},
        # the densification benchmark's scene, where the moments' memory counts
        {"name": "adamw8, 4M slots", "op": "adamw8", "layout": "scene", "n": 4_000_000, "k": 16, "active": 0.75, "grad": "f32"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "adamw32", "adamw8"])
    if rng.random() < 0.6:
        case = {"op": op, "layout": "scene", "n": _log_uniform(rng, 300, 1_500_000 if op == "adamw32" else 4_000_000),
                "k": rng.choice([1, 4, 9, 16]), "active": round(rng.uniform(0.05, 1.0), 3), "grad": "f32"}
    else:
        elements = _log_uniform(rng, 5000, 80_000_000 if op == "adamw32" else 200_000_000)
        case = {"op": op, "layout": "list", "tensors": min(_log_uniform(rng, 1, 700), max(1, elements // 200)),
                "elements": elements, "grad": rng.choice(["f32", "bf16", "f16"])}
        if op != "norm" and rng.random() < 0.5:
            case["copy"] = rng.choice(["bf16", "f16"])
    return case


def _sizes(case):
    """The tensors' sizes: the five groups of a scene, or ragged ones (a third of them short vectors)."""
    if case["layout"] == "scene":
        return [case["n"] * w for w in (3, 3, 4, 1, 3 * case["k"])]
    rng = random.Random(case["tensors"] * 7919 + case["elements"])
    weight = [rng.lognormvariate(0.0, 1.5) * (0.001 if rng.random() < 0.33 else 1.0) for _ in range(case["tensors"])]
    total = sum(weight)
    return [max(1, int(case["elements"] * w / total)) for w in weight]


def _up(x):
    return -(-x // BLOCK) * BLOCK


def _starts(sizes, padded):
    out, at = [], 0
    for s in sizes:
        out.append(at)
        at += _up(s) if padded else s
    return out, at


def work(case):
    e = sum(_sizes(case))
    blocks = sum(_up(s) // BLOCK for s in _sizes(case))
    mask = case["n"] if case["layout"] == "scene" else 0
    g = BYTES[case["grad"]]
    if case["op"] == "norm":
        return {"bytes": e * g, "flops": 2 * e}
    if case["op"] == "adamw32":
        return {"bytes": e * (24 + g + BYTES[case.get("copy", "")]) + mask, "flops": 14 * e}
    # the codes in and out, and the values that they stand for, in 16 bits
    return {"bytes": e * (12 + g + BYTES[case.get("copy", "")] + 4) + 4 * blocks + mask, "flops": 14 * e}


def _segments(state, flat):
    return [flat[a:a + s] for a, s in zip(state["starts"], state["sizes"])]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=dev)

    sizes = _sizes(case)
    scene = case["layout"] == "scene"
    starts, total = _starts(sizes, not scene)
    state = {"case": dict(case), "sizes": sizes, "starts": starts, "total": total, "seed": seed & 0x7FFFFFFF}
    params, grads, mus, nus = (torch.zeros(total, device=dev) for _ in range(4))
    if scene:
        n = case["n"]
        active = torch.arange(n, device=dev) < max(1, round(case["active"] * n))
        seen = active & (uniform(n) < 0.6)  # a view's gradient is zero where it does not see the Gaussian
        once = active & (uniform(n) < 0.95)  # slots that no view has seen yet have zero moments
        row = torch.exp(1.5 * normal(n))  # gradients differ by orders of magnitude between Gaussians
        scale = [2e-4, 5e-5, 2e-5, 1e-4, 1e-5]
        widths = [3, 3, 4, 1, 3 * case["k"]]
        for i, (a, s, w) in enumerate(zip(starts, sizes, widths)):
            r = (scale[i] * row)[:, None]
            params[a:a + s] = normal(n, w).reshape(-1)
            grads[a:a + s] = (normal(n, w) * r * seen[:, None]).reshape(-1)
            mus[a:a + s] = (0.3 * normal(n, w) * r * once[:, None]).reshape(-1)
            nus[a:a + s] = ((0.05 + 0.5 * uniform(n, w)) * r * r * once[:, None]).reshape(-1)
        state["active"] = active
        state["lr"] = [0.00016 * 3.0, 0.005, 0.001, 0.05, 0.0025]
        state["decay"] = [0.01, 1.0, 1.0, 1.0, 1.0]
        state["wd"] = [0.0, 0.01, 0.0, 0.02, 0.001]
        state["widths"] = widths
    else:
        state["active"] = None
        state["lr"] = [3e-4 * (1 + i % 3) for i in range(len(sizes))]
        state["decay"] = [0.1] * len(sizes)
        state["wd"] = [0.1 if s > 4096 else 0.0 for s in sizes]
        state["widths"] = [1] * len(sizes)
        level = torch.exp(normal(len(sizes))).cpu().tolist()
        for i, (a, s) in enumerate(zip(starts, sizes)):
            r = 1e-3 * level[i]
            params[a:a + s] = 0.05 * normal(s)
            grads[a:a + s] = normal(s) * r
            mus[a:a + s] = 0.3 * r * normal(s)
            nus[a:a + s] = (0.05 + 0.5 * uniform(s)) * (r * r)
    state["steps"] = 30000.0
    state["p"], state["g"] = params, grads.to(TYPES[case["grad"]])
    if case["op"] == "norm":
        # a loss scale of 1024 is taken off again
        state["unscale"] = torch.full((), 2.0 ** -10, device=dev) if case["grad"] == "f16" else None
        if state["unscale"] is not None:
            state["g"] = (grads * 1024.0).to(torch.float16)
    else:
        state["scale"] = (0.25 + 0.5 * uniform(1))[0].clone()  # the clip factor, on the device
        if case["grad"] == "f16":
            state["g"] = (grads * 1024.0).to(torch.float16)
            state["scale"] = state["scale"] * 2.0 ** -10
        state["count0"] = 1 + seed % 5000
        state["count"] = torch.full((1,), state["count0"], dtype=torch.int32, device=dev)
        state["copy"] = torch.zeros(total, dtype=TYPES[case["copy"]], device=dev) if case.get("copy") else None
    if case["op"] == "adamw32":
        state["mu"], state["nu"] = mus, nus
    if case["op"] == "adamw8":
        pstarts, ptotal = _starts(sizes, True)
        pm, pv = torch.zeros(ptotal, device=dev), torch.zeros(ptotal, device=dev)
        for a, b, s in zip(starts, pstarts, sizes):
            pm[b:b + s] = mus[a:a + s]
            pv[b:b + s] = nus[a:a + s]
        half = torch.full((), 1 << 19, dtype=torch.int32, device=dev)
        state["mu8"], state["mu_exp"] = _encode(pm, half, True)
        state["nu8"], state["nu_exp"] = _encode(pv, half, False)
        state["pstarts"], state["ptotal"] = pstarts, ptotal
    if own:
        state["plan"] = _plan(state)
    return state


def _plan(state):
    """What a user's program keeps: the plan over its parameters and gradients."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "jax-gs_b200") not in sys.path:
        sys.path.insert(0, os.path.join(root, "jax-gs_b200"))
    from gs_b200.training.optimizer import AdamW, GradNorm, Moments8, ParamTensor
    case, sizes = state["case"], state["sizes"]
    grads = _segments(state, state["g"])
    if case["op"] == "norm":
        return GradNorm(grads, max_norm=MAX_NORM, unscale=state["unscale"])
    tensors = []
    copies = _segments(state, state["copy"]) if state["copy"] is not None else [None] * len(sizes)
    for i, (p, g, c) in enumerate(zip(_segments(state, state["p"]), grads, copies)):
        w = state["widths"][i]
        if state["active"] is not None:
            p, g = p.view(-1, w), g.view(-1, w)
        tensors.append(ParamTensor(p, g, lr=state["lr"][i], weight_decay=state["wd"][i], lr_decay_rate=state["decay"][i],
                                   lr_transition_steps=state["steps"], active=state["active"], copy=c))
    if case["op"] == "adamw32":
        moments = list(zip(_segments(state, state["mu"]), _segments(state, state["nu"])))
    else:
        moments = Moments8(sizes, mu=state["mu8"], nu=state["nu8"], mu_exp=state["mu_exp"], nu_exp=state["nu_exp"])
    return AdamW(tensors, b1=B1, b2=B2, eps=EPS, moments=moments, grad_scale=state["scale"], seed=state["seed"],
                 count=state["count0"])


# ---- plain forms -------------------------------------------------------------------------------------------


def _pow2(field):
    """2^(field - 127) as float32, for biased exponents 0 (2^-127, subnormal) to 254."""
    bits = torch.where(field == 0, 0x00400000, field << 23)
    return bits.to(torch.int32).view(torch.float32)


def _encode(x, noise, signed):
    """Codes and exponent bytes of a flat float32 tensor of whole blocks; noise in [0, 2^20)."""
    a = x.abs().view(-1, BLOCK)
    bits = a.contiguous().view(torch.int32)
    top = bits.amax(1).to(torch.int64)
    field = ((top + 0xFFFFF) >> 23).clamp(max=255)
    down = _pow2((254 - field).clamp(min=0))[:, None]
    y = a * down * (2.0 ** (-112 if signed else -96))
    code = (y.view(torch.int32) + noise.view(-1, BLOCK if noise.dim() else 1)) >> 20
    code = code.clamp(max=127 if signed else 255)
    if signed:
        code = code | torch.where(x.view(-1, BLOCK).view(torch.int32) < 0, 128, 0)
    else:
        code = torch.where((a > 0) & (code == 0), 1, code)
    code = torch.where(field[:, None] == 255, 0, code)
    return code.to(torch.uint8).view(-1), field.to(torch.uint8)


def _decode(code, field, signed):
    """Float32 values of codes."""
    c = code.view(-1, BLOCK).to(torch.int32)
    up = _pow2(field.to(torch.int64).clamp(max=254))[:, None]
    mag = (((c & 127) if signed else c) << 20).view(torch.float32) * (2.0 ** (112 if signed else 96)) * up
    if signed:
        mag = torch.where(c > 127, -mag, mag)
    return torch.where(field[:, None] == 255, math.nan, mag).view(-1)


def _mix(x):
    """A 32-bit integer hash (two multiplications, three shifts) on int64 tensors."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & M32
    return x ^ (x >> 16)


def _adamw(p, m, v, lr, wd, active, count, b1, b2, eps):
    """The parameter's update from the new moments."""
    t = count.double() + 1.0
    inv1 = (1.0 / (1.0 - b1 ** t)).float()
    inv2 = (1.0 / (1.0 - b2 ** t)).float()
    new = p - lr * ((m * inv1) / (torch.sqrt(v * inv2) + eps) + wd * p)
    return new if active is None else torch.where(active, new, p)


def _per_element(state, starts, total):
    """Tensor index, offset in the tensor and whether it is one of its elements, for every place of a flat buffer."""
    dev = state["p"].device
    start = torch.tensor(starts, device=dev)
    span = torch.tensor(starts[1:] + [total], device=dev) - start
    tid = torch.repeat_interleave(torch.arange(len(starts), device=dev), span)
    off = torch.arange(total, device=dev) - start[tid]
    return tid, off, off < torch.tensor(state["sizes"], device=dev)[tid]


def _rates(state, tid):
    dev = state["p"].device
    c = state["count"].double()
    lr = torch.tensor(state["lr"], dtype=torch.float64, device=dev)
    lr = lr * torch.tensor(state["decay"], dtype=torch.float64, device=dev) ** (c / state["steps"])
    wd = torch.tensor(state["wd"], dtype=torch.float64, device=dev)
    return lr.float()[tid], wd.float()[tid]


def _rows_active(state, tid, off, valid):
    if state["active"] is None:
        return None
    width = torch.tensor(state["widths"], device=off.device)[tid]
    return state["active"][torch.where(valid, off // width, 0)]


def _moments(m, v, g):
    return m * B1 + g * (1.0 - B1), v * B2 + (g * g) * (1.0 - B2)


def run(state):
    op = state["case"]["op"]
    if own:
        plan = state["plan"]
        if op == "norm":
            return plan()
        plan.step()
        if op == "adamw32":
            out = {"p": state["p"], "mu": state["mu"], "nu": state["nu"], "count": plan.count}
        else:
            mu, nu = plan.moments.values(torch.bfloat16)
            out = {"p": state["p"], "mu": mu, "nu": nu, "count": plan.count}
    elif op == "norm":
        g = state["g"].double()
        norm = torch.sqrt((g * g).sum())
        norm = norm if state["unscale"] is None else norm * state["unscale"].double()
        scale = torch.where(norm < MAX_NORM, 1.0, MAX_NORM / norm)  # the factor that the step applies to the gradient
        scale = scale if state["unscale"] is None else scale * state["unscale"].double()
        return torch.stack([norm, torch.where(torch.isfinite(norm), scale, math.nan)]).float()
    elif op == "adamw32":
        tid, off, valid = _per_element(state, state["starts"], state["total"])
        lr, wd = _rates(state, tid)
        active = _rows_active(state, tid, off, valid)
        g = state["g"].float() * state["scale"]
        m, v = _moments(state["mu"], state["nu"], g)
        state["p"].copy_(_adamw(state["p"], m, v, lr, wd, active, state["count"], B1, B2, EPS))
        state["mu"].copy_(m)
        state["nu"].copy_(v)
        out = {"p": state["p"], "mu": state["mu"], "nu": state["nu"]}
    else:
        tid, off, valid = _per_element(state, state["pstarts"], state["ptotal"])
        where = torch.where(valid, torch.tensor(state["starts"], device=off.device)[tid] + off, 0)
        lr, wd = _rates(state, tid)
        active = _rows_active(state, tid, off, valid)
        p = torch.where(valid, state["p"][where], 0.0)
        g = torch.where(valid, state["g"][where].float() * state["scale"], 0.0)
        m, v = _moments(_decode(state["mu8"], state["mu_exp"], True), _decode(state["nu8"], state["nu_exp"], False), g)
        new = _adamw(p, m, v, lr, wd, active, state["count"], B1, B2, EPS)
        state["p"][where[valid]] = new[valid]
        key = _mix((state["seed"] + GOLDEN * state["count"].long()) & M32)
        key = _mix((key + GOLDEN * tid) & M32)
        key = _mix(key ^ (off // BLOCK))
        noise = _mix((key + GOLDEN * (off % BLOCK)) & M32)
        low, high = ((noise & 0xFFFF) << 4).to(torch.int32), ((noise >> 16) << 4).to(torch.int32)
        state["mu8"], state["mu_exp"] = _encode(m, low, True)
        state["nu8"], state["nu_exp"] = _encode(v, high, False)
        out = {"p": state["p"], "mu": _decode(state["mu8"], state["mu_exp"], True).to(torch.bfloat16),
               "nu": _decode(state["nu8"], state["nu_exp"], False).to(torch.bfloat16)}
    if not own:
        state["count"] += 1
        if state["copy"] is not None:
            state["copy"].copy_(state["p"])
        out["count"] = state["count"]
    if state["copy"] is not None:
        out["copy"] = state["copy"]
    return out


# ---- the definition in 64 bits -----------------------------------------------------------------------------


def _value(code, field, signed):
    """The value of a code in 64 bits, from its exponent and mantissa digits."""
    c = code.long()
    mag = c % 128 if signed else c
    exponent, digits = mag // 8, (mag % 8).double() / 8
    top = 15 if signed else 31
    x = torch.where(exponent == 0, digits * 2.0, digits + 1.0)
    x = torch.ldexp(x, exponent - top)
    x = torch.ldexp(x, torch.repeat_interleave(field.long() - 127, BLOCK)[:c.numel()])
    return torch.where(c >= 128, -x, x) if signed else x


def _rounded(x, u, signed):
    """x (whole blocks, float64) rounded down or up to the block's format, up where the random u in [0, 1) says so."""
    top, most = (15, 1.875) if signed else (31, 1.875)
    a = x.abs()
    big = a.view(-1, BLOCK).amax(1)
    mant, exp = torch.frexp(big.clamp(min=2.0 ** -127))  # big = mant 2^exp, mant in [0.5, 1)
    exp = exp.long() - 1
    exp = torch.where(2 * mant > most, exp + 1, exp)
    shift = torch.repeat_interleave(exp, BLOCK)
    a = torch.ldexp(a, -shift)
    own_exp = (torch.frexp(a.clamp(min=2.0 ** -300))[1].long() - 1).clamp(min=1 - top)
    unit = torch.ldexp(torch.ones_like(a), own_exp - 3)
    q = (torch.floor(a / unit + u) * unit).clamp(max=most)
    if not signed:
        q = torch.where((a > 0) & (q == 0), 2.0 ** (1 - top - 3), q)
    q = torch.ldexp(q, shift)
    return torch.where(x < 0, -q, q)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = sum((part.double() ** 2).sum() for part in s["g"].split(1 << 24))
        norm = total.sqrt() * (1.0 if s["unscale"] is None else float(s["unscale"]))
        factor = torch.clamp(MAX_NORM / norm, max=1.0) * (1.0 if s["unscale"] is None else float(s["unscale"]))
        return torch.stack([norm, factor])
    eight = case["op"] == "adamw8"
    dev = s["p"].device
    t = s["count0"] + 1
    out = {"p": s["p"].double(), "mu": [], "nu": []}
    if eight:
        m_all, v_all = _value(s["mu8"], s["mu_exp"], True), _value(s["nu8"], s["nu_exp"], False)
    else:
        m_all, v_all = s["mu"].double(), s["nu"].double()
    out["mu"], out["nu"] = m_all, v_all
    for i, (a, size) in enumerate(zip(s["starts"], s["sizes"])):
        b = s["pstarts"][i] if eight else a
        g = s["g"][a:a + size].double() * s["scale"].double()
        m = B1 * m_all[b:b + size] + (1 - B1) * g
        v = B2 * v_all[b:b + size] + (1 - B2) * g ** 2
        lr = s["lr"][i] * s["decay"][i] ** (s["count0"] / s["steps"])
        p = s["p"][a:a + size].double()
        step = lr * (m / (1 - B1 ** t) / ((v / (1 - B2 ** t)).sqrt() + EPS) + s["wd"][i] * p)
        if s["active"] is not None:
            step = step * s["active"].repeat_interleave(s["widths"][i])
        out["p"][a:a + size] = p - step
        if eight:
            e = torch.arange(_up(size), device=dev)
            key = _mix(torch.full((1,), (s["seed"] + GOLDEN * s["count0"]) % 2 ** 32, dtype=torch.int64, device=dev))
            key = _mix((key + GOLDEN * i) % 2 ** 32)
            h = _mix((_mix(key ^ (e // BLOCK)) + GOLDEN * (e % BLOCK)) % 2 ** 32)
            pad = torch.zeros(_up(size) - size, dtype=torch.float64, device=dev)
            m = _rounded(torch.cat([m, pad]), (h % 65536).double() / 65536, True)[:size]
            v = _rounded(torch.cat([v, pad]), (h // 65536).double() / 65536, False)[:size]
        m_all[b:b + size] = m
        v_all[b:b + size] = v
    if s["copy"] is not None:
        out["copy"] = torch.zeros(s["total"], dtype=torch.float64, device=dev)
        for a, size in zip(s["starts"], s["sizes"]):
            out["copy"][a:a + size] = out["p"][a:a + size]
    out["count"] = None
    return out
