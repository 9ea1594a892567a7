"""AdamW over many tensors at once, its moments in 32 bits or in 8, and the
global gradient norm that clips it (gs_adamw_step, gs_grad_norm,
gs_moments8_*; no reference counterpart: the reference's optimizers are
optax.adam over fixed groups, train.py:129-156).

AdamW and GradNorm are plans: built once over the caller's tensors, whose
memory they read and write in place on every call, so a step is one library
call whatever the number of tensors. The step count, the clip factor and the
decision to skip a step whose gradient is not finite live on the device, so a
captured CUDA graph replays successive steps. Calls are ordered on the current
stream of the tensors' device; steps of one plan must not overlap.

    opt = AdamW([ParamTensor(w, w_grad, lr=1e-3, weight_decay=0.1),
                 ParamTensor(b, b_grad, lr=1e-3)], moment_bits=8, max_grad_norm=1.0)
    ...                     # fill w_grad, b_grad
    opt.step()
"""
from __future__ import annotations

import ctypes
import dataclasses
import math
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from gs_b200 import _lib

_TYPES = {torch.float32: _lib.GS_TYPE_F32, torch.bfloat16: _lib.GS_TYPE_BF16, torch.float16: _lib.GS_TYPE_F16}
BLOCK = _lib.GS_ADAMW_BLOCK


@dataclasses.dataclass
class ParamTensor:
    """One tensor of an AdamW plan.

    param is float32; grad has its number of elements in float32, bfloat16 or
    float16. The learning rate of the step that follows c others is
    lr * lr_decay_rate ** (c / lr_transition_steps) (optax.exponential_decay;
    with a rate of 0, lr for the first step and 0 from then on).
    active (bool or uint8, one flag per row of param's first dimension): rows
    whose flag is 0 keep their parameter. copy (bfloat16 or float16) receives
    the new parameter, rounded.
    """
    param: torch.Tensor
    grad: torch.Tensor
    lr: float
    weight_decay: float = 0.0
    lr_decay_rate: float = 1.0
    lr_transition_steps: float = 1.0
    active: Optional[torch.Tensor] = None
    copy: Optional[torch.Tensor] = None


def _check_cuda(name: str, t: torch.Tensor, dtypes, device=None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: libgsb200 needs CUDA tensors")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype}, expected one of {[str(d) for d in dtypes]}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: libgsb200 needs contiguous tensors")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")


def _check_scalar(name: str, t: Optional[torch.Tensor], device) -> None:
    if t is None:
        return
    _check_cuda(name, t, (torch.float32,), device)
    if t.numel() != 1:
        raise ValueError(f"{name}: expected one value")


def _check_overlap(written: Sequence[Tuple[str, torch.Tensor]], read: Sequence[Tuple[str, torch.Tensor]]) -> None:
    """Raise if memory that is written is also another tensor's."""
    spans = []
    for is_written, group in ((True, written), (False, read)):
        for name, t in group:
            if t is not None and t.numel() > 0:
                spans.append((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), is_written, name))
    spans.sort(key=lambda x: x[0])
    end_w, name_w, end_r, name_r = 0, "", 0, ""  # furthest end of a written / a read span so far
    for a, b, is_written, name in spans:
        if a < end_w:
            raise ValueError(f"{name} shares memory with {name_w}, which the step writes")
        if is_written and a < end_r:
            raise ValueError(f"{name}, which the step writes, shares memory with {name_r}")
        if is_written and b > end_w:
            end_w, name_w = b, name
        if not is_written and b > end_r:
            end_r, name_r = b, name


def _stream(device: torch.device) -> int:
    """The current stream's handle, without building torch's Stream object (2 us of a 5 us call)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw is not None else _lib.stream(device)


class _Plan:
    """The device, and the plan's own tensors kept from reuse on the streams that use them."""

    def __init__(self, device: torch.device):
        self.device = device
        self._owned: List[torch.Tensor] = []
        self._streams = {_stream(device)}

    def _own(self, *tensors: torch.Tensor) -> None:
        self._owned += tensors

    def _call(self, fn: str, *args) -> None:
        """One library call on the current stream of the plan's device."""
        st = _stream(self.device)
        if st not in self._streams and not torch.cuda.is_current_stream_capturing():
            s = torch.cuda.current_stream(self.device)
            for t in self._owned:
                t.record_stream(s)
            self._streams.add(st)
        if torch.cuda.current_device() == self.device.index:
            _lib.call(fn, *args, st)
        else:
            with torch.cuda.device(self.device):
                _lib.call(fn, *args, st)


class GradNorm(_Plan):
    """Global norm of a list of gradients and the factor that clips it.

    A call computes norm = u * sqrt(sum of squares) (u: the one value of
    `unscale`, or 1) and scale = u * min(1, max_norm / norm), NaN if the norm
    is not finite, and returns them as a float32 device tensor [norm, scale]
    (the plan's own buffer). `scale`, a view of the second, is a grad_scale for
    AdamW.
    """

    def __init__(self, grads: Sequence[torch.Tensor], max_norm: float = math.inf,
                 unscale: Optional[torch.Tensor] = None):
        grads = [g.detach() if isinstance(g, torch.Tensor) else g for g in grads]
        if not grads:
            raise ValueError("no gradients")
        if not float(max_norm) > 0.0:
            raise ValueError("max_norm must be positive")
        for i, g in enumerate(grads):
            _check_cuda(f"grads[{i}]", g, _TYPES, grads[0].device)
        super().__init__(grads[0].device)
        _check_scalar("unscale", unscale, self.device)
        self.grads, self.unscale, self.max_norm = grads, unscale, float(max_norm)
        self._table = (_lib.GsGradTensor * len(grads))()
        for d, g in zip(self._table, grads):
            d.grad, d.count, d.type = g.data_ptr(), g.numel(), _TYPES[g.dtype]
        self._buf = torch.zeros(4, dtype=torch.float32, device=self.device)  # GsGradNorm
        self._ws = torch.empty(_lib.lib().gs_grad_norm_workspace_bytes(len(grads)), dtype=torch.uint8,
                               device=self.device)
        self._own(self._buf, self._ws)
        self.out = self._buf[:2]
        self.norm, self.scale = self._buf[0], self._buf[1]
        self._args = (self._table, len(self._table), self.max_norm, _lib.ptr(self.unscale), self._buf.data_ptr(),
                      self._ws.data_ptr(), self._ws.numel())

    def __call__(self) -> torch.Tensor:
        self._call("gs_grad_norm", *self._args)
        return self.out


class Moments8(_Plan):
    """Both Adam moments of a list of tensors as 8-bit codes with one exponent
    byte for each 128 elements (the format of gs_adamw_step), in flat buffers
    in which every tensor starts at a multiple of 128 elements. `sizes` are the
    tensors' element counts; the buffers are created (all moments 0) or given.
    """

    def __init__(self, sizes: Sequence[int], device=None, mu: Optional[torch.Tensor] = None,
                 nu: Optional[torch.Tensor] = None, mu_exp: Optional[torch.Tensor] = None,
                 nu_exp: Optional[torch.Tensor] = None):
        self.sizes = [int(s) for s in sizes]
        self.starts, total = [], 0
        for s in self.sizes:
            if s < 0:
                raise ValueError("negative size")
            self.starts.append(total)
            total += -(-s // BLOCK) * BLOCK
        self.total = total
        given = [mu, nu, mu_exp, nu_exp]
        if all(t is None for t in given):
            if device is None:
                raise ValueError("a device or the four buffers are needed")
            given = [torch.zeros(n, dtype=torch.uint8, device=device)
                     for n in (total, total, total // BLOCK, total // BLOCK)]
        for name, t, n in zip(("mu", "nu", "mu_exp", "nu_exp"), given, (total, total, total // BLOCK, total // BLOCK)):
            if t is None:
                raise ValueError(f"{name} is missing")
            _check_cuda(name, t, (torch.uint8,), given[0].device)
            if t.numel() != n:
                raise ValueError(f"{name}: {t.numel()} bytes, expected {n}")
        for name, t in zip(("mu", "nu"), given):
            if t.data_ptr() % 4:
                raise ValueError(f"{name}: not 4-byte aligned")
        self.mu, self.nu, self.mu_exp, self.nu_exp = given
        super().__init__(self.mu.device)
        self._own(*given)
        self._codes = tuple(t.data_ptr() for t in given)

    def values(self, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """(mu, nu) that the codes stand for, in the layout of the flat buffers
        (0 between the tensors), in float32 or bfloat16 (exact in both)."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("dtype must be float32 or bfloat16")
        mu, nu = (torch.empty(self.total, dtype=dtype, device=self.device) for _ in range(2))
        self._call("gs_moments8_decode", *self._codes, self.total, _TYPES[dtype], mu.data_ptr(), nu.data_ptr())
        return mu, nu

    def set_values(self, mu: torch.Tensor, nu: torch.Tensor) -> None:
        """Round float32 values in the layout of values() to the nearest codes
        (the values of a block's codes are kept exactly; nu >= 0)."""
        for name, t in (("mu", mu), ("nu", nu)):
            _check_cuda(name, t, (torch.float32,), self.device)
            if t.numel() != self.total:
                raise ValueError(f"{name}: {t.numel()} values, expected {self.total}")
        self._call("gs_moments8_encode", mu.data_ptr(), nu.data_ptr(), self.total, *self._codes)

    def split(self, flat: torch.Tensor) -> List[torch.Tensor]:
        """The tensors' parts of a buffer in the layout of values()."""
        return [flat[a:a + s] for a, s in zip(self.starts, self.sizes)]


class AdamW(_Plan):
    """AdamW over `tensors` (see ParamTensor); step() updates parameters,
    moments and copies in place.

    moment_bits: 32 or 8. moments: the moments to use, a list of (mu, nu)
    float32 tensors (32 bits) or a Moments8 (8 bits); created as zeros if not
    given. grad_scale: one float32 value on the device that multiplies every
    gradient (GradNorm.scale, or 1 / loss scale); while it is not finite, steps
    change nothing and are counted in `skipped`. max_grad_norm: clip by the
    global norm (optax.clip_by_global_norm) of the gradients, which step() then
    computes first (`norm`, a GradNorm, with grad_scale as its unscale). seed:
    of the 8-bit moments' stochastic rounding. count: steps already taken, or
    state: the int32 device tensor [steps taken, 0, steps skipped, 0] to use.
    """

    def __init__(self, tensors: Sequence[ParamTensor], b1: float = 0.9, b2: float = 0.999, eps: float = 1e-8,
                 moment_bits: Optional[int] = None,
                 moments: Union[None, Moments8, Sequence[Tuple[torch.Tensor, torch.Tensor]]] = None,
                 grad_scale: Optional[torch.Tensor] = None, max_grad_norm: Optional[float] = None, seed: int = 0,
                 count: int = 0, state: Optional[torch.Tensor] = None):
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("no tensors")
        _check_cuda("tensors[0].param", self.tensors[0].param, (torch.float32,))
        super().__init__(self.tensors[0].param.device)
        if moment_bits is None:
            moment_bits = 8 if isinstance(moments, Moments8) else 32
        if moment_bits not in (8, 32):
            raise ValueError("moment_bits must be 8 or 32")
        if moments is not None and isinstance(moments, Moments8) != (moment_bits == 8):
            raise ValueError("moments do not have moment_bits bits")
        if not 0 <= int(count) < 2 ** 31 - 1:
            raise ValueError("count out of range")
        self.moment_bits = moment_bits
        sizes = [t.param.numel() for t in self.tensors]
        if moments is None:
            if moment_bits == 8:
                moments = Moments8(sizes, self.device)
            else:
                moments = [(torch.zeros_like(t.param.detach()), torch.zeros_like(t.param.detach()))
                           for t in self.tensors]
        self.moments = moments
        self._check(sizes)
        if state is None:
            state = torch.zeros(4, dtype=torch.int32, device=self.device)
            state[0] = int(count)
        else:
            _check_cuda("state", state, (torch.int32,), self.device)
            if state.numel() != 4:
                raise ValueError("state: expected four int32")
        self._state = state
        self.count, self.skipped = self._state[0:1], self._state[2:3]
        self.norm = None
        if max_grad_norm is not None:
            self.norm = GradNorm([t.grad for t in self.tensors], max_grad_norm, grad_scale)
            grad_scale = self.norm.scale
        _check_scalar("grad_scale", grad_scale, self.device)
        self.grad_scale = grad_scale
        self._config = _lib.GsAdamwConfig()
        self._config.b1, self._config.b2, self._config.eps = float(b1), float(b2), float(eps)
        self._config.moment_bits, self._config.seed = moment_bits, int(seed) & 0xFFFFFFFF
        self._table = (_lib.GsAdamwTensor * len(self.tensors))()
        self._fill()
        self._bumped = self._written()
        self._args = (self._table, len(self._table), ctypes.byref(self._config), _lib.ptr(self.grad_scale),
                      self._state.data_ptr())
        self._own(self._state, *self._moment_buffers())

    def _moment_buffers(self) -> List[torch.Tensor]:
        m = self.moments
        if self.moment_bits == 8:
            return [m.mu, m.nu, m.mu_exp, m.nu_exp]
        return [t for pair in m for t in pair]

    def _written(self) -> List[torch.Tensor]:
        out = [t.param for t in self.tensors] + [t.copy for t in self.tensors if t.copy is not None]
        return [t for t in out if not t.is_inference()]

    def _check(self, sizes: List[int]) -> None:
        dev = self.device
        if self.moment_bits == 8:
            if self.moments.sizes != sizes:
                raise ValueError("moments: sizes differ from the tensors'")
            if self.moments.device != dev:
                raise ValueError(f"moments: on {self.moments.device}, expected {dev}")
        elif len(self.moments) != len(sizes):
            raise ValueError(f"moments: {len(self.moments)} pairs, expected {len(sizes)}")
        written, read = [], []
        for i, t in enumerate(self.tensors):
            name = f"tensors[{i}]"
            _check_cuda(f"{name}.param", t.param, (torch.float32,), dev)
            _check_cuda(f"{name}.grad", t.grad, _TYPES, dev)
            n = t.param.numel()
            if t.grad.numel() != n:
                raise ValueError(f"{name}.grad: {t.grad.numel()} elements, expected {n}")
            written.append((f"{name}.param", t.param))
            read.append((f"{name}.grad", t.grad))
            if t.copy is not None:
                _check_cuda(f"{name}.copy", t.copy, (torch.bfloat16, torch.float16), dev)
                if t.copy.numel() != n:
                    raise ValueError(f"{name}.copy: {t.copy.numel()} elements, expected {n}")
                written.append((f"{name}.copy", t.copy))
            if t.active is not None:
                _check_cuda(f"{name}.active", t.active, (torch.bool, torch.uint8), dev)
                rows = t.param.shape[0] if t.param.dim() else 1
                if t.active.numel() != rows:
                    raise ValueError(f"{name}.active: {t.active.numel()} flags, expected {rows}")
                if rows and n // rows > 32768:
                    raise ValueError(f"{name}.active: rows of {n // rows} elements, at most 32768")
                read.append((f"{name}.active", t.active))
            if self.moment_bits == 32:
                for key, m in zip(("mu", "nu"), self.moments[i]):
                    _check_cuda(f"moments[{i}].{key}", m, (torch.float32,), dev)
                    if m.numel() != n:
                        raise ValueError(f"moments[{i}].{key}: {m.numel()} elements, expected {n}")
                    written.append((f"moments[{i}].{key}", m))
        if self.moment_bits == 8:
            written += [("moments", t) for t in self._moment_buffers()]
        _check_overlap(written, read)

    def _fill(self) -> None:
        for i, (d, t) in enumerate(zip(self._table, self.tensors)):
            n = t.param.numel()
            d.param, d.grad, d.count = t.param.data_ptr(), t.grad.data_ptr(), n
            d.grad_type = _TYPES[t.grad.dtype]
            d.width = 1
            if t.active is not None:
                d.active = t.active.data_ptr()
                d.width = max(1, n // max(1, t.active.numel()))
            if t.copy is not None:
                d.copy, d.copy_type = t.copy.data_ptr(), _TYPES[t.copy.dtype]
            if self.moment_bits == 8:
                m = self.moments
                a = m.starts[i]
                d.mu, d.nu = m.mu.data_ptr() + a, m.nu.data_ptr() + a
                d.mu_exp, d.nu_exp = m.mu_exp.data_ptr() + a // BLOCK, m.nu_exp.data_ptr() + a // BLOCK
            else:
                d.mu, d.nu = (x.data_ptr() for x in self.moments[i])
        self.refresh()

    def refresh(self) -> None:
        """Take over learning rates and weight decays changed in `tensors`
        (not into graphs captured before)."""
        for d, t in zip(self._table, self.tensors):
            d.lr_init, d.weight_decay = float(t.lr), float(t.weight_decay)
            d.decay_rate, d.transition_steps = float(t.lr_decay_rate), float(t.lr_transition_steps)
            if d.decay_rate == 0.0 and d.transition_steps > 0.0:
                # 0 ^ (c / steps) is 1 at c = 0 and 0 behind it, as is 2^-126 ^ (1024 c) in float32: the library
                # takes the logarithm of the rate
                d.decay_rate, d.transition_steps = 2.0 ** -126, 2.0 ** -10

    def step(self) -> None:
        """One step on the gradients as they are."""
        self.clip()
        self.update()

    def clip(self) -> Optional[torch.Tensor]:
        """The first half of step(): the gradients' norm, with max_grad_norm.
        Returns grad_scale, the device value while which is not finite
        update() changes nothing (None: nothing is skipped)."""
        if self.norm is not None:
            self.norm()
        return self.grad_scale

    def update(self) -> None:
        """The second half of step(): parameters, moments and copies."""
        self._call("gs_adamw_step", *self._args)
        # the library writes through raw pointers: tell autograd, as an in-place operation does
        torch.autograd.graph.increment_version(self._bumped)

    def moment_values(self) -> List[Tuple[torch.Tensor, torch.Tensor]]:
        """(mu, nu) of every tensor in float32 (8 bits: decoded copies; 32 bits: the buffers)."""
        if self.moment_bits == 32:
            return [tuple(pair) for pair in self.moments]
        mu, nu = (self.moments.split(x) for x in self.moments.values())
        return [(m.view(t.param.shape), v.view(t.param.shape)) for m, v, t in zip(mu, nu, self.tensors)]

    def state_dict(self) -> Dict:
        """Copies of the step count, the steps skipped and the moments, with the tensors' sizes."""
        return {"state": self._state.clone(), "moment_bits": self.moment_bits,
                "sizes": [t.param.numel() for t in self.tensors],
                "moments": [t.clone() for t in self._moment_buffers()]}

    def load_state_dict(self, state: Dict) -> None:
        """Take over what state_dict() of a plan over tensors of the same sizes returned."""
        buffers = self._moment_buffers()
        if state["moment_bits"] != self.moment_bits:
            raise ValueError("moment_bits differ")
        # 8-bit moments lie in flat buffers, whose lengths do not tell the tensors' order (a state saved without its
        # sizes is taken by the lengths)
        sizes = [t.param.numel() for t in self.tensors]
        if (state.get("sizes", sizes) != sizes
                or [t.numel() for t in state["moments"]] != [t.numel() for t in buffers]):
            raise ValueError("sizes of the moments differ")
        self._state.copy_(state["state"])
        for t, s in zip(buffers, state["moments"]):
            t.copy_(s.view(t.shape))
