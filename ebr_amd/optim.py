"""The optimizer's step on gfx950 (kernels ``ebr_amd/csrc/ebr_optim.hip``, C ABI ``include/ebr_optim.h``):

- ``AdamW(params, lr, betas, eps, weight_decay, max_norm, state_bits)``   a ``torch.optim.Optimizer``
- ``adamw_(params, grads, exp_avgs, exp_avg_sqs, steps, ...)``   one step over lists of tensors
- ``grad_norm(grads)``   the gradients' global norm

All tensors of a step go together, in a launch for each 48 of them, with moments in fp32 or as 8-bit numbers of blocks of 256
(``state_bits``). Clipping by the global norm (the reference clips too, utils/optim.py:122-244) happens inside the step, on the
device: nothing waits for the norm. Step counts are the device's, so a captured step counts on at every replay.

Ops (``torch.ops.ebr_fused.*``, HIP device only; a missing library raises): ``grad_norm``, ``adamw``.
"""

# No ``from __future__ import annotations``: custom_op schema inference needs real type objects.
import bisect
import ctypes
import math
from collections import OrderedDict
from typing import Any, Callable, Dict, List, Optional, Sequence, Tuple, Union

import torch

from ebr_amd import _capi, _host
from ebr_amd.fused_attn.loader import hip_library
from ebr_amd.fused_attn.ops import _DTYPE_CODE, _stream

Tensor = torch.Tensor

BLOCK = 256  # elements of one scale
STATE8 = torch.float8_e4m3fn
_HALF = (torch.bfloat16, torch.float16)


def _scratch(n: int, like: Tensor) -> Tensor:
    if n < 0:
        raise ValueError("optim: sizes out of range")
    return torch.empty((n,), device=like.device, dtype=torch.uint8)


@torch.library.custom_op("ebr_fused::grad_norm", mutates_args=(), device_types="cuda")
def grad_norm_op(grads: Sequence[Tensor]) -> Tuple[Tensor, Tensor]:
    """The norm in fp64 and in fp32."""
    lib = hip_library()
    _check_grads(grads)
    like = grads[0]
    grads = [g.contiguous() for g in grads]
    norm, single = (torch.empty((), device=like.device, dtype=d) for d in (torch.float64, torch.float32))
    table = (_capi.OptimGrad * len(grads))(*((g.data_ptr(), g.numel(), _DTYPE_CODE[g.dtype], 0) for g in grads))
    scratch = _scratch(lib.ebr_block_grad_norm_scratch(len(grads), ctypes.addressof(table)), like)
    with torch.cuda.device(like.device):
        rc = lib.ebr_block_grad_norm(len(grads), ctypes.addressof(table), norm.data_ptr(), single.data_ptr(),
                                     scratch.data_ptr(), _stream(like))
    _capi.check(rc, "ebr_block_grad_norm")
    return norm, single


@grad_norm_op.register_fake
def _(grads):
    return grads[0].new_empty((), dtype=torch.float64), grads[0].new_empty((), dtype=torch.float32)


@torch.library.custom_op("ebr_fused::adamw", device_types="cuda",
                         mutates_args=("params", "exp_avgs", "exp_avg_sqs", "steps", "scales"))
def adamw_op(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
             steps: Sequence[Tensor], scales: Sequence[Tensor], lr: float, lr_dev: Optional[Tensor], beta1: float,
             beta2: float, eps: float, weight_decay: float, norm: Optional[Tensor], max_norm: float) -> None:
    """A step; scales: the first moments' and then the roots' in turn for each parameter, or none."""
    lib = hip_library()
    _check_step(params, grads, exp_avgs, exp_avg_sqs, steps, list(zip(scales[::2], scales[1::2])) or None, lr_dev)
    grads = [g.contiguous() for g in grads]
    kinds: Dict[Any, List[int]] = {}
    for i, (p, g) in enumerate(zip(params, grads)):
        kinds.setdefault((p.dtype, g.dtype), []).append(i)
    for (pt, gt), at in kinds.items():
        table = (_capi.OptimTensor * len(at))(*(
            (params[i].data_ptr(), grads[i].data_ptr(), exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(),
             scales[2 * i].data_ptr() if scales else 0, scales[2 * i + 1].data_ptr() if scales else 0, steps[i].data_ptr(),
             params[i].numel()) for i in at))  # fmt: skip
        like = params[at[0]]
        scratch = _scratch(lib.ebr_block_adamw_scratch(len(at)), like)
        with torch.cuda.device(like.device):
            rc = lib.ebr_block_adamw(
                _DTYPE_CODE[pt], _DTYPE_CODE[gt], 8 if scales else 32, len(at), ctypes.addressof(table), lr,
                0 if lr_dev is None else lr_dev.data_ptr(), beta1, beta2, eps, weight_decay,
                0 if norm is None else norm.data_ptr(), max_norm, scratch.data_ptr(), _stream(like),
            )  # fmt: skip
        _capi.check(rc, "ebr_block_adamw")


def _check_grads(grads: Sequence[Tensor]) -> None:
    if len(grads) == 0:
        raise ValueError("optim: no gradients")
    for g in grads:
        if g.layout != torch.strided:
            raise TypeError(f"optim: gradients must be dense, got {g.layout}")
        if g.dtype not in _DTYPE_CODE:
            raise TypeError(f"optim: unsupported dtype {g.dtype} of a gradient")
        if g.device != grads[0].device:
            raise ValueError(f"optim: gradients are on {grads[0].device} and {g.device}: one device a step")


def _check_step(params, grads, exp_avgs, exp_avg_sqs, steps, scales, lr) -> None:
    n = len(params)
    lists = (("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs), ("steps", steps), ("scales", scales))
    for name, ts in lists:
        if ts is not None and len(ts) != n:
            raise ValueError(f"optim: {len(ts)} {name} for {n} parameters")
    if n == 0:
        raise ValueError("optim: no parameters")
    _check_grads(grads)
    dev = params[0].device
    if grads[0].device != dev:
        raise ValueError(f"optim: parameters are on {dev}, gradients on {grads[0].device}")
    for k, (p, g, m, v, t) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, steps)):
        if p.dtype not in _DTYPE_CODE or (scales is not None and p.dtype == torch.float64):
            raise TypeError(f"optim: unsupported dtype {p.dtype} of parameter {k}{'' if scales is None else ' with 8-bit moments'}")
        if g.dtype != p.dtype and not (p.dtype == torch.float32 and g.dtype in _HALF):
            raise TypeError(f"optim: parameter {k} is {p.dtype}, its gradient {g.dtype}")
        if g.shape != p.shape:
            raise ValueError(f"optim: parameter {k} is {tuple(p.shape)}, its gradient {tuple(g.shape)}")
        want = STATE8 if scales is not None else torch.float64 if p.dtype == torch.float64 else torch.float32
        held = [("parameter", p, p.dtype, p.numel()), ("exp_avg", m, want, p.numel()), ("exp_avg_sq", v, want, p.numel()),
                ("step", t, torch.int64, 1)]
        if scales is not None:
            held += [("scale", s, torch.float32, -(-p.numel() // BLOCK)) for s in scales[k]]
            if len(scales[k]) != 2:
                raise ValueError(f"optim: scales of parameter {k}: one tensor for each moment")
        for name, x, dtype, numel in held:
            if x.dtype != dtype:
                raise TypeError(f"optim: {name} {k} is {x.dtype}, expected {dtype}")
            if x.numel() != numel or not x.is_contiguous():
                raise ValueError(f"optim: {name} {k} must be {numel} contiguous elements, got {tuple(x.shape)} with strides "
                                 f"{x.stride()}")
            if x.device != dev:
                raise ValueError(f"optim: {name} {k} is on {x.device}, parameter 0 on {dev}: one device a step")
    for name, ts in (("parameter", params), ("step", steps)):
        at = [x.data_ptr() for x in ts if x.numel() > 0]
        if len(set(at)) < len(at):
            raise ValueError(f"optim: the same {name} twice in one step")
    written = [x for ts in (params, exp_avgs, exp_avg_sqs, steps, *(scales or ())) for x in ts if x.numel() > 0]
    ends = sorted(_range(x) for x in written)
    if any(a[1] > b[0] for a, b in zip(ends, ends[1:])):
        raise ValueError("optim: two of the tensors that a step writes share memory")
    read = [g for p, g in zip(params, grads) if g.numel() > 0 and g.is_contiguous() and _range(g) != _range(p)]
    for x in read + ([lr] if isinstance(lr, Tensor) else []):
        start, end = _range(x)
        at = bisect.bisect_left(ends, (end,))
        if at > 0 and ends[at - 1][1] > start:
            raise ValueError("optim: a step writes to a gradient or to its lr")


def _range(x: Tensor) -> Tuple[int, int]:
    """The addresses of a contiguous tensor, the end past its last."""
    return x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()


def _check_numbers(lr, betas, eps, weight_decay, max_norm, device=None) -> None:
    if isinstance(lr, Tensor):
        if lr.numel() != 1 or lr.dtype != torch.float32 or (device is not None and lr.device != device):
            raise ValueError(f"optim: a tensor lr must be one fp32 number on the parameters' device, got {tuple(lr.shape)} "
                             f"{lr.dtype} on {lr.device}")
    elif not (math.isfinite(lr) and lr >= 0):
        raise ValueError(f"optim: lr must be a number from 0 on, got {lr}")
    if not all(0 <= b < 1 for b in betas) or len(betas) != 2:
        raise ValueError(f"optim: betas must be two numbers from 0 to below 1, got {betas}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"optim: eps must be a number from 0 on, got {eps}")
    if not (math.isfinite(weight_decay) and weight_decay >= 0):
        raise ValueError(f"optim: weight_decay must be a number from 0 on, got {weight_decay}")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"optim: max_norm must be above 0, got {max_norm}")


def _check_options(group: Dict[str, Any]) -> None:
    """Refuses options of a group that make AdamW another step than this one."""
    for name in ("amsgrad", "maximize"):
        if group.get(name):
            raise ValueError(f"optim: AdamW has no {name}")
    if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
        raise ValueError("optim: AdamW's weight decay is decoupled from the gradients")


def _check_saved(group: Dict[str, Any]) -> None:
    """Refuses the saved group of another optimizer than this one, ``torch.optim.AdamW``, or an Adam that takes the same steps."""
    missing = {"lr", "betas", "eps", "weight_decay"} - set(group)
    if missing or ("maximize" in group and "amsgrad" not in group):
        raise ValueError(f"optim: a group of another optimizer, with {sorted(group)}")
    _check_options(group)


def _norms(grads: Sequence[Tensor]) -> Tuple[Tensor, Tensor]:
    host = _host.module()
    out = None if host is None else host.grad_norms(grads)
    if out is None:
        _check_grads(grads)
        with torch.no_grad():
            out = torch.ops.ebr_fused.grad_norm(list(grads))
    return out


def grad_norm(grads: Sequence[Tensor]) -> Tensor:
    """The 2-norm of all the gradients together, summed in fp64 in a fixed order: one fp32 number on their device. The
    gradients may be of different dtypes."""
    return _norms(grads)[1]


def _launch(params, grads, exp_avgs, exp_avg_sqs, steps, scales, lr, betas, eps, weight_decay, norm, max_norm) -> None:
    by_tensor = isinstance(lr, Tensor)
    number, lr_dev = (0.0, lr) if by_tensor else (float(lr), None)
    clip = math.inf if max_norm is None else float(max_norm)
    host = _host.module()
    if host is not None and host.adamw(params, grads, exp_avgs, exp_avg_sqs, steps, scales, number, lr_dev, betas[0], betas[1],
                                       eps, weight_decay, norm, clip):
        return
    _check_step(params, grads, exp_avgs, exp_avg_sqs, steps, scales, lr)
    with torch.no_grad():
        torch.ops.ebr_fused.adamw(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), list(steps),
                                  [s for pair in scales or () for s in pair], number, lr_dev, betas[0], betas[1], eps,
                                  weight_decay, norm, clip)


def adamw_(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
           steps: Sequence[Tensor], *, lr: Union[float, Tensor], betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
           weight_decay: float = 1e-2, max_norm: Optional[float] = None,
           scales: Optional[Sequence[Tuple[Tensor, Tensor]]] = None) -> Optional[Tensor]:
    """One AdamW step in place over lists of contiguous tensors on one device, t being a parameter's step count after it:

        g <- g min(1, max_norm / (n + 1e-6)),  n the norm of all ``grads`` together (with ``max_norm``; returned, in fp32)
        m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
        p <- p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    Parameters are fp32, bfloat16, float16 or fp64; gradients of the same dtype, or 16-bit with fp32 parameters. ``exp_avgs``
    and ``exp_avg_sqs`` (m and v) are fp32 (fp64 for fp64), ``steps`` one int64 each. ``lr`` is a number or one fp32 number on
    the device. What a step writes shares no memory with anything else of it, but a gradient may be its own parameter.

    With ``scales``, moments are in 8 bits: ``exp_avgs`` holds m and ``exp_avg_sqs`` the root of v as float8_e4m3fn, and scales[k]
    is a pair of fp32 vectors, a scale for each 256 consecutive elements, that the numbers are multiplied with. They are rounded
    up or down in turn over the steps, in proportion to what lies on either side (``include/ebr_optim.h`` states the rule), so
    that small changes add up."""
    _check_numbers(lr, betas, eps, weight_decay, max_norm, params[0].device if len(params) else None)
    norm, single = (None, None) if max_norm is None else _norms(grads)
    _launch(params, grads, exp_avgs, exp_avg_sqs, steps, scales, lr, betas, eps, weight_decay, norm, max_norm)
    return single


def _dense(t: Tensor) -> bool:
    """Whether t's elements fill its memory from its first to its last, each once."""
    at = 1
    for stride, size in sorted((st, s) for st, s in zip(t.stride(), t.shape) if s > 1):
        if stride != at:
            return False
        at *= size
    return True


def _in_order(t: Tensor, like: Tensor) -> Tensor:
    """The elements of t as a vector in the order that ``like`` (dense) has them in memory; t itself where it can be."""
    if t.is_contiguous() and like.is_contiguous():
        return t
    if t.stride() != like.stride():
        t = torch.empty_like(like, dtype=t.dtype).copy_(t)
    return t.as_strided((t.numel(),), (1,))


class AdamW(torch.optim.Optimizer):
    """AdamW (``adamw_``) with all parameters of a group in one go.

    ``state_bits``: 32, or 8 for moments of a byte each (and 8 bytes for 256 elements). ``max_norm``: the gradients of all
    groups together are clipped to this norm, on one device; ``grad_norm`` then is their norm before that in the last step.
    ``lr`` may be a number or, for steps captured into a graph, one fp32 number on the device. For a capture, allocate the
    state before it with ``init_state``. ``load_state_dict`` takes the moments as they were saved; with 32 bits also those of
    ``torch.optim.AdamW``. ``amsgrad``, ``maximize`` and a weight decay that is part of the gradients, in a group or in a saved
    one, are refused, as is the state of another optimizer."""

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_norm: Optional[float] = None, state_bits: int = 32) -> None:
        _check_numbers(lr, betas, eps, weight_decay, max_norm)
        if state_bits not in (8, 32):
            raise ValueError(f"optim: state_bits must be 8 or 32, got {state_bits}")
        self.max_norm, self.state_bits = max_norm, state_bits
        self.grad_norm: Optional[Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("grad_norm", None)

    def __getstate__(self):
        return super().__getstate__() | dict(max_norm=self.max_norm, state_bits=self.state_bits)

    def _state_of(self, p: Tensor) -> Dict[str, Tensor]:
        st = self.state[p]
        if not st:
            if p.dtype not in _DTYPE_CODE or (self.state_bits == 8 and p.dtype == torch.float64):
                raise TypeError(f"optim: unsupported dtype {p.dtype} of a parameter with {self.state_bits}-bit moments")
            if p.layout != torch.strided or not _dense(p):
                raise ValueError(f"optim: a parameter of {tuple(p.shape)} with strides {p.stride()} does not fill its memory")
            st["step"] = torch.zeros((), device=p.device, dtype=torch.int64)
            kind = STATE8 if self.state_bits == 8 else torch.float64 if p.dtype == torch.float64 else torch.float32
            names = ("exp_avg", "exp_avg_root") if self.state_bits == 8 else ("exp_avg", "exp_avg_sq")
            for name in names:
                st[name] = torch.empty_like(p, dtype=torch.uint8 if self.state_bits == 8 else kind).zero_().view(kind)
                if self.state_bits == 8:
                    st[name + "_scale"] = torch.zeros((-(-p.numel() // BLOCK),), device=p.device, dtype=torch.float32)
        return st

    def init_state(self) -> None:
        """Allocates the state of every parameter that has none, as the first step would."""
        with torch.no_grad():
            for group in self.param_groups:
                for p in group["params"]:
                    self._state_of(p)

    def moments(self, p: Tensor) -> Tuple[Tensor, Tensor]:
        """The first and second moments that a parameter's state stands for, in fp32 (fp64 for fp64), of its shape."""
        st = self._state_of(p)
        if self.state_bits == 32:
            return st["exp_avg"].clone(), st["exp_avg_sq"].clone()
        out = []
        for name in ("exp_avg", "exp_avg_root"):
            scale = st[name + "_scale"].repeat_interleave(BLOCK)[: p.numel()]
            values = _in_order(st[name].view(torch.uint8), p).reshape(-1).view(STATE8).float() * scale
            out.append(torch.empty_like(p, dtype=torch.float32))
            _in_order(out[-1], p).view(-1).copy_(values)
        return out[0], out[1].square_()

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], Any]] = None) -> Any:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(group, [p for p in group["params"] if p.grad is not None]) for group in self.param_groups]
        for _, ps in groups:
            for p in ps:
                if p.grad.layout != torch.strided:
                    raise TypeError(f"optim: gradients must be dense, got {p.grad.layout}")
        norm = None
        if self.max_norm is not None:
            grads = [p.grad for _, ps in groups for p in ps]
            norm, self.grad_norm = _norms(grads) if grads else (None, None)
        for group, ps in groups:
            devices: Dict[torch.device, List[Tensor]] = {}
            for p in ps:
                devices.setdefault(p.device, []).append(p)
            for dev, some in devices.items():
                self._step_on(dev, some, group, norm)
        return loss

    def _step_on(self, dev: torch.device, ps: List[Tensor], group: Dict[str, Any], norm: Optional[Tensor]) -> None:
        _check_numbers(group["lr"], group["betas"], group["eps"], group["weight_decay"], None, dev)
        states = [self._state_of(p) for p in ps]
        flat = [_in_order(p, p) for p in ps]
        grads = [_in_order(p.grad, p) for p in ps]
        first, second, scales = "exp_avg", "exp_avg_sq", None
        if self.state_bits == 8:
            second = "exp_avg_root"
            scales = [(st[first + "_scale"], st[second + "_scale"]) for st in states]
        for st, p in zip(states, ps):
            for name in (first, second):
                if st[name].stride() != p.stride():  # as loaded: in p's order from now on
                    order = torch.empty_like(p, dtype=torch.uint8 if self.state_bits == 8 else st[name].dtype)
                    st[name] = order.copy_(st[name].view(order.dtype)).view(st[name].dtype)
        moments = [[_in_order(st[name], p) for st, p in zip(states, ps)] for name in (first, second)]
        _launch(flat, grads, *moments, [st["step"] for st in states], scales, group["lr"], group["betas"], group["eps"],
                group["weight_decay"], norm, self.max_norm)

    @torch.no_grad()
    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        # hooks run here: torch's turn would be between its copies and the moments as they are kept
        before, after = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        state_dict = state_dict.copy()
        for hook in before.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        names = {"step", "exp_avg", "exp_avg_sq"}
        if self.state_bits == 8:
            names = {"step", "exp_avg", "exp_avg_root", "exp_avg_scale", "exp_avg_root_scale"}
        for st in state_dict["state"].values():
            if set(st) != names:
                raise ValueError(f"optim: the state of a parameter has {sorted(st)}, expected {sorted(names)}")
        for group in state_dict["param_groups"]:
            _check_saved(group)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        ps = [p for group in self.param_groups for p in group["params"]]
        pairs = [(state_dict["state"][i], p) for i, p in zip(ids, ps) if i in state_dict["state"]]
        for st, p in pairs:
            for name in names:
                given = torch.as_tensor(st[name])
                shape = () if name == "step" else (-(-p.numel() // BLOCK),) if name.endswith("_scale") else p.shape
                if given.shape != shape and not (name == "step" and given.numel() == 1):
                    raise ValueError(f"optim: {name} is {tuple(given.shape)}, expected {tuple(shape)}")
                if name in ("exp_avg", "exp_avg_root") and self.state_bits == 8 and given.dtype != STATE8:
                    raise TypeError(f"optim: {name} is {given.dtype}, expected {STATE8}")
        self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = OrderedDict(), OrderedDict()
        try:
            super().load_state_dict(state_dict)
        finally:
            self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = before, after
        for st, p in pairs:
            own = self.state[p]  # torch casts what it loads to the parameter's dtype: the moments have their own
            own.clear()
            for name, fresh in self._state_of(p).items():
                given = torch.as_tensor(st[name])
                if fresh.dtype == STATE8:
                    fresh, given = fresh.view(torch.uint8), given.view(torch.uint8)
                fresh.copy_(given.reshape(fresh.shape))
        for hook in after.values():
            hook(self)


__all__ = ["AdamW", "adamw_", "grad_norm"]
