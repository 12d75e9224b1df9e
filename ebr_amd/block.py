"""Fused pointwise work of the energy network's blocks on gfx950 (kernels ``ebr_amd/csrc/ebr_block.hip``, C ABI
``include/ebr_block.h``): ``rms_norm`` over the last dimension and the SwiGLU activation ``silu(gate) * up``, each
differentiable twice, as the graded latent descent needs (the energy's gradient is taken with ``create_graph`` and the
training loss differentiates it again).

- ``rms_norm(x, eps)``      reference models/layers.py:37-42
- ``swiglu(gate_up)``       reference models/layers.py:74-84 (``gate, up = gate_up.chunk(2, -1)``; ``silu(gate) * up``)
- ``group_norm(x, groups, weight, bias, eps, activation)``   over a board's cells, channels last, with its activation
  (kernels ``ebr_amd/csrc/ebr_groupnorm.hip``)

Ops (``torch.ops.ebr_fused.*``, HIP device only; a missing library raises): ``block_rmsnorm``, ``block_rmsnorm_bwd``,
``block_rmsnorm_bwd2``, ``block_swiglu``, ``block_swiglu_bwd``, ``block_swiglu_bwd2``, ``block_groupnorm``,
``block_groupnorm_bwd``, ``block_groupnorm_bwd2``. Autograd: each op's backward
is the next op, so the functions are differentiable to second order; the second backward is not itself
differentiable. The arithmetic is fp32 (fp64 for fp64 tensors), each output rounded once to the dtype where eager
autograd chains several rounded kernels, so 16-bit results differ from eager by rounding only.
"""

# No ``from __future__ import annotations``: custom_op schema inference needs real type objects.
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ebr_amd import _capi, _host
from ebr_amd.fused_attn.loader import hip_library
from ebr_amd.fused_attn.ops import _DTYPE_CODE, _stream

Tensor = torch.Tensor


def _code(t: Tensor) -> int:
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"fused block: unsupported dtype {t.dtype}")
    return code


def _c(t: Tensor) -> Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _rows(x: Tensor) -> Tuple[int, int]:
    if x.dim() < 1:
        raise ValueError(f"fused block: expected a tensor with a last dim, got {tuple(x.shape)}")
    return x.numel() // max(1, x.shape[-1]), x.shape[-1]


def _like(t: Tensor, shape, ref: Tensor, name: str) -> None:
    """An operand the kernels index by ``ref``'s rows (the C ABI takes only ``ref``'s sizes)."""
    if tuple(t.shape) != tuple(shape) or t.device != ref.device:
        raise ValueError(f"fused block: {name} is {tuple(t.shape)} on {t.device}, expected {tuple(shape)} on "
                         f"{ref.device}")


def _half(gu: Tensor) -> int:
    if gu.dim() < 1 or gu.shape[-1] % 2:
        raise ValueError(f"fused block: swiglu needs an even last dim, got {tuple(gu.shape)}")
    return gu.shape[-1] // 2


# ---------------------------------------------------------------------------------------------------------------------
# rms_norm
# ---------------------------------------------------------------------------------------------------------------------


@torch.library.custom_op("ebr_fused::block_rmsnorm", mutates_args=(), device_types="cuda")
def rmsnorm_op(x: Tensor, eps: float) -> Tensor:
    lib = hip_library()
    x = _c(x)
    rows, C = _rows(x)
    y = torch.empty_like(x)
    if y.numel() == 0:
        return y
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_rmsnorm(_code(x), rows, C, eps, x.data_ptr(), y.data_ptr(), _stream(x))
    _capi.check(rc, "ebr_block_rmsnorm")
    return y


@rmsnorm_op.register_fake
def _(x, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("ebr_fused::block_rmsnorm_bwd", mutates_args=(), device_types="cuda")
def rmsnorm_bwd_op(x: Tensor, dy: Tensor, eps: float) -> Tensor:
    lib = hip_library()
    _like(dy, x.shape, x, "dy")
    x, dy = _c(x), _c(dy.to(x.dtype))
    rows, C = _rows(x)
    dx = torch.empty_like(x)
    if dx.numel() == 0:
        return dx
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_rmsnorm_bwd(_code(x), rows, C, eps, x.data_ptr(), dy.data_ptr(), dx.data_ptr(), _stream(x))
    _capi.check(rc, "ebr_block_rmsnorm_bwd")
    return dx


@rmsnorm_bwd_op.register_fake
def _(x, dy, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("ebr_fused::block_rmsnorm_bwd2", mutates_args=(), device_types="cuda")
def rmsnorm_bwd2_op(x: Tensor, dy: Tensor, c: Tensor, eps: float) -> Tuple[Tensor, Tensor]:
    lib = hip_library()
    _like(dy, x.shape, x, "dy")
    _like(c, x.shape, x, "c")
    x, dy, c = _c(x), _c(dy.to(x.dtype)), _c(c.to(x.dtype))
    rows, C = _rows(x)
    gx, gdy = torch.empty_like(x), torch.empty_like(x)
    if gx.numel() == 0:
        return gx, gdy
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_rmsnorm_bwd2(
            _code(x), rows, C, eps, x.data_ptr(), dy.data_ptr(), c.data_ptr(), gx.data_ptr(), gdy.data_ptr(),
            _stream(x),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_rmsnorm_bwd2")
    return gx, gdy


@rmsnorm_bwd2_op.register_fake
def _(x, dy, c, eps):
    like = torch.empty_like(x, memory_format=torch.contiguous_format)
    return like, torch.empty_like(like)


class _RmsNormBwd(torch.autograd.Function):
    @staticmethod
    def forward(x, dy, eps):
        return torch.ops.ebr_fused.block_rmsnorm_bwd(x, dy, eps)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, dy, eps = inputs
        ctx.save_for_backward(x, dy)
        ctx.eps = eps

    @staticmethod
    @once_differentiable
    def backward(ctx, c):
        x, dy = ctx.saved_tensors
        gx, gdy = torch.ops.ebr_fused.block_rmsnorm_bwd2(x, dy, c, ctx.eps)
        return gx, gdy, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(x, eps):
        return torch.ops.ebr_fused.block_rmsnorm(x, eps)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, eps = inputs
        ctx.save_for_backward(x)
        ctx.eps = eps

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        return _RmsNormBwd.apply(x, dy, ctx.eps), None


@_host.gradient("rms_norm")
def _rms_norm_grads(x, eps, dy, acc):
    dx = _RmsNormBwd.apply(x, dy, eps)
    return (dx if acc is None else dx + acc,)


@_host.gradient("rms_norm_bwd")
def _rms_norm_bwd_grads(x, dy, eps, c):
    return torch.ops.ebr_fused.block_rmsnorm_bwd2(x, dy, c, eps)


# ---------------------------------------------------------------------------------------------------------------------
# SwiGLU
# ---------------------------------------------------------------------------------------------------------------------


@torch.library.custom_op("ebr_fused::block_swiglu", mutates_args=(), device_types="cuda")
def swiglu_op(gu: Tensor) -> Tensor:
    lib = hip_library()
    _half(gu)
    gu = _c(gu)
    rows, two_i = _rows(gu)
    y = gu.new_empty((*gu.shape[:-1], two_i // 2))
    if y.numel() == 0:
        return y
    with torch.cuda.device(gu.device):
        rc = lib.ebr_block_swiglu(_code(gu), rows, two_i // 2, gu.data_ptr(), y.data_ptr(), _stream(gu))
    _capi.check(rc, "ebr_block_swiglu")
    return y


@swiglu_op.register_fake
def _(gu):
    return gu.new_empty((*gu.shape[:-1], gu.shape[-1] // 2))


@torch.library.custom_op("ebr_fused::block_swiglu_bwd", mutates_args=(), device_types="cuda")
def swiglu_bwd_op(gu: Tensor, dy: Tensor) -> Tensor:
    lib = hip_library()
    _like(dy, (*gu.shape[:-1], _half(gu)), gu, "dy")
    gu, dy = _c(gu), _c(dy.to(gu.dtype))
    rows, two_i = _rows(gu)
    dgu = torch.empty_like(gu)
    if dgu.numel() == 0:
        return dgu
    with torch.cuda.device(gu.device):
        rc = lib.ebr_block_swiglu_bwd(_code(gu), rows, two_i // 2, gu.data_ptr(), dy.data_ptr(), dgu.data_ptr(),
                                      _stream(gu))
    _capi.check(rc, "ebr_block_swiglu_bwd")
    return dgu


@swiglu_bwd_op.register_fake
def _(gu, dy):
    return torch.empty_like(gu, memory_format=torch.contiguous_format)


@torch.library.custom_op("ebr_fused::block_swiglu_bwd2", mutates_args=(), device_types="cuda")
def swiglu_bwd2_op(gu: Tensor, dy: Tensor, c: Tensor) -> Tuple[Tensor, Tensor]:
    lib = hip_library()
    _like(dy, (*gu.shape[:-1], _half(gu)), gu, "dy")
    _like(c, gu.shape, gu, "c")
    gu, dy, c = _c(gu), _c(dy.to(gu.dtype)), _c(c.to(gu.dtype))
    rows, two_i = _rows(gu)
    ggu, gdy = torch.empty_like(gu), torch.empty_like(dy)
    if ggu.numel() == 0:
        return ggu, gdy
    with torch.cuda.device(gu.device):
        rc = lib.ebr_block_swiglu_bwd2(
            _code(gu), rows, two_i // 2, gu.data_ptr(), dy.data_ptr(), c.data_ptr(), ggu.data_ptr(), gdy.data_ptr(),
            _stream(gu),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_swiglu_bwd2")
    return ggu, gdy


@swiglu_bwd2_op.register_fake
def _(gu, dy, c):
    return torch.empty_like(gu, memory_format=torch.contiguous_format), torch.empty_like(
        dy, memory_format=torch.contiguous_format
    )


class _SwiGLUBwd(torch.autograd.Function):
    @staticmethod
    def forward(gu, dy):
        return torch.ops.ebr_fused.block_swiglu_bwd(gu, dy)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs)

    @staticmethod
    @once_differentiable
    def backward(ctx, c):
        gu, dy = ctx.saved_tensors
        return torch.ops.ebr_fused.block_swiglu_bwd2(gu, dy, c)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(gu):
        return torch.ops.ebr_fused.block_swiglu(gu)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(inputs[0])

    @staticmethod
    def backward(ctx, dy):
        (gu,) = ctx.saved_tensors
        return _SwiGLUBwd.apply(gu, dy)


@_host.gradient("swiglu")
def _swiglu_grads(gu, dy, acc):
    dgu = _SwiGLUBwd.apply(gu, dy)
    return (dgu if acc is None else dgu + acc,)


@_host.gradient("swiglu_bwd")
def _swiglu_bwd_grads(gu, dy, c):
    return torch.ops.ebr_fused.block_swiglu_bwd2(gu, dy, c)


# ---------------------------------------------------------------------------------------------------------------------
# Group norm
# ---------------------------------------------------------------------------------------------------------------------

ACTIVATIONS = {None: 0, "silu": 1}  # EBR_ACT_*


def _board(x: Tensor, groups: int) -> Tuple[int, int, int]:
    """B, L and C of a channels-last tensor [B, ..., C]."""
    if x.dim() < 2:
        raise ValueError(f"fused block: group_norm needs [B, ..., C], got {tuple(x.shape)}")
    B, C = x.shape[0], x.shape[-1]
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"fused block: {C} channels do not split into {groups} groups")
    return B, x.numel() // max(1, B * C), C


def _acc(x: Tensor) -> torch.dtype:
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _param(p: Optional[Tensor], x: Tensor, name: str) -> Optional[Tensor]:
    """A weight or bias [C] as the kernels read it: contiguous, of the accumulation type."""
    if p is None:
        return None
    if tuple(p.shape) != (x.shape[-1],) or p.device != x.device:
        raise ValueError(f"fused block: {name} is {tuple(p.shape)} on {p.device}, expected ({x.shape[-1]},) on {x.device}")
    if p.dtype not in _DTYPE_CODE:
        raise TypeError(f"fused block: unsupported dtype {p.dtype} of {name}")
    return _c(p.to(_acc(x)))


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _norm_scratch(x: Tensor, order: int, B: int, L: int, C: int, groups: int) -> Tensor:
    n = hip_library().ebr_block_groupnorm_scratch(_code(x), order, B, L, C, groups)
    if n < 0:
        _capi.check(2, "ebr_block_groupnorm")
    return torch.empty((n,), device=x.device, dtype=torch.uint8)


@torch.library.custom_op("ebr_fused::block_groupnorm", mutates_args=(), device_types="cuda")
def groupnorm_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float,
                 act: int) -> Tuple[Tensor, Tensor]:
    """(y, stats [B, groups, 2]: each group's mean and 1 / sqrt(variance + eps))."""
    lib = hip_library()
    code, (B, L, C) = _code(x), _board(x, groups)
    x = _c(x)
    w, b = _param(weight, x, "weight"), _param(bias, x, "bias")
    y = torch.empty_like(x)
    stats = torch.empty((B, groups, 2), device=x.device, dtype=_acc(x))
    if y.numel() == 0:
        return y, stats.zero_()
    scratch = _norm_scratch(x, 0, B, L, C, groups)
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_groupnorm(code, act, B, L, C, groups, eps, x.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(),
                                     stats.data_ptr(), scratch.data_ptr(), _stream(x))
    _capi.check(rc, "ebr_block_groupnorm")
    return y, stats


@groupnorm_op.register_fake
def _(x, weight, bias, groups, eps, act):
    return (torch.empty_like(x, memory_format=torch.contiguous_format),
            x.new_empty((x.shape[0], groups, 2), dtype=_acc(x)))


def _check_stats(stats: Tensor, x: Tensor, groups: int) -> Tensor:
    _like(stats, (x.shape[0], groups, 2), x, "stats")
    if stats.dtype != _acc(x):
        raise TypeError(f"fused block: stats are {stats.dtype}, expected {_acc(x)}")
    return _c(stats)


@torch.library.custom_op("ebr_fused::block_groupnorm_bwd", mutates_args=(), device_types="cuda")
def groupnorm_bwd_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, dy: Tensor, groups: int,
                     act: int, params: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """(dx, dw, db); the latter of the accumulation type, and empty without ``params``."""
    lib = hip_library()
    code, (B, L, C) = _code(x), _board(x, groups)
    _like(dy, x.shape, x, "dy")
    stats = _check_stats(stats, x, groups)
    x, dy = _c(x), _c(dy.to(x.dtype))
    w, b = _param(weight, x, "weight"), _param(bias, x, "bias")
    dx = torch.empty_like(x)
    dw, db = (torch.empty((C if params else 0,), device=x.device, dtype=_acc(x)) for _ in range(2))
    if dx.numel() == 0:
        return dx, dw.zero_(), db.zero_()
    scratch = _norm_scratch(x, 1, B, L, C, groups)
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_groupnorm_bwd(
            code, act, B, L, C, groups, x.data_ptr(), _ptr(w), _ptr(b), stats.data_ptr(), dy.data_ptr(), dx.data_ptr(),
            dw.data_ptr() if params else 0, db.data_ptr() if params else 0, scratch.data_ptr(), _stream(x),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_groupnorm_bwd")
    return dx, dw, db


@groupnorm_bwd_op.register_fake
def _(x, weight, bias, stats, dy, groups, act, params):
    dw = x.new_empty((x.shape[-1] if params else 0,), dtype=_acc(x))
    return torch.empty_like(x, memory_format=torch.contiguous_format), dw, torch.empty_like(dw)


@torch.library.custom_op("ebr_fused::block_groupnorm_bwd2", mutates_args=(), device_types="cuda")
def groupnorm_bwd2_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, dy: Tensor, u: Tensor,
                      uw: Optional[Tensor], ub: Optional[Tensor], groups: int, act: int,
                      params: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """(gx, gdy, gw, gb): the gradients of <u, dx> + <uw, dw> + <ub, db>; gw and gb of the accumulation type, and empty
    without ``params``."""
    lib = hip_library()
    code, (B, L, C) = _code(x), _board(x, groups)
    _like(dy, x.shape, x, "dy")
    _like(u, x.shape, x, "u")
    stats = _check_stats(stats, x, groups)
    x, dy, u = _c(x), _c(dy.to(x.dtype)), _c(u.to(x.dtype))
    w, b = _param(weight, x, "weight"), _param(bias, x, "bias")
    uw, ub = _param(uw, x, "uw"), _param(ub, x, "ub")
    gx, gdy = torch.empty_like(x), torch.empty_like(x)
    gw, gb = (torch.empty((C if params else 0,), device=x.device, dtype=_acc(x)) for _ in range(2))
    if gx.numel() == 0:
        return gx, gdy, gw.zero_(), gb.zero_()
    scratch = _norm_scratch(x, 2, B, L, C, groups)
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_groupnorm_bwd2(
            code, act, B, L, C, groups, x.data_ptr(), _ptr(w), _ptr(b), stats.data_ptr(), dy.data_ptr(), u.data_ptr(),
            _ptr(uw), _ptr(ub), gx.data_ptr(), gdy.data_ptr(), gw.data_ptr() if params else 0,
            gb.data_ptr() if params else 0, scratch.data_ptr(), _stream(x),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_groupnorm_bwd2")
    return gx, gdy, gw, gb


@groupnorm_bwd2_op.register_fake
def _(x, weight, bias, stats, dy, u, uw, ub, groups, act, params):
    gx = torch.empty_like(x, memory_format=torch.contiguous_format)
    gw = x.new_empty((x.shape[-1] if params else 0,), dtype=_acc(x))
    return gx, torch.empty_like(gx), gw, torch.empty_like(gw)


def _wants_params(ctx, w: Optional[Tensor], b: Optional[Tensor]) -> bool:
    """Whether this pass uses the gradient of the weight or bias, the inputs after x: the descent's gradients for x alone
    leave theirs out. (A node lists its next functions for tensors only.)"""
    at = 1
    for i, p in ((1, w), (2, b)):
        if p is None:
            continue
        node, at = ctx.next_functions[at][0], at + 1
        if not ctx.needs_input_grad[i] or node is None:
            continue
        if node.name().endswith("AccumulateGrad") or torch._C._will_engine_execute_node(node):
            return True
    return False


def _as(t: Tensor, p: Optional[Tensor]) -> Optional[Tensor]:
    return None if p is None else t.to(p.dtype)


class _GroupNormBwd2(torch.autograd.Function):
    """A node of its own, so that a third derivative is an error: without it the gradients would pass for constants."""

    @staticmethod
    def forward(x, w, b, stats, dy, u, uw, ub, groups, act, params):
        gx, gdy, gw, gb = torch.ops.ebr_fused.block_groupnorm_bwd2(x, w, b, stats, dy, u, uw, ub, groups, act, params)
        return gx, gdy, _as(gw, w) if params else None, _as(gb, b) if params else None

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("trying to differentiate twice a function that was marked with @once_differentiable: "
                           "group_norm has no third derivative")


class _GroupNormBwd(torch.autograd.Function):
    @staticmethod
    def forward(x, w, b, stats, dy, groups, act, params):
        dx, dw, db = torch.ops.ebr_fused.block_groupnorm_bwd(x, w, b, stats, dy, groups, act, params)
        return dx, _as(dw, w) if params else None, _as(db, b) if params else None

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, b, stats, dy, ctx.groups, ctx.act, _ = inputs
        ctx.save_for_backward(x, w, b, stats, dy)
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, u, uw, ub):
        x, w, b, stats, dy = ctx.saved_tensors
        if u is None and uw is None and ub is None:
            return (None,) * 8
        params = _wants_params(ctx, w, b)
        u = torch.zeros_like(x) if u is None else u
        gx, gdy, gw, gb = _GroupNormBwd2.apply(x, w, b, stats, dy, u, uw, ub, ctx.groups, ctx.act, params)
        return gx, gw, gb, None, gdy, None, None, None


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(x, w, b, groups, eps, act):
        return torch.ops.ebr_fused.block_groupnorm(x, w, b, groups, eps, act)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, b, ctx.groups, _, ctx.act = inputs
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(x, w, b, output[1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, dy, _stats):
        x, w, b, stats = ctx.saved_tensors
        if dy is None:
            return (None,) * 6
        params = _wants_params(ctx, w, b)
        dx, dw, db = _GroupNormBwd.apply(x, w, b, stats, dy, ctx.groups, ctx.act, params)
        return dx, dw, db, None, None, None


@_host.gradient("group_norm")
def _group_norm_grads(x, w, b, stats, groups, act, params, dy):
    return _GroupNormBwd.apply(x, w, b, stats, dy, groups, act, params)


@_host.gradient("group_norm_bwd")
def _group_norm_bwd_grads(x, w, b, stats, dy, groups, act, params, u, uw, ub):
    u = torch.zeros_like(x) if u is None else u
    gx, gdy, gw, gb = _GroupNormBwd2.apply(x, w, b, stats, dy, u, uw, ub, groups, act, params)
    return gx, gw, gb, None, gdy


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               activation: Optional[str] = None) -> Tensor:
    """f(weight * h + bias) for a channels-last tensor [B, ..., C]: h is x less its mean and over the square root of its
    variance plus ``eps``, both taken for each sample and each group of C / groups neighbouring channels, over all cells.
    ``activation``: None, or "silu". ``weight`` and ``bias``: [C], or None (1 and 0). Statistics and sums are fp32 or wider
    (a group's squares about its mean have to stay in that range), outputs rounded once to x's dtype; differentiable twice,
    for x, weight and bias, and a third derivative raises."""
    host = _host.module()
    y = None if host is None or activation not in ACTIVATIONS else host.group_norm(x, groups, weight, bias, eps,
                                                                                   ACTIVATIONS[activation])
    if y is not None:
        return y
    if activation not in ACTIVATIONS:
        raise ValueError(f"fused block: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    _code(x), _board(x, groups)
    for p, name in ((weight, "weight"), (bias, "bias")):
        if p is not None and (tuple(p.shape) != (x.shape[-1],) or p.device != x.device):
            raise ValueError(f"fused block: {name} is {tuple(p.shape)} on {p.device}, expected ({x.shape[-1]},) on {x.device}")
    if not eps >= 0:
        raise ValueError(f"fused block: eps must not be negative, got {eps}")
    return _GroupNorm.apply(x, weight, bias, groups, float(eps), ACTIVATIONS[activation])[0]


def rms_norm(x: Tensor, eps: float) -> Tensor:
    """Unit RMS over the last dim (statistics in fp32), differentiable twice."""
    host = _host.module()
    y = None if host is None else host.rms_norm(x, eps)
    if y is not None:
        return y
    return _RmsNorm.apply(x, eps)


def add_rms_norm(x: Tensor, r: Tensor, eps: float) -> Tensor:
    """``rms_norm(x + r, eps)``: the residual sum rounded to the dtype, then its norm, in one kernel on the native path."""
    host = None if torch.compiler.is_compiling() else _host.module()
    y = None if host is None else host.add_rms_norm(x, r, eps)
    return rms_norm(x + r, eps) if y is None else y


def swiglu(gate_up: Tensor) -> Tensor:
    """silu(gate) * up of the two halves of the last dim, differentiable twice."""
    host = _host.module()
    y = None if host is None else host.swiglu(gate_up)
    if y is not None:
        return y
    _half(gate_up)
    return _SwiGLU.apply(gate_up)


rms_norm = torch._dynamo.allow_in_graph(rms_norm)
swiglu = torch._dynamo.allow_in_graph(swiglu)
group_norm = torch._dynamo.allow_in_graph(group_norm)

__all__ = ["add_rms_norm", "group_norm", "rms_norm", "swiglu"]
