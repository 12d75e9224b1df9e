"""The two ends of a training step on gfx950 (kernels ``ebr_amd/csrc/ebr_embed.hip`` and ``ebr_distill.hip``, C ABI
``include/ebr_block.h``):

- ``embedding(ids, weight, scale, dtype)``   rows of a table for tokens, scaled and cast, and the table's dense gradient
- ``distill_loss(logits, teacher_logits, teacher_ids, temperature, reduction)``   what the logits lack of a teacher's top
  logits, and its gradient

Ops (``torch.ops.ebr_fused.*``, HIP device only; a missing library raises): ``embed``, ``embed_bwd``, ``distill``,
``distill_bwd``. The arithmetic is fp32 (fp64 for fp64 tensors), each output rounded once; sums are always taken in the
same order, so equal calls give equal bits. The embedding is linear, and differentiable to any order (the gradient of its
gradient is the lookup again); the loss is differentiable once, and a second derivative raises.
"""

# No ``from __future__ import annotations``: custom_op schema inference needs real type objects.
import math
from typing import Optional, Tuple

import torch

from ebr_amd import _capi, _host
from ebr_amd.fused_attn.loader import hip_library
from ebr_amd.fused_attn.ops import _DTYPE_CODE, _stream

Tensor = torch.Tensor

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # EBR_REDUCE_*
MAX_TEACHER_ENTRIES = 1024


def _code(t: Tensor) -> int:
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"tokens: unsupported dtype {t.dtype}")
    return code


def _wide_ids(ids: Tensor, name: str) -> int:
    """1 for int64 tokens, 0 for int32."""
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens: {name} must be int64 or int32, got {ids.dtype}")
    return int(ids.dtype == torch.int64)


def _c(t: Tensor) -> Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _scratch(n: int, like: Tensor) -> Tensor:
    return torch.empty((n,), device=like.device, dtype=torch.uint8)


# ---------------------------------------------------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------------------------------------------------


def _check_embed(ids: Tensor, weight_dtype: torch.dtype, dtype: torch.dtype) -> None:
    _wide_ids(ids, "ids")
    for d in (weight_dtype, dtype):
        if d not in _DTYPE_CODE:
            raise TypeError(f"tokens: unsupported dtype {d}")
    if weight_dtype != dtype and not (weight_dtype == torch.float32 and dtype in (torch.bfloat16, torch.float16)):
        raise TypeError(f"tokens: a {weight_dtype} table gives {weight_dtype}"
                        f"{', bfloat16 or float16' if weight_dtype == torch.float32 else ''}, not {dtype}")


def _check_table(ids: Tensor, weight: Tensor) -> None:
    if weight.dim() != 2:
        raise ValueError(f"tokens: weight must be [V, C], got {tuple(weight.shape)}")
    if ids.device != weight.device:
        raise ValueError(f"tokens: ids are on {ids.device}, weight on {weight.device}")


@torch.library.custom_op("ebr_fused::embed", mutates_args=(), device_types="cuda")
def embed_op(ids: Tensor, weight: Tensor, scale: float, dtype: torch.dtype) -> Tensor:
    lib = hip_library()
    _check_embed(ids, weight.dtype, dtype)
    _check_table(ids, weight)
    ids, weight = _c(ids), _c(weight)
    V, C = weight.shape
    y = torch.empty((*ids.shape, C), device=weight.device, dtype=dtype)
    if y.numel() == 0:
        return y
    if V == 0:
        return y.zero_()
    with torch.cuda.device(weight.device):
        rc = lib.ebr_block_embed(_code(weight), _code(y), _wide_ids(ids, "ids"), ids.numel(), V, C, scale,
                                 ids.data_ptr(), weight.data_ptr(), y.data_ptr(), _stream(weight))
    _capi.check(rc, "ebr_block_embed")
    return y


@embed_op.register_fake
def _(ids, weight, scale, dtype):
    return weight.new_empty((*ids.shape, weight.shape[-1]), dtype=dtype)


@torch.library.custom_op("ebr_fused::embed_bwd", mutates_args=(), device_types="cuda")
def embed_bwd_op(ids: Tensor, dy: Tensor, V: int, scale: float, dtype: torch.dtype) -> Tensor:
    """dw [V, C] of ``dtype``, the table's."""
    lib = hip_library()
    _check_embed(ids, dtype, dy.dtype)
    if dy.dim() < 1 or tuple(dy.shape[:-1]) != tuple(ids.shape) or dy.device != ids.device:
        raise ValueError(f"tokens: dy is {tuple(dy.shape)} on {dy.device}, expected {tuple(ids.shape)} and a last dim on "
                         f"{ids.device}")
    ids, dy = _c(ids), _c(dy)
    C, N = dy.shape[-1], ids.numel()
    dw = torch.empty((V, C), device=dy.device, dtype=dtype)
    if dw.numel() == 0:
        return dw
    n = lib.ebr_block_embed_bwd_scratch(_code(dw), N, V, C)
    if n < 0:
        _capi.check(2, "ebr_block_embed_bwd")
    scratch = _scratch(n, dy)
    with torch.cuda.device(dy.device):
        rc = lib.ebr_block_embed_bwd(_code(dw), _code(dy), _wide_ids(ids, "ids"), N, V, C, scale, ids.data_ptr(),
                                     dy.data_ptr(), dw.data_ptr(), scratch.data_ptr(), _stream(dy))
    _capi.check(rc, "ebr_block_embed_bwd")
    return dw


@embed_bwd_op.register_fake
def _(ids, dy, V, scale, dtype):
    return dy.new_empty((V, dy.shape[-1]), dtype=dtype)


class _EmbedBwd(torch.autograd.Function):
    @staticmethod
    def forward(ids, dy, V, scale, dtype):
        return torch.ops.ebr_fused.embed_bwd(ids, dy, V, scale, dtype)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ids, dy, _, scale, _ = inputs
        ctx.save_for_backward(ids)
        ctx.scale, ctx.dtype = scale, dy.dtype

    @staticmethod
    def backward(ctx, c):
        (ids,) = ctx.saved_tensors
        return None, _Embed.apply(ids, c, ctx.scale, ctx.dtype), None, None, None


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ids, weight, scale, dtype):
        return torch.ops.ebr_fused.embed(ids, weight, scale, dtype)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ids, weight, scale, _ = inputs
        ctx.save_for_backward(ids)
        ctx.V, ctx.scale, ctx.dtype = weight.shape[0], scale, weight.dtype

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return None, _EmbedBwd.apply(ids, dy, ctx.V, ctx.scale, ctx.dtype), None, None


_DTYPES = {code: dtype for dtype, code in _DTYPE_CODE.items()}


@_host.gradient("embed")
def _embed_grads(ids, V, scale, code, dy):
    return None, _EmbedBwd.apply(ids, dy, V, scale, _DTYPES[code])


@_host.gradient("embed_bwd")
def _embed_bwd_grads(ids, scale, code, c):
    return None, _Embed.apply(ids, c, scale, _DTYPES[code])


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None) -> Tensor:
    """``scale * weight[ids]`` as [*ids.shape, C] in ``dtype`` (the table's, if not given; an fp32 table also gives
    bfloat16 and float16), taken in fp32 and rounded once. A token outside [0, V), such as a padding of -1, gives a row of
    zeros and no gradient. The table's gradient is dense, [V, C] in its dtype, summed in fp32 in a fixed order."""
    dtype = weight.dtype if dtype is None else dtype
    host = _host.module()
    y = None if host is None else host.embedding(ids, weight, scale, _DTYPE_CODE.get(dtype, -1))
    if y is not None:
        return y
    _check_embed(ids, weight.dtype, dtype)
    _check_table(ids, weight)
    if not math.isfinite(scale):
        raise ValueError(f"tokens: scale must be finite, got {scale}")
    return _Embed.apply(ids, weight, float(scale), dtype)


# ---------------------------------------------------------------------------------------------------------------------
# Distillation
# ---------------------------------------------------------------------------------------------------------------------


def _check_distill(logits: Tensor, teacher: Tensor, ids: Tensor, temperature: float) -> None:
    _wide_ids(ids, "teacher_ids")
    _code(logits), _code(teacher)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"tokens: logits must be [..., V], got {tuple(logits.shape)}")
    if teacher.dim() < 1 or tuple(teacher.shape[:-1]) != tuple(logits.shape[:-1]) or teacher.shape != ids.shape:
        raise ValueError(f"tokens: teacher_logits {tuple(teacher.shape)} and teacher_ids {tuple(ids.shape)} must both be "
                         f"{tuple(logits.shape[:-1])} and K")
    if not 1 <= teacher.shape[-1] <= MAX_TEACHER_ENTRIES:
        raise ValueError(f"tokens: K must be 1 to {MAX_TEACHER_ENTRIES} teacher entries, got {teacher.shape[-1]}")
    if teacher.device != logits.device or ids.device != logits.device:
        raise ValueError(f"tokens: logits are on {logits.device}, teacher_logits on {teacher.device}, teacher_ids on "
                         f"{ids.device}")
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError(f"tokens: temperature must be from 1e-15 to 1e15, got {temperature}")


def _rows(logits: Tensor) -> Tuple[Tensor, int]:
    """[N, V] with unit stride in a row, and the stride between rows (a slice of wider rows stays as it is)."""
    x = logits.reshape(-1, logits.shape[-1])
    V = x.shape[1]
    if (V > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < V):
        x = x.contiguous()
    return x, max(x.stride(0), V)


@torch.library.custom_op("ebr_fused::distill", mutates_args=(), device_types="cuda")
def distill_op(logits: Tensor, teacher: Tensor, ids: Tensor, temperature: float,
               reduction: int) -> Tuple[Tensor, Tensor, Tensor]:
    """(loss, stats [N, 4], scale): the latter two are what ``distill_bwd`` needs of the forward; scale is empty without
    a reduction."""
    lib = hip_library()
    _check_distill(logits, teacher, ids, temperature)
    x, row = _rows(logits)
    teacher, ids = _c(teacher), _c(ids)
    N, V, K = x.shape[0], x.shape[1], teacher.shape[-1]
    acc = torch.float64 if logits.dtype == torch.float64 else torch.float32
    none = reduction == REDUCTIONS["none"]
    loss = torch.empty(logits.shape[:-1] if none else (), device=x.device, dtype=acc)
    stats = torch.empty((N, 4), device=x.device, dtype=acc)
    scale = torch.empty((0,) if none else (1,), device=x.device, dtype=acc)
    if none and N == 0:
        return loss, stats, scale
    n = lib.ebr_block_distill_scratch(_code(logits), N, V, K)
    if n < 0:
        _capi.check(2, "ebr_block_distill")
    scratch = _scratch(n, x)
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_distill(
            _code(logits), _code(teacher), _wide_ids(ids, "teacher_ids"), N, V, K, row, temperature, reduction,
            x.data_ptr(), teacher.data_ptr(), ids.data_ptr(), stats.data_ptr(), loss.data_ptr(), scale.data_ptr(),
            scratch.data_ptr(), _stream(x),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_distill")
    return loss, stats, scale


@distill_op.register_fake
def _(logits, teacher, ids, temperature, reduction):
    acc = torch.float64 if logits.dtype == torch.float64 else torch.float32
    none = reduction == REDUCTIONS["none"]
    rows = math.prod(logits.shape[:-1])
    return (logits.new_empty(logits.shape[:-1] if none else (), dtype=acc), logits.new_empty((rows, 4), dtype=acc),
            logits.new_empty((0,) if none else (1,), dtype=acc))


@torch.library.custom_op("ebr_fused::distill_bwd", mutates_args=(), device_types="cuda")
def distill_bwd_op(logits: Tensor, teacher: Tensor, ids: Tensor, stats: Tensor, scale: Tensor, grad: Tensor,
                   temperature: float) -> Tensor:
    lib = hip_library()
    _check_distill(logits, teacher, ids, temperature)
    x, row = _rows(logits)
    teacher, ids = _c(teacher), _c(ids)
    N, V, K = x.shape[0], x.shape[1], teacher.shape[-1]
    none = scale.numel() == 0
    if grad.numel() != (N if none else 1) or tuple(stats.shape) != (N, 4):
        raise ValueError(f"tokens: grad is {tuple(grad.shape)} and stats {tuple(stats.shape)} for {N} rows")
    grad, stats = _c(grad.to(stats.dtype)), _c(stats)
    dx = torch.empty(logits.shape, device=x.device, dtype=logits.dtype)
    if N == 0:
        return dx
    with torch.cuda.device(x.device):
        rc = lib.ebr_block_distill_bwd(
            _code(logits), _code(teacher), _wide_ids(ids, "teacher_ids"), N, V, K, row, temperature, x.data_ptr(),
            teacher.data_ptr(), ids.data_ptr(), stats.data_ptr(), 0 if none else scale.data_ptr(), grad.data_ptr(),
            int(none), dx.data_ptr(), _stream(x),
        )  # fmt: skip
    _capi.check(rc, "ebr_block_distill_bwd")
    return dx


@distill_bwd_op.register_fake
def _(logits, teacher, ids, stats, scale, grad, temperature):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


class _DistillBwd(torch.autograd.Function):
    """A node of its own, so that a second derivative is an error: without it the gradient would pass for a constant."""

    @staticmethod
    def forward(logits, teacher, ids, stats, scale, grad, temperature):
        return torch.ops.ebr_fused.distill_bwd(logits, teacher, ids, stats, scale, grad, temperature)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, _c):
        raise RuntimeError("trying to differentiate twice a function that was marked with @once_differentiable: "
                           "distill_loss has no second derivative")


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(logits, teacher, ids, temperature, reduction):
        return torch.ops.ebr_fused.distill(logits, teacher, ids, temperature, reduction)

    @staticmethod
    def setup_context(ctx, inputs, output):
        logits, teacher, ids, temperature, _ = inputs
        _, stats, scale = output
        ctx.mark_non_differentiable(stats, scale)
        ctx.save_for_backward(logits, teacher, ids, stats, scale)
        ctx.temperature = temperature

    @staticmethod
    def backward(ctx, grad, _stats, _scale):
        logits, teacher, ids, stats, scale = ctx.saved_tensors
        dx = _DistillBwd.apply(logits, teacher, ids, stats, scale, grad, ctx.temperature)
        return dx, None, None, None, None


@_host.gradient("distill")
def _distill_grads(logits, teacher, ids, stats, scale, temperature, grad):
    return (_DistillBwd.apply(logits, teacher, ids, stats, scale, grad, temperature),)


def distill_loss(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor, temperature: float = 1.0,
                 reduction: str = "mean") -> Tensor:
    """Distillation of a student's ``logits`` [..., V] from a teacher's K largest logits, ``teacher_logits`` [..., K] at the
    columns ``teacher_ids`` [..., K]. With p the softmax of a row's teacher_logits / T over the entries whose ids lie in
    [0, V) (others, such as -1, are left out, whatever their logits), and q the softmax of its logits / T, a row's loss is

        T^2 sum_k p_k (log p_k - log q[ids_k])

    A row without an entry of positive probability has loss 0 and gradient 0. ``reduction``: "mean" over the other rows (0
    if there is none), "sum", or "none" for [...]. The loss is fp32 (fp64 for fp64 logits) whatever the logits' dtype. K is
    at most 1024, T from 1e-15 to 1e15; a teacher entry of one token with any logit is the cross entropy to it. Only the
    logits get a gradient."""
    host = _host.module()
    y = None if host is None or reduction not in REDUCTIONS else host.distill_loss(
        logits, teacher_logits, teacher_ids, temperature, REDUCTIONS[reduction])
    if y is not None:
        return y
    if reduction not in REDUCTIONS:
        raise ValueError(f"tokens: reduction must be one of {tuple(REDUCTIONS)}, got {reduction!r}")
    _check_distill(logits, teacher_logits, teacher_ids, temperature)
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("tokens: the teacher is a constant here (no gradient); detach teacher_logits")
    return _Distill.apply(logits, teacher_logits, teacher_ids, float(temperature), REDUCTIONS[reduction])[0]


embedding = torch._dynamo.allow_in_graph(embedding)
distill_loss = torch._dynamo.allow_in_graph(distill_loss)

__all__ = ["distill_loss", "embedding"]
