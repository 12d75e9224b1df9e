"""The attention path's caller side (drop-in for reference ``models/attention.py``).

- ``math_attention`` (reference :49-54): eager softmax attention, differentiable to any order; 16-bit inputs get an
  fp32 softmax.
- Backend table ``ATTENTION_BACKENDS`` / ``get_backend`` (:61-86): ``math``, ``sdpa_auto`` (first order only, for
  microsteps that keep no graph) and ``fused`` (``ebr_amd.fused_attn``, scale D**-0.5).
- The graded-tier flag ``second_order_window`` / ``second_order_required`` (:22-37), thread-local, and
  ``SecondOrderUnsafeError``.
- ``verify_second_order`` (:89-173): a backend's first and second derivatives against ``math_attention`` on a small
  attention-only energy; ``verify_rope_attention``: the same for the one node that takes the fused backend's place behind
  the fused RoPE split.
- ``EnergyAttention`` / ``EnergyReasoningBlock`` (:181-266): the energy network's attention (qkv projection, 2D RoPE,
  learned per-head temperature, backend, output projection) and its post-norm block.
"""

from __future__ import annotations

import threading
from contextlib import contextmanager
from dataclasses import dataclass
from typing import Any, Callable, Dict, Iterator, List, NamedTuple, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from torch import nn

from ebr_amd.layers import (
    RMS_NORM_EPS,
    CastedLinear,
    LayerNorm,
    RopeFused,
    RotaryTable2D,
    SwiGLU,
    apply_rope,
    group_norm,
    rms_norm,
)

Tensor = torch.Tensor
AttnFn = Callable[[Tensor, Tensor, Tensor], Tensor]


# ----------------------------------------------------------------------------------------------------------------------
# Graded tier
# ----------------------------------------------------------------------------------------------------------------------


class _Tier(threading.local):
    graded: bool = False


_TIER = _Tier()


def second_order_required() -> bool:
    """True inside a graded window on this thread: attention called now must carry a correct second derivative."""
    return _TIER.graded


@contextmanager
def second_order_window(active: bool) -> Iterator[None]:
    """Mark the calls inside as graded (``active``) or not, restoring the enclosing state on exit."""
    outer, _TIER.graded = _TIER.graded, bool(active)
    try:
        yield
    finally:
        _TIER.graded = outer


class SecondOrderUnsafeError(RuntimeError):
    """A backend without a correct second derivative reached a graded microstep."""


# ----------------------------------------------------------------------------------------------------------------------
# Backends ([B, H, N, D] in and out)
# ----------------------------------------------------------------------------------------------------------------------


def math_attention(q: Tensor, k: Tensor, v: Tensor) -> Tensor:
    """softmax(Q K^T * D**-0.5) V; bf16 / fp16 inputs are computed in fp32 and the result cast back."""
    wide = torch.float32 if q.dtype in (torch.bfloat16, torch.float16) else q.dtype
    logits = torch.matmul(q.to(wide), k.to(wide).transpose(-1, -2)) * q.shape[-1] ** -0.5
    return torch.matmul(logits.softmax(dim=-1), v.to(wide)).to(q.dtype)


def _sdpa_auto(q: Tensor, k: Tensor, v: Tensor) -> Tensor:
    return F.scaled_dot_product_attention(q, k, v)


def _fused(q: Tensor, k: Tensor, v: Tensor) -> Tensor:
    from ebr_amd.fused_attn import fused_attention

    return fused_attention(q, k, v, scale=q.shape[-1] ** -0.5)


@dataclass(frozen=True)
class AttentionBackend:
    name: str
    fn: AttnFn
    second_order: bool


ATTENTION_BACKENDS: Dict[str, AttentionBackend] = {
    b.name: b
    for b in (
        AttentionBackend("math", math_attention, True),
        AttentionBackend("sdpa_auto", _sdpa_auto, False),
        AttentionBackend("fused", _fused, True),
    )
}


def get_backend(name: str) -> AttentionBackend:
    backend = ATTENTION_BACKENDS.get(name)
    if backend is None:
        raise ValueError(f"unknown attention backend '{name}'; available: {sorted(ATTENTION_BACKENDS)}")
    return backend


# ----------------------------------------------------------------------------------------------------------------------
# Second-order self-test
# ----------------------------------------------------------------------------------------------------------------------


class _Derivatives(NamedTuple):
    grad_z: Tensor  # dE/dz (detached, fp32)
    hess_z: Optional[Tensor]  # d/dz <dE/dz, u>
    mixed: Tuple[Optional[Tensor], ...]  # d/dW <dE/dz, u> for each projection weight


class _Probe:
    """E(z) = sum(attn(z Wq, z Wk, z Wv) Wo) on a 2-row batch, with no residual around the attention, so every
    derivative of E passes through the backend.

    The draws are fixed (the gate must pass or fail exactly as the reference's): the global RNG is reseeded with
    ``seed``; the four weights come from a private CPU generator seeded 11, in the order Wq, Wk, Wv ([d, d]) then Wo
    ([d, 1]), each N(0, 1) * d**-0.5; then z0 = 0.5 * N(0, 1) [2, seq, d] and the direction u ~ N(0, 1) are drawn
    from the global RNG on ``device``."""

    ROWS = 2
    WEIGHT_SEED = 11

    def __init__(self, *, device: torch.device, dtype: torch.dtype, heads: int, seq: int, head_dim: int,
                 seed: int) -> None:
        torch.manual_seed(seed)
        self.heads, self.seq, self.head_dim = heads, seq, head_dim
        width = heads * head_dim
        gen = torch.Generator(device="cpu").manual_seed(self.WEIGHT_SEED)
        self.weights: List[Tensor] = [
            (torch.randn(width, cols, generator=gen) * width**-0.5).to(device=device, dtype=dtype).requires_grad_(True)
            for cols in (width, width, width, 1)
        ]
        self.z0 = torch.randn(self.ROWS, seq, width, device=device, dtype=dtype) * 0.5
        self.u = torch.randn_like(self.z0)

    def _to_heads(self, x: Tensor) -> Tensor:
        return x.view(self.ROWS, self.seq, self.heads, self.head_dim).transpose(1, 2).contiguous()

    def energy(self, attn: AttnFn, z: Tensor) -> Tensor:
        wq, wk, wv, wo = self.weights
        y = attn(self._to_heads(z @ wq), self._to_heads(z @ wk), self._to_heads(z @ wv))
        merged = y.transpose(1, 2).reshape(self.ROWS, self.seq, self.heads * self.head_dim)
        return (merged @ wo).float().sum()

    def derivatives(self, attn: AttnFn) -> _Derivatives:
        z = self.z0.detach().clone().requires_grad_(True)
        (gz,) = torch.autograd.grad(self.energy(attn, z), z, create_graph=True)
        directional = (gz * self.u).sum()
        (hz,) = torch.autograd.grad(directional, z, retain_graph=True, allow_unused=True)
        mixed = torch.autograd.grad(directional, self.weights, allow_unused=True)
        return _Derivatives(gz.detach().float(), hz, tuple(mixed))


def _max_rel(got: Optional[Tensor], want: Optional[Tensor]) -> float:
    """max|got - want| / max|want| (floored at 1e-12); 0 when nothing is expected, inf when something is missing."""
    if want is None:
        return 0.0
    if got is None:
        return float("inf")
    want = want.float()
    return float((got.float() - want).abs().max() / want.abs().max().clamp_min(1e-12))


def _absent_terms(want: _Derivatives, got: _Derivatives) -> List[str]:
    pairs = [("d2E/dz2", want.hess_z, got.hess_z)]
    pairs += [(f"d2E/dtheta dz (weight {i})", w, g) for i, (w, g) in enumerate(zip(want.mixed, got.mixed))]
    return [label for label, w, g in pairs if w is not None and g is None]


def _errors(want: _Derivatives, got: _Derivatives) -> Dict[str, float]:
    return {
        "dE/dz": _max_rel(got.grad_z, want.grad_z),
        "d2E/dz2": _max_rel(got.hess_z, want.hess_z),
        "d2E/dtheta dz": max(_max_rel(g, w) for g, w in zip(got.mixed, want.mixed)),
    }


def verify_second_order(
    backend: AttentionBackend,
    *,
    device: torch.device,
    dtype: torch.dtype = torch.float32,
    heads: int = 2,
    seq: int = 32,
    head_dim: int = 16,
    rtol: float = 5e-2,
    seed: int = 0,
) -> None:
    """Raise ``SecondOrderUnsafeError`` unless ``backend`` gives math_attention's dE/dz, d2E/dz2 . u and
    d2E/dW dz . u on the probe energy, each within ``rtol`` in max-abs relative error. Reseeds the global RNG."""
    probe = _Probe(device=device, dtype=dtype, heads=heads, seq=seq, head_dim=head_dim, seed=seed)
    want = probe.derivatives(math_attention)
    try:
        got = probe.derivatives(backend.fn)
    except Exception as exc:
        raise SecondOrderUnsafeError(
            f"self-test of attention backend '{backend.name}' raised {type(exc).__name__}: {exc}"
        ) from exc
    _require_agreement(f"attention backend '{backend.name}'", want, got, rtol)


def _require_agreement(what: str, want: _Derivatives, got: _Derivatives, rtol: float) -> None:
    absent = _absent_terms(want, got)
    if absent:
        raise SecondOrderUnsafeError(f"{what} has no second derivative for {', '.join(absent)}")
    errs = _errors(want, got)
    worst = {name: e for name, e in errs.items() if not e < rtol}
    if worst:
        detail = ", ".join(f"{name} off by {e:.3e}" for name, e in errs.items())
        raise SecondOrderUnsafeError(f"{what} disagrees with math attention beyond {rtol}: {detail}")


def verify_rope_attention(*, device: torch.device, dtype: torch.dtype = torch.float32, heads: int = 2,
                          head_dim: int = 16, rtol: float = 5e-2) -> bool:
    """``verify_second_order`` for ``rope_attention``: E(z) = sum(rope_attention(z Wqkv, t) Wo) on 4 x 4 cells against
    the dense split, the temperature t as a product and ``math_attention``, with d2E/dtheta dz for Wqkv, t and Wo. All
    draws come from a private generator: the global RNG is left as it is. False where it does not take the call (off the
    GPU, under a mode or hooks): the parts run then, and there is nothing to test."""
    from ebr_amd.fused_attn.rope_split import dense_split, rope_attention

    width = heads * head_dim
    gen = torch.Generator(device="cpu").manual_seed(_Probe.WEIGHT_SEED)

    def draw(*shape: int, std: float = 1.0) -> Tensor:
        return (torch.randn(*shape, generator=gen) * std).to(device=device, dtype=dtype)

    cos, sin = RotaryTable2D(head_dim, 4, 4).to(device)()
    w_qkv, w_o = (draw(width, cols, std=width**-0.5).requires_grad_(True) for cols in (3 * width, 1))
    t = torch.linspace(0.8, 1.25, heads, device=device).requires_grad_(True)
    z0, u = draw(_Probe.ROWS, 16, width, std=0.5), draw(_Probe.ROWS, 16, width)

    def parts(qkv: Tensor) -> Tensor:
        q, k, v = dense_split(qkv, cos, sin, cos.new_zeros((0,)), heads)
        y = math_attention(q * t.to(q.dtype).view(1, heads, 1, 1), k, v)
        return y.transpose(1, 2).reshape(_Probe.ROWS, 16, width)

    def derivatives(fn: Callable[[Tensor], Tensor]) -> _Derivatives:
        z = z0.clone().requires_grad_(True)
        (gz,) = torch.autograd.grad((fn(z @ w_qkv) @ w_o).float().sum(), z, create_graph=True)
        hz, *mixed = torch.autograd.grad((gz * u).sum(), (z, w_qkv, t, w_o), allow_unused=True)
        return _Derivatives(gz.detach().float(), hz, tuple(mixed))

    with torch.enable_grad():
        if rope_attention((z0 @ w_qkv).detach(), cos, sin, heads, t) is None:
            return False
        node = derivatives(lambda qkv: rope_attention(qkv, cos, sin, heads, t))
        _require_agreement("rope_attention", derivatives(parts), node, rtol)
    return True


def _self_test_layers(model: nn.Module) -> List["EnergyAttention"]:
    return [m for m in model.modules() if isinstance(m, EnergyAttention)]


def prime_attention_self_test(model: nn.Module) -> None:
    """Run every attention layer's pending self-test now, inside a forked RNG so the caller's random stream is left
    as it was (reference utils/checkpoint.py:234-248: a trainer calls this before its own draws)."""
    params = list(model.parameters())
    if not params:
        return
    device = params[0].device
    node_tested: Dict[int, bool] = {}  # by head count: the node's test is the same for every layer
    with torch.random.fork_rng(devices=[device] if device.type == "cuda" else []):
        for layer in _self_test_layers(model):
            layer._ensure_verified(device, torch.float32)
            if layer.graded_backend.fn is _fused and not layer._node_verified:
                layer._node_verified = node_tested.get(layer.num_heads, False)
                layer._ensure_node_verified(device, torch.float32)
                node_tested[layer.num_heads] = layer._node_verified


def seed_attention_self_test(model: nn.Module, seed: int) -> None:
    """Seed that each attention layer's pending self-test reseeds the global RNG with (reference
    utils/checkpoint.py:251-255)."""
    for layer in _self_test_layers(model):
        layer.self_test_seed = int(seed)


# ----------------------------------------------------------------------------------------------------------------------
# Energy network modules
# ----------------------------------------------------------------------------------------------------------------------


class EnergyAttention(nn.Module):
    """Multi-head attention of the energy network: a bias-free qkv projection, 2D RoPE on q and k, a learned
    temperature per head on q, the tier's backend, and a bias-free output projection.

    The graded backend must have a second derivative; it is checked against ``math_attention`` (``verify_second_order``)
    once, before its first graded call. Parameter names match the reference's state dicts."""

    _node_verified = False  # on the class: a whole module unpickled from before it existed has no such attribute

    def __init__(self, hidden_size: int, head_dim: int, num_heads: int, *, backend: str, nograd_backend: str) -> None:
        super().__init__()
        self.hidden_size, self.head_dim, self.num_heads = hidden_size, head_dim, num_heads
        self.output_size = num_heads * head_dim
        graded = get_backend(backend)
        if not graded.second_order:
            raise SecondOrderUnsafeError(f"backend '{backend}' has no second derivative: not usable in graded steps")
        self.graded_backend, self.nograd_backend = graded, get_backend(nograd_backend)
        self.qkv_proj = CastedLinear(hidden_size, 3 * self.output_size, bias=False)
        self.o_proj = CastedLinear(self.output_size, hidden_size, bias=False)
        self.log_logit_scale = nn.Parameter(torch.zeros(num_heads))  # log temperature; 0 keeps scale D**-0.5
        self._verified = False
        self.self_test_seed = 0

    def _ensure_verified(self, device: torch.device, dtype: torch.dtype) -> None:
        """Self-test the graded backend once, in fp32 for 16-bit models, on at most 2 heads of at most 16 dims."""
        if self._verified:
            return
        verify_second_order(
            self.graded_backend,
            device=device,
            dtype=torch.float32 if dtype in (torch.bfloat16, torch.float16) else dtype,
            heads=min(2, self.num_heads),
            head_dim=min(16, self.head_dim),
            seed=self.self_test_seed,
        )
        self._verified = True

    def _ensure_node_verified(self, device: torch.device, dtype: torch.dtype) -> None:
        """Self-test ``rope_attention`` once, before it serves a graded call in the backend's place."""
        if not self._node_verified:
            self._node_verified = verify_rope_attention(
                device=device,
                dtype=torch.float32 if dtype in (torch.bfloat16, torch.float16) else dtype,
                heads=min(2, self.num_heads),
            )

    def _temperature(self, dtype: torch.dtype, track_grad: bool) -> Tensor:
        t = self.log_logit_scale.exp() if track_grad else self.log_logit_scale.detach().exp()
        return t.to(dtype)

    def _heads(self, cos_sin: Any, x: Tensor, qkv: Tensor, graded: bool) -> Tuple[Tensor, Tensor, Tensor]:
        """q (rotated, tempered), k (rotated), v as [B, H, N, D]."""
        b, n, _ = x.shape
        h, d = self.num_heads, self.head_dim
        if isinstance(cos_sin, RopeFused):
            from ebr_amd.fused_attn.rope_split import rope_split

            # One kernel splits, rotates and lays out q, k, v. Outside graded steps it also applies the temperature;
            # graded steps apply it as a separate product so that log_logit_scale receives its gradient.
            if not graded:
                return rope_split(qkv, cos_sin.cos, cos_sin.sin, h, self._temperature(x.dtype, False))
            q, k, v = rope_split(qkv, cos_sin.cos, cos_sin.sin, h)
        else:
            q, k, v = (t.view(b, n, h, d) for t in qkv.split(self.output_size, dim=-1))
            if cos_sin is not None:
                q, k = apply_rope(cos_sin, q, k)
            q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        return q * self._temperature(q.dtype, True).view(1, h, 1, 1), k, v

    def forward(self, cos_sin: Any, hidden_states: Tensor) -> Tensor:
        graded = second_order_required()
        if graded:
            self._ensure_verified(hidden_states.device, hidden_states.dtype)
        backend = self.graded_backend if graded else self.nograd_backend
        qkv = self.qkv_proj(hidden_states)
        if isinstance(cos_sin, RopeFused) and backend.fn is _fused:
            from ebr_amd.fused_attn.rope_split import rope_attention

            # split, rotation, temperature, attention and merge as one node where the native path takes the call
            t = self.log_logit_scale if graded else self.log_logit_scale.detach()
            y = rope_attention(qkv, cos_sin.cos, cos_sin.sin, self.num_heads, t.exp())
            if y is not None:
                if graded:
                    self._ensure_node_verified(hidden_states.device, hidden_states.dtype)
                return self.o_proj(y)
        q, k, v = self._heads(cos_sin, hidden_states, qkv, graded)
        y = backend.fn(q, k, v)
        b, n, _ = hidden_states.shape
        return self.o_proj(y.transpose(1, 2).reshape(b, n, self.output_size))

    def extra_repr(self) -> str:
        return (f"heads={self.num_heads}, head_dim={self.head_dim}, graded={self.graded_backend.name}, "
                f"nograd={self.nograd_backend.name}")


class EnergyReasoningBlock(nn.Module):
    """Post-norm block: h <- rms_norm(h + sublayer(h)) for the attention, then for the SwiGLU MLP. ``norm="group"`` takes a
    group norm over the board's cells (``norm_groups`` groups of channels) in rms_norm's place, ``norm="layer"`` a layer norm
    with a learned weight and bias. ``mlp_impl``: the MLP's, ``block_impl`` if not given."""

    norm = "rms"  # on the class: a whole module unpickled from before it existed has no such attribute

    def __init__(self, config: Any) -> None:
        super().__init__()
        hidden, heads = config.hidden_size, config.num_heads
        if hidden % heads:
            raise ValueError(f"hidden_size {hidden} does not split into {heads} heads")
        self.block_impl = getattr(config, "block_impl", "eager")
        self.norm, self.norm_groups = getattr(config, "norm", "rms"), getattr(config, "norm_groups", 1)
        if self.norm not in ("rms", "group", "layer"):
            raise ValueError(f"norm must be 'rms', 'group' or 'layer', got {self.norm!r}")
        if self.norm == "group" and (self.norm_groups < 1 or hidden % self.norm_groups):
            raise ValueError(f"hidden_size {hidden} does not split into {self.norm_groups} norm groups")
        self.self_attn = EnergyAttention(hidden, hidden // heads, heads, backend=config.attn_backend,
                                         nograd_backend=config.attn_nograd_backend)
        mlp_impl = getattr(config, "mlp_impl", None)
        self.mlp = SwiGLU(hidden_size=hidden, expansion=config.expansion, impl=mlp_impl or self.block_impl)
        if self.norm == "layer":
            impl = "fused" if self.block_impl == "fused" else "eager"
            self.layer_norms = nn.ModuleList(LayerNorm(hidden, RMS_NORM_EPS, impl) for _ in range(2))

    def _add_norm(self, h: Tensor, r: Tensor, at: int = 0) -> Tensor:
        if self.norm == "layer":
            return self.layer_norms[at](h + r)
        if self.norm == "group":
            if self.block_impl == "fused":
                from ebr_amd import block

                return block.group_norm(h + r, self.norm_groups, eps=RMS_NORM_EPS)
            return group_norm(h + r, self.norm_groups, RMS_NORM_EPS)
        if self.block_impl == "fused":  # rms_norm with its first and second derivatives as HIP kernels
            from ebr_amd import block

            return block.add_rms_norm(h, r, RMS_NORM_EPS)
        return rms_norm(h + r, variance_epsilon=RMS_NORM_EPS)

    def _sublayers(self, cos_sin: Any) -> Sequence[Callable[[Tensor], Tensor]]:
        return (lambda x: self.self_attn(cos_sin, x), self.mlp)

    def forward(self, cos_sin: Any, hidden_states: Tensor) -> Tensor:
        h = hidden_states
        for at, sublayer in enumerate(self._sublayers(cos_sin)):
            h = self._add_norm(h, sublayer(h), at)
        return h


__all__ = [
    "ATTENTION_BACKENDS",
    "AttentionBackend",
    "EnergyAttention",
    "EnergyReasoningBlock",
    "SecondOrderUnsafeError",
    "get_backend",
    "math_attention",
    "prime_attention_self_test",
    "second_order_required",
    "seed_attention_self_test",
    "second_order_window",
    "verify_rope_attention",
    "verify_second_order",
]
