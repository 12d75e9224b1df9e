"""The host paths of the embedding, the distillation loss and the group norm: the native nodes give the Python nodes' bits,
leave modes, transforms and hooks to Python, take batched gradients there, and refuse the derivatives that there are none
of."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from ebr_amd import _host, block, tokens

pytestmark = pytest.mark.gpu

KINDS = ["embed", "distill", "distill_rows", "norm", "norm_plain", "norm_bias"]


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _case(kind):
    """The call, and the inputs that it is differentiable in."""
    g = torch.Generator("cuda").manual_seed(1)
    if kind == "embed":
        ids = torch.randint(-1, 9, (4, 50), generator=g, device="cuda")
        return (lambda w: tokens.embedding(ids, w, 0.7)), [_randn((9, 24), 2)]
    if kind.startswith("distill"):
        t, ids = _randn((6, 5, 3), 3), torch.randint(-1, 20, (6, 5, 3), generator=g, device="cuda")
        reduction = "none" if kind == "distill_rows" else "mean"
        return (lambda x: tokens.distill_loss(x, t, ids, 1.3, reduction)), [_randn((6, 5, 20), 4)]
    x, w, b = _randn((3, 7, 5, 24), 5), 1 + 0.1 * _randn((24,), 6), 0.1 * _randn((24,), 7)
    if kind == "norm":
        return (lambda x, w, b: block.group_norm(x, 4, w, b, activation="silu")), [x, w, b]
    if kind == "norm_bias":
        return (lambda x, b: block.group_norm(x, 4, None, b, activation="silu")), [x, b]
    return (lambda x: block.group_norm(x, 4)), [x]


def _orders(kind, fn, xs):
    xs = [x.detach().clone().requires_grad_(True) for x in xs]
    y = fn(*xs)
    dy = _randn(y.shape, 9).requires_grad_(True)
    out = [y, *torch.autograd.grad(y, xs, dy, create_graph=not kind.startswith("distill"))]
    if not kind.startswith("distill"):
        wrt = [dy] if kind == "embed" else [*xs, dy]
        out += torch.autograd.grad(out[1:], wrt, [_randn(o.shape, 10 + i) for i, o in enumerate(out[1:])])
    return [t.detach() for t in out]


@pytest.mark.parametrize("kind", KINDS)
def test_same_bits_as_the_python_nodes(monkeypatch, kind):
    fn, xs = _case(kind)
    assert "CppNode" in fn(*(x.requires_grad_(True) for x in xs)).grad_fn.name()
    got = _orders(kind, fn, xs)
    monkeypatch.setattr(_host, "_MODULE", None)
    assert "CppNode" not in fn(*xs).grad_fn.name()
    want = _orders(kind, fn, xs)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.ops.add(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("kind", KINDS)
def test_modes_see_the_ops(kind):
    fn, xs = _case(kind)
    native = _orders(kind, fn, xs)
    with _Seen() as seen:
        got = _orders(kind, fn, xs)
    names = {"embed": ["embed", "embed_bwd"], "dist": ["distill", "distill_bwd"],
             "norm": ["block_groupnorm", "block_groupnorm_bwd", "block_groupnorm_bwd2"]}[kind[:4] if kind != "embed" else kind]
    assert all(f"ebr_fused.{n}.default" in seen.ops for n in names)
    assert all(torch.equal(a, b) for a, b in zip(native, got))
    # a mode around the backward of a native forward
    xs = [x.detach().requires_grad_(True) for x in xs]
    y = fn(*xs)
    with _Seen() as seen:
        first = torch.autograd.grad(y, xs, _randn(y.shape, 9), create_graph=not kind.startswith("distill"))
    assert f"ebr_fused.{names[1]}.default" in seen.ops
    assert all(torch.equal(a, b) for a, b in zip(first, native[1:]))


@pytest.mark.parametrize("kind", KINDS)
def test_batched_gradients(kind):
    fn, xs = _case(kind)
    xs = [x.detach().requires_grad_(True) for x in xs]
    y = fn(*xs)

    def both(outs, wrt, seed):
        cots = [_randn((3, *o.shape), seed + i) for i, o in enumerate(outs)]
        got = torch.autograd.grad(outs, wrt, cots, is_grads_batched=True, retain_graph=True)
        want = [torch.autograd.grad(outs, wrt, [c[i] for c in cots], retain_graph=True) for i in range(3)]
        for i, g in enumerate(got):
            assert torch.equal(g, torch.stack([w[i] for w in want]))

    both([y], xs, 20)
    if kind.startswith("distill"):
        return
    dy = _randn(y.shape, 30).requires_grad_(True)
    first = torch.autograd.grad(y, xs, dy, create_graph=True)
    both(first, [dy] if kind == "embed" else [*xs, dy], 50)


def test_saved_tensor_hooks_see_what_is_saved():
    for kind in KINDS:
        fn, xs = _case(kind)
        xs = [x.detach().requires_grad_(True) for x in xs]
        ref = torch.autograd.grad(fn(*xs).sum(), xs)
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(1) or t.clone(), lambda t: t):
            y = fn(*xs)
        assert packed
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), xs), ref))


@pytest.mark.parametrize("native", [True, False])
def test_no_derivative_past_the_last(monkeypatch, native):
    if not native:
        monkeypatch.setattr(_host, "_MODULE", None)
    fn, (x,) = _case("distill")
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(fn(x), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dx.square().sum() + x.sum()).backward()
    fn, xs = _case("norm")
    x = xs[0].requires_grad_(True)
    (dx,) = torch.autograd.grad(fn(*xs).square().sum(), x, create_graph=True)
    (gx,) = torch.autograd.grad(dx.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (gx.sum() + x.sum()).backward()


def test_gradients_that_are_not_asked_for(monkeypatch):
    """A descent's gradient of the input alone leaves the parameters' out, on both paths; and each alone is the same."""
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_host, "_MODULE", None)
        fn, xs = _case("norm")
        x, w, b = (t.requires_grad_(True) for t in xs)
        x = x * 1.0  # inner nodes, as in a network: a leaf's gradient is always computed
        w, b = w * 1.0, b * 1.0
        y = fn(x, w, b)
        every = torch.autograd.grad(y.sum(), (x, w, b), retain_graph=True)
        for i, t in enumerate((x, w, b)):
            assert torch.equal(torch.autograd.grad(y.sum(), t, retain_graph=True)[0], every[i])
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        for t in (x, w, b):
            assert bool(torch.isfinite(torch.autograd.grad(dx.sum(), t, retain_graph=True)[0]).all())


def test_refused_calls_stay_refused():
    """What the native entry points leave is refused by the Python ones."""
    w = _randn((5, 8), 1)
    with pytest.raises(TypeError):
        tokens.embedding(torch.zeros(3, device="cuda"), w)
    with pytest.raises(ValueError):
        tokens.embedding(torch.zeros(3, dtype=torch.int64), w)
    with pytest.raises(ValueError):
        tokens.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), _randn((1, 1 << 18), 1))
    ids = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(NotImplementedError):
        tokens.distill_loss(_randn((3, 9), 1), _randn((3, 2), 2).requires_grad_(True), ids)
    with pytest.raises(ValueError):
        tokens.distill_loss(_randn((3, 9), 1), _randn((4, 2), 2), ids)
    with pytest.raises(ValueError):
        tokens.distill_loss(_randn((3, 9), 1), _randn((3, 2), 2), ids, reduction="batchmean")
    with pytest.raises(ValueError):
        block.group_norm(_randn((3, 9), 1), 2)
    with pytest.raises(ValueError):
        block.group_norm(_randn((3, 8), 1), 2, activation="tanh")
    with pytest.raises(ValueError):
        block.group_norm(_randn((3, 8), 1), 2, _randn((9,), 1))
