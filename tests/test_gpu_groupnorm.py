"""GPU parity of the group norm (``ebr_amd.block.group_norm``) and its first and second derivatives against 64-bit autograd
of the plain formula on the same inputs, and the operators of a training step together.

Tolerances: half a step of the output's type, and for what comes before it in 32 bits (u = 2^-24; fp64: 2^-53) a multiple
of u times the size of the terms that an output adds up, each taken without its sign (``_sizes``): no term passes through
more than about 30 roundings on its way (the normalised value 4, the activation's derivatives 15 with the exponential's and
the reciprocal's errors, products and the last sums 10), and a mean of m terms adds at most the depth of its chain of
additions, 2 L / 16 + 64 for L cells. Channels are within a few deviations of each other, so the normalised value is
not a small difference of large numbers; ``test_far_from_zero`` looks at the other case."""

import pytest
import torch

from ebr_amd import block, tokens
from ebr_amd import energy as en

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-24, torch.float16: 2.0**-24, torch.float64: 2.0**-53}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _plain(x, G, w, b, act):
    B, C = x.shape[0], x.shape[-1]
    v = x.reshape(B, -1, G, C // G)
    c = v - v.mean(dim=(1, 3), keepdim=True)
    h = (c * torch.rsqrt(c.square().mean(dim=(1, 3), keepdim=True) + EPS)).reshape(x.shape)
    a = h if w is None else h * w
    a = a if b is None else a + b
    return torch.nn.functional.silu(a) if act == "silu" else a


def _orders(fn, x, dy, u, w, b, uw=None, ub=None):
    """y; dx, dw, db; and the gradients of <u, dx> + <uw, dw> + <ub, db> for x, dy, w, b."""
    ps = [p for p in (w, b) if p is not None]
    y = fn(x, w, b)
    first = torch.autograd.grad(y, [x, *ps], dy, create_graph=True)
    cots = [u] + ([uw] if w is not None else []) + ([ub] if b is not None else [])
    some = [(o, c) for o, c in zip(first, cots) if c is not None]
    second = torch.autograd.grad([o for o, _ in some], [x, dy, *ps], [c for _, c in some], allow_unused=True)
    second = [torch.zeros_like(p) if s is None else s for s, p in zip(second, [x, dy, *ps])]
    return [t.detach() for t in (y, *first, *second)]


def _sizes(x, G, w, b, dy, u, uw, ub):
    """For each output of ``_orders`` the size of the terms it adds up (64 bits)."""
    B, C = x.shape[0], x.shape[-1]
    L = x.numel() // (B * C)

    def mean(v):
        v = v.reshape(B, L, G, C // G)
        return v.mean(dim=(1, 3), keepdim=True).expand(B, L, G, C // G).reshape(B, L, C)

    x, dy, u = (t.reshape(B, L, C) for t in (x, dy.abs(), u.abs()))
    mu = mean(x)
    r = (mean((x - mu).square()) + EPS).rsqrt()
    h = (x.abs() + mu.abs()) * r  # with what a difference from the mean can lose
    wa, ba = (torch.ones(C, dtype=x.dtype, device=x.device) if w is None else w.abs()), (0 if b is None else b.abs())
    uwa, uba = (0 if uw is None else uw.abs()), (0 if ub is None else ub.abs())
    a = wa * h + ba
    lip = 1 + a  # how an error of a, relative to it, grows in the activation's derivatives (each at most about 1)

    def proj(v):
        return r * (v + mean(v) + h * mean(v * h))

    k = wa * dy * lip
    q = wa * proj(u) + uwa * h + uba
    t = dy * q * lip
    v = wa * t + uwa * dy * lip + r * (u * mean(k * h) + k * mean(u * h))
    along = mean(k * u) + mean(k) * mean(u) + mean(u * h) * mean(k * h)
    sums = lambda v: v.sum((0, 1))  # noqa: E731
    out = [a * lip, proj(k)]
    ps = [sums(k / wa.clamp(min=1e-3) * h), sums(k / wa.clamp(min=1e-3))]
    out += [p for p, given in zip(ps, (w, b)) if given is not None]
    out += [proj(v) + r * r * h * along, q * lip]
    qs = [sums(dy * lip * proj(u) + t * h), sums(t)]
    return out + [p for p, given in zip(qs, (w, b)) if given is not None]


NAMES = ["y", "dx", "dw", "db", "gx", "gdy", "gw", "gb"]


def _check(x, G, w, b, act, dy, u, uw=None, ub=None):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, dy, w, b)]
    got = _orders(lambda x, w, b: block.group_norm(x, G, w, b, EPS, act), leaves[0], leaves[1], u, leaves[2], leaves[3], uw, ub)
    d = [None if t is None else t.detach().double() for t in (x, dy, w, b, u, uw, ub)]
    for t in d[:4]:
        if t is not None:
            t.requires_grad_(True)
    ref = _orders(lambda x, w, b: _plain(x, G, w, b, act), d[0], d[1], d[4], d[2], d[3], d[5], d[6])
    size = _sizes(d[0].detach(), G, None if w is None else d[2].detach(), None if b is None else d[3].detach(), d[1].detach(), d[4], d[5], d[6])
    names = [n for n in NAMES if (w is not None or n[1:] != "w") and (b is not None or n[1:] != "b")]
    L = x.numel() // (x.shape[0] * x.shape[-1])
    u_ = U[x.dtype] * (30 + 2 * L / 16 + 64)
    for n, a, e, s in zip(names, got, ref, size, strict=True):
        assert a.shape == e.shape, n
        f = torch.finfo(a.dtype)
        tol = (f.eps / 2 * e.abs()).clamp(min=f.tiny * f.eps / 2) + u_ * s.reshape(e.shape)
        off = (a.double() - e).abs() - tol
        assert bool((off <= 0).all()), f"{n}: off by {float((a.double() - e).abs().max()):.3e}, {float(off.max()):.3e} over its bound"
    return got


def _inputs(cuda, shape, dtype, seed, affine=True, pt=torch.float32):
    g = torch.Generator(cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    C = shape[-1]
    pt = torch.float64 if dtype == torch.float64 else pt
    ts = dict(x=(r(*shape) + 0.5 * r(C)).to(dtype), dy=r(*shape).to(dtype), u=r(*shape).to(dtype))
    ts["w"], ts["b"] = ((1 + 0.3 * r(C)).to(pt), (0.3 * r(C)).to(pt)) if affine else (None, None)
    ts["uw"], ts["ub"] = (r(C).to(pt), r(C).to(pt)) if affine else (None, None)
    return ts


DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
SHAPES = [
    ((2, 81, 512), 32), ((1, 1, 64), 2), ((3, 9, 24), 4), ((2, 7, 5, 30), 3), ((5, 33, 7), 7), ((1, 900, 512), 16),
    ((3, 2, 96), 1), ((2, 300, 320), 32), ((1, 4100, 16), 2), ((2, 40, 1032), 3), ((9, 16, 8), 8),
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_group_norm(cuda, dtype, act, shape, G):
    _say(f"group_norm {shape} {G} {act} {dtype}")
    ts = _inputs(cuda, shape, dtype, seed=shape[-1] + G)
    _check(ts["x"], G, ts["w"], ts["b"], act, ts["dy"], ts["u"], ts["uw"], ts["ub"])


# groups that a workgroup holds: tiles of every width, an end of the channels and of the cells inside a tile, four and eight
# cells a thread, 4 and 16 waves; and the sizes on either side of where it no longer does
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [
    ((2, 32, 64), 8), ((2, 33, 64), 4), ((3, 128, 96), 4), ((2, 129, 96), 4), ((2, 256, 64), 2), ((2, 257, 64), 2), ((2, 5, 512), 1),
    ((2, 130, 256), 2), ((1, 1024, 64), 8), ((1, 1025, 64), 8), ((2, 500, 128), 2), ((3, 17, 144), 3), ((1, 60, 2048), 4), ((700, 4, 64), 4),
    ((3, 4, 1024), 32), ((2, 16, 1024), 1), ((2, 7, 2048), 1), ((2, 1, 512), 2), ((2, 3, 96), 2), ((5, 2, 264), 1), ((2, 9, 4096), 2), ((2, 30, 320), 32), ((1, 193, 60), 6), ((2, 256, 128), 64),
])  # fmt: skip
def test_held_groups(cuda, dtype, shape, G):
    _say(f"group_norm held {shape} {G} {dtype}")
    ts = _inputs(cuda, shape, dtype, seed=shape[-1] + G)
    _check(ts["x"], G, ts["w"], ts["b"], "silu", ts["dy"], ts["u"], ts["uw"], ts["ub"])


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("have", ["", "w", "b"])
def test_parameters_left_out(cuda, act, have):
    _say(f"group_norm parameters {have!r} {act}")
    ts = _inputs(cuda, (3, 50, 48), torch.bfloat16, seed=1, pt=torch.bfloat16 if have else torch.float32)
    w, b = (ts[n] if n in have else None for n in "wb")
    _check(ts["x"], 6, w, b, act, ts["dy"], ts["u"], ts["uw"] if w is not None else None, None)


def test_far_from_zero(cuda):
    """Cells around 1000 with deviation 1, the first a zero as padding leaves it: a variance as a difference of squares, or
    one taken about the first cell, would be off by percents. Here x loses 1000 u against its deviation, so the statistics are
    within that, and h within 2000 u plus the sums'."""
    _say("group_norm far from zero")
    g = torch.Generator(cuda).manual_seed(4)
    x = 1000 + torch.randn(2, 700, 64, generator=g, device=cuda)
    y = block.group_norm(x, 4, eps=EPS)
    ref = _plain(x.double(), 4, None, None, None)
    assert float((y - ref).abs().max()) <= 3000 * 2.0**-24 * 5
    x[:, 0] = 0
    y, ref = block.group_norm(x, 4, eps=EPS), _plain(x.double(), 4, None, None, None)
    assert float((y - ref).abs().max() / ref.abs().max()) <= 3000 * 2.0**-24


def test_constant_groups_and_extremes(cuda):
    """A group of one value has h = 0 and the factor 1 / sqrt(eps); an infinity or NaN stays in its sample and group."""
    _say("group_norm constant")
    b = torch.linspace(-1, 1, 32, device=cuda)
    y = block.group_norm(torch.full((2, 20, 32), 3.0, device=cuda, dtype=torch.bfloat16), 4, None, b)
    assert torch.equal(y, b.to(torch.bfloat16).expand(2, 20, 32))
    for shape in ((2, 20, 32), (1, 900, 512), (1, 3000, 12)):  # held by a workgroup, by 16 waves, read twice
        b = torch.linspace(-1, 1, shape[-1], device=cuda)
        for value in (1000.1, -3e4, 7e-3):
            assert torch.equal(block.group_norm(torch.full(shape, value, device=cuda), 4, None, b), b.expand(shape))
    b = torch.linspace(-1, 1, 32, device=cuda)
    x = torch.randn(3, 20, 32, generator=torch.Generator(cuda).manual_seed(1), device=cuda)
    good = block.group_norm(x, 4, None, b, EPS, "silu")
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[1, 7, 9] = bad
        y = block.group_norm(z, 4, None, b, EPS, "silu")
        assert bool(torch.isnan(y[1, :, 8:16]).any())
        y[1, :, 8:16] = good[1, :, 8:16]
        assert torch.equal(y, good)


# read twice: threads and lanes without cells, one part and many, one channel a thread and vectors
@pytest.mark.parametrize("shape,G", [((1, 3000, 12), 4), ((2, 9, 7), 7), ((3, 40, 9), 1), ((1, 5000, 512), 16), ((2, 4100, 16), 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_groups_of_one_large_value(cuda, dtype, shape, G):
    """A group of one value has h = 0 whatever the value, whose square need not be a number of 32 bits; and cells around 1e20
    with deviation 1e16: x loses 10^4 u against it, and h as in ``test_far_from_zero``."""
    _say(f"group_norm large {shape} {dtype}")
    b = torch.linspace(-1, 1, shape[-1], device=cuda)
    for value in (1e20, torch.finfo(dtype).max, torch.finfo(dtype).min):
        x = torch.full(shape, value, device=cuda, dtype=dtype).requires_grad_(True)
        y = block.group_norm(x, G, None, b)
        assert torch.equal(y, b.to(dtype).expand(shape)), value
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool(torch.isfinite(dx).all()), value
    if dtype == torch.float32 and shape[1] * shape[2] // G > 1000:
        x = 1e20 * (1 + 1e-4 * torch.randn(shape, generator=torch.Generator(cuda).manual_seed(1), device=cuda))
        ref = _plain(x.double(), G, None, None, None)
        assert float((block.group_norm(x, G, eps=EPS) - ref).abs().max()) <= 3 * 1e4 * 2.0**-24 * float(ref.abs().max())


# few cells a thread and many, 4 waves and 16, a tile of several groups and one of all channels
@pytest.mark.parametrize("shape,G", [((2, 20, 32), 4), ((1, 900, 512), 16), ((2, 256, 64), 2), ((2, 5, 512), 1), ((1, 1024, 64), 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_held_groups_of_one_large_value(cuda, dtype, shape, G):
    """As ``test_long_groups_of_one_large_value`` where a workgroup holds the group: its elements' sum need not be a number of
    32 bits either."""
    _say(f"group_norm held large {shape} {dtype}")
    b = torch.linspace(-1, 1, shape[-1], device=cuda)
    for value in (1e20, 1e36, torch.finfo(dtype).max, torch.finfo(dtype).min):
        x = torch.full(shape, value, device=cuda, dtype=dtype).requires_grad_(True)
        y = block.group_norm(x, G, None, b)
        assert torch.equal(y, b.to(dtype).expand(shape)), value
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool(torch.isfinite(dx).all()), value


def test_views_and_empty_calls(cuda):
    _say("group_norm views")
    ts = _inputs(cuda, (4, 12, 48), torch.bfloat16, seed=3)
    a = _check(ts["x"], 6, ts["w"], ts["b"], "silu", ts["dy"], ts["u"])
    buf = torch.empty(4 * 12 * 48 + 1, device=cuda, dtype=torch.bfloat16)
    off = [buf.clone()[1:].view(4, 12, 48).copy_(ts[n]) for n in ("x", "dy", "u")]
    assert off[0].data_ptr() % 16
    _check(off[0], 6, ts["w"], ts["b"], "silu", off[1], off[2])
    _check(ts["x"].transpose(0, 1), 6, ts["w"], ts["b"], "silu", ts["dy"].transpose(0, 1), ts["u"].transpose(0, 1))
    _check(ts["x"][:, ::2], 6, ts["w"], ts["b"], "silu", ts["dy"][:, 1::2], ts["u"][:, :6])
    for _ in range(2):  # equal bits every time
        assert all(torch.equal(p, q) for p, q in zip(a, _check(ts["x"], 6, ts["w"], ts["b"], "silu", ts["dy"], ts["u"])))
    x = ts["x"].float().requires_grad_(True)
    (dx,) = torch.autograd.grad(block.group_norm(x, 6).sum(), x)  # an expanded cotangent
    assert float(dx.abs().max()) <= 200 * 2.0**-24 * float(x.std())
    for shape in ((0, 5, 8), (3, 0, 8)):
        e = torch.zeros(shape, device=cuda, requires_grad=True)
        w = torch.ones(8, device=cuda, requires_grad=True)
        y = block.group_norm(e, 2, w)
        dx, dw = torch.autograd.grad(y.sum(), (e, w))
        assert y.shape == dx.shape == shape and bool((dw == 0).all())


def test_gradients_by_differences(cuda):
    _say("group_norm gradcheck")
    g = torch.Generator(cuda).manual_seed(5)
    x, w, b = (torch.randn(*s, generator=g, device=cuda, dtype=torch.float64, requires_grad=True) for s in ((2, 3, 6), (6,), (6,)))
    for act in (None, "silu"):
        for args in ((x, w, b), (x, w), (x,)):
            fn = lambda *t: block.group_norm(t[0], 2, *t[1:], activation=act)  # noqa: E731, B023
            assert torch.autograd.gradcheck(fn, args)
            assert torch.autograd.gradgradcheck(fn, args)
    (dx,) = torch.autograd.grad(block.group_norm(x, 2, w, b).pow(2).sum(), x, create_graph=True)
    (gx,) = torch.autograd.grad(dx.pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_a_grid_past_32_bit_offsets(cuda):
    _say("group_norm 64-bit offsets")
    B, L, C = 2, (1 << 20) + 9, 1024
    x = torch.empty(B, L, C, device=cuda, dtype=torch.bfloat16).normal_(generator=torch.Generator(cuda).manual_seed(1))
    assert x.numel() >= 1 << 31
    y = block.group_norm(x, 8, activation="silu")
    ref = _plain(x[1:, :, -128:].double(), 1, None, None, "silu")
    assert float((y[1:, :, -128:] - ref).abs().max()) <= 2.0**-8 * float(ref.abs().max())


# -- a training step's operators together ------------------------------------------------------------------------------


def _model(cuda, **kw):
    kw = dict(hidden_size=64, num_heads=4, grid=(4, 4), vocab_size=7, norm="group", norm_groups=4) | kw
    return en.build(en.EnergyConfig(**kw), cuda, seed=3)


def _batch(cuda, B=3, L=16, C=64, V=7):
    g = torch.Generator(cuda).manual_seed(6)
    x = torch.randint(0, V, (B, L), generator=g, device=cuda)
    z = torch.randn(B, L, C, generator=g, device=cuda)
    teacher = torch.randn(B, L, 3, generator=g, device=cuda).sort(-1, descending=True).values, torch.rand(B, L, V, generator=g, device=cuda).topk(3, -1).indices
    return x, z, teacher


def _ce_distill(logits, teacher, T):
    """The distillation loss in plain torch ops."""
    values, ids = teacher
    p = torch.softmax(values / T, -1)
    logq = torch.log_softmax(logits / T, -1).gather(-1, ids)
    return T * T * (p * (torch.log(p) - logq)).sum(-1).mean()


def test_distilled_step_of_an_energy_with_group_norms(cuda, monkeypatch):
    """``train_step`` with the embedding, the group norms inside graded descent and the distillation loss, fp32, against the
    same network with each in plain torch ops. Bound 1e-4 relative: two graded steps through two blocks are some 10^3
    roundings of 2^-24 in a row."""
    _say("distilled step")
    x, z, teacher = _batch(cuda)
    fused, dec = _model(cuda, block_impl="fused", embed_impl="fused")
    plain, dec2 = _model(cuda)
    plain.load_state_dict(fused.state_dict())
    dec2.load_state_dict(dec.state_dict())
    loss = en.train_step(fused, dec, x, z, None, steps=2, teacher=teacher, temperature=2.0)
    monkeypatch.setattr(tokens, "distill_loss", lambda lg, v, i, temperature: _ce_distill(lg, (v, i), temperature))
    ref = en.train_step(plain, dec2, x, z, None, steps=2, teacher=teacher, temperature=2.0)
    assert abs(float(loss) - float(ref)) <= 1e-4 * abs(float(ref))
    for (n, p), q in zip([*fused.named_parameters(), *dec.named_parameters()], [*plain.parameters(), *dec2.parameters()]):
        if q.grad is None:
            assert p.grad is None, n
            continue
        assert float((p.grad - q.grad).norm()) <= 1e-4 * float(q.grad.norm().clamp(min=1e-6)), n


def test_compiled_gradient_of_an_energy_with_group_norms(cuda):
    """The energy's gradient under torch.compile agrees with eager to second order (the gate that training runs)."""
    _say("compiled group norm")
    model, _ = _model(cuda, block_impl="fused", embed_impl="fused")
    x, z, _ = _batch(cuda)
    errs = en.verify_compiled_energy_grad(model, en.compiled_energy_grad(model), z, model.puzzle_embedding(x, z.dtype))
    assert max(errs.values()) < 1e-3


def test_distilled_step_replays(cuda):
    """The bf16 step captured, replayed on new contents with eager work between, equal to the eager step every time."""
    _say("distilled step graph")
    x, z, teacher = _batch(cuda, B=8)
    z = z.bfloat16()
    model, dec = _model(cuda, block_impl="fused", embed_impl="fused", rope_impl="fused")
    params = [p for p in [*model.parameters(), *dec.parameters()]]

    def step():
        for p in params:
            p.grad = None
        return en.train_step(model, dec, x, z, None, steps=2, teacher=teacher, temperature=2.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    grads = [p.grad for p in params]
    for turn in range(3):
        x.copy_((x + turn) % 7)
        z.mul_(0.9)
        ref = step()
        want = [p.grad for p in params]
        for g in grads:
            if g is not None:
                g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ref, loss)
        for g, w in zip(grads, want):
            assert (g is None) == (w is None) and (g is None or torch.equal(g, w))
