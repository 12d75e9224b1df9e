"""GPU parity of the gated projection (``ebr_amd.block.swiglu_linear``) and its first and second derivatives against the closed
forms in 64 bits on the same inputs, by differences, and against its parts.

Tolerances, elementwise, with u = 2^-24 (fp64: 2^-53) and half a step H of the 16-bit type (u for the others): a product over K
terms is off by at most (K + 2) u of the sum of its terms without their signs; the activation and its derivatives are at most
1.1 in slope, and their own roundings (the exponential's argument among them, |g| of its size) fewer than 16 (1 + |g|) of
theirs; what passes through a rounded [dg|du] or [gg|gu] is H off there, and every output H at the end."""

import pytest
import torch

from ebr_amd import block, linear
from ebr_amd.fused_attn.loader import hip_library

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-24, torch.float16: 2.0**-24, torch.float64: 2.0**-53}
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float64: 2.0**-53}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float64: 1e-300}


def _say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.fixture
def cuda():
    return torch.device("cuda", 0)


def _inputs(dev, N, C, I, dtype, seed=0):
    g = torch.Generator(dev).manual_seed(seed)

    def randn(*s, scale=1.0):
        return (scale * torch.randn(s, generator=g, device=dev, dtype=torch.float64)).to(dtype)

    return dict(x=randn(N, C), w=randn(2 * I, C, scale=C**-0.5), dy=randn(N, I), c=randn(N, C))


def _forms(x, w, dy, c):
    """(y, dx, dw, gx, gdy, gw) and how far each may be off, in 64 bits."""
    dt = x.dtype
    u, H, tiny = U[dt], HALF[dt], TINY[dt]
    mid = 2 * u if dt in (torch.float32, torch.float64) else H
    x, w, dy, c = (t.double() for t in (x, w, dy, c))
    N, C = x.shape
    I = w.shape[0] // 2

    def product(a, ea, b, eb):
        """a b^T of operands that are off by ea and eb."""
        K = a.shape[1]
        e = (K + 2) * u * (a.abs() @ b.abs().T)
        if ea is not None:
            e = e + ea @ (b.abs().T + (eb.T if eb is not None else 0))
        if eb is not None:
            e = e + a.abs() @ eb.T
        return a @ b.T, e

    gu, eg = product(x, None, w, None)
    cc, ec = product(c, None, w, None)
    g, up, cg, cu = gu[:, :I], gu[:, I:], cc[:, :I], cc[:, I:]
    e_g, e_u, e_cg, e_cu = eg[:, :I], eg[:, I:], ec[:, :I], ec[:, I:]
    s = torch.sigmoid(g)
    f0, f1, f2 = g * s, s * (1 + g * (1 - s)), s * (1 - s) * (2 + g * (1 - 2 * s))
    own = 16 * u * (1 + g.abs())
    e0, e1, e2 = e_g * 1.1 + own * (f0.abs() + s), e_g * 0.5 + own * (s * (1 + g.abs())), e_g * 0.5 + own * (s * (2 + g.abs()))

    def times(*fs):
        """A product of values with their errors."""
        v, e = fs[0]
        for w_, ew in fs[1:]:
            v, e = v * w_, e * w_.abs() + v.abs() * ew + e * ew
        return v, e + 4 * u * v.abs()

    def plus(*fs):
        return sum(f[0] for f in fs), sum(f[1] + 2 * u * f[0].abs() for f in fs)

    zero = torch.zeros_like(dy)
    F0, F1, F2, UP, DY, CG, CU = (f0, e0), (f1, e1), (f2, e2), (up, e_u), (dy, zero), (cg, e_cg), (cu, e_cu)
    y = times(F0, UP)
    d = [torch.cat(p, 1) for p in zip(times(DY, UP, F1), times(DY, F0))]
    gg = plus(times(CG, DY, UP, F2), times(CU, DY, F1))
    e = [torch.cat(p, 1) for p in zip(gg, times(CG, DY, F1))]
    gdy = plus(times(CG, UP, F1), times(CU, F0))
    d[1], e[1] = d[1] + mid * d[0].abs() + tiny, e[1] + mid * e[0].abs() + tiny
    dx = product(*d, w.T, None)
    dw = product(d[0].T, d[1].T, x.T, None)
    gx = product(*e, w.T, None)
    gw = plus(product(e[0].T, e[1].T, x.T, None), product(d[0].T, d[1].T, c.T, None))
    out = (y, dx, dw, gx, gdy, gw)
    return [v for v, _ in out], [er + H * (v.abs() + er) + tiny for v, er in out]


NAMES = ("y", "dx", "dw", "gx", "gdy", "gw")


def _run(x, w, dy, c):
    x, w, dy = (t.detach().requires_grad_(True) for t in (x, w, dy))
    y = block.swiglu_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy.detach(), retain_graph=True)
    (dx2,) = torch.autograd.grad(y, x, dy, create_graph=True)
    assert torch.equal(dx.nan_to_num(), dx2.nan_to_num())
    gx, gdy, gw = torch.autograd.grad(dx2, (x, dy, w), c)
    with torch.no_grad():
        assert torch.equal(block.swiglu_linear(x, w).nan_to_num(), y.nan_to_num())
    return [t.detach() for t in (y, dx, dw, gx, gdy, gw)]


def _check(x, w, dy, c):
    got = _run(x, w, dy, c)
    shapes = dict(zip(NAMES, (dy.shape, x.shape, w.shape, x.shape, dy.shape, w.shape)))
    want, tol = _forms(x.reshape(-1, x.shape[-1]), w, dy.reshape(-1, dy.shape[-1]), c.reshape(-1, c.shape[-1]))
    for name, g, r, t in zip(NAMES, got, want, tol):
        assert g.dtype == x.dtype and g.shape == shapes[name], name
        off = (g.double().reshape(r.shape) - r).abs() - t
        assert bool((off <= 0).all()), (name, float(off.max()), float(r.abs().max()))
    return got


# one row and few, less and more than a tile, tiles of 64, 128 and 256, odd numbers of stages, widths off the vectors, one column
@pytest.mark.parametrize("N,C,I", [
    (1, 64, 32), (1, 2048, 520), (2, 8, 8), (3, 1, 1), (5, 7, 9), (33, 72, 40), (64, 128, 64), (65, 130, 66), (81, 256, 768),
    (130, 520, 264), (200, 64, 3), (257, 333, 129), (700, 192, 1000), (1500, 264, 1032), (5000, 136, 520), (20000, 40, 24),
])  # fmt: skip
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sizes(cuda, N, C, I, dtype):
    _say(f"swiglu_linear {N} {C} {I} {dtype}")
    _check(*_inputs(cuda, N, C, I, dtype, seed=N).values())


# up to 32 rows, whose gates read the weight straight into registers: rows off 16, a last turn that is not full, many turns, widths off
# 16 and off the vectors
@pytest.mark.parametrize("N", [1, 3, 15, 16, 17, 31, 32])
@pytest.mark.parametrize("C,I", [(8, 8), (72, 24), (520, 16), (2056, 40), (5000, 1000), (9, 33), (1031, 15), (2047, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_few_rows(cuda, N, C, I, dtype):
    _say(f"swiglu_linear few rows {N} {C} {I} {dtype}")
    ts = _inputs(cuda, N, C, I, dtype, seed=N + C)
    y = _check(**ts)[0]
    one = block.swiglu_linear(ts["x"][N - 1], ts["w"])  # a row alone, of one dimension: the same sums
    assert N > 16 or torch.equal(one, y[N - 1])


@pytest.mark.parametrize("N,C,I", [(1, 5, 3), (70, 65, 66), (129, 31, 40)])
def test_fp64(cuda, N, C, I):
    _say(f"swiglu_linear fp64 {N} {C} {I}")
    _check(*_inputs(cuda, N, C, I, torch.float64, seed=N).values())


def test_the_large_tiles(cuda):
    """Tiles of 256 in every product: many rows, many columns, and rows split among workgroups in the weight's gradient."""
    _say("swiglu_linear large tiles")
    for N, C, I in ((6144, 2048, 1280), (40000, 520, 264), (9000, 1024, 2056)):
        _check(*_inputs(cuda, N, C, I, torch.bfloat16, seed=C).values())


def test_more_tiles_than_a_round(cuda):
    """The weight's gradient in 288 tiles of 256, the last 32 of which split their rows, some with an edge."""
    _say("swiglu_linear more tiles than a round")
    a = _check(*_inputs(cuda, 4100, 4096, 2184, torch.bfloat16, seed=6).values())
    b = _run(*_inputs(cuda, 4100, 4096, 2184, torch.bfloat16, seed=6).values())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("N,C,I", [(40, 1, 1), (33, 9, 8), (700, 1031, 8), (3000, 264, 521), (5000, 263, 1025)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_widths_off_the_vectors(cuda, N, C, I, dtype):
    """Copies with zeros up to whole chunks, of either width and of both; nothing of them is left in the outputs."""
    _say(f"swiglu_linear off the vectors {N} {C} {I} {dtype}")
    ts = _inputs(cuda, N, C, I, dtype, seed=I)
    a = _check(**ts)
    off = {n: torch.empty(t.numel() + 1, device=cuda, dtype=dtype)[1:].view(t.shape).copy_(t) for n, t in ts.items()}
    assert all(torch.equal(x, y) for x, y in zip(a, _run(**off)))


def test_refused_alignment(cuda):
    """Tensors off 16 bytes where the widths are whole, and a scratch that is missing, at the C entry."""
    lib = hip_library()
    x, w, y = (torch.zeros(n + 8, device=cuda, dtype=torch.bfloat16) for n in (40 * 16, 48 * 16, 40 * 24))
    p = [t.data_ptr() for t in (x, w, y)]
    call = lambda *a: lib.ebr_block_swiglu_linear(1, 40, 16, 24, *a, 0, torch.cuda.current_stream().cuda_stream)  # noqa: E731
    codes = {call(p[0] + 2, p[1], p[2]), call(p[0], p[1] + 2, p[2]), call(p[0], p[1], p[2] + 8)}
    assert len(codes) == 1 and 0 not in codes and call(*p) == 0
    assert lib.ebr_block_swiglu_linear(1, 40, 15, 24, *p, 0, 0) != 0  # padded rows want scratch
    assert lib.ebr_block_swiglu_linear_scratch(1, 0, 40, 16, 24) == 0 < lib.ebr_block_swiglu_linear_scratch(1, 0, 40, 15, 24)
    torch.cuda.synchronize()


def test_large_gates(cuda):
    """Gates of some hundreds, whose exponentials leave the range on either side."""
    _say("swiglu_linear large gates")
    ts = _inputs(cuda, 96, 64, 40, torch.bfloat16, seed=2)
    ts["x"] = ts["x"] * 100
    _check(*ts.values())
    x = torch.full((3, 8), 1e4, device=cuda)
    w = torch.cat([torch.ones(4, 8, device=cuda), torch.ones(4, 8, device=cuda)])
    assert torch.equal(block.swiglu_linear(-x, w).abs(), torch.zeros(3, 4, device=cuda))  # silu of -80,000 is -0
    assert torch.equal(block.swiglu_linear(x, w), torch.full((3, 4), 6.4e9, device=cuda))


def test_nan_and_infinity_stay_in_their_row(cuda):
    _say("swiglu_linear nan")
    for N, C, I in ((70, 72, 40), (700, 264, 520)):
        ts = _inputs(cuda, N, C, I, torch.bfloat16, seed=4)
        good = _run(**ts)
        for bad in (float("nan"), float("inf")):
            x = ts["x"].clone()
            x[5, 3] = bad
            got = _run(x, ts["w"], ts["dy"], ts["c"])
            keep = torch.arange(N, device=cuda) != 5
            for i in (0, 1, 3, 4):
                assert bool(torch.isnan(got[i][5]).any())
                assert torch.equal(got[i][keep], good[i][keep])


def test_views_shapes_streams_and_empty_calls(cuda):
    _say("swiglu_linear views")
    ts = _inputs(cuda, 66, 48, 40, torch.bfloat16, seed=3)
    a = _check(**ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # equal bits every time, on any stream
        again = _run(**ts)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, again))
    off = {n: torch.empty(t.numel() + 1, device=cuda, dtype=t.dtype)[1:].view(t.shape).copy_(t) for n, t in ts.items()}
    assert off["w"].data_ptr() % 16
    _check(**off)
    _check(ts["x"].t().contiguous().t(), ts["w"].t().contiguous().t(), ts["dy"][:, ::2].repeat(1, 2), ts["c"])
    shaped = {n: t if n == "w" else t.view(2, 3, 11, -1) for n, t in ts.items()}
    assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(_run(**shaped), a))
    x = ts["x"].clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(block.swiglu_linear(x, ts["w"]).sum(), x)  # an expanded cotangent
    want, tol = _forms(ts["x"], ts["w"], torch.ones_like(ts["dy"]), ts["c"])
    assert bool(((dx.double() - want[1]).abs() <= tol[1]).all())
    e, w = torch.zeros(0, 48, device=cuda, dtype=torch.bfloat16, requires_grad=True), ts["w"].clone().requires_grad_(True)
    y = block.swiglu_linear(e, w)
    dx, dw = torch.autograd.grad(y.sum(), (e, w))
    assert y.shape == (0, 40) and dx.shape == (0, 48) and bool((dw == 0).all())


def test_gradients_by_differences(cuda):
    _say("swiglu_linear gradcheck")
    g = torch.Generator(cuda).manual_seed(5)
    x, w = (torch.randn(*s, generator=g, device=cuda, dtype=torch.float64, requires_grad=True) for s in ((3, 5), (8, 5)))
    assert torch.autograd.gradcheck(block.swiglu_linear, (x, w))
    assert torch.autograd.gradgradcheck(block.swiglu_linear, (x, w))
    assert torch.autograd.gradgradcheck(lambda t: block.swiglu_linear(t, w.detach()), (x,))
    assert torch.autograd.gradgradcheck(lambda t: block.swiglu_linear(x.detach(), t), (w,))
    (dx,) = torch.autograd.grad(block.swiglu_linear(x, w).pow(2).sum(), x, create_graph=True)
    (gx,) = torch.autograd.grad(dx.pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_python_path_gives_the_same_bits(cuda, monkeypatch):
    _say("swiglu_linear python path")
    ts = _inputs(cuda, 40, 72, 48, torch.bfloat16, seed=6)
    native = _run(**ts)
    x = ts["x"].clone().requires_grad_(True)
    y = block.swiglu_linear(x, ts["w"])
    cots = torch.stack([ts["dy"], ts["dy"].flip(0)])
    (batched,) = torch.autograd.grad(y, x, cots, is_grads_batched=True, retain_graph=True)
    for c, d in zip(cots, batched):
        assert torch.equal(torch.autograd.grad(y, x, c, retain_graph=True)[0], d)
    monkeypatch.setattr(block._host, "module", lambda: None)
    monkeypatch.setattr(linear._host, "module", lambda: None)
    with torch.no_grad():
        y = block.swiglu_linear(ts["x"], ts["w"])
    dx, dw = torch.ops.ebr_fused.block_swiglu_linear_bwd(ts["x"], ts["w"], ts["dy"], True, True)
    gx, gdy, gw = torch.ops.ebr_fused.block_swiglu_linear_bwd2(ts["x"], ts["w"], ts["dy"], ts["c"], True, True)
    again = [y, dx, dw, gx, gdy, gw]
    assert all(torch.equal(p, q) for p, q in zip(native, again))
    x, w = (ts[n].float().requires_grad_(True) for n in ("x", "w"))
    y = block.swiglu_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), ts["dy"].float(), create_graph=True)
    ((dx * ts["c"].float()).sum() + dw.square().sum()).backward()
    xr, wr = (t.detach().double().requires_grad_(True) for t in (x, w))
    yr = block.swiglu(xr @ wr.t())
    dxr, dwr = torch.autograd.grad(yr, (xr, wr), ts["dy"].double(), create_graph=True)
    ((dxr * ts["c"].double()).sum() + dwr.square().sum()).backward()
    for a, r in ((dx, dxr), (dw, dwr), (x.grad, xr.grad), (w.grad, wr.grad)):  # a few hundred roundings in a row
        assert float((a - r).norm()) <= 1e-4 * float(r.norm())


def test_a_weight_past_32_bit_offsets(cuda):
    """[dg|du] of more than 2^31 elements, and the weight's gradient over its rows."""
    _say("swiglu_linear 64-bit offsets")
    N, C, I = (1 << 19) + 77, 64, 2104
    ts = _inputs(cuda, 4096, C, I, torch.bfloat16, seed=7)
    assert N * 2 * I >= 1 << 31
    x = torch.zeros(N, C, device=cuda, dtype=torch.bfloat16)
    dy = torch.zeros(N, I, device=cuda, dtype=torch.bfloat16)
    x[-4096:], dy[-4096:] = ts["x"], ts["dy"]
    x.requires_grad_(True)
    w = ts["w"].clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(block.swiglu_linear(x, w), (x, w), dy)
    want, tol = _forms(*ts.values())
    assert bool(((dx[-4096:].double() - want[1]).abs() <= tol[1]).all()) and float(dx[:-4096].abs().max()) == 0.0
    assert bool(((dw.double() - want[2]).abs() <= tol[2]).all())


@pytest.mark.parametrize("N,C,I", [(3000, 136, 264), (700, 133, 263), (5, 72, 40), (6, 1031, 1500)])
def test_replays(cuda, N, C, I):
    """All derivatives captured, replayed on new contents with eager work between, equal to eager every time."""
    _say(f"swiglu_linear graph {N} {C} {I}")
    ts = list(_inputs(cuda, N, C, I, torch.bfloat16, seed=9).values())

    def run():
        x, w, dy = (t.detach().requires_grad_(True) for t in ts[:3])
        y = block.swiglu_linear(x, w)
        first = torch.autograd.grad(y, (x, w), ts[2], retain_graph=True)
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        return [t.detach() for t in (y, *first, *torch.autograd.grad(dx, (x, dy, w), ts[3]))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for turn in range(3):
        for t in ts:
            t.copy_(t.roll(turn + 1, 0))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
