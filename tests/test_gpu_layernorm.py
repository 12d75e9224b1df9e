"""GPU parity of the layer norm (``ebr_amd.block.layer_norm``) and its first and second derivatives against the closed forms
in 64 bits on the same inputs, and by differences.

Tolerances: half a step of the output's type, and for what comes before it (u = 2^-24; fp64: 2^-53) a multiple of u times the
size of the terms that an output adds up, each taken without its sign. A sum over a row of C has chains of at most
``_depth(C)`` additions (a thread's own, at most 8 vectors of 8, then 16 over lanes and waves; rows of more than 32,768, C /
1024 a thread), so each mean is off by that many u of the mean size of its terms, the variance by as much and r by half of it;
h, r and the means enter each output at most twice a term, next to fewer than 20 roundings of its own. A weight's gradient
adds up at most all rows, one after another."""

import pytest
import torch

from ebr_amd import block

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-24, torch.float16: 2.0**-24, torch.float64: 2.0**-53}
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float64: 2.0**-53}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _depth(C):
    return 80 + C // 1024


def _mean(v):
    return v.mean(-1, keepdim=True)


def _forms(x, w, b, dy, u, uw, ub):
    """Outputs (y, dx, dw, db, gx, gdy, gw) and the sizes of their terms, in 64 bits."""
    C = x.shape[-1]
    x, dy, u = (t.double().reshape(-1, C) for t in (x, dy, u))
    w = torch.ones(C, device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, device=x.device, dtype=torch.float64) if b is None else b.double()
    uw, ub = (torch.zeros_like(w) if t is None else t.double() for t in (uw, ub))
    r = ((x - _mean(x)).square().mean(-1, keepdim=True) + EPS).rsqrt()
    h = (x - _mean(x)) * r
    k, t = w * dy, uw * dy

    def project(v):
        return r * (v - _mean(v) - h * _mean(v * h))

    def project_size(v):
        return r * (v + _mean(v) + ha * _mean(v * ha))

    kh, uh = _mean(k * h), _mean(u * h)
    along = _mean(k * u) - _mean(k) * _mean(u) - uh * kh
    out = [w * h + b, project(k), (dy * h).sum(0), dy.sum(0),
           project(t - r * (u * kh + k * uh)) - r * r * h * along, w * project(u) + uw * h + ub, (dy * project(u)).sum(0)]
    ha = h.abs() + _mean(h.abs())  # with the mean's error in it
    ka, ua, ta, da, wa = k.abs(), u.abs(), t.abs(), dy.abs(), w.abs()
    kha, uha = _mean(ka * ha), _mean(ua * ha)
    size = [wa * ha + b.abs(), project_size(ka), (da * ha).sum(0), da.sum(0),
            project_size(ta) + r * r * (ha * (3 * uha * kha + _mean(ka * ua) + _mean(ka) * _mean(ua))
                                        + kha * (ua + _mean(ua)) + uha * (ka + _mean(ka))),
            wa * project_size(ua) + uw.abs() * ha + ub.abs(), (da * project_size(ua)).sum(0)]
    return out, size


def _run(x, w, b, dy, u, uw, ub, eps=EPS):
    x, dy = x.detach().requires_grad_(True), dy.detach().requires_grad_(True)
    ps = [None if p is None else p.detach().requires_grad_(True) for p in (w, b)]
    y = block.layer_norm(x, *ps, eps)
    some = [p for p in ps if p is not None]
    first = list(torch.autograd.grad(y, [x, *some], dy, create_graph=True))
    dx, rest = first[0], first[1:]
    dw = rest.pop(0) if w is not None else None
    db = rest.pop(0) if b is not None else None
    pairs = [(o, c) for o, c in ((dx, u), (dw, uw), (db, ub)) if o is not None and c is not None]
    gx, gdy, *gw = torch.autograd.grad([o for o, _ in pairs], [x, dy, *([ps[0]] if w is not None else [])], [c for _, c in pairs])
    return [None if t is None else t.detach() for t in (y, dx, dw, db, gx, gdy, gw[0] if gw else None)]


NAMES = ("y", "dx", "dw", "db", "gx", "gdy", "gw")


def _check(x, w, b, dy, u, uw=None, ub=None):
    got = _run(x, w, b, dy, u, uw, ub)
    want, size = _forms(x, w, b, dy, u, uw, ub)
    C = x.shape[-1]
    rows = x.numel() // C
    for name, g, r, s in zip(NAMES, got, want, size):
        if g is None:
            continue
        param = name in ("dw", "db", "gw")
        p = {"dw": w, "gw": w, "db": b}.get(name)
        assert g.dtype == (p.dtype if param else x.dtype) and g.shape == (p.shape if param else x.shape), name
        chain = {"y": 1, "dx": 3, "dw": 2, "db": 0, "gx": 6, "gdy": 4, "gw": 4}[name] * _depth(C) + 60 + (rows if param else 0)
        r, s = r.reshape(g.shape), s.reshape(g.shape)
        off = (g.double() - r).abs() - (HALF[g.dtype] * r.abs() * (1 + 1e-6) + U[x.dtype] * chain * s + 1e-300)
        assert bool((off <= 0).all()), (name, float(off.max()), float(r.abs().max()))
    return got


def _inputs(dev, shape, dtype, seed=0, pt=torch.float32):
    g = torch.Generator(dev).manual_seed(seed)

    def randn(*s, t=dtype):
        return torch.randn(s, generator=g, device=dev, dtype=torch.float64).to(t)

    C = shape[-1]
    return dict(x=(randn(*shape, t=torch.float64) + 0.5 * randn(C, t=torch.float64)).to(dtype), dy=randn(*shape), u=randn(*shape),
                w=1 + 0.3 * randn(C, t=pt), b=randn(C, t=pt), uw=randn(C, t=pt), ub=randn(C, t=pt))


@pytest.fixture
def cuda():
    return torch.device("cuda", 0)


# 16, 32 and 64 threads a row with whole vectors, one to four vectors; 256 and 1,024 threads; single elements at each; rows
# through two kernels, of vectors and of single elements
@pytest.mark.parametrize("C", [1, 2, 8, 64, 100, 128, 136, 255, 256, 512, 520, 777, 1032, 1536, 2048, 2056, 4096, 5003, 8200, 9001, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_widths(cuda, C, dtype):
    _say(f"layer_norm C={C} {dtype}")
    ts = _inputs(cuda, (37 if C < 3000 else 9, C), dtype, seed=C, pt=torch.float64 if dtype == torch.float64 else torch.float32)
    _check(ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"], ts["uw"], ts["ub"])


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 81, 4099, 20000])
@pytest.mark.parametrize("C", [48, 512, 777])
def test_rows(cuda, rows, C):
    _say(f"layer_norm rows={rows} C={C}")
    ts = _inputs(cuda, (rows, C), torch.bfloat16, seed=rows)
    _check(ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"])


@pytest.mark.parametrize("have,pt", [("", torch.float32), ("w", torch.bfloat16), ("b", torch.float16), ("wb", torch.bfloat16), ("wb", torch.float64)])
@pytest.mark.parametrize("C", [96, 40000])
def test_parameters_and_their_types(cuda, have, pt, C):
    _say(f"layer_norm parameters {have!r} {pt} C={C}")
    ts = _inputs(cuda, (3, 5, C), torch.bfloat16, seed=1, pt=pt)
    w, b = (ts[n] if n in have else None for n in "wb")
    _check(ts["x"], w, b, ts["dy"], ts["u"], ts["uw"] if w is not None else None, ts["ub"] if b is not None else None)


def test_weight_and_bias_of_two_types(cuda):
    _say("layer_norm mixed parameters")
    ts = _inputs(cuda, (7, 64), torch.bfloat16, seed=2)
    _check(ts["x"], ts["w"].bfloat16(), ts["b"], ts["dy"], ts["u"])


@pytest.mark.parametrize("C", [96, 1000, 5003, 40000])
def test_rows_of_one_value_and_far_from_zero(cuda, C):
    """A row of one value gives the bias, whatever the value. Around 1000 with deviation 1, x is itself exact here, so h stays
    within the general bound times the 1000 of the first mean's error, which the second mean takes out again: 3,000 u."""
    _say(f"layer_norm constant rows C={C}")
    b = torch.linspace(-1, 1, C, device=cuda)
    for dtype in (torch.float32, torch.bfloat16):
        for value in (0.0, 3.0, 1000.1, -3e4, 7e-3, 1e20, torch.finfo(dtype).max, torch.finfo(dtype).min):
            x = torch.full((3, C), value, device=cuda, dtype=dtype).requires_grad_(True)
            y = block.layer_norm(x, None, b)
            assert torch.equal(y, b.to(dtype).expand(3, C)), value
            (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
            assert bool(torch.isfinite(dx).all()), value
    x = 1000 + torch.randn(4, C, generator=torch.Generator(cuda).manual_seed(C), device=cuda)
    ref = _forms(x, None, None, x, x, None, None)[0][0]
    assert float((block.layer_norm(x) - ref).abs().max()) <= 3000 * 2.0**-24


@pytest.mark.parametrize("C", [64, 512, 777, 9001])
def test_nan_and_infinity_stay_in_their_row(cuda, C):
    _say(f"layer_norm nan C={C}")
    ts = _inputs(cuda, (6, C), torch.float32, seed=3)
    good = _run(ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"], None, None)
    for bad in (float("nan"), float("inf")):
        x = ts["x"].clone()
        x[2, C // 2] = bad
        got = _run(x, ts["w"], ts["b"], ts["dy"], ts["u"], None, None)
        for i in (0, 1, 4, 5):
            assert bool(torch.isnan(got[i][2]).any())
            keep = torch.arange(6, device=cuda) != 2
            assert torch.equal(got[i][keep], good[i][keep])


def test_views_streams_and_empty_calls(cuda):
    _say("layer_norm views")
    ts = _inputs(cuda, (12, 48), torch.bfloat16, seed=3)
    a = _check(ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"])
    off = [torch.empty(12 * 48 + 1, device=cuda, dtype=torch.bfloat16)[1:].view(12, 48).copy_(ts[n]) for n in ("x", "dy", "u")]
    assert off[0].data_ptr() % 16
    _check(off[0], ts["w"], ts["b"], off[1], off[2])
    _check(ts["x"].t()[:12], ts["w"][:12], ts["b"][:12], ts["dy"].t()[:12], ts["u"].t()[:12])
    _check(ts["x"][::2, ::3], ts["w"][::3], ts["b"][::3], ts["dy"][1::2, ::3], ts["u"][:6, :16])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # equal bits every time, on any stream
        again = _run(ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"], None, None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, again))
    x = ts["x"].float().requires_grad_(True)
    (dx,) = torch.autograd.grad(block.layer_norm(x).sum(), x)  # an expanded cotangent
    assert float(dx.abs().max()) <= 400 * 2.0**-24 * 4
    e, w = torch.zeros(0, 8, device=cuda, requires_grad=True), torch.ones(8, device=cuda, requires_grad=True)
    y = block.layer_norm(e, w)
    dx, dw = torch.autograd.grad(y.sum(), (e, w))
    assert y.shape == dx.shape == (0, 8) and bool((dw == 0).all())


def test_gradients_by_differences(cuda):
    _say("layer_norm gradcheck")
    g = torch.Generator(cuda).manual_seed(5)
    x, w, b = (torch.randn(*s, generator=g, device=cuda, dtype=torch.float64, requires_grad=True) for s in ((3, 5), (5,), (5,)))
    for args in ((x, w, b), (x, w), (x,)):
        assert torch.autograd.gradcheck(block.layer_norm, args)
        assert torch.autograd.gradgradcheck(block.layer_norm, args)
    (dx,) = torch.autograd.grad(block.layer_norm(x, w, b).pow(2).sum(), x, create_graph=True)
    (gx,) = torch.autograd.grad(dx.pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_python_path_gives_the_same_bits(cuda, monkeypatch):
    """The ops of the Python layer, which runs where the native host path does not, and gradients under a transform."""
    _say("layer_norm python path")
    ts = _inputs(cuda, (20, 72), torch.bfloat16, seed=4)
    args = (ts["x"], ts["w"], ts["b"], ts["dy"], ts["u"], ts["uw"], ts["ub"])
    native = _run(*args)
    x = ts["x"].float().requires_grad_(True)
    y = block.layer_norm(x, ts["w"], ts["b"])
    cots = torch.stack([ts["dy"].float(), ts["u"].float()])
    (batched,) = torch.autograd.grad(y, x, cots, is_grads_batched=True, retain_graph=True)
    for c, d in zip(cots, batched):
        assert torch.equal(torch.autograd.grad(y, x, c, retain_graph=True)[0], d)
    monkeypatch.setattr(block._host, "module", lambda: None)
    assert all(torch.equal(p, q) for p, q in zip(native, _run(*args)))


def test_rows_past_32_bit_offsets(cuda):
    _say("layer_norm 64-bit offsets")
    C = 2048
    rows = (1 << 20) + 9
    x = torch.empty(rows, C, device=cuda, dtype=torch.bfloat16).normal_(generator=torch.Generator(cuda).manual_seed(1)).requires_grad_(True)
    assert x.numel() >= 1 << 31
    y = block.layer_norm(x)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    for part in (slice(rows - 20, rows), slice(0, 20)):
        _, want = _run(x[part], None, None, x.detach()[part], x.detach()[part], None, None)[:2]
        assert torch.equal(dx[part], want)


def test_replays(cuda):
    """Both derivatives captured, replayed on new contents with eager work between, equal to eager every time."""
    _say("layer_norm graph")
    ts = _inputs(cuda, (300, 264), torch.bfloat16, seed=9)
    args = [ts[n] for n in ("x", "w", "b", "dy", "u", "uw", "ub")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(*args)
    for turn in range(3):
        for t in args:
            t.copy_(t.roll(turn + 1, 0))
        want = _run(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
