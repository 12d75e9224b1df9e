"""GPU parity of the optimizer's step (``ebr_amd.optim``) and the gradients' norm against the formulas in 64 bits on the same
inputs, and a training step of the energy network with the layer norm, the gated projection and the step together.

Tolerances, with u = 2^-24: a moment is two products and a sum of rounded factors, within 6 u of its terms' size (the second
squares a clipped gradient: 10 u); a parameter's change adds a root, a division and rounded factors to that, within 24 u of its
size, and the sum half a step of the parameter's type and u of its terms. Moments in 8 bits are taken in 64: their numbers are
exactly those of the rule, and the parameter is held to the bound above. A scale is that of the element that is largest in fp32,
rounded: another that fp32 does not tell from it, each moment being off by 4.5 u of its terms, may be larger by 9 u of these, that
is of the largest and twice the old largest times beta1; each root by 6 u, so by 12 u."""

import copy
import math

import pytest
import torch

from ebr_amd import energy as en
from ebr_amd import optim

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float64: 2.0**-53}
F8 = torch.float8_e4m3fn
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-6, weight_decay=0.05)


def _say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.fixture
def cuda():
    return torch.device("cuda", 0)


def _coded(x):
    """e4m3 numbers and scales of a moment."""
    b = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
    scale = b.abs().amax(1) / 448
    return (b / scale.clamp(min=1e-30)[:, None]).to(F8).view(-1)[: x.numel()].contiguous(), scale


def _inputs(dev, sizes, ptype=torch.float32, gtype=None, bits=32, seed=0, step=4, offset=0):
    """Lists for ``adamw_``; with ``offset``, views that begin so many elements into their memory."""
    gen = torch.Generator(dev).manual_seed(seed)
    wide = torch.float64 if ptype == torch.float64 else torch.float32

    def place(t):
        if not offset:
            return t
        room = torch.empty(t.numel() + offset, device=dev, dtype=torch.uint8 if t.dtype == F8 else t.dtype)
        room[offset:].copy_(t.view(room.dtype).reshape(-1))
        return room[offset:].view(t.dtype).view(t.shape)

    def randn(shape, dtype, scale):
        return (scale * torch.randn(shape, generator=gen, device=dev, dtype=torch.float64)).to(dtype)

    out = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], steps=[], scales=[] if bits == 8 else None)
    for k, s in enumerate(sizes):
        out["params"].append(place(randn(s, ptype, 0.3)))
        out["grads"].append(place(randn(s, gtype or ptype, 0.02)))
        n = out["params"][-1].numel()
        m, r = randn((n,), wide, 0.01), randn((n,), wide, 0.01).abs() + 0.004
        if bits == 8:
            (qm, sm), (qr, sr) = _coded(m), _coded(r)
            out["exp_avgs"].append(place(qm))
            out["exp_avg_sqs"].append(place(qr))
            out["scales"].append((sm, sr))
        else:
            out["exp_avgs"].append(place(m))
            out["exp_avg_sqs"].append(place(r.square()))
        out["steps"].append(torch.full((), step + k % 3, device=dev, dtype=torch.int64))
    return out


def _clone(ts):
    def one(t):
        return t.view(torch.uint8).clone().view(F8) if t.dtype == F8 else t.clone()

    return {n: None if v is None else [tuple(map(one, t)) if isinstance(t, tuple) else one(t) for t in v] for n, v in ts.items()}


def _quantized(x, t, start):
    """The numbers and scales that the rule gives moments x, in 64 bits."""
    n = x.numel()
    b = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    scale = b.abs().amax(1) / 448
    scale = torch.where(scale < 2.0**-126, torch.zeros_like(scale), scale)
    y = torch.where(scale[:, None] > 0, b.abs() / scale[:, None], torch.zeros_like(b)).view(-1)[:n]
    i = torch.arange(n, device=x.device)
    dither = ((i * 0x85EBCA77 + t * 0x9E3779B1 + start) % 2**32 // 256).double() / 2**24
    s = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0**-6))) - 3)
    q = (torch.floor(y / s + dither) * s).clamp(max=448)
    if start:
        q = torch.where(y > 0, q.clamp(min=2.0**-9), q)
    return torch.copysign(q, x), scale


def _check(ts, hyper, got_norm=None, max_norm=None, before=None):
    """``ts`` after a step from ``before``."""
    b1, b2 = hyper["betas"]
    lr, wd, eps = float(hyper["lr"]), hyper["weight_decay"], hyper["eps"]
    factor = 1.0
    if max_norm is not None:
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
        assert abs(float(got_norm) - norm) <= 2 * U * norm and got_norm.dtype == torch.float32 and got_norm.shape == ()
        factor = min(1.0, max_norm / (norm + 1e-6))
    eight = before["scales"] is not None
    for k, p0 in enumerate(before["params"]):
        t = int(before["steps"][k]) + 1
        assert int(ts["steps"][k]) == t
        u = 2.0**-53 if p0.dtype == torch.float64 else U
        p0d, g = p0.double().reshape(-1), before["grads"][k].double().reshape(-1) * factor
        m0, v0 = (before[n][k].float().double() if eight else before[n][k].double() for n in ("exp_avgs", "exp_avg_sqs"))
        m0, v0 = m0.reshape(-1), v0.reshape(-1)
        if eight:
            sm, sr = (s.double().repeat_interleave(256)[: g.numel()] for s in before["scales"][k])
            m0, v0 = m0 * sm, (v0 * sr).square()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g.square()
        ma = b1 * m0.abs() + (1 - b1) * g.abs()
        change = lr / (1 - b1**t) * m / (v.sqrt() / math.sqrt(1 - b2**t) + eps)
        change_a = lr / (1 - b1**t) * ma / (v.sqrt() / math.sqrt(1 - b2**t) + eps)
        p = p0d * (1 - lr * wd) - change
        # (fp16 below 2^-14 has steps of 2^-24 whatever the value: half of one is 2^-25)
        tol = HALF[p0.dtype] * p.abs() + (2.0**-25 if p0.dtype == torch.float16 else 0.0) + 3 * u * (p0d.abs() + change.abs()) + 24 * u * change_a + 1e-300
        off = (ts["params"][k].double().reshape(-1) - p).abs() - tol * (1 + 1e-6)
        assert off.numel() == 0 or float(off.max()) <= 0, (k, float(off.max()))
        if eight:
            for name, x, start, scale in (("exp_avgs", m, 0, 0), ("exp_avg_sqs", v.sqrt(), 2**31, 1)):
                q, s = _quantized(x, t, start)
                assert torch.equal(ts[name][k].float().double().reshape(-1), q), (k, name)
                near = 12 * U * s if scale else 9 * U * (s + 2 * b1 * before["scales"][k][0].double())
                assert bool(((ts["scales"][k][scale].double() - s).abs() <= 1.01 * U * s + near).all())
        else:
            assert bool(((ts["exp_avgs"][k].double().reshape(-1) - m).abs() <= 6 * u * ma + 1e-300).all())
            assert bool(((ts["exp_avg_sqs"][k].double().reshape(-1) - v).abs() <= 10 * u * v + 1e-300).all())


def _step(ts, **kw):
    return optim.adamw_(ts["params"], ts["grads"], ts["exp_avgs"], ts["exp_avg_sqs"], ts["steps"], scales=ts["scales"], **kw)


SIZES = {
    "one": [(1,)],
    "odd": [(3,), (255,), (256,), (257,), (1, 1), (4096,), (4097,), (5, 77), (0,), (513,)],
    "large": [(1 << 20, 3), (7,), (1000, 1001)],
    "many": [(17 * (k % 5) + 1,) for k in range(151)],
}
KINDS = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float64, torch.float64)]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_steps(cuda, sizes, kind, bits, max_norm):
    if bits == 8 and kind[0] == torch.float64:
        pytest.skip("fp64 parameters have fp64 moments")
    _say(f"adamw {sizes} {kind} {bits} {max_norm}")
    ts = _inputs(cuda, SIZES[sizes], *kind, bits=bits, seed=len(sizes))
    before = _clone(ts)
    norm = _step(ts, max_norm=max_norm, **HYPER)
    assert (norm is None) == (max_norm is None)
    _check(ts, HYPER, norm, max_norm, before)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_any_alignment(cuda, bits, offset):
    _say(f"adamw offset {offset} {bits}")
    for kind in ((torch.float32, torch.bfloat16), (torch.float16, torch.float16)):
        ts = _inputs(cuda, [(777,), (4, 1031), (256,)], *kind, bits=bits, offset=offset)
        before = _clone(ts)
        norm = _step(ts, max_norm=0.1, **HYPER)
        _check(ts, HYPER, norm, 0.1, before)


def test_kinds_together_and_a_learning_rate_on_the_device(cuda):
    _say("adamw mixed")
    parts = [_inputs(cuda, [(300,), (70, 11)], *kind, seed=k) for k, kind in enumerate(KINDS)]
    ts = {n: None if n == "scales" else sum((p[n] for p in parts), []) for n in parts[0]}
    before = _clone(ts)
    lr = torch.tensor(2.0**-8, device=cuda)
    norm = _step(ts, max_norm=0.3, **(HYPER | dict(lr=lr)))
    _check(ts, HYPER | dict(lr=2.0**-8), norm, 0.3, before)


def test_edges_of_the_numbers(cuda):
    """No clipping below the norm, a norm of zero, first steps, betas of 0, no decay; gradients that are not finite spoil what
    they touch and nothing beyond."""
    _say("adamw edges")
    ts = _inputs(cuda, [(1000,)], step=0)
    before = _clone(ts)
    hyper = HYPER | dict(betas=(0.0, 0.0), weight_decay=0.0)
    norm = _step(ts, max_norm=1e6, **hyper)
    _check(ts, hyper, norm, 1e6, before)
    for bits in (32, 8):
        ts = _inputs(cuda, [(1000,)], bits=bits)
        ts["grads"][0].zero_()
        before = _clone(ts)
        norm = _step(ts, max_norm=1.0, **HYPER)
        assert float(norm) == 0
        _check(ts, HYPER, norm, 1.0, before)
        for bad in (float("nan"), float("inf")):
            ts = _inputs(cuda, [(1000,), (300,)], bits=bits)
            ts["grads"][0][600] = bad
            good = _clone(ts)
            good["grads"][0][600] = 0.0
            _step(ts, **HYPER)
            _step(good, **HYPER)
            keep = torch.ones(1000, device=cuda, dtype=torch.bool)
            keep[600] = False
            assert not math.isfinite(float(ts["params"][0][600])) or bad == float("inf")
            assert torch.equal(ts["params"][0][keep], good["params"][0][keep]) and torch.equal(ts["params"][1], good["params"][1])
            if bits == 8:
                keep[512:768] = False  # the block of one scale
            for n in ("exp_avgs", "exp_avg_sqs"):
                assert torch.equal(ts[n][0].float()[keep], good[n][0].float()[keep])
                assert torch.equal(ts[n][1].float(), good[n][1].float())
        ts = _inputs(cuda, [(1000,)], bits=bits)
        ts["grads"][0][1] = float("nan")
        assert math.isnan(float(_step(ts, max_norm=1.0, **HYPER))) and bool(torch.isnan(ts["params"][0]).all())


def test_eight_bits_follow_their_rule_and_stick_nowhere(cuda):
    """Many steps, each to the bit what the rule gives from the one before; then gradients of half of the elements stop. A root
    of k steps (8 to 15) decays to 0.995 k, and is rounded down once t falls below 0.04: the t of 250 steps in a row lie at most
    2.62 / 250 apart (a golden-ratio sequence), so every root gets smaller. A first moment decays a tenth a step, in 100 steps
    past the normal numbers, of whose 8 steps the k-th takes at most 2.62 / (0.1 k) steps: all are 0 after 250."""
    _say("adamw 8-bit rule")
    ts = _inputs(cuda, [(2000,)], bits=8, seed=5)
    hyper = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0)
    for _ in range(20):
        before = _clone(ts)
        _step(ts, **hyper)
        _check(ts, hyper, before=before)
    n = 4096
    gen = torch.Generator(cuda).manual_seed(3)
    grad = 1e-3 * (1.0 + torch.rand(n, generator=gen, device=cuda))
    alive = torch.arange(n, device=cuda) % 2 == 0
    p = torch.zeros(n, device=cuda)
    q = [torch.zeros(n, device=cuda, dtype=torch.uint8).view(F8) for _ in range(2)]
    scales, s = [(torch.zeros(n // 256, device=cuda), torch.zeros(n // 256, device=cuda))], torch.zeros((), device=cuda, dtype=torch.int64)

    def root():
        return q[1].float() * scales[0][1].repeat_interleave(256)

    for t in range(450):
        if t == 200:
            start = root()
        optim.adamw_([p], [grad if t < 200 else grad * alive], [q[0]], [q[1]], [s], scales=scales, **hyper)
    assert bool((root() < start)[~alive].all()) and float(q[0].float()[~alive].abs().max()) == 0.0
    assert bool((q[1].float() > 0).all())  # and a root stays above 0


def test_norm_of_many_kinds(cuda):
    _say("grad_norm")
    gen = torch.Generator(cuda).manual_seed(1)
    ts = [torch.randn(n, generator=gen, device=cuda).to(dt) for n, dt in
          [(1, torch.float32), (1000, torch.bfloat16), (0, torch.float16), (77777, torch.float16), (33, torch.float64)] * 40]
    want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    got = [optim.grad_norm(ts) for _ in range(3)]
    assert abs(float(got[0]) - want) <= 2 * U * want and all(torch.equal(got[0], g) for g in got)
    view = torch.randn(40, 60, generator=gen, device=cuda)
    assert abs(float(optim.grad_norm([view.t()[::2], view[:0]])) - float(view[:, ::2].double().norm())) <= 2 * U * float(view.norm())
    assert float(optim.grad_norm([torch.full((4,), 3e38, device=cuda)])) == float("inf")  # past fp32 in the single number
    huge = torch.full(((1 << 31) + 5,), 1.0, device=cuda, dtype=torch.bfloat16)  # past 32-bit offsets
    assert float(optim.grad_norm([huge[1:], huge[:3]])) == float(torch.tensor(math.sqrt((1 << 31) + 7), dtype=torch.float32))


def test_python_path_gives_the_same_bits(cuda, monkeypatch):
    _say("adamw python path")
    for bits in (32, 8):
        ts = _inputs(cuda, SIZES["odd"], bits=bits)
        other = _clone(ts)
        version = ts["params"][0]._version
        a = _step(ts, max_norm=0.1, **HYPER)
        assert ts["params"][0]._version > version  # autograd sees the write
        with monkeypatch.context() as mp:
            mp.setattr(optim._host, "module", lambda: None)
            b = _step(other, max_norm=0.1, **HYPER)
        assert torch.equal(a, b)
        for n in ("params", "exp_avgs", "exp_avg_sqs", "steps"):
            assert all(torch.equal(p.float(), q.float()) for p, q in zip(ts[n], other[n]))


@pytest.mark.parametrize("native", [True, False])
def test_refusals(cuda, native, monkeypatch):
    _say(f"adamw refusals {native}")
    if not native:
        monkeypatch.setattr(optim._host, "module", lambda: None)

    def call(bits=32, **change):
        ts = _inputs(cuda, [(30,), (20, 2)], bits=bits)
        ts |= {n: f(ts[n]) for n, f in change.items() if callable(f)}
        kept = _clone(ts)
        try:
            _step(ts, **(HYPER | {n: v for n, v in change.items() if not callable(v)}))
        finally:
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(ts["params"], kept["params"]))

    for error, kw in [
        (ValueError, dict(params=lambda p: [p[0], p[0]], grads=lambda g: [g[0], g[0]], exp_avgs=lambda m: [m[0], m[0].clone()],
                          exp_avg_sqs=lambda v: [v[0], v[0].clone()])),
        (ValueError, dict(steps=lambda s: [s[0], s[0]])),
        (ValueError, dict(params=lambda p: [p[0], p[1].t()], grads=lambda g: [g[0], g[1].t()])),
        (ValueError, dict(grads=lambda g: [g[0], g[1].t()])),
        (ValueError, dict(exp_avgs=lambda m: [m[0][:29], m[1]])),
        (ValueError, dict(exp_avgs=lambda m: m[:1])),
        (ValueError, dict(params=lambda p: [p[0], p[1].cpu()])),
        (TypeError, dict(exp_avgs=lambda m: [m[0].bfloat16(), m[1]])),
        (TypeError, dict(steps=lambda s: [s[0].float(), s[1]])),
        (TypeError, dict(grads=lambda g: [g[0].double(), g[1]])),
        (TypeError, dict(params=lambda p: [p[0].int(), p[1]])),
        (ValueError, dict(lr=-1.0)), (ValueError, dict(lr=float("nan"))), (ValueError, dict(betas=(0.9, 1.0))),
        (ValueError, dict(eps=-1e-8)), (ValueError, dict(max_norm=0.0)), (ValueError, dict(weight_decay=-0.1)),
        (ValueError, dict(lr=torch.ones(2, device=cuda))), (ValueError, dict(lr=torch.ones(()))),
        (ValueError, dict(bits=8, scales=lambda s: [(s[0][0][:0], s[0][1]), s[1]])),
        (TypeError, dict(bits=8, scales=lambda s: [(s[0][0].double(), s[0][1]), s[1]])),
        (TypeError, dict(bits=8, exp_avgs=lambda m: [t.view(torch.uint8) for t in m])),
        (TypeError, dict(scales=lambda s: [(torch.zeros(1, device=cuda),) * 2] * 2)),
    ]:  # fmt: skip
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(ValueError):
        optim.adamw_([], [], [], [], [], lr=1e-3)
    with pytest.raises(ValueError):
        optim.grad_norm([])
    with pytest.raises(TypeError):
        optim.grad_norm([torch.zeros(3, device=cuda, dtype=torch.int32)])


# -- the optimizer ------------------------------------------------------------------------------------------------------


def _net(cuda, dtype=torch.float32):
    torch.manual_seed(2)
    net = torch.nn.Sequential(torch.nn.Linear(33, 70), torch.nn.Tanh(), torch.nn.Linear(70, 5)).to(cuda, dtype)
    net.register_parameter("order", torch.nn.Parameter(torch.randn(6, 40, device=cuda, dtype=dtype).t()))  # not contiguous
    net.register_parameter("unused", torch.nn.Parameter(torch.randn(9, device=cuda, dtype=dtype)))
    return net


def _loss(net, x):
    return net(x).square().mean() + (net.order * torch.arange(6, device=x.device)).square().mean()


def test_optimizer_follows_torch_s(cuda):
    """Ten clipped steps beside ``torch.optim.AdamW``, with groups of their own rates, a scheduler, and the state moved from one
    to the other. Each step is within some 50 u of the change and 3 u of the parameter, and later gradients see the difference:
    a hundred of these for ten steps."""
    _say("optimizer and torch's")
    ours, theirs = _net(cuda), _net(cuda)
    groups = lambda net: [dict(params=[*net[0].parameters(), net.order], lr=1e-2), dict(params=[*net[2].parameters(), net.unused], weight_decay=0.2)]  # noqa: E731
    a = optim.AdamW(groups(ours), lr=3e-3, betas=(0.9, 0.98), max_norm=0.5)
    b = torch.optim.AdamW(groups(theirs), lr=3e-3, betas=(0.9, 0.98))
    sa, sb = (torch.optim.lr_scheduler.StepLR(o, 3, 0.5) for o in (a, b))
    x = torch.randn(20, 33, generator=torch.Generator(cuda).manual_seed(1), device=cuda)
    for turn in range(10):
        for o, net in ((a, ours), (b, theirs)):
            o.zero_grad()
            _loss(net, x).backward()
        norm = torch.nn.utils.clip_grad_norm_([p for p in theirs.parameters() if p.grad is not None], 0.5)
        a.step(), b.step(), sa.step(), sb.step()
        assert abs(float(a.grad_norm) - float(norm)) <= 1e-4 * float(norm)
        for p, q in zip(ours.parameters(), theirs.parameters()):
            assert float((p - q).detach().abs().max()) <= 1e-4 * float(q.detach().abs().max())
    assert torch.equal(ours.unused, theirs.unused) and ours.unused not in a.state
    a.load_state_dict(b.state_dict())
    for p, q in zip(ours.parameters(), theirs.parameters()):
        if p.grad is not None:
            assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"]) and int(a.state[p]["step"]) == 10


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (32, torch.bfloat16), (8, torch.float32), (8, torch.bfloat16)])
def test_state_saved_and_loaded(cuda, bits, dtype, tmp_path):
    """A run continued from a saved state takes the same steps, to the bit; the moments keep their own types."""
    _say(f"state {bits} {dtype}")
    net = _net(cuda, dtype)
    opt = optim.AdamW(net.parameters(), lr=1e-2, max_norm=1.0, state_bits=bits)
    x = torch.randn(20, 33, generator=torch.Generator(cuda).manual_seed(1), device=cuda).to(dtype)

    def step(net, opt):
        opt.zero_grad()
        _loss(net, x).backward()
        opt.step()

    for _ in range(3):
        step(net, opt)
    torch.save(dict(net=net.state_dict(), opt=opt.state_dict()), tmp_path / "s.pt")
    saved = torch.load(tmp_path / "s.pt", weights_only=True, map_location="cpu")
    net2 = _net(cuda, dtype)
    net2.load_state_dict(saved["net"])
    opt2 = optim.AdamW(net2.parameters(), lr=1e-2, max_norm=1.0, state_bits=bits)
    opt2.load_state_dict(saved["opt"])
    opt3 = copy.deepcopy(opt)
    assert opt3.max_norm == 1.0 and opt3.state_bits == bits
    for _ in range(3):
        step(net, opt), step(net2, opt2)
    for p, q in zip(net.parameters(), net2.parameters()):
        assert torch.equal(p, q)
        if p.grad is not None:
            m, v = opt.moments(p)
            assert m.dtype == torch.float32 and m.shape == p.shape and torch.equal(m, opt2.moments(q)[0])
            assert opt.state[p]["exp_avg"].dtype == (F8 if bits == 8 else torch.float32)
            assert bool((v >= 0).all()) and torch.equal(v, opt2.moments(q)[1])
    with pytest.raises(ValueError):
        optim.AdamW(net.parameters(), state_bits=40 - bits).load_state_dict(saved["opt"])


def test_optimizer_refuses(cuda):
    _say("optimizer refusals")
    p = torch.nn.Parameter(torch.ones(10, 4, device=cuda))
    for kw in (dict(lr=-1), dict(betas=(1.0, 0.9)), dict(eps=-1), dict(weight_decay=-1), dict(max_norm=-1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    emb = torch.nn.Embedding(10, 4, sparse=True, device=cuda)
    emb(torch.tensor([1, 2], device=cuda)).sum().backward()
    with pytest.raises(TypeError):
        optim.AdamW(emb.parameters()).step()
    wide = torch.nn.Parameter(torch.ones(3, device=cuda, dtype=torch.float64))
    wide.grad = torch.ones_like(wide)
    with pytest.raises(TypeError):
        optim.AdamW([wide], state_bits=8).step()
    optim.AdamW([p]).step()  # no gradients: nothing to do
    assert torch.equal(p, torch.ones_like(p))


# -- a training step's operators together ------------------------------------------------------------------------------


def _model(cuda, **kw):
    kw = dict(hidden_size=64, num_heads=4, grid=(4, 4), vocab_size=7, norm="layer") | kw
    return en.build(en.EnergyConfig(**kw), cuda, seed=3)


def _batch(cuda, B=3, L=16, C=64, V=7):
    g = torch.Generator(cuda).manual_seed(6)
    return (torch.randint(0, V, (B, L), generator=g, device=cuda), torch.randn(B, L, C, generator=g, device=cuda),
            torch.randint(0, V, (B, L), generator=g, device=cuda))


FUSED = dict(block_impl="fused", mlp_impl="projected", embed_impl="fused")


def test_step_of_an_energy_with_these_operators(cuda):
    """``train_step`` with layer norms and gated projections inside graded descent and the optimizer's step, fp32, against the
    same network in plain torch ops. Bound 1e-4 relative for the gradients: two graded steps through two blocks are some 10^3
    roundings of 2^-24 in a row. The first step of AdamW moves each parameter by lr in its gradient's direction, so parameters
    are compared where the gradient is well above its error."""
    _say("energy step")
    x, z, target = _batch(cuda)
    fused, dec = _model(cuda, **FUSED)
    plain, dec2 = _model(cuda)
    plain.load_state_dict(fused.state_dict())
    dec2.load_state_dict(dec.state_dict())
    grads = {}
    for net, d, tag in ((fused, dec, "a"), (plain, dec2, "b")):
        en.train_step(net, d, x, z, target, steps=2)
        grads[tag] = [p.grad for p in [*net.parameters(), *d.parameters()]]
        for p in [*net.parameters(), *d.parameters()]:
            p.grad = None
    names = [n for n, _ in [*fused.named_parameters(), *dec.named_parameters()]]
    for n, a, b in zip(names, grads["a"], grads["b"]):
        assert (a is None) == (b is None), n
        assert a is None or float((a - b).norm()) <= 1e-4 * float(b.norm().clamp(min=1e-6)), n
    assert any("layer_norms" in n and g is not None for n, g in zip(names, grads["a"]))
    for bits in (32, 8):
        params, params2 = ([*m.parameters(), *d.parameters()] for m, d in ((copy.deepcopy(fused), copy.deepcopy(dec)), (plain, dec2)))
        kept = [p.detach().clone() for p in params]
        opt = optim.AdamW(params, lr=1e-3, weight_decay=0.0, max_norm=1.0, state_bits=bits)
        for p, g in zip(params, grads["a"]):
            p.grad = g
        opt.step()
        for p, k, g in zip(params, kept, grads["b"]):
            if g is None:
                assert torch.equal(p, k)
                continue
            sure = g.abs() > 1e-2 * g.norm()
            assert not sure.any() or float(((p - k) + 1e-3 * g.sign())[sure].detach().abs().max()) <= 2e-5


def test_training_steps_run_and_learn_nothing_undefined(cuda):
    _say("energy steps bf16")
    x, z, target = _batch(cuda, B=8)
    model, dec = _model(cuda, **FUSED, rope_impl="fused")
    params = [*model.parameters(), *dec.parameters()]
    for bits in (32, 8):
        opt = optim.AdamW(params, lr=1e-3, max_norm=1.0, state_bits=bits)
        for _ in range(3):
            before = [p.detach().clone() for p in params]
            loss = en.train_step(model, dec, x, z.bfloat16(), target, steps=2, optimizer=opt)
            assert math.isfinite(float(loss)) and all(p.grad is None for p in params)
            moved = [not torch.equal(p, q) for p, q in zip(params, before)]
            assert all(bool(torch.isfinite(p).all()) for p in params) and sum(moved) >= len(moved) - 1


def test_compiled_gradient_of_an_energy_with_these_operators(cuda):
    _say("compiled energy")
    model, _ = _model(cuda, **FUSED)
    x, z, _ = _batch(cuda)
    errs = en.verify_compiled_energy_grad(model, en.compiled_energy_grad(model), z, model.puzzle_embedding(x, z.dtype))
    assert max(errs.values()) < 1e-3


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(cuda, bits):
    """The whole step with the optimizer captured: replays take the steps that eager runs take, on the same contents."""
    _say(f"captured step {bits}")
    x, z, target = _batch(cuda, B=8)
    z = z.bfloat16()
    model, dec = _model(cuda, **FUSED, rope_impl="fused")
    twin, dec2 = copy.deepcopy(model), copy.deepcopy(dec)
    lr = torch.tensor(1e-3, device=cuda)
    opt, opt2 = (optim.AdamW([*m.parameters(), *d.parameters()], lr=lr, max_norm=0.5, state_bits=bits) for m, d in ((model, dec), (twin, dec2)))
    graph, loss = en.graph_train_step(model, dec, x, z, target, steps=2, optimizer=opt)
    for turn in range(4):
        x.copy_((x + turn) % 7)
        z.mul_(0.9)
        if turn == 2:
            lr.fill_(5e-4)
        want = en.train_step(twin, dec2, x, z, target, steps=2, optimizer=opt2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, loss) and torch.equal(opt.grad_norm, opt2.grad_norm)
        for p, q in zip([*model.parameters(), *dec.parameters()], [*twin.parameters(), *dec2.parameters()]):
            assert torch.equal(p, q)
            if p in opt.state and q in opt2.state:
                assert int(opt2.state[q]["step"]) == int(opt.state[p]["step"]) == turn + 1


def test_two_captured_steps_do_not_share_scratch(cuda):
    _say("two captured steps")
    sets = [_inputs(cuda, SIZES["odd"], bits=b, seed=s) for s, b in ((1, 32), (2, 8))]
    eager = [_clone(t) for t in sets]
    graphs = []
    for t in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        warm = _clone(t)
        with torch.cuda.stream(side):
            _step(warm, max_norm=0.05, **HYPER)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = _step(t, max_norm=0.05, **HYPER)
        graphs.append((g, norm))
    for turn in range(3):
        want = [_step(t, max_norm=0.05, **HYPER) for t in eager]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, norm), w, t, e in zip(graphs, want, sets, eager):
            assert torch.equal(norm, w)
            for n in ("params", "exp_avgs", "exp_avg_sqs", "steps"):
                assert all(torch.equal(p.float(), q.float()) for p, q in zip(t[n], e[n]))
