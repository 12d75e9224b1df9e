"""Performance cases of a training step's layer norm, gated projection and optimizer step: the calls that a training or
serving program makes of them, from one token or one board to the largest batches and parameter lists.

A case is a dict of plain values. ``kind`` says which operator it is:

- ``layer``  layer norm over the last dimension of ``N`` rows of ``C``, with a weight and a bias in fp32. ``order`` 1: output
             and the gradients of the input, weight and bias; ``order`` 2: a graded step, which takes the input's gradient
             and then the derivatives of that gradient for the input, the output's cotangent and the weight.
- ``glu``    the gated projection silu(x Wg^T) * (x Wu^T) of ``N`` rows of ``C`` to ``I``, Wg and Wu the halves of one weight
             [2 I, C]. ``order`` 0: the output alone, as serving does; 1: with the gradients of input and weight; 2: a graded
             step, as above.
- ``adamw``  one AdamW step over ``tensors`` parameters of ``total`` elements together, with the gradients' global norm
             clipped where ``clip``. ``dtype`` is the parameters' type, ``grad`` the gradients'. ``bits`` is 32 (fp32 moments)
             or 8: the first moment and the root of the second as e4m3 numbers with one fp32 scale for 256 elements.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
F8 = torch.float8_e4m3fn
BLOCK = 256
LR, BETAS, ADAM_EPS, DECAY, MAX_NORM = 3e-4, (0.9, 0.95), 1e-8, 0.1, 1.0


def listed():
    return [
        # One 9 x 9 board in a graded step: launches and the host path.
        dict(name="layer_one_board", kind="layer", N=81, C=512, dtype="bf16", order=2),
        # The 768-board training batch in a graded step: short rows, very many of them.
        dict(name="layer_boards", kind="layer", N=768 * 81, C=256, dtype="bf16", order=2),
        # Text: long rows, forward and gradient.
        dict(name="layer_text", kind="layer", N=16384, C=2048, dtype="bf16", order=1),
        # Few wide fp32 rows of an odd width: no vector is aligned in every row.
        dict(name="layer_odd_width", kind="layer", N=1000, C=5003, dtype="fp32", order=1),
        # Serving a single token: the weight is read once.
        dict(name="glu_one_token", kind="glu", N=1, C=2048, I=5632, dtype="bf16", order=0),
        # One board in a graded step.
        dict(name="glu_one_board", kind="glu", N=81, C=256, I=768, dtype="bf16", order=2),
        # The 768-board training batch in a graded step: products of a short inner dimension.
        dict(name="glu_boards", kind="glu", N=768 * 81, C=256, I=768, dtype="bf16", order=2),
        # Text: large products, forward and gradients.
        dict(name="glu_text", kind="glu", N=8192, C=2048, I=5632, dtype="bf16", order=1),
        # An energy network of two layers: a dozen fp32 tensors, clipped.
        dict(name="adamw_network", kind="adamw", tensors=13, total=6_300_000, dtype="fp32", grad="fp32", bits=32, clip=True),
        # A large model's share on one card: fp32 moments.
        dict(name="adamw_large", kind="adamw", tensors=80, total=160_000_000, dtype="fp32", grad="fp32", bits=32, clip=True),
        # The same with moments in 8 bits and bf16 gradients for fp32 parameters.
        dict(name="adamw_large_8bit", kind="adamw", tensors=80, total=160_000_000, dtype="fp32", grad="bf16", bits=8, clip=True),
        # Many small bf16 tensors of odd sizes, one after another in a buffer, moments in 8 bits.
        dict(name="adamw_small_8bit", kind="adamw", tensors=60, total=900_001, dtype="bf16", grad="bf16", bits=8, clip=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    kind = rng.choice(("layer", "glu", "adamw"))
    if kind == "layer":
        # rows of 64 elements and more: in a row of a few, nothing but rounding is left of the projected gradients
        C = 8 * _log_int(rng, 8, 1024) if rng.random() < 0.7 else _log_int(rng, 64, 12000)
        return dict(kind="layer", N=_log_int(rng, 1, max(1, min(65536, int(3.2e7 / C)))), C=C,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), order=rng.choice((1, 2)))
    if kind == "glu":
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
        C, I = (8 * _log_int(rng, 8, 512) if rng.random() < 0.7 else _log_int(rng, 64, 4096) for _ in range(2))
        most = 4e9 if dtype == "fp32" else 3e10
        return dict(kind="glu", N=_log_int(rng, 1, max(1, min(16384, int(most / (C * I))))), C=C, I=I, dtype=dtype,
                    order=rng.choice((0, 1, 2)))
    dtype, grad = rng.choice((("fp32", "fp32"), ("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp16")))
    tensors = _log_int(rng, 1, 80)
    return dict(kind="adamw", tensors=tensors, total=max(tensors, _log_int(rng, 1000, 100_000_000)), dtype=dtype, grad=grad,
                bits=rng.choice((32, 8)), clip=rng.random() < 0.5)


# -- inputs ------------------------------------------------------------------------------------------------------------


def _sizes(case):
    """The elements of each parameter: of very different sizes, as a network's matrices and vectors are."""
    n = case["tensors"]
    share = [1.0 + 40.0 * (k % 3 == 0) + 15.0 * (k % 5 == 1) for k in range(n)]
    left = case["total"] - n
    sizes = [1 + int(left * s / sum(share)) for s in share]
    sizes[0] += case["total"] - sum(sizes)
    return sizes


def _cut(flat, sizes):
    """A buffer's parts of these sizes, one after another."""
    return list(torch.split(flat, sizes))


def _inputs(case, seed):
    """The tensors of a case, in a fixed order of draws, on the GPU."""
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return (scale * torch.randn(shape, generator=g, device=dev, dtype=torch.float32)).to(dtype)

    if case["kind"] == "layer":
        N, C = case["N"], case["C"]
        x = randn(N, C, dtype=torch.float32) + 0.5 * randn(C, dtype=torch.float32)
        return dict(x=x.to(dt), dy=randn(N, C), u=randn(N, C), weight=1.0 + 0.1 * randn(C, dtype=torch.float32),
                    bias=0.1 * randn(C, dtype=torch.float32))
    if case["kind"] == "glu":
        N, C, I = case["N"], case["C"], case["I"]
        return dict(x=randn(N, C), weight=randn(2 * I, C, scale=C**-0.5), dy=randn(N, I), u=randn(N, C))
    total, sizes = case["total"], _sizes(case)
    ts = dict(p=randn(total, scale=0.02), g=randn(total, dtype=DTYPES[case["grad"]], scale=2e-3))
    m = randn(total, dtype=torch.float32, scale=4e-4)
    r = (randn(total, dtype=torch.float32, scale=5e-4).abs() + 1.5e-3)
    if case["bits"] == 32:
        ts |= dict(m=m, v=r.square())
    else:
        coded = [(_coded(a), _coded(b)) for a, b in zip(_cut(m, sizes), _cut(r, sizes))]
        ts |= dict(m=torch.cat([a[0].view(torch.uint8) for a, _ in coded]).view(F8),
                   r=torch.cat([b[0].view(torch.uint8) for _, b in coded]).view(F8),
                   ms=torch.cat([a[1] for a, _ in coded]), rs=torch.cat([b[1] for _, b in coded]))
    ts["steps"] = [torch.full((), 40, device=dev, dtype=torch.int64) for _ in sizes]
    return ts


def _blocks(x):
    """[blocks, 256] of a vector, the last one filled up with zeros."""
    n = -(-x.numel() // BLOCK) * BLOCK
    return torch.nn.functional.pad(x, (0, n - x.numel())).view(-1, BLOCK)


def _coded(x):
    """A moment that a run before this one has left: e4m3 numbers, and a scale for each 256 of them."""
    b = _blocks(x)
    scale = b.abs().amax(1) / 448.0
    return (b / scale.clamp(min=1e-30)[:, None]).to(F8).view(-1)[: x.numel()], scale


def prepare(case, seed):
    ts = _inputs(case, seed)
    if case["kind"] == "adamw":
        sizes = _sizes(case)
        parts = {n: _cut(ts[n].view(torch.uint8), sizes) if ts[n].dtype == F8 else _cut(ts[n], sizes)
                 for n in ("p", "g", "m", "v", "r") if n in ts}
        parts |= {n: [t.view(F8) for t in parts[n]] for n in ("m", "r") if case["bits"] == 8}
        parts |= {n: _cut(ts[n], [-(-s // BLOCK) for s in sizes]) for n in ("ms", "rs") if n in ts}
        return dict(case=case, flat=ts, **parts, steps=ts["steps"])
    for n in ("x", "weight", "bias"):
        if n in ts and (case["order"] > 0):
            ts[n].requires_grad_(True)
    ts["dy"].requires_grad_(case["order"] == 2)
    return dict(case=case, **ts)


# -- one pass ----------------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"layer": _own_layer, "glu": _own_glu, "adamw": _own_adamw}[kind](state)
    return {"layer": _plain_layer, "glu": _plain_glu, "adamw": _plain_adamw}[kind](state)


def _own_layer(s):
    from ebr_amd import block

    return _layer_grads(s["case"], block.layer_norm(s["x"], s["weight"], s["bias"], EPS), s["x"], s["dy"], s["u"], s["weight"], s["bias"])


def _plain_layer(s):
    dt = DTYPES[s["case"]["dtype"]]
    x, dy = (s[n].detach().float().requires_grad_(True) for n in ("x", "dy"))
    c = x - x.mean(dim=1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(dim=1, keepdim=True) + EPS) * s["weight"] + s["bias"]
    out = _layer_grads(s["case"], y, x, dy, s["u"].float(), s["weight"], s["bias"])
    return {n: t if n in ("dw", "db", "gw") else t.to(dt) for n, t in out.items()}


def _layer_grads(case, y, x, dy, u, w, b):
    """What a step takes from y."""
    out = {"y": y.detach()}
    if case["order"] == 1:
        return out | dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)))
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    return out | {"dx": dx.detach()} | dict(zip(("gx", "gdy", "gw"), torch.autograd.grad(dx, (x, dy, w), u)))


def _own_glu(s):
    from ebr_amd import block

    if s["case"]["order"] == 0:
        with torch.no_grad():
            return {"y": block.swiglu_linear(s["x"], s["weight"])}
    return _glu_grads(s["case"], block.swiglu_linear(s["x"], s["weight"]), s["x"], s["dy"], s["u"], s["weight"])


def _plain_glu(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w, dy = (s[n].detach().float().requires_grad_(case["order"] > 0) for n in ("x", "weight", "dy"))
    gate, up = (x @ w.t()).chunk(2, dim=1)
    y = gate / (1.0 + torch.exp(-gate)) * up
    out = {"y": y} if case["order"] == 0 else _glu_grads(case, y, x, dy, s["u"].float(), w)
    return {n: t.to(dt) for n, t in out.items()}


def _glu_grads(case, y, x, dy, u, w):
    out = {"y": y.detach()}
    if case["order"] == 1:
        return out | dict(zip(("dx", "dw"), torch.autograd.grad(y, (x, w), dy.detach())))
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    return out | {"dx": dx.detach()} | dict(zip(("gx", "gdy", "gw"), torch.autograd.grad(dx, (x, dy, w), u)))


def _own_adamw(s):
    from ebr_amd import optim

    case = s["case"]
    eight = case["bits"] == 8
    norm = optim.adamw_(s["p"], s["g"], s["m"], s["r"] if eight else s["v"], s["steps"], lr=LR, betas=BETAS, eps=ADAM_EPS,
                        weight_decay=DECAY, max_norm=MAX_NORM if case["clip"] else None,
                        scales=list(zip(s["ms"], s["rs"])) if eight else None)
    return _adamw_out(s, norm)


def _adamw_out(s, norm):
    out = {n: s["flat"][n] for n in ("p", "m", "v", "r", "ms", "rs") if n in s["flat"]} | {"steps": list(s["steps"][:4])}
    return out if norm is None else out | {"norm": norm}


def _plain_adamw(s):
    case = s["case"]
    norm, factor = None, 1.0
    if case["clip"]:
        # a sum over every gradient: 64 bits
        norm = torch.stack([g.double().square().sum() for g in s["g"]]).sum().sqrt()
        factor = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
        norm = norm.float()
    step = _plain_step8 if case["bits"] == 8 else _plain_step
    for k in range(len(s["p"])):
        step(s, k, s["g"][k].float() * factor)
    return _adamw_out(s, norm)


def _plain_update(p, t, m, root):
    """The parameter after the step from the moments, the second's root."""
    c1, c2 = (1.0 - b ** t.double() for b in BETAS)
    p.copy_(p.float() * (1.0 - LR * DECAY) - (LR / c1).float() * m / (root / c2.sqrt().float() + ADAM_EPS))


def _plain_step(s, k, g):
    m, v, t = s["m"][k], s["v"][k], s["steps"][k]
    t.add_(1)
    m.copy_(BETAS[0] * m + (1.0 - BETAS[0]) * g)
    v.copy_(BETAS[1] * v + (1.0 - BETAS[1]) * g * g)
    _plain_update(s["p"][k], t, m, v.sqrt())


def _plain_step8(s, k, g):
    t, n = s["steps"][k], g.numel()
    t.add_(1)
    g = _blocks(g)
    m, r = (_blocks(s[c][k].float()) * s[c + "s"][k][:, None] for c in ("m", "r"))
    m = BETAS[0] * m + (1.0 - BETAS[0]) * g
    r = (BETAS[1] * r * r + (1.0 - BETAS[1]) * g * g).sqrt()
    _plain_update(s["p"][k], t, m.view(-1)[:n], r.view(-1)[:n])
    i = torch.arange(n, device=g.device) * 0x85EBCA77 + t * 0x9E3779B1
    for c, x, start in (("m", m, 0), ("r", r, 0x80000000)):
        scale = x.abs().amax(1) / 448.0
        scale = torch.where(scale < 2.0**-126, torch.zeros_like(scale), scale)
        y = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x)).view(-1)[:n]
        dither = (((i + start) & 0xFFFFFFFF) >> 8).float() * 2.0**-24
        e = (torch.frexp(y.abs()).exponent - 1).clamp(min=-6)
        q = torch.ldexp(torch.floor(torch.ldexp(y.abs(), 3 - e) + dither), e - 3).clamp(max=448.0)
        if c == "r":
            q = torch.where(y > 0, q.clamp(min=2.0**-9), q)
        s[c][k].view(torch.uint8).copy_(torch.copysign(q, y).to(F8).view(torch.uint8))
        s[c + "s"][k].copy_(scale)


# -- what a pass cannot do without -------------------------------------------------------------------------------------


def work(case):
    es = SIZES[case["dtype"]]
    if case["kind"] == "layer":
        n = case["N"] * case["C"]
        # y of x; dx of x and dy; gx and gdy of x, dy and u: x and dy are read once in all
        return {"bytes": float((4 if case["order"] == 1 else 7) * n * es + 16.0 * case["C"]),
                "flops": (16.0 if case["order"] == 1 else 40.0) * n}
    if case["kind"] == "glu":
        N, C, I = (float(case[n]) for n in ("N", "C", "I"))
        # x, weight -> y; dy -> dx, dw; u -> gx, gdy, gw with dx
        tensors = (N * C + 2 * I * C + N * I, 2 * N * C + 4 * I * C + 2 * N * I, 4 * N * C + 4 * I * C + 3 * N * I)[case["order"]]
        # a product of N x C x 2 I: one forward, one each for dx and dw; dx's derivatives take three, two of them for the weight
        return {"bytes": tensors * es, "flops": 4.0 * N * C * I * (1, 3, 6)[case["order"]]}
    n = float(case["total"])
    states = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    return {"bytes": n * (2 * es + SIZES[case["grad"]] + states), "flops": 20.0 * n}


# -- the same values in 64 bits, from the definitions ------------------------------------------------------------------


def exact(case, seed):
    return {"layer": _exact_layer, "glu": _exact_glu, "adamw": _exact_adamw}[case["kind"]](case, _inputs(case, seed))


def _exact_layer(case, ts):
    """The closed forms of the layer norm's first and second derivatives."""
    x, dy, u, w, b = (ts[n].double() for n in ("x", "dy", "u", "weight", "bias"))

    def mean(v):
        return v.mean(dim=1, keepdim=True)

    mu = mean(x)
    r = (mean((x - mu) ** 2) + EPS) ** -0.5
    h = (x - mu) * r

    def project(v):
        return r * (v - mean(v) - h * mean(v * h))

    k = w * dy
    out = {"y": w * h + b, "dx": project(k)}
    if case["order"] == 1:
        return out | {"dw": (dy * h).sum(0), "db": dy.sum(0)}
    pu = project(u)
    along = mean(k * u) - mean(k) * mean(u) - mean(u * h) * mean(k * h)
    out["gx"] = project(-r * (u * mean(k * h) + k * mean(u * h))) - r * r * h * along
    return out | {"gdy": w * pu, "gw": (dy * pu).sum(0)}


def _exact_glu(case, ts):
    """The closed forms of the gated projection's first and second derivatives."""
    x, w = ts["x"].double(), ts["weight"].double()
    I = case["I"]
    gu = x @ w.T
    g, up = gu[:, :I], gu[:, I:]
    sg = torch.sigmoid(g)
    f0 = g * sg
    if case["order"] == 0:
        return {"y": f0 * up}
    f1 = sg * (1 + g * (1 - sg))
    dy = ts["dy"].double()
    d = torch.cat((dy * up * f1, dy * f0), dim=1)
    out = {"y": f0 * up, "dx": d @ w}
    if case["order"] == 1:
        return out | {"dw": d.T @ x}
    u = ts["u"].double()
    c = u @ w.T
    cg, cu = c[:, :I], c[:, I:]
    f2 = sg * (1 - sg) * (2 + g * (1 - 2 * sg))
    e = torch.cat((cg * dy * up * f2 + cu * dy * f1, cg * dy * f1), dim=1)
    return out | {"gx": e @ w, "gdy": cg * up * f1 + cu * f0, "gw": e.T @ x + d.T @ u}


def _exact_adamw(case, ts):
    sizes = _sizes(case)
    eight = case["bits"] == 8
    norm = ts["g"].double().norm()
    factor = min(1.0, MAX_NORM / (float(norm) + 1e-6)) if case["clip"] else 1.0
    b1, b2 = BETAS
    t = int(ts["steps"][0]) + 1
    p = ts["p"].double()
    g = ts["g"].double() * factor
    if eight:
        counts = [-(-n // BLOCK) for n in sizes]
        first = torch.cat([k + torch.arange(n, device=p.device) // BLOCK for n, k in zip(sizes, [sum(counts[:j]) for j in range(len(counts))])])
        m = ts["m"].float().double() * ts["ms"].double()[first]
        root = ts["r"].float().double() * ts["rs"].double()[first]
    else:
        m, root = ts["m"].double(), None
    m = b1 * m + (1 - b1) * g
    v = b2 * (root.square() if eight else ts["v"].double()) + (1 - b2) * g.square()
    root = v.sqrt()
    out = {"p": p * (1 - LR * DECAY) - LR / (1 - b1**t) * m / (root / math.sqrt(1 - b2**t) + ADAM_EPS)}
    out["steps"] = [None] * min(4, len(sizes))
    if case["clip"]:
        out["norm"] = norm
    if not eight:
        return out | {"m": m, "v": v}
    at = torch.cat([torch.arange(n, device=p.device) for n in sizes])
    for name, x, start in (("m", m, 0), ("r", root, 0x80000000)):
        top = torch.zeros(sum(counts), device=p.device, dtype=torch.float64).index_reduce_(0, first, x.abs(), "amax")
        scale = (top / 448.0)
        y = torch.where(scale[first] > 0, x / scale[first].clamp(min=1e-300), torch.zeros_like(x))
        dither = ((at * 0x85EBCA77 + t * 0x9E3779B1 + start) % 2**32 // 256).double() / 2**24
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
        q = (torch.floor(y.abs() / step + dither) * step).clamp(max=448.0)
        if name == "r":
            q = torch.where(y > 0, q.clamp(min=2.0**-9), q)
        out[name], out[name + "s"] = q * torch.sign(y), scale
    return out
