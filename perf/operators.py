"""Performance cases of the operators at the ends of a training step and of the group norm inside it: the calls that a
training program makes of them, from one board to the largest batches and vocabularies.

A case is a dict of plain values. ``kind`` says which operator it is:

- ``embed``    the embedding of ``N`` tokens from a table [V, C], scaled, and the table's gradient. ``dtype`` is the
               output's type, ``table`` the table's (an fp32 master table read at 16 bits, or a table of the same type).
               ``ids`` is "uniform" (a board's cell values) or "zipf" (text); ``pad`` is the share of padded tokens (-1).
- ``distill``  the distillation loss of ``N`` rows of ``V`` logits from a teacher's ``K`` top logits, and the logits'
               gradient. ``ragged`` rows have fewer than K valid entries, or none.
- ``norm``     group norm over [B, L, C], channels last, with its activation. ``order`` 1: output and the gradients of
               the input, weight and bias; ``order`` 2: a graded step, which takes the input's gradient and then the
               derivatives of that gradient for the input, the output's cotangent, the weight and the bias.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
IGNORE = -1


def listed():
    return [
        # One 9 x 9 board of 11 cell values: nothing but launches and the host path.
        dict(name="embed_one_board", kind="embed", N=81, V=11, C=512, table="fp32", dtype="bf16", ids="uniform", pad=0.0, scale=1.0),
        # The 384-board training batch: every one of the 11 table rows gathers thousands of gradient rows.
        dict(name="embed_boards", kind="embed", N=384 * 81, V=11, C=512, table="fp32", dtype="bf16", ids="uniform", pad=0.0, scale=1.0),
        # Text: an odd vocabulary, a few tokens very frequent, most absent, padded sequence ends.
        dict(name="embed_text", kind="embed", N=16384, V=50021, C=1024, table="bf16", dtype="bf16", ids="zipf", pad=0.1, scale=32.0),
        # A large fp32 master table: writing its dense gradient is nearly all of the work.
        dict(name="embed_large_table", kind="embed", N=32768, V=100003, C=2048, table="fp32", dtype="bf16", ids="zipf", pad=0.0, scale=1.0),
        # One board's cells, taught by another descent's top 4 of 11 logits: launches.
        dict(name="distill_one_board", kind="distill", N=81, V=11, K=4, dtype="bf16", T=2.0, ragged=False),
        # The training batch's cells: very many very short rows.
        dict(name="distill_boards", kind="distill", N=384 * 81, V=11, K=4, dtype="bf16", T=2.0, ragged=False),
        # Text: long rows, the teacher's top 64, padded positions without a teacher.
        dict(name="distill_text", kind="distill", N=4096, V=50021, K=64, dtype="bf16", T=1.0, ragged=True),
        # A few long fp32 rows: a short answer's loss, too few rows to fill the card one by one.
        dict(name="distill_few_rows", kind="distill", N=24, V=131072, K=128, dtype="fp32", T=1.5, ragged=False),
        # One board in a graded step: launches.
        dict(name="norm_one_board", kind="norm", B=1, L=81, C=512, G=32, dtype="bf16", act="silu", affine=True, order=2),
        # The 768-board training batch in a graded step.
        dict(name="norm_boards", kind="norm", B=768, L=81, C=512, G=32, dtype="bf16", act="silu", affine=True, order=2),
        # 30 x 30 boards, forward and gradient.
        dict(name="norm_maze", kind="norm", B=64, L=900, C=512, G=16, dtype="bf16", act="silu", affine=True, order=1),
        # Two large fp32 grids with groups of 10 channels: statistics over rows far longer than a workgroup holds.
        dict(name="norm_large_grid", kind="norm", B=2, L=128 * 128, C=320, G=32, dtype="fp32", act="silu", affine=True, order=2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("embed", "distill", "norm"))
    if kind == "embed":
        C = 8 * _log_int(rng, 2, 256) if rng.random() < 0.7 else _log_int(rng, 5, 1500)
        V = _log_int(rng, 3, max(3, min(131072, int(1.6e8 / C))))
        N = _log_int(rng, 1, max(1, min(65536, int(4e7 / C))))
        table, dtype = rng.choice((("fp32", "bf16"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")))
        return dict(kind="embed", N=N, V=V, C=C, table=table, dtype=dtype, ids=rng.choice(("uniform", "zipf")),
                    pad=rng.choice((0.0, 0.0, 0.2)), scale=rng.choice((1.0, round(math.sqrt(C), 3))))
    if kind == "distill":
        V = _log_int(rng, 2, 131072)
        N = _log_int(rng, 1, max(1, min(65536, int(1.9e8 / V))))
        return dict(kind="distill", N=N, V=V, K=_log_int(rng, 1, min(V, 256)), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    T=round(rng.uniform(0.7, 4.0), 2), ragged=rng.random() < 0.5)
    G = rng.choice((1, 2, 4, 8, 16, 32))
    L = _log_int(rng, 4, 16384)
    # groups of 64 elements and more: in a group of a few, nothing but rounding is left of the projected gradients
    C = G * _log_int(rng, max(1, -(-64 // L)), 1024 // G)
    B = _log_int(rng, 1, max(1, min(1024, int(1.6e7 / (L * C)))))
    return dict(kind="norm", B=B, L=L, C=C, G=G, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), act=rng.choice(("silu", "silu", "none")),
                affine=rng.random() < 0.7, order=rng.choice((1, 2)))


# -- inputs ------------------------------------------------------------------------------------------------------------


def _zipf(V):
    """The tokens' probabilities, by rank."""
    w = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    return w / w.sum()


def _inputs(case, seed):
    """The tensors of a case, in a fixed order of draws, on the GPU."""
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=g, device=dev)

    if case["kind"] == "embed":
        N, V, C = case["N"], case["V"], case["C"]
        if case["ids"] == "uniform":
            ids = torch.randint(0, V, (N,), generator=g, device=dev)
        else:
            cdf = _zipf(V).cumsum(0).to(dev)
            ids = torch.searchsorted(cdf, rand(N).double()).clamp_(max=V - 1)
        if case["pad"]:
            ids = torch.where(rand(N) < case["pad"], torch.full_like(ids, IGNORE), ids)
        return dict(ids=ids, weight=randn(V, C, dtype=DTYPES[case["table"]]), dy=randn(N, C))
    if case["kind"] == "distill":
        N, V, K = case["N"], case["V"], case["K"]
        # K distinct tokens per row, the teacher's logits falling off as a sorted distribution's do
        first = torch.randint(0, V, (N, 1), generator=g, device=dev)
        step = torch.randint(1, max(2, V // K + 1), (N, 1), generator=g, device=dev)
        k = torch.arange(K, device=dev)
        ids = (first + k * step) % V
        teacher = 8.0 - 1.5 * torch.log1p(k.float()) + 0.3 * randn(N, K, dtype=torch.float32)
        # the student has learnt some of it
        logits = 2.0 * randn(N, V, dtype=torch.float32)
        logits.scatter_add_(1, ids, 0.6 * teacher + 0.5 * randn(N, K, dtype=torch.float32))
        if case["ragged"]:
            have = (rand(N, 1) * (K + 1) * 1.25).long()  # valid entries of a row; a fifth of the rows have all
            have = torch.where(rand(N, 1) < 0.15, torch.zeros_like(have), have)
            ids = torch.where(k < have, ids, torch.full_like(ids, IGNORE))
        return dict(logits=logits.to(dt), teacher=teacher.to(dt), ids=ids)
    B, L, C = case["B"], case["L"], case["C"]
    x = randn(B, L, C, dtype=torch.float32) + 0.5 * randn(C, dtype=torch.float32)
    ts = dict(x=x.to(dt), dy=randn(B, L, C), u=randn(B, L, C), weight=None, bias=None)
    if case["affine"]:
        ts["weight"], ts["bias"] = 1.0 + 0.1 * randn(C, dtype=torch.float32), 0.1 * randn(C, dtype=torch.float32)
    return ts


def prepare(case, seed):
    ts = _inputs(case, seed)
    for n in ("weight", "bias", "logits", "x"):
        if ts.get(n) is not None:
            ts[n].requires_grad_(True)
    if case["kind"] == "norm":
        ts["dy"].requires_grad_(case["order"] == 2)
    return dict(case=case, **ts)


# -- one pass ----------------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"embed": _own_embed, "distill": _own_distill, "norm": _own_norm}[kind](state)
    return {"embed": _plain_embed, "distill": _plain_distill, "norm": _plain_norm}[kind](state)


def _own_embed(s):
    from ebr_amd import tokens

    y = tokens.embedding(s["ids"], s["weight"], scale=s["case"]["scale"], dtype=DTYPES[s["case"]["dtype"]])
    (dw,) = torch.autograd.grad(y, s["weight"], s["dy"])
    return {"y": y.detach(), "dw": dw}


def _plain_embed(s):
    with torch.no_grad():
        ids, w, scale = s["ids"], s["weight"], s["case"]["scale"]
        there = (ids >= 0)[:, None]
        at = ids.clamp(min=0)
        y = (w[at].float() * scale * there).to(DTYPES[s["case"]["dtype"]])
        dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
        dw.index_add_(0, at, s["dy"].float() * there)
        return {"y": y, "dw": (dw * scale).to(w.dtype)}


def _own_distill(s):
    from ebr_amd import tokens

    loss = tokens.distill_loss(s["logits"], s["teacher"], s["ids"], temperature=s["case"]["T"])
    (dx,) = torch.autograd.grad(loss, s["logits"])
    return {"loss": loss.detach(), "dx": dx}


def _plain_distill(s):
    with torch.no_grad():
        T = s["case"]["T"]
        z = s["logits"].float() / T
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        there = s["ids"] >= 0
        at = s["ids"].clamp(min=0)
        t = torch.where(there, s["teacher"].float() / T, torch.full((), -1e30, device=z.device))
        pe = torch.exp(t - t.amax(1, keepdim=True)) * there
        full = pe.sum(1, keepdim=True)
        counted = full > 0
        p = pe / full.clamp(min=1e-30)
        logp = t - t.amax(1, keepdim=True) - torch.log(full.clamp(min=1e-30))
        logq = torch.gather(z, 1, at) - top - torch.log(total)
        n = counted.sum().clamp(min=1)
        rows = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
        loss = rows.sum() * (T * T) / n
        dx = (e / total) * counted
        dx.scatter_add_(1, at, -p)
        return {"loss": loss, "dx": (dx * (T / n)).to(s["logits"].dtype)}


def _own_norm(s):
    from ebr_amd import block

    case = s["case"]
    x, w, b = s["x"], s["weight"], s["bias"]
    y = block.group_norm(x, case["G"], w, b, EPS, None if case["act"] == "none" else case["act"])
    return _norm_grads(case, y, x, s["dy"], s["u"], w, b)


def _plain_norm(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, dy = (s[n].detach().float().requires_grad_(True) for n in ("x", "dy"))
    B, L, C = x.shape
    v = x.view(B, L, case["G"], C // case["G"])
    c = v - v.mean(dim=(1, 3), keepdim=True)
    h = (c * torch.rsqrt((c * c).mean(dim=(1, 3), keepdim=True) + EPS)).view(B, L, C)
    a = h * s["weight"] + s["bias"] if case["affine"] else h
    y = a / (1.0 + torch.exp(-a)) if case["act"] == "silu" else a
    out = _norm_grads(case, y, x, dy, s["u"].float(), s["weight"], s["bias"])
    return {n: t if n in ("dw", "db", "gw", "gb") else t.to(dt) for n, t in out.items()}


def _norm_grads(case, y, x, dy, u, w, b):
    """What a step takes from y. A gradient that is zero by the formula (the bias's in the second derivative without an
    activation) is not asked for."""
    out = {"y": y.detach()}
    if case["order"] == 1:
        names, wrt = (("dx", "dw", "db"), (x, w, b)) if case["affine"] else (("dx",), (x,))
        return out | dict(zip(names, torch.autograd.grad(y, wrt, dy)))
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    names, wrt = ["gx", "gdy"], [x, dy]
    if case["affine"]:
        names, wrt = names + ["gw"], wrt + [w]
        if case["act"] == "silu":
            names, wrt = names + ["gb"], wrt + [b]
    return out | {"dx": dx.detach()} | dict(zip(names, torch.autograd.grad(dx, wrt, u)))


# -- what a pass cannot do without -------------------------------------------------------------------------------------


def work(case):
    es = SIZES[case["dtype"]]
    if case["kind"] == "embed":
        N, V, C, ws = case["N"], case["V"], case["C"], SIZES[case["table"]]
        p = _zipf(V) if case["ids"] == "zipf" else torch.full((V,), 1.0 / V, dtype=torch.float64)
        n = N * (1.0 - case["pad"])
        touched = float((1.0 - (1.0 - p) ** n).sum())  # rows of the table that are read: the expected number
        # tokens, the table's rows -> y; dy -> the whole dense gradient
        return {"bytes": 8.0 * N + touched * C * ws + 2.0 * N * C * es + float(V) * C * ws, "flops": 2.0 * N * C}
    if case["kind"] == "distill":
        N, V, K = case["N"], case["V"], case["K"]
        return {"bytes": 2.0 * N * V * es + N * K * (es + 8.0) + 4.0, "flops": 10.0 * N * V}
    n = case["B"] * case["L"] * case["C"]
    # y of x; dx of x and dy; gx and gdy of x, dy and u: x and dy are read once in all
    tensors = 4 if case["order"] == 1 else 7
    return {"bytes": float(tensors * n * es + (16.0 * case["C"] if case["affine"] else 0.0)), "flops": (30.0 if case["order"] == 1 else 90.0) * n}


# -- the same values in 64 bits, from the definitions ------------------------------------------------------------------


def exact(case, seed):
    return {"embed": _exact_embed, "distill": _exact_distill, "norm": _exact_norm}[case["kind"]](case, _inputs(case, seed))


def _exact_embed(case, ts):
    ids, w, dy = ts["ids"], ts["weight"], ts["dy"]
    keep = ids != IGNORE
    y = torch.zeros(dy.shape, device=w.device, dtype=torch.float64)
    y[keep] = w[ids[keep]].double() * case["scale"]
    dw = torch.zeros(w.shape, device=w.device, dtype=torch.float64)
    dw.index_put_((ids[keep],), dy[keep].double(), accumulate=True)
    return {"y": y, "dw": dw * case["scale"]}


def _exact_distill(case, ts):
    T = case["T"]
    z = (ts["logits"].double() / T).requires_grad_(True)
    there = ts["ids"] != IGNORE
    some = there.any(1)
    t = (ts["teacher"].double() / T).masked_fill(~there, -math.inf)
    t = torch.where(some[:, None], t, torch.zeros_like(t))
    p = torch.softmax(t, dim=1)
    logq = torch.log_softmax(z, dim=1).gather(1, ts["ids"].clamp(min=0))
    rows = torch.where(there, p * (torch.where(there, torch.log(p.clamp(min=1e-300)), torch.zeros_like(p)) - logq), torch.zeros_like(p)).sum(1)
    loss = T * T * rows[some].sum() / max(1, int(some.sum()))
    (dz,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "dx": dz / T}


def _exact_norm(case, ts):
    """The closed forms of the group norm's first and second derivatives."""
    x, dy, u = (ts[n].double() for n in ("x", "dy", "u"))
    B, L, C = x.shape
    G = case["G"]

    def mean(v):  # over a group, for each of its elements
        return v.view(B, L, G, C // G).mean(dim=(1, 3), keepdim=True).expand(B, L, G, C // G).reshape(B, L, C)

    w = ts["weight"].double() if case["affine"] else 1.0
    b = ts["bias"].double() if case["affine"] else 0.0
    mu = mean(x)
    r = (mean((x - mu) ** 2) + EPS) ** -0.5
    h = (x - mu) * r

    def project(v):
        return r * (v - mean(v) - h * mean(v * h))

    a = w * h + b
    if case["act"] == "silu":
        sg = torch.sigmoid(a)
        f0, f1, f2 = a * sg, sg * (1 + a * (1 - sg)), sg * (1 - sg) * (2 + a * (1 - 2 * sg))
    else:
        f0, f1, f2 = a, torch.ones_like(a), torch.zeros_like(a)
    da = dy * f1
    k = w * da
    out = {"y": f0, "dx": project(k)}
    if case["order"] == 1:
        if case["affine"]:
            out |= {"dw": (da * h).sum((0, 1)), "db": da.sum((0, 1))}
        return out
    pu = project(u)
    q = w * pu
    t = dy * f2 * q
    v = w * t - r * (u * mean(k * h) + k * mean(u * h))
    along = mean(k * u) - mean(k) * mean(u) - mean(u * h) * mean(k * h)
    out |= {"gx": project(v) - r * r * h * along, "gdy": f1 * q}
    if case["affine"]:
        out["gw"] = (da * pu + t * h).sum((0, 1))
        if case["act"] == "silu":
            out["gb"] = t.sum((0, 1))
    return out
