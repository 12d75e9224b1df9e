"""GPU parity of the token ends (``ebr_amd.tokens``) against plain 64-bit formulas on the same inputs.

Tolerances are bounds of the arithmetic: half a step of the output's type, relative to the value, and for what comes before
it in 32 bits (u = 2^-24) the standard bound of a sum of n terms, n u sum |term|, and of the exponentials named at
``_soft_bounds``."""

import math

import pytest
import torch

from ebr_amd import tokens

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-24, torch.float16: 2.0**-24, torch.float64: 2.0**-53}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _half_step(t, ref):
    """Half a step of t's type at ref's values; below the normal range half of the smallest step."""
    f = torch.finfo(t.dtype)
    return (f.eps / 2 * ref.abs()).clamp(min=f.tiny * f.eps / 2)


def _near(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, what
    off = (got - ref).abs() - tol
    assert bool((off <= 0).all()), f"{what}: off by {float((got - ref).abs().max()):.3e}, {float(off.max()):.3e} over its bound"


# -- embedding ---------------------------------------------------------------------------------------------------------

PAIRS = [(torch.float32, torch.bfloat16), (torch.float32, torch.float16), (torch.float32, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float64, torch.float64)]  # fmt: skip


def _check_embed(ids, w, scale, yt, seed=7):
    w = w.detach().requires_grad_(True)
    y = tokens.embedding(ids, w, scale=scale, dtype=yt)
    assert y.dtype == yt and y.shape == (*ids.shape, w.shape[1])
    dy = torch.randn(y.shape, generator=torch.Generator(w.device).manual_seed(seed), device=w.device).to(yt)
    (dw,) = torch.autograd.grad(y, w, dy)
    assert dw.dtype == w.dtype and dw.shape == w.shape
    V, C = w.shape
    flat, g = ids.reshape(-1).long(), dy.reshape(-1, C).double()
    keep = (flat >= 0) & (flat < V)
    ref = torch.zeros(flat.numel(), C, dtype=torch.float64, device=w.device)
    ref[keep] = w.detach().double()[flat[keep]] * scale
    u = U[w.dtype]
    _near(y.reshape(-1, C), ref, _half_step(y, ref) + u * ref.abs(), "y")
    s, size = (torch.zeros(V, C, dtype=torch.float64, device=w.device) for _ in range(2))
    s.index_add_(0, flat[keep], g[keep])
    size.index_add_(0, flat[keep], g[keep].abs())
    n = torch.bincount(flat[keep], minlength=V)[:, None]
    s, size = s * scale, size * abs(scale)
    # n terms, then the product by the scale (itself rounded to 32 bits)
    _near(dw, s, _half_step(dw, s) * (s != 0) + 1.01 * u * ((n + 2) * size), "dw")
    assert bool((dw[n[:, 0] == 0] == 0).all())
    return y, dw, dy


@pytest.mark.parametrize("wt,yt", PAIRS)
@pytest.mark.parametrize("N,V,C", [(1, 1, 1), (81, 11, 512), (63, 3, 20), (130, 700, 264), (5000, 513, 24), (4096, 9, 7)])
def test_embedding(cuda, wt, yt, N, V, C):
    _say(f"embedding {N} {V} {C} {wt} {yt}")
    g = torch.Generator(cuda).manual_seed(N + V)
    ids = torch.randint(-1, V + 1, (N,), generator=g, device=cuda)
    w = torch.randn(V, C, generator=g, device=cuda).to(wt)
    _check_embed(ids, w, 1.0 if C % 2 else -1.7, yt)


# the most tokens and rows that go without a sort, and one more of each; columns that end inside a tile and off the vectors
@pytest.mark.parametrize("N,V,C", [(256, 11, 520), (257, 11, 520), (255, 32768, 8), (256, 32769, 8), (3, 32768, 9), (256, 2, 1537),
                                   (64, 5, 513), (65, 1, 24)])  # fmt: skip
@pytest.mark.parametrize("wt,yt", PAIRS[:4])
def test_embedding_of_few_tokens(cuda, wt, yt, N, V, C):
    _say(f"embedding of few {N} {V} {C} {wt} {yt}")
    g = torch.Generator(cuda).manual_seed(N)
    ids = (torch.rand(N, generator=g, device=cuda) ** 3 * V).long()
    ids[N // 2 :: 9] = -1
    ids[-1] = V - 1
    _check_embed(ids.int() if C % 2 else ids, torch.randn(V, C, generator=g, device=cuda).to(wt), 2.5, yt)


# columns that take half a vector each, or a quarter: few tokens, sorted ones in one workgroup and in many
@pytest.mark.parametrize("N,V,C", [(200, 9, 12), (200, 9, 6), (300, 40, 12), (300, 40, 10), (5000, 700, 1500), (5000, 700, 6)])
@pytest.mark.parametrize("wt,yt", PAIRS)
def test_embedding_of_half_vectors(cuda, wt, yt, N, V, C):
    _say(f"embedding of half vectors {N} {V} {C} {wt} {yt}")
    g = torch.Generator(cuda).manual_seed(N + C)
    ids = (torch.rand(N, generator=g, device=cuda) ** 3 * (V + 1)).long()
    _check_embed(ids, torch.randn(V, C, generator=g, device=cuda).to(wt), 1.5, yt)


# the largest tables whose sums a workgroup holds, with one chunk and many, and the first that do not fit
@pytest.mark.parametrize("N,V,C", [(257, 16, 130), (700, 17, 64), (5000, 32, 129), (31104, 11, 512), (20000, 32, 1679), (20000, 32, 1677),
                                   (70001, 2, 3), (300, 33, 8), (1025, 1, 66), (300000, 40, 16)])  # fmt: skip
@pytest.mark.parametrize("wt,yt", [PAIRS[0], PAIRS[2], PAIRS[4], PAIRS[5]])
def test_embedding_of_small_tables(cuda, wt, yt, N, V, C):
    _say(f"embedding of a small table {N} {V} {C} {wt} {yt}")
    g = torch.Generator(cuda).manual_seed(N)
    ids = (torch.rand(N, generator=g, device=cuda) ** 3 * V).long()
    ids[N // 3 :: 11] = -1
    ids[-1] = V - 1
    _check_embed(ids, torch.randn(V, C, generator=g, device=cuda).to(wt), 0.75, yt)


# as below, with more tokens than go without a sort, of a small table and of one whose positions are sorted
@pytest.mark.parametrize("V", [7, 40])
@pytest.mark.parametrize("ids", [
    [-1] * 290, [3] * 900, [0, 2**32 + 3, 2**40, -(2**32) + 1, 6] * 60, list(range(7)) * 50 + [7], [5] * 264 + [6] * 64, [5] * 63 + [6] * 630,
])  # fmt: skip
def test_embedding_of_special_tokens_sorted(cuda, ids, V):
    _say(f"embedding of {len(ids)} {ids[:5]}.. {V}")
    w = torch.randn(V, 16, generator=torch.Generator(cuda).manual_seed(1), device=cuda)
    _check_embed(torch.tensor(ids, device=cuda), w, 1.0, torch.float32)


# more than one workgroup's sort (4096), two and three passes of 9 bits, more than a tile a sort group (from 2^17 on), and chunks
# of more than 64 positions (from 2^19 on); the tables of 5 and 11 rows are summed without a sort
@pytest.mark.parametrize("N,V,C", [(4097, 11, 64), (20000, 50021, 40), (9000, 300001, 9), (300000, 5, 16), (1100000, 70000, 2)])
def test_embedding_sorts(cuda, N, V, C):
    _say(f"embedding sorts {N} {V} {C}")
    g = torch.Generator(cuda).manual_seed(N)
    ids = (torch.rand(N, generator=g, device=cuda) ** 4 * V).long()
    ids[:: 7] = -1
    _check_embed(ids.view(2, -1) if N % 2 == 0 else ids, torch.randn(V, C, generator=g, device=cuda), 0.5, torch.bfloat16)


@pytest.mark.parametrize("ids", [
    [-1] * 70, [3] * 200, [0, 2**32 + 3, 2**40, -(2**32) + 1, 6], list(range(7)) * 30 + [7], [5] * 64 + [6] * 64, [5] * 63 + [6] * 130,
])  # fmt: skip
def test_embedding_of_special_tokens(cuda, ids):
    _say(f"embedding of {ids[:5]}..")
    w = torch.randn(7, 16, generator=torch.Generator(cuda).manual_seed(1), device=cuda)
    _check_embed(torch.tensor(ids, device=cuda), w, 1.0, torch.float32)


def test_embedding_takes_what_users_hold(cuda):
    """int32 tokens, token and table views, a cotangent that is an expanded scalar, empty calls, a cotangent off alignment."""
    _say("embedding views")
    g = torch.Generator(cuda).manual_seed(2)
    ids = torch.randint(0, 9, (6, 10), generator=g, device=cuda, dtype=torch.int32)
    w = torch.randn(16, 9, generator=g, device=cuda).t()
    _check_embed(ids, w, 2.0, torch.bfloat16)
    _check_embed(ids.t()[1:, ::2], w, 2.0, torch.float32)
    wide = torch.randn(9, 17, generator=g, device=cuda)
    _check_embed(ids, wide.view(-1)[1:145].view(9, 16), 2.0, torch.bfloat16)
    leaf = w.detach().clone().requires_grad_(True)
    tokens.embedding(ids, leaf).sum().backward()
    assert torch.equal(leaf.grad[:, 0], torch.bincount(ids.reshape(-1).long(), minlength=9).float())
    dy = torch.randn(961, generator=g, device=cuda)[1:].view(6, 10, 16)
    (dw,) = torch.autograd.grad(tokens.embedding(ids, leaf), leaf, dy)
    assert torch.equal(dw, torch.autograd.grad(tokens.embedding(ids, leaf), leaf, dy.clone())[0])
    assert torch.equal(tokens.embedding(torch.tensor(3, device=cuda), leaf), leaf[3])  # one token, no batch
    for shape, V, C in (((0,), 5, 8), ((2, 0), 5, 8), ((3,), 5, 0), ((3,), 0, 8)):
        t = torch.zeros(V, C, device=cuda, requires_grad=True)
        y = tokens.embedding(torch.zeros(shape, dtype=torch.int64, device=cuda), t)
        assert y.shape == (*shape, C) and bool((y == 0).all())
        (dw,) = torch.autograd.grad(y.sum(), t)
        assert dw.shape == t.shape and bool((dw == 0).all())


def test_embedding_repeats_its_bits_and_differentiates_again(cuda):
    _say("embedding again")
    g = torch.Generator(cuda).manual_seed(3)
    ids = torch.randint(0, 5, (3000,), generator=g, device=cuda)
    w = torch.randn(5, 96, generator=g, device=cuda)
    first = _check_embed(ids, w, 1.0, torch.bfloat16)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _check_embed(ids, w, 1.0, torch.bfloat16)))
    few = torch.tensor([0, 2, 2, -1, 4, 1], device=cuda)
    table = torch.randn(5, 3, generator=g, device=cuda, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: tokens.embedding(few, t, 1.5), (table,))
    assert torch.autograd.gradgradcheck(lambda t: tokens.embedding(few, t, 1.5).pow(3), (table,))
    # the gradient's own gradient is the lookup: exactly c[ids] of a cotangent c
    dy = torch.randn(6, 3, generator=g, device=cuda, requires_grad=True)
    t32 = table.detach().float().requires_grad_(True)
    (dw,) = torch.autograd.grad(tokens.embedding(few, t32), t32, dy, create_graph=True)
    c = torch.randn(5, 3, generator=g, device=cuda)
    (back,) = torch.autograd.grad(dw, dy, c)
    assert torch.equal(back, torch.where((few >= 0)[:, None], c[few.clamp(min=0)], torch.zeros_like(back)))


# sorted in many workgroups (more than 4,096 positions, and more than 16 rows or, of many, 32): one pass of 9 bits and two, a
# tile of 1,024 a workgroup and more (from 2^17 positions on), chunks of 64 positions and more (from 2^19 on), sixteen bits
# and 32, and half and single vectors; every other position the same token, whose run goes over most chunks' borders
@pytest.mark.parametrize("wt,yt", [PAIRS[0], PAIRS[2], PAIRS[3]])
@pytest.mark.parametrize("N,V,C", [(4097, 33, 64), (31104, 40, 512), (140000, 600, 12), (300000, 50021, 16), (530001, 37, 8), (70001, 300, 5)])
def test_embedding_sorts_in_many_workgroups_and_repeats_its_bits(cuda, wt, yt, N, V, C):
    _say(f"embedding sorts, again {N} {V} {C} {wt} {yt}")
    g = torch.Generator(cuda).manual_seed(N)
    ids = (torch.rand(N, generator=g, device=cuda) ** 2 * V).long()
    ids[::2] = V // 2
    ids[::5] = -1
    w = torch.randn(V, C, generator=g, device=cuda).to(wt).requires_grad_(True)
    dy = torch.randn(N, C, generator=g, device=cuda).to(yt)
    dw = [torch.autograd.grad(tokens.embedding(ids, w, 0.5, yt), w, dy)[0] for _ in range(4)]
    assert all(torch.equal(dw[0], d) for d in dw[1:])
    flat, d = ids.cpu(), dy.cpu().double()  # (half of the rows to one: on the GPU that takes seconds)
    keep = flat >= 0
    ref, size = (torch.zeros(V, C, dtype=torch.float64).index_add_(0, flat[keep], v[keep]) * 0.5 for v in (d, d.abs()))
    n = torch.bincount(flat[keep], minlength=V)[:, None]
    got = dw[0].cpu()
    _near(got, ref, _half_step(got, ref) * (ref != 0) + 1.01 * U[wt] * (n + 2) * size, "dw")  # the bound of _check_embed


def test_embedding_gradient_of_the_most_positions(cuda):
    """The most tokens that a call takes, sorted: the last chunk's end passes 32 bits. Ones are counted: whole numbers below
    2^24 exactly, the others by at most 8,192 additions of parts (2^-24 each)."""
    _say("embedding of 2^31 - 4097 tokens")
    N, V = 2**31 - 4097, 40
    ids = torch.full((N,), 3, dtype=torch.int32, device=cuda)
    ids[::7159] = V - 1
    w = torch.randn(V, 1, generator=torch.Generator(cuda).manual_seed(1), device=cuda, requires_grad=True)
    y = tokens.embedding(ids, w, dtype=torch.bfloat16)
    last = -(-N // 7159)
    assert y[7159 * (last - 1)] == w[V - 1].bfloat16() and y[N - 1] == w[3 if (N - 1) % 7159 else V - 1].bfloat16()
    (dw,) = torch.autograd.grad(y, w, torch.ones(1, 1, device=cuda, dtype=torch.bfloat16).expand(N, 1))
    assert dw[V - 1].item() == last
    assert abs(dw[3].item() - (N - last)) <= 8192 * 2.0**-24 * N
    dw[3], dw[V - 1] = 0, 0
    assert bool((dw == 0).all())


# -- distillation ------------------------------------------------------------------------------------------------------


def _soft_bounds(x, T, n, u, finite):
    """A bound of the relative error of softmax(x / T) in arithmetic of unit u, where the sum of a row goes through chains of
    n additions, and its largest exponent. The exponent (x - max) log2(e) / T is rounded three times (the difference, log2(e) /
    T, the product) and once more minus the sum's log2: 4 u of its size; the two powers of two and the logarithm are each
    within two steps (4 u); every addition of the chain may rescale (one more power, exponent and product)."""
    z = torch.where(finite, x / T, torch.full_like(x, -math.inf))
    top = z.amax(-1, keepdim=True)
    far = torch.where(torch.isfinite(z), top - z, torch.zeros_like(z)).amax().item() + math.log(x.shape[-1] + 1.0)
    return u * (5 * far * 1.5 + 12 + 8 * n), far


def _reference(x, t, ids, T):
    """Row losses, gradients of each row's loss, p summed by column, q: in 64 bits."""
    V = x.shape[-1]
    there = (ids >= 0) & (ids < V)
    x = x.double()
    logq = torch.log_softmax(x / T, dim=-1)
    tz = torch.where(there, t.double() / T, torch.full((), -math.inf, device=x.device, dtype=torch.float64))
    some = torch.isfinite(tz).any(-1) & (tz > -math.inf).any(-1)
    p = torch.where(some[..., None], torch.softmax(torch.where(some[..., None], tz, torch.zeros_like(tz)), -1), torch.zeros_like(tz))
    at = ids.clamp(0, V - 1).long()
    lq = logq.gather(-1, at)
    term = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)) - lq), torch.zeros_like(p))
    size = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)).abs() + lq.abs() + 1), torch.zeros_like(p))
    byc = torch.zeros_like(x).scatter_add_(-1, at, p)
    q = logq.exp() * some[..., None]
    return term.sum(-1) * T * T, size.sum(-1) * T * T, T * (q - byc), byc, q, some


def _check_distill(x, t, ids, T=1.0, reduction="mean", upstream=None):
    x = x.detach().requires_grad_(True)
    loss = tokens.distill_loss(x, t, ids, temperature=T, reduction=reduction)
    K, V = t.shape[-1], x.shape[-1]
    u = U[x.dtype]
    assert loss.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    rows, size, drow, byc, q, some = _reference(x.detach(), t, ids, T)
    n = max(1, int(some.sum()))
    rel, far = _soft_bounds(x.detach().double(), T, V // 8 + K + 64, u, torch.isfinite(x.detach().double()))
    there = (ids >= 0) & (ids < V) & torch.isfinite(t.double())
    prel, pfar = _soft_bounds(t.double(), T, K + 64, u, there)
    row_tol = size * (rel + prel) * 2 + (rel + prel) * 2 * T * T * (1 + far + pfar) * some
    if reduction == "none":
        ref, tol, each = rows, row_tol, 1.0
    else:
        each = 1.0 / n if reduction == "mean" else 1.0
        ref, tol = rows.sum() * each, row_tol.sum() * each
    _near(loss.detach(), ref, tol + _half_step(loss, ref), "loss")
    g = torch.ones_like(loss) if upstream is None else upstream.to(loss.dtype)
    (dx,) = torch.autograd.grad(loss, x, g)
    assert dx.dtype == x.dtype
    factor = g.double()[..., None] * each
    ref = drow * factor
    _near(dx, ref, _half_step(dx, ref) * (ref != 0) + (T * factor.abs()) * 2 * (q * rel + byc * (prel + K * u)) + 8 * u * ref.abs(), "dx")
    assert bool((dx[~some] == 0).all())
    return loss.detach(), dx


def _teacher(cuda, lead, V, K, seed, invalid=0.0):
    g = torch.Generator(cuda).manual_seed(seed)
    ids = torch.rand(*lead, V, generator=g, device=cuda).topk(K, dim=-1).indices
    if invalid:
        ids = torch.where(torch.rand(ids.shape, generator=g, device=cuda) < invalid, torch.full_like(ids, -1), ids)
    return torch.randn(*lead, K, generator=g, device=cuda) * 3, ids


DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,V,K", [((1,), 1, 1), ((81,), 11, 4), ((3, 7), 8, 8), ((5,), 17, 3), ((33,), 64, 64), ((9,), 65, 5),
                                      ((4, 3), 2048, 32), ((3,), 2049, 300), ((2,), 50021, 64), ((5,), 1000, 1000), ((40,), 33, 1)])  # fmt: skip
def test_distill(cuda, dtype, lead, V, K):
    _say(f"distill {lead} {V} {K} {dtype}")
    x = (torch.randn(*lead, V, generator=torch.Generator(cuda).manual_seed(V), device=cuda) * 3).to(dtype)
    t, ids = _teacher(cuda, lead, V, K, seed=K)
    _check_distill(x, t, ids, T=1.0 if K % 2 else 2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 97, 5000, 20000])
@pytest.mark.parametrize("T", [0.5, 1.0])
def test_distill_entry_whose_logit_a_mask_has_set_to_the_lowest_value(cuda, dtype, V, T):
    """The loss is p (max - lowest) T but for terms of order 1, half of the largest float at T = 1: finite in 32 bits, though
    the logarithm in base 2, or at T = 0.5, is not. p = 1/2 exactly, and 16 steps are far more than the roundings of the
    difference, the product and the result (half a step each)."""
    _say(f"distill lowest logit {V} {dtype} {T}")
    x = torch.randn(7, V, generator=torch.Generator().manual_seed(3)).to(cuda, dtype)
    x[:, 1] = torch.finfo(dtype).min
    ids = torch.tensor([[1, 2]], device=cuda).expand(7, 2)
    t = torch.zeros(7, 2, device=cuda)
    x.requires_grad_(True)
    ref = 0.5 * T * (x.detach().double().amax(-1) - torch.finfo(dtype).min)
    rows = tokens.distill_loss(x, t, ids, T, "none")
    loss = tokens.distill_loss(x, t, ids, T)
    assert bool(((rows.detach().double() - ref).abs() <= 16 * 2.0**-24 * ref).all())
    assert abs(loss.item() - ref.mean().item()) <= 16 * 2.0**-24 * ref.mean().item()
    (dx,) = torch.autograd.grad(loss, x)
    assert bool(torch.isfinite(dx).all())
    want = -T * 0.5 / 7  # no probability of its own
    assert bool(((dx[:, 1].double() - want).abs() <= torch.finfo(dtype).eps * abs(want)).all())


# every number of threads a row, rows that end inside a workgroup, and many entries for short rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("N,V,K", [(70, 32, 5), (70, 33, 33), (50, 97, 8), (37, 130, 100), (19, 300, 256), (9, 500, 500), (6, 1024, 1024),
                                   (3, 2000, 1024), (700, 2100, 3), (2, 140000, 1024), (2, 300000, 700)])  # fmt: skip
def test_distill_teams(cuda, dtype, N, V, K):
    _say(f"distill teams {N} {V} {K} {dtype}")
    g = torch.Generator(cuda).manual_seed(N)
    x = (torch.randn(N, V, generator=g, device=cuda) * 2).to(dtype)
    t, ids = _teacher(cuda, (N,), V, K, seed=K)
    _check_distill(x, t, ids, T=1.5)
    ids[::2] = torch.randint(0, V, ids[::2].shape, generator=g, device=cuda)  # with tokens named twice
    _check_distill(x, t, ids, T=1.5)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("V,K", [(11, 5), (700, 20), (5000, 70)])
def test_distill_ragged_rows(cuda, reduction, V, K):
    """Rows with some entries, one, or none; what the entries that do not count hold is never used."""
    _say(f"distill ragged {reduction} {V} {K}")
    lead = (4, 9)
    x = torch.randn(*lead, V, generator=torch.Generator(cuda).manual_seed(V), device=cuda) * 3
    t, ids = _teacher(cuda, lead, V, K, seed=K, invalid=0.5)
    ids[0, :3], ids[1, 1, 1:] = -1, -100
    ids[2, 2, 0] = V  # just outside
    t[0, 0], t[0, 1], t[0, 2] = math.nan, math.inf, torch.finfo(torch.float32).min
    up = torch.rand(lead, generator=torch.Generator(cuda).manual_seed(1), device=cuda) if reduction == "none" else torch.tensor(0.3, device=cuda)
    a = _check_distill(x, t, ids, T=0.8, reduction=reduction, upstream=up)
    b = _check_distill(x, torch.where((ids >= 0) & (ids < V), t, torch.full_like(t, math.nan)), ids, T=0.8, reduction=reduction, upstream=up)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("V", [11, 300, 4000])
def test_distill_masked_logits(cuda, V):
    """Student logits of -inf or the type's lowest value, and teacher entries of -inf, in a row with others."""
    _say(f"distill masked {V}")
    x = torch.randn(6, V, generator=torch.Generator(cuda).manual_seed(V), device=cuda)
    t, ids = _teacher(cuda, (6,), V, 4, seed=3)
    off = torch.ones(6, V, dtype=torch.bool, device=cuda).scatter_(1, ids, False) & (torch.arange(V, device=cuda) % 3 > 0)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        _check_distill(x.masked_fill(off, low).to(torch.bfloat16), t, ids)
    for dtype in (torch.float32, torch.bfloat16):  # a row whose mask leaves nothing: as if all were equal
        y = x.to(dtype)
        y[4] = torch.finfo(dtype).min
        _check_distill(y, t, ids, T=0.9)
    t[0, 1:], t[1, 0], t[2] = -math.inf, -math.inf, -math.inf  # one entry left, one gone, a row without any
    _check_distill(x, t, ids)
    # the teacher wants what the student rules out: infinite, by the formula
    x[3, ids[3, 0]] = -math.inf
    leaf = x.detach().requires_grad_(True)
    loss = tokens.distill_loss(leaf, t, ids, reduction="none")
    assert bool(torch.isinf(loss[3])) and bool(torch.isfinite(loss[4]))
    bad = x.clone()
    bad[5, 1] = math.nan
    assert bool(torch.isnan(tokens.distill_loss(bad, t, ids, reduction="none")[5]))


@pytest.mark.parametrize("V,K", [(11, 9), (700, 40), (3000, 40)])
def test_distill_same_token_twice(cuda, V, K):
    _say(f"distill twice {V} {K}")
    g = torch.Generator(cuda).manual_seed(4)
    x, t = torch.randn(5, V, generator=g, device=cuda), torch.randn(5, K, generator=g, device=cuda)
    ids = torch.randint(0, min(V, 6), (5, K), generator=g, device=cuda)
    _check_distill(x, t, ids)


def test_distill_is_the_cross_entropy_to_one_token(cuda):
    _say("distill cross entropy")
    g = torch.Generator(cuda).manual_seed(5)
    x = torch.randn(50, 97, generator=g, device=cuda, requires_grad=True)
    y = torch.randint(0, 97, (50,), generator=g, device=cuda)
    loss = tokens.distill_loss(x, torch.zeros(50, 1, device=cuda), y[:, None].int())
    ref = torch.nn.functional.cross_entropy(x.double(), y)
    assert abs(float(loss) - float(ref)) <= 40 * 2.0**-24 * float(ref)


def test_distill_takes_what_users_hold(cuda):
    """A slice of padded rows, a transposed tensor, an expanded row, misaligned rows, 16-bit teachers, empty calls; equal bits
    every time."""
    _say("distill views")
    g = torch.Generator(cuda).manual_seed(6)
    t, ids = _teacher(cuda, (3, 5), 100, 7, seed=8)
    wide = torch.randn(3, 5, 128, generator=g, device=cuda)
    a = _check_distill(wide[..., :100], t, ids)
    b = _check_distill(wide[..., :100].contiguous(), t.clone(), ids.int())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    _check_distill(wide[..., 1:101].bfloat16(), t.bfloat16(), ids)
    _check_distill(torch.randn(100, 5, 3, generator=g, device=cuda).permute(2, 1, 0), t.half(), ids)
    _check_distill(wide[:1, :1, :100].expand(3, 5, 100), t, ids)
    _check_distill(wide.view(-1)[1:1501].view(3, 5, 100), t.double(), ids)
    _check_distill(wide[0, 0, :100], t[0, 0], ids[0, 0])  # one row without a batch
    for reduction, want in (("mean", ()), ("sum", ()), ("none", (0, 5))):
        x = torch.zeros(0, 5, 100, device=cuda, requires_grad=True)
        loss = tokens.distill_loss(x, t[:0], ids[:0], reduction=reduction)
        assert loss.shape == want and bool((loss == 0).all())
        assert torch.autograd.grad(loss.sum(), x)[0].shape == x.shape
    nothing = tokens.distill_loss(wide[..., :100], t, torch.full_like(ids, -1))
    assert float(nothing) == 0.0


def test_distill_gradients_by_differences(cuda):
    _say("distill gradcheck")
    g = torch.Generator(cuda).manual_seed(9)
    ids = torch.tensor([[0, 3, 3], [-1, 2, 1], [-1, -1, -1]], device=cuda)
    t = torch.randn(3, 3, generator=g, device=cuda, dtype=torch.float64)
    x = torch.randn(3, 5, generator=g, device=cuda, dtype=torch.float64, requires_grad=True)
    for reduction in ("mean", "sum", "none"):
        assert torch.autograd.gradcheck(lambda v: tokens.distill_loss(v, t, ids, 1.7, reduction), (x,))
    (dx,) = torch.autograd.grad(tokens.distill_loss(x, t, ids), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [8191, 8192, 50021, 300000])
def test_distill_of_no_rows_of_a_long_vocabulary(cuda, dtype, V):
    """Few long rows are split into parts; no rows have none: the sum and the mean are 0, the gradient is empty."""
    _say(f"distill no rows {V} {dtype}")
    t, ids = torch.zeros(0, 3, 4, device=cuda), torch.zeros(0, 3, 4, dtype=torch.int64, device=cuda)
    for reduction, want in (("mean", ()), ("sum", ()), ("none", (0, 3))):
        x = torch.zeros(0, 3, V, device=cuda, dtype=dtype, requires_grad=True)
        loss = tokens.distill_loss(x, t, ids, 2.0, reduction)
        assert loss.shape == want and bool((loss == 0).all())
        assert torch.autograd.grad(loss.sum(), x)[0].shape == x.shape


# -- streams and graphs ------------------------------------------------------------------------------------------------


def _step(ids, w, out_w, t, tids):
    y = tokens.embedding(ids, w, dtype=torch.bfloat16)
    loss = tokens.distill_loss(y.float() @ out_w, t, tids, 2.0)
    return loss, *torch.autograd.grad(loss, (w, out_w))


def _step_inputs(cuda, n=600, V=40, C=32):
    g = torch.Generator(cuda).manual_seed(12)
    ids = torch.randint(0, V, (n,), generator=g, device=cuda)
    w = torch.randn(V, C, generator=g, device=cuda, requires_grad=True)
    out_w = torch.randn(C, V, generator=g, device=cuda, requires_grad=True)
    t, tids = _teacher(cuda, (n,), V, 5, seed=1)
    return ids, w, out_w, t, tids


def test_tokens_compiled(cuda):
    """Under torch.compile (no Triton) the same ops run, with the eager call's bits."""
    _say("tokens compiled")
    a = _step_inputs(cuda)

    def loss_of(ids, w, out_w, t, tids):
        return tokens.distill_loss(tokens.embedding(ids, w, dtype=torch.bfloat16).float() @ out_w, t, tids, 2.0)

    loss = torch.compile(loss_of, backend="aot_eager")(*a)
    got = loss, *torch.autograd.grad(loss, (a[1], a[2]))
    assert all(torch.equal(p, q) for p, q in zip(got, _step(*a)))


def test_tokens_from_two_threads(cuda):
    """Two programs' calls at once, each on a stream of its own."""
    _say("tokens threads")
    import threading

    a = _step_inputs(cuda)
    ref = _step(*a)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            own = [p.detach().clone().requires_grad_(p.requires_grad) for p in a]
            for _ in range(5):
                got[i] = _step(*own)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(p, q) for i in range(2) for p, q in zip(ref, got[i]))


def test_tokens_on_another_stream(cuda):
    _say("tokens stream")
    a = _step_inputs(cuda)
    ref = _step(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(*a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(ref, got))


def test_tokens_captured(cuda):
    """A captured step replays on new contents, with eager work between the replays; two graphs do not share scratch."""
    _say("tokens graph")
    ids, w, out_w, t, tids = _step_inputs(cuda)
    leaf = [p.detach().clone().requires_grad_(True) for p in (w, out_w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(ids, *leaf, t, tids)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(ids, *leaf, t, tids)
        graphs.append((graph, out))
    for turn in range(3):
        ids.copy_((ids * 7 + turn) % 40)
        with torch.no_grad():
            leaf[0].mul_(0.9)
        ref = _step(ids, *(p.detach().clone().requires_grad_(True) for p in leaf), t, tids)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(ref, out))
