"""GPU parity of the layer norm, the gated projection and the optimizer's step next to the borders of their plans and arguments.

Tolerances of the gated projection are those of ``tests/test_gpu_swiglu_linear.py``, whose closed forms in 64 bits are used."""

import pytest
import torch
from test_gpu_swiglu_linear import _check, _forms, _inputs, _say

from ebr_amd import block, optim
from ebr_amd.fused_attn.loader import hip_library

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}


@pytest.fixture
def cuda():
    return torch.device("cuda", 0)


# on both sides of where gate and up would go in tiles of 128 (I above 12,736) and of 256 (from 25,600 on) for these rows, and of
# 64 rows, up to which the products take what [dg|du] and [gg|gu] lack of their values before rounding
@pytest.mark.parametrize("N", [33, 48, 64, 65])
@pytest.mark.parametrize("C,I", [(72, 12736), (72, 12744), (264, 14336), (40, 25608), (71, 12745)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_projection_of_some_rows_against_a_wide_weight(cuda, N, C, I, dtype):
    _say(f"swiglu_linear wide weight {N} {C} {I} {dtype}")
    ts = _inputs(cuda, N, C, I, dtype, seed=N + I)
    got = _check(*ts.values())
    lib, code, stream = hip_library(), CODE[dtype], torch.cuda.current_stream().cuda_stream
    for order in (1, 2):  # scratch of NaN: whatever of it is read has been written
        scratch = torch.full((lib.ebr_block_swiglu_linear_scratch(code, order, N, C, I),), 255, device=cuda, dtype=torch.uint8)
        gx, gdy, gw = (torch.empty_like(ts[n]) for n in ("x", "dy", "w"))
        p = [ts[n].data_ptr() for n in ("x", "w", "dy", "c")[: order + 2]]
        if order == 1:
            rc = lib.ebr_block_swiglu_linear_bwd(code, N, C, I, *p, gx.data_ptr(), gw.data_ptr(), scratch.data_ptr(), stream)
        else:
            rc = lib.ebr_block_swiglu_linear_bwd2(code, N, C, I, *p, gx.data_ptr(), gdy.data_ptr(), gw.data_ptr(),
                                                  scratch.data_ptr(), stream)
        assert rc == 0
        assert torch.equal(gx, got[1 if order == 1 else 3]) and torch.equal(gw, got[2 if order == 1 else 5])
        assert order == 1 or torch.equal(gdy, got[4])


def test_gated_projection_carries_both_parts_up_to_64_rows(cuda):
    """Of a wide weight as of a narrow one. A rounding to bf16 is off by 2^-8 / sqrt(3) of a number's binade in the mean square,
    and a number is sqrt(1.5 / ln 2) of its binade (evenly spread over its logarithm): 1.54e-3. Values rounded once stay near that,
    those of sums whose operands were rounded too are sqrt(2) of it off, 2.2e-3; 1.9e-3 lies between."""
    _say("swiglu_linear both parts")
    for I in (520, 14336):
        ts = _inputs(cuda, 48, 136, I, torch.bfloat16, seed=I)
        got = _check(*ts.values())
        want, _ = _forms(**ts)
        for k in (1, 2, 3, 5):
            assert float((got[k].double() - want[k]).norm() / want[k].norm()) < 1.9e-3, (I, k)


@pytest.mark.parametrize("rows,C,dtype", [((1 << 22) + 5, 6, torch.float64), ((1 << 24) + 5, 2, torch.float64)])
def test_layer_norm_of_more_rows_than_a_launch_has_workgroups(cuda, rows, C, dtype):
    """fp64 rows go through workgroups of 1,024 threads, of which a launch holds fewer than 2^22: the same rows again and again give
    the same bits as once (differences there are off by at most 8 u, times r of at most 317 and a weight below 6). The parameters'
    sums are off by at most a rounding a row, and 20 of a term's own, of their terms without their signs."""
    _say(f"layer norm {rows} rows of {C}")
    g = torch.Generator(cuda).manual_seed(3)
    few, turns = 4096, -(-rows // 4096)
    base = {n: torch.randn(few, C, generator=g, device=cuda, dtype=dtype).clamp(-4, 4) for n in ("x", "dy", "u")}
    w, b = (torch.randn(C, generator=g, device=cuda, dtype=dtype).clamp(-4, 4) for _ in range(2))
    full = {n: t.repeat(turns, 1)[:rows] for n, t in base.items()}
    out = []
    for ts in (base, full):
        x, p, q = ts["x"].clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = block.layer_norm(x, p, q)
        dy = ts["dy"].clone().requires_grad_(True)
        dx, dw, db = torch.autograd.grad(y, (x, p, q), dy, create_graph=True)
        out.append([t.detach() for t in (y, dx, dw, db, *torch.autograd.grad(dx, (x, dy), ts["u"]))])
    h = base["x"] - base["x"].mean(1, keepdim=True)
    h = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
    assert float((out[0][0] - (w * h + b)).abs().max()) <= 2.0**-53 * 8 * 317 * 6
    rest = rows - (turns - 1) * few
    for one, all_ in zip(*out):
        if one.dim() == 2:
            assert torch.equal(all_[: (turns - 1) * few].view(-1, few, C), one.expand(turns - 1, few, C))
            assert torch.equal(all_[-rest:], one[:rest])
    times = torch.full((few, 1), turns - 1, device=cuda, dtype=dtype)
    times[:rest] += 1
    for got, term in ((out[1][2], base["dy"] * h), (out[1][3], base["dy"])):
        assert bool(((got - (times * term).sum(0)).abs() <= (rows + few + 20) * 2.0**-53 * (times * term.abs()).sum(0)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,C,I", [(1, 64, 32), (3, 72, 20), (17, 520, 40), (32, 71, 36), (2, 64, 6)])
def test_gated_projection_of_few_rows_at_any_address(cuda, N, C, I, dtype):
    """The C entry, whose x, w and y lie off the vectors by one to seven elements: the bits of aligned ones, and nothing beside y."""
    _say(f"swiglu_linear unaligned {N} {C} {I} {dtype}")
    ts = _inputs(cuda, N, C, I, dtype, seed=I)
    y = block.swiglu_linear(ts["x"], ts["w"])
    for off in (1, 2, 3, 7):
        x, w = (torch.empty(ts[n].numel() + off, device=cuda, dtype=dtype)[off:].copy_(ts[n].view(-1)) for n in ("x", "w"))
        out = torch.full((N * I + 16,), -7.0, device=cuda, dtype=dtype)
        rc = hip_library().ebr_block_swiglu_linear(CODE[dtype], N, C, I, x.data_ptr(), w.data_ptr(), out[off:].data_ptr(), None,
                                                   torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(out[off : off + N * I].view(N, I), y)
        assert bool((out[:off] == -7).all()) and bool((out[off + N * I :] == -7).all())


def test_gated_projection_of_more_rows_than_tiles_of_64_fit_a_launch(cuda):
    """2^29 rows and some, whose tiles of 64 would be too many and whose tiles of 256 are not: the same rows again and again give the
    same bits as once."""
    N, few, C, I = (1 << 29) + 64, 4096, 8, 8
    _say(f"swiglu_linear {N} rows")
    ts = _inputs(cuda, few, C, I, torch.bfloat16, seed=1)
    once = _check(*ts.values())
    x = ts["x"].repeat(N // few + 1, 1)[:N].requires_grad_(True)
    y = block.swiglu_linear(x, ts["w"])
    dy = ts["dy"].repeat(N // few + 1, 1)[:N]
    (dx,) = torch.autograd.grad(y, x, dy)
    for got, one in ((y.detach(), once[0]), (dx, once[1])):
        for part in got[: N // few * few].view(8, -1, few, 8):
            assert torch.equal(part, one.expand(part.shape))
        assert torch.equal(got[N // few * few :], one[: N % few])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_its_parameter(cuda, bits):
    """The bits of a step on a copy; a gradient in another's parameter is refused before anything is written."""
    _say(f"adamw on its own parameter {bits}")
    g = torch.Generator(cuda).manual_seed(1)
    start = [torch.randn(n, generator=g, device=cuda) for n in (5, 3001)]
    out = []
    for copied in (False, True):
        p = [t.clone() for t in start]
        kind = optim.STATE8 if bits == 8 else torch.float32
        m, v = ([torch.zeros(t.numel() * kind.itemsize, device=cuda, dtype=torch.uint8).view(kind) for t in p] for _ in range(2))
        s = [torch.zeros((), device=cuda, dtype=torch.int64) for _ in p]
        scales = [tuple(torch.zeros(-(-t.numel() // 256), device=cuda) for _ in range(2)) for t in p] if bits == 8 else None
        for _ in range(3):
            optim.adamw_(p, [t.clone() for t in p] if copied else p, m, v, s, lr=0.1, max_norm=1.0, scales=scales)
        out.append([*p, *m, *v, *s])
    held = [t.clone() for t in out[0][:2]]
    for grads, lr in (([p[0], p[1].clone()], p[1][7]), ([p[1][:5], p[1].clone()], 0.1)):
        with pytest.raises(ValueError, match="writes to a gradient"):
            optim.adamw_(p, grads, m, v, s, lr=lr, scales=scales)
    assert all(torch.equal(a, b) for a, b in zip(p, held))
    for a, b in zip(*out):
        assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


@pytest.mark.parametrize("N,C,I", [(5, 72, 40), (6, 71, 41), (48, 72, 12744), (48, 264, 40), (200, 136, 264), (700, 264, 1032), (9000, 520, 1032)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gated_projection_s_gradients_alone(cuda, N, C, I, dtype):
    """What is wanted alone has the bits that it has beside the rest."""
    _say(f"swiglu_linear wanted alone {N} {C} {I} {dtype}")
    x, w, dy, c = _inputs(cuda, N, C, I, dtype, seed=N).values()
    ops = torch.ops.ebr_fused
    dx, dw = ops.block_swiglu_linear_bwd(x, w, dy, True, True)
    assert torch.equal(ops.block_swiglu_linear_bwd(x, w, dy, True, False)[0], dx)
    assert torch.equal(ops.block_swiglu_linear_bwd(x, w, dy, False, True)[1], dw)
    gx, gdy, gw = ops.block_swiglu_linear_bwd2(x, w, dy, c, True, True)
    for want_x, want_w in ((True, False), (False, True), (False, False)):
        a = ops.block_swiglu_linear_bwd2(x, w, dy, c, want_x, want_w)
        assert torch.equal(a[1], gdy)
        assert torch.equal(a[0], gx) if want_x else a[0].numel() == 0
        assert torch.equal(a[2], gw) if want_w else a[2].numel() == 0
