"""Host-side checks of the layer norm, the gated projection and the optimizer's step, no GPU: the ops' fakes give the shapes and
types that the kernels write, wrong arguments are refused before anything runs, here and at the C entry points, the scratch
sizes, and the network's plain forms. Parity of the kernels is in ``tests/test_gpu_layernorm.py``,
``tests/test_gpu_swiglu_linear.py`` and ``tests/test_gpu_optim.py``."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ebr_amd import _capi, block, layers, optim
from ebr_amd import energy as en

P = 0x100000  # a placeholder that no refused call reads


@pytest.mark.parametrize("dtype,acc", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float64, torch.float64)])
def test_fakes(dtype, acc):
    ops = torch.ops.ebr_fused
    with FakeTensorMode():
        x, w = torch.empty(2, 5, 12, dtype=dtype), torch.empty(12, dtype=torch.bfloat16)
        y, stats = ops.block_layernorm(x, w, None, 1e-5)
        assert y.shape == x.shape and y.dtype == dtype and stats.shape == (10, 4) and stats.dtype == acc
        dx, dw, db = ops.block_layernorm_bwd(x, w, stats, y, torch.bfloat16, True)
        assert dx.shape == x.shape and dw.shape == db.shape == (12,) and dw.dtype == torch.bfloat16
        gx, gdy, gw = ops.block_layernorm_bwd2(x, w, stats, y, x, None, None, torch.bfloat16, False)
        assert gx.shape == gdy.shape == x.shape and gw.shape == (0,)
        w2 = torch.empty(14, 12, dtype=dtype)
        y = ops.block_swiglu_linear(x, w2)
        assert y.shape == (2, 5, 7) and y.dtype == dtype
        dx, dw = ops.block_swiglu_linear_bwd(x, w2, y, True, False)
        assert dx.shape == x.shape and dw.shape == (0,)
        gx, gdy, gw = ops.block_swiglu_linear_bwd2(x, w2, y, x, False, True)
        assert gx.shape == (0,) and gdy.shape == y.shape and gw.shape == w2.shape
        norm, single = ops.grad_norm([x, w])
        assert norm.dtype == torch.float64 and single.dtype == torch.float32 and norm.shape == single.shape == ()


def _norm(x=(3, 8), w=(8,), b=(8,), xt=torch.float32, wt=torch.float32, **kw):
    return block.layer_norm(torch.zeros(x, dtype=xt), torch.zeros(w, dtype=wt), torch.zeros(b), **kw)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: _norm(xt=torch.int32)),
    (TypeError, lambda: _norm(wt=torch.int64)),
    (ValueError, lambda: _norm(x=())),
    (ValueError, lambda: _norm(x=(3, 0), w=(0,), b=(0,))),
    (ValueError, lambda: _norm(w=(7,))),
    (ValueError, lambda: _norm(b=(1, 8))),
    (ValueError, lambda: _norm(eps=-1e-5)),
    (ValueError, lambda: _norm(eps=float("nan"))),
    (ValueError, lambda: block.layer_norm(torch.zeros(3, 8), torch.zeros(8, device="meta"))),
    (NotImplementedError, lambda: _norm()),  # no kernel off the GPU
])  # fmt: skip
def test_layer_norm_refuses(error, call):
    with pytest.raises(error):
        call()


def _glu(x=(3, 8), w=(6, 8), xt=torch.float32, wt=torch.float32):
    return block.swiglu_linear(torch.zeros(x, dtype=xt), torch.zeros(w, dtype=wt))


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: _glu(xt=torch.int32, wt=torch.int32)),
    (TypeError, lambda: _glu(wt=torch.bfloat16)),
    (ValueError, lambda: _glu(w=(6, 7))),
    (ValueError, lambda: _glu(w=(5, 8))),
    (ValueError, lambda: _glu(w=(0, 8))),
    (ValueError, lambda: _glu(w=(8,))),
    (ValueError, lambda: _glu(x=())),
    (ValueError, lambda: _glu(x=(3, 0), w=(6, 0))),
    (ValueError, lambda: block.swiglu_linear(torch.zeros(3, 8), torch.zeros(6, 8, device="meta"))),
    (NotImplementedError, lambda: _glu()),  # no kernel off the GPU
])  # fmt: skip
def test_swiglu_linear_refuses(error, call):
    with pytest.raises(error):
        call()


def _step(n=2, bits=32, **kw):
    p, g = ([torch.zeros(4) for _ in range(n)] for _ in range(2))
    state = torch.float8_e4m3fn if bits == 8 else torch.float32
    m, v = ([torch.zeros(4, dtype=torch.uint8).view(state) if bits == 8 else torch.zeros(4) for _ in range(n)] for _ in range(2))
    s = [torch.zeros((), dtype=torch.int64) for _ in range(n)]
    scales = [(torch.zeros(1), torch.zeros(1)) for _ in range(n)] if bits == 8 else None
    a = dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, steps=s, scales=scales, lr=1e-3) | kw
    return optim.adamw_(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), a.pop("steps"), **a)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(n=0)),
    (ValueError, dict(grads=[torch.zeros(4)])),
    (ValueError, dict(params=[torch.zeros(5), torch.zeros(4)])),
    (ValueError, dict(exp_avgs=[torch.zeros(8)[::2], torch.zeros(4)])),
    (ValueError, dict(lr=-1e-3)), (ValueError, dict(lr=float("inf"))), (ValueError, dict(lr=torch.zeros(2))),
    (ValueError, dict(betas=(0.9, 1.0))), (ValueError, dict(betas=(-0.1, 0.9))), (ValueError, dict(eps=-1.0)),
    (ValueError, dict(weight_decay=float("nan"))), (ValueError, dict(max_norm=0.0)), (ValueError, dict(max_norm=float("nan"))),
    (TypeError, dict(grads=[torch.zeros(4, dtype=torch.float64)] * 2)),
    (TypeError, dict(exp_avgs=[torch.zeros(4, dtype=torch.float16)] * 2)),
    (TypeError, dict(steps=[torch.zeros(())] * 2)),
    (ValueError, dict(bits=8, scales=[(torch.zeros(2), torch.zeros(1))] * 2)),
    (TypeError, dict(bits=8, exp_avgs=[torch.zeros(4)] * 2)),
    (NotImplementedError, dict()),  # no kernel off the GPU
    (NotImplementedError, dict(bits=8)),
])  # fmt: skip
def test_adamw_refuses(error, kw):
    with pytest.raises(error):
        _step(**kw)


def test_the_same_tensor_twice():
    p = torch.zeros(4)
    with pytest.raises(ValueError, match="twice"):
        _step(params=[p, p])
    s = torch.zeros((), dtype=torch.int64)
    with pytest.raises(ValueError, match="twice"):
        _step(steps=[s, s])


def test_tensors_that_share_memory():
    m = torch.zeros(10)
    with pytest.raises(ValueError, match="share memory"):
        _step(exp_avgs=[m[:4], m[4:8]], exp_avg_sqs=[m[6:], torch.zeros(4)])
    with pytest.raises(NotImplementedError):  # side by side: no kernel off the GPU
        _step(exp_avgs=[m[:4], m[4:8]])


def test_entries_refuse():
    lib = _capi.load()
    ln, ln1, ln2 = lib.ebr_block_layernorm, lib.ebr_block_layernorm_bwd, lib.ebr_block_layernorm_bwd2
    assert ln(4, 0, 3, 8, 1e-5, P, P, P, P, P, None) == 1 and ln(1, 7, 3, 8, 1e-5, P, P, P, P, P, None) == 1
    for rows, C in ((0, 8), (-1, 8), (3, 0), (3, (1 << 24) + 1), (1 << 37, 8), (1 << 62, 8)):
        assert ln(1, 0, rows, C, 1e-5, P, P, P, P, P, None) == 2
        assert ln1(1, 0, rows, C, P, P, P, P, P, P, P, P, None) == 2
        assert lib.ebr_block_layernorm_scratch(1, 1, rows, C) == -1
    assert ln(1, 0, 3, 8, 1e-5, 0, P, P, P, P, None) == 4 and ln(1, 0, 3, 8, 1e-5, P, P, P, P, 0, None) == 4
    assert ln1(1, 0, 3, 8, P, P, P, 0, P, P, P, P, None) == 4
    assert ln1(1, 0, 3, 8, P, P, P, P, P, P, P, 0, None) == 5 and ln1(1, 0, 3, 8, P, P, P, P, P, P, P, P + 8, None) == 3
    assert ln2(1, 0, 3, 8, P, P, P, P, P, P, P, P, 0, P, P, None) == 4
    assert ln2(1, 0, 3, 8, P, P, P, P, P, P, P, P, P, P, 0, None) == 5

    f, b1, b2 = lib.ebr_block_swiglu_linear, lib.ebr_block_swiglu_linear_bwd, lib.ebr_block_swiglu_linear_bwd2
    assert f(4, 3, 8, 8, P, P, P, P, None) == 1
    for N, C, I in ((0, 8, 8), (3, 0, 8), (3, 8, 0), (1 << 31, 8, 8), (3, (1 << 20) - 7, 8), (3, 8, (1 << 19) - 7),
                    ((1 << 31) - 1, 8, 1 << 18)):
        assert f(1, N, C, I, P, P, P, P, None) == 2
        assert b1(1, N, C, I, P, P, P, P, P, P, None) == 2
        assert b2(1, N, C, I, P, P, P, P, P, P, P, P, None) == 2
        assert lib.ebr_block_swiglu_linear_scratch(1, 1, N, C, I) == -1
    assert f(1, 40, 8, 9, P, P, P, 0, None) == 5 and f(1, 40, 8, 9, P, P, P, P + 8, None) == 3  # copies want scratch
    assert f(1, 40, 8, 8, P + 2, P, P, 0, None) == 3 and f(1, 40, 8, 8, P, P, P + 8, 0, None) == 3
    assert b1(1, 3, 8, 8, P, P + 2, P, P, P, P, None) == 3 and b2(1, 3, 8, 8, P, P, P, P + 4, P, P, P, P, None) == 3
    assert lib.ebr_block_swiglu_linear_scratch(1, 0, 40, 8, 8) == lib.ebr_block_swiglu_linear_scratch(1, 0, 3, 9, 9) == 0
    assert f(1, 3, 8, 8, P, P, 0, P, None) == 4 and b1(1, 3, 8, 8, P, 0, P, P, P, P, None) == 4
    assert b1(1, 3, 8, 8, P, P, P, P, P, 0, None) == 5 and b1(1, 3, 8, 8, P, P, P, P, P, P + 4, None) == 3
    assert b1(1, 3, 8, 8, P, P, P, 0, 0, P, None) == 0  # nothing wanted, nothing done
    assert b2(1, 3, 8, 8, P, P, P, P, P, 0, P, P, None) == 4


def _table(rows=2, **kw):
    table = [dict(p=P + 4096 * k, g=P, m=P + 4096 * (k + 16), v=P + 4096 * (k + 32), ms=P + 4096 * (k + 48), vs=P + 4096 * (k + 64),
                  step=P + 4096 * 80 + 8 * k, n=100) | kw for k in range(rows)]
    return (_capi.OptimTensor * rows)(*(tuple(r[f] for f, _ in _capi.OptimTensor._fields_) for r in table))


@pytest.mark.parametrize("code,kw", [
    (1, dict(pt=4)), (1, dict(gt=-1)), (1, dict(pt=1, gt=0)), (1, dict(pt=0, gt=3)), (1, dict(bits=16)), (1, dict(pt=3, gt=3, bits=8)),
    (2, dict(count=-1)), (2, dict(b1=1.0)), (2, dict(b2=float("nan"))), (2, dict(eps=-1.0)), (2, dict(row=dict(n=-1))),
    (2, dict(row=dict(n=1 << 40))), (2, dict(row=dict(m=P + 4096 * 32 + 396))), (2, dict(bits=8, row=dict(vs=P + 4096 * 16 + 96))), (2, dict(row=dict(p=P))), (2, dict(row=dict(step=P))),
    (4, dict(row=dict(g=0))), (4, dict(row=dict(step=0))), (4, dict(bits=8, row=dict(vs=0))), (4, dict(table=0)),
    (5, dict(scratch=0)), (3, dict(scratch=P + 8)), (0, dict(count=0)),
])  # fmt: skip
def test_adamw_entry_refuses(code, kw):
    a = dict(pt=0, gt=0, bits=32, count=2, b1=0.9, b2=0.99, eps=1e-8, scratch=P, row={}) | kw
    table = _table(**a["row"])
    at = a.get("table", ctypes.addressof(table))
    rc = _capi.load().ebr_block_adamw(a["pt"], a["gt"], a["bits"], a["count"], at, 1e-3, None, a["b1"], a["b2"], a["eps"], 0.0, None,
                                      0.0, a["scratch"], None)
    assert rc == code


def test_grad_norm_entry_refuses():
    lib = _capi.load()

    def call(g=P, n=100, dtype=0, count=1, norm=P, scratch=P):
        table = (_capi.OptimGrad * 1)((g, n, dtype, 0))
        return lib.ebr_block_grad_norm(count, ctypes.addressof(table), norm, None, scratch, None)

    assert [call(count=0), call(n=-1), call(n=1 << 40), call(dtype=9), call(g=0), call(norm=0), call(scratch=0), call(scratch=P + 8)] == [
        2, 2, 2, 1, 4, 4, 5, 3]
    assert lib.ebr_block_grad_norm_scratch(0, None) == -1 and lib.ebr_block_adamw_scratch(-1) == -1


def test_scratch_sizes():
    lib = _capi.load()
    assert lib.ebr_block_layernorm_scratch(1, 1, 81, 512) >= 21 * 2 * 512 * 4
    assert lib.ebr_block_layernorm_scratch(3, 2, 81, 512) >= 81 * 8 * 8
    assert lib.ebr_block_layernorm_scratch(1, 3, 81, 512) == -1
    # [dg | du], and beside them what few rows' roundings leave
    assert lib.ebr_block_swiglu_linear_scratch(1, 1, 1000, 64, 32) >= 1000 * 64 * 2
    assert lib.ebr_block_swiglu_linear_scratch(1, 2, 64, 64, 32) >= 4 * 64 * 64 * 2
    assert lib.ebr_block_swiglu_linear_scratch(1, 3, 64, 64, 32) == -1


def test_the_network_s_options():
    cfg = dict(hidden_size=32, num_heads=2, grid=(2, 2), attn_backend="math", attn_nograd_backend="math")
    with pytest.raises(ValueError, match="norm must be"):
        en.ScalarEnergy(en.EnergyConfig(**cfg, norm="batch"))
    with pytest.raises(ValueError, match="SwiGLU impl"):
        en.ScalarEnergy(en.EnergyConfig(**cfg, mlp_impl="other"))
    with pytest.raises(ValueError, match="LayerNorm impl"):
        layers.LayerNorm(8, impl="other")
    assert not any("layer_norms" in n for n, _ in en.ScalarEnergy(en.EnergyConfig(**cfg)).named_parameters())
    model, dec = en.build(en.EnergyConfig(**cfg, norm="layer"), torch.device("cpu"))
    names = [n for n, _ in model.named_parameters() if "layer_norms" in n]
    assert len(names) == 2 * 2 * 2  # a weight and a bias for each norm of each layer
    x, z = torch.zeros(2, 4, dtype=torch.int64), torch.randn(2, 4, 32)
    params = [*model.parameters(), *dec.parameters()]
    before = [p.detach().clone() for p in params]
    opt = torch.optim.SGD(params, lr=0.1)
    en.train_step(model, dec, x, z, torch.zeros(2, 4, dtype=torch.int64), steps=2, optimizer=opt)
    assert all(p.grad is None for p in params) and any(not torch.equal(p, q) for p, q in zip(params, before))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plain_layer_norm(dtype):
    """Against torch's own: both in fp32, rounded once; some 20 roundings of terms below 8."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 40, generator=g).to(dtype)
    norm = layers.LayerNorm(40)
    with torch.no_grad():
        norm.weight.copy_(torch.randn(40, generator=g)), norm.bias.copy_(torch.randn(40, generator=g))
    want = torch.nn.functional.layer_norm(x.double(), (40,), norm.weight.double(), norm.bias.double(), layers.RMS_NORM_EPS)
    y = norm(x)
    assert y.dtype == dtype
    step = torch.finfo(dtype).eps / 2
    assert bool(((y.double() - want).abs() <= step * want.abs() + 20 * 2.0**-24 * 16).all())


def test_in_order():
    p = torch.randn(4, 6).t()
    assert optim._dense(p) and not optim._dense(torch.randn(4, 6)[:, ::2]) and not optim._dense(torch.randn(3).expand(2, 3))
    assert torch.equal(optim._in_order(p, p), p.t().reshape(-1))
    g = torch.randn(6, 4)
    assert torch.equal(optim._in_order(g, p).view(4, 6).t(), g)
