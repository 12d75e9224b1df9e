"""Host-side checks of the token ends (``ebr_amd.tokens``), no GPU: the ops' fakes give the shapes and types that the
kernels write, wrong arguments are refused before anything runs, here and at the C entry points, and the scratch sizes.
Parity of the kernels is in ``tests/test_gpu_tokens.py``."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ebr_amd import _capi, tokens

IDS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("wt,yt", [(torch.float32, torch.bfloat16), (torch.float16, torch.float16), (torch.float64, torch.float64)])
def test_embed_fakes(wt, yt):
    with FakeTensorMode():
        ids, w = torch.empty(2, 5, dtype=torch.int64), torch.empty(7, 12, dtype=wt)
        y = torch.ops.ebr_fused.embed(ids, w, 1.0, yt)
        assert y.shape == (2, 5, 12) and y.dtype == yt
        dw = torch.ops.ebr_fused.embed_bwd(ids, y, 7, 1.0, wt)
        assert dw.shape == w.shape and dw.dtype == wt


@pytest.mark.parametrize("reduction,shape", [(0, (2, 5)), (1, ()), (2, ())])
def test_distill_fakes(reduction, shape):
    with FakeTensorMode():
        x = torch.empty(2, 5, 17, dtype=torch.bfloat16)
        t, ids = torch.empty(2, 5, 4), torch.empty(2, 5, 4, dtype=torch.int32)
        loss, stats, scale = torch.ops.ebr_fused.distill(x, t, ids, 1.0, reduction)
        assert loss.shape == shape and loss.dtype == torch.float32 and stats.shape == (10, 4)
        dx = torch.ops.ebr_fused.distill_bwd(x, t, ids, stats, scale, loss, 1.0)
        assert dx.shape == x.shape and dx.dtype == x.dtype


def _embed(ids=IDS, w=None, **kw):
    return tokens.embedding(ids, torch.zeros(4, 8) if w is None else w, **kw)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: _embed(ids=IDS.float())),
    (TypeError, lambda: _embed(ids=IDS.to(torch.int16))),
    (TypeError, lambda: _embed(w=torch.zeros(4, 8, dtype=torch.int32))),
    (TypeError, lambda: _embed(w=torch.zeros(4, 8, dtype=torch.bfloat16), dtype=torch.float32)),
    (TypeError, lambda: _embed(dtype=torch.float64)),
    (ValueError, lambda: _embed(w=torch.zeros(4))),
    (ValueError, lambda: _embed(w=torch.zeros(4, 8, device="meta"))),
    (ValueError, lambda: _embed(scale=float("inf"))),
    (NotImplementedError, lambda: _embed()),  # no kernel off the GPU
])  # fmt: skip
def test_embedding_refuses(error, call):
    with pytest.raises(error):
        call()


def _distill(x=(3, 9), t=(3, 2), ids=None, xt=torch.float32, it=torch.int64, **kw):
    ids = t if ids is None else ids
    return tokens.distill_loss(torch.zeros(x, dtype=xt), torch.zeros(t), torch.zeros(ids, dtype=it), **kw)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: _distill(it=torch.float32)),
    (TypeError, lambda: _distill(xt=torch.int64)),
    (ValueError, lambda: _distill(t=(2, 2))),
    (ValueError, lambda: _distill(ids=(3, 1))),
    (ValueError, lambda: _distill(t=(3, 0))),
    (ValueError, lambda: _distill(t=(3, 1025))),
    (ValueError, lambda: _distill(x=(3, 0))),
    (ValueError, lambda: _distill(temperature=0.0)),
    (ValueError, lambda: _distill(temperature=float("nan"))),
    (ValueError, lambda: _distill(reduction="batchmean")),
    (NotImplementedError, lambda: tokens.distill_loss(torch.zeros(3, 9), torch.zeros(3, 2, requires_grad=True), torch.zeros(3, 2, dtype=torch.int64))),
    (NotImplementedError, lambda: _distill()),  # no kernel off the GPU
])  # fmt: skip
def test_distill_refuses(error, call):
    with pytest.raises(error):
        call()


P = 0x100000  # a placeholder that no refused call reads


@pytest.mark.parametrize("kw,code", [
    (dict(wt=4), 1), (dict(yt=0), 1), (dict(wt=3), 1), (dict(V=0), 2), (dict(N=-1), 2), (dict(N=2**31 - 1), 2),
    (dict(V=2**31), 2), (dict(C=0), 2), (dict(C=2**18), 2), (dict(ids=0), 4), (dict(w=0), 4), (dict(y=0), 4),
])  # fmt: skip
def test_embed_entry_refuses(kw, code):
    a = dict(wt=1, yt=1, N=5, V=7, C=8, ids=P, w=P, y=P) | kw
    lib = _capi.load()
    assert lib.ebr_block_embed(a["wt"], a["yt"], 1, a["N"], a["V"], a["C"], 1.0, a["ids"], a["w"], a["y"], None) == code
    if code != 4:
        assert lib.ebr_block_embed_bwd(a["wt"], a["yt"], 1, a["N"], a["V"], a["C"], 1.0, P, P, P, P, None) == code


def test_embed_bwd_entry_refuses_pointers():
    call = _capi.load().ebr_block_embed_bwd
    assert call(1, 1, 1, 5, 7, 8, 1.0, P, P, 0, P, None) == 4
    assert call(1, 1, 1, 5, 7, 8, 1.0, P, P, P, 0, None) == 5
    assert call(1, 1, 1, 5, 7, 8, 1.0, P, P, P, P + 8, None) == 3


@pytest.mark.parametrize("kw,code", [
    (dict(dt=4), 1), (dict(tt=7), 1), (dict(N=-1), 2), (dict(V=0), 2), (dict(K=0), 2), (dict(K=1025), 2), (dict(row=8), 2),
    (dict(T=0.0), 2), (dict(T=float("nan")), 2), (dict(reduction=3), 2), (dict(N=2**25, V=4000, row=4000), 2),
    (dict(x=0), 4), (dict(loss=0), 4), (dict(scale=0), 4), (dict(scratch=0), 5), (dict(stats=P + 4), 3),
])  # fmt: skip
def test_distill_entry_refuses(kw, code):
    a = dict(dt=1, tt=0, N=5, V=9, K=2, row=9, T=1.0, reduction=2, x=P, loss=P, scale=P, scratch=P, stats=P) | kw
    lib = _capi.load()
    rc = lib.ebr_block_distill(a["dt"], a["tt"], 1, a["N"], a["V"], a["K"], a["row"], ctypes.c_double(a["T"]), a["reduction"],
                               a["x"], P, P, a["stats"], a["loss"], a["scale"], a["scratch"], None)
    assert rc == code
    if not kw.keys() & {"reduction", "loss", "scale", "scratch"}:
        assert lib.ebr_block_distill_bwd(a["dt"], a["tt"], 1, a["N"], a["V"], a["K"], a["row"], ctypes.c_double(a["T"]), a["x"],
                                         P, P, a["stats"], P, P, 0, P, None) == code


def test_scratch_sizes():
    lib = _capi.load()
    assert lib.ebr_block_embed_bwd_scratch(0, 0, 11, 512) >= 0
    assert lib.ebr_block_embed_bwd_scratch(0, 5000, 11, 512) >= 4 * 5000 * 4
    assert lib.ebr_block_embed_bwd_scratch(0, 5000, 0, 512) == -1
    assert lib.ebr_block_distill_scratch(1, 100, 11, 4) > 0
    assert lib.ebr_block_distill_scratch(1, 100, 11, 0) == -1


@pytest.mark.parametrize("temperature", [9e-16, 1.1e15, float("inf"), -1.0])
def test_distill_refuses_temperatures_whose_square_leaves_fp32(temperature):
    with pytest.raises(ValueError, match="temperature"):
        _distill(temperature=temperature)


def test_the_guide_s_loss_calls_the_entries_with_their_arguments():
    """The launcher-level loss of the integration guide compiles, and passes as many arguments as the entry points take (its
    GPU test runs it)."""
    import ast
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    (src,) = (b for b in re.findall(r"```python\n(.*?)```", text, re.S) if b.startswith("# training/distill_hip.py"))
    called = {n.func.attr: len(n.args) for n in ast.walk(ast.parse(src))
              if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and n.func.attr.startswith("ebr_block")}
    assert called == {n: len(_capi.SIGNATURES[n][1]) for n in ("ebr_block_distill_scratch", "ebr_block_distill", "ebr_block_distill_bwd")}
