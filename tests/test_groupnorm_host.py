"""Host-side checks of the group norm (``ebr_amd.block.group_norm``) and of the options that reach the new operators, no
GPU: fakes, refusals here and at the C entry points, scratch sizes, and the block's eager group norm."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ebr_amd import _capi, block, layers
from ebr_amd import energy as en


@pytest.mark.parametrize("dtype,acc", [(torch.bfloat16, torch.float32), (torch.float64, torch.float64)])
def test_fakes(dtype, acc):
    with FakeTensorMode():
        x, w = torch.empty(3, 4, 5, 24, dtype=dtype), torch.empty(24)
        y, stats = torch.ops.ebr_fused.block_groupnorm(x, w, None, 4, 1e-5, 1)
        assert y.shape == x.shape and y.dtype == dtype and stats.shape == (3, 4, 2) and stats.dtype == acc
        dx, dw, db = torch.ops.ebr_fused.block_groupnorm_bwd(x, w, None, stats, y, 4, 1, True)
        assert dx.shape == x.shape and dw.shape == db.shape == (24,) and dw.dtype == acc
        out = torch.ops.ebr_fused.block_groupnorm_bwd2(x, w, None, stats, y, dx, None, None, 4, 1, False)
        assert [t.shape for t in out] == [x.shape, x.shape, (0,), (0,)]


X = torch.zeros(2, 5, 12)


@pytest.mark.parametrize("error,call", [
    (ValueError, lambda: block.group_norm(X[0, 0], 4)),
    (ValueError, lambda: block.group_norm(X, 5)),
    (ValueError, lambda: block.group_norm(X, 0)),
    (ValueError, lambda: block.group_norm(X, 4, torch.zeros(11))),
    (ValueError, lambda: block.group_norm(X, 4, None, torch.zeros(12, device="meta"))),
    (ValueError, lambda: block.group_norm(X, 4, activation="tanh")),
    (ValueError, lambda: block.group_norm(X, 4, eps=-1.0)),
    (ValueError, lambda: block.group_norm(X, 4, eps=float("nan"))),
    (TypeError, lambda: block.group_norm(X.int(), 4)),
    (NotImplementedError, lambda: block.group_norm(X, 4)),  # no kernel off the GPU
])  # fmt: skip
def test_group_norm_refuses(error, call):
    with pytest.raises(error):
        call()


P = 0x100000  # a placeholder that no refused call reads


@pytest.mark.parametrize("kw,code", [
    (dict(dt=4), 1), (dict(act=2), 2), (dict(B=0), 2), (dict(L=0), 2), (dict(C=0), 2), (dict(G=0), 2), (dict(G=5), 2),
    (dict(C=2**21, G=1), 2), (dict(B=2**30, L=2**30), 2), (dict(B=2**25, L=1), 2), (dict(B=2**25, L=1, C=9, G=1), 2), (dict(x=0), 4), (dict(stats=0), 4), (dict(y=0), 4),
    (dict(scratch=0), 5), (dict(scratch=P + 4), 3),
])  # fmt: skip
def test_entries_refuse(kw, code):
    a = dict(dt=1, act=1, B=2, L=9, C=24, G=4, x=P, stats=P, y=P, scratch=P) | kw
    lib = _capi.load()
    head = (a["dt"], a["act"], a["B"], a["L"], a["C"], a["G"])
    assert lib.ebr_block_groupnorm(*head, 1e-5, a["x"], P, P, a["y"], a["stats"], a["scratch"], None) == code
    assert lib.ebr_block_groupnorm_bwd(*head, a["x"], P, P, a["stats"], P, a["y"], P, P, a["scratch"], None) == code
    assert lib.ebr_block_groupnorm_bwd2(*head, a["x"], P, P, a["stats"], P, P, P, P, a["y"], P, P, P, a["scratch"], None) == code


def test_scratch_sizes():
    lib = _capi.load()
    sizes = [lib.ebr_block_groupnorm_scratch(1, order, 2, 81, 512, 32) for order in (0, 1, 2)]
    assert all(n >= 0 for n in sizes)
    assert lib.ebr_block_groupnorm_scratch(1, 3, 2, 81, 512, 32) == -1
    assert lib.ebr_block_groupnorm_scratch(1, 0, 2, 81, 512, 31) == -1


@pytest.mark.parametrize("B,L,C", [(2**30, 2**34, 1), (2**26, 2**38, 16), (2**25, 2**39, 3), (2**30, 2**33, 8)])
def test_scratch_refuses_sizes_whose_product_passes_64_bits(B, L, C):
    assert [_capi.load().ebr_block_groupnorm_scratch(1, order, B, L, C, 1) for order in (0, 1, 2)] == [-1, -1, -1]


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("dtype,B,L,C,G,fits", [
    (1, 2**25, 1, 8, 1, False), (1, 2**24, 1, 64, 8, False), (1, 2**24 - 1, 1, 64, 8, True),  # a workgroup for each sample
    (0, 2**23, 2, 5, 5, False), (0, 2**21, 2, 5, 5, True),                                    # one for each group
    # several for each sample: 5 of vectors of 2 (21 million in all), 3 of single elements (12.6), which tensors off alignment take
    (3, 2**22, 1, 130, 1, True), (3, 2**24, 1, 130, 1, False), (3, 2**21, 1, 130, 1, True),
])  # fmt: skip
def test_scratch_refuses_what_a_launch_does_not_hold(dtype, B, L, C, G, fits, order):
    assert (_capi.load().ebr_block_groupnorm_scratch(dtype, order, B, L, C, G) >= 0) == fits


def test_eager_group_norm_is_torch_s():
    x = torch.randn(3, 6, 7, 24, generator=torch.Generator().manual_seed(0), dtype=torch.float32)
    ref = torch.nn.functional.group_norm(x.double().permute(0, 3, 1, 2), 4, eps=1e-5).permute(0, 2, 3, 1)
    # mean and variance over 252 values in 32 bits: a few hundred roundings of 2^-24 at most
    assert float((layers.group_norm(x, 4, 1e-5) - ref).abs().max()) <= 300 * 2.0**-24 * float(ref.abs().max())


def test_options_are_checked_and_off_by_default():
    cfg = en.EnergyConfig()
    assert cfg.embed_impl == "eager" and cfg.norm == "rms"
    for bad in (dict(embed_impl="fast"), dict(norm="batch"), dict(norm="group", norm_groups=7), dict(norm="group", norm_groups=0)):
        with pytest.raises(ValueError):
            en.build(en.EnergyConfig(hidden_size=32, num_heads=2, grid=(3, 3), **bad), torch.device("cpu"))


def test_a_block_with_group_norms_trains_off_the_gpu():
    cfg = en.EnergyConfig(hidden_size=32, num_heads=2, grid=(3, 3), vocab_size=5, norm="group", norm_groups=4,
                          attn_backend="math", attn_nograd_backend="math")
    model, dec = en.build(cfg, torch.device("cpu"), seed=1)
    g = torch.Generator().manual_seed(2)
    x, targets = (torch.randint(0, 5, (2, 9), generator=g) for _ in range(2))
    loss = en.train_step(model, dec, x, torch.randn(2, 9, 32, generator=g), targets, steps=2)
    assert bool(torch.isfinite(loss)) and all(bool(torch.isfinite(p.grad).all()) for p in model.parameters() if p.grad is not None)
    values, ids = en.teacher_logits(model, dec, x, torch.randn(2, 9, 32, generator=g), 3, steps=2)
    assert values.shape == ids.shape == (2, 9, 3) and bool((values[..., 0] >= values[..., 2]).all())
