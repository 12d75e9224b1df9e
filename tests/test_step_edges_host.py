"""Host-side checks, no GPU, of what the layer norm, the gated projection and the optimizer's step do next to the borders of their
plans and arguments. Parity of the kernels there is in ``tests/test_gpu_step_edges.py``."""

import ctypes
import os
import random
import subprocess
from pathlib import Path

import pytest
import torch

from ebr_amd import _capi, block, layers, optim

PLAN = r"""
#include "glu_plan.hpp"
#include <cstdio>
using namespace ebr_glu;
int main() {
    long seen = 0, wrong = 0;
    const int64_t widths[] = {1, 8, 24, 64, 1000, 5632, 6400, 6408, 12736, 12744, 14336, 25600, 25608, 28672, (1 << 19) - 8};
    for (int dtype = 0; dtype < 4; ++dtype)
        for (int order = 1; order <= 2; ++order)
            for (const int64_t C : {8, 72, 4096, (1 << 20) - 8})
                for (const int64_t I : widths)
                    for (int64_t N = 1; N <= 130; ++N) {
                        const bool rest = with_rest(dtype, N);
                        if (rest != (N <= 64 && (dtype == EBR_DTYPE_BF16 || dtype == EBR_DTYPE_F16))) ++wrong;
                        if (is_few(dtype, N, C)) continue;
                        const int tile = gates_cut(dtype, order, N, C, I).tile;
                        if (tile != 64 && tile != 128 && tile != 256) ++wrong;
                        if (rest && staged(size_of(dtype), tile)) {
                            ++wrong;
                            std::printf("%d %d %lld %lld %d\n", dtype, order, (long long)N, (long long)I, tile);
                        }
                        if (!rest) seen += staged(size_of(dtype), tile);
                    }
    return wrong ? 1 : seen ? 0 : 2;
}
"""


def _host_program(tmp_path, source):
    """A program of plain C++ beside the library's sources, run; its exit status and output."""
    csrc = Path(block.__file__).parent / "csrc"
    (tmp_path / "t.cpp").write_text(source)
    cc = [os.environ.get("CXX", "g++"), "-std=c++17", "-O1", f"-I{csrc}", str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")]
    subprocess.run(cc, check=True, capture_output=True)
    run = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    return run.returncode, run.stdout


def test_gated_projection_of_few_rows_writes_what_its_products_read(tmp_path):
    """What [dg|du] lacks of its values before rounding enters the derivatives' products of up to 64 rows in 16 bits: no tile
    that leaves it unwritten stands before them."""
    rc, out = _host_program(tmp_path, PLAN)
    assert rc == 0, out


def _saved(cls, steps=1, **kw):
    p = torch.nn.Parameter(torch.ones(6))
    opt = cls([p], **kw)
    for _ in range(steps):
        p.grad = torch.ones(6)
        opt.step()
    return opt.state_dict()


@pytest.mark.parametrize("steps", [0, 1])
@pytest.mark.parametrize("cls,kw", [
    (torch.optim.AdamW, dict(maximize=True)), (torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.Adam, dict(weight_decay=0.1)),
    (torch.optim.RAdam, {}), (torch.optim.NAdam, {}), (torch.optim.Adamax, {}), (torch.optim.SGD, dict(lr=0.1)),
])  # fmt: skip
def test_states_of_other_steps_are_refused(cls, kw, steps):
    ours = optim.AdamW([torch.nn.Parameter(torch.zeros(6))], lr=3e-4)
    with pytest.raises(ValueError, match="optim:"):
        ours.load_state_dict(_saved(cls, steps, **kw))
    assert ours.param_groups[0]["lr"] == 3e-4 and len(ours.state) == 0


@pytest.mark.parametrize("cls,kw", [(torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.Adam, {}), (torch.optim.AdamW, dict(foreach=False))])
def test_states_of_the_same_steps_are_taken(cls, kw):
    p = torch.nn.Parameter(torch.zeros(6))
    ours, saved = optim.AdamW([p]), _saved(cls, 2, **kw)
    for again in (False, True):  # theirs, then ours as it is after that
        ours.load_state_dict(ours.state_dict() if again else saved)
        assert int(ours.state[p]["step"]) == 2 and torch.equal(ours.state[p]["exp_avg_sq"], saved["state"][0]["exp_avg_sq"])
        assert ours.param_groups[0]["weight_decay"] == saved["param_groups"][0]["weight_decay"]


def test_groups_of_other_steps_are_refused():
    p, q = (torch.nn.Parameter(torch.zeros(6)) for _ in range(2))
    for kw in (dict(maximize=True), dict(amsgrad=True), dict(decoupled_weight_decay=False)):
        with pytest.raises(ValueError, match="AdamW"):
            optim.AdamW([dict(params=[p], **kw)])
        ours = optim.AdamW([p])
        with pytest.raises(ValueError, match="AdamW"):
            ours.add_param_group(dict(params=[q], **kw))
        assert len(ours.param_groups) == 1
    assert len(optim.AdamW([dict(params=[p], maximize=False), dict(params=[q], lr=1e-4)]).param_groups) == 2


@pytest.mark.parametrize("error,name,value", [
    (ValueError, "exp_avg", torch.zeros(3, 2, dtype=torch.uint8).view(optim.STATE8)), (ValueError, "exp_avg_root_scale", torch.zeros(2)), (ValueError, "step", torch.zeros(2)),
    (TypeError, "exp_avg_root", torch.zeros(2, 3)),
])  # fmt: skip
def test_a_refused_state_leaves_the_optimizer_as_it_was(error, name, value):
    ps = [torch.nn.Parameter(torch.zeros(2, 3)) for _ in range(2)]
    ours, other = (optim.AdamW(ps, lr=lr, state_bits=8) for lr in (3e-4, 1e-3))
    for opt, t in ((ours, 5), (other, 7)):
        opt.init_state()
        for p in ps:
            opt.state[p]["step"].fill_(t)
    saved = other.state_dict()
    saved["state"][1][name] = value
    with pytest.raises(error, match="optim:"):
        ours.load_state_dict(saved)
    assert ours.param_groups[0]["lr"] == 3e-4 and [int(ours.state[p]["step"]) for p in ps] == [5, 5]
    saved["state"][1] = saved["state"][0]
    ours.load_state_dict(saved)
    assert ours.param_groups[0]["lr"] == 1e-3 and [int(ours.state[p]["step"]) for p in ps] == [7, 7]


@pytest.mark.parametrize("dtype", [0, 1, 2, 3])
def test_sizes_that_the_gated_projection_takes(dtype):
    """What the header says is always taken is, and what would be a launch of 2^32 threads and more is not."""
    lib, rng = _capi.load(), random.Random(dtype)

    def up(n):
        return (n + 255) // 256 * 256

    seen = 0
    for _ in range(20000):
        N, C, I = (int(2 ** rng.uniform(0, bits)) for bits in (30, 20, 19))
        C, I = min(C, (1 << 20) - 8), min(I, (1 << 19) - 8)
        if N < 1 << 30 and max(up(N) * up(C), up(N) * up(I), 2 * up(C) * up(I)) < 1 << 36:
            seen += 1
            assert all(lib.ebr_block_swiglu_linear_scratch(dtype, order, N, C, I) >= 0 for order in range(3)), (N, C, I)
    assert seen > 1000
    for N, C, I in ((2_000_000, 2048, 11008), ((1 << 29) + 64, 8, 8), (33, 16384, 1 << 16)):
        assert all(lib.ebr_block_swiglu_linear_scratch(dtype, order, N, C, I) >= 0 for order in range(3)), (N, C, I)
    for N, C, I in (((1 << 31) - 1, 8, 1 << 18), ((1 << 31) - 1, 8, 512), ((1 << 30) + 1, (1 << 20) - 8, (1 << 19) - 8)):
        assert all(lib.ebr_block_swiglu_linear_scratch(dtype, order, N, C, I) == -1 for order in range(3)), (N, C, I)


def test_more_tensors_than_a_step_takes():
    lib = _capi.load()
    assert lib.ebr_block_adamw_scratch((1 << 24) - 1) > 0
    for count in (1 << 24, (1 << 31) - 1, 1 << 40):
        assert lib.ebr_block_adamw_scratch(count) == -1
        assert lib.ebr_block_adamw(0, 0, 32, count, None, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, None, 0.0, None, None) == 2


def _step(params, grads, lr=1e-3, **kw):
    zeros = [[torch.zeros(p.shape) for p in params] for _ in range(2)]
    steps = [torch.zeros((), dtype=torch.int64) for _ in params]
    return optim.adamw_(params, grads, *zeros, steps, lr=lr, **kw)


def test_a_step_that_writes_to_what_it_reads():
    """A gradient in another's parameter, or a place further on in its own, would be read before or after it is written, as it comes."""
    both = torch.zeros(12)
    p, q, r = both[:4], both[4:8], torch.zeros(4)
    for params, grads in (((p, q), (r, p)), ((p, q), (both[2:6], r)), ((p, q), (both[1:5], r)), ((p, q), (r, both[7:11]))):
        with pytest.raises(ValueError, match="writes to a gradient"):
            _step(params, grads)
    with pytest.raises(ValueError, match="its lr"):
        _step((p, q), (r, r), lr=both[5])
    for grads in ((p, r), (r, both[8:]), (both.view(4, 3)[:, 0], r)):  # its own, one beside, and one that is copied: no kernel off the GPU
        with pytest.raises(NotImplementedError):
            _step((p, q), grads)


@pytest.mark.parametrize("kw", [dict(g=0x101000), dict(g=0x100004), dict(lr=0x100018), dict(norm=0x102010), dict(scratch=0x101FF0)])
def test_adamw_entry_refuses_to_write_to_what_it_reads(kw):
    at = 0x100000
    rows = [(at + 4096 * k, kw.get("g", 0x200000), at + 4096 * (2 + k), at + 4096 * (4 + k), 0, 0, at + 4096 * 6 + 8 * k, 1000)
            for k in range(2)]
    table = (_capi.OptimTensor * 2)(*rows)
    rc = _capi.load().ebr_block_adamw(0, 0, 32, 2, ctypes.addressof(table), 1e-3, kw.get("lr"), 0.9, 0.99, 1e-8, 0.0, kw.get("norm"),
                                      1.0, kw.get("scratch", 0x300000), None)
    assert rc == 2


CUTS = r"""
#include "glu_plan.hpp"
#include <cmath>
#include <cstdio>
#include <random>
#include <set>
#include <string>
using namespace ebr_glu;
int main() {
    std::mt19937_64 rng(1);
    const auto size = [&](double bits) { return (int64_t)std::exp2(std::uniform_real_distribution<double>(0, bits)(rng)); };
    std::set<std::string> seen;
    for (int k = 0; k < 3000000; ++k) {
        const int dtype = k % 4, order = 1 + k / 4 % 2;
        const int64_t N = size(22), C = padded(dtype, size(14)), I = padded(dtype, size(15));
        const int each = with_rest(dtype, N) ? 2 : 1, bytes = size_of(dtype);
        const Cut in = input_cut(dtype, N, C, I, each), w = weight_cut(dtype, N, C, I, order * each);
        const auto say = [&](const char* what, int tile) { seen.insert(std::to_string(bytes) + what + std::to_string(tile)); };
        for (int o = 0; o < 3; ++o)
            if (!is_few(dtype, N, C)) say(o == 0 ? " forward " : o == 1 ? " first " : " second ", gates_cut(dtype, o, N, C, I).tile);
        if (in.whole) say(" dx ", in.tile);
        if (in.splits > 1) say(" dx split ", in.tile);
        if (w.whole) say(" dw ", w.tile);
        if (w.splits > 1) say(" dw split ", w.tile);
    }
    for (const std::string& s : seen) std::puts(s.c_str());
}
"""


def test_the_gated_projection_s_kernels_are_all_taken(tmp_path):
    """Every tile of every product is some size's, and no size takes another."""
    rc, out = _host_program(tmp_path, CUTS)
    want = {"8 forward 64", "8 first 64", "8 second 64", "8 dx 64", "8 dw 64", "4 dx split 64", "2 dx split 64"}
    for bytes, tiles in ((4, (64, 128)), (2, (64, 128, 256))):
        want |= {f"{bytes} {p} {t}" for t in tiles for p in ("forward", "first", "second", "dx", "dw", "dw split")}
    assert rc == 0 and set(out.splitlines()) == want


def test_hooks_of_the_projection_run(monkeypatch):
    """``impl="projected"`` takes the projection's weight alone, but where the module has hooks it is called."""

    def plain(gu):
        gate, up = gu.chunk(2, -1)
        return torch.nn.functional.silu(gate) * up

    monkeypatch.setattr(block, "swiglu", plain)
    monkeypatch.setattr(block, "swiglu_linear", lambda x, w: plain(x @ w.t()))
    net, x, seen = layers.SwiGLU(8, 2.0, impl="projected"), torch.randn(3, 8), []
    want = net(x)
    at = net.gate_up_proj
    for put in (lambda: at.register_forward_hook(lambda m, i, o: seen.append("after")),
                lambda: at.register_forward_pre_hook(lambda m, i: seen.append("before")),
                lambda: at.register_full_backward_hook(lambda m, i, o: seen.append("backward")),
                lambda: at.register_full_backward_pre_hook(lambda m, o: seen.append("before backward"))):
        handle = put()
        y = net(x.clone().requires_grad_(True))
        y.sum().backward()
        assert torch.allclose(y, want)
        handle.remove()
        assert torch.allclose(net(x), want)
    assert seen == ["after", "before", "backward", "before backward"]


def test_hooks_of_a_load_see_and_change_what_is_loaded():
    """What a hook gives in a saved state's place is what is loaded, once; a hook that follows finds the moments as they are kept."""
    p = torch.nn.Parameter(torch.zeros(6, dtype=torch.bfloat16))
    ours, saved, seen = optim.AdamW([p]), _saved(torch.optim.AdamW, 2), []

    def wider(opt, state_dict):
        state = {k: dict(st, exp_avg=st["exp_avg"] + 2.0**-20) for k, st in state_dict["state"].items()}
        seen.append("before")
        return dict(state_dict, state=state)

    ours.register_load_state_dict_pre_hook(wider)
    ours.register_load_state_dict_post_hook(lambda opt: seen.append(opt.state[p]["exp_avg"].clone()))
    for _ in range(2):
        ours.load_state_dict(saved)
    want = saved["state"][0]["exp_avg"] + 2.0**-20
    assert seen[0] == seen[2] == "before" and len(seen) == 4
    assert torch.equal(seen[1], want) and torch.equal(seen[3], want) and torch.equal(ours.state[p]["exp_avg"], want)
