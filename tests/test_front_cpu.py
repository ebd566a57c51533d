"""Norm, routing and balance loss without a GPU: what is refused before anything is launched, and their cases."""
import random
import re
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))


def test_tensors_on_the_cpu_are_refused():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    x, w = torch.randn(4, 256), torch.ones(256)
    for call in (lambda: rms_norm(x, w), lambda: rms_norm(x.requires_grad_(True), w), lambda: rms_norm_fp8(x.detach(), w), lambda: route(x, 4),
                 lambda: balance_loss(x, torch.zeros(4, 2, dtype=torch.int64)), lambda: rms_norm(x.to("meta"), w.to("meta"))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def _traced():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    w, idx = torch.ones(256), torch.zeros(4, 2, dtype=torch.int64)
    return (lambda x: rms_norm(x, w.to(x.device)), lambda x: rms_norm(x, w.to(x.device), residual=x)[0], lambda x: rms_norm_fp8(x, w.to(x.device))[0][1],
            lambda x: route(x, 4)[1], lambda x: balance_loss(x, idx.to(x.device)))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tracing_is_refused(device):
    """A tracer would keep the example's outputs as constants."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 256, device=device)
    for call in _traced():
        with pytest.raises(RuntimeError, match="tracing"):
            torch.jit.trace(call, (x,))
        with pytest.raises(RuntimeError, match="tracing"):
            make_fx(call)(x)
        if device == "cuda":
            assert call(x).device == x.device


def test_kernels_placed_before_their_inputs_are_complete_read_them_coherently():
    """Launches in stream order overlap the kernel before: the non-coherent path (and what lets the compiler take it) is for
    data that nobody writes while the kernel is there, and such loads may be moved in front of the wait."""
    csrc = Path(__file__).resolve().parent.parent / "csrc"
    for part in ("norm", "route"):
        for f in sorted(csrc.glob(f"{part}/*.cu*")):
            for n, line in enumerate(f.read_text().splitlines(), 1):
                assert not any(s in line for s in ("__ldg(", "ld_global_nc", "ld.global.nc", "__restrict__")), f"{f.name}:{n}"
    # in an exchange: the layout's results in the counts, the counts' results in the dispatch
    for f in ("layout", "dispatch"):
        assert not re.search(r"const \w+\* __restrict__ (is_in_rank|num_tokens_per_expert|item_rank|chunk_base)\b", (csrc / "ep" / f"{f}.cu").read_text())


def test_layer_stored_before_it_had_a_norm_and_a_choice_of_routers():
    """Whole modules that earlier versions pickled: the same attributes but those that came with the options."""
    from gpu_data_transfer_profile_b200.models.moe_layer import MoELayer
    layer = MoELayer(64, 64, 4, 2, None, dtype=torch.float32, device="cpu", expert_backend="torch")
    state = layer.__getstate__()
    new = ("_choice", "_balance", "_plain_choice", "norm_eps", "aux_loss")
    old = {k: dict(v) if k in ("_buffers", "_parameters") else v for k, v in state.items() if k not in new}
    del old["_buffers"]["expert_bias"], old["_parameters"]["norm_weight"]
    again = MoELayer.__new__(MoELayer)
    again.__setstate__(old)
    assert sorted(again.state_dict()) == sorted(layer.state_dict()) and all(getattr(again, n) == getattr(layer, n) for n in new)
    x = torch.randn(5, 64)
    for a, b in zip(again._route(x, None, True), layer._route(x, None, True)):
        assert torch.equal(a, b)
    again._mix = lambda *a: a[0]
    assert again(x) is x and again.aux_loss is None


@pytest.mark.parametrize("kw", [dict(topk_groups=2), dict(topk_groups=0), dict(num_groups=2, topk_groups=3), dict(group_best=0), dict(group_best=3)])
def test_layer_refuses_groups_that_it_could_not_choose(kw):
    from gpu_data_transfer_profile_b200.models.moe_layer import MoELayer
    with pytest.raises(ValueError, match="group"):
        MoELayer(64, 64, 4, 2, None, dtype=torch.float32, device="cpu", expert_backend="torch", **kw)
    for good in (dict(topk_groups=1), dict(group_best=2), dict(num_groups=2, topk_groups=2)):
        MoELayer(64, 64, 4, 2, None, dtype=torch.float32, device="cpu", expert_backend="torch", **good)


def test_unknown_scores_are_refused():
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    for call in (lambda: route(torch.randn(2, 8), 2, score="relu"), lambda: balance_loss(torch.randn(2, 8), torch.zeros(2, 2, dtype=torch.int64), score="")):
        with pytest.raises(ValueError, match="score"):
            call()


def test_cases_fit_what_the_operators_take():
    import importlib.util
    spec = importlib.util.spec_from_file_location("operator_cases", Path(__file__).resolve().parent.parent / "perf" / "operators.py")
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    assert M.own is False
    listed = M.listed()
    most = max(M.work(c)["bytes"] for c in listed)
    assert 4 <= len(listed) <= 12 and most >= 16 * min(M.work(c)["bytes"] for c in listed)
    rng = random.Random(0)
    for c in listed + [M.draw(rng) for _ in range(3000)]:
        assert M.work(c)["bytes"] <= most
        if c["kind"].startswith("norm"):
            assert 1 <= c["hidden"] <= 32768 and (c["kind"] != "norm_fp8" or c["hidden"] % 128 == 0)
        elif c["kind"] != "balance_grad":
            size = c["experts"] // c["groups"]
            assert size * c["groups"] == c["experts"] <= 1024 and c["topk_groups"] <= c["groups"] and c["topk"] <= size * c["topk_groups"] and size >= c["group_best"]
        assert c["kind"].startswith("norm") or c["padded"] < c["tokens"] or c["tokens"] == 0
