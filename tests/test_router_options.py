"""The router's options are looked at where they are given, whichever kernel makes the selection. No GPU needed."""
import pytest
import torch


def test_unknown_names_are_refused_by_route():
    from lazylora_amd.router import route, select_experts
    x, w = torch.randn(3, 8), torch.randn(16, 8)
    for kw in ({"group_score": "mean"}, {"scoring": "tanh"}, {"group_score": None}, {"scoring": "softmax", "group_score": "mean"},
               {"num_groups": 4, "group_score": "mean"}, {"group_score": ["max"]}):
        with pytest.raises(ValueError, match="unknown"):
            route(x, w, top_k=2, **kw)
        with pytest.raises(ValueError, match="unknown"):
            select_experts(x, 2, **kw)


def test_unknown_names_are_refused_at_construction():
    from lazylora_amd.router import KimiK3MoERouter
    for kw in ({"group_score": "mean"}, {"scoring": "tanh"}):
        with pytest.raises(ValueError, match="unknown"):
            KimiK3MoERouter(8, 16, 2, **kw)
    KimiK3MoERouter(8, 16, 2, scoring="softmax", num_groups=4, topk_groups=2, group_score="max")


def test_unknown_names_are_refused_by_the_block():
    from lazylora_amd.int4 import Int4Experts, Int4Weight
    from lazylora_amd.latent_moe import LatentMoEBlock
    w = Int4Weight(torch.zeros(4, 32, 16, dtype=torch.uint8), torch.ones(4, 32, 1, dtype=torch.bfloat16))
    r = lambda *s: torch.zeros(*s)
    for kw in ({"group_score": "mean"}, {"scoring": "tanh"}):
        with pytest.raises(ValueError, match="unknown"):
            LatentMoEBlock(Int4Experts(w, w, w), r(4, 8), None, r(8, 8), r(8, 8), r(8, 8), r(32, 8), r(8, 32), **kw)
