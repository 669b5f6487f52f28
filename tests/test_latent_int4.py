"""The latent MoE block over 4-bit experts, on the host: what it refuses around `cached` and adapters. No GPU needed
(the router is replaced, and no routed product is launched)."""
import pytest
import torch

E, H, Dl, F, Ds, k = 4, 32, 64, 32, 16, 2


@pytest.fixture
def block(monkeypatch):
    from lazylora_amd import latent_moe
    from lazylora_amd.int4 import Int4Experts, Int4Weight
    w = lambda R, K: Int4Weight(torch.zeros(E, R, K // 2, dtype=torch.uint8), torch.ones(E, R, K // 32, dtype=torch.bfloat16))

    def route(x, weight, bias, top_k, *_):
        v, idx = torch.sigmoid(x @ weight.T).topk(top_k)
        return idx, v

    monkeypatch.setattr(latent_moe, "route", route)
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(sum(s)))
    return latent_moe.LatentMoEBlock(Int4Experts(w(F, Dl), w(F, Dl), w(Dl, F)), r(E, H), None, r(Ds, H), r(Ds, H), r(H, Ds),
                                     r(Dl, H), r(H, Dl), top_k=k)


def test_cached_sum_does_not_drop_a_gradient(block):
    """The routed sum of an earlier call is no function of this call's input: where a gradient is recorded there is
    nothing that could carry it, through the latent projection or through the router's weights."""
    x, cached = torch.randn(3, H), torch.randn(3, Dl)
    with pytest.raises(NotImplementedError, match="no backward"):
        block(x.clone().requires_grad_(True), cached=cached)
    block.gate_weight.requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no backward"):
        block(x, cached=cached)
    block.gate_weight.requires_grad_(False)
    block.latent_down.requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no backward"):
        block(x, cached=cached)


def test_cached_sum_without_a_gradient(block):
    x, cached = torch.randn(3, H), torch.randn(3, Dl)
    want = block._shared(x, None) + cached @ block.latent_up.T
    torch.testing.assert_close(block(x, cached=cached)[0], want)
    with torch.no_grad():
        torch.testing.assert_close(block(x.clone().requires_grad_(True), cached=cached)[0], want)
    # in any floating type, as with an ExpertLayer
    low = cached.bfloat16()
    torch.testing.assert_close(block(x, cached=low)[0], block._shared(x, None) + low.float() @ block.latent_up.T)


def test_routed_adapters_are_refused_whenever_they_come(block):
    """`lora` may be set on a block that is there already: routed adapters are not left out of the sum in silence."""
    class Adapter:
        lora_A, lora_B, scaling, dropout_rate = torch.zeros(4, Dl), torch.zeros(F, 4), 1.0, 0.0

    class Bundle:
        gate_lora = up_lora = down_lora = Adapter()

    block.lora = Bundle()
    with torch.no_grad(), pytest.raises(ValueError, match="adapters"):
        block(torch.randn(3, H))
    with torch.no_grad(), pytest.raises(ValueError, match="adapters"):
        block(torch.randn(3, H), cached=torch.randn(3, Dl))
