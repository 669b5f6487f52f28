"""The latent MoE block with group-limited softmax routing and 4-bit experts, as it decodes, against 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def block(act="situ", dt=torch.bfloat16, **kw):
    from lazylora_amd.latent_moe import LatentMoEBlock
    from test_gpu_int4 import gen_of, layer
    gen = gen_of(21)
    E, H, Dl, F, Ds = 16, 192, 128, 64, 96
    ex = layer(gen, E, Dl, F, 64, True, dt)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen) / s[-1] ** 0.5
    w = dict(gate_weight=4 * r(E, H), gate_bias=0.02 * torch.randn(E, device="cuda", generator=gen), shared_w1=r(Ds, H),
             shared_w3=r(Ds, H), shared_w2=r(H, Ds), latent_down=r(Dl, H), latent_up=r(H, Dl),
             latent_norm=1 + 0.1 * torch.randn(Dl, device="cuda", generator=gen))
    return LatentMoEBlock(ex, **w, top_k=4, routed_scaling_factor=2.0, act=act, scoring="softmax", num_groups=4,
                          topk_groups=2, group_score="max", **kw), w, ex, gen


def block64(w, ex, h, act):
    """The block's formulas in 64 bits, its choice included."""
    from test_gpu_int4 import routed64
    from test_gpu_select import oracle_select
    n = {k: v.double().cpu().numpy() for k, v in w.items()}
    h = h.double().cpu().numpy()
    glu = lambda g, u: 4 * np.tanh(g / 4) / (1 + np.exp(-g)) * 25 * np.tanh(u / 25) if act == "situ" else g / (1 + np.exp(-g)) * u
    idx, tw = oracle_select(h @ n["gate_weight"].T, 4, n["gate_bias"], "softmax", 4, 2, "max", True, 2.0)
    latent = torch.from_numpy(h @ n["latent_down"].T)
    routed, _ = routed64(latent, torch.from_numpy(idx), torch.from_numpy(tw), ex, act, None)
    routed = routed / np.sqrt((routed ** 2).mean(1, keepdims=True) + 1e-5) * n["latent_norm"]
    return glu(h @ n["shared_w1"].T, h @ n["shared_w3"].T) @ n["shared_w2"].T + routed @ n["latent_up"].T, idx, tw


@pytest.mark.parametrize("N", [1, 3, 40, 200])
@pytest.mark.parametrize("act", ["situ", "swiglu"])
def test_block(N, act):
    b, w, ex, gen = block(act)
    h = torch.randn(N, 192, device="cuda", generator=gen)
    with torch.no_grad():
        out, idx, tw = b(h)
    want, want_i, want_w = block64(w, ex, h, act)
    np.testing.assert_array_equal(idx.cpu().numpy(), want_i)
    # the logits are fp32 products here: the weights follow their rounding
    np.testing.assert_allclose(tw.cpu().numpy(), want_w, rtol=1e-4)
    # bfloat16 in front of the experts, between their products and behind them: three half steps, each averaged over
    # the terms of a sum, on a part of the result
    err = np.linalg.norm(out.double().cpu().numpy() - want) / np.linalg.norm(want)
    assert err < 3 * 2.0 ** -9
    with torch.no_grad():
        again = b(h, cached=torch.zeros(N, 128, device="cuda"))[0]
    assert not torch.equal(again, out)


def test_gradients_and_adapters_are_refused():
    class Adapter:
        lora_A, lora_B, scaling, dropout_rate = torch.zeros(4, 128), torch.zeros(64, 4), 1.0, 0.0

    class Bundle:
        gate_lora = up_lora = down_lora = Adapter()

    b, _, _, gen = block()
    h = torch.randn(3, 192, device="cuda", generator=gen, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no backward"):
        b(h)
    with pytest.raises(ValueError, match="adapters"):
        block(lora=Bundle())


def test_grouped_choice_trains():
    """The same routing over MXFP4 experts, with gradients through the weights."""
    from lazylora_amd.experts import ExpertLayer
    from lazylora_amd.latent_moe import LatentMoEBlock
    import oracle
    rng = np.random.default_rng(3)
    e = oracle.random_experts(rng, 8, 128, 64, 119, 123)
    ex = ExpertLayer(*[torch.from_numpy(a).cuda() for a in (e.w1p, e.w1s, e.w3p, e.w3s, e.w2p, e.w2s)])
    r = lambda *s: torch.randn(*s, device="cuda") / s[-1] ** 0.5
    b = LatentMoEBlock(ex, 4 * r(8, 64), torch.zeros(8), r(32, 64), r(32, 64), r(64, 32), r(128, 64), r(64, 128), top_k=2,
                       scoring="softmax", num_groups=4, topk_groups=2)
    x = torch.randn(9, 64, device="cuda", requires_grad=True)
    out, idx, w = b(x)
    # the gradient along a direction, through the weights alone, against the block's forward on both sides
    c = torch.randn_like(w)
    g = torch.autograd.grad((w * c).sum(), x, retain_graph=True)[0]
    v = torch.randn_like(x)
    f = lambda y: b(y)[1:]
    step = 2.0 ** -9
    (i0, w0), (i1, w1) = f((x + step * v).detach()), f((x - step * v).detach())
    same = (i0 == idx).all(1) & (i1 == idx).all(1)  # rows whose choice the step does not change
    assert same.sum() >= 4
    diff = ((w0 - w1) * c).sum(1) / (2 * step)
    slope = (g * v).sum(1)
    assert (diff - slope)[same].abs().max() < 0.05 * (1 + slope.abs().max())
    out.sum().backward()
    assert torch.isfinite(x.grad).all()
