"""The latent MoE block with its dense half in the kernels (dense="native"): shared expert with adapters
and their dropout, norm of the routed sum, as one training step, against the block in float64.

Bars: a rounding to bfloat16 moves a tensor by at most 2^-8 / sqrt(3) = 2.3e-3 of its norm. The output
carries two of them (h, y) beside the routed path's own error (measured below 1.2e-3 in the block's other
tests): 5e-3. The gradients carry three (of the upstream gradient, of gate | up's, of dx) in their shared
part, 4e-3, beside the routed backward's: 5e-3."""
import types

import numpy as np
import pytest
import torch

import oracle
from tests.conftest import assert_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


def keep_mask(shape, p, seed, stream):
    """Philox4x32-7 in numpy, uint64 products."""
    n = int(np.prod(shape))
    b = np.arange((n + 3) // 4, dtype=np.uint64)
    m = np.uint64(0xFFFFFFFF)
    c = [b & m, b >> np.uint64(32), np.full_like(b, stream & 0xFFFFFFFF), np.full_like(b, stream >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(7):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack(c, 1).reshape(-1)[:n]
    return torch.from_numpy((words >= int(p * 2 ** 32)).reshape(shape))


def bf(a):
    return torch.tensor(np.asarray(a), dtype=torch.float32).bfloat16().double().numpy()


class Adapter:
    def __init__(self, rng, n_in, n_out, r, p):
        self.lora_A = torch.tensor(rng.standard_normal((r, n_in)) * n_in ** -0.5, dtype=torch.float32, device="cuda")
        self.lora_B = torch.tensor(rng.standard_normal((n_out, r)) * 0.3, dtype=torch.float32, device="cuda")
        self.scaling, self.dropout_rate = 2.0, p
        self.lora_A.requires_grad_(True)
        self.lora_B.requires_grad_(True)


def make(rng, N, dense, adapters=True, act="situ"):
    from lazylora_amd.experts import ExpertLayer
    from lazylora_amd.latent_moe import LatentMoEBlock
    H, Dl, Fm, E, topk, Ds = 256, 128, 64, 8, 2, 136
    ex = oracle.random_experts(rng, E, Dl, Fm, 121, 125)
    g = lambda *s: bf(rng.standard_normal(s) * 0.05)
    p = {"gate": g(E, H), "bias": g(E), "w1": g(Ds, H), "w3": g(Ds, H), "w2": g(H, Ds), "down": g(Dl, H) * 4,
         "up": g(H, Dl), "norm": 1 + g(Dl)}
    bundle = None
    if adapters:
        bundle = types.SimpleNamespace(shared_gate_lora=Adapter(rng, H, Ds, 8, 0.1),
                                       shared_up_lora=Adapter(rng, H, Ds, 8, 0.25),
                                       shared_down_lora=Adapter(rng, Ds, H, 8, 0.5))
    L = ExpertLayer(*[torch.from_numpy(np.ascontiguousarray(a)).cuda()
                      for a in (ex.w1p, ex.w1s, ex.w3p, ex.w3s, ex.w2p, ex.w2s)])
    t = lambda a: torch.tensor(a, dtype=torch.float32)
    blk = LatentMoEBlock(L, t(p["gate"]), t(p["bias"]), t(p["w1"]), t(p["w3"]), t(p["w2"]), t(p["down"]), t(p["up"]),
                         t(p["norm"]), top_k=topk, routed_scaling_factor=2.5, act=act, lora=bundle, dense=dense)
    x = torch.tensor(bf(rng.standard_normal((N, H))), dtype=torch.float32, device="cuda", requires_grad=True)
    return blk, x, p, ex, bundle


def reference(x, p, ex, idx, bundle, seed, act="situ"):
    """The block in float64 torch on the CPU, the selection and the dropout masks given."""
    from lazylora_amd.latent_moe import glu, rms_norm
    d = {n: torch.tensor(a, dtype=torch.float64) for n, a in p.items()}
    ab = {}

    def delta(v, name, stream):
        if bundle is None:
            return 0.0
        mod = getattr(bundle, name)
        A, B = (t.detach().cpu().double().requires_grad_(True) for t in (mod.lora_A, mod.lora_B))
        ab[name] = (A, B)
        if seed is not None:
            v = torch.where(keep_mask(v.shape, mod.dropout_rate, seed, stream), v / (1 - mod.dropout_rate), 0.0)
        return mod.scaling * (v @ A.T) @ B.T

    scores = torch.sigmoid(x @ d["gate"].T)
    w = torch.gather(scores, -1, idx)
    w = w / (w.sum(-1, keepdim=True) + 1e-20) * 2.5
    s_act = glu(x @ d["w1"].T + delta(x, "shared_gate_lora", 0), x @ d["w3"].T + delta(x, "shared_up_lora", 1), act)
    shared = s_act @ d["w2"].T + delta(s_act, "shared_down_lora", 2)
    hl = x @ d["down"].T
    routed = torch.zeros_like(hl)
    for e in range(ex.E):
        W1, W3, W2 = (torch.from_numpy(m) for m in ex.dense(e))
        wt = ((idx == e).to(torch.float64) * w).sum(-1, keepdim=True)
        routed = routed + wt * (glu(hl @ W1.T, hl @ W3.T, act) @ W2.T)
    return shared + rms_norm(routed, d["norm"], 1e-5) @ d["up"].T, ab


@pytest.mark.parametrize("N,adapters,seed,act", [(1, False, None, "situ"), (24, True, None, "swiglu"),
                                                 (70, True, 12345678901, "situ"), (300, True, 7, "swiglu")])
def test_native_block_step(k, N, adapters, seed, act):
    print(f"\n[case] native block: {N} tokens, adapters {adapters}, seed {seed}, {act}", flush=True)
    rng = np.random.default_rng(900 + N)
    blk, x, p, ex, bundle = make(rng, N, "native", adapters, act)
    gout = torch.tensor(bf(rng.standard_normal((N, 256))), dtype=torch.float32, device="cuda")
    out, idx, _ = blk.forward(x, dropout_seed=seed)
    out.backward(gout)
    xr = x.detach().cpu().double().requires_grad_(True)
    ref, ab = reference(xr, p, ex, idx.cpu(), bundle, seed, act)
    ref.backward(gout.cpu().double())
    assert_close(out.detach().cpu().numpy(), ref.detach().numpy(), "block output")
    assert_close(x.grad.cpu().numpy(), xr.grad.numpy(), "dL/dx")
    for name, (A, B) in ab.items():
        mod = getattr(bundle, name)
        assert_close(mod.lora_A.grad.cpu().numpy(), A.grad.numpy(), f"{name} dL/dA")
        assert_close(mod.lora_B.grad.cpu().numpy(), B.grad.numpy(), f"{name} dL/dB")
    if seed is not None:  # the replayed forward of a recomputed layer drops the same elements
        again = blk.forward(x.detach(), dropout_seed=seed)[0]
        other = blk.forward(x.detach(), dropout_seed=seed + 1)[0]
        assert torch.equal(again, out.detach()) and not torch.equal(other, again)


def test_torch_block_with_dropout(k):
    """The fp32 block takes the adapters' dropout too; without a seed it is what it was."""
    print("\n[case] fp32 block with adapter dropout", flush=True)
    rng = np.random.default_rng(77)
    blk, x, p, ex, bundle = make(rng, 40, "torch")
    out, idx, _ = blk.forward(x, dropout_seed=99)
    ref, _ = reference(x.detach().cpu().double(), p, ex, idx.cpu(), bundle, 99)
    assert_close(out.detach().cpu().numpy(), ref.detach().numpy(), "block output")
    off, _ = reference(x.detach().cpu().double(), p, ex, idx.cpu(), bundle, None)
    assert_close(blk.forward(x)[0].detach().cpu().numpy(), off.detach().numpy(), "without a seed")


def test_native_block_refusals(k):
    from lazylora_amd.latent_moe import LatentMoEBlock
    print("\n[case] native block refusals", flush=True)
    rng = np.random.default_rng(5)
    blk, *_ = make(rng, 4, "native")
    z = lambda *s: torch.zeros(s)
    args = lambda H=256, Ds=136: (blk.experts, z(8, H), z(8), z(Ds, H), z(Ds, H), z(H, Ds), z(128, H), z(H, 128))
    for kw in (dict(dense="hip"), dict(dense="native", dense_dtype=torch.float32)):
        with pytest.raises(ValueError):
            LatentMoEBlock(*args(), **kw)
    for a in (args(H=252), args(Ds=100)):
        with pytest.raises(ValueError):
            LatentMoEBlock(*a, dense="native")
        LatentMoEBlock(*a)  # the fp32 block takes any width
