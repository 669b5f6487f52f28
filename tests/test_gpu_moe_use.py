"""Expert selection and 4-bit experts as programs use them together: threads, batched gradients, long stacks, prompts of
thousands of tokens."""
import threading

import numpy as np
import pytest
import torch

from test_gpu_int4 import gen_of, layer, routed64, weight

pytestmark = pytest.mark.gpu


def test_batched_gradients_are_refused():
    from lazylora_amd.router import select_experts
    x = torch.randn(5, 16, device="cuda", requires_grad=True)
    _, w = select_experts(x, 3, scoring="softmax")
    v = torch.randn(4, 5, 3, device="cuda")
    with pytest.raises(NotImplementedError, match="vmap"):
        torch.autograd.grad(w, x, v, is_grads_batched=True, retain_graph=True)
    one = torch.autograd.grad(w, x, v[0])[0]
    assert torch.isfinite(one).all()


def test_two_threads():
    """Calls from two threads, each on a stream of its own, right ones and refused ones: results and messages are
    each thread's own."""
    from lazylora_amd.int4 import int4_gemm, int4_routed
    from lazylora_amd.router import select_experts
    gen = gen_of(77)
    ex = layer(gen, 16, 256, 128, 64, True, torch.bfloat16)
    wt = weight(gen, (), 96, 256, 32, True, torch.bfloat16)
    inputs = [torch.randn(n, 256, device="cuda", generator=gen).bfloat16() for n in (1, 40)]
    gate = torch.randn(16, 256, device="cuda", generator=gen) / 4

    def step(h):
        x = (h.float() @ gate.T).requires_grad_(True)
        idx, w = select_experts(x, 4, torch.zeros(16, device="cuda"), num_groups=4, topk_groups=2)
        g = torch.autograd.grad(w, x, torch.ones_like(w))[0]
        return idx, w.detach(), g, int4_routed(h, idx, w.detach(), ex), int4_gemm(h, wt)

    want = [step(h) for h in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = step(inputs[i])
                    try:
                        select_experts(inputs[i], 0) if i else int4_gemm(inputs[i][:, :64], wt)
                    except ValueError as exc:
                        if ("top_k" if i else "width") not in str(exc):
                            wrong.append(str(exc))
                    torch.cuda.current_stream().synchronize()
                    wrong.extend(n for n, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as exc:  # noqa: BLE001 (the other thread's assertion shows it)
            wrong.append(repr(exc))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("N", [1, 5, 40])
def test_stacked_codes_past_32_bits(N):
    """Experts whose codes and scales lie more than 2^31 bytes (and 2^32 codes) behind the first, on each path."""
    from lazylora_amd.int4 import Int4Experts, Int4Weight, int4_routed
    E, D, F, group, dt = 70, 8192, 8192, 32, torch.bfloat16
    gen = gen_of(N, 70)

    def stack(R, K):
        packed = torch.empty(E, R, K // 2, device="cuda", dtype=torch.uint8)
        scales = torch.empty(E, R, K // group, device="cuda", dtype=dt)
        for e in range(E):  # cheap to make, and other codes in every expert
            packed[e] = (torch.arange(R * K // 2, device="cuda") * (2 * e + 3) // 7 % 251).view(R, K // 2).to(torch.uint8)
            scales[e] = 2.0 ** -10 * (1 + e % 3)
        return Int4Weight(packed, scales, None)

    whole = Int4Experts(stack(F, D), stack(F, D), stack(D, F))
    assert whole.w1.packed.numel() > 2 ** 31 and whole.w1.packed.numel() * 2 > 2 ** 32
    pick = [0, 64, 69]
    part = Int4Experts(*(Int4Weight(w.packed[pick].clone(), w.scales[pick].clone()) for w in (whole.w1, whole.w3, whole.w2)))
    h = torch.randn(N, D, device="cuda", generator=gen).to(dt)
    idx = torch.randint(0, 3, (N, 2), device="cuda", generator=gen)
    w = torch.rand(N, 2, device="cuda", generator=gen)
    got = int4_routed(h, torch.tensor(pick, device="cuda")[idx], w, whole).float()
    want = int4_routed(h, idx, w, part).float()
    # the forms may differ with the number of experts: hidden values and results a rounding step apart
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_a_prompt_of_thousands_of_tokens():
    """Many more pairs than the routing's threads, an expert with most of them and experts with none."""
    from lazylora_amd.int4 import int4_routed
    N, k, E, D, F, dt = 5000, 4, 40, 128, 64, torch.bfloat16
    gen = gen_of(N)
    ex = layer(gen, E, D, F, 32, True, dt)
    h = torch.randn(N, D, device="cuda", generator=gen).to(dt)
    idx = torch.randint(0, E - 3, (N, k), device="cuda", generator=gen)
    idx[:, 0] = 7
    w = torch.rand(N, k, device="cuda", generator=gen)
    out = int4_routed(h, idx, w, ex)
    want, size = routed64(h, idx, w, ex, "swiglu", dt)
    eps = torch.finfo(dt).eps
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= 0.75 * eps * size * 1.5 + eps / 2 * np.abs(want) + torch.finfo(dt).tiny).all()
    # the order in which the routing places pairs does not change a result
    assert all(torch.equal(int4_routed(h, idx, w, ex), out) for _ in range(5))


def test_saved_tensor_hooks():
    """Saved logits and indices that come back from a hook strided, in another type or on the host."""
    from lazylora_amd.router import select_experts
    x = torch.randn(7, 32, device="cuda").requires_grad_(True)
    dw = torch.randn(7, 4, device="cuda")
    run = lambda: select_experts(x, 4, scoring="softmax", num_groups=4, topk_groups=2)[1]
    want = torch.autograd.grad(run(), x, dw)[0]

    def strided(t):
        wide = torch.full((*t.shape, 2), -1, device=t.device, dtype=t.dtype)
        wide[..., 0] = t.detach()
        return wide[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(strided, lambda t: t):
        w = run()
    assert torch.equal(torch.autograd.grad(w, x, dw)[0], want)
    with torch.autograd.graph.save_on_cpu():
        w = run()
    assert torch.equal(torch.autograd.grad(w, x, dw)[0], want)
    for bad in (lambda t: t.cpu(), lambda t: t[:3], lambda t: t[:, :2], lambda t: t.double() if t.is_floating_point() else t.int()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), bad):
            w = run()
        with pytest.raises(ValueError):
            torch.autograd.grad(w, x, dw)
