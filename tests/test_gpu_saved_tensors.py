"""Backward passes over what saved-tensor hooks hand back: the dense operators' tensors strided, in another type, of
another size or on the host."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

pytestmark = pytest.mark.gpu


def calls():
    """name -> (function of its leaves, leaves)."""
    from lazylora_amd.dense import dropout, gated_ffn, layer_norm
    gen = torch.Generator("cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    seed = torch.tensor([5], device="cuda")
    low = lambda *s: r(*s).bfloat16().requires_grad_(True)
    return {"norm": (layer_norm, [r(5, 3, 24).requires_grad_(True), r(24).requires_grad_(True), r(24).requires_grad_(True)]),
            "dropout": (lambda x: dropout(x, 0.5, seed), [r(5, 24).requires_grad_(True)]),
            "gated_ffn": (gated_ffn, [low(2, 9, 24), low(16, 24), low(16, 24), low(32, 16)])}


def strided(t):
    wide = torch.zeros((*t.shape, 2), device=t.device, dtype=t.dtype)
    wide[..., 0] = t.detach()
    return wide[..., 0]


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
def test_other_layouts(name):
    fn, leaves = calls()[name]
    y = fn(*leaves)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dy)
    for hooks in (saved_tensors_hooks(strided, lambda t: t), save_on_cpu()):
        with hooks:
            y = fn(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: torch.cat([t, t]), lambda t: t[..., :0],
                                    lambda t: t.half() if t.dtype != torch.float16 else t.float()],
                         ids=["host", "longer", "empty", "type"])
def test_what_does_not_fit_is_refused(name, unpack):
    fn, leaves = calls()[name]
    with saved_tensors_hooks(lambda t: t.detach(), unpack):
        y = fn(*leaves)
    with pytest.raises(ValueError):
        torch.autograd.grad(y, leaves, torch.randn_like(y))


@pytest.mark.parametrize("which", range(6))
def test_each_saved_tensor_of_the_feed_forward_block(which):
    """One of the tensors alone comes back a row short."""
    fn, leaves = calls()["gated_ffn"]
    count = iter(range(100))
    with saved_tensors_hooks(lambda t: (next(count), t.detach()), lambda p: p[1][:-1] if p[0] == which else p[1]):
        y = fn(*leaves)
    assert next(count) == 6
    with pytest.raises(ValueError):
        torch.autograd.grad(y, leaves, torch.randn_like(y))
