"""The dense operators' backward passes under forward-mode differentiation, and the calls that remain as
they were beside it."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")


def case(*a):
    print("\n[case]", *a, flush=True)


def graphs():
    """name -> (an output recorded outside every mode, its leaves)."""
    from lazylora_amd.dense import dropout, gated_ffn, layer_norm
    r = lambda *s: torch.randn(*s, device="cuda")
    x, w = r(5, 24).requires_grad_(True), r(24).requires_grad_(True)
    f = [r(5, 24), r(16, 24), r(16, 24), r(32, 16)]
    f = [t.bfloat16().requires_grad_(True) for t in f]
    return {"norm": (layer_norm(x, w, w), [x, w]), "dropout": (dropout(x, 0.5, 3), [x]),
            "gated_ffn": (gated_ffn(*f), f)}


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
def test_upstream_tangents_are_refused(name):
    """The derivative of a backward pass along its upstream gradient would come out as zero."""
    case("tangent upstream", name)
    y, leaves = graphs()[name]
    dy = torch.randn_like(y)
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaves, fwad.make_dual(dy, dy), retain_graph=True)
        # no tangent among its tensors: an open level changes nothing
        inside = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    outside = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(inside, outside))


def test_inputs_with_tangents_are_refused():
    from lazylora_amd.dense import rms_norm
    case("tangent of an input")
    x = torch.randn(4, 16, device="cuda")
    plain = rms_norm(x)
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rms_norm(fwad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(rms_norm(x), plain)
