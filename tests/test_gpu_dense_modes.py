"""The dense operators' backward passes under forward-mode differentiation and under tracers, and the calls
that remain as they were beside them."""
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


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
def test_traced_backward_is_refused(name):
    """A graph recorded before, differentiated while a tracer runs."""
    from torch.fx.experimental.proxy_tensor import make_fx
    case("traced backward", name)
    y, leaves = graphs()[name]
    dy = torch.randn_like(y)
    for pre in (False, True):
        with pytest.raises(NotImplementedError, match="trace"):
            make_fx(lambda g: torch.autograd.grad(y, leaves, g, retain_graph=True), pre_dispatch=pre)(dy)
    with pytest.raises(RuntimeError):  # torch itself refuses to trace over recorded tensors
        torch.jit.trace(lambda g: torch.autograd.grad(y, leaves, g, retain_graph=True), (dy,), check_trace=False)
    assert all(g.isfinite().all() for g in torch.autograd.grad(y, leaves, dy))


def test_modes_that_watch():
    """Under a flop counter and inside a compiled function (whose graph breaks at the call) results stay."""
    from torch.utils.flop_counter import FlopCounterMode
    from lazylora_amd.dense import rms_norm
    case("watching modes")
    x = torch.randn(4, 16, device="cuda")
    plain = rms_norm(x)
    with FlopCounterMode(display=False):
        assert torch.equal(rms_norm(x), plain)
    assert torch.equal(torch.compile(lambda t: rms_norm(t) + 1, backend="eager")(x), plain + 1)
