"""The dense operators under forward-mode differentiation and under tracers: their launches record nothing
there, so such a call raises instead of dropping a derivative or tracing memory that nobody writes. The
refusal comes before every other check, so no GPU is needed to see it."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def _calls():
    """name -> (the module's function of its tensors, those tensors)."""
    from lazylora_amd import _dense_autograd as m
    x, w, b = torch.randn(3, 8), torch.ones(8), torch.zeros(8)
    h = torch.randn(3, 16)
    wg, wu, wd = torch.randn(16, 8), torch.randn(16, 8), torch.randn(8, 16)
    return {"norm": (lambda x, w, b: m.norm(x, w, b, 1e-5, 1), [x, w, b]),
            "dropout": (lambda x: m.dropout(x, 0.5, 1, None, 0), [x]),
            "gated_ffn": (lambda x, wg, wu, wd, gd, ud: m.gated_ffn(x, wg, wu, wd, 0, gd, ud, True)[0],
                          [x, wg, wu, wd, h, h.clone()])}


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    """A dual tensor in any place, whether or not the call records a gradient."""
    fn, args = _calls()[name]
    for i in range(len(args)):
        with fwad.dual_level():
            moved = [a.detach().requires_grad_(grad) for a in args]
            moved[i] = fwad.make_dual(moved[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*moved)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*moved)
    with pytest.raises(ValueError, match="HIP device|bfloat16"):  # without a tangent: the ordinary checks
        fn(*args)


@pytest.mark.parametrize("name", ["norm", "dropout", "gated_ffn"])
def test_tracers_are_refused(name):
    """torch.jit.trace and make_fx (before and after the dispatcher) would record the outputs' allocation and
    nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    fn, args = _calls()[name]
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(fn, tuple(args), check_trace=False)
    for mode in ("real", "fake"):
        for pre in (False, True):
            with pytest.raises(NotImplementedError, match="trace"):
                make_fx(fn, tracing_mode=mode, pre_dispatch=pre)(*args)
    with pytest.raises(ValueError, match="HIP device|bfloat16"):  # outside again: the ordinary checks
        fn(*args)


def test_other_dispatch_modes_are_not_tracers():
    """A mode that only watches (a flop counter, selective checkpointing) does not stop the call."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    fn, args = _calls()["norm"]
    with Watch(), pytest.raises(ValueError, match="HIP device"):
        fn(*args)
