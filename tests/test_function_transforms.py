"""The operators under torch.func transforms and batched gradients: a launch takes memory, and a transform's tensors
have none of their own, so such a call says so before anything else. No GPU needed."""
import pytest
import torch
from torch.func import functionalize, grad, vmap


def _calls():
    """name -> (the module's function of its first tensor, that tensor)."""
    from lazylora_amd import _dense_autograd as m
    b, w = torch.zeros(8), torch.ones(8)
    wg, wd = torch.randn(16, 8), torch.randn(8, 16)
    q, s = torch.zeros(4, 4, dtype=torch.uint8), torch.ones(4, 1).bfloat16()
    return {"select": lambda x: m.select_experts(x, b, 2, 0, 1, 1, 0, 1.0, True)[1],
            "int4_gemm": lambda x: m.int4_gemm(x, q, s, None),
            "norm": lambda x: m.norm(x, w, b, 1e-5, 1), "dropout": lambda x: m.dropout(x, 0.5, 1, None, 0),
            "gated_ffn": lambda x: m.gated_ffn(x, wg, wg, wd, 0, None, None, False)[0]}


@pytest.mark.parametrize("name", ["select", "int4_gemm", "norm", "dropout", "gated_ffn"])
def test_transformed_tensors_are_refused(name):
    fn, x = _calls()[name], torch.randn(3, 4, 8)
    for transform in (vmap, lambda f: vmap(f, in_dims=1), lambda f: grad(lambda t: f(t).sum()), functionalize):
        with torch.no_grad(), pytest.raises(NotImplementedError, match="vmap"):
            transform(fn)(x)
        with pytest.raises(NotImplementedError, match="vmap"):
            transform(fn)(x)
    # a tensor that is not the transform's own is an ordinary one
    with pytest.raises((ValueError, NotImplementedError), match="HIP device|bfloat16"):
        vmap(lambda t: fn(x[0]))(x)
    with pytest.raises((ValueError, NotImplementedError), match="HIP device|bfloat16"):
        fn(x[0])
