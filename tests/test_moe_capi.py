"""Host-side refusals of the selection's and the 4-bit products' C entry points, and their operators under tracers and
forward-mode differentiation: nothing is launched. No GPU needed."""
import ctypes
import os

import pytest
import torch
import torch.autograd.forward_ad as fwad

vp = ctypes.c_void_p
P = vp(1 << 20)  # never dereferenced: every call below fails its checks, or has nothing to do, first
F32, BF16, I32, I64, F16 = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    from lazylora_amd import native
    if not os.path.exists(native.LIB_PATH):
        pytest.fail(f"{native.LIB_PATH} is not built: run __graft_entry__.build() first")
    return native._load_library()


def select(lib, idx=P, w=P, logits=P, dtype=F32, bias=P, N=4, E=64, k=6, scoring=1, groups=8, kept=3, score=0):
    return lib.mxfp4_select_topk(idx, w, logits, dtype, bias, N, E, k, scoring, groups, kept, score, 1.0, 1, None)


def test_select_refusals(lib):
    for kw in ({"idx": None}, {"w": None}, {"logits": None}, {"dtype": I32}, {"N": -1}, {"E": 0}, {"E": 4097, "groups": 1},
               {"k": 0}, {"k": 65, "groups": 1, "kept": 1}, {"k": 25}, {"scoring": 2}, {"groups": 0}, {"groups": 5},
               {"groups": 65, "E": 650}, {"kept": 0}, {"kept": 9}, {"score": 2}, {"E": 33 * 124, "groups": 33}):
        assert select(lib, **kw) == -1, kw
        assert b"select_topk" in lib.mxfp4_last_error()
    assert select(lib, N=0, idx=None, w=None, logits=None, bias=None) == 0


def test_select_backward_refusals(lib):
    call = lambda g=P, idx=P, gw=P, x=P, dtype=BF16, N=4, E=64, k=6, scoring=0: lib.mxfp4_select_topk_backward(
        g, idx, gw, x, dtype, N, E, k, scoring, 1.0, 1, None)
    for kw in ({"g": None}, {"idx": None}, {"gw": None}, {"x": None}, {"dtype": I64}, {"N": -1}, {"E": 4097}, {"k": 0},
               {"k": 65}, {"E": 5}, {"scoring": -1}):
        assert call(**kw) == -1, kw
    assert call(N=0, g=None, idx=None, gw=None, x=None) == 0


def test_int4_gemm_refusals(lib):
    call = lambda y=P, x=P, q=P, s=P, z=P, dtype=BF16, M=3, K=256, R=16, group=64: lib.mxfp4_int4_gemm(
        y, x, q, s, z, dtype, M, K, R, group, None)
    odd = vp((1 << 20) + 8)
    for kw in ({"y": None}, {"x": None}, {"q": None}, {"s": None}, {"y": odd}, {"x": odd}, {"q": odd}, {"s": odd}, {"z": odd},
               {"dtype": F32}, {"M": -1}, {"M": (1 << 24) + 1}, {"K": 0}, {"K": 224}, {"K": (1 << 20) + 64}, {"R": 0},
               {"R": (1 << 20) + 1}, {"group": 16}, {"group": 256}, {"group": 0}):
        assert call(**kw) == -1, kw
        assert b"int4_gemm" in lib.mxfp4_last_error()
    assert call(M=0, y=None, x=None, q=None, s=None, z=None) == 0


def moe(lib, out=P, h=P, dtype=BF16, idx=P, it=I64, w=P, N=4, k=2, codes=(P, P, P), scales=(P, P, P), zeros=None, E=8, D=256,
        F=128, group=64, act=0, ws=P, n=1 << 40):
    arr = lambda t: None if t is None else (vp * 3)(*[x if x is None else x.value for x in t])
    return lib.mxfp4_int4_moe_forward(out, h, dtype, idx, it, w, N, k, arr(codes), arr(scales), arr(zeros), E, D, F, group, act,
                                      ws, n, None)


def test_int4_moe_refusals(lib):
    odd = vp((1 << 20) + 8)
    for kw in ({"out": None}, {"h": None}, {"idx": None}, {"w": None}, {"ws": None}, {"codes": None}, {"scales": None},
               {"codes": (P, None, P)}, {"scales": (P, P, None)}, {"zeros": (P, None, P)}, {"zeros": (None, None, P)},
               {"out": odd}, {"h": odd}, {"codes": (P, P, odd)}, {"scales": (odd, P, P)}, {"zeros": (P, odd, P)},
               {"ws": vp((1 << 20) + 16)}, {"dtype": F32}, {"it": F16}, {"N": -1}, {"k": 0}, {"N": 1 << 24}, {"E": 0},
               {"E": 4097}, {"D": 224}, {"F": 96}, {"F": 0}, {"group": 48}, {"act": 2}, {"N": (1 << 23) + 1, "D": 1 << 10}):
        assert moe(lib, **kw) == -1, kw
        assert b"int4_moe_forward" in lib.mxfp4_last_error()
    size = lib.mxfp4_int4_moe_workspace_size(4, 2, 8, 256, 128)
    assert size > 0 and moe(lib, n=size - 1) == -2
    assert moe(lib, N=0, out=None, h=None, idx=None, w=None, ws=None, n=0) == 0
    for args in ((0, 2, 8, 256, 128), (4, 0, 8, 256, 128), (1 << 24, 2, 8, 256, 128), (4, 2, 0, 256, 128)):
        assert lib.mxfp4_int4_moe_workspace_size(*args) == 0


def _calls():
    from lazylora_amd import _dense_autograd as m
    x, b, h = torch.randn(3, 8), torch.zeros(8), torch.randn(2, 64).bfloat16()
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 2).bfloat16()
    return {"select": (lambda x, b: m.select_experts(x, b, 2, 0, 1, 1, 0, 1.0, True)[1], [x, b]),
            "int4_gemm": (lambda h, s: m.int4_gemm(h, q, s, None), [h, s])}


@pytest.mark.parametrize("name", ["select", "int4_gemm"])
def test_tangents_and_tracers_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    fn, args = _calls()[name]
    for i in range(len(args)):
        with fwad.dual_level():
            moved = list(args)
            moved[i] = fwad.make_dual(moved[i], torch.ones_like(args[i]))
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*moved)
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(fn, tuple(args), check_trace=False)
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(fn)(*args)
    with pytest.raises(ValueError, match="HIP device"):  # otherwise: the ordinary checks
        fn(*args)
