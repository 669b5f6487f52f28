"""Host-side refusals of the dense operators' C entry points: nothing is launched. No GPU needed."""
import ctypes
import os

import pytest

vp = ctypes.c_void_p
P = vp(1 << 20)  # never dereferenced: every call below fails its checks, or has nothing to do, first
BF16, I32, F16, F32 = 1, 2, 4, 0


@pytest.fixture(scope="module")
def lib():
    from lazylora_amd import native
    if not os.path.exists(native.LIB_PATH):
        pytest.fail(f"{native.LIB_PATH} is not built: run __graft_entry__.build() first")
    return native._load_library()


def ffn_fwd(lib, ptrs=None, dtype=BF16, M=4, D=64, F=32, Do=64, act=0, ws=P, nws=1 << 40):
    p = dict.fromkeys(("y", "h", "gu", "x", "wg", "wu", "wd", "gd", "ud"), P)
    p.update(ptrs or {})
    return lib.mxfp4_ffn_forward(*p.values(), dtype, M, D, F, Do, act, ws, nws, None)


def ffn_bwd(lib, ptrs=None, dtype=BF16, M=4, D=64, F=32, Do=64, act=0, ws=P, nws=1 << 40):
    p = dict.fromkeys(("dx", "dwg", "dwu", "dwd", "dgu", "dy", "gh", "x", "h", "gu", "wg", "wu", "wd"), P)
    p.update(ptrs or {})
    return lib.mxfp4_ffn_backward(*p.values(), dtype, M, D, F, Do, act, ws, nws, None)


@pytest.mark.parametrize("call", [ffn_fwd, ffn_bwd])
def test_ffn_refusals(lib, call):
    for kw in ({"dtype": F32}, {"dtype": I32}, {"act": 2}, {"act": -1}, {"M": -1}, {"M": (1 << 24) + 1}, {"D": 60},
               {"F": 4}, {"Do": 0}, {"D": -8}, {"F": (1 << 20) + 8}):
        assert call(lib, **kw) == -1, kw
    for name in ("x", "wg", "wu", "wd"):
        assert call(lib, {name: vp((1 << 20) + 8)}) == -1
        assert b"aligned" in lib.mxfp4_last_error()
    for name in ("wg", "wu", "wd"):
        assert call(lib, {name: None}) == -1
        assert b"null" in lib.mxfp4_last_error()


def test_ffn_forward_nulls_and_empty(lib):
    for name in ("y", "h", "x"):
        assert ffn_fwd(lib, {name: None}) == -1
    assert ffn_fwd(lib, M=0, ptrs=dict.fromkeys(("y", "h", "gu", "x"))) == 0  # no rows: nothing to do


def test_ffn_backward_nulls(lib):
    for name in ("dgu", "dy", "gu", "x", "h", "dwg", "dwu"):  # dw_gate and dw_up go together
        assert ffn_bwd(lib, {name: None}) == -1
    nothing = dict.fromkeys(("dx", "dwg", "dwu", "dwd", "gh", "x", "h", "dgu", "dy", "gu"))
    assert ffn_bwd(lib, nothing, M=0) == 0


def test_ffn_workspace_refused_when_small(lib):
    n = lib.mxfp4_ffn_workspace_size(4, 4096, 256, 4096)
    if n:
        assert ffn_fwd(lib, D=4096, F=256, Do=4096, nws=n - 1) == -2
        assert ffn_bwd(lib, D=4096, F=256, Do=4096, nws=n - 1) == -2


def test_norm_refusals(lib):
    fwd = lambda y=P, x=P, M=4, D=8, kind=0, dtype=F32: lib.mxfp4_norm_forward(y, P, x, P, P, M, D, 1e-5, kind, dtype,
                                                                               None)
    for kw in ({"y": None}, {"x": None}, {"M": -1}, {"D": 0}, {"D": (1 << 20) + 1}, {"kind": 2}, {"dtype": I32}):
        assert fwd(**kw) == -1, kw
    assert fwd(M=0, x=None, y=None) == 0
    bwd = lambda dx=P, dw=P, db=P, dy=P, x=P, st=P, M=4, D=8, kind=1, dtype=BF16, ws=P, n=1 << 30: \
        lib.mxfp4_norm_backward(dx, dw, db, dy, x, P, st, M, D, kind, dtype, ws, n, None)
    for kw in ({"dx": None}, {"dy": None}, {"x": None}, {"st": None}, {"M": -1}, {"D": 0}, {"kind": 5}, {"dtype": 3},
               {"ws": None}, {"ws": vp(8)}):
        assert bwd(**kw) == -1, kw
    assert bwd(n=lib.mxfp4_norm_workspace_size(4, 8) - 1) == -2
    assert bwd(M=0, dw=None, db=None, dx=None, dy=None, x=None, st=None, ws=None, n=0) == 0


def test_dropout_refusals(lib):
    call = lambda y=P, x=P, n=8, p=0.5, dtype=F32: lib.mxfp4_dropout(y, x, n, p, 1, None, 0, dtype, None)
    for kw in ({"y": None}, {"x": None}, {"n": -1}, {"n": (1 << 40) + 1}, {"p": -0.1}, {"p": 1.1},
               {"p": float("nan")}, {"dtype": I32}):
        assert call(**kw) == -1, kw
    assert call(n=0, x=None, y=None) == 0


def test_operators_raise_where_the_library_is_off(monkeypatch):
    import torch
    from lazylora_amd import dense
    monkeypatch.setenv("LAZYLORA_NO_NATIVE", "1")
    x = torch.zeros(4, 8)
    for call in (lambda: dense.rms_norm(x), lambda: dense.layer_norm(x), lambda: dense.dropout(x, 0.5, 1),
                 lambda: dense.gated_ffn(x, x, x, x.T)):
        with pytest.raises(RuntimeError, match="unavailable"):
            call()


def test_autograd_module_is_built():
    from lazylora_amd import _dense_autograd
    assert all(hasattr(_dense_autograd, n) for n in ("norm", "dropout", "gated_ffn"))


def test_sizes_past_the_c_types_are_refused(lib):
    """Sizes that 32 bits would wrap to small ones (the call would compute those rows and leave the rest
    unwritten); expanded tensors, nothing is allocated. The size is looked at before the device."""
    import torch
    from lazylora_amd.native import MXFP4Kernel
    k = MXFP4Kernel(lib)
    z = lambda *s: torch.zeros((1,) * len(s), dtype=torch.bfloat16).expand(*s)
    f32 = lambda *s: torch.zeros((1,) * len(s)).expand(*s)
    for M, D in ((2 ** 32 + 5, 1), (2 ** 31, 1), (1, 2 ** 32 + 8), (1, 2 ** 20 + 1)):
        with pytest.raises(ValueError, match="too many rows or columns"):
            k.norm_forward(z(M, D))
        with pytest.raises(ValueError, match="too many rows or columns"):
            k.norm_backward(z(M, D), z(M, D), None, f32(2, M))
    big = 2 ** 32 + 8
    for M, D, F, Do in ((2 ** 32 + 4, 8, 8, 8), (2 ** 24 + 1, 8, 8, 8), (2, big, 8, 8), (2, 8, big, 8), (2, 8, 8, big),
                        (2, 8, 2 ** 20 + 8, 8)):
        w = (z(F, D), z(F, D), z(Do, F))
        with pytest.raises(ValueError, match=r"2\^24 rows"):
            k.ffn_forward(z(M, D), *w)
        with pytest.raises(ValueError, match=r"2\^24 rows"):
            k.ffn_backward(z(M, Do), f32(M, 2 * F), *w)


def test_ffn_backward_without_the_gate_and_up_gradient(lib):
    """dgu may be NULL only where neither dx nor dw_gate is asked for; then what its product reads may be too."""
    unread = dict.fromkeys(("dx", "dwg", "dwu", "dgu", "gu", "wg", "wu", "wd", "x"))
    for name in ("dy", "h"):
        assert ffn_bwd(lib, {**unread, name: None}) == -1
        assert b"null" in lib.mxfp4_last_error()
    assert ffn_bwd(lib, {**unread, "dx": P}) == -1
    assert ffn_bwd(lib, {**unread, "dwg": P, "dwu": P, "x": P}) == -1
    assert ffn_bwd(lib, {**unread, "dgu": P}) == -1
    assert ffn_bwd(lib, {**unread, "dwd": None}) == 0  # nothing asked for: nothing to do


def test_only_the_entry_points_have_c_names(lib):
    """Any other C name that the library exports could meet a host program's function of that name."""
    import re
    import subprocess
    from lazylora_amd import native
    out = subprocess.run(["nm", "-D", "--defined-only", native.LIB_PATH], capture_output=True, text=True, check=True)
    names = [l.split()[-1] for l in out.stdout.splitlines() if " T " in l]
    assert "mxfp4_gemm" in names
    assert [n for n in names if not n.startswith(("mxfp4_", "_Z", "_init", "_fini"))] == []
