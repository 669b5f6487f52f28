"""Norms and dropout of more rows and elements than one launch holds: HIP takes fewer than 2^32 threads per
launch, and the operators take 16 to 1024 threads per row, or one per eight elements. The border between two
launches and the end against calls on those rows alone, or against the formula."""
import pytest
import torch

from tests.test_gpu_norm_dropout import check, norm_reference, philox7

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


@pytest.fixture(autouse=True)
def empty_cache():
    yield
    torch.cuda.empty_cache()


def case(*a):
    print("\n[case]", *a, flush=True)


def filled(M, D):
    """[M, D] bfloat16 rows that differ within any 4097 neighbours, made a piece at a time."""
    piece = torch.randn(4097, D, device="cuda").bfloat16()
    x = torch.empty(M, D, dtype=torch.bfloat16, device="cuda")
    for i in range(0, M, 4097 * 4096):
        part = x[i:i + 4097 * 4096]
        part.copy_(piece.repeat((len(part) + 4096) // 4097, 1)[:len(part)])
    return x


# threads per row of each form: rows past 2^32 threads where that is little memory, else past a launch
@pytest.mark.parametrize("D,M", [(1, 2 ** 28 + 21), (3, 2 ** 28 + 5), (136, 2 ** 26 + 3), (520, 2 ** 24 + 1),
                                 (2056, 2 ** 21 + 2), (4104, 2 ** 20 + 3), (8200, 2 ** 19 + 1), (16392, 2 ** 19 + 3)])
@pytest.mark.parametrize("layer", [0, 1])
def test_norm_rows(k, D, M, layer):
    case("norm of", M, "rows of", D, "layer" if layer else "rms")
    x = filled(M, D)
    w = 1 + 0.2 * torch.randn(D, device="cuda")
    eps = 0.1
    y, st = k.norm_forward(x, w, None, eps, layer, True)
    threads = 16 if D <= 128 else 64 if D <= 512 else 256 if D <= 4096 else 512 if D <= 8192 else 1024
    border = 2 ** 29 // threads
    for first in (min(border - 300, M - 600), M - 600):
        part = x[first:first + 600].contiguous()
        want, stw = k.norm_forward(part, w, None, eps, layer, True)
        assert torch.equal(y[first:first + 600], want)
        assert torch.equal(st[0, first:first + 600], stw[0]) and (not layer or torch.equal(st[1, first:first + 600], stw[1]))
        (ref, eref), (dref, edref), _, _ = norm_reference(part, w, None, want, layer, eps)
        check("y", want, ref, eref)
        got, _, _ = k.norm_backward(want, part, w, stw, layer)
        check("dx", got, dref, edref)
    dx, _, _ = k.norm_backward(y, x, w, st, layer)
    for first in (min(border - 300, M - 600), M - 600):
        part = x[first:first + 600].contiguous()
        want, _, _ = k.norm_backward(y[first:first + 600].contiguous(), part, w, st[:, first:first + 600].contiguous(), layer)
        assert torch.equal(dx[first:first + 600], want)


def test_most_rows(k):
    """2^31 - 1 rows, the most that are taken; column gradients too."""
    M = 2 ** 31 - 1
    case("norm of", M, "rows of one element")
    x = torch.ones(M, 1, dtype=torch.bfloat16, device="cuda")
    x[-5:] = 2
    y, st = k.norm_forward(x, None, None, 3.0, 0, True)  # 1 / sqrt(1 + 3), 2 / sqrt(4 + 3)
    last = torch.tensor(2 / 7 ** 0.5).bfloat16().item()
    assert (y[:5] == 0.5).all() and (y[2 ** 25 - 5:2 ** 25 + 5] == 0.5).all() and (y[-5:] == last).all()
    dy = torch.zeros_like(x)
    dy[7], dy[-3] = 1, 1
    dx, dw, db = k.norm_backward(dy, x, None, st, 0, need_weight=True, need_bias=True)
    assert db.item() == 2 and abs(dw.item() - (0.5 + 2 / 7 ** 0.5)) < 1e-6
    assert dx[7].item() == 0.375 and not dx[8:1000].any()  # r - r^3 x^2 = 1/2 - 1/8


def test_dropout_elements(k):
    """2^35 + 13 elements, in place: more than 2^32 threads of eight."""
    n = 2 ** 35 + 13
    case("dropout of", n, "elements")
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert k.lib.mxfp4_dropout(x.data_ptr(), x.data_ptr(), n, 0.5, 99, None, 3, 1, s) == 0
    for first in (0, 2 ** 32 - 20, 2 ** 34 - 20, 2 ** 35 - 20, n - 30):
        keep = torch.tensor([philox7(i, 99, 3) >= 2 ** 31 for i in range(first, first + 30)], device="cuda")
        assert torch.equal(x[first:first + 30], keep * torch.tensor(2, dtype=torch.bfloat16, device="cuda"))
