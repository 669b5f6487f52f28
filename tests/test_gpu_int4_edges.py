"""Products with group-scaled 4-bit weights where waves, rounds and widths do not divide evenly, against 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_int4 import DT, bound, dense64, gen_of, layer, matrix64, weight

pytestmark = pytest.mark.gpu


# Of the form for 16 rows: 17 units of 256 codes in two rounds of 9 waves (the last wave has none in the second), with
# groups of 32 of 23 in three of 8; all its waves with all its batches, which takes more than 64 KiB of LDS.
@pytest.mark.parametrize("M,K,R", [(5, 4352, 17), (16, 4352, 33), (7, 5888, 16), (16, 4096, 16400)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_waves_without_a_last_unit(M, K, R, group, dtype):
    from lazylora_amd.int4 import int4_gemm
    dt = DT[dtype]
    for zeros in (False, True):
        gen = gen_of(M, K, R, group, zeros)
        x = torch.randn(M, K, device="cuda", generator=gen).to(dt)
        w = weight(gen, (), R, K, group, zeros, dt)
        xs = x.double().cpu().numpy()
        want = xs @ dense64(w).T
        err = np.abs(int4_gemm(x, w).double().cpu().numpy() - want)
        assert (err <= bound(xs, w, want, dt)).all(), (zeros, err.max())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_routed_waves_without_a_last_unit(group, dtype):
    """Gate/up over 9 units in two rounds of 5 waves, down over 17 in two of 9. Small whole numbers with scales of
    powers of two: gate and up products are exact, so a hidden value is off by its rounding and the activation's
    error alone."""
    from lazylora_amd.int4 import int4_routed
    dt, N, k, E, D, F = DT[dtype], 9, 2, 3, 2304, 4352
    for zeros in (False, True):
        gen = gen_of(group, zeros)
        ex = layer(gen, E, D, F, group, zeros, dt)
        for m in (ex.w1, ex.w3):
            m.scales.copy_(2.0 ** torch.randint(-8, -6, m.scales.shape, device="cuda", generator=gen))
        h = torch.randint(-2, 3, (N, D), device="cuda", generator=gen).to(dt)
        idx = torch.randn(N, E, device="cuda", generator=gen).topk(k, -1).indices
        w = torch.rand(N, k, device="cuda", generator=gen)
        got = int4_routed(h, idx, w, ex).double().cpu().numpy()
        hs, ids, ws = h.double().cpu().numpy(), idx.cpu().numpy(), w.double().cpu().numpy()
        want, tol = np.zeros((N, D)), np.zeros((N, D))
        eps = torch.finfo(dt).eps
        for e in range(E):
            t, j = np.nonzero(ids == e)
            w1, w3, w2 = (matrix64(m.packed[e], m.scales[e], None if m.zeros is None else m.zeros[e])
                          for m in (ex.w1, ex.w3, ex.w2))
            scale = np.repeat(ex.w2.scales[e].double().cpu().numpy(), group, -1)
            g, u = hs[t] @ w1.T, hs[t] @ w3.T
            a = g / (1 + np.exp(-g)) * u
            np.add.at(want, t, ws[t, j, None] * (a @ w2.T))
            # half a step and the activation's 2^-18 of each hidden value; the sums' as in bound()
            hidden = (eps / 2 + 2.0 ** -18) * (np.abs(a) @ np.abs(w2).T) + torch.finfo(dt).tiny * np.abs(w2).sum(1)
            sums = (F / 4 + 16) * 2.0 ** -24 * (np.abs(a) @ (62 * np.abs(scale)).T)
            np.add.at(tol, t, ws[t, j, None] * (hidden + sums))
        tol += eps / 2 * (np.abs(want) + tol) + torch.finfo(dt).tiny
        assert (np.abs(got - want) <= tol).all(), zeros


# every form: one, two and four rows, 16 rows, and the tiles'
FORMS = [(1, 1152, 40), (2, 1152, 40), (4, 1152, 40), (6, 1152, 40), (20, 1152, 40), (64, 1152, 2100), (200, 384, 2100),
         (300, 384, 2100), (600, 384, 2100), (1100, 128, 2100)]


@pytest.mark.parametrize("M,K,R", FORMS)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_largest_numbers(M, K, R, group):
    """Rows of numbers up to 2^112 with every zero point: a group's sums stay in 32 bits, whatever the signs."""
    from lazylora_amd.int4 import Int4Weight, int4_gemm
    gen, dt = gen_of(M, K, group), torch.bfloat16
    x = (2.0 ** 111 * (1 + torch.rand(M, K, device="cuda", generator=gen))).to(dt)
    x[x > 2.0 ** 112] = 2.0 ** 112
    x[M // 2:] *= 1 - 2 * torch.randint(0, 2, (M - M // 2, K), device="cuda", generator=gen)
    packed = torch.randint(0, 256, (R, K // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = (2.0 ** torch.randint(-120, -110, (R, K // group), device="cuda", generator=gen).float()).to(dt)
    zeros = torch.randint(0, 256, scales.shape, device="cuda", generator=gen, dtype=torch.uint8)
    zeros[0] = 255
    w = Int4Weight(packed, scales, zeros)
    xs = x.double().cpu().numpy()
    want = xs @ dense64(w).T
    # as bound(), with 31 of a code and 16 + z of the sum
    each = (47 + zeros.double().cpu().numpy()) * scales.double().cpu().numpy()
    tol = ((K / 4 + 16) * 2.0 ** -24 * (np.abs(xs) @ np.repeat(each, group, -1).T) + torch.finfo(dt).eps / 2 * np.abs(want)
           + torch.finfo(dt).tiny)
    assert (np.abs(int4_gemm(x, w).double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("M,K,R", FORMS)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_scales_that_are_not_finite(M, K, R, value):
    """Their rows of weights give infinities or NaN, the others what they give without them."""
    from lazylora_amd.int4 import int4_gemm
    gen = gen_of(M, K, R)
    for k in (K, K + 32):  # also in a last block that is not full
        x = torch.randn(M, k, device="cuda", generator=gen).half()
        w = weight(gen, (), R, k, 32, True, torch.float16)
        want = int4_gemm(x, w)
        rows = torch.tensor([0, R // 2, R - 1], device="cuda")
        w.scales[rows, torch.tensor([0, 1, k // 32 - 1], device="cuda")] = value
        got = int4_gemm(x, w)
        clean = torch.ones(R, dtype=torch.bool, device="cuda")
        clean[rows] = False
        assert not torch.isfinite(got[:, rows]).any() and torch.equal(got[:, clean], want[:, clean])
