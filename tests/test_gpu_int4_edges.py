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
