"""Layer and RMS norm and the counter-based dropout against their formulas in 64 bits.

Norm bounds per element: fp32 sums over D terms in a tree (no partial sum is longer than 64 terms per
lane and step), so (64 + log2 D) 2^-24 relative to sums of absolute values covers a mean; everything is
carried through the formulas, plus u = eps / 2 of the type for the final rounding. Dropout is exact up to
the product's rounding; its mask is compared bit for bit with Philox4x32-7 in Python integers."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


def case(*a):
    print("\n[case]", *a, flush=True)


def check(name, got, want, bound):
    over = ((got.double() - want).abs() / bound)
    assert got.shape == want.shape and not torch.isnan(over).any(), name
    worst = over.max().item() if over.numel() else 0.0
    print(f"{name}: largest error {worst:.3f} of its bound")
    assert worst <= 1.0, f"{name}: {worst:.2f} times its bound"


def norm_reference(x, w, b, dy, layer, eps):
    """float64 outputs and gradients with bounds: (y, dx, dw, db)."""
    dt = x.dtype
    u, s = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    M, D = x.shape
    f = (64 + max(D, 2).bit_length()) * 2.0 ** -24
    X, G = x.double(), dy.double()
    W = torch.ones(D, dtype=torch.float64, device="cuda") if w is None else w.double()
    mean = X.mean(1, keepdim=True) if layer else torch.zeros(M, 1, dtype=torch.float64, device="cuda")
    em = f * X.abs().mean(1, keepdim=True) if layer else 0 * mean
    c = X - mean
    r = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    # relative error of r: half of the mean square's, whose terms are off by em each (to first order their
    # sum cancels; second order em^2) and by the difference's own rounding
    er = f + 2.0 ** -22 + 0.5 * (em * r) ** 2 + 2.0 ** -23 * (X.abs() * c.abs()).mean(1, keepdim=True) * r * r
    xh = c * r
    exh = em * r + xh.abs() * er + 2.0 ** -23 * X.abs() * r
    y = xh * W + (0 if b is None else b.double())
    ey = exh * W.abs() + 2.0 ** -22 * (xh * W).abs() + 2.0 ** -23 * y.abs() + u * y.abs() + s
    t = G * W
    m1 = (t * xh).mean(1, keepdim=True)
    m0 = t.mean(1, keepdim=True) if layer else 0 * m1
    em1 = f * (t * xh).abs().mean(1, keepdim=True) + (t.abs() * exh).mean(1, keepdim=True)
    em0 = f * t.abs().mean(1, keepdim=True) if layer else 0 * m1
    dx = r * (t - m0 - xh * m1)
    edx = r * (em0 + xh.abs() * em1 + exh * m1.abs() + 2.0 ** -21 * (t.abs() + m0.abs() + (xh * m1).abs())) \
        + er * dx.abs() + u * dx.abs() + s
    fr = (M + 8) * 2.0 ** -24  # sums over rows, in runs
    dw, db = (G * xh).sum(0), G.sum(0)
    edw = fr * (G * xh).abs().sum(0) + (G.abs() * exh).sum(0) + 1e-37
    edb = fr * G.abs().sum(0) + 1e-37
    return (y, ey), (dx, edx), (dw, edw), (db, edb)


NORM_SIZES = [(1, 1), (3, 2), (5, 7), (64, 8), (1000, 64), (257, 127), (130, 128), (33, 129), (70, 512), (9, 513),
              (41, 1000), (300, 2048), (21, 2049), (7, 3584), (1, 7168), (600, 7168), (3, 8191), (2, 8193), (5, 16384),
              (4, 16385), (3, 40001)]


@pytest.mark.parametrize("M,D", NORM_SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layer", [0, 1])
def test_norm(k, M, D, dt, layer):
    case("norm", M, D, dt, "layer" if layer else "rms")
    g = torch.Generator(device="cuda").manual_seed(M + D)
    x = (torch.randn(M, D, device="cuda", generator=g) * 2 + 0.5).to(dt)
    w = 1 + 0.2 * torch.randn(D, device="cuda", generator=g)
    b = 0.3 * torch.randn(D, device="cuda", generator=g) if layer else None
    dy = torch.randn(M, D, device="cuda", generator=g).to(dt)
    eps = 1e-5 if D > 1 else 0.1  # a layer norm of one element divides by sqrt(eps) alone
    (y, ey), (dx, edx), (dw, edw), (db, edb) = norm_reference(x, w, b, dy, layer, eps)
    got, stats = k.norm_forward(x, w, b, eps, layer, save_for_backward=True)
    assert torch.equal(got, k.norm_forward(x, w, b, eps, layer)[0])
    check("y", got, y, ey)
    gx, gw, gb = k.norm_backward(dy, x, w, stats, layer, need_weight=True, need_bias=True)
    check("dx", gx, dx, edx)
    check("dw", gw, dw, edw)
    check("db", gb, db, edb)
    gx2, none, gb2 = k.norm_backward(dy, x, w, stats, layer, need_bias=True)
    assert none is None and torch.equal(gx, gx2) and torch.equal(gb, gb2)
    gx3, none, _ = k.norm_backward(dy, x, w, stats, layer)
    assert none is None and torch.equal(gx, gx3)


@pytest.mark.parametrize("D", [24, 1001])
def test_norm_autograd(k, D):
    """No weight, weights of other types, higher axes, strided inputs, gradients against differences."""
    from lazylora_amd.dense import layer_norm, rms_norm
    case("norm autograd", D)
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(D, 6, 5, device="cuda", generator=g).permute(1, 2, 0).requires_grad_(True)  # [6, 5, D], strided
    assert not x.is_contiguous()
    dy = torch.randn(6, 5, D, device="cuda", generator=g)
    wb = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16().requires_grad_(True)
    bb = (0.1 * torch.randn(D, device="cuda", generator=g)).half().requires_grad_(True)
    for layer in (False, True):
        for w, b in ((None, None), (wb, None), (wb, bb)):
            if b is not None and not layer:
                continue
            y = layer_norm(x, w, b) if layer else rms_norm(x, w)
            leaves = [t for t in (x, w, b) if t is not None]
            grads = torch.autograd.grad(y, leaves, dy)
            assert all(a.dtype == l.dtype and a.shape == l.shape for a, l in zip(grads, leaves))
            X = x.detach().double()
            V = {"x": X, "w": None if w is None else w.detach().double(), "b": None if b is None else b.detach().double()}

            def loss(**moved):
                v = {**V, **moved}
                c = v["x"] - v["x"].mean(-1, keepdim=True) if layer else v["x"]
                o = c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
                o = o if v["w"] is None else o * v["w"]
                return ((o if v["b"] is None else o + v["b"]) * dy.double()).sum()

            for n, got in zip([n for n in "xwb" if V[n] is not None], grads):
                dirn = torch.randn(V[n].shape, dtype=torch.float64, device="cuda",
                                   generator=torch.Generator(device="cuda").manual_seed(1))
                diff = (loss(**{n: V[n] + 1e-5 * dirn}) - loss(**{n: V[n] - 1e-5 * dirn})) / 2e-5
                u = torch.finfo(got.dtype).eps
                slack = (got.double().abs() * dirn.abs()).sum() * max(u, 1e-5) + 1e-5
                assert ((got.double() * dirn).sum() - diff).abs() <= slack, n
    flat = rms_norm(x.detach(), wb.detach())
    rows = k.norm_forward(x.detach().reshape(30, D), wb.detach().float())[0]
    assert torch.equal(flat.reshape(30, D), rows)


def test_norm_special_rows(k):
    """A constant row (variance 0), a zero row, rows with NaN and infinity: each only its own outputs."""
    from lazylora_amd.dense import layer_norm, rms_norm
    case("special rows")
    x = torch.randn(8, 300, device="cuda")
    x[1], x[2], x[3, 7], x[4, 9] = 2.5, 0.0, float("nan"), float("inf")
    for y in (layer_norm(x), rms_norm(x)):
        assert torch.isfinite(y[[0, 1, 2, 5, 6, 7]]).all()
        assert torch.isnan(y[3]).all() and torch.isnan(y[4, 9])
        assert not y[2].any()
    assert layer_norm(x)[1].abs().max() < 1e-3


def test_norm_empty_and_refusals(k):
    from lazylora_amd.dense import layer_norm, rms_norm
    case("norm: empty, refusals")
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and not gw.any()
    ok = torch.zeros(4, 64, device="cuda")
    for bad in (lambda: rms_norm(ok.cpu()), lambda: rms_norm(ok.double()), lambda: rms_norm(ok.long()),
                lambda: rms_norm(ok, w[:63].detach()), lambda: layer_norm(ok, w.detach(), w.detach()[None]),
                lambda: rms_norm(ok, w.detach().cpu()), lambda: rms_norm(torch.zeros((), device="cuda")),
                lambda: rms_norm(torch.zeros(3, 0, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    _, st = k.norm_forward(ok, save_for_backward=True)
    for bad in (lambda: k.norm_backward(ok[:3], ok, None, st), lambda: k.norm_backward(ok, ok, None, st[:, :3]),
                lambda: k.norm_backward(ok.half(), ok, None, st), lambda: k.norm_backward(ok, ok, w.half(), st)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------- dropout
def philox7(i, seed, stream):
    m = 0xFFFFFFFF
    c = [(i >> 2) & m, i >> 34, stream & m, stream >> 32]
    k0, k1 = seed & m, seed >> 32
    for _ in range(7):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k0, b & m, (a >> 32) ^ c[3] ^ k1, a & m]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return c[i & 3]


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 255, 2047, 2048, 2049, 10001])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("p,seed,stream", [(0.1, 1234567890123456789, 0), (0.5, 2 ** 64 - 1, 2 ** 64 - 5),
                                           (0.999, 0, 2 ** 32)])
def test_dropout_mask_and_values(k, n, dt, p, seed, stream):
    case("dropout", n, dt, p)
    x = (torch.randn(n, device="cuda") + 3).to(dt)
    x = torch.where(x == 0, torch.ones_like(x), x)
    y = k.dropout(x, p, seed, stream)
    thr = int(p * 2 ** 32)
    keep = torch.tensor([philox7(i, seed, stream) >= thr for i in range(n)], device="cuda")
    assert torch.equal(y != 0, keep)
    want = torch.where(keep, x.float() * (1.0 / (1.0 - p)), torch.zeros((), device="cuda")).to(dt)
    assert torch.equal(y, want)  # one fp32 product, one rounding


def test_dropout_autograd_and_properties(k):
    from lazylora_amd.dense import dropout
    case("dropout properties")
    x = torch.randn(300, 1001, device="cuda").T.requires_grad_(True)  # strided: numbered in row-major order
    y = dropout(x, 0.25, 42, 3)
    dy = torch.randn_like(y)
    (g,) = torch.autograd.grad(y, (x,), dy)
    assert torch.equal(g, dropout(dy, 0.25, 42, 3))
    assert torch.equal((g == 0) | (x == 0), (y == 0) | (dy == 0))  # x and dy may hold a zero themselves
    assert torch.equal(y.detach(), k.dropout(x.detach().contiguous(), 0.25, 42, 3))
    # kept counts: binomial, 6 standard deviations
    n = x.numel()
    assert abs((y != 0).sum().item() - 0.75 * n) < 6 * (n * 0.75 * 0.25) ** 0.5
    # another seed, stream: independent masks agree on (0.75^2 + 0.25^2) of the elements
    for other in (dropout(x, 0.25, 43, 3), dropout(x, 0.25, 42, 4)):
        same = ((other != 0) == (y != 0)).sum().item()
        assert abs(same - 0.625 * n) < 6 * (n * 0.625 * 0.375) ** 0.5
    assert torch.equal(dropout(x, 0.0, 1), x)
    assert not dropout(x, 1.0, 1).any()
    bad = torch.full((4096,), float("nan"), device="cuda")
    z = k.dropout(bad, 0.5, 9)
    assert 0 < (z == 0).sum().item() < 4096 and torch.isnan(z[z != 0]).all()  # dropped is 0 even for NaN
    assert dropout(torch.empty(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)
    off = torch.randn(1003, device="cuda").bfloat16()[3:]  # 2-byte aligned start
    assert torch.equal(k.dropout(off, 0.3, 5), k.dropout(off.clone(), 0.3, 5))


def test_dropout_seed_tensor_and_graph(k):
    """A seed in device memory gives the number's mask; a captured graph follows it between replays; a
    seed changed between a forward and its backward is noticed."""
    from lazylora_amd.dense import dropout
    case("seed tensor, graph")
    x = torch.randn(5000, device="cuda")
    seed = torch.tensor([77], device="cuda")
    assert torch.equal(dropout(x, 0.3, seed, 2), dropout(x, 0.3, 77, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = dropout(x, 0.3, seed, 2)
    for s in (77, 78, 2 ** 62, 5):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, dropout(x, 0.3, s, 2))
    xr = x.clone().requires_grad_(True)
    y = dropout(xr, 0.3, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_dropout_refusals(k):
    case("dropout refusals")
    x = torch.zeros(8, device="cuda")
    for kw in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(seed=-1), dict(seed=2 ** 64), dict(stream=-1),
               dict(stream=2 ** 64), dict(x=x.cpu()), dict(x=x.double()), dict(seed=torch.zeros(1, device="cuda")),
               dict(seed=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(seed=torch.zeros(1, dtype=torch.int64))):
        args = {**dict(x=x, p=0.5, seed=1, stream=0), **kw}
        with pytest.raises(ValueError):
            k.dropout(args["x"], args["p"], args["seed"], args["stream"])


def test_norm_and_dropout_on_a_side_stream_and_captured(k):
    from lazylora_amd.native import NORM_LAYER
    case("norm: stream, graph")
    x, dy = torch.randn(700, 1000, device="cuda").bfloat16(), torch.randn(700, 1000, device="cuda").bfloat16()
    w = torch.rand(1000, device="cuda") + 0.5

    def step():
        y, st = k.norm_forward(x, w, None, 1e-5, NORM_LAYER, True)
        return (y,) + k.norm_backward(dy, x, w, st, NORM_LAYER, True, True) + (k.dropout(y, 0.1, 3),)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        x.copy_(torch.randn(700, 1000, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


# rows enough that every work-group of the backward takes several, a last pass of fewer rows than teams among
# them: more than 16384 rows up to width 128, 4096 up to 512, 1024 up to 2048, 512 up to 4096, 256 above
MANY_ROWS = [(16400, 64), (33000, 127), (4101, 300), (8200, 512), (1030, 2048), (3001, 1000), (1000, 3584), (1600, 2049),
             (600, 4100), (700, 8192), (260, 8200), (515, 16384), (520, 16400), (1100, 16385)]


@pytest.mark.parametrize("M,D", MANY_ROWS)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layer", [0, 1])
def test_norm_many_rows(k, M, D, dt, layer):
    case("norm, many rows", M, D, dt, "layer" if layer else "rms")
    g = torch.Generator(device="cuda").manual_seed(M + D)
    x = (torch.randn(M, D, device="cuda", generator=g) * 2 + 0.5).to(dt)
    w = 1 + 0.2 * torch.randn(D, device="cuda", generator=g)
    b = 0.3 * torch.randn(D, device="cuda", generator=g) if layer else None
    dy = torch.randn(M, D, device="cuda", generator=g).to(dt)
    (y, ey), (dx, edx), (dw, edw), (db, edb) = norm_reference(x, w, b, dy, layer, 1e-5)
    got, stats = k.norm_forward(x, w, b, 1e-5, layer, save_for_backward=True)
    check("y", got, y, ey)
    gx, gw, gb = k.norm_backward(dy, x, w, stats, layer, need_weight=True, need_bias=True)
    check("dx", gx, dx, edx)
    check("dw", gw, dw, edw)
    check("db", gb, db, edb)
    gx2, gw2, none = k.norm_backward(dy, x, w, stats, layer, need_weight=True)
    assert none is None and torch.equal(gx, gx2) and torch.equal(gw, gw2)
    plain, none, _ = k.norm_backward(dy, x, None, stats, layer)  # no weight, no column sums
    (_, _), (dx1, edx1), _, _ = norm_reference(x, None, b, dy, layer, 1e-5)
    check("dx without a weight", plain, dx1, edx1)
    assert none is None
