"""The gated feed-forward block's kernels against its formulas in float64, element by element.

The bound of each element is what the roundings can add up to: u = eps / 2 of the type per rounding to
16 bits, 2^-24 per fp32 term of a sum, 2e-6 relative for an activation function (its exponential,
reciprocal and products), carried through the formulas with absolute values."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(1, 8, 8, 8), (1, 64, 16, 24), (2, 4096, 128, 4096), (3, 72, 40, 56), (16, 512, 256, 512), (17, 200, 136, 264),
         (33, 1032, 392, 72), (64, 2048, 512, 1024), (128, 128, 128, 128), (129, 264, 392, 136), (257, 640, 264, 520),
         (300, 1032, 72, 64), (515, 328, 776, 1288)]


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


def case(*a):
    print("\n[case]", *a, flush=True)


def inputs(seed, M, D, F, Do, dt, deltas=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)
    t = {"x": r(M, D), "wg": r(F, D) / D ** 0.5, "wu": r(F, D) / D ** 0.5, "wd": r(Do, F) / F ** 0.5, "dy": r(M, Do),
         "dh": r(M, F), "gd": r(M, F), "ud": r(M, F)}
    t = {n: v.to(dt) for n, v in t.items()}
    if not deltas:
        t["gd"] = t["ud"] = None
    return t


def act64(g, u, act):
    if act == "swiglu":
        return g * torch.sigmoid(g) * u
    return 4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25)


def reference(t, act, grad_h):
    """float64 values and element bounds of every output."""
    dt = t["x"].dtype
    u_, s_ = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    d = {n: None if v is None else v.double() for n, v in t.items()}
    x, wg, wu, wd, dy = d["x"], d["wg"], d["wu"], d["wd"], d["dy"]
    M, D = x.shape
    F, Do = wg.shape[0], wd.shape[0]
    f = 2.0 ** -24
    gd, ud = d["gd"] if d["gd"] is not None else 0, d["ud"] if d["ud"] is not None else 0
    g, u = (x @ wg.T + gd).requires_grad_(True), (x @ wu.T + ud).requires_grad_(True)
    h = act64(g, u, act)
    hg, hu = torch.autograd.grad(h.sum(), (g, u))
    g, u, h = g.detach(), u.detach(), h.detach()
    eg = (D + 2) * f * (x.abs() @ wg.abs().T + (gd.abs() if torch.is_tensor(gd) else 0))
    eu = (D + 2) * f * (x.abs() @ wu.abs().T + (ud.abs() if torch.is_tensor(ud) else 0))
    eh = hg.abs() * eg + hu.abs() * eu + 2e-6 * h.abs() + u_ * h.abs() + s_
    y = h @ wd.T
    ey = eh @ wd.abs().T + (F + 2) * f * (h.abs() @ wd.abs().T) + u_ * y.abs() + s_
    dh = dy @ wd + (d["dh"] if grad_h else 0)
    edh = (Do + 2) * f * (dy.abs() @ wd.abs() + (d["dh"].abs() if grad_h else 0))
    dg, du = dh * hg, dh * hu
    # second derivatives of both activations stay below 1 + |g| + |u|; the derivative's factors are sums of
    # terms up to (1 + |g|)(1 + |u|) in size
    second = (1 + g.abs() + u.abs()) * (eg + eu) + 2e-6 * (1 + g.abs()) * (1 + u.abs())
    edg = edh * hg.abs() + dh.abs() * second + u_ * dg.abs() + s_
    edu = edh * hu.abs() + dh.abs() * second + u_ * du.abs() + s_
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + (2 * F + 2) * f * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) \
        + u_ * dx.abs() + s_
    dwg, dwu, dwd = dg.T @ x, du.T @ x, dy.T @ h
    grow = lambda e, v, b, w: e.T @ b.abs() + (M + 2) * f * (v.abs().T @ b.abs()) + u_ * w.abs() + s_
    out = {"y": (y, ey), "h": (h, eh), "dg": (dg, edg), "du": (du, edu), "dx": (dx, edx),
           "dwg": (dwg, grow(edg, dg, x, dwg)), "dwu": (dwu, grow(edu, du, x, dwu)),
           "dwd": (dwd, dy.abs().T @ eh + (M + 2) * f * (dy.abs().T @ h.abs()) + u_ * dwd.abs() + s_)}
    return out


def check(name, got, want):
    v, bound = want
    assert got.shape == v.shape, name
    over = ((got.double() - v).abs() / bound.clamp_min(1e-300))
    assert not torch.isnan(over).any(), f"{name}: NaN"
    worst = over.max().item() if over.numel() else 0.0
    print(f"{name}: largest error {worst:.3f} of its bound")
    assert worst <= 1.0, f"{name}: an element is {worst:.2f} times its bound off"


@pytest.mark.parametrize("M,D,F,Do", SIZES)
@pytest.mark.parametrize("act,dt", [("swiglu", torch.bfloat16), ("situ", torch.bfloat16), ("swiglu", torch.float16),
                                    ("situ", torch.float16)])
def test_forward_and_backward(k, M, D, F, Do, act, dt):
    case("ffn", M, D, F, Do, act, dt)
    t = inputs(M + D, M, D, F, Do, dt)
    want = reference(t, act, True)
    y, h, gu = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], act, t["gd"], t["ud"], save_for_backward=True)
    check("y", y, want["y"])
    check("h", h, want["h"])
    dgu, dx, dwg, dwu, dwd = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"], act, t["dh"], t["x"], h,
                                            need_w_in=True, need_w_down=True)
    for name, got in (("dg", dgu[:, :F]), ("du", dgu[:, F:]), ("dx", dx), ("dwg", dwg), ("dwu", dwu), ("dwd", dwd)):
        check(name, got, want[name])


@pytest.mark.parametrize("M,D,F,Do", [(4099, 520, 2056, 4104), (2050, 328, 1544, 2312), (1100, 1032, 776, 3080),
                                      (700, 2056, 392, 1544), (3330, 2568, 4104, 2056), (1000, 7176, 520, 1544),
                                      (1000, 1032, 2056, 264), (4096, 264, 2056, 7176), (9, 264, 2056, 4104),
                                      (25, 136, 2056, 4104), (40, 264, 2056, 4104), (60, 328, 2056, 4104)])
@pytest.mark.parametrize("act,dt", [("situ", torch.bfloat16), ("swiglu", torch.float16)])
def test_large_tiles(k, M, D, F, Do, act, dt):
    """Sizes that the large tiles take, whole and cut, with ragged last rows, columns and steps, and wide
    products of few rows."""
    case("large", M, D, F, Do, act, dt)
    t = inputs(M, M, D, F, Do, dt)
    want = reference(t, act, True)
    y, h, gu = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], act, t["gd"], t["ud"], save_for_backward=True)
    check("y", y, want["y"])
    check("h", h, want["h"])
    dgu, dx, dwg, dwu, dwd = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"], act, t["dh"], t["x"], h,
                                            need_w_in=True, need_w_down=True)
    for name, got in (("dg", dgu[:, :F]), ("du", dgu[:, F:]), ("dx", dx), ("dwg", dwg), ("dwu", dwu), ("dwd", dwd)):
        check(name, got, want[name])


@pytest.mark.parametrize("M", [1, 5, 16, 31, 48, 63, 65, 96, 127, 130, 191, 200, 255, 384])
def test_every_row_count(k, M):
    """The row count decides which kernel runs; no deltas, no grad_h, frozen weights."""
    D, F, Do = 776, 264, 520
    case("rows", M)
    t = inputs(M, M, D, F, Do, torch.bfloat16, deltas=False)
    want = reference(t, "swiglu", False)
    y, h, gu = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], save_for_backward=True)
    y2, h2, none = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"])
    assert none is None and torch.equal(y, y2) and torch.equal(h, h2)  # keeping gate | up changes nothing
    check("y", y, want["y"])
    dgu, dx, *rest = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"])
    assert rest == [None, None, None]
    check("dx", dx, want["dx"])
    again = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"])
    assert torch.equal(dx, again[1]) and torch.equal(dgu, again[0])


def test_autograd_against_differences(k):
    """Every gradient against central differences of the float64 block along random directions: the
    difference's own error at step 1e-5 is below 1e-8 of values of order 1; the gradients' roundings stay
    below the element bounds summed along the direction."""
    from lazylora_amd.dense import gated_ffn
    for act in ("swiglu", "situ"):
        case("differences", act)
        t = inputs(7, 37, 136, 72, 104, torch.bfloat16)
        leaves = {n: t[n].requires_grad_(True) for n in ("x", "wg", "wu", "wd", "gd", "ud")}
        y, h = gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], act, t["gd"], t["ud"], return_hidden=True)
        grads = dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (t["dy"], t["dh"]))))
        d = {n: v.detach().double() for n, v in t.items()}

        def loss(**moved):
            v = {**d, **moved}
            hh = act64(v["x"] @ v["wg"].T + v["gd"], v["x"] @ v["wu"].T + v["ud"], act)
            return ((hh @ v["wd"].T) * d["dy"]).sum() + (hh * d["dh"]).sum()

        bounds = reference({n: v.detach() for n, v in t.items()}, act, True)
        names = {"x": "dx", "wg": "dwg", "wu": "dwu", "wd": "dwd", "gd": "dg", "ud": "du"}
        for n in leaves:
            dirn = torch.randn(d[n].shape, dtype=torch.float64, device="cuda",
                               generator=torch.Generator(device="cuda").manual_seed(3))
            diff = (loss(**{n: d[n] + 1e-5 * dirn}) - loss(**{n: d[n] - 1e-5 * dirn})) / 2e-5
            got = (grads[n].double() * dirn).sum()
            slack = (bounds[names[n]][1] * dirn.abs()).sum() + 1e-6 * diff.abs() + 1e-6
            print(n, got.item(), diff.item(), "slack", slack.item())
            assert (got - diff).abs() <= slack, n


def test_autograd_partial_needs(k):
    """Only what needs a gradient gets one; h's gradient alone; higher axes; strided inputs."""
    from lazylora_amd.dense import gated_ffn
    case("partial needs")
    t = inputs(11, 24, 64, 48, 40, torch.float16)
    x3 = t["x"].reshape(2, 12, 64).transpose(0, 1)  # not contiguous
    y0 = gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])
    y3 = gated_ffn(x3, t["wg"], t["wu"], t["wd"])
    assert y3.shape == (12, 2, 40) and torch.equal(y3.transpose(0, 1).reshape(24, 40), y0)
    assert not y0.requires_grad
    wu = t["wu"].clone().requires_grad_(True)
    y = gated_ffn(t["x"], t["wg"], wu, t["wd"])
    (g,) = torch.autograd.grad(y, (wu,), t["dy"])
    check("dwu alone", g, reference({**t, "gd": None, "ud": None}, "swiglu", False)["dwu"])
    x = t["x"].clone().requires_grad_(True)
    _, h = gated_ffn(x, t["wg"], t["wu"], t["wd"], return_hidden=True)
    (gx,) = torch.autograd.grad(h, (x,), t["dh"])
    zero = {**t, "gd": None, "ud": None, "dy": torch.zeros_like(t["dy"])}
    check("dx from h alone", gx, reference(zero, "swiglu", True)["dx"])
    yy = gated_ffn(x, t["wg"], t["wu"], t["wd"])
    (g1,) = torch.autograd.grad(yy, (x,), torch.ones_like(yy), create_graph=True)
    with pytest.raises(RuntimeError):
        g1.sum().backward()


def test_no_rows(k):
    from lazylora_amd.dense import gated_ffn
    case("no rows")
    t = inputs(1, 0, 64, 32, 48, torch.bfloat16, deltas=False)
    for n in ("x", "wg", "wu", "wd"):
        t[n].requires_grad_(True)
    y = gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])
    assert y.shape == (0, 48)
    gx, gg, gu, gd = torch.autograd.grad(y, [t[n] for n in ("x", "wg", "wu", "wd")], torch.empty_like(y))
    assert gx.shape == (0, 64) and not gg.any() and not gu.any() and not gd.any()


@pytest.mark.parametrize("M", [1, 40, 130])
def test_rows_behind_the_last_are_left(k, M):
    """Through the C ABI, outputs with rows to spare: those keep what they held."""
    D, F, Do = 136, 72, 200
    case("spare rows", M)
    lib = k.lib
    t = inputs(5, M, D, F, Do, torch.bfloat16)
    mark = 123.0
    buf = lambda n, w, dt=torch.bfloat16: torch.full((n + 3, w), mark, dtype=dt, device="cuda")
    y, h, gu, dgu, dx = buf(M, Do), buf(M, F), buf(M, 2 * F, torch.float32), buf(M, 2 * F), buf(M, D)
    dw = [buf(F, D), buf(F, D), buf(Do, F)]
    n = lib.mxfp4_ffn_workspace_size(M, D, F, Do)
    ws = torch.full((n + 256,), 77, dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    p = lambda v: v.data_ptr()
    w = [p(t[q]) for q in ("wg", "wu", "wd")]
    assert lib.mxfp4_ffn_forward(p(y), p(h), p(gu), p(t["x"]), *w, p(t["gd"]), p(t["ud"]), 1, M, D, F, Do, 1, p(ws), n,
                                 s) == 0
    assert lib.mxfp4_ffn_backward(p(dx), *[p(v) for v in dw], p(dgu), p(t["dy"]), p(t["dh"]), p(t["x"]), p(h), p(gu), *w,
                                  1, M, D, F, Do, 1, p(ws), n, s) == 0
    torch.cuda.synchronize()
    for v in (y, h, gu, dgu, dx, *dw):
        assert (v[-3:] == mark).all()
    assert (ws[n:] == 77).all()
    want = reference(t, "situ", True)
    check("y", y[:M], want["y"])
    check("dx", dx[:M], want["dx"])
    check("dwd", dw[2][:Do], want["dwd"])


def test_special_values(k):
    """Infinities and NaN stay in their rows (and reach that row's outputs); others are untouched."""
    case("special values")
    M, D, F, Do = 70, 136, 72, 40
    t = inputs(3, M, D, F, Do, torch.bfloat16, deltas=False)
    y0, _, _ = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"])
    x = t["x"].clone()
    x[5, 135], x[69, 0] = float("nan"), float("inf")
    y, _, _ = k.ffn_forward(x, t["wg"], t["wu"], t["wd"])
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[5] = keep[69] = False
    assert torch.equal(y[keep], y0[keep])
    assert torch.isnan(y[5]).all() and not torch.isfinite(y[69]).all()


def test_other_stream_and_graph(k):
    """On a side stream, and captured: replays with changed inputs equal the eager call, with eager work and
    synchronisations between them."""
    from lazylora_amd.dense import gated_ffn
    case("stream and graph")
    for M in (1, 40, 300):
        t = inputs(9, M, 520, 264, 392, torch.bfloat16)
        eager = lambda: k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], "situ", t["gd"], t["ud"], True)

        def step():
            y, h, gu = eager()
            return (y, h, gu) + k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"], "situ", t["dh"], t["x"], h,
                                               need_w_in=True, need_w_down=True)

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
        for r in range(4):
            t["x"].copy_(torch.randn_like(t["x"].float()).to(torch.bfloat16))
            t["dy"].mul_(-1)
            graph.replay()
            torch.cuda.synchronize()
            want = step()
            gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])  # eager work between replays
            assert all(torch.equal(a, b) for a, b in zip(held, want)), f"replay {r} of {M} rows"


def test_refusals(k):
    from lazylora_amd.dense import gated_ffn
    case("refusals")
    t = inputs(2, 4, 64, 32, 48, torch.bfloat16)
    ok = dict(x=t["x"], w_gate=t["wg"], w_up=t["wu"], w_down=t["wd"])
    bad = [dict(x=t["x"].float()), dict(x=t["x"].cpu()), dict(w_gate=t["wg"].half()), dict(w_up=t["wu"][:, :56]),
           dict(w_down=t["wd"].T), dict(act="gelu"), dict(gate_delta=t["gd"].float()), dict(up_delta=t["ud"][:3]),
           dict(w_gate=t["wg"][:30], w_up=t["wu"][:30]), dict(x=t["x"][:, :63]), dict(w_down=t["wd"].cpu()),
           dict(x=torch.zeros((), device="cuda", dtype=torch.bfloat16))]
    for change in bad:
        with pytest.raises(ValueError):
            gated_ffn(**{**ok, **change})
    y, h, gu = k.ffn_forward(*ok.values(), save_for_backward=True)
    w = list(ok.values())[1:]
    for kw in (dict(gu=gu.bfloat16()), dict(gu=gu[:3]), dict(grad_y=t["dy"].float()), dict(grad_y=t["dy"][:, :40]),
               dict(grad_h=t["dh"].float()), dict(need_w_in=True), dict(need_w_down=True),
               dict(need_w_down=True, h=h[:3])):
        args = {**dict(grad_y=t["dy"], gu=gu, w_gate=w[0], w_up=w[1], w_down=w[2]), **kw}
        with pytest.raises(ValueError):
            k.ffn_backward(**args)
