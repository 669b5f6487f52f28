"""The dense operators as programs use them: a whole training step captured into a graph, two streams at
once, offsets past 32 bits, strided weights, expanded gradients, saved tensors changed in between."""
import pytest
import torch

from tests.test_gpu_dense_ffn import check, inputs, reference
from tests.test_gpu_norm_dropout import philox7

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


def case(*a):
    print("\n[case]", *a, flush=True)


def block(t, seed):
    """Norm, dropout, feed-forward with deltas, residual: one step's outputs and gradients."""
    from lazylora_amd.dense import dropout, gated_ffn, layer_norm, rms_norm
    xn = rms_norm(t["x"], t["w"])
    y, h = gated_ffn(dropout(xn, 0.1, t["seed"], 1), t["wg"], t["wu"], t["wd"], "situ", t["gd"], t["ud"], True)
    z = layer_norm(y + t["x"], t["w"], t["b"])
    leaves = [t[n] for n in ("x", "w", "b", "wg", "wu", "wd", "gd", "ud")]
    grads = torch.autograd.grad((z, h), leaves, (t["dy"], t["dh"]))
    return (z.detach(), h.detach()) + grads  # no graph of the leaves outlives the step


def tensors(seed, M, D, F, dt=torch.bfloat16):
    t = inputs(seed, M, D, F, D, dt)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t["w"], t["b"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g), 0.1 * torch.randn(D, device="cuda", generator=g)
    t["seed"] = torch.tensor([seed], device="cuda")
    for n in ("x", "w", "b", "wg", "wu", "wd", "gd", "ud"):
        t[n].requires_grad_(True)
    return t


@pytest.mark.parametrize("M", [3, 200])
def test_captured_training_step(k, M):
    """Forward and backward through autograd in one graph, replayed with new inputs and seeds between eager
    steps; every replay equals the eager step."""
    case("captured step", M)
    t = tensors(5, M, 520, 264)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(t, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block(t, 1)
    for r in range(4):
        with torch.no_grad():
            t["x"].copy_(torch.randn_like(t["x"], dtype=torch.float32))
            t["dy"].neg_()
            t["seed"].add_(17)
        graph.replay()
        torch.cuda.synchronize()
        want = block(t, 1)
        for i, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), f"replay {r}, output {i}"


def test_two_streams_at_once(k):
    case("two streams")
    ts = [tensors(6, 300, 776, 264), tensors(7, 40, 776, 264)]
    want = [block(t, 1) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(block(ts[i], 1))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_strided_and_expanded(k):
    """Transposed weights, sliced deltas and a sum's expanded gradient give what their copies give."""
    from lazylora_amd.dense import gated_ffn, rms_norm
    case("strides")
    t = inputs(8, 30, 72, 40, 48, torch.float16)
    wide = torch.randn(30, 80, device="cuda").half()
    wgt = t["wg"].T.contiguous().T  # column-major storage
    x = t["x"].clone().requires_grad_(True)
    y = gated_ffn(x, wgt, t["wu"], t["wd"], gate_delta=wide[:, ::2])
    y2 = gated_ffn(x, t["wg"], t["wu"], t["wd"], gate_delta=wide[:, ::2].contiguous())
    assert torch.equal(y, y2)
    (g,) = torch.autograd.grad(y.sum(), (x,))
    (g2,) = torch.autograd.grad(y2, (x,), torch.ones_like(y2))
    assert torch.equal(g, g2)
    odd = torch.randn(31 * 33 + 1, device="cuda").half()[1:].view(31, 33)  # starts at an odd element
    assert torch.equal(rms_norm(odd), rms_norm(odd.clone()))


def test_saved_tensors_are_guarded(k):
    """Changing in place what a backward will read raises instead of giving a wrong gradient."""
    from lazylora_amd.dense import gated_ffn, rms_norm
    case("saved tensors")
    t = inputs(9, 8, 64, 32, 48, torch.bfloat16)
    wu = t["wu"].clone().requires_grad_(True)
    for change in ("x", "wd"):
        y = gated_ffn(t["x"], t["wg"], wu, t["wd"])
        t[change].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda")
    y = rms_norm(x, w)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_offsets_past_32_bits(k):
    """More elements than 32 bits count: the last rows against a call on them alone, or the formula."""
    from lazylora_amd.dense import dropout
    case("dropout of 2^32 + 13 elements")
    n = 2 ** 32 + 13
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.5, 99, 3)
    for first in (2 ** 31 - 20, 2 ** 32 - 20, n - 30):
        keep = torch.tensor([philox7(i, 99, 3) >= 2 ** 31 for i in range(first, first + 30)], device="cuda")
        assert torch.equal(y[first:first + 30] != 0, keep)
    del x, y
    case("norm of 300,001 rows of 7168")
    M, D = 300001, 7168
    x = torch.randn(M, D, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(D, device="cuda")
    y, st = k.norm_forward(x, w, None, 1e-5, 1, True)
    tail, st2 = k.norm_forward(x[-600:].contiguous(), w, None, 1e-5, 1, True)  # as many rows: the same kernel
    assert torch.equal(y[-600:], tail) and torch.equal(st[:, -600:], st2)
    dx, _, _ = k.norm_backward(y, x, w, st, 1)
    dx2, _, _ = k.norm_backward(tail, x[-600:].contiguous(), w, st2, 1)
    assert torch.equal(dx[-600:], dx2)
    del x, y, dx
    case("feed-forward block of 1,100,003 rows, 2 x 1024 hidden features")
    t = inputs(10, 1100003, 64, 1024, 72, torch.bfloat16)
    y, h, gu = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], "situ", t["gd"], t["ud"], save_for_backward=True)
    dgu, dx, *_ = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"], "situ", t["dh"])
    last = {**t, **{n: t[n][-300:].contiguous() for n in ("x", "dy", "dh", "gd", "ud")}}
    want = reference(last, "situ", True)
    for name, got in (("y", y), ("h", h), ("dg", dgu[:, :1024]), ("du", dgu[:, 1024:]), ("dx", dx)):
        check(name, got[-300:], want[name])


def test_gradients_not_asked_for_are_not_made(k):
    """A backward for some of the leaves allocates no gradient of the others: dx of a trainable block no weight
    gradients, a down weight alone no gradient of gate | up. What is asked for is what the whole backward gives."""
    from lazylora_amd.dense import gated_ffn
    case("gradients asked for")

    def peak(t, names):
        y = gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])
        whole = torch.autograd.grad(y, [t[n] for n in ("x", "wg", "wu", "wd")], t["dy"], retain_graph=True)
        whole = dict(zip(("x", "wg", "wu", "wd"), whole))
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, [t[n] for n in names], t["dy"])
        torch.cuda.synchronize()
        assert all(torch.equal(g, whole[n]) for g, n in zip(got, names)), names
        return torch.cuda.max_memory_allocated() - before

    def leaves(*sizes):
        t = inputs(12, *sizes, torch.bfloat16, deltas=False)
        for n in ("x", "wg", "wu", "wd"):
            t[n].requires_grad_(True)
        return t

    # 8 rows: dx and the split sums are small, a weight gradient 16 MiB
    t = leaves(8, 2048, 4096, 2048)
    assert peak(t, ["x"]) < 2 ** 24
    assert 2 ** 24 <= peak(t, ["x", "wd"]) < 2 ** 25
    # 4096 rows: gate | up's gradient is 32 MiB, the down weight's 1/4 MiB
    assert peak(leaves(4096, 64, 2048, 64), ["wd"]) < 2 ** 25


def test_one_optional_input_alone(k):
    """A bias without a weight, an up delta without a gate delta: each gradient goes to its own input."""
    from lazylora_amd.dense import gated_ffn, layer_norm
    case("optional inputs")
    x, dy = torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda")
    bias = torch.randn(40, device="cuda", requires_grad=True)
    for lead in (x, x.clone().requires_grad_(True)):
        y = layer_norm(lead, None, bias)
        (gb,) = torch.autograd.grad(y, (bias,), dy, retain_graph=True)
        assert ((gb.double() - dy.double().sum(0)).abs() <= 8 * 2.0 ** -24 * dy.double().abs().sum(0)).all()
        assert torch.equal(y.detach(), layer_norm(x, torch.ones(40, device="cuda"), bias.detach()))
    t = inputs(13, 20, 72, 40, 48, torch.bfloat16)
    t["ud"].requires_grad_(True)
    want = reference({**{n: v.detach() for n, v in t.items()}, "gd": None}, "situ", False)
    y = gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], "situ", None, t["ud"])
    check("y", y.detach(), want["y"])
    (gu,) = torch.autograd.grad(y, (t["ud"],), t["dy"])
    check("du", gu, want["du"])


def test_negative_views(k):
    """The imaginary part of a conjugate is a view that stands for its negative: read with its sign, of inputs,
    weights and upstream gradients (of one element such a view is contiguous and is not copied first)."""
    from lazylora_amd.dense import dropout, layer_norm, rms_norm
    case("negative views")
    z = lambda *s: torch.randn(*s, dtype=torch.cfloat, device="cuda").conj().imag
    for shape in ((1, 1), (1,), (3, 8)):
        x, plain = z(*shape), None
        plain = x.resolve_neg().clone()
        assert x.is_neg() and not plain.is_neg()
        w = z(shape[-1])
        wp = w.resolve_neg().clone()
        assert torch.equal(dropout(x, 0.0, 1), plain)
        assert torch.equal(k.dropout(x, 0.0, 1), plain)
        assert torch.equal(rms_norm(x, w), rms_norm(plain, wp))
        assert torch.equal(layer_norm(x, w, w), layer_norm(plain, wp, wp))
        leaf = torch.randn(*shape, device="cuda", requires_grad=True)
        for fn in (lambda v: dropout(v, 0.0, 1), lambda v: rms_norm(v, w, 0.1)):
            (got,) = torch.autograd.grad(fn(leaf), (leaf,), x)
            (want,) = torch.autograd.grad(fn(leaf), (leaf,), plain)
            assert torch.equal(got, want)
        if len(shape) == 2:
            y, st = k.norm_forward(x, w.resolve_neg(), None, 0.1, 0, True)
            assert torch.equal(y, rms_norm(plain, wp, 0.1))
            assert torch.equal(k.norm_backward(x, plain, wp, st)[0], k.norm_backward(plain, plain, wp, st)[0])
            assert torch.equal(k.norm_backward(plain, x, w, st)[0], k.norm_backward(plain, plain, wp, st)[0])
