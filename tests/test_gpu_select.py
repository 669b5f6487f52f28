"""Expert selection with softmax or sigmoid scores and groups against its definition in 64 bits, forward and
backward. Indices are compared for equality: the order is that of exact arithmetic."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def select():
    from lazylora_amd.router import select_experts
    return select_experts


def oracle_scores(x, scoring):
    """x float64 [N, E] -> scores; a row without a finite logit has softmax scores 0."""
    with np.errstate(over="ignore", invalid="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-x))
        top = x.max(1, keepdims=True)
        e = np.exp(x - np.where(top == -np.inf, 0, top))
        total = e.sum(1, keepdims=True)
        return e / np.where(total == 0, 1, total)


def largest_first(v):
    """Positions along the last axis in descending order, NaN first, ties by position."""
    nan = np.isnan(v)
    return np.lexsort((-np.where(nan, 0, v), ~nan), axis=-1)


def oracle_select(x, top_k, bias=None, scoring="sigmoid", num_groups=1, topk_groups=None, group_score="top2",
                  renormalize=True, routed_scaling_factor=1.0):
    x = x.astype(np.float64)
    N, E = x.shape
    s = oracle_scores(x, scoring)
    choice = x if bias is None else s + bias.astype(np.float64)
    kept = num_groups if topk_groups is None else topk_groups
    size = E // num_groups
    idx = np.empty((N, top_k), np.int64)
    for t in range(N):
        groups = choice[t].reshape(num_groups, size)
        if group_score == "max":
            nan = np.isnan(groups).any(1)
            value = np.where(nan, np.nan, groups.max(1))
        else:
            g = (s[t] if bias is None else choice[t]).reshape(num_groups, size)
            first = np.take_along_axis(g, largest_first(g), 1)[:, :2]
            value = first.sum(1)
        on = np.sort(largest_first(value)[:kept])
        ids = (on[:, None] * size + np.arange(size)).ravel()
        idx[t] = ids[largest_first(choice[t][ids])[:top_k]]
    w = np.take_along_axis(s, idx, 1)
    if renormalize and top_k > 1:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return idx, w * routed_scaling_factor


# Relative error of a weight, in steps of 2^-24: the exponential and its argument (the argument's own rounding
# moves it by |x - max| <= 32 steps wherever the score is not negligible), the sum of up to 64 + 7 terms in a row,
# the quotients, the sum of up to 64 chosen scores: below 256.
W_TOL = 256 * 2.0 ** -24


def run(select, x, dtype, bias, **kw):
    t = torch.from_numpy(x).cuda().to(DTYPES[dtype])
    b = None if bias is None else torch.from_numpy(bias).cuda()
    idx, w = select(t, bias=b, **kw)
    assert idx.dtype == torch.int64 and w.dtype == torch.float32
    want_i, want_w = oracle_select(t.float().cpu().numpy(), bias=None if bias is None else bias, **kw)
    got_i, got_w = idx.cpu().numpy(), w.cpu().numpy()
    np.testing.assert_array_equal(got_i, want_i)
    # scores below the smallest normal numbers are off by steps of their own
    np.testing.assert_allclose(got_w, want_w, rtol=W_TOL, atol=1e-18)
    return idx, w


CASES = [  # N, E, top_k, groups, kept
    (1, 8, 2, 1, 1), (3, 1, 1, 1, 1), (5, 2, 2, 2, 2), (7, 60, 6, 1, 1), (33, 64, 8, 8, 3), (9, 256, 8, 8, 4),
    (4, 257, 5, 1, 1), (6, 84, 7, 7, 3), (5, 84, 7, 12, 5), (3, 896, 16, 1, 1), (3, 896, 16, 7, 3), (2, 1024, 64, 4, 1),
    (2, 4096, 64, 1, 1), (2, 4096, 3, 64, 9), (3, 64, 4, 64, 4), (2, 2046, 9, 33, 5), (65, 33, 33, 1, 1), (3, 70, 70 // 2, 5, 3),
]


@pytest.mark.parametrize("N,E,top_k,groups,kept", CASES)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_against_definition(select, N, E, top_k, groups, kept, scoring, with_bias):
    rng = np.random.default_rng(E + 7 * top_k)
    for dtype in DTYPES:
        for group_score in ("top2", "max") if groups > 1 else ("top2",):
            x = (1.5 * rng.standard_normal((N, E))).astype(np.float32)
            bias = (0.1 * rng.standard_normal(E)).astype(np.float32) if with_bias else None
            run(select, x, dtype, bias, top_k=top_k, scoring=scoring, num_groups=groups, topk_groups=kept,
                group_score=group_score, renormalize=dtype != "f16", routed_scaling_factor=2.5)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3), (7, 3)])
def test_many_tokens_are_ordered_exactly(select, scoring, groups, kept):
    """Enough tokens for neighbours that 32-bit sums of score and bias cannot tell apart."""
    rng = np.random.default_rng(5)
    E = 56 * 8
    x = rng.standard_normal((6000, E)).astype(np.float32)
    bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
    run(select, x, "f32", bias, top_k=16, scoring=scoring, num_groups=groups, topk_groups=kept)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("ulps", [0, 1, 3])
def test_neighbours_closer_than_32_bits(select, scoring, ulps):
    """Experts whose score + bias agree to 32 bits and differ behind them: pairs, and runs longer than top_k and
    longer than a wave."""
    rng = np.random.default_rng(11)
    for E, run_len, groups in ((64, 2, 1), (64, 12, 1), (256, 100, 1), (256, 100, 4), (256, 250, 8), (66, 20, 3)):
        x = rng.standard_normal((4, E)).astype(np.float32)
        bias = np.zeros(E, np.float32)
        at = rng.permutation(E)[:run_len]
        for t in range(4):
            v = np.float32(2.0 + t / 8)
            steps = rng.integers(0, ulps + 1, run_len)
            x[t, at] = v + steps.astype(np.float32) * np.spacing(v)
        bias[rng.permutation(E)[:5]] = 2.0 ** -27
        for kept in {1, max(1, groups // 2), groups}:
            for group_score in ("top2", "max"):
                run(select, x, "f32", bias, top_k=6, scoring=scoring, num_groups=groups, topk_groups=kept,
                    group_score=group_score)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_equal_values_and_masks(select, scoring, with_bias):
    """Rows of one value, masked experts (-inf, the type's lowest value), rows with nothing left, infinities and
    NaN; biases that switch experts off."""
    rng = np.random.default_rng(3)
    for E, groups, kept, k in ((64, 1, 1, 6), (64, 8, 3, 6), (896, 7, 2, 16), (60, 12, 12, 60)):
        rows = [np.zeros(E), np.full(E, -np.inf), np.full(E, np.finfo(np.float32).min), np.full(E, np.nan),
                np.where(np.arange(E) == E // 2, 1.0, -np.inf), np.where(np.arange(E) % 3 == 0, -np.inf, 0.5),
                np.where(np.arange(E) % 5 == 0, np.finfo(np.float32).min, rng.standard_normal(E)),
                np.where(np.arange(E) == 3, np.nan, rng.standard_normal(E)),
                np.where(np.arange(E) == E - 2, np.inf, rng.standard_normal(E)), np.full(E, -200.0), np.full(E, 200.0),
                rng.integers(-2, 3, E).astype(np.float64)]
        x = np.stack(rows).astype(np.float32)
        biases = [None]
        if with_bias:
            b = (0.1 * rng.standard_normal(E)).astype(np.float32)
            off = b.copy()
            off[::4] = -np.inf
            biases = [np.zeros(E, np.float32), b, off, np.full(E, 3.0, np.float32)]
        for bias in biases:
            for group_score in ("top2", "max"):
                run(select, x, "f32", bias, top_k=k if k < E else kept * (E // groups), scoring=scoring,
                    num_groups=groups, topk_groups=kept, group_score=group_score)


def grad64(x, dw, idx, scoring, renormalize, scale):
    t = torch.from_numpy(x.astype(np.float64)).requires_grad_(True)
    s = (t.sigmoid() if scoring == "sigmoid" else t.softmax(1)).gather(1, idx)
    w = scale * (s / (s.sum(1, True) + 1e-20) if renormalize and idx.shape[1] > 1 else s)
    return torch.autograd.grad(w, t, dw.double())[0].numpy()


@pytest.mark.parametrize("N,E,top_k", [(1, 1, 1), (5, 8, 1), (37, 60, 6), (9, 256, 8), (3, 896, 16), (2, 4096, 64), (4, 7, 7)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_backward(select, N, E, top_k, scoring, renormalize):
    rng = np.random.default_rng(E)
    for dtype, dt in DTYPES.items():
        t = torch.from_numpy((1.5 * rng.standard_normal((N, E))).astype(np.float32)).cuda().to(dt).requires_grad_(True)
        dw = torch.from_numpy(rng.standard_normal((N, top_k)).astype(np.float32))
        idx, w = select(t, top_k, scoring=scoring, renormalize=renormalize, routed_scaling_factor=1.5)
        got = torch.autograd.grad(w, t, dw.cuda())[0]
        assert got.dtype == dt and got.shape == t.shape
        want = grad64(t.detach().float().cpu().numpy(), dw, idx.cpu(), scoring, renormalize, 1.5)
        # a result is a score times a difference of terms: their errors, as W_TOL, count against the terms' size; one
        # rounding to the logits' type
        s = oracle_scores(t.detach().float().cpu().numpy().astype(np.float64), scoring)
        chosen = np.take_along_axis(s, idx.cpu().numpy(), 1)
        size = 1.5 * np.abs(dw.numpy()).max(1, keepdims=True) / (chosen.sum(1, keepdims=True) if renormalize else 1)
        bound = 4 * W_TOL * 2 * s * size + torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -25
        assert (np.abs(got.float().cpu().numpy() - want) <= bound).all()


def test_backward_against_differences(select):
    """The gradient of a weighted sum of the weights along a direction, against the forward on both sides of the
    logits, in steps that leave the choice as it is."""
    rng = np.random.default_rng(2)
    x = torch.from_numpy((3 * rng.permutation(40).reshape(4, 10) / 10).astype(np.float32)).cuda()
    v, c = torch.randn_like(x), torch.randn(4, 3, device="cuda")
    for scoring in ("sigmoid", "softmax"):
        for renorm in (False, True):
            t = x.clone().requires_grad_(True)
            _, w = select(t, 3, scoring=scoring, renormalize=renorm)
            slope = (torch.autograd.grad((w * c).sum(), t)[0] * v).sum().double().item()
            h = 2.0 ** -7
            f = lambda y: (select(y, 3, scoring=scoring, renormalize=renorm)[1] * c).sum().double().item()
            # truncation: h^2 / 6 times a third derivative of order 1 per element; rounding: 2^-22 / h
            assert abs((f(x + h * v) - f(x - h * v)) / (2 * h) - slope) < 2e-3


def test_masked_rows_have_finite_gradients(select):
    x = torch.full((3, 16), -torch.inf, device="cuda")
    x[1, 4] = 1.0
    x[2, ::2] = 0.25
    for scoring in ("sigmoid", "softmax"):
        t = x.clone().requires_grad_(True)
        idx, w = select(t, 4, scoring=scoring)
        g = torch.autograd.grad(w, t, torch.randn_like(w))[0]
        assert torch.isfinite(w).all() and torch.isfinite(g).all()
        assert (w[0] == 0).all() and (g[0] == 0).all()


def test_layouts_devices_and_empty_inputs(select):
    """Strided, broadcast and offset logits, leading axes, a 64-bit bias, no tokens, another stream."""
    base = torch.randn(6, 5, 130, device="cuda")
    x = base[::2, 1:, 1:129]
    idx, w = select(x, 4, scoring="softmax", num_groups=4, topk_groups=2)
    i2, w2 = select(x.contiguous().view(-1, 128), 4, scoring="softmax", num_groups=4, topk_groups=2)
    assert idx.shape == (3, 4, 4) and torch.equal(idx.view(-1, 4), i2) and torch.equal(w.view(-1, 4), w2)
    row = torch.randn(128, device="cuda")
    i3, _ = select(row.expand(5, 128), 4)
    assert torch.equal(i3, select(row, 4)[0].expand(5, 4))
    bias = torch.randn(128, device="cuda", dtype=torch.float64).float().double()
    assert torch.equal(select(row, 4, bias)[0], select(row, 4, bias.float())[0])
    e = torch.empty(0, 128, device="cuda", requires_grad=True)
    idx, w = select(e, 4, scoring="softmax")
    assert idx.shape == (0, 4) and torch.autograd.grad(w.sum(), e)[0].shape == (0, 128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = select(row, 4)
    s.synchronize()
    assert torch.equal(got[0], select(row, 4)[0])


def test_more_tokens_than_one_launch_takes(select):
    """2^25 tokens to a launch: the ones on both sides of the line, and the last, forward and backward."""
    N = 2 ** 25 + 5
    x = torch.zeros(N, 2, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, N - 1], device="cuda")
    x[at, 1] = 1.0
    x.requires_grad_(True)
    idx, w = select(x, 1, scoring="softmax", renormalize=False)
    want = torch.zeros(N, device="cuda", dtype=torch.int64)
    want[at] = 1
    assert torch.equal(idx[:, 0], want)
    hot = 1 / (1 + np.exp(-1.0))
    assert (w[at, 0] - hot).abs().max() < 1e-6 and int((w == 0.5).sum()) == N - len(at)
    g = torch.autograd.grad(w, x, torch.ones_like(w))[0]
    assert int((g == torch.tensor([0.25, -0.25], device="cuda").bfloat16()).all(1).sum()) == N - len(at)
    assert (g[at, 1].float() - hot * (1 - hot)).abs().max() < 2e-3


def test_refusals(select):
    x = torch.randn(3, 64, device="cuda")
    for kw in ({"top_k": 0}, {"top_k": 65}, {"top_k": 4, "num_groups": 5}, {"top_k": 4, "num_groups": 0},
               {"top_k": 4, "num_groups": 8, "topk_groups": 9}, {"top_k": 4, "num_groups": 8, "topk_groups": 0},
               {"top_k": 17, "num_groups": 8, "topk_groups": 2}, {"top_k": 2, "scoring": "tanh"},
               {"top_k": 2, "group_score": "mean"}, {"top_k": 2, "bias": torch.zeros(63, device="cuda")},
               {"top_k": 2, "bias": torch.zeros(64)}, {"top_k": 2, "bias": torch.zeros(64, device="cuda").long()},
               {"top_k": 2, "num_groups": 2 ** 40}):
        with pytest.raises(ValueError):
            select(x, **kw)
    for bad in (x.cpu(), x.double(), x.long(), torch.randn(3, 4097, device="cuda"), torch.randn((), device="cuda"),
                torch.empty(3, 0, device="cuda")):
        with pytest.raises(ValueError):
            select(bad, 1)
    with pytest.raises(ValueError):  # 33 groups of 124 do not fit the runs
        select(torch.randn(2, 33 * 124, device="cuda"), 2, num_groups=33, topk_groups=2)
    t = x.clone().requires_grad_(True)
    g = torch.autograd.grad(select(t, 4, scoring="softmax")[1].sum(), t, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


def test_router_options():
    """route, KimiK3MoERouter and the plain selection agree; the reference's form is the router's own kernel."""
    from lazylora_amd.router import KimiK3MoERouter, route, select_experts
    torch.manual_seed(0)
    r = KimiK3MoERouter(96, 64, 6, 2.5, device="cuda", scoring="softmax", num_groups=8, topk_groups=3, group_score="max")
    torch.nn.init.normal_(r.bias, std=0.02)
    x = torch.randn(11, 96, device="cuda", requires_grad=True)
    idx, w = r(x)
    logits = torch.nn.functional.linear(x, r.weight)
    i2, w2 = select_experts(logits, 6, r.bias, "softmax", 8, 3, "max", True, 2.5)
    assert torch.equal(idx, i2) and torch.equal(w, w2)
    w.sum().backward()
    assert torch.isfinite(x.grad).all() and x.grad.abs().sum() > 0 and r.weight.grad is not None
    old = route(x, r.weight, r.bias, 6)
    new = select_experts(logits, 6, r.bias)
    assert torch.equal(old[0], new[0]) and torch.allclose(old[1], new[1], rtol=1e-5)
    with pytest.raises(ValueError):
        route(x, r.weight, r.bias, 6, scoring="linear")


def test_captured_and_replayed(select):
    """Forward and backward in a graph, replayed over changed logits with eager work between."""
    x = torch.randn(17, 64, device="cuda")
    bias = 0.1 * torch.randn(64, device="cuda")
    dw = torch.randn(17, 6, device="cuda")

    def step(t):
        t = t.detach().requires_grad_(True)
        idx, w = select(t, 6, bias, "softmax", 8, 4)
        return idx, w.detach(), torch.autograd.grad(w, t, dw)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step(x)):
            assert torch.equal(got, want)
