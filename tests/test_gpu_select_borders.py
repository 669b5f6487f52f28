"""Expert selection where the border of a choice is hard to see in 32 bits, or infinite, against its definition in 64
bits."""
import numpy as np
import pytest
import torch

from test_gpu_select import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def select():
    from lazylora_amd.router import select_experts
    return select_experts


def test_group_kept_by_its_rounding(select):
    """One expert of group 0 is forced and the other banned by 2^20: the group's sum of two is 0.9440, in 32 bits 1.0.
    Groups 1 (0.9860) and 2 (0.9580) stay, though neither is near group 0's 32-bit value."""
    x = np.array([[0.3317167, -0.5672482, -0.0279773, -0.0279773, -0.0839758, -0.0839758]], np.float32)
    bias = np.array([2.0 ** 20, -2.0 ** 20, 0, 0, 0, 0], np.float32)
    idx, _ = run(select, x, "f32", bias, top_k=4, num_groups=3, topk_groups=2)
    assert idx[0].tolist() == [2, 3, 4, 5]


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [2.0 ** 4, 2.0 ** 10, 2.0 ** 20, 2.0 ** 30])
@pytest.mark.parametrize("E,groups,kept", [(6, 3, 2), (64, 8, 3), (64, 8, 7), (84, 7, 4), (256, 8, 4), (896, 7, 3)])
def test_biases_of_mixed_sign(select, scoring, size, E, groups, kept):
    """Some groups of one forced and otherwise banned experts, in random places of the groups' order: their sums of two
    cancel to the size of a score."""
    rng = np.random.default_rng(int(size) + E)
    x = (0.1 * rng.standard_normal((512, E))).astype(np.float32)
    per = E // groups
    for n in (1, 2, groups // 2, groups):
        bias = (1e-6 * rng.standard_normal(E)).astype(np.float32)
        for g in rng.permutation(groups)[:n]:
            bias[g * per:(g + 1) * per] = -size
            bias[g * per + rng.integers(per)] = size
        run(select, x, "f32", bias, top_k=min(4, kept * per), scoring=scoring, num_groups=groups, topk_groups=kept)


@pytest.mark.parametrize("kept", [1, 2, 3])
def test_sums_past_32_bits(select, kept):
    """Sums of two finite choices that 32 bits cannot hold are no infinities."""
    big = np.finfo(np.float32).max
    x = np.zeros((2, 8), np.float32)
    x[1] = [0, 1, 2, 3, 0, 1, 2, 3]
    for bias in ([-big, -big, -big / 2, -big * 0.75, 0, 0, -np.inf, 0], [big, big * 0.5, big, big * 0.75, 0, big, np.inf, -big],
                 [np.inf, -np.inf, big, big, -big, -big, -np.inf, -np.inf], [-np.inf, -np.inf, -big, -big, -np.inf, -big, -big, -big]):
        with np.errstate(invalid="ignore"):  # inf - inf is NaN, in the definition too
            run(select, x, "f32", np.array(bias, np.float32), top_k=min(2 * kept, 4), num_groups=4, topk_groups=kept)


def shortest(call, n=20):
    """The shortest of several timings of n calls in a graph, in seconds per call."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    times = []
    for _ in range(10):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e-3 / n)
    return min(times)


@pytest.mark.parametrize("off", [-np.inf, float(np.finfo(np.float32).min), np.inf])
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_switched_experts_cost_no_64_bit_choice(select, off, group_score):
    """A group switched off, or an expert forced, by an infinite or the lowest bias: the choice is as clear in 32 bits
    as without (11 us; every token's groups and order again in 64 bits took 18 to 21)."""
    x = 1.5 * torch.randn(8192, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    plain = 0.02 * torch.randn(256, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    bias = plain.clone()
    bias[32:33 if off > 0 else 64] = off
    run(select, x[:256].cpu().numpy(), "f32", bias.cpu().numpy(), top_k=8, num_groups=8, topk_groups=4, group_score=group_score)
    time = lambda b: shortest(lambda: select(x, 8, b, num_groups=8, topk_groups=4, group_score=group_score))
    assert time(bias) < 1.3 * time(plain)


@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_infinite_groups_on_both_sides(select, group_score):
    """More or fewer groups switched off, forced or NaN than the kept ones leave room for."""
    rng = np.random.default_rng(8)
    for n in range(9):
        for value in (-np.inf, np.inf, np.nan, np.finfo(np.float32).min, np.finfo(np.float32).max):
            x = rng.standard_normal((8, 64)).astype(np.float32)
            bias = (0.02 * rng.standard_normal(64)).astype(np.float32)
            for g in rng.permutation(8)[:n]:
                bias[8 * g:8 * g + rng.integers(1, 9)] = value
            run(select, x, "f32", bias, top_k=6, num_groups=8, topk_groups=4, group_score=group_score)
            run(select, x, "f32", bias, top_k=6, scoring="softmax", num_groups=8, topk_groups=4, group_score=group_score)


def test_saturated_scores(select):
    """Scores that 64 bits hold as equal: without a bias the order is the logits', with one the ids' (written down
    here, not computed); a 64-bit bias counts as its 32-bit value."""
    x = torch.tensor([[45.0, 38.0, 50.0, 40.0, -60.0, -42.0, -50.0, 0.0]], device="cuda")
    pick = lambda b, k=8: select(x, k, b, renormalize=False)[0][0].tolist()
    assert pick(None) == [2, 0, 3, 1, 7, 5, 6, 4]
    assert pick(torch.zeros(8, device="cuda")) == [0, 1, 2, 3, 7, 5, 6, 4]  # small scores differ, those next to 1 do not
    assert pick(torch.full((8,), 0.02, device="cuda")) == [0, 1, 2, 3, 7, 4, 5, 6]
    # 1 - 9.4e-14 and 1 - 3.4e-14 differ in 64 bits, though not in 32
    y = torch.tensor([[30.0, 31.0, 30.5, -1.0]], device="cuda")
    assert select(y, 3, torch.zeros(4, device="cuda"))[0][0].tolist() == [1, 2, 0]
    b = torch.zeros(8, device="cuda", dtype=torch.float64)
    b[3] = 2.0 ** -30
    assert pick(1 + b) == pick(torch.ones(8, device="cuda")) and pick(b)[0] == 3


def grads64(x, g, idx, scoring, renormalize, scale):
    """(dL/dlogits, size of what is added) in 64 bits, with the differences of the upstream gradients taken before they
    are weighted: dL/ds_j of the renormalised weights is (sum_i s_i (g_j - g_i) + 1e-20 g_j) / S^2, and softmax's own
    term likewise over all experts."""
    N, E = x.shape
    if scoring == "sigmoid":
        s, rest = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    else:
        e = np.exp(x - x.max(1, keepdims=True))
        s = e / e.sum(1, keepdims=True)
    dx, size = np.zeros((N, E)), np.zeros((N, E))
    for t in range(N):
        c, u = s[t, idx[t]], scale * g[t]
        out = np.ones(E, bool)
        out[idx[t]] = False
        diff = u[:, None] - u[None, :]
        both = np.abs(u[:, None]) + np.abs(u[None, :])
        np.fill_diagonal(both, 0)
        a, b = (diff * c).sum(1), (both * c).sum(1)
        if renormalize:
            S = c.sum() + 1e-20
            a, b, d = (a + 1e-20 * u) / S ** 2, (b + 1e-20 * np.abs(u)) / S ** 2, (u * c).sum() * 1e-20 / S ** 2
        elif scoring == "sigmoid":
            a, b, d = u, np.abs(u), 0.0
        else:
            left = s[t, out].sum()
            a, b, d = a + u * left, b + np.abs(u) * left, (u * c).sum()
        if scoring == "sigmoid":
            dx[t, idx[t]], size[t, idx[t]] = (v * c * rest[t, idx[t]] for v in (a, b))
        else:
            dx[t], size[t] = -s[t] * d, s[t] * np.abs(u * c).sum() * (1e-20 / S ** 2 if renormalize else 1)
            dx[t, idx[t]], size[t, idx[t]] = c * (a - d if renormalize else a), c * (b + abs(d) * renormalize)
    return dx, size


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E,top_k", [(8, 1), (8, 2), (64, 6), (300, 16), (1024, 64), (4096, 5)])
def test_gradients_of_confident_routers(select, scoring, renormalize, E, top_k):
    """Rows in which one expert has nearly all of the score: its gradient is as small as the others' scores, and is
    right to 32 bits of that, not of the upstream gradient."""
    rng = np.random.default_rng(E + top_k)
    x = rng.standard_normal((24, E)).astype(np.float32)
    for t in range(24):
        x[t] -= 0.75 * t * (scoring == "sigmoid")
        x[t, rng.integers(E)] += 0.75 * t
    g = rng.standard_normal((24, top_k)).astype(np.float32)
    logits = torch.from_numpy(x).cuda().requires_grad_(True)
    idx, w = select(logits, top_k, scoring=scoring, renormalize=renormalize, routed_scaling_factor=2.5)
    got = torch.autograd.grad(w, logits, torch.from_numpy(g).cuda())[0].double().cpu().numpy()
    want, size = grads64(x.astype(np.float64), g.astype(np.float64), idx.cpu().numpy(), scoring, renormalize and top_k > 1, 2.5)
    # scores as in W_TOL (their exponents' rounding up to 2^-24 times the distance of a logit from the largest, 32 where
    # they matter), three of them in a product, the sums of 64 and of 4096 / 64 terms in a row
    tol = 1024 * 2.0 ** -24
    assert (np.abs(got - want) <= tol * size + 1e-30).all(), (np.abs(got - want) / (size + 1e-30)).max()
