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
        run(select, x, "f32", np.array(bias, np.float32), top_k=min(2 * kept, 4), num_groups=4, topk_groups=kept)
