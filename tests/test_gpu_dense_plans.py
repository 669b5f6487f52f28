"""Every kernel form that the feed-forward block's plan chooses, cuts of the last rows among them, element by
element against float64. tests/test_dense_plans.py asserts that these sizes reach every form there is, so a change
of the plan that loses one is noticed."""
import pytest
import torch

from tests.test_gpu_dense_ffn import check, inputs, reference

pytestmark = pytest.mark.gpu

# (M, D, F, Do): a frozen and a full step of large widths, then ragged sizes, each for forms that those before it miss
PLAN_SIZES = [(1000, 7168, 2048, 7168), (4099, 7168, 2048, 7168), (1, 216, 2168, 216), (1894, 208, 336, 1440),
              (74, 5408, 680, 3280), (17, 1760, 608, 6648), (6947, 304, 344, 552), (18, 6616, 4328, 1296),
              (39, 208, 240, 264), (51, 232, 224, 264), (19, 224, 2296, 224), (33, 200, 2248, 4592),
              (55, 472, 2072, 7880), (2663, 200, 6160, 248), (2054, 1608, 208, 7984), (13305, 392, 648, 1032),
              (4212, 3888, 208, 336), (5702, 264, 264, 6376), (129, 6520, 5664, 1800), (163, 816, 4128, 5728),
              (4292, 4128, 472, 2008), (2820, 5800, 296, 2208), (1588, 216, 3528, 2536), (1172, 208, 7992, 2128)]


@pytest.fixture(scope="module")
def k():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    from lazylora_amd.native import kernel
    return kernel()


@pytest.mark.parametrize("M,D,F,Do", PLAN_SIZES)
@pytest.mark.parametrize("act,dt", [("situ", torch.bfloat16), ("swiglu", torch.float16)])
def test_every_form(k, M, D, F, Do, act, dt):
    print("\n[case] form", M, D, F, Do, act, dt, flush=True)
    t = inputs(M + F, M, D, F, Do, dt)
    want = reference(t, act, True)
    y, h, gu = k.ffn_forward(t["x"], t["wg"], t["wu"], t["wd"], act, t["gd"], t["ud"], save_for_backward=True)
    check("y", y, want["y"])
    check("h", h, want["h"])
    dgu, dx, dwg, dwu, dwd = k.ffn_backward(t["dy"], gu, t["wg"], t["wu"], t["wd"], act, t["dh"], t["x"], h,
                                            need_w_in=True, need_w_down=True)
    for name, got in (("dg", dgu[:, :F]), ("du", dgu[:, F:]), ("dx", dx), ("dwg", dwg), ("dwu", dwu), ("dwd", dwd)):
        check(name, got, want[name])
