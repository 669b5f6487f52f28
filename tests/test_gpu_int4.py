"""Products with group-scaled 4-bit integer weights and the routed layer over them, against 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def weight(gen, lead, R, K, group, zeros, dt):
    from lazylora_amd.int4 import Int4Weight
    packed = torch.randint(0, 256, (*lead, R, K // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((*lead, R, K // group), device="cuda", generator=gen)) / (4.6 * K ** 0.5)).to(dt)
    z = torch.randint(0, 16, scales.shape, device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    return Int4Weight(packed, scales, z)


def matrix64(packed, scales, zeros):
    """[R, K] in 64 bits on the CPU."""
    p = packed.cpu().numpy()
    q = np.empty(p.shape[:-1] + (2 * p.shape[-1],))
    q[..., 0::2], q[..., 1::2] = p & 15, p >> 4
    group = q.shape[-1] // scales.shape[-1]
    z = 8.0 if zeros is None else np.repeat(zeros.cpu().numpy().astype(np.float64), group, -1)
    return (q - z) * np.repeat(scales.double().cpu().numpy(), group, -1)


def dense64(w):
    return matrix64(w.packed, w.scales, w.zeros)


def gen_of(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(sum((i + 1) * 7919 ** i * int(k) for i, k in enumerate(key)) % 2 ** 31)
    return g


def bound(x, w, y, dt):
    """The product's error: fp32 sums of the terms x (16 + q) and of x itself times 16 + z, K / 4 additions and more
    in a row at most, against the size of what is added (|x| times 31 + 31 at most, times the scale); one rounding to
    the type (half a step, and half the smallest number)."""
    K = w.shape[-1]
    scale = np.repeat(w.scales.double().cpu().numpy(), w.group, -1)
    terms = np.abs(x) @ (62 * np.abs(scale)).T
    return (K / 4 + 16) * 2.0 ** -24 * terms + torch.finfo(dt).eps / 2 * np.abs(y) + torch.finfo(dt).tiny


SIZES = [  # M, K, R
    (1, 128, 16), (1, 256, 1), (2, 384, 17), (3, 640, 40), (15, 128, 33), (16, 1024, 16), (17, 512, 20), (31, 256, 18),
    (32, 128, 5), (33, 384, 31), (64, 256, 16), (65, 128, 16), (130, 512, 49), (1, 7168, 24),
    # each form of the tiles: two by eight waves, two by two by four, four by two by four, four by four by two and by one
    (64, 1152, 2100), (200, 384, 2100), (300, 384, 2100), (600, 384, 2100), (1100, 128, 2100), (4, 512, 70000),
]


@pytest.mark.parametrize("M,K,R", SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gemm(M, K, R, group, dtype):
    from lazylora_amd.int4 import int4_gemm
    dt = DT[dtype]
    # widths that end inside a block of 128 wherever the group allows it
    for k in {K, K + group} if group < 128 else {K}:
        for zeros in (False, True):
            gen = gen_of(M, k, R, group, zeros)
            x = torch.randn(M, k, device="cuda", generator=gen).to(dt)
            w = weight(gen, (), R, k, group, zeros, dt)
            y = int4_gemm(x, w)
            assert y.dtype == dt and y.shape == (M, R)
            xs = x.double().cpu().numpy()
            want = xs @ dense64(w).T
            err = np.abs(y.double().cpu().numpy() - want)
            assert (err <= bound(xs, w, want, dt)).all(), (k, zeros, err.max())


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("K,R", [(1024, 8), (1152, 1), (2048, 13), (2176, 40), (7168, 100), (16384, 9), (20480, 19), (3584, 4100)])
def test_gemm_long_rows(M, K, R):
    """The lengths that one wave, a whole work-group and several rounds of one cover; rows past a batch."""
    from lazylora_amd.int4 import int4_gemm
    for dt, group, zeros in ((torch.bfloat16, 128, True), (torch.float16, 32, False), (torch.bfloat16, 64, True)):
        gen = gen_of(M, K, R, group)
        x = torch.randn(M, K, device="cuda", generator=gen).to(dt)
        w = weight(gen, (), R, K, group, zeros, dt)
        y = int4_gemm(x, w)
        xs = x.double().cpu().numpy()
        want = xs @ dense64(w).T
        assert (np.abs(y.double().cpu().numpy() - want) <= bound(xs, w, want, dt)).all()


def test_small_numbers_are_kept():
    """Rows of x in the type's subnormal range, in every form of the product."""
    from lazylora_amd.int4 import int4_gemm
    for dt, tiny in ((torch.float16, 2.0 ** -24), (torch.float16, 2.0 ** -20), (torch.bfloat16, 2.0 ** -120)):
        for M in (1, 3, 6, 20):
            gen = gen_of(M)
            x = (torch.randint(-3, 4, (M, 1024), device="cuda", generator=gen) * tiny).to(dt)
            w = weight(gen, (), 24, 1024, 32, True, dt)
            w.scales.copy_(torch.full_like(w.scales, 64.0))  # results in the normal range
            want = x.double().cpu().numpy() @ dense64(w).T
            err = np.abs(int4_gemm(x, w).double().cpu().numpy() - want)
            assert (err <= torch.finfo(dt).eps * np.abs(want) + 1e-3 * np.abs(want).max()).all()


def test_codes_are_exact():
    """Every code and zero point in every place of a group: one-hot rows give the weights themselves."""
    from lazylora_amd.int4 import Int4Weight, int4_gemm
    for dt in DT.values():
        for group in (32, 64, 128):
            K, R = 256, 32
            gen = gen_of(group)
            packed = torch.randint(0, 256, (R, K // 2), device="cuda", generator=gen, dtype=torch.uint8)
            scales = 2.0 ** torch.randint(-3, 4, (R, K // group), device="cuda", generator=gen)
            zeros = torch.randint(0, 256, (R, K // group), device="cuda", generator=gen, dtype=torch.uint8)
            zeros[::2] &= 15
            w = Int4Weight(packed, scales.to(dt), zeros)
            y = int4_gemm(torch.eye(K, device="cuda", dtype=dt), w)
            assert torch.equal(y.T.double().cpu(), torch.from_numpy(dense64(w)))  # whole numbers up to 255 in 8 bits


def routed64(h, idx, w, ex, act, dt):
    """(out, size of what is added) in 64 bits; the hidden rows are rounded to dt as the layer does."""
    h, idx, w = h.double().cpu().numpy(), idx.cpu().numpy(), w.double().cpu().numpy()
    out, size = np.zeros_like(h), np.zeros_like(h)
    parts = lambda m, e: (m.packed[e], m.scales[e], None if m.zeros is None else m.zeros[e])
    for e in range(ex.E):
        t, j = np.nonzero(idx == e)
        if len(t) == 0:
            continue
        w1, w3, w2 = (matrix64(*parts(m, e)) for m in (ex.w1, ex.w3, ex.w2))
        g, u = h[t] @ w1.T, h[t] @ w3.T
        s = 1 / (1 + np.exp(-g))
        a = g * s * u if act == "swiglu" else 4 * np.tanh(g / 4) * s * 25 * np.tanh(u / 25)
        np.add.at(out, t, w[t, j, None] * (a @ w2.T))
        np.add.at(size, t, np.abs(w[t, j, None]) * (np.abs(a) @ np.abs(w2).T))
    return out, size


ROUTED = [  # N, k, E, D, F, group, zeros, dtype, act
    (1, 1, 1, 128, 128, 128, False, "bf16", "swiglu"), (1, 8, 16, 256, 128, 64, True, "bf16", "swiglu"),
    (3, 2, 4, 160, 96, 32, False, "f16", "situ"), (8, 8, 8, 128, 256, 128, True, "f16", "swiglu"),
    (9, 8, 8, 128, 256, 64, False, "bf16", "situ"), (64, 1, 2, 96, 160, 32, True, "bf16", "swiglu"),
    (65, 1, 2, 96, 160, 32, False, "f16", "swiglu"), (100, 4, 5, 192, 64, 64, True, "bf16", "situ"),
    (300, 3, 70, 128, 128, 64, False, "f16", "swiglu"), (200, 2, 1200, 64, 64, 32, True, "bf16", "swiglu"),
    (150, 2, 2, 128, 128, 128, False, "bf16", "swiglu"), (1, 8, 12, 1024, 1152, 64, True, "bf16", "swiglu"),
    (1, 3, 4, 2176, 1024, 128, False, "f16", "situ"), (1, 11, 16, 1024, 1024, 32, False, "bf16", "situ"),
    (2, 8, 12, 1024, 1152, 64, True, "bf16", "swiglu"),
    # by tokens up to 8 (pairs that share experts among them), by experts past 8 and where the pairs are many for the experts
    (3, 8, 12, 1024, 1024, 64, True, "f16", "swiglu"), (8, 3, 12, 1280, 1024, 128, False, "bf16", "situ"),
    (8, 4, 12, 1024, 1056, 32, True, "bf16", "swiglu"), (9, 2, 12, 1024, 1024, 64, False, "f16", "swiglu"),
    # 32 rows to a tile in each form (few, some, many weight rows), then 64
    (50, 2, 4, 96, 64, 32, True, "f16", "swiglu"), (50, 2, 4, 160, 1024, 32, False, "bf16", "swiglu"),
    (50, 2, 4, 128, 4096, 64, True, "bf16", "situ"), (50, 2, 4, 4096, 160, 32, False, "f16", "swiglu"),
    (128, 2, 4, 128, 2048, 128, True, "bf16", "swiglu"), (512, 2, 16, 96, 2048, 32, True, "f16", "swiglu"),
    (512, 2, 16, 2048, 96, 32, False, "bf16", "situ"),
]


def layer(gen, E, D, F, group, zeros, dt):
    from lazylora_amd.int4 import Int4Experts
    return Int4Experts(weight(gen, (E,), F, D, group, zeros, dt), weight(gen, (E,), F, D, group, zeros, dt),
                       weight(gen, (E,), D, F, group, zeros, dt))


@pytest.mark.parametrize("N,k,E,D,F,group,zeros,dtype,act", ROUTED)
def test_routed(N, k, E, D, F, group, zeros, dtype, act):
    from lazylora_amd.int4 import int4_routed
    dt = DT[dtype]
    gen = gen_of(N, k, E, D, F)
    ex = layer(gen, E, D, F, group, zeros, dt)
    h = torch.randn(N, D, device="cuda", generator=gen).to(dt)
    if k <= E:
        idx = (torch.randn(N, E, device="cuda", generator=gen) + torch.randn(E, device="cuda", generator=gen)).topk(k, -1).indices
    else:
        idx = torch.randint(0, E, (N, k), device="cuda", generator=gen)
    w = torch.rand(N, k, device="cuda", generator=gen)
    idx[N // 2, 0] = -1          # no expert
    if N > 2:
        idx[1] = E + 5           # a token with none at all
        idx[2, -1] = 2 ** 40
    out = int4_routed(h, idx, w, ex, act)
    assert out.dtype == dt and out.shape == (N, D)
    want, size = routed64(h, idx, w, ex, act, dt)
    # a hidden value is off by half a step of its type and by the errors of its two products and the activation,
    # all below a quarter step together at these widths; the output by half a step
    eps = torch.finfo(dt).eps
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= 0.75 * eps * size * 1.5 + eps / 2 * np.abs(want) + torch.finfo(dt).tiny).all(), (err / (eps * size + 1e-30)).max()
    if N > 2:
        assert (out[1] == 0).all()
    # a row's result does not depend on the others, nor on the ids' type
    again = int4_routed(h[: max(1, N // 3)], idx[: max(1, N // 3)], w[: max(1, N // 3)], ex, act)
    err = (again.float() - out[: again.shape[0]].float()).abs().max()
    assert err <= 2 * eps * float(np.abs(want).max() + 1)
    ids32 = torch.where((idx >= 0) & (idx < E), idx, -1).int()
    assert torch.equal(int4_routed(h, ids32, w, ex, act), out)


def test_same_expert_many_times():
    """Every pair with one expert (tiles end to end), a token whose slots all name it, and one expert alone."""
    from lazylora_amd.int4 import int4_routed
    dt = torch.bfloat16
    gen = gen_of(9)
    for N, k in ((1, 3), (20, 3), (33, 2), (90, 4)):
        if N == 1:
            ex = layer(gen, 4, 1024, 1024, 64, True, dt)
        else:
            ex = layer(gen, 4, 128, 128, 64, True, dt)
        h = torch.randn(N, ex.D, device="cuda", generator=gen).to(dt)
        idx = torch.full((N, k), 2, device="cuda")
        w = torch.rand(N, k, device="cuda", generator=gen)
        out = int4_routed(h, idx, w, ex)
        want, size = routed64(h, idx, w, ex, "swiglu", dt)
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= torch.finfo(dt).eps * (1.125 * size + np.abs(want) / 2)).all()


def test_layouts_and_streams():
    from lazylora_amd.int4 import Int4Weight, int4_gemm
    gen = gen_of(3)
    w = weight(gen, (), 48, 256, 64, True, torch.bfloat16)
    x = torch.randn(4, 6, 512, device="cuda", generator=gen).bfloat16()[:, ::2, 1::2]
    y = int4_gemm(x, w)
    assert y.shape == (4, 3, 48) and torch.equal(y.view(-1, 48), int4_gemm(x.contiguous().view(-1, 256), w))
    assert torch.equal(int4_gemm(x[0, 0], w), y[0, 0])
    # offset by one element, and strided weights
    flat = torch.zeros(256 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = x[0, 0]
    assert torch.equal(int4_gemm(flat[1:], w), y[0, 0])
    wide = torch.zeros(48, 256, device="cuda", dtype=torch.uint8)
    wide[:, ::2] = w.packed
    assert torch.equal(int4_gemm(x, Int4Weight(wide[:, ::2], w.scales, w.zeros)), y)
    assert int4_gemm(x[:, :0], w).shape == (4, 0, 48)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = int4_gemm(x, w)
    s.synchronize()
    assert torch.equal(z, y)


def test_rows_outside_the_call_stay():
    """Outputs are written in their rows and columns only: a result of a guarded C call."""
    from lazylora_amd.native import kernel
    lib = kernel().lib
    gen = gen_of(4)
    for M, R in ((1, 5), (17, 30), (40, 16)):
        w = weight(gen, (), R, 128, 32, True, torch.float16)
        x = torch.randn(M, 128, device="cuda", generator=gen).half()
        buf = torch.full((M * R + 64,), 7.0, device="cuda", dtype=torch.float16)
        rc = lib.mxfp4_int4_gemm(buf.data_ptr(), x.data_ptr(), w.packed.data_ptr(), w.scales.data_ptr(), w.zeros.data_ptr(),
                                 4, M, 128, R, 32, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert (buf[M * R:] == 7).all()


@pytest.mark.parametrize("N,k,E,D,F", [(1, 8, 12, 1024, 1152), (5, 8, 12, 128, 64), (40, 4, 12, 160, 96), (300, 4, 6, 128, 96)])
def test_workspace_and_output_bounds(N, k, E, D, F):
    """A routed call writes its output and its workspace and nothing behind them, on each path."""
    import ctypes
    from lazylora_amd.native import kernel
    lib = kernel().lib
    gen = gen_of(N, k, D)
    ex = layer(gen, E, D, F, 32, True, torch.bfloat16)
    h = torch.randn(N, D, device="cuda", generator=gen).bfloat16()
    idx = torch.randint(-1, E, (N, k), device="cuda", generator=gen)
    w = torch.rand(N, k, device="cuda", generator=gen)
    out = torch.full((N * D + 512,), 7.0, device="cuda", dtype=torch.bfloat16)
    n = lib.mxfp4_int4_moe_workspace_size(N, k, E, D, F)
    ws = torch.full((n + 4096,), 0xA5, device="cuda", dtype=torch.uint8)
    arr = lambda name: (ctypes.c_void_p * 3)(*[getattr(m, name).data_ptr() for m in (ex.w1, ex.w3, ex.w2)])
    rc = lib.mxfp4_int4_moe_forward(out.data_ptr(), h.data_ptr(), 1, idx.data_ptr(), 3, w.data_ptr(), N, k, arr("packed"),
                                    arr("scales"), arr("zeros"), E, D, F, 32, 0, ws.data_ptr(), n,
                                    torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (out[N * D:] == 7).all() and (ws[n:] == 0xA5).all()
    from lazylora_amd.int4 import int4_routed
    assert torch.equal(out[: N * D].view(N, D), int4_routed(h, idx, w, ex))


def test_two_streams_at_once():
    """Calls of different sizes on two streams, each with its own workspace, give what they give alone."""
    from lazylora_amd.int4 import int4_gemm, int4_routed
    gen = gen_of(31)
    ex = layer(gen, 16, 256, 128, 64, True, torch.bfloat16)
    wt = weight(gen, (), 512, 256, 64, False, torch.bfloat16)
    calls = []
    for N in (1, 3, 33, 200):
        h = torch.randn(N, 256, device="cuda", generator=gen).bfloat16()
        idx = torch.randn(N, 16, device="cuda", generator=gen).topk(4, -1).indices
        w = torch.rand(N, 4, device="cuda", generator=gen)
        calls.append(lambda h=h, idx=idx, w=w: (int4_routed(h, idx, w, ex), int4_gemm(h, wt)))
    want = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for r in range(6):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[(i + r) % 2]):
                got.append((i, c()))
    torch.cuda.synchronize()
    for i, g in got:
        assert torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1])


def test_non_finite_rows():
    """An infinity or NaN stays in its row."""
    from lazylora_amd.int4 import int4_gemm
    gen = gen_of(5)
    w = weight(gen, (), 32, 256, 128, False, torch.bfloat16)
    x = torch.randn(20, 256, device="cuda", generator=gen).bfloat16()
    want = int4_gemm(x, w)
    x[3, 7], x[11, 200] = float("inf"), float("nan")
    y = int4_gemm(x, w)
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[3] = bad[11] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], want[~bad])


def test_refusals():
    from lazylora_amd.int4 import Int4Experts, Int4Weight, int4_gemm, int4_routed
    gen = gen_of(6)
    w = weight(gen, (), 16, 128, 32, True, torch.bfloat16)
    x = torch.randn(2, 128, device="cuda").bfloat16()
    for bad in (x.float(), x.half(), x[:, :96], x.cpu(), x.int(), torch.zeros((), device="cuda").bfloat16()):
        with pytest.raises(ValueError):
            int4_gemm(bad, w)
    with pytest.raises(NotImplementedError):
        int4_gemm(x.clone().requires_grad_(True), w)
    with torch.no_grad():
        int4_gemm(x.clone().requires_grad_(True), w)
    for args in ((w.packed.int(), w.scales), (w.packed, w.scales.float()), (w.packed, w.scales[:, :3]),
                 (w.packed, w.scales[:8]), (w.packed, w.scales, w.zeros.int()), (w.packed, w.scales, w.zeros[:, :2]),
                 (w.packed[0], w.scales[0]), (w.packed, w.scales.repeat(1, 2)), (w.packed, w.scales.cpu())):
        with pytest.raises(ValueError):
            Int4Weight(*args)
    ex = layer(gen, 3, 128, 64, 32, False, torch.bfloat16)
    idx, tw = torch.zeros(2, 2, device="cuda", dtype=torch.int64), torch.ones(2, 2, device="cuda")
    for args in ((x[0], idx, tw), (x, idx[:1], tw), (x, idx.float(), tw), (x, idx, tw[:, :1]), (x, idx, tw.long()),
                 (x, idx.cpu(), tw), (x.half(), idx, tw), (x[:, :64], idx, tw), (x, idx[:, :0], tw[:, :0])):
        with pytest.raises(ValueError):
            int4_routed(*args, ex)
    with pytest.raises(ValueError):
        int4_routed(x, idx, tw, ex, act="relu")
    with pytest.raises(NotImplementedError):
        int4_routed(x, idx, tw.clone().requires_grad_(True), ex)
    with pytest.raises(ValueError):
        Int4Experts(ex.w1, ex.w3, ex.w1)
    with pytest.raises(ValueError):
        Int4Experts(ex.w1, ex.w3, weight(gen, (3,), 128, 64, 64, False, torch.bfloat16))
    with pytest.raises(ValueError):
        Int4Experts(w, w, w)
    with pytest.raises(ValueError):
        Int4Experts(ex.w1, ex.w3, weight(gen, (3,), 128, 64, 32, True, torch.bfloat16))


def test_captured_and_replayed():
    """A decoding step, selection and routed layer, in one graph, replayed over changed tokens."""
    from lazylora_amd.int4 import int4_gemm, int4_routed
    from lazylora_amd.router import select_experts
    gen = gen_of(8)
    dt = torch.bfloat16
    for N in (2, 40):
        ex = layer(gen, 16, 256, 128, 64, True, dt)
        wp = weight(gen, (), 256, 256, 64, False, dt)
        gate = torch.randn(16, 256, device="cuda", generator=gen) / 16
        h = torch.randn(N, 256, device="cuda", generator=gen).to(dt)

        def step(h):
            x = int4_gemm(h, wp)
            idx, w = select_experts(x.float() @ gate.T, 4, scoring="softmax", num_groups=4, topk_groups=2)
            return x, idx, int4_routed(x, idx, w, ex)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(h)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(h)
        for _ in range(4):
            h.copy_(torch.randn(N, 256, device="cuda", generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            for got, want in zip(out, step(h)):
                assert torch.equal(got, want)
