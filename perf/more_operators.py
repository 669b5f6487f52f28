"""Routing to experts and the experts' products with 4-bit integer weights, as programs call them:
expert selection (softmax or sigmoid scores, balance bias, groups, renormalised weights, with its
gradient), the product with group-scaled 4-bit weights and the routed expert layer over them.

Where `own` is true a pass calls lazylora_amd.router and lazylora_amd.int4; else the same values come
from elementary torch operations. `listed()` names the cases, `draw()` makes more of the same ranges
and `exact()` computes a case in 64 bits from the operator's definition.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST_LOGITS = 8192 * 256        # a drawn selection stays below the largest listed one,
LARGEST_MACS = 1000 * 7168 * 2048  # a drawn product too,
LARGEST_WEIGHTS = 8192 * 28672
LARGEST_LAYER = 64 * 7168 * 2048   # and so does a routed layer: elements of one of its three matrices,
LARGEST_ACTIVE = 112 * 3584 * 1536  # those of the experts that its tokens choose,
LARGEST_PAIR_MACS = 2000 * 3584 * 1536  # and one product's multiplications


# ---------------------------------------------------------------- the cases
def _select(name, N, E, k, scoring, dtype="f32", bias=True, groups=1, kept=1, group_score="top2", renorm=True,
            mode="forward", masked=False):
    """mode "step" adds the gradient of the logits; masked: some experts are off (-inf for every token)."""
    return {"name": name, "kind": "select", "N": N, "E": E, "k": k, "scoring": scoring, "dtype": dtype, "bias": bias,
            "groups": groups, "kept": kept, "group_score": group_score, "renorm": renorm, "mode": mode,
            "masked": masked}


def _gemm(name, M, K, R, group, dtype="bf16", zeros=True):
    return {"name": name, "kind": "gemm", "M": M, "K": K, "R": R, "group": group, "dtype": dtype, "zeros": zeros}


def _routed(name, N, k, E, D, F, group, dtype="bf16", zeros=False, act="swiglu"):
    return {"name": name, "kind": "routed", "N": N, "k": k, "E": E, "D": D, "F": F, "group": group, "dtype": dtype,
            "zeros": zeros, "act": act}


def listed():
    return [
        # serving, one token: launch latency
        _select("select_token", 1, 256, 8, "sigmoid", groups=8, kept=4),
        # prefill of a long prompt, group-limited choice
        _select("select_prefill", 8192, 256, 8, "sigmoid", groups=8, kept=4),
        # a ragged training step of a small softmax mixture, 16-bit logits, no bias
        _select("select_softmax_step", 4099, 64, 6, "softmax", "bf16", bias=False, mode="step"),
        # a training step over many experts in seven groups of 128, some of them off
        _select("select_wide_step", 1024, 896, 16, "softmax", groups=7, kept=3, group_score="max", mode="step",
                masked=True),
        # one token through the gate and up projections of a shared expert, with zero points
        _gemm("gemm_token", 1, 7168, 4096, 128),
        # two tokens (one with its draft) through a wide projection
        _gemm("gemm_wide", 2, 8192, 28672, 64),
        # a ragged batch of decoding requests through the latent up projection, half precision, symmetric codes
        _gemm("gemm_few_rows", 13, 3584, 7168, 32, "f16", False),
        # a short prompt
        _gemm("gemm_prompt", 1000, 7168, 2048, 64),
        # one token's eight experts
        _routed("routed_token", 1, 8, 64, 7168, 2048, 32),
        # a batch of decoding requests over the experts of a latent layer
        _routed("routed_batch", 32, 8, 128, 3584, 1536, 128, "f16", True, "situ"),
        # a ragged short prompt over few experts
        _routed("routed_prompt", 500, 4, 32, 3584, 1536, 64),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(("select", "gemm", "routed"))
    group, zeros = rng.choice((32, 64, 128)), rng.random() < 0.5
    if kind == "select":
        groups = rng.choice((1, 1, 2, 4, 7, 8, 12))
        E = groups * _log(rng, max(2, 8 // groups), 1024 // groups)
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(16, kept * (E // groups)))
        return _select("", _log(rng, 1, min(8192, LARGEST_LOGITS // E)), E, k, rng.choice(("sigmoid", "softmax")),
                       rng.choice(("f32", "f32", "bf16", "f16")), rng.random() < 0.7, groups, kept,
                       rng.choice(("top2", "max")), rng.random() < 0.8, rng.choice(("forward", "step")),
                       rng.random() < 0.3)
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "gemm":
        K = group * _log(rng, max(1, 256 // group), 8192 // group)
        R = _log(rng, 16, min(28672, LARGEST_WEIGHTS // K))
        return _gemm("", _log(rng, 1, min(1024, max(1, LARGEST_MACS // (K * R)))), K, R, group, dtype, zeros)
    D = group * _log(rng, max(1, 256 // group), 7168 // group)
    F = group * _log(rng, max(1, 128 // group), 2048 // group)
    E = _log(rng, 4, min(128, LARGEST_LAYER // (D * F)))
    k = rng.randint(1, min(8, E))
    N = _log(rng, 1, min(512, max(1, LARGEST_PAIR_MACS // (k * D * F))))
    while N > 1 and _active(N, k, E) * D * F > LARGEST_ACTIVE:
        N //= 2
    return _routed("", N, k, E, D, F, group, dtype, zeros, rng.choice(("swiglu", "situ")))


# ---------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _codes(gen, lead, R, K, group, zeros, dt):
    """(packed, scales, zeros) of random matrices [*lead, R, K] whose products keep the activations' size."""
    packed = torch.randint(0, 256, (*lead, R, K // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = (0.5 + torch.rand((*lead, R, K // group), device="cuda", generator=gen)) / (4.6 * math.sqrt(K))
    z = torch.randint(5, 12, scales.shape, device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    return packed, scales.to(dt), z


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DT[case["dtype"]]
    st = {"case": case}
    if case["kind"] == "select":
        N, E = case["N"], case["E"]
        # some experts are liked better than others, and the bias works against it
        liked = 0.5 * _randn(gen, E)
        logits = 1.5 * _randn(gen, N, E) + liked
        st["bias"] = 0.02 * _randn(gen, E) - 0.05 * liked if case["bias"] else None
        if case["masked"]:
            logits[:, torch.rand(E, device="cuda", generator=gen) < 0.05] = -math.inf
        st["logits"] = logits.to(dt)
        if case["mode"] == "step":
            st["logits"].requires_grad_(True)
            st["dw"] = _randn(gen, N, case["k"])
    elif case["kind"] == "gemm":
        st["x"] = _randn(gen, case["M"], case["K"]).to(dt)
        st["w"] = _codes(gen, (), case["R"], case["K"], case["group"], case["zeros"], dt)
    else:
        N, E, D, F = case["N"], case["E"], case["D"], case["F"]
        st["h"] = _randn(gen, N, D).to(dt)
        for name, R, K in (("w1", F, D), ("w3", F, D), ("w2", D, F)):
            st[name] = _codes(gen, (E,), R, K, case["group"], case["zeros"], dt)
        # a router's choice: some experts are liked better, weights that sum to one
        top = (_randn(gen, N, E) + 0.5 * _randn(gen, E)).topk(case["k"], -1)
        st["idx"], st["weights"] = top.indices, torch.softmax(top.values, -1)
    if own:
        _handles(st)
    return st


def _handles(st):
    """The weights as a program that uses the package keeps them."""
    from lazylora_amd.int4 import Int4Experts, Int4Weight
    case = st["case"]
    if case["kind"] == "gemm":
        st["weight"] = Int4Weight(*st["w"])
    elif case["kind"] == "routed":
        st["experts"] = Int4Experts(*(Int4Weight(*st[n]) for n in ("w1", "w3", "w2")))


# ---------------------------------------------------------------- a pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return {"select": _plain_select, "gemm": _plain_gemm, "routed": _plain_routed}[case["kind"]](case, state)


def _run_own(case, st):
    if case["kind"] == "select":
        from lazylora_amd.router import select_experts
        idx, w = select_experts(st["logits"], case["k"], st["bias"], scoring=case["scoring"],
                                num_groups=case["groups"], topk_groups=case["kept"], group_score=case["group_score"],
                                renormalize=case["renorm"], routed_scaling_factor=SCALE)
        if case["mode"] == "forward":
            return idx, w
        return (idx, w) + torch.autograd.grad(w, [st["logits"]], st["dw"])
    if "weight" not in st and "experts" not in st:
        _handles(st)
    from lazylora_amd.int4 import int4_gemm, int4_routed
    if case["kind"] == "gemm":
        return (int4_gemm(st["x"], st["weight"]),)
    return (int4_routed(st["h"], st["idx"], st["weights"], st["experts"], act=case["act"]),)


SCALE = 2.5  # the routed scaling factor


# ---------------------------------------------------------------- plain forms
def _plain_select(case, st):
    x = st["logits"].double()  # next to the border of a choice 32 bits lose which value is the larger
    N, E = x.shape
    G, size = case["groups"], E // case["groups"]
    if case["scoring"] == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
    else:
        s = torch.exp(x - x.max(-1, keepdim=True).values)
        s = s / s.sum(-1, keepdim=True)
    choice = x if st["bias"] is None else s + st["bias"].double()  # without a bias the scores' order is the logits'
    if G > 1:
        if case["group_score"] == "max":
            score = choice.view(N, G, size).max(-1).values
        else:
            best = (s if st["bias"] is None else choice).view(N, G, size).sort(dim=-1, descending=True).values
            score = best[..., 0] + best[..., 1] if size > 1 else best[..., 0]
        kept = score.sort(dim=-1, descending=True, stable=True).indices[:, :case["kept"]].sort(-1).values
        open_ = (kept[..., None] * size + torch.arange(size, device=x.device)).view(N, -1)
        order = choice.gather(1, open_).sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
        idx = open_.gather(1, order)
    else:
        idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
    chosen = s.gather(1, idx)
    total = chosen.sum(-1, keepdim=True) + 1e-20
    norm = case["renorm"] and case["k"] > 1
    w = SCALE * (chosen / total if norm else chosen)
    if case["mode"] == "forward":
        return idx, w.float()
    g = SCALE * st["dw"].double()
    if norm:
        g = (g - (g * chosen).sum(-1, keepdim=True) / total) / total
    ds = torch.zeros_like(s).scatter_(1, idx, g)
    if case["scoring"] == "sigmoid":
        dx = ds * s * (1 - s)
    else:
        dx = s * (ds - (g * chosen).sum(-1, keepdim=True))
    return idx, w.float(), dx.to(st["logits"].dtype)


def _matrix(packed, scales, zeros):
    """[R, K] in 32 bits."""
    R, K = packed.shape[0], 2 * packed.shape[1]
    q = torch.stack((packed & 15, packed >> 4), -1).view(R, scales.shape[1], -1).float()
    q -= 8.0 if zeros is None else zeros[..., None].float()
    return (q * scales[..., None].float()).view(R, K)


def _plain_gemm(case, st):
    return ((st["x"].float() @ _matrix(*st["w"]).T).to(DT[case["dtype"]]),)


def _plain_routed(case, st):
    x, idx, w = st["h"].float(), st["idx"], st["weights"]
    out = torch.zeros_like(x)
    for e in torch.unique(idx).tolist():
        w1, w3, w2 = (_matrix(*(None if t is None else t[e] for t in st[n])) for n in ("w1", "w3", "w2"))
        t, j = (idx == e).nonzero(as_tuple=True)
        g, u = x[t] @ w1.T, x[t] @ w3.T
        s = 1 / (1 + torch.exp(-g))
        h = g * s * u if case["act"] == "swiglu" else 4 * torch.tanh(g / 4) * s * 25 * torch.tanh(u / 25)
        out[t] += w[t, j, None] * (h @ w2.T)
    return (out.to(DT[case["dtype"]]),)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"select": _exact_select, "gemm": _exact_gemm, "routed": _exact_routed}[case["kind"]](case, st)


def _exact_select(case, st):
    import numpy as np
    logits = st["logits"].detach().double().cpu()
    N, E = logits.shape
    scores = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, 1)
    keys = logits if st["bias"] is None else scores + st["bias"].double().cpu()
    top2 = (scores if st["bias"] is None else keys).numpy().reshape(N, case["groups"], -1)
    keys = keys.numpy()
    if case["group_score"] == "max":
        value = keys.reshape(top2.shape).max(2)
    else:
        value = np.sort(top2, 2)[:, :, -2:].sum(2)
    # a group's rank: the groups before it are the better ones and the equal ones of lower number
    number = np.arange(case["groups"])
    before = (value[:, None, :] > value[:, :, None]) | ((value[:, None, :] == value[:, :, None]) &
                                                       (number[None, None, :] < number[None, :, None]))
    on = np.repeat(before.sum(2) < case["kept"], E // case["groups"], 1)
    ids = np.broadcast_to(np.arange(E), (N, E))
    idx = torch.from_numpy(np.lexsort((ids, -keys, ~on), axis=1)[:, :case["k"]].copy()).cuda()
    x = st["logits"].detach().double().requires_grad_(True)
    s = (x.sigmoid() if case["scoring"] == "sigmoid" else x.softmax(1)).gather(1, idx)
    w = SCALE * (s / (s.sum(1, True) + 1e-20) if case["renorm"] and case["k"] > 1 else s)
    if case["mode"] == "forward":
        return idx, w.detach()
    return (idx, w.detach()) + torch.autograd.grad(w, [x], st["dw"].double())


def _exact_product(x, packed, scales, zeros):
    """x [M, K] in 64 bits times the transposed matrix, some rows of it at a time."""
    group = 2 * packed.shape[1] // scales.shape[1]
    out = []
    for p, s, r in zip(packed.split(4096), scales.split(4096), range(0, packed.shape[0], 4096)):
        w = torch.empty(p.shape[0], 2 * p.shape[1], dtype=torch.float64, device=p.device)
        w[:, 0::2], w[:, 1::2] = p % 16, p // 16
        w -= 8 if zeros is None else zeros[r:r + 4096].double().repeat_interleave(group, 1)
        w *= s.double().repeat_interleave(group, 1)
        out.append(x.mm(w.t()))
    return torch.cat(out, 1)


def _exact_gemm(case, st):
    return (_exact_product(st["x"].double(), *st["w"]),)


def _exact_routed(case, st):
    h, out = st["h"].double(), torch.zeros(st["h"].shape, dtype=torch.float64, device="cuda")
    part = lambda name, e: [None if t is None else t[e] for t in st[name]]
    for e in range(case["E"]):
        share = ((st["idx"] == e) * st["weights"].double()).sum(1)
        rows = share.nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        g, u = _exact_product(h[rows], *part("w1", e)), _exact_product(h[rows], *part("w3", e))
        if case["act"] == "situ":
            a = 100 * (g / 4).tanh() * g.sigmoid() * (u / 25).tanh()
        else:
            a = g * g.sigmoid() * u
        out.index_add_(0, rows, share[rows, None] * _exact_product(a, *part("w2", e)))
    return (out,)


# ---------------------------------------------------------------- what a pass cannot do without
def _active(N, k, E):
    """Experts that N tokens choose, on average, where all are liked the same."""
    return E * (1 - (1 - k / E) ** N)


def _weight_bytes(R, K, case):
    return R * K / 2 + R * (K // case["group"]) * (BYTES[case["dtype"]] + (1 if case["zeros"] else 0))


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "select":
        N, E, k = case["N"], case["E"], case["k"]
        bias = 4 * E if case["bias"] else 0
        if case["mode"] == "forward":
            return {"bytes": N * E * e + bias + 12 * N * k, "flops": 10.0 * N * E}
        return {"bytes": 2 * N * E * e + bias + 16 * N * k, "flops": 15.0 * N * E}
    if case["kind"] == "gemm":
        M, K, R = case["M"], case["K"], case["R"]
        return {"bytes": _weight_bytes(R, K, case) + e * M * (K + R), "flops": 2.0 * M * K * R}
    N, k, D, F = case["N"], case["k"], case["D"], case["F"]
    one = 2 * _weight_bytes(F, D, case) + _weight_bytes(D, F, case)
    return {"bytes": _active(N, k, case["E"]) * one + N * (2 * D * e + 12 * k), "flops": 6.0 * N * k * D * F}
