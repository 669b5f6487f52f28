"""The dense operators of the latent MoE block as programs call them, as cases that can be timed
and compared: the gated feed-forward block (the shared expert), layer / RMS norm and the adapters'
dropout.

Where `own` is true a pass calls lazylora_amd.dense; else the same values come from elementary
torch operations in 32 bits. `listed()` names the cases, `draw()` makes more of the same ranges and
`exact()` computes a case in 64 bits from the operator's definition.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST_FLOPS = 1.1e12  # a feed-forward pass of a drawn case stays below the largest listed one
LARGEST_ELEMENTS = 8192 * 7168  # and so does a norm or dropout pass


# ---------------------------------------------------------------- the cases
def _ffn(name, M, D, F, Do, mode, act="swiglu", dtype="bf16"):
    """mode: "forward"; "adapters" = a step with frozen weights, the adapters' deltas on gate and up
    and the hidden activations returned for the down adapter; "train" = a step with weight gradients."""
    return {"name": name, "kind": "ffn", "M": M, "D": D, "F": F, "Do": Do, "mode": mode, "act": act, "dtype": dtype}


def _norm(name, M, D, norm, mode, dtype, affine="full"):
    """affine: "full" = weight (and bias for layer norm), "weight" = no bias, "none" = neither."""
    return {"name": name, "kind": "norm", "M": M, "D": D, "norm": norm, "mode": mode, "dtype": dtype, "affine": affine}


def _dropout(name, M, D, p, mode, dtype):
    return {"name": name, "kind": "dropout", "M": M, "D": D, "p": p, "mode": mode, "dtype": dtype}


def listed():
    return [
        # serving, one token through the shared expert: every weight read for one row
        _ffn("ffn_token", 1, 7168, 2048, 7168, "forward"),
        # a ragged batch of decoding requests (or a short prompt), the latent width, half precision
        _ffn("ffn_few_rows", 37, 3584, 1536, 3584, "forward", "situ", "f16"),
        # a ragged LoRA step: frozen weights, the adapters' deltas and the hidden output for the down adapter
        _ffn("ffn_adapter_step", 1000, 7168, 2048, 7168, "adapters", "situ"),
        # prefill of a long prompt
        _ffn("ffn_prefill", 8192, 7168, 2048, 7168, "forward"),
        # a full fine-tuning step: all weight gradients, a token count off every tile
        _ffn("ffn_train", 4099, 7168, 2048, 7168, "train"),
        # the norm in front of a layer while one token is decoded
        _norm("norm_token", 1, 7168, "rms", "forward", "bf16"),
        # the norm of the routed sum in a LoRA step of the latent block: fp32, weight gradient
        _norm("norm_latent_step", 1000, 3584, "rms", "step", "f32"),
        # layer norm over a long batch, forward and backward, weight and bias gradients
        _norm("norm_train", 8192, 7168, "layer", "step", "bf16"),
        # adapter dropout of one decoded row (a one-token training sequence): launch latency
        _dropout("dropout_row", 1, 2049, 0.1, "forward", "f32"),
        # adapter dropout in the LoRA step above: fp32 inputs, forward and backward
        _dropout("dropout_adapter", 1000, 7168, 0.05, "step", "f32"),
        # the same over a long batch in 16 bits
        _dropout("dropout_long", 8192, 7168, 0.1, "step", "bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("ffn", "ffn", "norm", "dropout"))
    if kind == "ffn":
        mode = rng.choice(("forward", "forward", "adapters", "train"))
        # widths of small models up to the listed ones, any multiple of 8
        D, F = 8 * _log(rng, 16, 896), 8 * _log(rng, 16, 256)
        Do = D if rng.random() < 0.7 else 8 * _log(rng, 16, 896)
        per_row = 2.0 * F * (2 * D + Do) * {"forward": 1, "adapters": 2, "train": 3}[mode]
        M = _log(rng, 1, min(8192, max(1, int(LARGEST_FLOPS / per_row))))
        return _ffn("", M, D, F, Do, mode, rng.choice(("swiglu", "situ")), rng.choice(("bf16", "bf16", "f16")))
    D = _log(rng, 64, 16384)
    M = _log(rng, 1, max(1, LARGEST_ELEMENTS // D))
    mode, dtype = rng.choice(("forward", "step")), rng.choice(("bf16", "f16", "f32"))
    if dtype == "f32":
        M = max(1, M // 2)
    if kind == "norm":
        return _norm("", M, D, rng.choice(("rms", "layer")), mode, dtype, rng.choice(("full", "full", "weight", "none")))
    return _dropout("", M, D, rng.choice((0.05, 0.1, 0.25, 0.5)), mode, dtype)


# ---------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DT[case["dtype"]]
    M, D = case["M"], case["D"]
    st = {"case": case}
    if case["kind"] == "ffn":
        F, Do, mode = case["F"], case["Do"], case["mode"]
        # normed hidden states, weights that keep the activations' size
        st["x"] = _randn(gen, M, D).to(dt)
        st["wg"] = (_randn(gen, F, D) / math.sqrt(D)).to(dt)
        st["wu"] = (_randn(gen, F, D) / math.sqrt(D)).to(dt)
        st["wd"] = (_randn(gen, Do, F) / math.sqrt(F)).to(dt)
        if mode == "adapters":
            st["gd"], st["ud"] = (0.1 * _randn(gen, M, F)).to(dt), (0.1 * _randn(gen, M, F)).to(dt)
            st["dh"] = (0.1 * _randn(gen, M, F)).to(dt)
        if mode != "forward":
            st["dy"] = _randn(gen, M, Do).to(dt)
            st["leaves"] = ["x", "gd", "ud"] if mode == "adapters" else ["x", "wg", "wu", "wd"]
    else:
        # rows of different size and offset, as residual streams have
        x = _randn(gen, M, D) * (0.5 + _randn(gen, M, 1).abs()) + 0.3 * _randn(gen, M, 1)
        st["x"] = x.to(dt)
        if case["mode"] == "step":
            st["dy"] = _randn(gen, M, D).to(dt)
            st["leaves"] = ["x"]
        if case["kind"] == "norm":
            st["w"] = st["b"] = None
            if case["affine"] != "none":
                st["w"] = 1 + 0.1 * _randn(gen, D)
                if case["affine"] == "full" and case["norm"] == "layer":
                    st["b"] = 0.1 * _randn(gen, D)
            if case["mode"] == "step":
                st["leaves"] += [n for n in ("w", "b") if st[n] is not None]
        else:
            st["seed"] = int(torch.randint(0, 2 ** 62, (1,), device="cuda", generator=gen).item())
            st["stream"] = seed % 7
    for n in st.get("leaves", ()):
        st[n].requires_grad_(True)
    return st


# ---------------------------------------------------------------- a pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return {"ffn": _plain_ffn, "norm": _plain_norm, "dropout": _plain_dropout}[case["kind"]](case, state)


def _run_own(case, st):
    from lazylora_amd import dense
    if case["kind"] == "ffn":
        if case["mode"] == "adapters":
            y, h = dense.gated_ffn(st["x"], st["wg"], st["wu"], st["wd"], act=case["act"], gate_delta=st["gd"],
                                   up_delta=st["ud"], return_hidden=True)
            return (y, h) + torch.autograd.grad((y, h), [st[n] for n in st["leaves"]], (st["dy"], st["dh"]))
        y = dense.gated_ffn(st["x"], st["wg"], st["wu"], st["wd"], act=case["act"])
    elif case["kind"] == "norm":
        if case["norm"] == "rms":
            y = dense.rms_norm(st["x"], st["w"], EPS)
        else:
            y = dense.layer_norm(st["x"], st["w"], st["b"], EPS)
    else:
        y = dense.dropout(st["x"], case["p"], st["seed"], st["stream"])
    if case["mode"] == "forward":
        return (y,)
    return (y,) + torch.autograd.grad(y, [st[n] for n in st["leaves"]], st["dy"])


EPS = 1e-5


# ---------------------------------------------------------------- plain forms
def _plain_ffn(case, st):
    dt, mode, act = DT[case["dtype"]], case["mode"], case["act"]
    x, wg, wu, wd = (st[n].float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.T, x @ wu.T
    if mode == "adapters":
        g, u = g + st["gd"].float(), u + st["ud"].float()
    s = 1 / (1 + torch.exp(-g))
    if act == "swiglu":
        a, b = g * s, u
    else:
        tg, tu = torch.tanh(g / 4), torch.tanh(u / 25)
        a, b = 4 * tg * s, 25 * tu
    h = a * b
    y = (h @ wd.T).to(dt)
    if mode == "forward":
        return (y,)
    dy = st["dy"].float()
    dh = dy @ wd
    if mode == "adapters":
        dh = dh + st["dh"].float()
    if act == "swiglu":
        da, db = s * (1 + g * (1 - s)), 1.0
    else:
        da, db = (1 - tg * tg) * s + 4 * tg * s * (1 - s), 1 - tu * tu
    dg, du = dh * b * da, dh * a * db
    dx = (dg @ wg + du @ wu).to(dt)
    if mode == "adapters":
        return (y, h.to(dt), dx, dg.to(dt), du.to(dt))
    return (y, dx, (dg.T @ x).to(dt), (du.T @ x).to(dt), (dy.T @ h).to(dt))


def _plain_norm(case, st):
    dt, layer = DT[case["dtype"]], case["norm"] == "layer"
    x = st["x"].float()
    xc = x - x.mean(-1, keepdim=True) if layer else x
    r = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * r
    y = xh if st["w"] is None else xh * st["w"]
    if st["b"] is not None:
        y = y + st["b"]
    if case["mode"] == "forward":
        return (y.to(dt),)
    dy = st["dy"].float()
    dxh = dy if st["w"] is None else dy * st["w"]
    dx = dxh - xh * (dxh * xh).mean(-1, keepdim=True)
    if layer:
        dx = dx - dxh.mean(-1, keepdim=True)
    out = [y.to(dt), (dx * r).to(dt)]
    if st["w"] is not None:
        out.append((dy * xh).sum(0))
    if st["b"] is not None:
        out.append(dy.sum(0))
    return tuple(out)


def _words(n, seed, stream):
    """The first n 32-bit words of Philox4x32-7 under `seed`, as int64: word i is lane i % 4 of the
    block with counter (i // 4 low, high, stream low, high)."""
    lo32 = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c = [block & lo32, block >> 32, torch.full_like(block, stream & lo32), torch.full_like(block, stream >> 32)]
    k0, k1 = seed & lo32, seed >> 32

    def mul(m, v):  # low and high half of a 32 x 32 bit product
        a, b = m * (v & 0xFFFF), m * (v >> 16)
        t = (a >> 16) + b
        return (a & 0xFFFF) | ((t & 0xFFFF) << 16), t >> 16

    for _ in range(7):
        l0, h0 = mul(0xD2511F53, c[0])
        l1, h1 = mul(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & lo32, (k1 + 0xBB67AE85) & lo32
    return torch.stack(c, 1).reshape(-1)[:n]


def _plain_dropout(case, st):
    x = st["x"]
    keep = (_words(x.numel(), st["seed"], st["stream"]) >= math.floor(case["p"] * 2 ** 32)).view_as(x)
    scale = 1 / (1 - case["p"])
    zero = torch.zeros((), device="cuda")
    y = torch.where(keep, x.float() * scale, zero).to(x.dtype)
    if case["mode"] == "forward":
        return (y,)
    return (y, torch.where(keep, st["dy"].float() * scale, zero).to(x.dtype))


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    v = {n: t.detach().double() for n, t in st.items() if torch.is_tensor(t)}
    for n in st.get("leaves", ()):
        v[n].requires_grad_(True)
    if case["kind"] == "ffn":
        g, u = v["x"].mm(v["wg"].t()), v["x"].mm(v["wu"].t())
        if "gd" in v:
            g, u = g + v["gd"], u + v["ud"]
        if case["act"] == "situ":
            h = 4 * (g / 4).tanh() * g.sigmoid() * 25 * (u / 25).tanh()
        else:
            h = g * g.sigmoid() * u
        y = h.mm(v["wd"].t())
        outs, ups = ((y, h), (v["dy"], v["dh"])) if case["mode"] == "adapters" else ((y,), (v.get("dy"),))
    elif case["kind"] == "norm":
        x = v["x"]
        if case["norm"] == "layer":
            y = (x - x.mean(1, True)) / (x.var(1, unbiased=False, keepdim=True) + EPS).sqrt()
        else:
            y = x / (x.square().mean(1, True) + EPS).sqrt()
        y = y * v["w"] if "w" in v else y
        y = y + v["b"] if "b" in v else y
        outs, ups = (y,), (v.get("dy"),)
    else:
        x = v["x"]
        rows = [w >= int(case["p"] * 4294967296) for w in _counted_words(x.numel(), st["seed"], st["stream"])]
        keep = torch.stack(rows, 1).flatten()[:x.numel()].reshape(x.shape)
        y = (x / (1 - case["p"])).masked_fill(~keep, 0)
        outs, ups = (y,), (v.get("dy"),)
    if case["mode"] == "forward":
        return tuple(o.detach() for o in outs)
    grads = torch.autograd.grad(outs, [v[n] for n in st["leaves"]], ups)
    return tuple(o.detach() for o in outs) + grads


def _counted_words(n, seed, stream):
    """The four words of each Philox4x32-7 block, products taken modulo 2^64 in two's complement."""
    m32 = 4294967295

    def wide(a, b):
        p = a * b
        return p & m32, (p >> 32) & m32

    i = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    x0, x1 = i & m32, (i >> 32) & m32
    x2, x3 = torch.full_like(i, stream & m32), torch.full_like(i, (stream >> 32) & m32)
    for r in range(7):
        ka, kb = ((seed & m32) + r * 0x9E3779B9) & m32, ((seed >> 32) + r * 0xBB67AE85) & m32
        la, ha = wide(x0, 0xD2511F53)
        lb, hb = wide(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = hb ^ x1 ^ ka, lb, ha ^ x3 ^ kb, la
    return x0, x1, x2, x3


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    M, D, e = case["M"], case["D"], BYTES[case["dtype"]]
    if case["kind"] == "ffn":
        F, Do, mode = case["F"], case["Do"], case["mode"]
        weights = 2 * F * D + Do * F
        forward = 2.0 * M * weights
        if mode == "forward":
            return {"bytes": e * (M * D + weights + M * Do), "flops": forward}
        step = e * (2 * M * D + weights + 2 * M * Do)  # x, dx, the weights, y, dy
        if mode == "adapters":  # two deltas and their gradients, h and its upstream gradient
            return {"bytes": step + 6 * e * M * F, "flops": 2 * forward}
        return {"bytes": step + e * weights, "flops": 3 * forward}
    n = M * D
    tensors = 4 if case["mode"] == "step" else 2  # x, y, dy, dx
    if case["kind"] == "dropout":
        return {"bytes": tensors * n * e, "flops": 0.0}
    vectors = 0
    if case["affine"] != "none":
        vectors = 2 if case["norm"] == "layer" and case["affine"] == "full" else 1
    vectors *= 2 if case["mode"] == "step" else 1
    return {"bytes": tensors * n * e + 4 * vectors * D, "flops": (12.0 if case["mode"] == "step" else 5.0) * n}
