"""
The dense operators of the latent MoE block on MI355X, differentiable: the gated feed-forward
block (the shared expert, lazy_lora/trainer/lazy_trainer.py:702-708), layer and RMS norm
(RMSNormFunction, lazy_lora/streaming/trunk_streamer.py:23-34) and the adapters' dropout
(LazyLoRALinear.forward_lora_only, lazy_lora/core/lora_layer.py:104-139).

    from lazylora_amd.dense import gated_ffn, layer_norm, rms_norm, dropout

They run in hand-written kernels (csrc/mx_dense.hip, csrc/mx_rows.hip) on the current stream of
their tensors' device and raise ValueError for tensors they do not take; nothing falls back to torch.
Sums, statistics and activation functions are fp32 whatever the tensors' type, and each result is
rounded once. Results do not depend on timing (no atomics). Without a gradient to record a call
saves nothing; a second derivative is refused by autograd.
"""
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from lazylora_amd.native import _ACTS, _FLOATS, NORM_LAYER, NORM_RMS, _aligned, kernel


def _native():
    k = kernel()
    if k is None:
        raise RuntimeError("the MI355X dense operators are unavailable: LAZYLORA_NO_NATIVE=1 is set, or the native "
                           "library failed to load, or no HIP device is visible (set LAZYLORA_NATIVE_STRICT=1 to see "
                           "the underlying error)")
    return k


def _records(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# The backward functions run in autograd's own thread, where host work costs several times what it does in
# the caller's (a step of a small norm: 123 us with the checks and conversions of a public call in its
# backward, 91 without), so they take what their forward has checked and call the inner entry points.
def _once(impl):
    """A backward that autograd may run but not differentiate: once_differentiable where a graph of it
    is asked for (create_graph=True), the plain function, which is quicker, elsewhere."""
    guarded = once_differentiable(impl)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else impl(ctx, *grads)

    return staticmethod(backward)


def _tidy(t):
    return t if t is None else _aligned(t.contiguous())


def _ffn_grads(ctx, grad_y, grad_h=None):
    x, w_gate, w_up, w_down, h, gu = ctx.saved_tensors
    if grad_y is None and grad_h is None:
        return (None,) * 8
    need = ctx.needs_input_grad
    if grad_y is None:  # only h was used
        grad_y = grad_h.new_zeros((grad_h.shape[0], w_down.shape[0]))
    dgu, dx, dwg, dwu, dwd = ctx.k._ffn_backward(
        _tidy(grad_y), gu, (_tidy(w_gate), _tidy(w_up), _tidy(w_down)), _FLOATS[w_gate.dtype], _ACTS[ctx.act],
        _tidy(grad_h), _tidy(x), _tidy(h), need[0])
    F = w_gate.shape[0]
    return (dx, dwg if need[1] else None, dwu if need[2] else None, dwd, dgu[:, :F] if need[4] else None,
            dgu[:, F:] if need[5] else None, None, None)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, gate_delta, up_delta, act, return_hidden):
        ctx.k = _native()
        y, h, gu = ctx.k.ffn_forward(x, w_gate, w_up, w_down, act, gate_delta, up_delta, save_for_backward=True)
        need = ctx.needs_input_grad
        # what the products of the wanted gradients read: x for the gate and up weights, h for the down weight
        ctx.save_for_backward(x if need[1] or need[2] else None, w_gate, w_up, w_down, h if need[3] else None, gu)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return (y, h) if return_hidden else y

    backward = _once(_ffn_grads)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, act: str = "swiglu",
              gate_delta: Optional[torch.Tensor] = None, up_delta: Optional[torch.Tensor] = None,
              return_hidden: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y = GLU(x Wg^T + gate_delta, x Wu^T + up_delta) Wd^T for x [..., D], w_gate and w_up [F, D], w_down
    [Do, F], all bfloat16 or all float16, D, F and Do multiples of 8; act "swiglu" or "situ".

    gate_delta and up_delta [..., F] are added to the products before the activation (an adapter's terms;
    either may be None). With return_hidden the result is (y, h), h the hidden activations [..., F] that
    the down product reads: a down adapter takes them, and its gradient comes back through h.
    Differentiable in x, the weights and the deltas. For a backward the fp32 gate and up sums are kept
    (8 bytes per row and hidden feature): rounded to 16 bits they would add the same error again that
    the rounding of their gradients has."""
    lead = x.shape[:-1]
    flat = lambda t: t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if x.dim() == 0 or any(t is not None and t.shape[:-1] != lead for t in (gate_delta, up_delta)):
        raise ValueError("x and the deltas must agree in all axes but the last")
    x, gate_delta, up_delta = flat(x), flat(gate_delta), flat(up_delta)
    if _records(x, w_gate, w_up, w_down, gate_delta, up_delta):
        out = _GatedFfn.apply(x, w_gate, w_up, w_down, gate_delta, up_delta, act, return_hidden)
        y, h = out if return_hidden else (out, None)
    else:
        y, h, _ = _native().ffn_forward(x, w_gate, w_up, w_down, act, gate_delta, up_delta)
    if len(lead) != 1:
        y = y.reshape(lead + y.shape[-1:])
        h = h if h is None else h.reshape(lead + h.shape[-1:])
    return (y, h) if return_hidden else y


def _norm_grads(ctx, grad_y):
    x, weight, stats = ctx.saved_tensors
    _, need_w, need_b, _, _ = ctx.needs_input_grad
    dx, dw, db = ctx.k._norm_backward(grad_y, x, weight, stats, ctx.kind, need_w, need_b)
    if need_w and ctx.weight_dtype != torch.float32:
        dw = dw.to(ctx.weight_dtype)
    if need_b and ctx.bias_dtype != torch.float32:
        db = db.to(ctx.bias_dtype)
    return dx, dw, db, None, None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, kind):
        ctx.k = _native()
        if weight is not None:
            ctx.weight_dtype = weight.dtype
            weight = weight.float().contiguous()
        if bias is not None:
            ctx.bias_dtype = bias.dtype
            bias = bias.float()
        x = x.contiguous()
        y, stats = ctx.k.norm_forward(x, weight, bias, eps, kind, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.kind = kind
        return y

    backward = _once(_norm_grads)


def _norm(x, weight, bias, eps, kind):
    if x.dim() == 0:
        raise ValueError("x must have at least one axis")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.reshape(0, 0)
    if _records(x2, weight, bias):
        y = _Norm.apply(x2, weight, bias, eps, kind)
    else:
        w, b = (None if t is None else t.float() for t in (weight, bias))
        y, _ = _native().norm_forward(x2, w, b, eps, kind)
    return y if x.dim() == 2 else y.reshape(x.shape)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, var the mean square distance
    from the mean. x float32, bfloat16 or float16; weight and bias [D] of any floating type, or None.
    Differentiable in all three."""
    return _norm(x, weight, bias, eps, NORM_LAYER)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last axis (trunk_streamer.py:23-34); types as in
    layer_norm. Differentiable in x and weight."""
    return _norm(x, weight, None, eps, NORM_RMS)


def _dropout_grad(ctx, grad_y):
    seed = ctx.seed if ctx.seed is not None else ctx.saved_tensors[0]
    return ctx.k._dropout(grad_y, ctx.p, seed, ctx.stream), None, None, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, stream):
        ctx.k, ctx.p, ctx.seed, ctx.stream = _native(), p, seed, stream
        if torch.is_tensor(seed):  # saved, so that autograd notices a seed changed before the backward
            ctx.save_for_backward(seed)
            ctx.seed = None
        return ctx.k.dropout(x, p, seed, stream)

    backward = _once(_dropout_grad)


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], stream: int = 0) -> torch.Tensor:
    """x / (1 - p) where kept, 0 where dropped (each element with probability p, to 2^-32). The mask is a
    function of (seed, stream, element number in row-major order) and of nothing else: nothing is stored
    for the backward, and a recomputed forward with the same numbers drops the same elements. seed: a
    whole number in [0, 2^64), or a one-element int64 tensor on x's device, which the kernel reads (a
    captured graph draws a new mask when it changes between replays). stream tells the calls under one
    seed apart (one number per adapter, say). x float32, bfloat16 or float16; p in [0, 1]."""
    if _records(x):
        return _Dropout.apply(x, p, seed, stream)
    return _native().dropout(x, p, seed, stream)
