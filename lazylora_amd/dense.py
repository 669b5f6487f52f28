"""
The dense operators of the latent MoE block on MI355X, differentiable: the gated feed-forward
block (the shared expert, lazy_lora/trainer/lazy_trainer.py:702-708), layer and RMS norm
(RMSNormFunction, lazy_lora/streaming/trunk_streamer.py:23-34) and the adapters' dropout
(LazyLoRALinear.forward_lora_only, lazy_lora/core/lora_layer.py:104-139).

    from lazylora_amd.dense import gated_ffn, layer_norm, rms_norm, dropout

They run in hand-written kernels (csrc/mx_dense.hip, csrc/mx_rows.hip), as autograd functions in C++
(csrc/dense_autograd.cpp), on the current stream of their tensors' device, and raise ValueError for
tensors they do not take; nothing falls back to torch. Sums, statistics and activation functions are
fp32 whatever the tensors' type, and each result is rounded once. Results do not depend on timing (no
atomics). Without a gradient to record a call saves nothing; a second derivative raises. So do
forward-mode differentiation and tracing (torch.jit.trace, make_fx; NotImplementedError): a launch
would drop a tangent and leave no trace. torch.compile breaks its graph at a call.
"""
from typing import Optional, Tuple, Union

import torch

from lazylora_amd.native import _ACTS, NORM_LAYER, NORM_RMS, kernel

_ext = None


def _module():
    """The autograd module; RuntimeError where the native library is off or unavailable."""
    global _ext
    if kernel() is None:
        raise RuntimeError("the MI355X dense operators are unavailable: LAZYLORA_NO_NATIVE=1 is set, or the native "
                           "library failed to load, or no HIP device is visible (set LAZYLORA_NATIVE_STRICT=1 to see "
                           "the underlying error)")
    if _ext is None:
        try:
            from lazylora_amd import _dense_autograd
        except ImportError as exc:
            raise RuntimeError("lazylora_amd/_dense_autograd is missing or does not load: build it with "
                               f"`python -m lazylora_amd.build` (or __graft_entry__.build()): {exc}") from exc
        _ext = _dense_autograd
    return _ext


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
    if act not in _ACTS:
        raise ValueError(f"unknown activation {act!r}")
    out = _module().gated_ffn(x, w_gate, w_up, w_down, _ACTS[act], gate_delta, up_delta, return_hidden)
    return tuple(out) if return_hidden else out[0]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, var the mean square distance
    from the mean. x float32, bfloat16 or float16; weight and bias [D] of any floating type (float64 too is
    taken as float32), or None.
    Differentiable in all three."""
    return _module().norm(x, weight, bias, eps, NORM_LAYER)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last axis (trunk_streamer.py:23-34); types as in
    layer_norm. Differentiable in x and weight."""
    return _module().norm(x, weight, None, eps, NORM_RMS)


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], stream: int = 0) -> torch.Tensor:
    """x / (1 - p) where kept, 0 where dropped (each element with probability p, to 2^-32). The mask is a
    function of (seed, stream, element number in row-major order) and of nothing else: nothing is stored
    for the backward, and a recomputed forward with the same numbers drops the same elements. seed: a
    whole number in [0, 2^64), or a one-element int64 tensor on x's device, which the kernel reads (a
    captured graph draws a new mask when it changes between replays; changed between a forward and its
    backward it raises). stream tells the calls under one seed apart (one number per adapter, say).
    x float32, bfloat16 or float16; p in [0, 1]."""
    where = seed if isinstance(seed, torch.Tensor) else None
    number = 0 if where is not None else seed
    if not (0 <= number < 2 ** 64 and 0 <= stream < 2 ** 64):
        raise ValueError(f"seed and stream must lie in [0, 2^64), got {seed} and {stream}")
    return _module().dropout(x, p, number, where, stream)
