"""
Products with 4-bit integer weights on MI355X, for serving: a matrix [R, K] as codes, two to a byte (low
nibble = even element, as in the MXFP4 checkpoints, lazy_lora/native/mxfp4_gemm.c:12-15), with a 16-bit
scale and a zero point for every 32, 64 or 128 codes of a row,

    W[r, k] = scales[r, k // group] * (code[r, k] - zeros[r, k // group]).

    from lazylora_amd.int4 import Int4Experts, Int4Weight, int4_gemm, int4_routed

`int4_gemm` is one product, `int4_routed` a routed expert layer over stacked matrices, from one token on.
Both run in hand-written kernels (csrc/mx_int4.hip) on the current stream of their tensors' device, raise
ValueError for tensors they do not take and have no backward pass (NotImplementedError where a gradient
would be recorded); nothing falls back to torch. The codes enter the products exactly, sums are fp32, each
result is rounded once.
"""
from typing import Optional, Tuple

import torch

from lazylora_amd.dense import _module
from lazylora_amd.native import _ACTS

GROUPS = (32, 64, 128)


def _tidy(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned, as the kernels take it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class Int4Weight:
    """A matrix [R, K] of 4-bit codes, or E of them stacked: packed uint8 [(E,) R, K / 2], scales bfloat16 or
    float16 [(E,) R, K / group], zeros uint8 of the scales' shape, or None: 8 everywhere (symmetric codes). The
    tensors are kept as they are where they are contiguous and 16-byte aligned; `shape` is [(E,) R, K]."""

    __slots__ = ("packed", "scales", "zeros", "shape", "group")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None):
        if packed.dtype != torch.uint8 or packed.dim() not in (2, 3):
            raise ValueError(f"packed must be uint8 [R, K / 2] or [E, R, K / 2], got {packed.dtype} {tuple(packed.shape)}")
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"scales must be bfloat16 or float16, got {scales.dtype}")
        K, n = 2 * packed.shape[-1], scales.shape[-1] if scales.dim() else 0
        if scales.shape[:-1] != packed.shape[:-1] or n == 0 or K % n or K // n not in GROUPS:
            raise ValueError(f"scales {tuple(scales.shape)} do not hold one number for every 32, 64 or 128 codes of a row "
                             f"of {tuple(packed.shape[:-1]) + (K,)}")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError(f"zeros must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
        if scales.device != packed.device or (zeros is not None and zeros.device != packed.device):
            raise ValueError("codes, scales and zeros must lie on one device")
        self.packed, self.scales, self.zeros = _tidy(packed), _tidy(scales), None if zeros is None else _tidy(zeros)
        self.shape: Tuple[int, ...] = tuple(packed.shape[:-1]) + (K,)
        self.group = K // n

    def to(self, device) -> "Int4Weight":
        return Int4Weight(self.packed.to(device), self.scales.to(device),
                          None if self.zeros is None else self.zeros.to(device))


class Int4Experts:
    """One layer's experts with 4-bit weights: w1 (gate) and w3 (up) [E, F, D], w2 (down) [E, D, F], all of one
    group size. LatentMoEBlock takes it in an ExpertLayer's place, for inference."""

    def __init__(self, w1: Int4Weight, w3: Int4Weight, w2: Int4Weight):
        if any(len(w.shape) != 3 for w in (w1, w3, w2)):
            raise ValueError("an expert layer needs stacked matrices [E, R, K]")
        self.E, self.F, self.D = w1.shape
        if w3.shape != w1.shape or w2.shape != (self.E, self.D, self.F):
            raise ValueError(f"w1 and w3 must be [E, F, D] and w2 [E, D, F], got {w1.shape}, {w3.shape} and {w2.shape}")
        if not w1.group == w3.group == w2.group:
            raise ValueError(f"the matrices must have one group size, got {w1.group}, {w3.group} and {w2.group}")
        if any((w.zeros is None) != (w1.zeros is None) for w in (w3, w2)):
            raise ValueError("zero points must be given for all three matrices or for none")
        if any(w.scales.dtype != w1.scales.dtype or w.packed.device != w1.packed.device for w in (w3, w2)):
            raise ValueError("the matrices must have scales of one type and lie on one device")
        self.w1, self.w3, self.w2 = w1, w3, w2

    @property
    def device(self) -> torch.device:
        return self.w1.packed.device

    @property
    def dtype(self) -> torch.dtype:
        """The type of the scales, which is that of the activations."""
        return self.w1.scales.dtype


def int4_gemm(x: torch.Tensor, weight: Int4Weight) -> torch.Tensor:
    """y [..., R] = x [..., K] W^T, x and y of the scales' type (bfloat16 or float16). A row of x with an infinity
    gives NaN, and so does one with numbers past fp32's range in the sum of |x| max(31, 16 + zero) over a group (none
    below 2^111 is, and no float16). Scales have to be finite."""
    return _module().int4_gemm(x, weight.packed, weight.scales, weight.zeros)


def int4_routed(h: torch.Tensor, topk_indices: torch.Tensor, topk_weights: torch.Tensor, experts: Int4Experts,
                act: str = "swiglu") -> torch.Tensor:
    """sum over the slots j of topk_weights[t, j] * W2_e GLU(W1_e h[t], W3_e h[t]), e = topk_indices[t, j], for h
    [N, D] of the scales' type; the result is of that type too, and so are the GLU's results in between (a SwiGLU
    value past float16's 65504 is an infinity, and the token's result NaN; bfloat16 and "situ" do not reach that).
    topk_indices int32 or int64 [N, k], as the router gives them (ids outside [0, E) contribute nothing),
    topk_weights [N, k] of any floating type; act "swiglu" or "situ"."""
    if act not in _ACTS:
        raise ValueError(f"unknown activation {act!r}")
    w1, w3, w2 = experts.w1, experts.w3, experts.w2
    return _module().int4_routed(h, topk_indices, topk_weights, w1.packed, w1.scales, w1.zeros, w3.packed, w3.scales,
                                 w3.zeros, w2.packed, w2.scales, w2.zeros, _ACTS[act])
