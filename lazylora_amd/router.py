"""
The Kimi-K3 MoE router on MI355X, with the interface of lazy_lora/core/moe_router.py.

`KimiK3MoERouter.forward(x, weight, bias)` returns (topk_indices [N, k] int64, topk_weights
[N, k] fp32) like the reference (moe_router.py:55-123): the gate product logits = x . W^T runs
in fp32 in the platform BLAS (a plain dense GEMM), and the selection -- sigmoid scores, bias
added for selection only, top-k in descending order, unbiased scores gathered, renormalised
with +1e-20, scaled -- runs in one HIP kernel, one wave per token, so the indices feed the
routed-expert layer without a host round trip. Gradients flow from topk_weights back through
the logits into x (and the gate weight, if it requires grad), as torch autograd does through the
reference's torch branch; the trainer relies on that (lazy_lora/trainer/lazy_trainer.py:842-844).

`select_experts` is the same step for routers of other forms, from logits of any floating type: softmax or
sigmoid scores, a choice limited to the best groups of experts, with its gradient; `route`,
KimiK3MoERouter and LatentMoEBlock take its options.

Differences from the reference, all deliberate:
  * equal biased scores go to the lower expert id first (torch.topk leaves their order
    unspecified; the NumPy branch's argsort is not stable either);
  * results land on x's device (CPU and NumPy inputs are computed on the GPU and copied
    back); a missing library raises instead of falling back to a CPU path;
  * top_k <= 64 and num_experts <= 4096 (the reference configurations use 16 of 896).
"""
from typing import List, Optional, Tuple, Union

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F

from lazylora_amd.dense import _module
from lazylora_amd.native import GROUP_SCORES, SCORINGS, kernel


def _native():
    k = kernel()
    if k is None:
        raise RuntimeError("LAZYLORA_NO_NATIVE=1: the MI355X router is disabled")
    return k


class _Select(torch.autograd.Function):
    """Selection on device logits; backward gives dL/dlogits from dL/dtopk_weights."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, scale, renormalize):
        idx, w = _native().router_topk(logits, bias, top_k, scale, renormalize)
        ctx.mark_non_differentiable(idx)
        ctx.save_for_backward(logits, idx)
        ctx.scale, ctx.renormalize = scale, renormalize
        return idx, w

    @staticmethod
    def backward(ctx, _grad_idx, grad_w):
        logits, idx = ctx.saved_tensors
        grad_logits = None
        if grad_w is not None and ctx.needs_input_grad[0]:
            grad_logits = _native().router_topk_backward(logits, idx, grad_w, ctx.scale, ctx.renormalize)
        # the bias only steers the (non-differentiable) selection: no gradient, as in torch
        return grad_logits, None, None, None, None


def check_options(scoring: str, group_score: str) -> None:
    if not (isinstance(scoring, str) and scoring in SCORINGS):
        raise ValueError(f"unknown scoring {scoring!r}")
    if not (isinstance(group_score, str) and group_score in GROUP_SCORES):
        raise ValueError(f"unknown group score {group_score!r}")


def select_experts(logits: torch.Tensor, top_k: int, bias: Optional[torch.Tensor] = None, scoring: str = "sigmoid",
                   num_groups: int = 1, topk_groups: Optional[int] = None, group_score: str = "top2",
                   renormalize: bool = True, routed_scaling_factor: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(topk_indices [..., top_k] int64, topk_weights [..., top_k] fp32) from router logits [..., E] (float32,
    bfloat16 or float16, on the HIP device), differentiable in the logits.

    Scores are sigmoid(logits) or softmax(logits) (`scoring`); the choice goes by score + bias (bias [E] of any
    floating type, float64 too taken as float32; for the choice only: no gradient), the weights are the chosen scores, divided by their sum +
    1e-20 with `renormalize` (and top_k > 1), times routed_scaling_factor. With num_groups > 1 the experts form
    that many equal runs and only the topk_groups best of them (None: all) can be chosen from, by the sum of
    each group's two largest values of score + bias (group_score "top2") or by its largest ("max").

    Indices are in descending order of score + bias in 64 bits (without a bias: of the logits), and so are the
    groups; values that are equal there, as sigmoid(38) and sigmoid(45) under one bias are, go to the lower id,
    equal groups to the lower number, NaN comes first. A softmax row of -inf alone has weights 0. E <= 4096 (where num_groups is no power of two, 64 * 64 experts
    for the next power of two of groups), num_groups <= 64, top_k <= min(64, experts of the kept groups).
    Second derivatives, forward-mode differentiation, tracing and function transforms raise, as in lazylora_amd.dense."""
    check_options(scoring, group_score)
    return _module().select_experts(logits, bias, top_k, SCORINGS[scoring], num_groups,
                            num_groups if topk_groups is None else topk_groups, GROUP_SCORES[group_score],
                            routed_scaling_factor, renormalize)


def route(x: Union[torch.Tensor, np.ndarray], weight: Union[torch.Tensor, np.ndarray],
          bias: Optional[Union[torch.Tensor, np.ndarray]] = None, top_k: int = 16,
          routed_scaling_factor: float = 1.0, renormalize: bool = True, scoring: str = "sigmoid",
          num_groups: int = 1, topk_groups: Optional[int] = None, group_score: str = "top2"):
    """(topk_indices [N, k] int64, topk_weights [N, k] fp32) for tokens x [..., hidden] and gate
    weight [E, hidden] (moe_router.py:81-99). NumPy in, NumPy out; torch tensors come back on
    x's device. scoring, num_groups, topk_groups and group_score as in select_experts, which makes the
    selection unless they are the reference's (sigmoid, one group)."""
    check_options(scoring, group_score)
    as_numpy = isinstance(x, np.ndarray)
    xt = torch.from_numpy(np.asarray(x, np.float32)) if as_numpy else x
    if xt.is_cuda:
        dev = xt.device
    elif torch.cuda.is_available():
        dev = torch.device("cuda", torch.cuda.current_device())
    else:
        raise RuntimeError("the MI355X router needs a HIP device (torch.cuda.is_available() is False)")
    w = torch.as_tensor(weight).to(dev, torch.float32)
    if w.dim() != 2:
        raise ValueError(f"weight must be [num_experts, hidden], got {tuple(w.shape)}")
    hidden = w.shape[1]
    if xt.shape[-1] != hidden:
        raise ValueError(f"x has width {xt.shape[-1]} but the gate takes {hidden}")
    b = None if bias is None else torch.as_tensor(bias).to(dev, torch.float32)
    logits = F.linear(xt.reshape(-1, hidden).to(dev, torch.float32), w)   # [N, E] fp32
    if scoring == "sigmoid" and num_groups == 1 and topk_groups in (None, 1):
        idx, tw = _Select.apply(logits, b, int(top_k), float(routed_scaling_factor), bool(renormalize))
    else:
        idx, tw = select_experts(logits, int(top_k), b, scoring, num_groups, topk_groups, group_score,
                                 bool(renormalize), float(routed_scaling_factor))
    if as_numpy:
        return idx.cpu().numpy(), tw.detach().cpu().numpy()
    if not xt.is_cuda:
        return idx.to(xt.device), tw.to(xt.device)
    return idx, tw


class KimiK3MoERouter(nn.Module):
    """KimiK3MoERouter (lazy_lora/core/moe_router.py:23-135) with the selection on MI355X; scoring and the
    group arguments as in select_experts."""

    scoring, num_groups, topk_groups, group_score = "sigmoid", 1, None, "top2"  # of modules saved without them

    def __init__(self, hidden_size: int = 7168, num_experts: int = 896, top_k: int = 16,
                 routed_scaling_factor: float = 1.0, renormalize: bool = True, use_bias: bool = True,
                 device: Optional[Union[str, torch.device]] = None, scoring: str = "sigmoid", num_groups: int = 1,
                 topk_groups: Optional[int] = None, group_score: str = "top2"):
        check_options(scoring, group_score)
        super().__init__()
        self.weight = nn.Parameter(torch.empty(num_experts, hidden_size, device=device))
        self.bias = nn.Parameter(torch.zeros(num_experts, device=device)) if use_bias else None
        nn.init.normal_(self.weight, std=0.02)
        self.hidden_size = hidden_size
        self.num_experts = num_experts
        self.top_k = top_k
        self.routed_scaling_factor = routed_scaling_factor
        self.renormalize = renormalize
        self.use_bias = use_bias
        self.scoring, self.num_groups, self.topk_groups, self.group_score = scoring, num_groups, topk_groups, group_score

    def forward(self, x, weight=None, bias=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(topk_indices [N, top_k] int64, topk_weights [N, top_k] fp32). `weight`/`bias`
        override the module's own (each layer streams its own gate, moe_router.py:68-73)."""
        if weight is None:
            weight = self.weight
        if bias is None:
            bias = self.bias
        return route(x, weight, bias, self.top_k, self.routed_scaling_factor, self.renormalize, self.scoring,
                     self.num_groups, self.topk_groups, self.group_score)

    @staticmethod
    def get_active_expert_set(topk_indices) -> List[int]:
        """Sorted unique expert ids of a batch (moe_router.py:125-135)."""
        if isinstance(topk_indices, torch.Tensor):
            ids = torch.unique(topk_indices).cpu().tolist()
        else:
            ids = np.unique(np.asarray(topk_indices)).tolist()
        return sorted(int(e) for e in ids)
