"""
The Kimi-K3 latent MoE block of one layer on MI355X, around the routed-expert kernels.

Mirrors LazyLoRATrainer._run_layer's MoE half and _moe_forward
(lazy_lora/trainer/lazy_trainer.py:689-737):
  * route: KimiK3MoERouter on the normed hidden state (moe_router.py:55-123; here the device
    router of lazylora_amd.router, so indices never leave the GPU);
  * shared expert at full width: GLU(x W1^T + LoRA, x W3^T + LoRA) W2^T + LoRA (:703-708);
  * routed experts in the latent space: h_latent = x W_down^T (:727), the routed sum
    (RoutedExpertsFunction, :728-730, the MXFP4 kernels), RMSNorm of the sum with its weight
    (RMSNormFunction, lazy_lora/streaming/trunk_streamer.py:23-34; :733), up-projection (:734);
  * out = shared + routed (:736).
The dense projections (shared expert, latent down/up) are plain GEMMs and run in the platform
BLAS through torch, in fp32; the whole block is differentiable in x (through the router's
weights too, as in the reference) and in any LoRA factor that requires grad; the routed
adapters' gradients are accumulated into them by the routed node, as in the reference.

With dense="native" the shared expert runs in 16 bits through the gated feed-forward kernels
(lazylora_amd.dense.gated_ffn; the checkpoint's dense weights are bfloat16, so bfloat16 holds them
exactly) and the norm of the routed sum through the norm kernels, forward and backward.

For inference the experts can be an Int4Experts (lazylora_amd.int4), 4-bit integer weights with group scales; and
the router may have softmax scores or choose among groups of experts (lazylora_amd.router.select_experts).
"""
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn.functional as F

from lazylora_amd.dense import dropout, gated_ffn
from lazylora_amd.dense import rms_norm as native_rms_norm
from lazylora_amd.experts import ExpertLayer
from lazylora_amd.int4 import Int4Experts, int4_routed
from lazylora_amd.routed import RoutedExpertsFunction
from lazylora_amd.router import check_options, route

SITU_BETA, SITU_LINEAR_BETA = 4.0, 25.0  # lazy_lora/core/situ_activation.py:22-23


def glu(g: torch.Tensor, u: torch.Tensor, act: str) -> torch.Tensor:
    """SiTU-GLU (situ_activation.py:47-75) or SwiGLU, in torch (the shared expert's dense path)."""
    if act in ("situ", "situ_glu"):
        return SITU_BETA * torch.tanh(g / SITU_BETA) * torch.sigmoid(g) * (SITU_LINEAR_BETA * torch.tanh(u / SITU_LINEAR_BETA))
    if act == "swiglu":
        return F.silu(g) * u
    raise ValueError(f"unknown activation {act!r}")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-5) -> torch.Tensor:
    """RMSNormFunction.forward (trunk_streamer.py:23-34)."""
    out = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    return out * weight if weight is not None else out


def lora_delta(x: torch.Tensor, mod, dropout_seed=None, stream: int = 0) -> torch.Tensor:
    """forward_lora_only (lora_layer.py:104-139): s (drop(x) A^T) B^T, fp32. Dropout at the adapter's
    dropout_rate with a seed (and a number that tells adapters under it apart), off without one."""
    if mod is None:
        return 0.0
    p = float(getattr(mod, "dropout_rate", 0.0) or 0.0)
    if dropout_seed is not None and p > 0.0:
        x = dropout(x, p, dropout_seed, stream)
    A = mod.lora_A.to(x.device, torch.float32)
    B = mod.lora_B.to(x.device, torch.float32)
    return float(mod.scaling) * F.linear(F.linear(x, A), B)


class LatentMoEBlock:
    """One MoE layer: router, shared expert, latent projections, routed MXFP4 experts, norm.

    Weights follow the checkpoint's names (scripts/make_tiny_model.py:134-146 lists them):
    gate.weight [E, H], gate.e_score_correction_bias [E], shared_experts.{gate,up,down}_proj
    [Ds, H] / [Ds, H] / [H, Ds], routed_expert_down_proj [Dl, H], routed_expert_up_proj [H, Dl],
    routed_expert_norm [Dl]; the experts as an ExpertLayer of the latent width Dl. `lora` is the
    layer's adapter bundle (gate_lora / up_lora / down_lora for the routed experts and
    shared_gate_lora / shared_up_lora / shared_down_lora for the shared expert, any of them absent
    or None), as the reference's LayerLoRABundle (lazy_trainer.py:124-134).

    dense: "torch" (fp32 BLAS) or "native" (the shared expert in dense_dtype, torch.bfloat16 or
    torch.float16, through the feed-forward kernels, and the norm through the norm kernels; the hidden
    and shared widths must be multiples of 8).

    scoring, num_groups, topk_groups and group_score as in select_experts. experts may be an Int4Experts: the
    routed products then run in its scales' type, without routed adapters, and where a gradient would be
    recorded a call raises NotImplementedError, with a cached sum as without.
    """

    def __init__(self, experts: Union[ExpertLayer, Int4Experts], gate_weight, gate_bias, shared_w1, shared_w3, shared_w2, latent_down,
                 latent_up, latent_norm=None, top_k: int = 16, routed_scaling_factor: float = 1.0,
                 renormalize: bool = True, act: str = "situ", rms_eps: float = 1e-5, lora=None,
                 dense: str = "torch", dense_dtype: torch.dtype = torch.bfloat16, scoring: str = "sigmoid",
                 num_groups: int = 1, topk_groups: Optional[int] = None, group_score: str = "top2"):
        if dense not in ("torch", "native"):
            raise ValueError(f'dense must be "torch" or "native", got {dense!r}')
        check_options(scoring, group_score)
        dev = experts.device
        f32 = lambda t: None if t is None else torch.as_tensor(t).to(dev, torch.float32)
        self.experts = experts
        self.gate_weight, self.gate_bias = f32(gate_weight), f32(gate_bias)
        self.native, self.dense_dtype = dense == "native", dense_dtype
        shared_dtype = dense_dtype if self.native else torch.float32
        self.shared = tuple(torch.as_tensor(t).to(dev, shared_dtype) for t in (shared_w1, shared_w3, shared_w2))
        self.latent_down, self.latent_up, self.latent_norm = f32(latent_down), f32(latent_up), f32(latent_norm)
        self.top_k, self.routed_scaling_factor, self.renormalize = top_k, routed_scaling_factor, renormalize
        self.act, self.rms_eps, self.lora = act, rms_eps, lora
        self.scoring, self.num_groups, self.topk_groups, self.group_score = scoring, num_groups, topk_groups, group_score
        self._check_adapters()
        H = self.gate_weight.shape[1]
        if self.latent_down.shape != (experts.D, H) or self.latent_up.shape != (H, experts.D):
            raise ValueError(f"latent projections must be [{experts.D}, {H}] and [{H}, {experts.D}]")
        if self.native:
            if dense_dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"dense_dtype must be torch.bfloat16 or torch.float16, got {dense_dtype}")
            if H % 8 or self.shared[0].shape[0] % 8:
                raise ValueError(f'dense="native" needs hidden and shared widths that are multiples of 8, got {H} and '
                                 f"{self.shared[0].shape[0]}")
        self.hidden = H

    def _adapter(self, name: str):
        return getattr(self.lora, name, None) if self.lora is not None else None

    def _routed_lora(self):
        mods = tuple(self._adapter(n) for n in ("gate_lora", "up_lora", "down_lora"))
        return mods if all(m is not None for m in mods) else None

    def _shared(self, x: torch.Tensor, seed) -> torch.Tensor:
        """The shared expert with its adapters (lazy_trainer.py:703-708), fp32."""
        W1, W3, W2 = self.shared
        delta = lambda v, name, stream: lora_delta(v, self._adapter(name), seed, stream)
        d_gate, d_up = delta(x, "shared_gate_lora", 0), delta(x, "shared_up_lora", 1)
        if not self.native:
            s_act = glu(F.linear(x, W1) + d_gate, F.linear(x, W3) + d_up, self.act)
            return F.linear(s_act, W2) + delta(s_act, "shared_down_lora", 2)
        low = lambda d: d.to(self.dense_dtype) if torch.is_tensor(d) else None
        y, s_act = gated_ffn(x.to(self.dense_dtype), W1, W3, W2, self.act, low(d_gate), low(d_up), return_hidden=True)
        if self._adapter("shared_down_lora") is None:
            return y.float()
        return y.float() + delta(s_act.float(), "shared_down_lora", 2)

    def _check_adapters(self) -> None:
        if isinstance(self.experts, Int4Experts) and self._routed_lora() is not None:
            raise ValueError("routed adapters need an ExpertLayer: the products with 4-bit integer weights take none")

    def _routed(self, h_latent: torch.Tensor, w: torch.Tensor, idx: torch.Tensor, cached) -> torch.Tensor:
        """The routed experts' sum, fp32 (`cached`: an earlier call's)."""
        if not isinstance(self.experts, Int4Experts):
            return RoutedExpertsFunction.apply(h_latent, w, idx, self.experts, self.act, cached, self._routed_lora())
        self._check_adapters()
        if cached is not None:
            # nothing recorded with the call that made it, and nothing here, would carry a gradient to h_latent or w
            if torch.is_grad_enabled() and (h_latent.requires_grad or w.requires_grad):
                raise NotImplementedError("the products with 4-bit integer weights have no backward pass: call the block "
                                          "under torch.no_grad() or on detached tensors, with cached as without")
            return cached.to(torch.float32)
        return int4_routed(h_latent.to(self.experts.dtype), idx, w, self.experts, self.act).float()

    def forward(self, h_moe_norm: torch.Tensor, cached: Optional[torch.Tensor] = None, dropout_seed=None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(out in h's dtype and shape, topk_indices, topk_weights) for the normed hidden state.

        dropout_seed: a whole number (or one-element int64 device tensor) that turns on the shared
        adapters' dropout at their dropout_rate; the masks depend on it and the element alone, so a
        replayed forward with the same seed (the reference's backward replays each layer) drops the same
        elements. Give every layer and step its own. The routed adapters take no dropout."""
        shape, dtype = h_moe_norm.shape, h_moe_norm.dtype
        x = h_moe_norm.reshape(-1, self.hidden).to(self.experts.device, torch.float32)
        idx, w = route(x, self.gate_weight, self.gate_bias, self.top_k, self.routed_scaling_factor, self.renormalize,
                       self.scoring, self.num_groups, self.topk_groups, self.group_score)
        shared = self._shared(x, dropout_seed)
        h_latent = F.linear(x, self.latent_down)
        routed = self._routed(h_latent, w, idx, cached)
        if self.latent_norm is not None:
            norm = native_rms_norm if self.native else rms_norm
            routed = norm(routed, self.latent_norm, self.rms_eps)
        out = shared + F.linear(routed, self.latent_up)
        return out.reshape(shape).to(dtype), idx, w

    __call__ = forward
