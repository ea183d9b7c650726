"""``mxfp4`` quantization config and linear method: MXFP4 weights and activations on scaled MFMAs.

No counterpart in the reference; the interface is that of its methods (base_config.py:22-91).  A checkpoint holds
``weight`` uint8 [N, K/2] (two codes a byte, the lower k in the low bits) and ``weight_scale`` uint8 [N, K/32]
(exponent bytes) for every projection, which the loader shards and merges like a dense weight (weight_loader.py:40-77);
with ``is_checkpoint_mxfp4_serialized`` false it holds 16- or 32-bit ``weight`` [N, K], quantised once after loading.
Activations are quantised by the products (``ops.mx4_gemm``).  The configuration is this framework's own: published
ones of the same method name mean weight-only experts beside 16-bit layers, which it does not implement and refuses.
"""

from typing import Any, Dict, List, Optional

import torch
from torch.nn.parameter import Parameter

from .. import ops
from .base_config import LinearMethodBase, QuantizationConfig, set_weight_attrs


class MXFP4Config(QuantizationConfig):
    """MXFP4 in blocks of 32."""

    def __init__(self, is_checkpoint_mxfp4_serialized: bool = True, weight_bits: int = 4,
                 group_size: int = ops.MX4_BLOCK) -> None:
        if weight_bits != 4 or group_size != ops.MX4_BLOCK:
            raise ValueError(f"MXFP4 has 4 bits and blocks of {ops.MX4_BLOCK}, got {weight_bits} bits and groups of "
                             f"{group_size}")
        self.is_checkpoint_mxfp4_serialized = is_checkpoint_mxfp4_serialized
        self.weight_bits = weight_bits
        self.group_size = group_size

    def __repr__(self) -> str:
        return f"MXFP4Config(is_checkpoint_mxfp4_serialized={self.is_checkpoint_mxfp4_serialized})"

    def get_name(self) -> str:
        return "mxfp4"

    def get_supported_act_dtypes(self) -> List[torch.dtype]:
        return [torch.half, torch.bfloat16]

    def get_min_capability(self) -> int:
        return 95  # the products are gfx950's scaled MFMAs

    @staticmethod
    def get_config_filenames() -> List[str]:
        return ["quant_config.json", "quantize_config.json"]

    @classmethod
    def from_config(cls, config: Dict[str, Any]) -> "MXFP4Config":
        """Every linear layer's weights and activations in MXFP4; what else a config asks for is refused by name."""
        known = ("quant_method", "is_checkpoint_mxfp4_serialized", "bits", "group_size")
        others = sorted(k for k, v in config.items() if k not in known and v not in (None, False, [], {}, ""))
        if others:
            raise ValueError(f"the mxfp4 method quantises all linear layers, weights and activations; it does not "
                             f"implement {others}")
        return cls(bool(config.get("is_checkpoint_mxfp4_serialized", True)), config.get("bits", 4),
                   config.get("group_size", ops.MX4_BLOCK))

    def get_linear_method(self) -> "MXFP4LinearMethod":
        return MXFP4LinearMethod(self)

    def get_scaled_act_names(self) -> List[str]:
        return []


class MXFP4LinearMethod(LinearMethodBase):
    """y = Q(x) W^T (+ bias), W in MXFP4, Q the quantisation of activations to it."""

    def __init__(self, quant_config: MXFP4Config):
        self.quant_config = quant_config

    def create_weights(self, input_size: int, output_size: int) -> Dict[str, Any]:
        if input_size % ops.MX4_BLOCK:
            raise ValueError(f"input_size={input_size} is not divisible by the block of {ops.MX4_BLOCK}. "
                             "This can be caused by too large tensor parallel size.")
        if output_size % 8:
            raise ValueError(f"output_size={output_size} is not divisible by 8. "
                             "This can be caused by too large tensor parallel size.")
        meta = {"_input_size": input_size, "_output_size": output_size, "_weights_processed": False}
        if not self.quant_config.is_checkpoint_mxfp4_serialized:
            weight = Parameter(torch.empty(output_size, input_size), requires_grad=False)
            set_weight_attrs(weight, {"input_dim": 1, "output_dim": 0})
            return {"weight": weight, **meta}
        weight = Parameter(torch.empty(output_size, input_size // 2, dtype=torch.uint8), requires_grad=False)
        set_weight_attrs(weight, {"input_dim": 1, "output_dim": 0, "packed_dim": 1, "pack_factor": 2})
        scale = Parameter(torch.empty(output_size, input_size // ops.MX4_BLOCK, dtype=torch.uint8), requires_grad=False)
        set_weight_attrs(scale, {"input_dim": 1, "output_dim": 0})
        return {"weight": weight, "weight_scale": scale, **meta}

    def process_weights_after_loading(self, weights: Dict[str, Any]) -> Dict[str, Any]:
        """Lay the weight out for the products, on its device, a 16- or 32-bit one quantised first; the loaded
        tensors are dropped."""
        if weights.get("_weights_processed", False):
            return weights
        if self.quant_config.is_checkpoint_mxfp4_serialized:
            q = ops.Mx4(weights["weight"].data, weights["weight_scale"].data)
        else:
            q = ops.mx4_quantize(weights["weight"].data)
        w = ops.mx4_repack(q)
        return {
            "weight": Parameter(w.w, requires_grad=False),
            "weight_scale": Parameter(w.s, requires_grad=False),
            "_input_size": w.K,
            "_output_size": w.N,
            "_weights_processed": True,
        }

    def _apply(self, weights: Dict[str, Any], x: torch.Tensor, bias: Optional[torch.Tensor],
               activation: Optional[str]) -> torch.Tensor:
        if not weights.get("_weights_processed", False):
            weights = self.process_weights_after_loading(weights)
        w = ops.Mx4Weight(weights["weight"], weights["weight_scale"], weights["_output_size"], weights["_input_size"])
        if x.dim() == 2:
            return ops.mx4_gemm(x, w, bias=bias, activation=activation)
        y = ops.mx4_gemm(x.reshape(-1, x.shape[-1]), w, bias=bias, activation=activation)
        return y.reshape(x.shape[:-1] + y.shape[-1:])

    def apply_weights(self, weights: Dict[str, Any], x: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        return self._apply(weights, x, bias, None)

    def apply_weights_act(self, weights: Dict[str, Any], x: torch.Tensor, activation: str,
                          bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """act(gate) * up in the gate/up product (halves that are no multiple of a block go the base class's way)."""
        if weights["_output_size"] % (2 * ops.MX4_BLOCK):
            return super().apply_weights_act(weights, x, activation, bias)
        return self._apply(weights, x, bias, activation)
