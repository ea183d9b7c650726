"""Tensor-parallel linear layers that drive a linear method's lifecycle.

Mirror of python/sglite/srt/model_executor/layers/linear.py:15-194 (the caller
side of the plugin boundary):

* construction calls ``create_weights(local_in, local_out)`` and keeps
  ``_``-prefixed entries out of the state dict (linear.py:32-45);
* ``load_state_dict`` pops this layer's tensors with exact shape/dtype checks,
  re-points the method's weight map, restores metadata and runs
  ``process_weights_after_loading`` once, re-binding only attributes that
  already exist (linear.py:50-99);
* ``forward`` is ``apply_weights(weights, x, bias)``; a row-parallel layer
  all-reduces its partial output when tp_size > 1 (linear.py:101-103, 189-194).

Tensor-parallel sizes are explicit arguments here (tp_rank, tp_size) instead
of the reference's process-group globals.

Beyond the reference, a layer can hold low-rank adapters beside its weight:
``add_adapters`` makes the slots, ``load_adapter`` fills one, and ``forward``
with a step's ``ops.lora_route`` adds each row's adapter to its output.
"""

from __future__ import annotations

from typing import Any, Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import ops
from .quantization import LinearMethodBase, UnquantizedLinearMethod


def div_even(a: int, b: int, allow_replicate: bool = False) -> int:
    """a / b, which must divide evenly; with ``allow_replicate`` a < b gives 1."""
    if allow_replicate and a < b:
        if b % a:
            raise ValueError(f"{b} is not a multiple of {a}")
        return 1
    if a % b:
        raise ValueError(f"{a} is not divisible by {b}")
    return a // b


def _concat_prefix(prefix: str, name: str) -> str:
    return f"{prefix}.{name}" if prefix else name


class _TPLinearBase:
    def __init__(self, full_isize: int, full_osize: int, local_isize: int, local_osize: int, has_bias: bool,
                 linear_method: Optional[LinearMethodBase] = None, tp_size: int = 1):
        self.full_input_size = full_isize
        self.full_output_size = full_osize
        self.local_input_size = local_isize
        self.local_output_size = local_osize
        self._tp_size = tp_size
        self._linear_method = linear_method or UnquantizedLinearMethod()
        self._weights: Dict[str, Any] = self._linear_method.create_weights(local_isize, local_osize)
        self._weight_metadata: Dict[str, Any] = {}
        for name in list(self._weights.keys()):
            if name.startswith("_"):
                self._weight_metadata[name] = self._weights.pop(name)
        for name, tensor in self._weights.items():
            setattr(self, name, tensor)
        self.bias = torch.empty(local_osize) if has_bias else None
        self._weights_processed = False
        self._parts: Tuple[int, ...] = (local_osize,)  # columns of the projections merged into this one
        self._lora: Optional[ops.LoraStack] = None     # adapter slots; not in the state dict

    def state_dict_keys(self, prefix: str = "") -> List[str]:
        return [_concat_prefix(prefix, n) for n, v in self.__dict__.items()
                if not n.startswith("_") and isinstance(v, torch.Tensor)]

    def load_state_dict(self, state_dict: Dict[str, torch.Tensor], *, prefix: str = "", _internal: bool = False) -> None:
        for name, param in list(self.__dict__.items()):
            if name.startswith("_") or not isinstance(param, torch.Tensor):
                continue
            item = state_dict.pop(_concat_prefix(prefix, name))
            assert isinstance(item, torch.Tensor)
            assert param.shape == item.shape and param.dtype == item.dtype, (
                f"{name}: expected {tuple(param.shape)} {param.dtype}, got {tuple(item.shape)} {item.dtype}")
            setattr(self, name, item)
        for name in list(self._weights.keys()):
            if hasattr(self, name):
                self._weights[name] = getattr(self, name)
        for name, value in self._weight_metadata.items():
            self._weights[name] = value
        if not self._weights_processed:
            processed = self._linear_method.process_weights_after_loading(self._weights)
            self._weight_metadata = {}
            for name, value in processed.items():
                if name.startswith("_"):
                    self._weight_metadata[name] = value
                else:
                    self._weights[name] = value
                    if hasattr(self, name):  # runtime tensors (workspace) stay out of the state dict
                        setattr(self, name, value)
            self._weights.update(self._weight_metadata)
            self._weights_processed = True
        if not _internal and state_dict:
            raise RuntimeError(f"Unexpected keys in state_dict: {list(state_dict.keys())}")

    def add_adapters(self, num_adapters: int, max_rank: int, dtype: torch.dtype,
                     device: Optional[torch.device] = None) -> None:
        """Make ``num_adapters`` empty adapter slots (an empty slot adds nothing) of ranks up to ``max_rank``,
        rounded up to a multiple of 8, on ``device`` (that of the loaded weights if None; before they are loaded, the
        current GPU).  Replaces slots made before: a step captured with those is captured anew.  Layers whose sizes
        the adapters' kernels cannot take (input and every merged projection in multiples of 8, at most four merged)
        are refused."""
        if not 1 <= num_adapters <= ops.LORA_MAX_ADAPTERS:
            raise ValueError(f"num_adapters must be in [1, {ops.LORA_MAX_ADAPTERS}], got {num_adapters}")
        rank = (max_rank + 7) // 8 * 8
        if not 8 <= rank <= ops.LORA_MAX_RANK:
            raise ValueError(f"max_rank must be in [1, {ops.LORA_MAX_RANK}], got {max_rank}")
        if device is None:
            loaded = [t for t in self._weights.values() if isinstance(t, torch.Tensor)] if self._weights_processed else []
            device = loaded[0].device if loaded else torch.device("cuda")
        self._lora = ops.make_lora_stack(num_adapters, rank, self.local_input_size, self._parts, dtype, device)

    def _lora_slot(self, slot: int) -> ops.LoraStack:
        if self._lora is None:
            raise RuntimeError("this layer has no adapter slots (call add_adapters first)")
        if not 0 <= slot < self._lora.ranks.numel():
            raise ValueError(f"slot must be in [0, {self._lora.ranks.numel()}), got {slot}")
        return self._lora

    @torch.no_grad()
    def load_adapter(self, slot: int, lora_a: Union[torch.Tensor, Sequence[Optional[torch.Tensor]]],
                     lora_b: Union[torch.Tensor, Sequence[Optional[torch.Tensor]]], scaling: float = 1.0) -> None:
        """Fill a slot with an adapter: A [rank, K] and B [columns, rank] for every merged projection in order (one
        tensor each for a layer of one projection, None where the adapter leaves a projection alone), each the
        layer's own shard.  ``scaling`` is alpha / rank.  The slot holds values alone: trained Parameters are copied
        without their gradients' graph.  Copies on the current stream: the caller orders it
        against steps on other streams."""
        stack = self._lora_slot(slot)
        a_list = [lora_a] if isinstance(lora_a, torch.Tensor) else list(lora_a)
        b_list = [lora_b] if isinstance(lora_b, torch.Tensor) else list(lora_b)
        if len(a_list) != len(stack.parts) or len(b_list) != len(stack.parts):
            raise ValueError(f"this layer merges {len(stack.parts)} projections, got {len(a_list)} A and "
                             f"{len(b_list)} B")
        R, K = stack.b.shape[2], stack.a.shape[2]
        rank = 0
        for i, (a, b) in enumerate(zip(a_list, b_list)):  # check everything before any copy
            if (a is None) != (b is None):
                raise ValueError(f"projection {i} has only one of A and B")
            if a is None:
                continue
            if a.dim() != 2 or a.shape[1] != K or not 1 <= a.shape[0] <= R:
                raise ValueError(f"A of projection {i} must be [rank, {K}] with rank in [1, {R}], got {tuple(a.shape)}")
            if tuple(b.shape) != (stack.parts[i], a.shape[0]):
                raise ValueError(f"B of projection {i} must be {(stack.parts[i], a.shape[0])}, got {tuple(b.shape)}")
            rank = max(rank, a.shape[0])
        self.clear_adapter(slot)
        col = 0
        for i, (a, b) in enumerate(zip(a_list, b_list)):
            if a is not None:
                stack.a[slot, i * R:i * R + a.shape[0]].copy_(a)
                stack.b[slot, col:col + stack.parts[i], :a.shape[0]].copy_(b)
            col += stack.parts[i]
        stack.scaling[slot] = float(scaling)
        stack.ranks[slot] = rank

    def clear_adapter(self, slot: int) -> None:
        """Empty a slot: rows that name it get the projection alone."""
        stack = self._lora_slot(slot)
        for t in (stack.a, stack.b, stack.scaling, stack.ranks):
            t[slot].zero_()

    def _add_lora(self, y: torch.Tensor, x: torch.Tensor, adapters: ops.LoraBatch,
                  activation: Optional[str] = None) -> torch.Tensor:
        rows, cols = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
        out = ops.lora_add(cols, rows, self._lora, adapters, activation, out=cols if activation is None else None)
        return out.reshape(y.shape[:-1] + out.shape[-1:])

    def forward(self, x: torch.Tensor, adapters: Optional[ops.LoraBatch] = None) -> torch.Tensor:
        """The projection of x, with ``adapters`` (``ops.lora_route`` of the rows' slots) and slots made, plus each
        row's adapter: added in fp32 to the projection as stored, and rounded once more."""
        y = self._linear_method.apply_weights(self._weights, x, self.bias)
        if adapters is not None and self._lora is not None:
            y = self._add_lora(y, x, adapters)
        return y

    __call__ = forward


class ReplicatedLinear(_TPLinearBase):
    def __init__(self, input_size: int, output_size: int, has_bias: bool,
                 linear_method: Optional[LinearMethodBase] = None):
        super().__init__(input_size, output_size, input_size, output_size, has_bias, linear_method)


class MergedColumnParallelLinear(_TPLinearBase):
    """Fused column-parallel projection (gate_up): local N = sum(size / tp) (linear.py:127-143)."""

    def __init__(self, input_size: int, output_sizes: List[int], has_bias: bool,
                 linear_method: Optional[LinearMethodBase] = None, tp_size: int = 1):
        tp_sizes = [div_even(s, tp_size) for s in output_sizes]
        super().__init__(input_size, sum(output_sizes), input_size, sum(tp_sizes), has_bias, linear_method, tp_size)
        self._parts = tuple(tp_sizes)

    def forward_act(self, x: torch.Tensor, activation: str,
                    adapters: Optional[ops.LoraBatch] = None) -> torch.Tensor:
        """act(gate) * up of a two-part (gate, up) projection: the layer's forward
        followed by silu_and_mul / gelu_and_mul (blocks.py:53-55), fused into the
        GEMM when the linear method has a fused kernel, or with ``adapters`` into
        the step that adds them."""
        if adapters is not None and self._lora is not None:
            y = self._linear_method.apply_weights(self._weights, x, self.bias)
            return self._add_lora(y, x, adapters, activation)
        return self._linear_method.apply_weights_act(self._weights, x, activation, self.bias)


class QKVParallelLinear(_TPLinearBase):
    """Fused q/k/v projection: local N = (Hq/tp + 2 Hkv/tp) * d (linear.py:146-168)."""

    def __init__(self, hidden_size: int, head_dim: int, num_qo_heads: int, num_kv_heads: int, has_bias: bool,
                 linear_method: Optional[LinearMethodBase] = None, tp_size: int = 1):
        local_qo = div_even(num_qo_heads, tp_size)
        local_kv = div_even(num_kv_heads, tp_size, allow_replicate=True)
        super().__init__(hidden_size, (num_qo_heads + 2 * num_kv_heads) * head_dim, hidden_size,
                         (local_qo + 2 * local_kv) * head_dim, has_bias, linear_method, tp_size)
        self._parts = (local_qo * head_dim, local_kv * head_dim, local_kv * head_dim)


class RowParallelLinear(_TPLinearBase):
    """Row-parallel projection (o, down): local K = K / tp, all-reduce of the output (linear.py:171-194)."""

    def __init__(self, input_size: int, output_size: int, has_bias: bool,
                 linear_method: Optional[LinearMethodBase] = None, tp_size: int = 1, process_group=None):
        self._group = process_group
        super().__init__(input_size, output_size, div_even(input_size, tp_size), output_size, has_bias,
                         linear_method, tp_size)

    def forward(self, x: torch.Tensor, adapters: Optional[ops.LoraBatch] = None) -> torch.Tensor:
        # Each rank adds B (A_rank x_rank) to its partial output: the all-reduce sums both.
        y = super().forward(x, adapters)
        if self._tp_size > 1:
            torch.distributed.all_reduce(y, group=self._group)
        return y

    __call__ = forward
