"""Adapter slots that the kernels cannot serve are refused when they are made; where slots lie (no GPU)."""
import pytest
import torch

from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, ReplicatedLinear, RowParallelLinear

CPU = torch.device("cpu")


@pytest.mark.parametrize("layer", [
    ReplicatedLinear(64, 100, False), ReplicatedLinear(60, 96, False), RowParallelLinear(72, 64, False, tp_size=2),
    MergedColumnParallelLinear(64, [16, 12], False), MergedColumnParallelLinear(64, [16] * 5, False)])
def test_sizes_the_kernels_cannot_take(layer):
    with pytest.raises(ValueError):
        layer.add_adapters(2, 8, torch.float16, CPU)
    assert layer._lora is None


def test_refused_slots_leave_the_ones_before():
    layer = MergedColumnParallelLinear(64, [16, 24, 8, 8], False)
    layer.add_adapters(2, 8, torch.float16, CPU)
    before = layer._lora
    for bad in (dict(num_adapters=512, max_rank=8), dict(num_adapters=2, max_rank=300)):
        with pytest.raises(ValueError):
            layer.add_adapters(dtype=torch.float16, device=CPU, **bad)
    assert layer._lora is before


def test_stacks_the_kernels_cannot_take():
    ok = dict(num_adapters=2, max_rank=8, K=64, parts=(16, 8), dtype=torch.float16, device=CPU)
    assert ops.make_lora_stack(**ok).b.shape == (2, 24, 8)
    for bad in (dict(num_adapters=0), dict(num_adapters=512), dict(max_rank=0), dict(max_rank=12), dict(max_rank=264),
                dict(K=0), dict(K=60), dict(parts=()), dict(parts=(8,) * 5), dict(parts=(16, 0)), dict(parts=(20, 12)),
                dict(parts=(1 << 27,)), dict(K=1 << 24), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            ops.make_lora_stack(**{**ok, **bad})


def test_slots_lie_with_the_loaded_weights():
    layer = ReplicatedLinear(64, 32, False)
    layer.load_state_dict({"weight": torch.zeros(32, 64)})
    layer.add_adapters(2, 8, torch.float16)
    assert layer._lora.a.device == CPU
    layer.load_adapter(1, torch.ones(4, 64), torch.ones(32, 4))
    assert layer._lora.ranks.tolist() == [0, 4]


def test_trained_parameters_leave_no_graph_in_the_slots():
    layer = ReplicatedLinear(64, 32, False)
    layer.add_adapters(2, 8, torch.float16, CPU)
    a, b = torch.nn.Parameter(torch.ones(4, 64)), torch.nn.Parameter(torch.ones(32, 4))
    assert torch.is_grad_enabled()
    layer.load_adapter(0, a, b, 0.5)
    assert not any(t.requires_grad or t.grad_fn is not None for t in layer._lora[:4])
    assert torch.equal(layer._lora.a[0, :4].float(), torch.ones(4, 64)) and layer._lora.ranks.tolist() == [4, 0]
    assert a.requires_grad and a.grad is None
