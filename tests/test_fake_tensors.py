"""Shapes of the adapters and dense experts without data: the public calls under FakeTensorMode (no GPU)."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, ReplicatedLinear
from sglite_amd.mlp import GatedMLP

DEV = torch.device("cuda")
H = torch.float16


@pytest.fixture(autouse=True)
def fake():
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # a fake tensor's address is 0, with a warning
        with FakeTensorMode():
            yield


def empty(*shape, dtype=H):
    return torch.empty(shape, dtype=dtype, device=DEV)


@pytest.mark.parametrize("M", [4, 20])
def test_lora_add(M):
    stack = ops.make_lora_stack(3, 16, 64, (24, 24), H, DEV)
    y, x, batch = empty(M, 48), empty(M, 64), ops.lora_route(empty(M, dtype=torch.int32), 3)
    assert ops.lora_add(y, x, stack, batch).shape == (M, 48)
    assert ops.lora_add(y, x, stack, batch, "silu").shape == (M, 24)
    assert ops.lora_add(y, x, stack, batch, out=y) is y
    out = empty(M, 48)
    assert ops.lora_add(y, x, stack, batch, out=out) is out
    with pytest.raises(ValueError, match="shape"):
        ops.lora_add(y, x, stack, batch, out=empty(M, 40))


def test_moe_dense_gemm():
    a, w = empty(10, 64), empty(4, 32, 64)
    align = ops.moe_align_block_size(empty(10, 2, dtype=torch.int32), 16, 4)
    out = empty(20, 16)
    assert ops.moe_dense_gemm(a, w, align, None, 20, 2, "silu", out=out) is out
    assert ops.moe_dense_gemm(a, w, align, None, 20, 2).shape == (20, 32)


def test_layers_with_adapters():
    batch = ops.lora_route(empty(20, dtype=torch.int32), 3)
    torch.set_default_dtype(H)
    try:
        one, two = ReplicatedLinear(64, 40, False), MergedColumnParallelLinear(64, [48, 48], False)
        mlp = GatedMLP(64, 48)
    finally:
        torch.set_default_dtype(torch.float32)
    one.load_state_dict({"weight": empty(40, 64)})
    two.load_state_dict({"weight": empty(96, 64)})
    mlp.load_state_dict({"gate_up_proj.weight": empty(96, 64), "down_proj.weight": empty(64, 48)})
    for layer in (one, two, mlp.gate_up_proj, mlp.down_proj):
        layer.add_adapters(3, 8, H, DEV)
    x = empty(20, 64)
    assert one(x, batch).shape == (20, 40) and one(x.view(2, 10, 64), batch).shape == (2, 10, 40)
    assert two(x, batch).shape == (20, 96) and two.forward_act(x, "silu", batch).shape == (20, 48)
    assert mlp(x, batch).shape == (20, 64)
