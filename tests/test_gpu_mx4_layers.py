"""MXFP4 layers on the GPU: linears, a gated block, experts and adapters as a model runs them."""
import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import checkpoint as ck
from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, QKVParallelLinear, ReplicatedLinear
from sglite_amd.mlp import GatedMLP
from sglite_amd.moe import MXFP4MoELayer
from sglite_amd.quantization import MXFP4Config
from tests.test_gpu_mx4_gemm import HALF, close
from tests.test_gpu_mx4_moe import formula

pytestmark = pytest.mark.gpu
DEV = "cuda"


def normal(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


@pytest.fixture
def half_default():
    torch.set_default_dtype(torch.float16)
    yield
    torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("serialized", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_layers(serialized, dtype):
    H, D, Hq, Hkv = 256, 64, 4, 2
    N = (Hq + 2 * Hkv) * D
    torch.set_default_dtype(dtype)
    try:
        layer = QKVParallelLinear(H, D, Hq, Hkv, True, MXFP4Config(serialized).get_linear_method())
    finally:
        torch.set_default_dtype(torch.float32)
    w, bias = normal((N, H), 0, dtype, H ** -0.5), normal((N,), 1, dtype)
    codes, scales = oracle.quantize(w)
    state = {"weight": codes, "weight_scale": scales} if serialized else {"weight": w}
    layer.load_state_dict({**state, "bias": bias})
    values = oracle.values(codes, scales)
    for shape in ((1, H), (5, H), (3, 50, H)):
        x = normal(shape, len(shape), dtype)
        y = layer(x)
        assert y.shape == shape[:-1] + (N,) and y.dtype == dtype
        close(y.reshape(-1, N), *oracle.product(oracle.quantized(x.reshape(-1, H)), values, bias))


def test_halves_that_are_no_whole_blocks(half_default):
    layer = MergedColumnParallelLinear(64, [40, 40], False, MXFP4Config().get_linear_method())  # 40 is no multiple of 32
    codes, scales = oracle.quantize(normal((80, 64), 2))
    layer.load_state_dict({"weight": codes, "weight_scale": scales})
    x = normal((6, 64), 3, torch.float16)
    y = layer(x).float()
    want = (torch.nn.functional.silu(y[:, :40]) * y[:, 40:]).half()
    assert torch.equal(layer.forward_act(x, "silu"), want)


@pytest.mark.parametrize("M", [1, 7, 40, 300, 2100])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_block(M, act, half_default):
    """Each product of the block against the formula on what the one before it gave."""
    H, I = 256, 384
    mlp = GatedMLP(H, I, act, MXFP4Config().get_linear_method())
    gu, dn = oracle.quantize(normal((2 * I, H), 0, scale=H ** -0.5)), oracle.quantize(normal((H, I), 1, scale=I ** -0.5))
    mlp.load_state_dict({"m.gate_up_proj.weight": gu[0], "m.gate_up_proj.weight_scale": gu[1],
                         "m.down_proj.weight": dn[0], "m.down_proj.weight_scale": dn[1]}, prefix="m")
    x = normal((M, H), 2, torch.float16)
    h = mlp.gate_up_proj.forward_act(x, act)
    close(h, *oracle.gated(*oracle.product(oracle.quantized(x), oracle.values(*gu)), act))
    y = mlp(x)
    close(y, *oracle.product(oracle.quantized(h), oracle.values(*dn)))
    if M <= 40:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mlp(x)
        for seed in (5, 6):
            x.copy_(normal((M, H), seed, torch.float16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, mlp(x))


@pytest.mark.parametrize("M", [3, 60])
def test_adapters_beside(M, half_default):
    H, N = 128, 96
    layer = ReplicatedLinear(H, N, False, MXFP4Config().get_linear_method())
    codes, scales = oracle.quantize(normal((N, H), 0, scale=H ** -0.5))
    layer.load_state_dict({"weight": codes, "weight_scale": scales})
    layer.add_adapters(4, 8, torch.float16)
    a, b = normal((8, H), 1, torch.float16, H ** -0.5), normal((N, 8), 2, torch.float16, 0.1)
    layer.load_adapter(2, a, b, 0.5)
    x = normal((M, H), 3, torch.float16)
    ids = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    ids[::2] = 2
    y, base = layer(x, ops.lora_route(ids, 4)), layer(x)
    assert torch.equal(y[1::2], base[1::2])
    add = 0.5 * (x.double() @ a.double().t()) @ b.double().t()
    want = base.double() + add
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -18 * (x.double().abs() @ a.double().abs().t()) @ b.double().abs().t()
    assert ((y.double() - want).abs() <= tol + 2.0 ** -25)[::2].all()


def test_shards_sum_to_the_whole():
    """Two ranks' halves of K and of the columns give what the whole layer gives."""
    K, N, M = 256, 96, 20
    stream = dict(zip(("l.down_proj.weight", "l.down_proj.weight_scale"), oracle.quantize(normal((N, K), 0))))
    x = normal((M, K), 1, torch.float16)
    method = MXFP4Config().get_linear_method()
    parts = []
    for rank in range(2):
        shard = dict(ck.ingest(iter(stream.items()), rank=rank, world=2))
        w = method.process_weights_after_loading({"weight": shard["l.down_proj.weight"],
                                                  "weight_scale": shard["l.down_proj.weight_scale"]})
        parts.append(method.apply_weights(w, x.chunk(2, 1)[rank]).double())
    y, err = oracle.product(oracle.quantized(x), oracle.values(*stream.values()))
    tol = err + 2.0 ** -11 * (parts[0].abs() + parts[1].abs()) + 2.0 ** -24
    assert ((parts[0] + parts[1] - y).abs() <= tol).all()


@pytest.mark.parametrize("serialized", [True, False])
@pytest.mark.parametrize("T", [1, 13, 200])
def test_expert_layer(T, serialized):
    E, k, H, I, dtype = 8, 2, 256, 160, torch.bfloat16
    w1, w2 = normal((E, 2 * I, H), 0, dtype, H ** -0.5), normal((E, H, I), 1, dtype, I ** -0.5)
    q1, q2 = oracle.quantize(w1), oracle.quantize(w2)
    layer = MXFP4MoELayer(E, k, H, I, serialized=serialized, params_dtype=dtype)
    state = ({"gate_up_proj": q1[0], "gate_up_proj.weight_scale": q1[1], "down_proj": q2[0],
              "down_proj.weight_scale": q2[1]} if serialized else {"gate_up_proj": w1, "down_proj": w2})
    layer.load_state_dict(state)
    assert not state
    x, logits = normal((T, H), 2, dtype), normal((T, E), 3)
    # Stage by stage, each on what the one before it gave.
    weights, ids, align = ops.moe_route(logits, k, True, 16)
    e1, e2 = layer._expert_weights()
    h = ops.mx4_moe_gemm(x, e1, align, weights, T * k, k, "silu")
    close(h, *formula(x, *q1, ids, k, None, "silu"))
    y = ops.mx4_moe_gemm(h, e2, align, weights, T * k, 1, mul_routed_weight=True)
    close(y, *formula(h, *q2, ids, 1, weights, None))
    want = y.double().view(T, k, H).sum(1)
    got = layer(x.clone(), logits)
    tol = HALF[dtype] * want.abs() + 2.0 ** -22 * y.double().view(T, k, H).abs().sum(1) + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all()
    if T <= 13:
        buf = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer(buf, logits)
        for seed in (4, 5):
            fresh = normal((T, H), seed, dtype)
            logits.copy_(normal((T, E), seed + 10))
            buf.copy_(fresh)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(buf, layer(fresh.clone(), logits))


def test_experts_with_no_tokens():
    layer = MXFP4MoELayer(4, 2, 64, 64, serialized=False)
    layer.load_state_dict({"gate_up_proj": normal((4, 128, 64), 0, torch.float16),
                           "down_proj": normal((4, 64, 64), 1, torch.float16)})
    x = torch.empty((0, 64), dtype=torch.float16, device=DEV)
    assert layer(x, torch.empty((0, 4), device=DEV)).shape == (0, 64)
