"""MXFP4 calls and layers under torch.compile: one graph, and the eager results.  Without a GPU the tracing alone: its
tensors stand in for a device's."""
import pytest
import torch

from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, ReplicatedLinear
from sglite_amd.mlp import GatedMLP
from sglite_amd.moe import MXFP4MoELayer
from sglite_amd.quantization import MXFP4Config

H = torch.float16


class Traced(Exception):
    pass


def traced_whole(monkeypatch, fn, *args):
    """Whether Dynamo takes fn in one graph (the graph itself would need a GPU)."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    calls = []

    def backend(graph, inputs):
        calls.extend(str(n.target) for n in graph.graph.nodes if "sglite_awq" in str(n.target))
        raise Traced
    torch._dynamo.reset()
    with pytest.raises(Exception) as e:
        torch.compile(fn, backend=backend, fullgraph=True)(*args)
    assert "Traced" in repr(e.value) or isinstance(e.value.__cause__, Traced), e.value
    return calls


def weight(N, K, E=None):
    wb, sb = ops._mx4_layout_bytes(N, K)
    lead = () if E is None else (E,)
    return ops.Mx4Weight(torch.zeros(lead + (wb,), dtype=torch.uint8), torch.zeros(lead + (sb,), dtype=torch.uint8), N, K)


def test_products_trace(monkeypatch):
    x, w, bias, out = torch.zeros(20, 96).to(H), weight(128, 96), torch.zeros(128), torch.zeros(20, 128).to(H)
    wide = torch.zeros(20, 200).to(H)[:, 8:104]
    for fn, arg in ((lambda v: ops.mx4_gemm(v, w) * 2, x), (lambda v: ops.mx4_gemm(v, w, bias=bias), x),
                    (lambda v: ops.mx4_gemm(v, w, activation="silu"), wide),
                    (lambda v: ops.mx4_gemm(v, w, out=out) + 1, x),
                    (lambda v: ops.mx4_dequantize(ops.mx4_quantize(v), H), x)):
        assert traced_whole(monkeypatch, fn, arg)
    some = torch.zeros(20, 96).to(H)
    torch._dynamo.mark_dynamic(some, 0)  # a batch of any size
    assert traced_whole(monkeypatch, lambda v: ops.mx4_gemm(v, w, bias=bias, activation="gelu"), some)
    ex, ids, tw = weight(64, 96, 4), torch.zeros(20, 2, dtype=torch.int32), torch.ones(20, 2)
    assert len(traced_whole(monkeypatch, lambda v: ops.mx4_moe_gemm(v, ex, ops.moe_align_block_size(ids, 16, 4), tw, 40,
                                                                    2, "silu", True), x)) == 2


def processed(layer, N, K):
    """A layer as it is after loading, without the device that lays its weight out."""
    w = weight(N, K)
    layer._weights.update(weight=w.w, weight_scale=w.s, _output_size=N, _input_size=K, _weights_processed=True)
    return layer


def test_layers_trace(monkeypatch):
    method = MXFP4Config().get_linear_method()
    x = torch.zeros(20, 96).to(H)
    one = processed(ReplicatedLinear(96, 64, True, method), 64, 96)
    assert len(traced_whole(monkeypatch, lambda v: one(v) * 2, x)) == 1
    assert len(traced_whole(monkeypatch, lambda v: one(v), x.view(2, 10, 96))) == 1
    two = processed(MergedColumnParallelLinear(96, [64, 64], False, method), 128, 96)
    assert len(traced_whole(monkeypatch, lambda v: two.forward_act(v, "silu"), x)) == 1
    mlp = GatedMLP(96, 64, "silu", method)
    processed(mlp.gate_up_proj, 128, 96), processed(mlp.down_proj, 96, 64)
    assert len(traced_whole(monkeypatch, lambda v: mlp(v), x)) == 2
    moe = MXFP4MoELayer(4, 2, 96, 64)
    moe._experts = (weight(128, 96, 4), weight(96, 64, 4))
    logits = torch.zeros(20, 4)
    assert len(traced_whole(monkeypatch, lambda v: moe(v, logits), x)) >= 4


def compiled(fn):
    torch._dynamo.reset()
    return torch.compile(fn, backend="aot_eager", fullgraph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 20, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_products(M, dtype):
    g = torch.Generator(device="cuda").manual_seed(M)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)
    w = ops.mx4_repack(ops.mx4_quantize(normal(128, 96)))
    x, bias = normal(M, 96), normal(128).float()
    assert torch.equal(compiled(lambda v: ops.mx4_gemm(v, w, bias=bias) * 2.0)(x), ops.mx4_gemm(x, w, bias=bias) * 2.0)
    odd = normal(M * 96 + 1)[1:].view(M, 96)  # an odd address
    wide = normal(M, 200)[:, 8:104]
    fn = compiled(lambda v: ops.mx4_gemm(v, w, activation="gelu") + 1.0)
    for v in (x, odd, wide):
        assert torch.equal(fn(v), ops.mx4_gemm(v, w, activation="gelu") + 1.0)
    for more in (M + 1, 2 * M + 40):  # other batches of the same function
        v = normal(more, 96)
        assert torch.equal(fn(v), ops.mx4_gemm(v, w, activation="gelu") + 1.0)
    out = torch.zeros((M, 128), dtype=dtype, device="cuda")
    assert torch.equal(compiled(lambda v: ops.mx4_gemm(v, w, out=out) + 1.0)(x), ops.mx4_gemm(x, w) + 1.0)
    assert torch.equal(out, ops.mx4_gemm(x, w))
    back = compiled(lambda v: ops.mx4_dequantize(ops.mx4_quantize(v), torch.float32))
    assert torch.equal(back(odd), ops.mx4_dequantize(ops.mx4_quantize(odd), torch.float32))
    ex = ops.mx4_repack(ops.mx4_quantize(normal(4, 64, 96)))
    ids = torch.randint(0, 4, (M, 2), generator=g, device="cuda").int()
    tw = torch.rand((M, 2), generator=g, device="cuda")

    def experts(v):
        return ops.mx4_moe_gemm(v, ex, ops.moe_align_block_size(ids, 16, 4), tw, 2 * M, 2, "silu", True)
    assert torch.equal(compiled(experts)(odd), experts(odd))


@pytest.mark.gpu
def test_layers():
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(H)
    torch.set_default_dtype(H)
    try:
        one = ReplicatedLinear(96, 64, True, MXFP4Config(False).get_linear_method())
        mlp = GatedMLP(96, 64, "silu", MXFP4Config(False).get_linear_method())
    finally:
        torch.set_default_dtype(torch.float32)
    one.load_state_dict({"weight": normal(64, 96), "bias": normal(64)})
    mlp.load_state_dict({"gate_up_proj.weight": normal(128, 96), "down_proj.weight": normal(96, 64)})
    moe = MXFP4MoELayer(4, 2, 96, 64, serialized=False)
    moe.load_state_dict({"gate_up_proj": normal(4, 128, 96), "down_proj": normal(4, 96, 64)})
    x, logits = normal(20, 96), normal(20, 4)
    assert torch.equal(compiled(lambda v: one(v) * 2.0)(x), one(x) * 2.0)
    assert torch.equal(compiled(lambda v: mlp(v) * 2.0)(x), mlp(x) * 2.0)
    want = moe(x.clone(), logits)
    assert torch.equal(compiled(lambda v: moe(v, logits) * 1.0)(x.clone()), want)
