"""MXFP4 layers without a GPU: configuration, what checkpoints yield, refusals."""
import json

import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import checkpoint as ck
from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear
from sglite_amd.model_config import load_quantization_config
from sglite_amd.moe import MoELayer, MXFP4FusedMoe, MXFP4MoELayer, create_moe_backend, fused_experts_impl
from sglite_amd.moe import AWQMoELayer
from sglite_amd.quantization import LinearMethodBase, MXFP4Config, get_quantization_config

PRE = "model.layers.1.mlp.experts"


def test_config(tmp_path):
    assert get_quantization_config("MXFP4") is MXFP4Config
    cfg = load_quantization_config(str(tmp_path), {"quantization_config": {"quant_method": "mxfp4"}})
    assert isinstance(cfg, MXFP4Config) and cfg.is_checkpoint_mxfp4_serialized and cfg.get_name() == "mxfp4"
    (tmp_path / "quant_config.json").write_text(json.dumps({"quant_method": "mxfp4", "group_size": 32,
                                                            "is_checkpoint_mxfp4_serialized": False}))
    cfg = load_quantization_config(str(tmp_path))
    assert not cfg.is_checkpoint_mxfp4_serialized and isinstance(cfg.get_linear_method(), LinearMethodBase)
    for bad in ({"bits": 8}, {"group_size": 128}):
        with pytest.raises(ValueError, match="blocks of 32"):
            MXFP4Config.from_config(bad)


def test_create_weights():
    w = MXFP4Config().get_linear_method().create_weights(96, 40)
    assert w["weight"].shape == (40, 48) and w["weight_scale"].shape == (40, 3)
    assert w["weight"].dtype == w["weight_scale"].dtype == torch.uint8
    w = MXFP4Config(False).get_linear_method().create_weights(96, 40)
    assert w["weight"].shape == (40, 96) and "weight_scale" not in w
    for K, N in ((80, 40), (96, 44)):
        with pytest.raises(ValueError, match="not divisible"):
            MXFP4Config().get_linear_method().create_weights(K, N)


def projection(name, N, K, g):
    codes, scales = oracle.quantize(torch.randn((N, K), generator=g))
    return [(f"{name}.weight", codes), (f"{name}.weight_scale", scales)]


@pytest.mark.parametrize("world", [1, 2])
def test_ingestion_yields_what_the_layers_hold(world):
    """Shards and merges of codes and scales are those of the weight itself."""
    g = torch.Generator().manual_seed(0)
    pre, H, I, D = "model.layers.0", 64, 128, 16
    stream = [t for n, N, K in (("self_attn.q_proj", 4 * D, H), ("self_attn.k_proj", 2 * D, H),
                                ("self_attn.v_proj", 2 * D, H), ("self_attn.o_proj", H, 4 * D),
                                ("mlp.gate_proj", I, H), ("mlp.up_proj", I, H), ("mlp.down_proj", H, I))
              for t in projection(f"{pre}.{n}", N, K, g)]
    whole = dict(stream)
    for rank in range(world):
        got = dict(ck.ingest(iter(stream), rank=rank, world=world, num_kv_heads=2, dtype=torch.float16))
        method = MXFP4Config().get_linear_method()
        for name, layer in (("self_attn.qkv_proj", QKVParallelLinear(H, D, 4, 2, False, method, world)),
                            ("self_attn.o_proj", RowParallelLinear(4 * D, H, False, method, world)),
                            ("mlp.gate_up_proj", MergedColumnParallelLinear(H, [I, I], False, method, world)),
                            ("mlp.down_proj", RowParallelLinear(I, H, False, method, world))):
            for key in layer.state_dict_keys(f"{pre}.{name}"):
                item, param = got[key], getattr(layer, key.split(".")[-1])
                assert item.shape == param.shape and item.dtype == param.dtype, key
        n = "mlp.down_proj"
        mine = oracle.values(got[f"{pre}.{n}.weight"], got[f"{pre}.{n}.weight_scale"])
        full = oracle.values(whole[f"{pre}.{n}.weight"], whole[f"{pre}.{n}.weight_scale"])
        assert torch.equal(mine, full.chunk(world, 1)[rank])
        mine = oracle.values(got[f"{pre}.mlp.gate_up_proj.weight"], got[f"{pre}.mlp.gate_up_proj.weight_scale"])
        parts = [oracle.values(whole[f"{pre}.mlp.{p}.weight"], whole[f"{pre}.mlp.{p}.weight_scale"]).chunk(world)[rank]
                 for p in ("gate_proj", "up_proj")]
        assert torch.equal(mine, torch.cat(parts))


@pytest.mark.parametrize("tp", [1, 2])
def test_expert_layer_holds_what_ingestion_yields(tp):
    g = torch.Generator().manual_seed(1)
    E, H, I = 3, 64, 128
    stream = [t for e in range(E) for n, N, K in (("gate_proj", I, H), ("up_proj", I, H), ("down_proj", H, I))
              for t in projection(f"{PRE}.{e}.{n}", N, K, g)]
    for rank in range(tp):
        sd = dict(ck.ingest(iter(stream), rank=rank, world=tp, num_experts=E))
        layer = MXFP4MoELayer(E, 2, H, I, tp_size=tp)
        want = layer.state_dict(prefix=PRE)
        assert set(want) == set(sd) and layer.state_dict_keys(PRE) == list(want)
        for k, v in want.items():
            assert v.shape == sd[k].shape and v.dtype == sd[k].dtype
        with pytest.raises(RuntimeError, match="not loaded"):
            layer(torch.zeros(2, H).half(), torch.zeros(2, E))
        for bad in ({k: v.char() for k, v in sd.items()}, {k: v[:, :-1] for k, v in sd.items()}):
            with pytest.raises(AssertionError):
                layer.load_state_dict(bad, prefix=PRE)
        short = dict(sd)
        short.pop(f"{PRE}.down_proj.weight_scale")
        with pytest.raises(KeyError):
            layer.load_state_dict(short, prefix=PRE)
        assert len(short) == 3  # nothing was taken
        with pytest.raises(ValueError, match="device tensors"):
            layer.load_state_dict(dict(sd), prefix=PRE)
    dense = MXFP4MoELayer(E, 2, H, I, serialized=False, params_dtype=torch.bfloat16)
    assert {k: (tuple(v.shape), v.dtype) for k, v in dense.state_dict().items()} == {
        "gate_up_proj": ((E, 2 * I, H), torch.bfloat16), "down_proj": ((E, H, I), torch.bfloat16)}


def test_layer_and_backend_refusals():
    for kw in (dict(intermediate_size=80), dict(hidden_size=48), dict(params_dtype=torch.float64), dict(top_k=0),
               dict(activation="relu"), dict(tp_size=4), dict(backend="fused"), dict(backend="awq_fused")):
        with pytest.raises(ValueError):
            MXFP4MoELayer(**{**dict(num_experts=4, top_k=2, hidden_size=64, intermediate_size=64), **kw})
    for layer in (MoELayer, AWQMoELayer):
        with pytest.raises(ValueError, match="backend"):
            layer(4, 2, 128, 128, backend="mxfp4_fused")
    E, H, I, T = 4, 64, 96, 3

    def stack(N, K):
        wb, sb = ops.mx4_weight_bytes(N, K)
        return ops.Mx4Weight(torch.zeros(E, wb, dtype=torch.uint8), torch.zeros(E, sb, dtype=torch.uint8), N, K)
    m1, m2 = stack(2 * I, H), stack(H, I)
    d1, d2 = torch.zeros(E, 2 * I, H).half(), torch.zeros(E, H, I).half()
    x, logits = torch.zeros(T, H).half(), torch.zeros(T, E)
    backend = create_moe_backend("mxfp4_fused")
    assert isinstance(backend, MXFP4FusedMoe)
    for pair in ((d1, d2), (m1, d2), (d1, m2), (object(), m2)):
        with pytest.raises(ValueError, match="mxfp4_fused"):
            backend.forward(x, *pair, logits, 2, True)
    for name in ("fused", "awq_fused"):
        for pair in ((m1, m2), (m1, d2), (d1, m2)):
            with pytest.raises(ValueError, match="mxfp4_fused"):
                create_moe_backend(name).forward(x, *pair, logits, 2, True)
    for pair in ((m1, d2), (d1, m2)):
        with pytest.raises(ValueError, match="both"):
            fused_experts_impl(x, *pair, torch.zeros(T, 2), torch.zeros(T, 2, dtype=torch.int32))
    for pair in ((m1, stack(H, 2 * I)), (stack(2 * I, 32), m2), (m1, stack(96, I))):
        with pytest.raises(AssertionError):
            backend.forward(x, *pair, logits, 2, True)
    with pytest.raises(ValueError, match="device tensors"):
        backend.forward(x, m1, m2, logits, 2, True)
