"""Dense experts: the layer's state-dict contract and every refusal ahead of a launch (no GPU)."""
import pytest
import torch

from sglite_amd import _lib, ops
from sglite_amd import checkpoint as ck
from sglite_amd.moe import FusedMoe, MoELayer, create_moe_backend

PRE = "model.layers.1.mlp.experts"


def checkpoint(E, H, I, seed=0):
    g = torch.Generator().manual_seed(seed)
    for e in range(E):
        for n, shape in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
            yield f"{PRE}.{e}.{n}.weight", torch.randn(shape, generator=g).half()


@pytest.mark.parametrize("tp", [1, 2])
def test_layer_loads_what_ingestion_yields(tp):
    E, H, I = 3, 40, 48
    for rank in range(tp):
        sd = dict(ck.ingest(checkpoint(E, H, I), rank=rank, world=tp, num_experts=E))
        layer = MoELayer(E, 2, H, I, tp_size=tp)
        want = layer.state_dict(prefix=PRE)
        assert set(want) == set(sd) and layer.state_dict_keys(PRE) == list(want)
        for k, v in want.items():
            assert v.shape == sd[k].shape and v.dtype == sd[k].dtype
        with pytest.raises(RuntimeError, match="not loaded"):
            layer(torch.zeros(2, H).half(), torch.zeros(2, E))
        for bad in ({k: v.bfloat16() for k, v in sd.items()}, {k: v[:, :-1] for k, v in sd.items()}):
            with pytest.raises(AssertionError):
                layer.load_state_dict(bad, prefix=PRE)
        with pytest.raises(KeyError):
            layer.load_state_dict({f"{PRE}.gate_up_proj": sd[f"{PRE}.gate_up_proj"]}, prefix=PRE)
        assert layer.gate_up_proj.is_meta  # nothing was taken
        with pytest.raises(RuntimeError, match="Unexpected"):
            layer.load_state_dict({**sd, "other": torch.zeros(1)}, prefix=PRE)
        layer.load_state_dict(dict(sd), prefix=PRE)
        assert torch.equal(layer.down_proj, sd[f"{PRE}.down_proj"])
        with pytest.raises(ValueError, match="device tensors"):
            layer(torch.zeros(2, H).half(), torch.zeros(2, E))


def test_misaligned_checkpoint_tensors_are_moved():
    layer = MoELayer(2, 1, 16, 24)
    flat = torch.arange(2 * 48 * 16 + 2 * 16 * 24 + 1, dtype=torch.float16)[1:]
    up, down = flat[:2 * 48 * 16].view(2, 48, 16), flat[2 * 48 * 16:].view(2, 16, 24)
    layer.load_state_dict({"gate_up_proj": up, "down_proj": down})
    assert layer.gate_up_proj.data_ptr() % 16 == 0 and torch.equal(layer.gate_up_proj, up)
    assert layer.down_proj.data_ptr() % 16 == 0 and torch.equal(layer.down_proj, down)


def test_layer_and_backend_refusals():
    for kw in (dict(intermediate_size=20), dict(hidden_size=36), dict(params_dtype=torch.float32),
               dict(top_k=0), dict(top_k=5), dict(activation="relu"), dict(intermediate_size=40, tp_size=3)):
        with pytest.raises(ValueError):
            MoELayer(**{**dict(num_experts=4, top_k=2, hidden_size=32, intermediate_size=48), **kw})
    backend = create_moe_backend("fused")
    assert isinstance(backend, FusedMoe)
    x, logits = torch.zeros(2, 32).half(), torch.zeros(2, 4)
    w1, w2 = torch.zeros(4, 96, 32).half(), torch.zeros(4, 32, 48).half()
    with pytest.raises(ValueError, match="awq_fused"):
        backend.forward(x, object(), w2, logits, 2, True)
    for a, b in ((w1[:, :, :24], w2), (w1, w2[:3]), (w1, w2[:, :, :40]), (w1[:, :80], w2), (w1[0], w2)):
        with pytest.raises(AssertionError):
            backend.forward(x, a, b, logits, 2, True)
    with pytest.raises(ValueError):
        backend.forward(x, w1, w2, logits, 2, True, activation="relu")


def test_python_refusals():
    a, w = torch.zeros(4, 64).half(), torch.zeros(3, 32, 64).half()
    i32 = torch.int32
    al = ops.MoeAlignment(torch.zeros(53, dtype=i32), torch.zeros(4, dtype=i32), torch.zeros(1, dtype=i32),
                          torch.zeros(4, dtype=i32))
    tw = torch.ones(4, 2)
    ok = dict(a=a, w=w, align=al, topk_weights=tw, num_routed=8, top_k=2)
    for bad in (dict(w=w[0]), dict(a=a[0]), dict(a=a[:, :32]), dict(a=a.bfloat16()), dict(a=a.float(), w=w.float()),
                dict(w=torch.zeros(3, 64, 32).half().transpose(1, 2)),
                dict(w=torch.zeros(3 * 32 * 64 + 1).half()[1:].view(3, 32, 64)), dict(activation="relu"),
                dict(topk_weights=None, mul_routed_weight=True), dict(topk_weights=tw[:3]), dict(num_routed=-1),
                dict(top_k=0), dict(align=al._replace(expert_offsets=torch.zeros(5, dtype=i32))),
                dict(align=al._replace(sorted_ids=torch.zeros(53, dtype=torch.int64)))):
        with pytest.raises(ValueError):
            ops.moe_dense_gemm(**{**ok, **bad})
    with pytest.raises(ValueError, match="device tensors"):  # all else is in order
        ops.moe_dense_gemm(**ok)


def _call(lib, **kw):
    p = dict(a=4096, rows=4, w=8192, E=3, N=64, K=64, dtype=0, ids=64, cap=100, off=128, tw=256, n=8, k=2, act=0, mul=1,
             out=65536)
    p.update(kw)
    return lib.awq_moe_dense_gemm(p["a"], p["rows"], p["w"], p["E"], p["N"], p["K"], p["dtype"], p["ids"], p["cap"],
                                  p["off"], p["tw"], p["n"], p["k"], p["act"], p["mul"], p["out"], None)


def test_c_abi_refusals():
    """Every bad call is turned away before a launch (the pointers are never read)."""
    lib = _lib.load()
    inv, uns = _lib.AWQ_STATUS_INVALID_ARGUMENT, _lib.AWQ_STATUS_UNSUPPORTED
    for want, kw in [
            (inv, dict(dtype=2)), (inv, dict(N=60)), (inv, dict(K=60)), (inv, dict(N=0)), (inv, dict(K=-8)),
            (inv, dict(act=3)), (inv, dict(act=1, N=72)), (inv, dict(k=0)), (inv, dict(rows=3)), (inv, dict(a=None)),
            (inv, dict(w=None)), (inv, dict(ids=None)), (inv, dict(off=None)), (inv, dict(out=None)),
            (inv, dict(tw=None)), (inv, dict(a=4104)), (inv, dict(w=8194)), (inv, dict(out=65544)),
            (uns, dict(E=0)), (uns, dict(E=513)), (uns, dict(n=-1)), (uns, dict(n=1 << 24, rows=1 << 24)),
            (uns, dict(cap=1 << 30)), (uns, dict(N=1 << 24, K=64)), (uns, dict(n=1 << 22, rows=1 << 22, k=1, K=256)),
            (uns, dict(K=1 << 30)), (uns, dict(N=1 << 30, K=8))]:
        assert _call(lib, **kw) == want, kw
        assert lib.awq_last_error()
    assert _call(lib, n=0, a=None, out=None) == 0 and _call(lib, cap=0) == 0
