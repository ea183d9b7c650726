"""Dense experts end to end: checkpoint stream, layer, backend, against the block in 64 bits."""
import pytest
import torch

from sglite_amd import checkpoint as ck
from sglite_amd.moe import MoELayer, create_moe_backend, fused_experts_impl, fused_topk

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2e-2  # of the largest output, as the engine's fused MoE is held to
PRE = "model.layers.0.mlp.experts"


def stream(E, H, I, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [(f"{PRE}.{e}.{n}.weight", (torch.randn(shape, generator=g) / shape[1] ** 0.5).to(dtype))
            for e in range(E) for n, shape in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I)))]


def block(x, w1, w2, logits, k, renormalize, act="silu", on_input=False):
    p, ids = torch.sort(torch.softmax(logits.double(), -1), dim=-1, descending=True, stable=True)
    p, ids = p[:, :k], ids[:, :k]
    p = p / (p.sum(-1, keepdim=True) + 1e-8) if renormalize else p
    out = torch.zeros(x.shape, dtype=torch.float64)
    f = torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu
    for e in range(w1.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            s = p[t, j, None]
            g, u = (x[t].double() @ w1[e].double().t() * (s if on_input else 1)).chunk(2, -1)
            out.index_add_(0, t, f(g) * u @ w2[e].double().t() * (1 if on_input else s))
    return out


def close(got, want):
    assert torch.isfinite(got).all()
    assert (got.double().cpu() - want).abs().max() <= TOL * want.abs().max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 128, 8, 256, 96), (5, 8, 2, 264, 136), (37, 8, 2, 512, 256),
                                       (400, 6, 3, 192, 88), (900, 4, 1, 256, 320)])
def test_layer_from_checkpoint(T, E, k, H, I, dtype):
    sd = dict(ck.ingest(stream(E, H, I, dtype, T), num_experts=E))
    layer = MoELayer(E, k, H, I, params_dtype=dtype)
    layer.load_state_dict({n: v.to(DEV) for n, v in sd.items()}, prefix=PRE)
    g = torch.Generator().manual_seed(T)
    x, logits = torch.randn((T, H), generator=g).to(dtype), torch.randn((T, E), generator=g)
    w1, w2 = sd[f"{PRE}.gate_up_proj"], sd[f"{PRE}.down_proj"]
    xd = x.to(DEV)
    out = layer(xd, logits.to(DEV))
    assert out.data_ptr() == xd.data_ptr()  # the block writes its result over its input
    close(out, block(x, w1, w2, logits, k, True))
    backend = create_moe_backend("fused")
    for act, on_input, renorm in (("gelu", False, False), ("silu", True, False)):
        y = backend.forward(x.to(DEV), w1.to(DEV), w2.to(DEV), logits.to(DEV), k, renorm, act, on_input)
        close(y, block(x, w1, w2, logits, k, renorm, act, on_input))


def test_tensor_parallel_shards_sum_to_the_full_layer():
    E, H, I, k, T, tp = 8, 128, 192, 3, 29, 2
    w = stream(E, H, I, torch.float16, 7)
    full = dict(ck.ingest(w, num_experts=E))
    g = torch.Generator().manual_seed(9)
    x, logits = torch.randn((T, H), generator=g).half(), torch.randn((T, E), generator=g)
    total = torch.zeros((T, H), dtype=torch.float64)
    for rank in range(tp):
        sd = dict(ck.ingest(w, rank=rank, world=tp, num_experts=E))
        layer = MoELayer(E, k, H, I, renormalize=False, tp_size=tp)
        layer.load_state_dict({n: v.to(DEV) for n, v in sd.items()}, prefix=PRE)
        xd = x.to(DEV)
        tw, ids = fused_topk(xd, logits.to(DEV), k, False)
        total += fused_experts_impl(xd, layer.gate_up_proj, layer.down_proj, tw, ids).double().cpu()
    close(total, block(x, full[f"{PRE}.gate_up_proj"], full[f"{PRE}.down_proj"], logits, k, False))


def test_padded_tokens_leave_the_others_alone_and_no_tokens():
    E, H, I, k = 4, 64, 48, 2
    sd = dict(ck.ingest(stream(E, H, I, torch.float16, 1), num_experts=E))
    w1, w2 = sd[f"{PRE}.gate_up_proj"].to(DEV), sd[f"{PRE}.down_proj"].to(DEV)
    g = torch.Generator().manual_seed(2)
    x, logits = torch.randn((20, H), generator=g).half(), torch.randn((20, E), generator=g)
    x[13:] = float("nan")
    xd = x.to(DEV)
    tw, ids = fused_topk(xd, logits.to(DEV), k, True, num_token_non_padded=torch.tensor(13, device=DEV))
    assert (ids[13:] == -1).all()
    out = fused_experts_impl(xd, w1, w2, tw, ids)
    close(out[:13], block(x[:13], w1.cpu(), w2.cpu(), logits[:13], k, True))
    empty = create_moe_backend("fused").forward(xd[:0], w1, w2, logits[:0].to(DEV), k, True)
    assert empty.shape == (0, H)


def test_captured_block_follows_new_tokens():
    E, H, I, k, T = 16, 256, 128, 4, 24
    sd = dict(ck.ingest(stream(E, H, I, torch.bfloat16, 3), num_experts=E))
    layer = MoELayer(E, k, H, I, params_dtype=torch.bfloat16)
    layer.load_state_dict({n: v.to(DEV) for n, v in sd.items()}, prefix=PRE)
    x, logits = torch.randn((T, H), device=DEV).bfloat16(), torch.randn((T, E), device=DEV)
    layer(x.clone(), logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x.clone(), logits)
    for _ in range(4):
        x.copy_(torch.randn((T, H), device=DEV))
        logits.copy_(torch.randn((T, E), device=DEV))
        want = layer(x.clone(), logits)
        graph.replay()
        assert torch.equal(out, want)
