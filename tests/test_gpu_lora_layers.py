"""Adapters through the layers that hold them: AWQ projections and the gated MLP, alone and captured."""
import pytest
import torch

from oracle import awq_oracle as oracle
from sglite_amd import ops
from sglite_amd.linear import MergedColumnParallelLinear, QKVParallelLinear, ReplicatedLinear, RowParallelLinear
from sglite_amd.mlp import GatedMLP
from sglite_amd.quantization import get_quantization_config

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Half a step of the type; the projections themselves are held to the engine's GEMM tolerance.
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
GEMM_TOL = 2e-2
H, I, HEADS, KV, D = 256, 384, 4, 2, 64


def method():
    return get_quantization_config("awq").from_config(
        {"bits": 4, "group_size": 64, "zero_point": True, "quant_method": "awq"}).get_linear_method()


def awq(K, N, dtype, seed):
    t = oracle.make_awq_linear(K, N, 64, seed=seed)
    t = {k: t[k].to(dtype) if k == "scales" else t[k] for k in ("qweight", "qzeros", "scales")}
    W = oracle.dequantize(t["qweight"], t["qzeros"], t["scales"], 64).double().to(DEV)
    return {k: v.to(DEV) for k, v in t.items()}, W


def build(make, shape, dtype, seed):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        layer = make()
    finally:
        torch.set_default_dtype(before)
    tensors, W = awq(*shape, dtype, seed)
    layer.load_state_dict(tensors)
    return layer, W


def fill(layer, slots, dtype, seed, skip=()):
    """Adapters of different ranks; returns each slot's full delta weight [K, N] in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    layer.add_adapters(slots, 24, dtype)
    K, deltas = layer.local_input_size, []
    for s in range(slots):
        a, b, cols = [], [], []
        for p, n in enumerate(layer._parts):
            r = 24 - 5 * ((s + p) % 4)
            A = (torch.randn((r, K), generator=g) / K ** 0.5).to(dtype).to(DEV)
            B = (torch.randn((n, r), generator=g) * 0.2).to(dtype).to(DEV)
            if (s, p) in skip:
                a.append(None), b.append(None)
                cols.append(torch.zeros((K, n), dtype=torch.float64, device=DEV))
            else:
                a.append(A), b.append(B)
                cols.append((B.double() @ A.double()).t())
        one = len(a) == 1
        layer.load_adapter(s, a[0] if one else a, b[0] if one else b, 0.5 + s)
        deltas.append((0.5 + s) * torch.cat(cols, 1))
    return deltas


def plain(x, W, deltas, ids):
    y = x.double() @ W
    for s, dW in enumerate(deltas):
        rows = ids == s
        y[rows] += x[rows].double() @ dW
    return y


def close(got, want):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs().max()
    assert err <= GEMM_TOL * want.abs().max(), float(err)


def ids_for(M, slots, seed):
    return torch.randint(-1, slots, (M,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 3, 40, 200])
def test_projections(M, dtype):
    for make, shape, skip in [
            (lambda: QKVParallelLinear(H, D, HEADS, KV, False, method()), (H, (HEADS + 2 * KV) * D), ((1, 1), (2, 0))),
            (lambda: RowParallelLinear(HEADS * D, H, False, method()), (HEADS * D, H), ()),
            (lambda: MergedColumnParallelLinear(H, [I, I], False, method()), (H, 2 * I), ((0, 0),)),
            (lambda: ReplicatedLinear(H, 96, False, method()), (H, 96), ())]:
        layer, W = build(make, shape, dtype, seed=M)
        x = torch.randn((M, shape[0]), generator=torch.Generator().manual_seed(M)).to(dtype).to(DEV)
        ids = ids_for(M, 3, M)
        batch = ops.lora_route(ids, 3)
        base = layer(x)
        assert torch.equal(layer(x, batch), base)  # no slots yet
        deltas = fill(layer, 3, dtype, seed=M, skip=skip)
        y = layer(x, batch)
        close(y, plain(x, W, deltas, ids))
        assert torch.equal(y[ids < 0], base[ids < 0]) and torch.equal(layer(x), base)
        # The step that adds is lora_add on the projection as stored.
        assert torch.equal(y, ops.lora_add(base, x, layer._lora, batch))
        assert torch.equal(layer(x.view(1, M, -1), batch), y.view(1, M, -1))
        if isinstance(layer, MergedColumnParallelLinear):
            g, u = plain(x, W, deltas, ids).chunk(2, 1)
            close(layer.forward_act(x, "silu", batch), torch.nn.functional.silu(g) * u)
        layer.clear_adapter(0)
        cleared = layer(x, batch)
        assert torch.equal(cleared[ids == 0], base[ids == 0]) and torch.equal(cleared[ids != 0], y[ids != 0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,one_launch", [(1, True), (6, False), (150, False)])
def test_gated_mlp_with_adapters_on_either_or_both(M, one_launch, dtype):
    x = torch.randn((M, H), generator=torch.Generator().manual_seed(M)).to(dtype).to(DEV)
    ids = ids_for(M, 2, M)
    batch = ops.lora_route(ids, 2)
    for which in ("gate_up_proj", "down_proj", "both"):
        before = torch.get_default_dtype()
        torch.set_default_dtype(dtype)
        try:
            mlp = GatedMLP(H, I, "silu", method(), one_launch=one_launch)
        finally:
            torch.set_default_dtype(before)
        gu, Wg = awq(H, 2 * I, dtype, 1)
        dn, Wd = awq(I, H, dtype, 2)
        mlp.load_state_dict({**{f"gate_up_proj.{k}": v for k, v in gu.items()},
                             **{f"down_proj.{k}": v for k, v in dn.items()}})
        base = mlp(x)
        dg = fill(mlp.gate_up_proj, 2, dtype, 3) if which != "down_proj" else []
        dd = fill(mlp.down_proj, 2, dtype, 4) if which != "gate_up_proj" else []
        g, u = plain(x, Wg, dg, ids).chunk(2, 1)
        close(mlp(x, batch), plain(torch.nn.functional.silu(g) * u, Wd, dd, ids))
        assert torch.equal(mlp(x), base)


def test_a_decode_step_captured_once_serves_other_adapters():
    """qkv, o and the MLP of a layer in one graph: new rows, slots and adapter weights at each replay."""
    dtype, M, slots = torch.float16, 12, 4
    qkv, _ = build(lambda: QKVParallelLinear(H, D, HEADS, KV, False, method()), (H, (HEADS + 2 * KV) * D), dtype, 5)
    o, _ = build(lambda: RowParallelLinear(HEADS * D, H, False, method()), (HEADS * D, H), dtype, 6)
    torch.set_default_dtype(dtype)
    try:
        mlp = GatedMLP(H, I, "silu", method())
    finally:
        torch.set_default_dtype(torch.float32)
    gu, _ = awq(H, 2 * I, dtype, 7)
    dn, _ = awq(I, H, dtype, 8)
    mlp.load_state_dict({**{f"gate_up_proj.{k}": v for k, v in gu.items()},
                         **{f"down_proj.{k}": v for k, v in dn.items()}})
    layers = [qkv, o, mlp.gate_up_proj, mlp.down_proj]
    for n, layer in enumerate(layers):
        fill(layer, slots, dtype, n)
    x = torch.randn((M, H), device=DEV).to(dtype)
    ids = ids_for(M, slots, 0)

    def step():
        batch = ops.lora_route(ids, slots)
        t = qkv(x, batch)
        return mlp(o(t[:, :HEADS * D].contiguous(), batch) + x, batch)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(5):
        x.copy_(torch.randn((M, H), device=DEV))
        ids.copy_(ids_for(M, slots, 10 + n))
        K, N = o.local_input_size, o._parts[0]
        o.load_adapter(n % slots, torch.randn((3 + n, K), device=DEV) / 16, torch.randn((N, 3 + n), device=DEV), 0.25)
        want = step()
        graph.replay()
        assert torch.equal(out, want)
