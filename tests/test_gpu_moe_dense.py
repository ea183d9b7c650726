"""Grouped products of dense experts against the formula in 64 bits."""
import pytest
import torch

from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type


def make(T, E, k, K, N, dtype, seed=0, load="even"):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn((T, K), generator=g).to(dtype).to(DEV)
    w = (torch.randn((E, N, K), generator=g) / K ** 0.5).to(dtype).to(DEV)
    if load == "one":  # everything on one expert
        ids = torch.full((T, k), E // 2)
    else:
        bias = torch.randn(E, generator=g) * (2.0 if load == "skewed" else 0.0)
        ids = torch.topk(torch.randn((T, E), generator=g) + bias, k, -1).indices
    weights = torch.rand((T, k), generator=g) + 0.1
    return a, w, ids.to(torch.int32).to(DEV), weights.to(DEV)


def formula(a, w, ids, top_k, weights, act):
    """Every routed row's result and a bound of its error before the last rounding, in 64 bits."""
    flat = ids.reshape(-1).long()
    E, N, K = w.shape
    out = torch.zeros((flat.numel(), N), dtype=torch.float64, device=a.device)
    err = torch.zeros_like(out)
    for e in range(E):
        rows = (flat == e).nonzero().reshape(-1)
        if rows.numel():
            x, W = a[rows // top_k].double(), w[e].double()
            out[rows] = x @ W.t()
            err[rows] = (K + 8) * 2.0 ** -24 * (x.abs() @ W.abs().t())  # fp32 sums of K products
    if weights is not None:
        out, err = out * weights.reshape(-1, 1).double(), err * weights.reshape(-1, 1).double()
        err += 2.0 ** -23 * out.abs()
    if act is None:
        return out, err
    h = N // 2
    g, u, eg, eu = out[:, :h], out[:, h:], err[:, :h], err[:, h:]
    f = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    # Slopes of silu and gelu stay below 1.13; exp, erf and the divide within 2^-20 of the factors.
    return f * u, 1.13 * eg * (u.abs() + eu) + f.abs() * eu + 2.0 ** -20 * ((f * u).abs() + (g * u).abs())


def close(got, want, err):
    tol = err + HALF[got.dtype] * (want.abs() + err) + 2.0 ** -25
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float(((got.double() - want).abs() - tol).max()):.3e}"


SHAPES = [
    # T, E, k, K, N, load
    (1, 8, 2, 64, 32, "even"),
    (1, 128, 8, 2048, 1536, "even"),
    (3, 4, 1, 8, 16, "even"),
    (7, 16, 4, 72, 80, "even"),
    (16, 128, 8, 768, 2048, "even"),
    (33, 8, 2, 328, 208, "skewed"),
    (64, 512, 2, 64, 48, "even"),
    (100, 1, 1, 200, 336, "even"),
    (129, 6, 3, 1000, 272, "skewed"),
    (300, 4, 2, 136, 144, "one"),
    (512, 32, 4, 256, 512, "even"),
    (777, 5, 2, 520, 400, "skewed"),
    (1030, 3, 1, 384, 1040, "one"),
    (2048, 16, 4, 512, 528, "skewed"),
    (300, 200, 8, 64, 48, "even"),
    (1500, 300, 2, 72, 272, "skewed"),
    (700, 2, 1, 8, 16, "even"),
]


@pytest.mark.parametrize("E,n", [(4, 700), (2, 1), (300, 1300)])
def test_buckets_padded_to_long_blocks(E, n):
    """Tiles of padding alone in front of other experts' rows."""
    a, w, ids, _ = make(n, E, 1, 136, 48, torch.bfloat16, load="skewed")
    align = ops.moe_align_block_size(ids, 1024, E)
    close(ops.moe_dense_gemm(a, w, align, None, n, 1), *formula(a, w, ids, 1, None, None))


def test_weights_and_rows_on_another_stream():
    a, w, ids, weights = make(900, 4, 2, 512, 256, torch.float16)
    want, err = formula(a, w, ids, 2, weights, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        align = ops.moe_align_block_size(ids, 16, 4)
        got = [ops.moe_dense_gemm(a, w, align, weights, 1800, 2, "silu", True) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(got[0], t) for t in got)
    close(got[0], want, err)


def test_layers_share_a_graph_with_adapters_between():
    """A step's projections with adapters and expert products in one graph, replayed with other ids."""
    a, w, ids, weights = make(40, 8, 2, 256, 128, torch.float16)
    stack = ops.make_lora_stack(3, 16, 256, (256,), torch.float16, torch.device(DEV))
    stack.a.normal_(std=0.05), stack.b.normal_(std=0.2), stack.scaling.fill_(1.0), stack.ranks.fill_(16)
    slots = torch.randint(-1, 3, (40,), dtype=torch.int32, device=DEV)

    def step():
        x = ops.lora_add(a, a, stack, ops.lora_route(slots, 3))
        return ops.moe_dense_gemm(x, w, ops.moe_align_block_size(ids, 16, 8), weights, 80, 2, "gelu", True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        ids.copy_(torch.randint(0, 8, ids.shape, dtype=torch.int32, device=DEV))
        slots.copy_(torch.randint(-1, 3, slots.shape, dtype=torch.int32, device=DEV))
        want = step()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,K,N,load", SHAPES)
def test_products(T, E, k, K, N, load, dtype):
    a, w, ids, weights = make(T, E, k, K, N, dtype, seed=T, load=load)
    n = T * k
    for block in (16, 64):
        align = ops.moe_align_block_size(ids, block, E)
        close(ops.moe_dense_gemm(a, w, align, None, n, k), *formula(a, w, ids, k, None, None))
        close(ops.moe_dense_gemm(a, w, align, weights, n, k, mul_routed_weight=True),
              *formula(a, w, ids, k, weights, None))
        close(ops.moe_dense_gemm(a, w, align, weights, n, k), *formula(a, w, ids, k, None, None))
        close(ops.moe_dense_gemm(a, w, align, None, n, k, activation="silu"), *formula(a, w, ids, k, None, "silu"))
        close(ops.moe_dense_gemm(a, w, align, weights, n, k, activation="gelu", mul_routed_weight=True),
              *formula(a, w, ids, k, weights, "gelu"))
    # One activation row per routed row, as for the second product.
    rows = torch.randn((n, K), device=DEV).to(dtype)
    close(ops.moe_dense_gemm(rows, w, align, weights, n, 1, mul_routed_weight=True),
          *formula(rows, w, ids, 1, weights, None))


@pytest.mark.parametrize("T", [3, 200])
def test_rows_of_no_expert_are_not_written(T):
    a, w, ids, _ = make(T, 4, 2, 128, 96, torch.float16)
    ids[::3] = torch.tensor([-1, 4], dtype=torch.int32, device=DEV)
    align = ops.moe_align_block_size(ids, 16, 4)
    out = torch.full((2 * T, 96), 5.0, dtype=a.dtype, device=DEV)
    got = ops.moe_dense_gemm(a, w, align, None, 2 * T, 2, out=out)
    none = ((ids < 0) | (ids >= 4)).reshape(-1)
    want, err = formula(a, w, ids, 2, None, None)
    assert got is out and (out[none] == 5.0).all()
    close(out[~none], want[~none], err[~none])
    ids[:] = -1
    out.fill_(3.0)
    ops.moe_dense_gemm(a, w, ops.moe_align_block_size(ids, 16, 4), None, 2 * T, 2, out=out)
    assert (out == 3.0).all()


def test_no_rows():
    a, w, ids, _ = make(0, 4, 2, 64, 32, torch.bfloat16)
    assert ops.moe_dense_gemm(a, w, ops.moe_align_block_size(ids, 16, 4), None, 0, 2).shape == (0, 32)


@pytest.mark.parametrize("T", [20, 600])
def test_infinite_and_nan_values_stay_in_their_rows_and_experts(T):
    for dtype in (torch.float16, torch.bfloat16):
        a, w, ids, _ = make(T, 4, 2, 200, 72, dtype, load="skewed")
        want, err = formula(a, w, ids, 2, None, None)
        a[3, 199], w[1] = float("inf"), float("nan")
        got = ops.moe_dense_gemm(a, w, ops.moe_align_block_size(ids, 16, 4), None, 2 * T, 2)
        flat = ids.reshape(-1)
        clean = flat != 1
        hit = torch.zeros_like(clean)
        hit[6:8] = True
        close(got[clean & ~hit], want[clean & ~hit], err[clean & ~hit])
        assert got[~clean].isnan().all() and not got[hit].isfinite().any()


def test_strided_and_offset_inputs():
    a, w, ids, weights = make(70, 4, 2, 128, 96, torch.bfloat16)
    align = ops.moe_align_block_size(ids, 16, 4)
    want, err = formula(a, w, ids, 2, weights, None)
    wide = torch.zeros((70, 131), dtype=a.dtype, device=DEV)
    wide[:, 3:] = a
    double = torch.zeros((70, 4), dtype=torch.float64, device=DEV)
    double[:, ::2] = weights.double()
    got = ops.moe_dense_gemm(wide[:, 3:], w, align, double[:, ::2], 140, 2, mul_routed_weight=True)
    close(got, want, err)
    more = torch.cat([a, torch.full((5, 128), float("nan"), dtype=a.dtype, device=DEV)])
    close(ops.moe_dense_gemm(more, w, align, weights, 140, 2, mul_routed_weight=True), want, err)


@pytest.mark.parametrize("T", [8, 400])
def test_same_bits_every_time_and_in_a_replayed_graph(T):
    a, w, ids, weights = make(T, 16, 4, 512, 256, torch.float16)
    n = T * 4

    def step():
        align = ops.moe_align_block_size(ids, 16, 16)
        return (ops.moe_dense_gemm(a, w, align, None, n, 4, activation="silu"),
                ops.moe_dense_gemm(a, w, align, weights, n, 4, mul_routed_weight=True))

    first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, first))
        ids.copy_(torch.randint(0, 16, ids.shape, dtype=torch.int32, device=DEV))
        first = step()
        if i % 2:
            torch.cuda.synchronize()


def test_registered_op():
    a, w, ids, weights = make(20, 4, 2, 64, 32, torch.float16)
    align = ops.moe_align_block_size(ids, 16, 4)
    out = torch.zeros((40, 16), dtype=a.dtype, device=DEV)
    args = (a, w, align.sorted_ids, align.expert_offsets, weights, out, 40, 2, "silu", True)
    torch.library.opcheck(torch.ops.sglite_awq.awq_moe_dense_gemm, args,
                          test_utils=("test_schema", "test_faketensor"))
    torch.ops.sglite_awq.awq_moe_dense_gemm(*args)
    assert torch.equal(out, ops.moe_dense_gemm(a, w, align, weights, 40, 2, "silu", True))
