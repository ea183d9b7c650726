"""Grouped products of MXFP4 experts against the formula in 64 bits."""
import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import ops
from tests.test_gpu_mx4_gemm import close, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def route(T, E, k, load="even", seed=0):
    g = torch.Generator().manual_seed(seed)
    if load == "one":  # everything on one expert
        ids = torch.full((T, k), E // 2)
    else:
        bias = torch.randn(E, generator=g) * (2.0 if load == "skewed" else 0.0)
        ids = torch.topk(torch.randn((T, E), generator=g) + bias, k, -1).indices
    return ids.to(torch.int32).to(DEV), (torch.rand((T, k), generator=g) + 0.1).to(DEV)


def formula(a, codes, scales, ids, top_k, weights, act):
    flat, xq = ids.reshape(-1).long(), oracle.quantized(a)
    N = codes.shape[1]
    out = torch.zeros((flat.numel(), N if act is None else N // 2), dtype=torch.float64, device=DEV)
    err = torch.zeros_like(out)
    for e in range(codes.shape[0]):
        rows = (flat == e).nonzero().reshape(-1)
        if rows.numel():
            rw = None if weights is None else weights.reshape(-1, 1)[rows].double()
            y, b = oracle.product(xq[rows // top_k], oracle.values(codes[e], scales[e]), None, rw)
            out[rows], err[rows] = (y, b) if act is None else oracle.gated(y, b, act)
    return out, err


SHAPES = [
    # T, E, k, K, N, load
    (1, 8, 2, 64, 64, "even"), (1, 128, 8, 2048, 1536, "even"), (3, 4, 1, 32, 64, "even"), (7, 16, 4, 96, 192, "even"),
    (24, 128, 8, 2048, 1536, "even"), (40, 5, 2, 544, 128, "skewed"), (64, 160, 6, 256, 192, "even"),
    (100, 300, 4, 128, 64, "skewed"), (200, 4, 2, 160, 448, "one"), (333, 16, 2, 1056, 320, "skewed"),
    (700, 8, 2, 512, 640, "even"), (512, 64, 8, 1024, 768, "skewed"), (1500, 3, 1, 288, 192, "skewed"),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,K,N,load", SHAPES)
def test_products(T, E, k, K, N, load, dtype):
    a, codes, scales, w = make(T, N, K, dtype, E=E)
    ids, tw = route(T, E, k, load)
    align = ops.moe_align_block_size(ids, 16, E)
    for act in ("silu", "gelu") if T < 300 else ("silu",):
        got = ops.mx4_moe_gemm(a, w, align, None, T * k, k, activation=act)
        close(got, *formula(a, codes, scales, ids, k, None, act))
    got = ops.mx4_moe_gemm(a, w, align, tw, T * k, k, activation="silu", mul_routed_weight=True)
    close(got, *formula(a, codes, scales, ids, k, tw, "silu"))
    h, codes, scales, w = make(T * k, 200, K, dtype, seed=1, E=E)
    got = ops.mx4_moe_gemm(h, w, align, tw, T * k, 1, mul_routed_weight=True)
    close(got, *formula(h, codes, scales, ids, 1, tw, None))


@pytest.mark.parametrize("T", [2, 9, 300])
def test_ids_outside_the_experts_leave_their_rows(T):
    a, codes, scales, w = make(T, 64, 96, torch.float16, E=6)
    ids, tw = route(T, 6, 2)
    ids[0, 1], ids[T // 2, 0] = -1, 6
    align = ops.moe_align_block_size(ids, 16, 6)
    out = torch.full((2 * T, 64), 7.0, dtype=torch.float16, device=DEV)
    assert ops.mx4_moe_gemm(a, w, align, tw, 2 * T, 2, out=out) is out
    live = ((ids >= 0) & (ids < 6)).reshape(-1)
    want, err = formula(a, codes, scales, ids, 2, None, None)
    close(out[live], want[live], err[live])
    assert (out[~live] == 7).all() and int((~live).sum()) == 2
    ids.fill_(-1)  # no row at all
    out.fill_(7)
    ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, 6), tw, 2 * T, 2, out=out)
    assert (out == 7).all()


@pytest.mark.parametrize("T", [3, 250])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_rows_aligned_to_larger_blocks(T, block):
    E, k = 9, 2
    a, codes, scales, w = make(T, 96, 160, torch.bfloat16, E=E)
    ids, tw = route(T, E, k, "skewed")
    got = ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, block, E), tw, T * k, k, mul_routed_weight=True)
    close(got, *formula(a, codes, scales, ids, k, tw, None))


@pytest.mark.parametrize("T", [2, 90])
def test_a_token_that_names_an_expert_twice(T):
    a, codes, scales, w = make(T, 64, 96, torch.float16, E=5)
    ids, tw = route(T, 5, 3)
    ids[:, 2] = ids[:, 0]
    got = ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, 5), tw, 3 * T, 3, "silu")
    close(got, *formula(a, codes, scales, ids, 3, None, "silu"))


def test_stacks_past_31_bits():
    E, N, K = 9, 16384, 31744
    g = torch.Generator(device=DEV).manual_seed(0)
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(118, 122, (E, N, K // 32), generator=g, device=DEV, dtype=torch.uint8)
    w = ops.mx4_repack(ops.Mx4(codes, scales))
    assert w.w.numel() > 1 << 31
    cols = torch.tensor([0, 9000, N - 1], device=DEV)
    for T in (2, 100):
        a = torch.randn((T, K), generator=g, device=DEV).half()
        ids, tw = route(T, E, 2)
        ids[0, 0] = E - 1
        got = ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, E), tw, 2 * T, 2)
        close(got[:, cols], *formula(a, codes[:, cols], scales[:, cols], ids, 2, None, None))


def test_no_tokens():
    _, _, _, w = make(1, 64, 96, torch.float16, E=6)
    ids = torch.empty((0, 2), dtype=torch.int32, device=DEV)
    y = ops.mx4_moe_gemm(torch.empty((0, 96), dtype=torch.float16, device=DEV), w, ops.moe_align_block_size(ids, 16, 6),
                         None, 0, 2)
    assert y.shape == (0, 64)


@pytest.mark.parametrize("T", [3, 200])
def test_rows_that_are_not_finite(T):
    a, codes, scales, w = make(T, 64, 352, torch.bfloat16, E=4)
    ids, tw = route(T, 4, 2)
    a[T // 2, 351] = float("nan")
    y = ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, 4), None, 2 * T, 2, "silu").view(T, 2, 32)
    bad = torch.zeros(T, dtype=torch.bool, device=DEV)
    bad[T // 2] = True
    assert torch.equal(torch.isnan(y).flatten(1).all(-1), bad) and torch.equal(torch.isnan(y).flatten(1).any(-1), bad)


@pytest.mark.parametrize("T", [2, 150])
def test_captured_replays_with_other_routes(T):
    E, k = 16, 4
    a, codes, scales, w = make(T, 128, 160, torch.bfloat16, E=E)
    ids, tw = route(T, E, k)
    ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, E), tw, T * k, k, "silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, E), tw, T * k, k, "silu", True)
    for seed in range(4):
        i, t = route(T, E, k, "skewed", seed)
        ids.copy_(i)
        tw.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.mx4_moe_gemm(a, w, ops.moe_align_block_size(ids, 16, E), tw, T * k, k, "silu", True))
