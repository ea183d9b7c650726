"""Which kernel an MXFP4 product takes, and the tiles of 128 columns against the formula in 64 bits: they run where
their grid gives half to all of the CUs a workgroup, through a ring of three stages of 512 k."""
import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import ops

DEV = "cuda"

# M, N, K, activation; stages of 512 k, what the last holds of them and of 128 k, row tiles of 2 to 8 m-tiles (the last
# one lower than the others), columns past N.  For 256 CUs.
NARROW = [
    (289, 5504, 512, None), (100, 24584, 352, None), (390, 4232, 544, None), (65, 32768, 672, None),
    (257, 6912, 1024, "silu"), (390, 4160, 1056, "silu"), (70, 16448, 1056, "gelu"), (1000, 2600, 1184, None),
    (130, 12288, 1600, "gelu"), (128, 16384, 2080, None), (333, 6144, 2560, None), (385, 4096, 2624, "gelu"),
    (128, 28672, 4096, "silu"), (1024, 2560, 9728, None), (2049, 1288, 1536, None),
]


def stages(K):
    return (K + 511) // 512


def narrow(M, N, K, act):
    p = ops.mx4_plan_info(M, N, K, act)
    return p.kernel == "mx4_tile_kernel" and p.columns == 128 and p.quantised_ahead


def test_the_shapes_below_take_tiles_of_128_columns():
    if ops.device_cu_count() != 256:
        pytest.skip("the shapes are for 256 CUs")
    for shape in NARROW:
        assert narrow(*shape), (shape, ops.mx4_plan_info(*shape))
    assert {stages(s[2]) for s in NARROW} >= {1, 2, 3, 4, 5, 8, 19}
    for M, N, act, kernel, columns in ((128, 16256, None, "mx4_rows_kernel", 32), (128, 16384, None, "mx4_tile_kernel", 128),
                                       (128, 32768, None, "mx4_tile_kernel", 128), (128, 32776, None, "mx4_tile_kernel", 256),
                                       (64, 32768, None, "mx4_rows_kernel", 32), (1, 64, "silu", "mx4_rows_kernel", 32)):
        p = ops.mx4_plan_info(M, N, 512, act)
        assert (p.kernel, p.columns) == (kernel, columns), (M, N, p)
    assert not ops.mx4_plan_info(8, 64, 64).quantised_ahead and ops.mx4_plan_info(8, 64, 64).workspace_bytes == 0
    assert ops.mx4_plan_info(9, 64, 64).quantised_ahead and ops.mx4_plan_info(9, 64, 64).workspace_bytes > 0


def test_refusals():
    for bad in ((0, 64, 64), (-1, 64, 64), (4, 60, 64), (4, 64, 60), (4, 32, 64, "silu"), (4, 64, 64, "relu")):
        with pytest.raises(ValueError):
            ops.mx4_plan_info(*bad)
    with pytest.raises(RuntimeError):
        ops.mx4_plan_info(1 << 24, 64, 64)


def inputs(M, N, K, dtype, seed):
    from tests.test_gpu_mx4_gemm import make

    x, codes, scales, w = make(M, N, K, dtype, seed)
    return x, codes, scales, w, torch.randn(N, generator=torch.Generator().manual_seed(seed + 1)).to(dtype).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K,act", NARROW)
def test_tiles_of_128_columns(M, N, K, act, dtype):
    from tests.test_gpu_mx4_gemm import close

    assert narrow(M, N, K, act)
    x, codes, scales, w, bias = inputs(M, N, K, dtype, M + K)
    xq, wv = oracle.quantized(x), oracle.values(codes, scales)
    for b in (bias, None):
        got = ops.mx4_gemm(x, w, bias=b, activation=act)
        y, err = oracle.product(xq, wv, b)
        close(got, *((y, err) if act is None else oracle.gated(y, err, act)))
        for _ in range(3):  # stages that had not landed would differ from run to run
            assert torch.equal(ops.mx4_gemm(x, w, bias=b, activation=act), got)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,act", [(390, 4232, 1184, None), (128, 24576, 2560, "silu")])
def test_rows_and_weights_that_are_not_finite(M, N, K, act):
    """In the last stage and in one before it; a stage that another unit left behind would spread them."""
    assert narrow(M, N, K, act)
    x, codes, scales, w, _ = inputs(M, N, K, torch.bfloat16, 5)
    x[3, K - 1], x[M - 1, 600] = float("nan"), float("inf")
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    bad[3] = bad[M - 1] = True
    y = ops.mx4_gemm(x, w, activation=act)
    assert torch.equal(torch.isnan(y).all(-1), bad) and torch.equal(torch.isnan(y).any(-1), bad)
    scales[7, K // 32 - 1], scales[40, 18] = 255, 255
    y = ops.mx4_gemm(x, ops.mx4_repack(ops.Mx4(codes, scales)), activation=act)[~bad]
    cols = torch.zeros(y.shape[1], dtype=torch.bool, device=DEV)
    cols[7] = cols[40] = True
    assert torch.equal(torch.isnan(y).all(0), cols) and torch.equal(torch.isnan(y).any(0), cols)


@pytest.mark.gpu
def test_captured_replays():
    M, N, K = 333, 6144, 1056
    assert narrow(M, N, K, None)
    x, _, _, w, bias = inputs(M, N, K, torch.float16, 1)
    ops.mx4_gemm(x, w, bias=bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx4_gemm(x, w, bias=bias)
    for seed in range(4):
        x.copy_(torch.randn((M, K), generator=torch.Generator().manual_seed(seed)))
        ops.mx4_gemm(x[:100], w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.mx4_gemm(x, w, bias=bias))
