"""MXFP4 blocks on the GPU: codes and bytes equal the oracle's, value by value; layouts there and back."""
import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(x):
    q = ops.mx4_quantize(x)
    codes, scales = oracle.quantize(x)
    assert torch.equal(q.scales, scales)
    live = (scales != 255).repeat_interleave(16, -1)
    assert torch.equal(q.codes[live], codes[live])
    for dtype in TYPES:
        got, want = ops.mx4_dequantize(q, dtype), oracle.values(codes, scales).to(dtype)
        assert got.dtype == dtype and got.shape == x.shape
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("order", ["sorted", "mixed"])
def test_every_16_bit_value(dtype, order):
    bits = torch.arange(1 << 16, dtype=torch.int32)
    if order == "mixed":
        bits = bits[torch.randperm(1 << 16, generator=torch.Generator().manual_seed(3))]
    check(bits.to(torch.int16).view(dtype).reshape(-1, 64).to(DEV))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_finite_value_under_larger_ones(dtype):
    """Each value in a block whose largest is 1 to 64 times it, of either sign."""
    v = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    for shift in range(7):
        x = v[:v.numel() // 16 * 16].reshape(-1, 16)
        top = (x.float() * 2.0 ** shift).amax(-1, keepdim=True).to(dtype)
        check(torch.cat((x, -top.expand(-1, 16)), -1).contiguous().to(DEV))


@pytest.mark.parametrize("scale", [2.0 ** -140, 2.0 ** -126, 1e-3, 1.0, 2.0 ** 125])
def test_fp32_values_at_the_borders(scale):
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    near = torch.cat((mids, torch.nextafter(mids, mids - 1), torch.nextafter(mids, mids + 1)))
    g = torch.Generator().manual_seed(5)
    rows = []
    for top in (4.0, 4.0000005, 5.5, 7.9999995):
        pick = near[torch.randint(0, near.numel(), (40, 31), generator=g)]
        rows.append(torch.cat((torch.full((40, 1), top), torch.minimum(pick, torch.tensor(top))), -1))
    x = torch.cat(rows) * torch.where(torch.rand((160, 32), generator=g) < 0.5, -1.0, 1.0)
    check((x * scale).to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 32), (7, 2560), (333, 96), (2, 5, 160), (1, 9728), (0, 64)])
def test_shapes(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[-1], generator=g))
    check(x.to(dtype).to(DEV))


def test_blocks_that_are_not_finite_or_empty():
    x = torch.ones((6, 96), device=DEV)
    x[0, 5], x[1, 40], x[2, 95], x[3, 32:64], x[4, :32] = float("inf"), float("-inf"), float("nan"), 0.0, -0.0
    for dtype in TYPES:
        check(x.to(dtype))
    y = ops.mx4_dequantize(ops.mx4_quantize(x))
    assert torch.isnan(y).sum() == 96 and torch.isnan(y[0, :32]).all() and (y[5] == 1).all()


def test_views():
    """Transposed, strided, offset and expanded inputs are read as they stand."""
    g = torch.Generator().manual_seed(9)
    big = torch.randn((130, 200), generator=g).to(DEV)
    for x in (big[:96, :7].t(), big[:, 8:72], big[3:9, 1:33], big[::3, 4:100], big[:1, :64].expand(5, 64)):
        for dtype in TYPES:
            check(x.to(dtype) if dtype != torch.float32 else x)
    half = big.half()
    check(half[:, 8:72])
    check(half[2:5, 3:35])
    q = ops.mx4_quantize(big[:, 8:72])
    wide = ops.Mx4(torch.zeros((130, 40), dtype=torch.uint8, device=DEV), torch.zeros((130, 3), dtype=torch.uint8, device=DEV))
    wide.codes[:, 3:35], wide.scales[:, 1:] = q.codes, q.scales
    got = ops.mx4_dequantize(ops.Mx4(wide.codes[:, 3:35], wide.scales[:, 1:]))
    assert torch.equal(got, ops.mx4_dequantize(q))


@pytest.mark.parametrize("shape", [(8, 32), (40, 96), (64, 128), (2560, 544), (3, 24, 160), (5, 64, 1056)])
def test_repack_there_and_back(shape):
    g = torch.Generator().manual_seed(1)
    q = ops.Mx4(torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), generator=g).to(torch.uint8).to(DEV),
                torch.randint(0, 256, shape[:-1] + (shape[-1] // 32,), generator=g).to(torch.uint8).to(DEV))
    w = ops.mx4_repack(q)
    assert (w.w.shape[-1], w.s.shape[-1]) == ops.mx4_weight_bytes(*shape[-2:])
    back = ops.mx4_unrepack(w)
    assert torch.equal(back.codes, q.codes) and torch.equal(back.scales, q.scales)
    if len(shape) == 3:
        one = ops.mx4_repack(ops.Mx4(q.codes[1], q.scales[1]))
        assert torch.equal(w.expert(1).w, one.w) and torch.equal(w.expert(1).s, one.s)


def test_captured_and_on_another_stream():
    x = torch.randn((40, 160), device=DEV, dtype=torch.bfloat16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops.mx4_dequantize(ops.mx4_quantize(x))
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, ops.mx4_dequantize(ops.mx4_quantize(x)))
    with torch.cuda.graph(graph):
        out = ops.mx4_dequantize(ops.mx4_quantize(x))
    for seed in range(3):
        x.copy_(torch.randn((40, 160), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.mx4_dequantize(ops.mx4_quantize(x)))
