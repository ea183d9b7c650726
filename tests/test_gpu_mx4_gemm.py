"""MXFP4 products against the formula in 64 bits."""
import pytest
import torch

from oracle import mx4_oracle as oracle
from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type


def make(M, N, K, dtype, seed=0, E=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((M, K), generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))).to(dtype).to(DEV)
    shape = (N, K) if E is None else (E, N, K)
    codes, scales = oracle.quantize(torch.randn(shape, generator=g).to(DEV) / K ** 0.5)
    return x, codes, scales, ops.mx4_repack(ops.Mx4(codes, scales))


def close(got, want, err):
    tol = err + HALF[got.dtype] * (want.abs() + err) + 2.0 ** -25
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float(((got.double() - want).abs() - tol).max()):.3e}"


def check(M, N, K, dtype, act=None, biased=False, seed=0):
    x, codes, scales, w = make(M, N, K, dtype, seed)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(7)).to(dtype).to(DEV) if biased else None
    got = ops.mx4_gemm(x, w, bias=bias, activation=act)
    y, err = oracle.product(oracle.quantized(x), oracle.values(codes, scales), bias)
    assert got.shape == (M, N if act is None else N // 2) and got.dtype == dtype
    close(got, *((y, err) if act is None else oracle.gated(y, err, act)))


SHAPES = [
    # M, N, K
    (1, 8, 32), (1, 2560, 4096), (2, 40, 96), (5, 64, 544), (16, 2560, 9728), (16, 200, 160), (17, 64, 128),
    (24, 256, 2560), (33, 1000, 672), (48, 96, 1056), (64, 512, 2048), (65, 64, 512), (100, 72, 224), (128, 6144, 512),
    (130, 8, 2560), (200, 640, 64), (257, 1536, 1024), (333, 320, 9728), (1000, 768, 640), (2049, 1280, 288),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, dtype):
    check(M, N, K, dtype)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 64, 32), (3, 19456, 2560), (16, 128, 4096), (31, 448, 96), (64, 1024, 512),
                                   (150, 192, 1120), (300, 2816, 256), (1111, 640, 384)])
def test_gated(M, N, K, dtype, act):
    check(M, N, K, dtype, act)


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("M", [1, 9, 40, 100, 700])
def test_bias(M, act):
    check(M, 320, 256, torch.bfloat16, act, biased=True)
    check(M, 1280, 1056, torch.float16, act, biased=True)


@pytest.mark.parametrize("M,N,K,act", [
    (2048, 8192, 160, None), (2305, 7432, 672, None), (9000, 2056, 96, None), (2600, 6144, 1024, None),
    (2500, 8256, 352, "silu"), (4097, 5184, 128, "gelu"), (2048, 8192, 1152, "silu")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large(M, N, K, act, dtype):
    check(M, N, K, dtype, act, biased=True)


@pytest.mark.parametrize("M", [1, 16, 17, 64, 200, 1500])
def test_rows_that_are_not_finite(M):
    x, codes, scales, w = make(M, 96, 352, torch.bfloat16)
    x[0, 0], x[M // 2, 351] = float("inf"), float("nan")
    y = ops.mx4_gemm(x, w)
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    bad[0] = bad[M // 2] = True
    assert torch.equal(torch.isnan(y).all(-1), bad) and torch.equal(torch.isnan(y).any(-1), bad)


@pytest.mark.parametrize("M", [1, 16, 64, 300])
def test_weights_that_are_nan_and_scales_at_the_ends(M):
    x, codes, scales, _ = make(M, 64, 256, torch.float16)
    scales[3, 2] = 255
    y = ops.mx4_gemm(x, ops.mx4_repack(ops.Mx4(codes, scales)))
    assert torch.isnan(y[:, 3]).all() and torch.isnan(y).sum() == M
    scales.fill_(0)  # 2^-127: far below what fp16 holds
    assert (ops.mx4_gemm(x, ops.mx4_repack(ops.Mx4(codes, scales))) == 0).all()
    scales.fill_(127 + 9)
    xs = (x * 2.0 ** -12).half()
    got = ops.mx4_gemm(xs, ops.mx4_repack(ops.Mx4(codes, scales)))
    close(got, *oracle.product(oracle.quantized(xs), oracle.values(codes, scales)))


@pytest.mark.parametrize("M", [0, 1, 70])
def test_zero_and_no_rows(M):
    _, _, _, w = make(1, 64, 96, torch.float16)
    x = torch.zeros((M, 96), dtype=torch.float16, device=DEV)
    bias = torch.arange(64, device=DEV)
    assert (ops.mx4_gemm(x, w) == 0).all() and ops.mx4_gemm(x, w).shape == (M, 64)
    assert torch.equal(ops.mx4_gemm(x, w, bias=bias), bias.half().expand(M, 64))


@pytest.mark.parametrize("M", [4, 40, 400])
def test_views_out_and_rows_alone(M):
    x, codes, scales, w = make(M, 96, 160, torch.bfloat16)
    want = ops.mx4_gemm(x, w)
    wide = torch.full((M, 200), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:168] = x
    assert torch.equal(ops.mx4_gemm(wide[:, 8:168], w), want)
    assert torch.equal(ops.mx4_gemm(x.t().contiguous().t(), w), want)
    buf = torch.full((M + 2, 96), 7.0, dtype=torch.bfloat16, device=DEV)
    assert ops.mx4_gemm(x, w, out=buf[1:-1]).data_ptr() == buf[1:].data_ptr()
    assert torch.equal(buf[1:-1], want) and (buf[0] == 7).all() and (buf[-1] == 7).all()
    with pytest.raises(ValueError):
        ops.mx4_gemm(x, w, out=torch.empty((M, 192), dtype=torch.bfloat16, device=DEV)[:, ::2])
    square, _, _, sw = make(M, 160, 160, torch.bfloat16)
    with pytest.raises(ValueError, match="share memory"):
        ops.mx4_gemm(square, sw, out=square)


@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_captured_replays_with_eager_work_between(M):
    x, codes, scales, w = make(M, 640, 1056, torch.float16)
    bias = torch.randn(640, device=DEV).half()
    ops.mx4_gemm(x, w)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx4_gemm(x, w, bias=bias, activation="silu")
    with torch.cuda.graph(other):
        out2 = ops.mx4_gemm(x, w)
    for seed in range(4):
        x.copy_(make(M, 8, 1056, torch.float16, seed)[0])
        ops.mx4_gemm(torch.randn((200, 1056), device=DEV).half(), w)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.mx4_gemm(x, w, bias=bias, activation="silu"))
        assert torch.equal(out2, ops.mx4_gemm(x, w))


def test_two_streams_at_once():
    pairs = [make(300, 1280, 2048, torch.float16, seed) for seed in range(2)]
    want = [ops.mx4_gemm(p[0], p[3]) for p in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (p, s) in enumerate(zip(pairs, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.mx4_gemm(p[0], p[3]))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


def test_threads_on_one_stream():
    """The quantised rows of a call lie in its thread's own workspace."""
    import threading

    pairs = [make(300, 640, 1024, torch.float16, seed) for seed in range(4)]
    want, bad = [ops.mx4_gemm(p[0], p[3]) for p in pairs], []

    def work(i):
        for _ in range(30):
            y = ops.mx4_gemm(pairs[i][0], pairs[i][3])
        torch.cuda.synchronize()
        if not torch.equal(y, want[i]):
            bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_offsets_past_31_bits():
    """A weight of more than 2 GiB, and an output of more than 2^32 bytes."""
    N, K = 65536, 69632
    g = torch.Generator(device=DEV).manual_seed(0)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(118, 122, (N, K // 32), generator=g, device=DEV, dtype=torch.uint8)
    w = ops.mx4_repack(ops.Mx4(codes, scales))
    cols = torch.tensor([0, 77, 40000, N - 1], device=DEV)
    values = oracle.values(codes[cols], scales[cols])
    back = ops.mx4_unrepack(w)
    assert torch.equal(back.codes[cols], codes[cols]) and torch.equal(back.scales[cols], scales[cols])
    del back, codes
    for M in (2, 70, 300):
        x = torch.randn((M, K), generator=g, device=DEV).bfloat16()
        close(ops.mx4_gemm(x, w)[:, cols], *oracle.product(oracle.quantized(x), values))
    del w
    M, N, K = 70000, 32768, 64
    x = torch.randn((M, K), generator=g, device=DEV).half()
    q = ops.mx4_quantize(torch.randn((N, K), generator=g, device=DEV))
    y = ops.mx4_gemm(x, ops.mx4_repack(q))
    rows = torch.tensor([0, 1, 40001, 65535, 65536, M - 1], device=DEV)
    close(y[rows], *oracle.product(oracle.quantized(x[rows]), oracle.values(*q)))


def test_compiled():
    x, codes, scales, w = make(20, 128, 96, torch.bfloat16)

    def op(v):
        return torch.ops.sglite_awq.awq_mx4_gemm(v, w.w, w.s, None, 128, 96, "none") * 2.0
    assert torch.equal(torch.compile(op, backend="aot_eager", fullgraph=True)(x), ops.mx4_gemm(x, w) * 2.0)
    assert torch.equal(torch.compile(lambda v: ops.mx4_gemm(v, w) * 2.0, backend="aot_eager")(x), ops.mx4_gemm(x, w) * 2.0)


def test_ops_called_by_themselves_check_too():
    x, codes, scales, w = make(20, 128, 96, torch.bfloat16)
    op = torch.ops.sglite_awq.awq_mx4_gemm
    wide = torch.zeros((20, 200), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:104] = x
    assert torch.equal(op(wide[:, 8:104], w.w, w.s, None, 128, 96, "none"), ops.mx4_gemm(x, w))
    for bad in ((x[:, :64], w.w, w.s, None, 128, 96, "none"), (x, w.w[:-16], w.s, None, 128, 96, "none"),
                (x, w.w, w.s, None, 160, 96, "none"), (x.float(), w.w, w.s, None, 128, 96, "none")):
        with pytest.raises(ValueError):
            op(*bad)


def test_registered_ops_meet_the_direct_calls():
    x, codes, scales, w = make(20, 128, 96, torch.bfloat16)
    y = torch.ops.sglite_awq.awq_mx4_gemm(x, w.w, w.s, None, 128, 96, "silu")
    assert torch.equal(y, ops.mx4_gemm(x, w, activation="silu"))
    q = torch.ops.sglite_awq.awq_mx4_quantize(x)
    assert all(torch.equal(a, b) for a, b in zip(q, ops.mx4_quantize(x)))
    assert torch.equal(torch.ops.sglite_awq.awq_mx4_dequantize(*q, torch.float32), ops.mx4_dequantize(ops.Mx4(*q), torch.float32))
