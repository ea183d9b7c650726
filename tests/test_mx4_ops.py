"""The registered MXFP4 ops called by themselves: everything that a kernel reads or writes is checked, in the bodies
and in the fake implementations alike."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from sglite_amd import ops

U8, I32, H = torch.uint8, torch.int32, torch.float16
OPS = torch.ops.sglite_awq
M, N, K, E = 20, 128, 96, 4


def good_and_bad(name, dev):
    """Arguments that an op takes, and changes to them that it must refuse."""
    def empty(*shape, dtype=H):
        return torch.zeros(shape, dtype=dtype, device=dev)
    wb, sb = ops._mx4_layout_bytes(N, K)
    w, s, x = empty(wb, dtype=U8), empty(sb, dtype=U8), empty(M, K)
    codes, scales = empty(N, K // 2, dtype=U8), empty(N, K // 32, dtype=U8)
    if name == "awq_mx4_quantize":
        return dict(x=x), [dict(x=empty(M, 48)), dict(x=empty(M, K, dtype=torch.int16)), dict(x=empty()),
                           dict(x=empty(M, 0))]
    if name == "awq_mx4_dequantize":
        return dict(codes=codes, scales=scales, dtype=H), [
            dict(scales=scales[:-1]), dict(scales=scales[:, :-1]), dict(codes=empty(N, K // 2, dtype=I32)),
            dict(scales=empty(N, K // 32, dtype=I32)), dict(dtype=torch.float64), dict(scales=scales.reshape(-1))]
    if name == "awq_mx4_repack":
        return dict(codes=codes, scales=scales), [
            dict(scales=scales[:-1]), dict(scales=scales[:, :-1]), dict(codes=empty(N, K // 2, dtype=torch.int8)),
            dict(codes=codes[0], scales=scales[0]),
            dict(codes=empty(1, 2, N, K // 2, dtype=U8), scales=empty(1, 2, N, K // 32, dtype=U8))]
    if name == "awq_mx4_unrepack":
        return dict(w=w, s=s, N=N, K=K), [dict(w=w[:-16]), dict(s=s[:-16]), dict(N=2 * N), dict(K=K + 512),
                                          dict(w=w.view(torch.int8)), dict(w=empty(2, wb, dtype=U8))]
    gemm = dict(x=x, w=w, s=s, bias=empty(N), N=N, K=K, activation="none")
    bad = [dict(x=x[:, :64]), dict(x=x[0]), dict(x=x.float()), dict(w=w[:-16]), dict(s=s[:-16]), dict(N=160), dict(K=64),
           dict(N=64), dict(bias=empty(N - 8)), dict(bias=empty(N + 8)), dict(bias=empty(N, dtype=torch.float32)),
           dict(bias=empty(N, dtype=torch.bfloat16)), dict(bias=torch.zeros(N, dtype=H, device="cpu")),
           dict(activation="relu")]
    if name == "awq_mx4_gemm":
        return gemm, bad
    if name == "awq_mx4_gemm_out":
        return dict(gemm, out=empty(M, N)), bad + [
            dict(out=empty(M - 1, N)), dict(out=empty(M, N // 2)), dict(out=empty(M, 2 * N)[:, ::2]),
            dict(out=empty(N, M).t()), dict(out=empty(M, N, dtype=torch.bfloat16)), dict(activation="silu"),
            dict(out=torch.zeros(M, N, dtype=H, device="cpu"))]
    n, k = 2 * M, 2
    moe = dict(a=x, w=empty(E, wb, dtype=U8), s=empty(E, sb, dtype=U8),
               sorted_ids=torch.full((n + 15 * E,), n, dtype=I32, device=dev), expert_offsets=empty(E + 1, dtype=I32),
               topk_weights=empty(n, dtype=torch.float32), out=empty(n, N), N=N, K=K, num_routed=n, top_k=k,
               activation="none", mul_routed_weight=True)
    return moe, [
        dict(a=x[:, :64]), dict(a=x.float()), dict(w=w), dict(w=empty(E + 1, wb, dtype=U8)), dict(N=160), dict(K=64),
        dict(sorted_ids=moe["sorted_ids"].long()), dict(sorted_ids=empty(2 * n, dtype=I32)[::2]),
        dict(sorted_ids=torch.full((n,), n, dtype=I32, device="cpu")), dict(expert_offsets=empty(E, dtype=I32)),
        dict(expert_offsets=empty(E + 2, dtype=I32)), dict(expert_offsets=empty(E + 1, dtype=torch.int64)),
        dict(expert_offsets=torch.zeros(E + 1, dtype=I32, device="cpu")), dict(topk_weights=None),
        dict(topk_weights=empty(n - 1, dtype=torch.float32)), dict(topk_weights=empty(n)),
        dict(topk_weights=torch.zeros(n, device="cpu")), dict(out=empty(n - 1, N)), dict(out=empty(n, N // 2)),
        dict(out=empty(n, 2 * N)[:, ::2]), dict(out=empty(n, N, dtype=torch.float32)), dict(activation="silu"),
        dict(out=torch.zeros(n, N, dtype=H, device="cpu")), dict(num_routed=-1), dict(num_routed=n + 1), dict(top_k=0),
        dict(activation="tanh")]


NAMES = [n for n in ops.REGISTERED_OPS if n.startswith("awq_mx4")]


def check_refusals(name, dev):
    ok, bad = good_and_bad(name, dev)
    getattr(OPS, name)(**ok)
    for change in bad:
        with pytest.raises(ValueError):
            getattr(OPS, name)(**{**ok, **change})


@pytest.mark.parametrize("name", NAMES)
def test_refusals_in_a_trace(name):
    with FakeTensorMode():
        check_refusals(name, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_refusals(name):
    check_refusals(name, "cuda")
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_overlaps_and_addresses():
    ok, _ = good_and_bad("awq_mx4_gemm_out", "cuda")
    square = torch.zeros((N, N), dtype=H, device="cuda")
    w = ops.mx4_repack(ops.mx4_quantize(square))
    with pytest.raises(ValueError, match="share memory"):
        OPS.awq_mx4_gemm_out(square, w.w, w.s, None, square, N, N, "none")
    odd = torch.zeros(M * N + 1, dtype=H, device="cuda")[1:].view(M, N)
    with pytest.raises(ValueError, match="aligned"):
        OPS.awq_mx4_gemm_out(**{**ok, "out": odd})
    bias = torch.randn(N + 1, device="cuda").half()[1:]  # an odd address and a strided one are copied
    x = torch.randn((M, N), device="cuda").half()
    want = ops.mx4_gemm(x, w, bias=bias)
    assert torch.equal(OPS.awq_mx4_gemm(x, w.w, w.s, bias, N, N, "none"), want)
    assert torch.equal(OPS.awq_mx4_gemm(x, w.w, w.s, bias.repeat_interleave(2)[::2], N, N, "none"), want)
