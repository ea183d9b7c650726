"""The registered AWQ ops called by themselves: what the kernels read or write is checked ahead of a launch.  Without
a GPU the checks alone, on tensors of the host."""
import pytest
import torch

from sglite_amd import ops

OPS, H, I32, I64 = torch.ops.sglite_awq, torch.float16, torch.int32, torch.int64
M, N, K, G = 5, 64, 256, 128


def repacked(empty):
    NT, NG = (N + 15) // 16, K // G
    return dict(w=empty(NT * ((K + 127) // 128) * 256, dtype=I32), s=empty(NT, NG, 16), z=empty(NT, NG, dtype=I64))


OTHER = {"cpu": "meta", "cuda": "cpu"}  # another device than the kernels'


def zeros(dev):
    return lambda *shape, dtype=H, device=dev: torch.zeros(shape, dtype=dtype, device=device)


def bad_weights(ok, empty, other):
    return [dict(w=ok["w"][:-4]), dict(w=ok["w"].long()), dict(w=empty(2 * ok["w"].numel(), dtype=I32)[::2]),
            dict(s=ok["s"][:-1]), dict(s=ok["s"].double()), dict(z=ok["z"][:-1]), dict(z=ok["z"].int()),
            dict(N=2 * N), dict(K=2 * K), dict(G=64), dict(G=0), dict(G=48), dict(K=0), dict(N=0),
            dict(z=ok["z"].to(other))]


def linear(name, dev):
    empty, other = zeros(dev), OTHER[dev]
    ok = dict(repacked(empty), K=K, N=N, G=G)
    bad = bad_weights(ok, empty, other)
    if name in ("awq_unrepack_cdna4", "awq_dequant_repacked"):
        return ok, bad
    ok.update(x=empty(M, K), bias=empty(N), counters=ops.make_counters(N, torch.device(dev)))
    bad += [dict(x=empty(M, K - 8)), dict(x=empty(K)), dict(x=empty(M, K, dtype=torch.bfloat16)), dict(bias=empty(N - 8)),
            dict(bias=empty(N, dtype=torch.float32)), dict(bias=empty(N, device=other)),
            dict(counters=ok["counters"].long()), dict(counters=ok["counters"][::2]),
            dict(counters=ok["counters"].to(other))]
    cols = N
    if "act" in name:
        ok["activation"] = "silu"
        bad.append(dict(activation="relu"))
        cols = N // 2
    if name.endswith("out"):
        ok["out"] = empty(M, cols)
        bad += [dict(out=empty(M - 1, cols)), dict(out=empty(M, cols + 8)), dict(out=empty(M, 2 * cols)[:, ::2]),
                dict(out=empty(cols, M).t()), dict(out=empty(M, cols, dtype=torch.float32)),
                dict(out=empty(M, cols, device=other))]
    return ok, bad


LINEAR = ["awq_unrepack_cdna4", "awq_dequant_repacked", "awq_w4a16_gemm", "awq_w4a16_gemm_out", "awq_w4a16_gemm_act",
          "awq_w4a16_gemm_act_out"]


def check_linear(name, a):
    """What the op's body checks."""
    if "gemm" not in name:
        return ops._check_repacked(**a)
    a = {"out": None, "activation": None, **a}
    return ops._check_gemm_op(**a)


@pytest.mark.parametrize("name", LINEAR)
def test_linear_checks(name):
    ok, bad = linear(name, "cpu")
    check_linear(name, ok)
    for change in bad:
        with pytest.raises(ValueError):
            check_linear(name, {**ok, **change})


def test_checkpoint_tensors_lie_on_one_device():
    q, z, s = torch.zeros(K, N // 8, dtype=I32), torch.zeros(K // G, N // 8, dtype=I32), torch.ones(K // G, N).half()
    ops._check_awq_shapes(q, z, s)
    for bad in ((q, z.to("meta"), s), (q, z, s.to("meta"))):
        with pytest.raises(ValueError, match="one device"):
            ops._check_awq_shapes(*bad)


def refused_by_the_op(name, ok, bad):
    getattr(OPS, name)(**ok)
    for change in bad:
        with pytest.raises(ValueError):
            getattr(OPS, name)(**{**ok, **change})
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("name", LINEAR)
def test_linear_ops(name):
    refused_by_the_op(name, *linear(name, "cuda"))


@pytest.mark.gpu
def test_strided_and_odd_operands_are_copied():
    from oracle import awq_oracle as oracle

    t = oracle.make_awq_linear(K, N, G, seed=1)
    r = ops.repack(*(t[k].to("cuda") for k in ("qweight", "qzeros", "scales")))
    cnt = ops.make_counters(N, torch.device("cuda"))
    x, bias = torch.randn((M, K), device="cuda").half(), torch.randn(N, device="cuda").half()
    want = ops.gemm(x, r, K, N, G, bias=bias, counters=cnt)
    wide = torch.zeros((M, K + 40), device="cuda").half()
    wide[:, 8:K + 8] = x
    odd = torch.cat((bias[:1], bias))[1:]
    assert torch.equal(OPS.awq_w4a16_gemm(wide[:, 8:K + 8], r.w, r.s, r.z, odd, cnt, K, N, G), want)
    out = torch.full((M, N), 7.0, dtype=H, device="cuda")
    assert ops.gemm(x, r, K, N, G, bias=bias, counters=cnt, out=out) is out and torch.equal(out, want)
    OPS.awq_w4a16_gemm_out(x.t().contiguous().t(), r.w, r.s, r.z, bias, cnt, out.zero_(), K, N, G)
    assert torch.equal(out, want) and ops.counters_settled(cnt)
