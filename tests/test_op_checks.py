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


def on_lines(t):
    """The same counters at a multiple of 128 bytes, which the host's allocator does not promise."""
    big = torch.zeros(t.numel() + 32, dtype=t.dtype, device=t.device)
    at = -big.data_ptr() % 128 // 4
    return big[at:at + t.numel()]


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
    ok.update(x=empty(M, K), bias=empty(N), counters=on_lines(ops.make_counters(N, torch.device(dev))))
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


E, TOP_K, ROWS = 4, 2, 2 * M


def routed(dev, cols):
    empty = zeros(dev)
    return dict(a=empty(M, K), sorted_ids=torch.full((ROWS + 15 * E,), ROWS, dtype=I32, device=dev),
                expert_offsets=empty(E + 1, dtype=I32), topk_weights=empty(ROWS, dtype=torch.float32),
                out=empty(ROWS, cols), num_routed=ROWS, top_k=TOP_K, activation="none", mul_routed_weight=True)


def bad_routed(ok, dev, cols):
    empty, other, ids, offsets = zeros(dev), OTHER[dev], ok["sorted_ids"], ok["expert_offsets"]
    return [dict(a=empty(M, K - 8)), dict(a=empty(K)), dict(a=empty(M, K, dtype=torch.bfloat16)),
            dict(sorted_ids=ids.long()), dict(sorted_ids=ids.repeat(2)[::2]), dict(sorted_ids=ids.to(other)),
            dict(expert_offsets=offsets[:-1]), dict(expert_offsets=empty(E + 2, dtype=I32)),
            dict(expert_offsets=offsets.long()), dict(expert_offsets=offsets.to(other)), dict(topk_weights=None),
            dict(topk_weights=ok["topk_weights"][:-1]), dict(topk_weights=empty(ROWS)),
            dict(topk_weights=ok["topk_weights"].to(other)), dict(out=empty(ROWS - 1, cols)), dict(out=empty(ROWS, cols + 8)),
            dict(out=empty(ROWS, 2 * cols)[:, ::2]), dict(out=empty(ROWS, cols, dtype=torch.float32)),
            dict(out=ok["out"].to(other)), dict(activation="silu"), dict(activation="relu"), dict(num_routed=-1),
            dict(num_routed=ROWS + 1), dict(top_k=0)]


def grouped(name, dev):
    empty, other = zeros(dev), OTHER[dev]
    ok = routed(dev, N)
    bad = bad_routed(ok, dev, N)
    if name == "awq_moe_dense_gemm":
        w = empty(E, N, K)
        ok["w"] = w
        return ok, bad + [dict(w=w[0]), dict(w=w[:, :, :-8]), dict(w=empty(E, K, N).transpose(1, 2)), dict(w=w.bfloat16()),
                          dict(w=empty(E + 1, N, K)), dict(w=empty(E, N + 8, K)), dict(w=w.to(other))]
    ws, ss, zs = ops.expert_strides(K, N, G)
    ok.update(w=empty(E, ws // 4, dtype=I32), s=empty(E, ss // 2), z=empty(E, zs // 8, dtype=I64), K=K, N=N, G=G)
    return ok, bad + [dict(w=ok["w"][:-1]), dict(w=ok["w"].long()), dict(w=ok["w"][0]), dict(s=ok["s"][:, :-8]),
                      dict(s=ok["s"].bfloat16()), dict(s=ok["s"][:-1]), dict(z=ok["z"][:, :-1]), dict(z=ok["z"].int()),
                      dict(z=ok["z"].to(other)), dict(N=2 * N), dict(K=2 * K), dict(G=64), dict(G=48), dict(K=0),
                      dict(N=0), dict(G=0)]


GROUPED = {"awq_moe_w4a16_gemm": ops._check_moe_gemm_op, "awq_moe_dense_gemm": ops._check_moe_dense_op}


@pytest.mark.parametrize("name", GROUPED)
def test_grouped_checks(name):
    ok, bad = grouped(name, "cpu")
    GROUPED[name](**ok)
    for change in bad:
        with pytest.raises(ValueError):
            GROUPED[name](**{**ok, **change})


def test_sum_and_stack_checks():
    one, out = torch.zeros(M, 2, 64).half(), torch.zeros(M, 64).half()
    ops._check_moe_sum(one, out)
    for bad in ((one[0], out), (one, out[:-1]), (one, out[:, :32]), (one, out.float()), (one[:, :, ::2], out[:, ::2]),
                (one, out.to("meta"))):
        with pytest.raises(ValueError):
            ops._check_moe_sum(*bad)
    q, z, s = torch.zeros(E, K, N // 8, dtype=I32), torch.zeros(E, K // G, N // 8, dtype=I32), torch.ones(E, K // G, N).half()
    assert ops._check_expert_stacks(q, z, s) == (E, K, N, G)
    for bad in ((q[0], z[0], s[0]), (q, z[1:], s), (q, z, s[1:]), (q, z.to("meta"), s), (q, z, s[:, :1])):
        with pytest.raises(ValueError):
            ops._check_expert_stacks(*bad)


def mlp(dev, I=384):
    """The one-launch block's arguments, K being its hidden size."""
    empty, other = zeros(dev), OTHER[dev]

    def layout(k, n):
        return (empty((n + 15) // 16 * ((k + 127) // 128) * 256, dtype=I32), empty((n + 15) // 16, k // G, 16),
                empty((n + 15) // 16, k // G, dtype=I64))
    gate, down = layout(K, 2 * I), layout(I, K)
    ok = dict(x=empty(M, K), **dict(zip(("gw", "gs", "gz"), gate)), **dict(zip(("dw", "ds", "dz"), down)),
              counters=on_lines(ops.make_mlp_counters(torch.device(dev))), out=empty(M, K), H=K, I=I, G=G, activation="silu")
    return ok, [{name: ok[name].reshape(-1)[:-1]} for name in ("gw", "gs", "gz", "dw", "ds", "dz")] + [
        dict(x=empty(M, K - 8)), dict(x=empty(M, K).bfloat16()), dict(gw=ok["gw"].long()), dict(dz=ok["dz"].int()),
        dict(dw=ok["dw"].to(other)), dict(counters=ok["counters"][:-32]), dict(counters=ok["counters"].long()),
        dict(counters=ok["counters"].to(other)), dict(out=empty(M - 1, K)), dict(out=empty(M, 2 * K)[:, ::2]),
        dict(out=empty(M, K).bfloat16()), dict(out=ok["out"].to(other)), dict(H=2 * K), dict(I=2 * I), dict(G=64),
        dict(activation="relu")]


def lora(dev, inplace, L=3, R=8):
    empty, other = zeros(dev), OTHER[dev]
    ok = dict(y=empty(M, N), x=empty(M, K), a=empty(L, 2 * R, K), b=empty(L, N, R), scaling=empty(L, dtype=torch.float32),
              ranks=empty(L, dtype=I32), adapter_ids=empty(M, dtype=I32), sorted_ids=None, block_adapters=None,
              parts=[N // 2, N // 2])
    tables = dict(sorted_ids=torch.full((M + 15 * (L + 1),), M, dtype=I32, device=dev),
                  block_adapters=torch.full((M // 16 + L + 2,), L, dtype=I32, device=dev))
    bad = [dict(y=empty(M, N - 8)), dict(y=empty(M - 1, N)), dict(x=empty(M, K - 8)), dict(x=empty(M, K).bfloat16()),
           dict(a=empty(L, 2 * R, K - 8)), dict(a=empty(L - 1, 2 * R, K)), dict(b=empty(L, N, 2 * R)), dict(b=empty()),
           dict(a=ok["a"].to(other)), dict(scaling=empty(L)), dict(scaling=empty(L - 1, dtype=torch.float32)),
           dict(ranks=ok["ranks"].long()), dict(ranks=ok["ranks"][:-1]), dict(adapter_ids=ok["adapter_ids"][:-1]),
           dict(adapter_ids=ok["adapter_ids"].long()), dict(adapter_ids=ok["adapter_ids"].to(other)),
           dict(sorted_ids=tables["sorted_ids"]), {**tables, "sorted_ids": tables["sorted_ids"][:-1]},
           {**tables, "block_adapters": tables["block_adapters"][:1]}, dict(parts=[N]), dict(parts=[N // 2, N // 2 - 8])]
    if inplace:
        return ok, bad + [dict(y=empty(M, 2 * N)[:, ::2])]
    return dict(ok, activation="none"), bad + [dict(activation="relu"), dict(parts=[N - 8, 8], activation="silu")]


def test_mlp_checks():
    ok, bad = mlp("cpu")
    ops._check_mlp_op(**ok)
    for change in bad:
        with pytest.raises(ValueError):
            ops._check_mlp_op(**{**ok, **change})


def test_lora_checks(monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    ok, bad = lora("cpu", False)
    ops._check_lora_op(**ok)
    for change in bad:
        with pytest.raises(ValueError):
            ops._check_lora_op(**{**ok, **change})
    for ids, n in ((torch.zeros(M, dtype=I64), 3), (torch.zeros(M, 1, dtype=I32), 3), (torch.zeros(M, dtype=I32), 0)):
        with pytest.raises(ValueError):
            ops._check_lora_ids(ids, n)


def refused_by_the_op(name, ok, bad):
    getattr(OPS, name)(**ok)
    for change in bad:
        with pytest.raises(ValueError):
            getattr(OPS, name)(**{**ok, **change})
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("name", GROUPED)
def test_grouped_ops(name):
    refused_by_the_op(name, *grouped(name, "cuda"))


@pytest.mark.gpu
def test_mlp_op():
    ok, bad = mlp("cuda", 128)
    if ops.gated_mlp_plan(M, K, 128, G) is None:  # then the C ABI refuses the shape, after the checks
        with pytest.raises(RuntimeError):
            OPS.awq_gated_mlp_out(**ok, polls=-1)
    else:
        OPS.awq_gated_mlp_out(**ok, polls=-1)
    for change in bad:
        with pytest.raises(ValueError):
            OPS.awq_gated_mlp_out(**{**ok, **change}, polls=-1)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_lora_ops():
    refused_by_the_op("awq_lora_add", *lora("cuda", False))
    refused_by_the_op("awq_lora_add_", *lora("cuda", True))
    for ids, n in ((torch.zeros(M, dtype=I64), 3), (torch.zeros(M, 1, dtype=I32), 3), (torch.zeros(M, dtype=I32), 0)):
        with pytest.raises(ValueError):
            OPS.awq_lora_route(ids.cuda(), n)
    ids = torch.arange(40, dtype=I32, device="cuda") % 4 - 1
    want = ops.lora_route(ids, 3)
    got = OPS.awq_lora_route(ids.repeat_interleave(2)[::2], 3)  # a strided one is copied
    assert torch.equal(got[0], want.sorted_ids)


@pytest.mark.gpu
def test_other_moe_ops():
    one, out = torch.ones((M, 2, 64), device="cuda").half(), torch.zeros((M, 64), device="cuda").half()
    OPS.awq_moe_sum_reduce(one, out)
    assert (out == 2).all()
    with pytest.raises(ValueError):
        OPS.awq_moe_sum_reduce(one, out[:-1])
    with pytest.raises(ValueError, match="int32"):
        OPS.awq_moe_align_block_size(torch.zeros((M, 2), dtype=I64, device="cuda"), 16, E)


@pytest.mark.gpu
def test_moe_gemm_checks_its_alignment():
    """The Python call too: an alignment for other experts or of another type is refused."""
    ok, _ = grouped("awq_moe_w4a16_gemm", "cuda")
    ex = ops.RepackedExperts(ok["w"], ok["s"], ok["z"], K, N, G)
    al = ops.moe_align_block_size(torch.zeros((M, TOP_K), dtype=I32, device="cuda"), 16, E)

    def call(align, n=N):
        return ops.moe_gemm(ok["a"], ex, K, n, G, align, ok["topk_weights"], ROWS, TOP_K)
    assert call(al).shape == (ROWS, N)
    for bad in (al._replace(expert_offsets=al.expert_offsets[:-1]), al._replace(sorted_ids=al.sorted_ids.long())):
        with pytest.raises(ValueError):
            call(bad)
    with pytest.raises(ValueError):
        call(al, 2 * N)


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
