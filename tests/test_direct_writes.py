"""An output that a direct launch writes counts as written, as one that a registered op writes: a backward pass that
saved it is refused and not wrong.  Without a GPU the launches are left out."""
import pytest
import torch

from sglite_amd import ops
from tests.test_op_checks import on_lines

M, K, N, E = 4, 256, 128, 3
H, I32 = torch.float16, torch.int32


def calls(dev):
    """Each call that writes a tensor of the caller's, as (name, function of the output, its shape)."""
    def zeros(*shape, dtype=H):
        return torch.zeros(shape, dtype=dtype, device=dev)

    def repacked(k, n):
        return ops.Repacked(zeros(n // 16 * (k // 128) * 256, dtype=I32), zeros(n // 16, k // 128, 16),
                            zeros(n // 16, k // 128, dtype=torch.int64))
    x, r, cnt = zeros(M, K), repacked(K, N), on_lines(ops.make_counters(N, torch.device(dev)))
    align = ops.MoeAlignment(torch.full((M + 15 * E,), M, dtype=I32, device=dev), zeros(1, dtype=I32), zeros(1, dtype=I32),
                             zeros(E + 1, dtype=I32))
    ws, ss, zs = ops.expert_strides(K, N, 128)
    ex = ops.RepackedExperts(zeros(E, ws // 4, dtype=I32), zeros(E, ss // 2), zeros(E, zs // 8, dtype=torch.int64), K, N, 128)
    wb, sb = ops.mx4_weight_bytes(N, K)
    w4, w4e = (ops.Mx4Weight(zeros(*lead, wb, dtype=torch.uint8), zeros(*lead, sb, dtype=torch.uint8), N, K)
               for lead in ((), (E,)))
    stack = ops.make_lora_stack(2, 8, K, (N,), H, torch.device(dev))
    batch = ops.LoraBatch(zeros(M, dtype=I32), None, None, 2)
    yield "gemm", lambda o: ops.gemm(x, r, K, N, 128, counters=cnt, out=o), (M, N)
    yield "moe_gemm", lambda o: ops.moe_gemm(x, ex, K, N, 128, align, None, M, 1, out=o), (M, N)
    yield "moe_dense_gemm", lambda o: ops.moe_dense_gemm(x, zeros(E, N, K), align, None, M, 1, out=o), (M, N)
    yield "moe_sum_reduce", lambda o: ops.moe_sum_reduce(zeros(M, 2, N), o), (M, N)
    yield "mx4_gemm", lambda o: ops.mx4_gemm(x, w4, out=o), (M, N)
    yield "mx4_moe_gemm", lambda o: ops.mx4_moe_gemm(x, w4e, align, None, M, 1, out=o), (M, N)
    yield "lora_add", lambda o: ops.lora_add(o, x, stack, batch, out=o), (M, N)
    if dev == "cpu" or ops.gated_mlp_plan(M, K, N, 128) is not None:
        gate, down, mlp = repacked(K, 2 * N), repacked(N, K), on_lines(ops.make_mlp_counters(torch.device(dev)))
        yield "gated_mlp", lambda o: ops.gated_mlp(x, gate, down, K, N, 128, mlp, out=o), (M, K)


NAMES = ["gemm", "moe_gemm", "moe_dense_gemm", "moe_sum_reduce", "mx4_gemm", "mx4_moe_gemm", "lora_add", "gated_mlp"]


@pytest.mark.parametrize("name", NAMES)
def test_versions(name, monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    launched = []
    for launch in ("_gemm_launch", "_moe_gemm_launch", "_moe_dense_launch", "_moe_sum_launch", "_mx4_gemm_launch",
                   "_mx4_moe_launch", "_lora_launch", "_mlp_launch"):
        monkeypatch.setattr(ops, launch, lambda *a, launch=launch: launched.append(launch))
    fn, shape = {n: (f, s) for n, f, s in calls("cpu")}[name]
    out = torch.zeros(shape, dtype=H)
    before = out._version
    assert fn(out) is out and len(launched) == 1 and out._version > before


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_backward_pass_that_saved_it(name):
    found = {n: (f, s) for n, f, s in calls("cuda")}
    if name not in found:
        pytest.skip("no one-launch plan for this block")
    fn, shape = found[name]
    weight = torch.ones(shape[1], dtype=H, device="cuda", requires_grad=True)
    out = torch.ones(shape, dtype=H, device="cuda")
    y = (out * weight).sum()  # saves out for the weight's gradient
    fn(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
