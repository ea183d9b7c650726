"""Which expert weights each MoE backend and layer takes (no GPU: every call is refused ahead of a launch)."""
import pytest
import torch

from sglite_amd import ops
from sglite_amd.moe import AWQFusedMoe, AWQMoeWeights, FusedMoe, create_moe_backend, fused_experts_impl

E, H, I, T = 4, 64, 48, 3


def dense():
    return torch.zeros(E, 2 * I, H).half(), torch.zeros(E, H, I).half()


def awq():
    def stack(K, N):
        return AWQMoeWeights(ops.RepackedExperts(*(torch.zeros(E, 1) for _ in ops.RepackedExperts._fields)), K, N, 32)
    return stack(H, 2 * I), stack(I, H)


def call(f, w1, w2):
    x, logits = torch.zeros(T, H).half(), torch.zeros(T, E)
    if f is fused_experts_impl:
        return f(x, w1, w2, torch.zeros(T, 2), torch.zeros(T, 2, dtype=torch.int32))
    return f.forward(x, w1, w2, logits, 2, True)


def test_backends_refuse_the_other_kind_and_mixed_pairs():
    (d1, d2), (a1, a2) = dense(), awq()
    for pair in ((d1, d2), (d1, a2), (a1, d2)):
        with pytest.raises(ValueError, match="awq_fused"):
            call(create_moe_backend("awq_fused"), *pair)
    for pair in ((a1, a2), (d1, a2), (a1, d2)):
        with pytest.raises(ValueError, match="dense"):
            call(create_moe_backend("fused"), *pair)
    for pair in ((d1, a2), (a1, d2)):
        with pytest.raises(ValueError, match="both"):
            call(fused_experts_impl, *pair)
    assert not issubclass(FusedMoe, AWQFusedMoe)
    # Their own kind goes on to the kernels, which need device tensors.
    for f, pair in (("awq_fused", (a1, a2)), ("fused", (d1, d2))):
        with pytest.raises(ValueError, match="device tensors"):
            call(create_moe_backend(f), *pair)
    with pytest.raises(ValueError, match="device tensors"):
        call(fused_experts_impl, d1, d2)
