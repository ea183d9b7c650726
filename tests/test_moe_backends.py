"""Which expert weights each MoE backend and layer takes (no GPU: every call is refused ahead of a launch)."""
import pytest
import torch

from sglite_amd import ops
from sglite_amd.moe import (SUPPORTED_MOE_BACKENDS, AWQFusedMoe, AWQMoELayer, AWQMoeWeights, BaseMoeBackend, FusedMoe,
                            MoELayer, create_moe_backend, fused_experts_impl)

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


def test_layers_refuse_the_other_kinds_backend_at_once():
    for layer, name, other in ((AWQMoELayer, "awq_fused", "fused"), (MoELayer, "fused", "awq_fused")):
        with pytest.raises(ValueError, match="backend"):
            layer(E, 2, 128, 128, backend=other)
        with pytest.raises(ValueError, match="unknown"):
            layer(E, 2, 128, 128, backend="none")
        assert layer(E, 2, 128, 128)._backend.__class__ is layer(E, 2, 128, 128, backend=name)._backend.__class__


def test_layers_take_a_backend_of_ones_own(monkeypatch):
    class Mine(BaseMoeBackend):
        def forward(self, hidden_states, **kw):
            return hidden_states

    monkeypatch.setitem(SUPPORTED_MOE_BACKENDS, "mine", Mine)
    for layer in (AWQMoELayer, MoELayer):
        assert isinstance(layer(E, 2, 128, 128, backend="mine")._backend, Mine)
