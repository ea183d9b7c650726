"""MXFP4 experts that cannot be loaded leave the caller's tensors, and the layer, as they are."""
import pytest
import torch

from sglite_amd import ops
from sglite_amd.moe import MXFP4MoELayer

E, H, I = 3, 64, 96


def state(serialized, prefix="l"):
    g = torch.Generator().manual_seed(0)
    layer = MXFP4MoELayer(E, 2, H, I, serialized=serialized)
    return layer, {k: torch.randint(0, 120, p.shape, generator=g).to(p.dtype)
                   for k, p in layer.state_dict(prefix=prefix).items()}


@pytest.mark.parametrize("serialized", [True, False])
def test_tensors_of_the_host(serialized):
    layer, sd = state(serialized)
    before = dict(sd)
    with pytest.raises(ValueError, match="device tensors"):
        layer.load_state_dict(sd, prefix="l")
    assert list(sd) == list(before) and all(sd[k] is v for k, v in before.items()) and layer._experts is None


def test_a_second_stack_that_fails(monkeypatch):
    """The first stack's layout is not kept beside the second's old one."""
    layer, sd = state(True)
    made = []

    def repack(q):
        if made:
            raise RuntimeError("out of memory")
        made.append(q)
        return ops.Mx4Weight(q.codes, q.scales, q.codes.shape[-2], q.codes.shape[-1] * 2)
    monkeypatch.setattr(ops, "mx4_repack", repack)
    layer._experts = old = (object(), object())
    with pytest.raises(RuntimeError, match="memory"):
        layer.load_state_dict(sd, prefix="l")
    assert len(sd) == 4 and layer._experts is old
    made.clear()
    monkeypatch.setattr(ops, "mx4_repack", lambda q: q)
    with pytest.raises(RuntimeError, match="Unexpected"):
        layer.load_state_dict({**sd, "more": torch.zeros(1)}, prefix="l")
    layer.load_state_dict(sd, prefix="l")
    assert not sd and layer._experts is not old
