"""Adapters beside a projection: slots, and every refusal ahead of a launch (no GPU)."""
import ctypes

import pytest
import torch

from sglite_amd import _lib, ops
from sglite_amd.linear import MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear
from sglite_amd.mlp import GatedMLP

CPU = torch.device("cpu")


def test_slots_hold_the_merged_projections_adapters():
    qkv = QKVParallelLinear(64, 8, 4, 2, False, tp_size=2)  # local q 16, k 8, v 8
    assert qkv._parts == (16, 8, 8)
    qkv.add_adapters(3, 11, torch.float16, CPU)
    st = qkv._lora
    assert st.a.shape == (3, 3 * 16, 64) and st.b.shape == (3, 32, 16) and st.parts == (16, 8, 8)
    keys = qkv.state_dict_keys("qkv")
    g = torch.Generator().manual_seed(0)
    aq, av = torch.randn((11, 64), generator=g), torch.randn((5, 64), generator=g)
    bq, bv = torch.randn((16, 11), generator=g), torch.randn((8, 5), generator=g)
    qkv.load_adapter(1, [aq, None, av], [bq, None, bv], 0.5)
    assert st.ranks.tolist() == [0, 11, 0] and st.scaling.tolist() == [0.0, 0.5, 0.0]
    assert torch.equal(st.a[1, :11], aq.half()) and torch.equal(st.a[1, 32:37], av.half())
    assert not st.a[1, 11:32].any() and not st.a[1, 37:].any() and not st.a[0].any() and not st.a[2].any()
    assert torch.equal(st.b[1, :16, :11], bq.half()) and torch.equal(st.b[1, 24:, :5], bv.half())
    assert not st.b[1, 16:24].any() and not st.b[1, 24:, 5:].any()
    # A smaller adapter leaves nothing of the one before; nothing shows in the state dict.
    qkv.load_adapter(1, [aq[:2], None, None], [bq[:, :2], None, None])
    assert st.ranks.tolist() == [0, 2, 0] and not st.a[1, 2:].any() and not st.b[1, 16:].any()
    qkv.clear_adapter(1)
    assert not st.a.any() and not st.b.any() and not st.ranks.any()
    assert qkv.state_dict_keys("qkv") == keys


def test_slot_refusals_change_nothing():
    o = RowParallelLinear(64, 32, False)
    with pytest.raises(RuntimeError, match="add_adapters"):
        o.load_adapter(0, torch.zeros(4, 64), torch.zeros(32, 4))
    for bad in (dict(num_adapters=0, max_rank=8), dict(num_adapters=512, max_rank=8),
                dict(num_adapters=2, max_rank=0), dict(num_adapters=2, max_rank=257)):
        with pytest.raises(ValueError):
            o.add_adapters(dtype=torch.float16, device=CPU, **bad)
    with pytest.raises(ValueError):
        o.add_adapters(2, 8, torch.float32, CPU)
    o.add_adapters(2, 8, torch.bfloat16, CPU)
    o.load_adapter(0, torch.ones(4, 64), torch.ones(32, 4))
    before = [t.clone() for t in o._lora[:4]]
    for a, b in ((torch.zeros(9, 64), torch.zeros(32, 9)), (torch.zeros(4, 63), torch.zeros(32, 4)),
                 (torch.zeros(4, 64), torch.zeros(32, 5)), (torch.zeros(4, 64), None), (None, torch.zeros(32, 4)),
                 ([torch.zeros(4, 64)] * 2, [torch.zeros(32, 4)] * 2), (torch.zeros(0, 64), torch.zeros(32, 0))):
        with pytest.raises(ValueError):
            o.load_adapter(0, a if a is not None else [None], b if b is not None else [None])
    for slot in (-1, 2):
        with pytest.raises(ValueError, match="slot"):
            o.load_adapter(slot, torch.zeros(4, 64), torch.zeros(32, 4))
        with pytest.raises(ValueError, match="slot"):
            o.clear_adapter(slot)
    assert all(torch.equal(p, q) for p, q in zip(before, o._lora[:4]))


def test_layers_without_slots_take_a_batch_and_ignore_it():
    batch = ops.LoraBatch(torch.zeros(5, dtype=torch.int32), None, None, 2)
    g = torch.Generator().manual_seed(1)
    o = RowParallelLinear(16, 8, False)
    o.load_state_dict({"weight": torch.randn((8, 16), generator=g)})
    x = torch.randn((5, 16), generator=g)
    assert torch.equal(o(x, batch), o(x))
    mlp = GatedMLP(16, 24)
    mlp.load_state_dict({"gate_up_proj.weight": torch.randn((48, 16), generator=g),
                         "down_proj.weight": torch.randn((16, 24), generator=g)})
    assert torch.equal(mlp(x, batch), mlp(x))
    assert MergedColumnParallelLinear(16, [24, 8], False)._parts == (24, 8)


def _stack(L=3, P=2, R=16, K=64, N=48, dtype=torch.float16):
    return ops.LoraStack(torch.zeros(L, P * R, K, dtype=dtype), torch.zeros(L, N, R, dtype=dtype), torch.zeros(L),
                         torch.zeros(L, dtype=torch.int32), (N // P,) * P)


def _batch(M=4, L=3):
    return ops.LoraBatch(torch.zeros(M, dtype=torch.int32), None, None, L)


def test_python_refusals():
    st, y, x = _stack(), torch.zeros(4, 48, dtype=torch.float16), torch.zeros(4, 64, dtype=torch.float16)
    h = torch.float16
    for bad_y, bad_x, bad_stack, bad_batch, act in [
            (y[:, :40], x, st, _batch(), None), (y[:3], x, st, _batch(), None), (y, x[:, :32], st, _batch(), None),
            (y, x[0], st, _batch(), None), (y.bfloat16(), x, st, _batch(), None), (y, x.float(), st, _batch(), None),
            (y, x, st._replace(parts=(24, 16)), _batch(), None), (y, x, st._replace(parts=(48,)), _batch(), None),
            (y, x, st._replace(a=st.a[0]), _batch(), None), (y, x, st._replace(b=st.b.bfloat16()), _batch(), None),
            (y, x, st._replace(scaling=st.scaling.half()), _batch(), None),
            (y, x, st._replace(scaling=st.scaling[:2]), _batch(), None),
            (y, x, st._replace(ranks=st.ranks.long()), _batch(), None),
            (y, x, st._replace(b=torch.zeros(3, 16, 48, dtype=h).transpose(1, 2)), _batch(), None),
            (y, x, st._replace(a=torch.zeros(3 * 32 * 64 + 1, dtype=h)[1:].view(3, 32, 64)), _batch(), None),
            (y, x, st, _batch(M=5), None), (y, x, st, _batch(L=4), None),
            (y, x, st, _batch()._replace(adapter_ids=torch.zeros(4, dtype=torch.int64)), None),
            (y, x, st, _batch()._replace(sorted_ids=torch.zeros(64, dtype=torch.int32)), None),
            (y, x, st, _batch()._replace(sorted_ids=torch.zeros(63, dtype=torch.int32),
                                         block_adapters=torch.zeros(4, dtype=torch.int32)), None),
            (y, x, st, _batch()._replace(sorted_ids=torch.zeros(64, dtype=torch.int32),
                                         block_adapters=torch.zeros(3, dtype=torch.int32)), None), (y, x, st, _batch(), "relu"),
            (y, x, st._replace(parts=(16, 32)), _batch(), "silu")]:
        with pytest.raises(ValueError):
            ops.lora_add(bad_y, bad_x, bad_stack, bad_batch, activation=act)
    with pytest.raises(ValueError, match="device tensors"):  # all else is in order
        ops.lora_add(y, x, st, _batch())
    for ids, n in ((torch.zeros(4, dtype=torch.int64), 3), (torch.zeros((2, 2), dtype=torch.int32), 3),
                   (torch.zeros(4, dtype=torch.int32), 0), (torch.zeros(4, dtype=torch.int32), 512)):
        with pytest.raises(ValueError):
            ops.lora_route(ids, n)
    with pytest.raises(ValueError, match="device tensors"):
        ops.lora_route(torch.zeros(4, dtype=torch.int32), 3)


def _call(lib, **kw):
    a = dict(y=4096, x=8192, a=16384, b=32768, scaling=64, ranks=128, out=65536, M=4, N=48, K=64, L=3, R=16, parts=2,
             cols=(24, 24), dtype=0, act=0, ids=192, sorted=256, blocks=512, ws=1 << 20, wsb=1 << 30)
    a.update(kw)
    cols = (ctypes.c_int64 * len(a["cols"]))(*a["cols"]) if a["cols"] else None
    return lib.awq_lora_add(a["y"], a["x"], a["a"], a["b"], a["scaling"], a["ranks"], a["out"], a["M"], a["N"], a["K"],
                            a["L"], a["R"], a["parts"], cols, a["dtype"], a["act"], a["ids"], a["sorted"], a["blocks"],
                            a["ws"], a["wsb"], None)


def test_c_abi_refusals():
    """Every bad call is turned away before a launch (the pointers are never read)."""
    lib = _lib.load()
    inv, uns, wsp = _lib.AWQ_STATUS_INVALID_ARGUMENT, _lib.AWQ_STATUS_UNSUPPORTED, _lib.AWQ_STATUS_WORKSPACE
    for want, kw in [
            (inv, dict(dtype=2)), (inv, dict(act=3)), (inv, dict(M=-1)), (inv, dict(K=60)), (inv, dict(R=12)),
            (inv, dict(N=44)), (inv, dict(R=0)), (inv, dict(cols=None)), (inv, dict(cols=(24, 16))),
            (inv, dict(cols=(20, 28))), (inv, dict(cols=(48, 0))), (inv, dict(cols=(56, -8))),
            (inv, dict(act=1, cols=(16, 32))), (inv, dict(act=1, parts=1, cols=(48,))), (inv, dict(act=1, out=4096)),
            (inv, dict(y=None)), (inv, dict(x=None)), (inv, dict(a=None)), (inv, dict(b=None)),
            (inv, dict(scaling=None)), (inv, dict(ranks=None)), (inv, dict(out=None)),
            (inv, dict(blocks=None)), (inv, dict(ids=None, sorted=None)),
            (uns, dict(M=257, sorted=None, blocks=None)),
            (uns, dict(M=256, N=1 << 24, R=8, cols=(1 << 23, 1 << 23), sorted=None, blocks=None)), (inv, dict(y=4104)), (inv, dict(x=8194)), (inv, dict(a=16392)),
            (inv, dict(b=32776)), (inv, dict(out=65544)),
            (uns, dict(R=264)), (uns, dict(L=0)), (uns, dict(L=512)), (uns, dict(parts=5, cols=(8,) * 6)),
            (uns, dict(parts=0, cols=(48,))), (uns, dict(M=1 << 24)), (uns, dict(M=1 << 23, K=128)),
            (uns, dict(K=1 << 24)), (uns, dict(N=1 << 30, cols=(1 << 29, 1 << 29))),
            (wsp, dict(ws=None)), (wsp, dict(wsb=16)), (wsp, dict(ws=(1 << 20) + 8))]:
        assert _call(lib, **kw) == want, kw
        assert lib.awq_last_error()
    assert _call(lib, M=0, y=None, x=None, ws=None) == 0
    for routed, rows in ((1, 4 + 4 * 15), (0, 4)):
        need = lib.awq_lora_workspace_bytes(4, 48, 64, 3, 16, 2, routed)
        assert need >= rows * 32 * 4
        assert _call(lib, wsb=need - 1, **({} if routed else dict(sorted=None, blocks=None))) == wsp
        assert lib.awq_lora_workspace_bytes(0, 48, 64, 3, 16, 2, routed) == 0
        assert lib.awq_lora_workspace_bytes(4, 48, 64, 3, 304, 2, routed) == uns
    for want, args in [(uns, (16, 4, 0, 16, 16, 16, 16, None)), (uns, (16, 4, 512, 16, 16, 16, 16, None)),
                       (uns, (16, -1, 3, 16, 16, 16, 16, None)), (uns, (16, 1 << 24, 3, 16, 16, 16, 16, None)),
                       (inv, (None, 4, 3, 16, 16, 16, 16, None)), (inv, (16, 4, 3, None, 16, 16, 16, None)),
                       (inv, (16, 4, 3, 16, None, 16, 16, None)), (inv, (16, 4, 3, 16, 16, None, 16, None)),
                       (inv, (16, 4, 3, 16, 16, 16, None, None))]:
        assert lib.awq_lora_route(*args) == want, args
