"""Adapters of many rows: the 64-row tiles at every rank's first sizes, and what must stay in its row there."""
import pytest
import torch

from sglite_amd import ops
from test_gpu_lora import DEV, close, deltas, gated, make

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,parts,L,R", [(511, 136, (72, 24), 3, 40), (512, 136, (72, 24), 3, 40),
                                           (1023, 64, (40,), 7, 24), (1024, 64, (40,), 7, 24),
                                           (1535, 200, (72, 24), 100, 16), (1536, 200, (72, 24), 100, 16),
                                           (1601, 72, (264,), 511, 8), (1700, 256, (64, 40, 24), 5, 32)])
def test_both_sides_of_the_lines(M, K, parts, L, R, dtype):
    y, x, stack, ids = make(M, K, parts, L, R, dtype, [(R, R // 2 + 1, 1, 0, R - 1)[e % 5] for e in range(L)], seed=M)
    for order in (ids, ids.sort().values, ids.sort(descending=True).values):  # scattered and in sequences
        ids.copy_(order)
        want, err = deltas(y, x, stack, ids)
        got = ops.lora_add(y, x, stack, ops.lora_route(ids, L))
        close(got, want, err)
        none = (ids < 0) | (stack.ranks[ids.clamp(min=0).long()] == 0)
        assert torch.equal(got[none], y[none])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,R", [(1550, 24), (600, 40), (600, 104)])
def test_gated(M, R, act, dtype):
    y, x, stack, ids = make(M, 264, (72, 72), 6, R, dtype, [R, 1, R // 2 + 1, 0, R - 1, 8])
    want, err = gated(*deltas(y, x, stack, ids), act)
    close(ops.lora_add(y, x, stack, ops.lora_route(ids, 6), activation=act), want, err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** -10, 1.0, 2.0 ** 9])
def test_large_and_small_sums(dtype, scale):
    """v = A x of 2^7 times x's size: beyond fp16's range in the last case."""
    y, x, stack, ids = make(1540, 512, (64,), 2, 16, dtype, scale=scale)
    stack.a.mul_(2.0 ** 7)
    stack.b.mul_(2.0 ** -12)
    close(ops.lora_add(y, x, stack, ops.lora_route(ids, 2)), *deltas(y, x, stack, ids))


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_and_nan_inputs_stay_in_their_rows(dtype):
    y, x, stack, ids = make(1600, 128, (64,), 2, 16, dtype)
    ids[:] = 1
    want, err = deltas(y, x, stack, ids)
    x[3, 5], x[1520, 127] = float("inf"), float("nan")
    got = ops.lora_add(y, x, stack, ops.lora_route(ids, 2))
    keep = torch.ones(1600, dtype=torch.bool, device=DEV)
    keep[3] = keep[1520] = False
    close(got[keep], want[keep], err[keep])
    assert got[1520].isnan().all() and not got[3].isfinite().any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_past_a_rank_does_not_count(bad):
    """NaN and infinities past an adapter's rank, in other adapters and in rows without one."""
    y, x, stack, ids = make(1600, 136, (40, 24), 3, 32, torch.bfloat16, [13, 32, 27])
    ids[:] = torch.arange(1600, device=DEV, dtype=torch.int32) % 4 - 1
    ids[ids == 1] = 0
    want, err = deltas(y, x, stack, ids)
    for p in range(2):
        stack.a[0, p * 32 + 13:p * 32 + 32] = bad
        stack.a[2, p * 32 + 27:p * 32 + 32] = bad
    stack.b[0, :, 13:] = bad
    stack.b[2, :, 27:] = bad
    stack.a[1], stack.b[1] = bad, bad
    x[ids < 0] = bad
    close(ops.lora_add(y, x, stack, ops.lora_route(ids, 3)), want, err)


def test_same_bits_every_time():
    y, x, stack, ids = make(2000, 1024, (256,), 5, 32, torch.bfloat16)
    first = ops.lora_add(y, x, stack, ops.lora_route(ids, 5))
    assert all(torch.equal(first, ops.lora_add(y, x, stack, ops.lora_route(ids, 5))) for _ in range(5))
