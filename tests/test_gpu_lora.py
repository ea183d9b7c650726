"""Adapters of many requests beside a projection, against the formula in 64 bits."""
import pytest
import torch

from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Half a step of the type, and what is left of a value that enters the MFMAs as
# two of the type (relative to the largest of its row).
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SPLIT = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def make(M, K, parts, L, R, dtype, ranks=None, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    N, P = sum(parts), len(parts)
    a = (torch.randn((L, P * R, K), generator=g) / K ** 0.5).to(dtype)
    b = (torch.randn((L, N, R), generator=g) * 0.3).to(dtype)
    ranks = torch.tensor([R] * L if ranks is None else ranks, dtype=torch.int32)
    stack = ops.LoraStack(a.to(DEV), b.to(DEV), torch.rand(L, generator=g).add(0.5).to(DEV), ranks.to(DEV),
                          tuple(parts))
    x = (torch.randn((M, K), generator=g) * scale).to(dtype).to(DEV)
    y = torch.randn((M, N), generator=g).to(dtype).to(DEV)
    ids = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32).to(DEV)
    return y, x, stack, ids


def routed(ids, L):
    """The sorted tables whatever the row count."""
    return ops.LoraBatch(ids, *torch.ops.sglite_awq.awq_lora_route(ids, L), L)


def deltas(y, x, stack, ids):
    """(y + scaling B A x, a bound of its error before the last rounding), row by row in 64 bits."""
    out, err = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    L, N, R = stack.b.shape
    K = x.shape[1]
    for e in range(L):
        r = min(max(int(stack.ranks[e]), 0), R)
        rows = (ids == e).nonzero().reshape(-1)
        if r == 0 or rows.numel() == 0:
            continue
        xe, s, c = x[rows].double(), float(stack.scaling[e]), 0
        for p, w in enumerate(stack.parts):
            A, B = stack.a[e, p * R:p * R + r].double(), stack.b[e, c:c + w, :r].double()
            v = xe @ A.t()
            out[rows, c:c + w] += s * (v @ B.t())
            # fp32 sums of K and of r products, the split of v, a few roundings of the result.
            mag = (xe.abs() @ A.abs().t()) @ B.abs().t()
            err[rows, c:c + w] = s * (SPLIT[x.dtype] * v.abs().amax(1, keepdim=True) * B.abs().sum(1)[None]
                                      + (K + r + 8) * 2.0 ** -24 * mag) + 2.0 ** -22 * out[rows, c:c + w].abs()
            c += w
    return out, err


def gated(out, err, act):
    h = out.shape[1] // 2
    g, u, eg, eu = out[:, :h], out[:, h:], err[:, :h], err[:, h:]
    f = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    # Slopes of silu and gelu stay below 1.13; exp, erf and the divide within 2^-20 of the result.
    return f * u, 1.13 * eg * (u.abs() + eu) + f.abs() * eu + 2.0 ** -20 * (f * u).abs() + 2.0 ** -20 * (g * u).abs()


def close(got, want, err):
    # Half a step of the type, or of its smallest values.
    tol = err + HALF[got.dtype] * (want.abs() + err) + 2.0 ** -25
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float(((got.double() - want).abs() - tol).max()):.3e}"


SHAPES = [
    # M, K, parts, L, R
    (1, 256, (64,), 1, 8),
    (1, 2560, (4096, 1024, 1024), 4, 16),
    (2, 8, (8,), 3, 8),
    (5, 72, (24, 8, 40), 2, 16),
    (16, 4096, (2560,), 16, 24),
    (17, 1000, (136,), 5, 40),
    (33, 520, (64, 64), 40, 64),
    (64, 512, (96, 32), 2, 128),
    (100, 384, (8, 16, 24, 32), 3, 256),
    (130, 256, (264,), 511, 8),
    (333, 1024, (512, 128, 128), 8, 8),
    (700, 640, (328,), 3, 72),
    (1111, 768, (640, 64), 6, 32),
    (2048, 256, (192,), 1, 200),
    (515, 136, (72, 24), 100, 16),
    (4100, 2048, (1024, 256, 256), 9, 64),
    (600, 64, (40, 40, 40, 8), 2, 256),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,K,parts,L,R", SHAPES)
def test_lora_add(M, K, parts, L, R, dtype):
    ranks = [(R, R // 2 + 1, 1, 0, R - 1)[e % 5] for e in range(L)]
    y, x, stack, ids = make(M, K, parts, L, R, dtype, ranks)
    if M == 1:
        ids[:] = 0
    y0 = y.clone()
    batch = ops.lora_route(ids, L)
    want, err = deltas(y, x, stack, ids)
    got = ops.lora_add(y, x, stack, batch)
    close(got, want, err)
    none = (ids < 0) | (stack.ranks[ids.clamp(min=0).long()] == 0)
    assert torch.equal(got[none], y0[none]) and torch.equal(y, y0)
    inplace = ops.lora_add(y, x, stack, batch, out=y)
    assert inplace is y and torch.equal(y, got)
    other = torch.full_like(y0, 7.0)
    assert torch.equal(ops.lora_add(y0, x, stack, batch, out=other), got)
    # Few rows by the tables of a larger step, a larger step row by row.
    assert (batch.sorted_ids is None) == (M <= 16)
    if M <= 256:
        for b in (routed(ids, L), ops.LoraBatch(ids, None, None, L)):
            got = ops.lora_add(y0, x, stack, b)
            close(got, want, err)
            assert torch.equal(got[none], y0[none])
            z = y0.clone()
            assert torch.equal(ops.lora_add(z, x, stack, b, out=z), got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,half,L,R", [(1, 2560, 9728, 4, 16), (7, 64, 8, 2, 8), (40, 512, 200, 9, 48),
                                          (90, 128, 72, 3, 136), (1500, 512, 168, 4, 64)])
def test_lora_add_gated(M, K, half, L, R, act, dtype):
    y, x, stack, ids = make(M, K, (half, half), L, R, dtype, [R - e % 3 for e in range(L)], seed=M)
    batch = ops.lora_route(ids, L)
    want, err = gated(*deltas(y, x, stack, ids), act)
    close(ops.lora_add(y, x, stack, batch, activation=act), want, err)
    if M <= 256:
        for b in (routed(ids, L), ops.LoraBatch(ids, None, None, L)):
            close(ops.lora_add(y, x, stack, b, activation=act), want, err)


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("L,R", [(9, 16), (9, 64), (6, 128), (5, 200)])
def test_blocks_of_many_columns(L, R, act):
    """Row blocks with two column steps a wave; the last one of a part, and its columns, are cut short."""
    parts = (9000, 9000) if act else (12872, 4104, 40)
    y, x, stack, ids = make(270, 64, parts, L, R, torch.float16, [(R, R - 3, 0, 1)[e % 4] for e in range(L)], seed=R)
    ids[:20] = -1
    y0 = y.clone()
    batch = ops.lora_route(ids, L)
    assert batch.sorted_ids is not None
    want, err = deltas(y, x, stack, ids)
    if act:
        close(ops.lora_add(y, x, stack, batch, activation=act), *gated(want, err, act))
        return
    got = ops.lora_add(y, x, stack, batch)
    close(got, want, err)
    assert torch.equal(got[ids < 0], y0[ids < 0])
    assert torch.equal(ops.lora_add(y, x, stack, batch, out=y), got)


def test_every_id_without_an_adapter_names_none():
    y, x, stack, ids = make(50, 128, (64,), 4, 16, torch.float16)
    ids[::2] = torch.tensor([-1, 4, 5, -7, 2 ** 31 - 1, -2 ** 31, 1000, 511, 512, 4, -1, -2, 99, 4, 5, 6, 7, 8, 9, 10,
                             11, 12, 13, 14, 15], dtype=torch.int32, device=DEV)
    batch = ops.lora_route(ids, 4)
    got = ops.lora_add(y, x, stack, batch)
    close(got, *deltas(y, x, stack, ids))
    assert torch.equal(got[::2], y[::2])


def test_all_rows_without_an_adapter_and_all_on_one():
    for M in (9, 200, 800):
        y, x, stack, ids = make(M, 128, (64, 64), 3, 16, torch.bfloat16)
        ids[:] = -1
        batch = ops.lora_route(ids, 3)
        assert torch.equal(ops.lora_add(y, x, stack, batch), y)
        close(ops.lora_add(y, x, stack, batch, activation="silu"), *gated(*deltas(y, x, stack, ids), "silu"))
        ids[:] = 2
        close(ops.lora_add(y, x, stack, ops.lora_route(ids, 3)), *deltas(y, x, stack, ids))


def test_no_rows():
    y, x, stack, ids = make(0, 128, (64,), 3, 16, torch.float16)
    batch = ops.lora_route(ids, 3)
    assert ops.lora_add(y, x, stack, batch).shape == (0, 64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** -10, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("M", [20, 40, 520])
def test_large_and_small_sums(M, dtype, scale):
    """v = A x of 2^7 times x's size: beyond fp16's range in the last case."""
    y, x, stack, ids = make(M, 512, (64,), 2, 16, dtype, scale=scale)
    stack.a.mul_(2.0 ** 7)
    stack.b.mul_(2.0 ** -12)
    close(ops.lora_add(y, x, stack, ops.lora_route(ids, 2)), *deltas(y, x, stack, ids))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_past_a_rank_does_not_count(bad):
    """NaN and infinities past an adapter's rank, in other adapters and in rows without one."""
    for dtype in (torch.float16, torch.bfloat16):
        for M in (3, 90, 600):
            y, x, stack, ids = make(M, 136, (40, 24), 3, 40, dtype, [13, 40, 33])
            ids[:] = torch.arange(M, device=DEV, dtype=torch.int32) % 4 - 1
            ids[ids == 1] = 0
            want, err = deltas(y, x, stack, ids)
            for p in range(2):
                stack.a[0, p * 40 + 13:p * 40 + 40] = bad
                stack.a[2, p * 40 + 33:p * 40 + 40] = bad
            stack.b[0, :, 13:] = bad
            stack.b[2, :, 33:] = bad
            stack.a[1], stack.b[1] = bad, bad
            x[ids < 0] = bad
            close(ops.lora_add(y, x, stack, ops.lora_route(ids, 3)), want, err)


def test_infinite_and_nan_inputs_stay_in_their_rows():
    for dtype, M in ((torch.float16, 30), (torch.bfloat16, 40), (torch.float16, 700)):
        y, x, stack, ids = make(M, 128, (64,), 2, 16, dtype)
        ids[:] = 1
        want, err = deltas(y, x, stack, ids)
        x[3, 5], x[20, 127] = float("inf"), float("nan")
        got = ops.lora_add(y, x, stack, ops.lora_route(ids, 2))
        keep = torch.ones(M, dtype=torch.bool, device=DEV)
        keep[3] = keep[20] = False
        close(got[keep], want[keep], err[keep])
        assert got[20].isnan().all() and not got[3].isfinite().any()


def test_strided_and_offset_inputs():
    y, x, stack, ids = make(30, 128, (64, 32), 3, 16, torch.float16)
    want, err = deltas(y, x, stack, ids)
    batch = ops.lora_route(ids, 3)
    wide = torch.zeros((30, 300), dtype=x.dtype, device=DEV)
    wide[:, 3:131] = x
    wide[:, 140:236] = y
    close(ops.lora_add(wide[:, 140:236], wide[:, 3:131], stack, batch), want, err)
    turned = y.t().contiguous().t()
    close(ops.lora_add(turned, x, stack, batch), want, err)
    odd = torch.zeros(ids.numel() + 1, dtype=torch.int32, device=DEV)
    odd[1:] = ids
    close(ops.lora_add(y, x, stack, ops.lora_route(odd[1:], 3)), want, err)


def test_same_bits_every_time_and_on_another_stream():
    y, x, stack, ids = make(300, 1024, (256,), 5, 32, torch.bfloat16)
    first = ops.lora_add(y, x, stack, ops.lora_route(ids, 5))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = [ops.lora_add(y, x, stack, ops.lora_route(ids, 5)) for _ in range(5)]
    here = [ops.lora_add(y, x, stack, ops.lora_route(ids, 5)) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, t) for t in here + there)


def test_two_graphs_replayed_in_turn_with_new_ids():
    """Captured routing follows the ids in place at each replay, whatever runs eagerly between."""
    sets = [make(M, 512, (128, 64), 4, 16, torch.float16, seed=M) for M in (24, 100)]
    graphs = []
    for y, x, stack, ids in sets:
        ops.lora_add(y, x, stack, ops.lora_route(ids, 4))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.lora_add(y, x, stack, ops.lora_route(ids, 4))
        graphs.append((g, out))
    for n in range(6):
        for (y, x, stack, ids), (g, out) in zip(sets, graphs):
            ids.copy_(torch.randint(-1, 4, ids.shape, dtype=torch.int32, device=DEV))
            want = ops.lora_add(y, x, stack, ops.lora_route(ids, 4))
            g.replay()
            if n % 2:
                torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_registered_ops_and_fakes():
    y, x, stack, ids = make(20, 128, (64, 64), 3, 16, torch.float16)
    eager = ops.lora_add(y, x, stack, routed(ids, 3))
    args = (stack.a, stack.b, stack.scaling, stack.ranks, *routed(ids, 3)[:3])
    assert torch.equal(torch.ops.sglite_awq.awq_lora_add(y, x, *args, [64, 64], "none"), eager)
    z = y.clone()
    torch.ops.sglite_awq.awq_lora_add_(z, x, *args, [64, 64])
    assert torch.equal(z, eager)
    torch.library.opcheck(torch.ops.sglite_awq.awq_lora_add, (y, x, *args, [64, 64], "silu"),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.sglite_awq.awq_lora_add_, (z, x, *args, [64, 64]),
                          test_utils=("test_schema", "test_faketensor"))
