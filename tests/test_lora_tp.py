"""Adapters under tensor parallelism: two ranks over gloo (CPU tensors), lora_add by its formula.

A column-parallel layer holds A whole and its columns of B, a row-parallel one its input slice of A and B whole: the
all-reduce of its partial outputs must sum the adapters' parts once, with those of the weight."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

H, I, T, SLOTS, R = 64, 96, 7, 3, 5


def _lora_add(y, x, stack, batch, activation=None, out=None):
    """The operator's definition, in float32 (the layers' own slots and arguments)."""
    res, rank = y.clone(), stack.b.shape[2]
    for m, e in enumerate(batch.adapter_ids.tolist()):
        col = 0
        for p, n in enumerate(stack.parts):
            if 0 <= e < batch.num_adapters:
                a, b = stack.a[e, p * rank:(p + 1) * rank].float(), stack.b[e, col:col + n].float()
                res[m, col:col + n] += stack.scaling[e] * (b @ (a @ x[m]))
            col += n
    if activation is not None:
        g, u = res.chunk(2, -1)
        return torch.nn.functional.silu(g) * u
    return res if out is None else out.copy_(res)


def _data():
    g = torch.Generator().manual_seed(11)
    r = lambda *shape: torch.randn(shape, generator=g) * 0.2  # noqa: E731
    adapters = [{n: ((r(R - s, k)).half().float(), r(o, R - s).half().float()) for n, k, o in
                 (("gate", H, I), ("up", H, I), ("down", I, H))} for s in range(SLOTS)]
    return r(T, H), {"gate": r(I, H), "up": r(I, H), "down": r(H, I)}, adapters, torch.tensor([0, -1, 2, 1, 1, 0, -1],
                                                                                              dtype=torch.int32)


def _whole(x, w, adapters, ids):
    def project(t, n):
        y = t @ w[n].t()
        for m, e in enumerate(ids.tolist()):
            if e >= 0:
                a, b = adapters[e][n]
                y[m] += (0.5 + e) * (b @ (a @ t[m]))
        return y
    return project(torch.nn.functional.silu(project(x, "gate")) * project(x, "up"), "down")


def _rank(rank, world, port, q):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from sglite_amd import ops
        from sglite_amd.linear import MergedColumnParallelLinear, RowParallelLinear

        ops.lora_add = _lora_add
        x, w, adapters, ids = _data()
        part = slice(rank * (I // world), (rank + 1) * (I // world))
        gate_up = MergedColumnParallelLinear(H, [I, I], False, tp_size=world)
        down = RowParallelLinear(I, H, False, tp_size=world)
        gate_up.load_state_dict({"weight": torch.cat([w["gate"][part], w["up"][part]])})
        down.load_state_dict({"weight": w["down"][:, part].contiguous()})
        for layer in (gate_up, down):
            layer.add_adapters(SLOTS, R, torch.float16)
        for s, ad in enumerate(adapters):
            gate_up.load_adapter(s, [ad["gate"][0], ad["up"][0]], [ad["gate"][1][part], ad["up"][1][part]], 0.5 + s)
            down.load_adapter(s, ad["down"][0][:, part], ad["down"][1], 0.5 + s)
        batch = ops.LoraBatch(ids, None, None, SLOTS)
        y = down(gate_up.forward_act(x, "silu", batch), batch)
        want = _whole(x, w, adapters, ids)
        q.put((rank, float((y - want).abs().max()), float(want.abs().max())))
    finally:
        dist.destroy_process_group()


def test_two_ranks_sum_the_adapters_once():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for rank, err, size in sorted(res):
        # float32 sums of at most 2 * (I + R) products in two orders, through one product of sums.
        assert err <= 8 * (I + R) * 2.0 ** -24 * max(1.0, size) * 10, (rank, err, size)
