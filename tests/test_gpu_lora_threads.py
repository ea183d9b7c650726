"""Adapters called from several threads on one stream."""
import threading

import pytest
import torch

from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [(1, 3), (40, 64), (600, 700)])
def test_two_threads_on_one_stream(rows):
    """Each thread's results are those of its calls alone: the launches of two calls may come in any order."""
    def inputs(M, seed):
        g = torch.Generator().manual_seed(seed)
        stack = ops.make_lora_stack(3, 16, 512, (128, 64), torch.float16, torch.device(DEV))
        stack.a.copy_(torch.randn(stack.a.shape, generator=g) / 20)
        stack.b.copy_(torch.randn(stack.b.shape, generator=g) / 3)
        stack.scaling.fill_(1.0), stack.ranks.fill_(16)
        x, y = torch.randn((M, 512), generator=g).half().to(DEV), torch.randn((M, 192), generator=g).half().to(DEV)
        return y, x, stack, torch.randint(0, 3, (M,), generator=g, dtype=torch.int32).to(DEV)

    sets = [inputs(M, seed) for seed, M in enumerate(rows)]
    want = [ops.lora_add(y, x, stack, ops.lora_route(ids, 3)) for y, x, stack, ids in sets]
    torch.cuda.synchronize()
    wrong, done = [], []

    def call(n):
        y, x, stack, ids = sets[n]
        got = [ops.lora_add(y, x, stack, ops.lora_route(ids, 3)) for _ in range(200)]
        torch.cuda.synchronize()
        wrong.append(sum(not torch.equal(want[n], t) for t in got))
        done.append(n)

    threads = [threading.Thread(target=call, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert sorted(done) == [0, 1] and wrong == [0, 0]
