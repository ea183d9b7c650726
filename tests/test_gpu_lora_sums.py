"""How much of v = A x reaches the second product: sums that cancel down to their last bits, exactly."""
import pytest
import torch

from sglite_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R", [8, 64, 128, 256])
@pytest.mark.parametrize("M", [1, 16, 40, 600, 1600])
def test_differences_of_large_sums_are_exact(M, R, dtype):
    """Each sum is a whole number of 23 bits, its digits in A and their places in x, so that fp32 adds them exactly;
    B takes the difference, at most 127, of two of them: every value on the way is exact, and so is the output."""
    K, L, N = 200, 3, 136
    g = torch.Generator().manual_seed(M + R)
    large = torch.randint(1 << 22, (1 << 23) - (1 << 16), (L, R // 2), generator=g)
    d = torch.randint(1, 128, (L, R // 2), generator=g)
    v = torch.stack([large + d, large], -1).reshape(L, R)
    a = torch.zeros((L, R, K))
    at = (3, K // 2, K - 1)
    for k, digit in zip(at, (v & 255, v >> 8 & 127, v >> 15)):
        a[:, :, k] = digit.float()
    x = torch.zeros((M, K))
    for k, place in zip(at, (1.0, 2.0 ** 8, 2.0 ** 15)):
        x[:, k] = place
    sign = torch.where(torch.arange(M) % 3 == 1, -1.0, 1.0)
    x *= sign[:, None]
    b = torch.zeros((L, N, R))
    n = torch.arange(N)
    pair = n % (R // 2)
    b[:, n, 2 * pair], b[:, n, 2 * pair + 1] = 1.0, -1.0
    scaling = torch.tensor([1.0, 0.5, 4.0])
    ids = torch.arange(M, dtype=torch.int32) // 5 % L
    stack = ops.LoraStack(a.to(dtype).to(DEV), b.to(dtype).to(DEV), scaling.to(DEV),
                          torch.full((L,), R, dtype=torch.int32, device=DEV), (N,))
    assert torch.equal(stack.a.float().cpu(), a)
    got = ops.lora_add(torch.zeros((M, N), dtype=dtype, device=DEV), x.to(dtype).to(DEV), stack,
                       ops.lora_route(ids.to(DEV), L))
    want = (d[ids.long()][:, pair].float() * scaling[ids.long()][:, None] * sign[:, None])
    assert torch.equal(got.float().cpu(), want)
