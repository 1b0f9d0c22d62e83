"""Row sums that blocks of a product's own launch write are read by tiles as they come: rows of a neighbouring tile, not yet written, must not be
read from a line that another tile brought into the cache.  Calls on two inputs in turn leave sums of the other one in memory; a call
on the same input again finds its own.  Row counts that are no multiple of 8 and of tiles, so that rows of two tiles are neighbours there."""
import pytest
import torch

from kiln_amd import marlin_gemm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [0, 16])
@pytest.mark.parametrize("m,k,n", [(1503, 2176, 5888), (1501, 2560, 5120), (777, 2560, 9216), (1031, 1152, 6144), (2045, 1280, 4096), (515, 640, 10240)])
def test_sums_are_the_calls_own(m, k, n, rank):
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    b = torch.randint(-2**31, 2**31, (k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    s = ((torch.rand(k // 128, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    x = [(torch.randn(m, k, device="cuda", generator=gen) + shift).bfloat16() for shift in (0.0, 40.0)]
    a_, b_ = (torch.randn(shape, device="cuda", generator=gen).bfloat16() for shape in ((max(rank, 1), k), (n, max(rank, 1))))

    def call(x):
        return marlin_gemm.marlin_w4a16_gemm_lora(x, b, s, 128, a_, b_, [rank], [0.5]) if rank else marlin_gemm.marlin_w4a16_gemm(x, b, s, 128)

    for x_ in x:                       # twice: the second finds the first one's sums
        call(x_)
    want = []
    for x_ in x:
        call(x_)
        want.append(call(x_).view(torch.int16))
    for i in range(24):
        assert torch.equal(call(x[i % 2]).view(torch.int16), want[i % 2]), i
