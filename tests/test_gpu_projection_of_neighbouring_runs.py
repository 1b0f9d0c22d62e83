"""A launch of the mid-M kernel that projects onto its adapters itself, in several runs of 64 rows: each run waits for its own rows of the
projection, and must not read those of the next run, not yet written, from a line that it brought into the cache.  Calls on two
inputs in turn leave the other one's projection in memory."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, marlin_gemm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n,rank", [(65, 2560, 18432, 40), (70, 9216, 2560, 48), (101, 2560, 18432, 40), (131, 4096, 2560, 40), (199, 2560, 4096, 40), (69, 2560, 2560, 16),
                                        (251, 2560, 2560, 40), (255, 2560, 2560, 64)])
def test_a_run_reads_its_own_projection(m, k, n, rank):
    L = _lib.load()
    out = (ctypes.c_size_t * 6)()
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert L.kiln_w4a16_debug_workspace_operands(m, n, k, cus, rank, 1 << 30, out) == 0 and out[4] > 1
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    b = torch.randint(-2**31, 2**31, (k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    s = ((torch.rand(k // 128, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    x = [(torch.randn(m, k, device="cuda", generator=gen) + shift).bfloat16() for shift in (0.0, 40.0)]
    a_ = (torch.randn(rank, k, device="cuda", generator=gen) / k ** 0.5).bfloat16()
    b_ = (torch.randn(n, rank, device="cuda", generator=gen) / rank ** 0.5).bfloat16()
    call = lambda x: marlin_gemm.marlin_w4a16_gemm_lora(x, b, s, 128, a_, b_, [rank], [0.5])
    want = []
    for x_ in x:
        call(x_)
        want.append(call(x_).view(torch.int16))
        # the term added to what the plain product has: two roundings to bf16 (2^-8 each) and T's own, and f32 sums
        plain = marlin_gemm.marlin_w4a16_gemm(x_, b, s, 128).double()
        low = 0.5 * (x_.double() @ a_.double().t()) @ b_.double().t()
        size = 0.5 * (x_.double().abs() @ a_.double().abs().t()) @ b_.double().abs().t()   # no less than the slices of T are in all
        base = (x_.double().abs().sum(1, keepdim=True) * s.double().max() * 280) * (k + 8) * 2.0 ** -24
        got = want[-1].view(torch.bfloat16).double()
        excess = (got - plain - low).abs() - (2.0 ** -8 * (plain.abs() + (plain + low).abs()) + (2.0 ** -8 + (k + 2 * rank) * 2.0 ** -24) * size + 2 * base) * (1 + 2.0 ** -8)
        assert excess.max().item() <= 0
    for i in range(24):
        assert torch.equal(call(x[i % 2]).view(torch.int16), want[i % 2]), i
