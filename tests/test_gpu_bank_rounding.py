"""Calls on a bank whose term lands on the f32 sums of the product round once, others twice, as the library says of a call.

Rounded once, a value is the bf16 value nearest to the formula's unless that lies as near to a border between two as the f32 sums are off.  Partial
sums of these products (codes of up to 144 times scales of s, rows of 1: sqrt(k) 150 s) round by 2^-25 of themselves on average, sqrt(k) of
them add up to k 150 s 2^-25, a few of 10^-2 s at k = 2560 where a step of y, of 4.6 sqrt(k) s and more, is 2^-8 of it, s: few in a hundred
are off.  Rounded in between, the base is off by up to half a step before the term is added: a quarter of the values and more."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, marlin_gemm
from tests.test_gpu_bank import forward, problem

pytestmark = pytest.mark.gpu
ONE_LAUNCH, BASE, BEHIND, IN_PRODUCT = range(4)


@pytest.mark.parametrize("method,shape", [
    (ONE_LAUNCH, (1, 2560, 2560, 128, 4, 8, "one")), (ONE_LAUNCH, (2, 256, 256, -1, 3, 16, "any")), (ONE_LAUNCH, (1, 640, 512, -1, 3, 64, "one")),
    (ONE_LAUNCH, (2, 128, 8192, 128, 5, 24, "runs")), (IN_PRODUCT, (2100, 2560, 8192, 128, 40, 24, "any")), (IN_PRODUCT, (2048, 2560, 8192, -1, 3, 64, "runs")),
    (IN_PRODUCT, (2177, 2560, 8192, 128, 300, 8, "any")),
    (BASE, (16, 2560, 2560, 128, 16, 16, "any")), (BEHIND, (77, 4096, 512, -1, 3, 32, "runs"))])
def test_values_that_are_the_nearest(method, shape):
    m, k, n, g, count, rank, pattern = shape
    out = (ctypes.c_int * 2)()
    assert _lib.load().kiln_w4a16_debug_bank_plan(m, n, k, rank, torch.cuda.get_device_properties(0).multi_processor_count, out) == 0 and out[0] == method
    p = problem(*shape, seed=30)
    p["of"] = p["of"].clamp(0, count - 1)
    want = p["x"].double() @ marlin_gemm.dequant_f32(p["b"], p["s"], g).double()
    for j in range(count):
        mine, s, a, b = p["of"] == j, p["sc"][j].double(), p["a_"][j].double(), p["b_"][j].double()
        want[mine] += s * ((p["x"][mine].double() @ a.t()) @ b.t())
    nearest = (forward(p) == want.to(torch.bfloat16)).double().mean().item()
    if method in (ONE_LAUNCH, IN_PRODUCT):
        assert nearest >= 0.9
    else:
        assert nearest <= 0.9
