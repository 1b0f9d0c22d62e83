"""The product behind a bank's gradient of the rows in every size of its blocks, with its contraction whole and in slices: against the
formulas in 64 bits, at row counts and widths that no block divides, with the adapters' runs crossing blocks."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, marlin_gemm
from tests.test_gpu_bank import backward, bits, check_backward, problem

pytestmark = pytest.mark.gpu

# block (rows, columns of k), slices of n: m, k, n, groupsize, adapters, rank, pattern
CASES = [
    ((128, 128), 1, (300, 1152, 768, 128, 5, 24, "any")), ((128, 128), 1, (65, 640, 512, -1, 3, 64, "any")), ((128, 128), 5, (300, 1152, 2560, 128, 4, 40, "runs")),
    ((128, 256), 1, (1301, 4736, 512, 128, 5, 24, "any")), ((128, 256), 3, (777, 2432, 4864, -1, 7, 40, "runs")),
    ((256, 256), 1, (1500, 9344, 768, 128, 6, 16, "any")), ((256, 256), 5, (2001, 1408, 9472, 128, 3, 24, "any")),
    ((256, 256), 3, (1301, 3200, 4864, -1, 40, 64, "runs")), ((256, 256), 3, (2048, 2560, 18432, 128, 1, 32, "one")),
]


def planned(block, slices, m, n, k):
    out = (ctypes.c_int * 3)()
    assert _lib.load().kiln_w4a16_debug_bank_backward_plan(m, n, k, out) == 0
    return (out[0], out[1]) == block and out[2] == slices


@pytest.mark.parametrize("block,slices,shape", CASES)
def test_against_the_formulas(block, slices, shape):
    m, k, n, *_ = shape
    assert planned(block, slices, m, n, k)
    p = problem(*shape, seed=20)
    made = backward(p)
    check_backward(p, *made)
    assert all(torch.equal(a, b) for a, b in zip(bits(made), bits(backward(p))))
    none = {**p, "of": torch.full_like(p["of"], -1)}
    assert torch.equal(bits(marlin_gemm.marlin_w4a16_gemm_backward(p["dy"], p["b"], p["s"], p["g"]))[0], bits(backward(none)[0])[0])


@pytest.mark.parametrize("block,slices,shape", [c for c in CASES if c[0] != (128, 128)])
def test_an_adapter_that_holds_no_numbers_stays_with_its_own_rows(block, slices, shape):
    p = problem(*shape, seed=21)
    if shape[4] == 1:
        p["of"][::3] = -1
    p["of"][0] = p["of"][-1] = 0
    bad = {**p, "a_": p["a_"].clone()}
    k = shape[1]
    odd = torch.zeros(k, dtype=torch.bool, device="cuda")
    odd[17] = odd[k - 1] = odd[k // 2] = True
    bad["a_"][0, 3, 17], bad["a_"][0, 5, k - 1], bad["a_"][0, 0, k // 2] = float("inf"), float("nan"), float("-inf")
    mine = p["of"] == 0
    da, ea = backward(p)[0], backward(bad)[0]
    assert torch.equal(bits(da[~mine])[0], bits(ea[~mine])[0])
    assert torch.equal(bits(da[mine][:, ~odd])[0], bits(ea[mine][:, ~odd])[0])
    assert not bool(torch.isfinite(ea[mine][:, odd]).any()) and bool(torch.isnan(ea[mine][:, k - 1]).all())
