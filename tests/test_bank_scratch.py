"""The scratch of a call on a bank holds what the plan of that call writes into it: the rows' order, the projection in the plan's slices
and, where the product adds the term, the ordered rows with their sums.  CPU only."""
import ctypes

import pytest

from kiln_amd import _lib

ONE_LAUNCH, BASE, BEHIND, IN_PRODUCT = range(4)


def up256(size):
    return -(-size // 256) * 256


def plan(m, n, k, rank, cus=256):
    out = (ctypes.c_int * 2)()
    assert _lib.load().kiln_w4a16_debug_bank_plan(m, n, k, rank, cus, out) == 0
    return tuple(out)


def written(m, n, k, count, rank):
    """The end of what a call writes: order and first, T, then the rows in order, their sums and their adapters."""
    method, slices = plan(m, n, k, rank)
    if method == ONE_LAUNCH:
        return 0
    end = up256(4 * m) + up256(4 * (count + 2)) + 4 * slices * m * rank
    if method == IN_PRODUCT:
        end = up256(end) + up256(2 * m * k) + 4 * m * (k // 128 + 1)
    return end


def test_scratch_holds_every_slice_of_the_projection():
    size = _lib.load().kiln_w4a16_gemm_bank_scratch_bytes
    for k in range(128, 131072 + 1, 128):
        for m in range(1, 18):
            for count, rank in ((1, 64), (4, 8)):
                assert written(m, 256, k, count, rank) <= size(m, 256, k, count, rank), (m, k, count, rank)


@pytest.mark.parametrize("n", [256, 2560, 9216, 18432])
def test_scratch_holds_what_larger_calls_write(n):
    size = _lib.load().kiln_w4a16_gemm_bank_scratch_bytes
    seen = set()
    for k in (128, 640, 2560, 4096, 5248, 8192, 9216, 14336, 32896, 43008, 65664):
        for m in (1, 2, 4, 5, 16, 17, 64, 256, 257, 300, 1029, 2048, 8191):
            seen.add(plan(m, n, k, 24)[0])
            assert written(m, n, k, 7, 24) <= size(m, n, k, 7, 24), (m, k)
    assert {BASE, BEHIND} <= seen


def test_plans_of_every_method():
    assert plan(1, 2560, 2560, 8)[0] == ONE_LAUNCH and plan(16, 18432, 2560, 16)[0] == BASE
    assert plan(77, 2560, 9216, 24)[0] == BEHIND and plan(2048, 18432, 2560, 32)[0] == IN_PRODUCT


def test_no_slice_of_a_plan_is_empty():
    for k in range(128, 131072 + 1, 128):
        for m in (1, 4, 16, 17):
            slices, groups = plan(m, 25600, k, 64)[1], k // 128
            each = -(-groups // slices)
            assert 1 <= slices <= 32 and (slices - 1) * each < groups, (m, k, slices)


def test_a_plan_query_refuses():
    out = (ctypes.c_int * 2)()
    for bad in ((0, 256, 128, 8), (1, 128, 128, 8), (1, 256, 64, 8), (1, 256, 128, 4), (1, 256, 128, 72), (1, 300, 128, 8), (1, 256, 200, 8)):
        assert _lib.load().kiln_w4a16_debug_bank_plan(*bad, 256, out) == 1, bad
