"""Which blocks products of sorted rows and their gradients take (kiln_w4a16_debug_experts_plan), for 256 compute units; no GPU is touched.
0: 32 rows, wavefronts sharing the contraction; 1, 2, 3: 32, 64, 128 rows; 4, 5: 32, 64 rows with two sets of wavefronts."""
import itertools

import pytest

from kiln_amd import _lib

ROWS = {0: 32, 1: 32, 2: 64, 3: 128, 4: 32, 5: 64}


def plan(rows, n, k, experts, backward):
    return _lib.load().kiln_w4a16_debug_experts_plan(rows, n, k, experts, backward, 256)


def counts():
    """Row counts from 1 to some 100000, every one of the first 300."""
    rows = 1
    while rows < 100000:
        yield rows
        rows = rows + 1 if rows < 300 else rows * 103 // 100


@pytest.mark.parametrize("n,k", [(256, 128), (512, 1024), (2048, 768), (2048, 2560), (2560, 1024), (9216, 2560), (28672, 4096)])
def test_blocks_of_128_rows_are_for_experts_that_have_them(n, k):
    """Their kernel has the rows' sums formed by a launch in front, which no smaller block reads.  In the gradient there is no such launch, and experts of a few
    rows run the same code whatever the block."""
    for experts, rows in itertools.product((1, 2, 3, 8, 16, 24, 64, 128, 256, 1024), counts()):
        each = rows / min(rows, experts)
        if plan(rows, n, k, experts, 0) == 3:
            assert rows > 64 and each >= 40, (rows, experts)
        if plan(rows, n, k, experts, 1) == 3:
            assert rows > 64 and (each <= 8 or each >= 100), (rows, experts)


@pytest.mark.parametrize("n,k,experts", [(2048, 2560, 64), (2560, 1024, 64), (2048, 768, 128), (768, 2048, 128)])
@pytest.mark.parametrize("backward", [0, 1])
def test_more_rows_never_take_smaller_blocks(n, k, experts, backward):
    blocks = [ROWS[plan(rows, n, k, experts, backward)] for rows in range(1, 20000)]
    assert blocks == sorted(blocks) and blocks[0] == 32 and blocks[-1] == 128


@pytest.mark.parametrize("rows,n,k,experts,backward", [(40, 2048, 2560, 64, 0), (62, 2048, 2560, 64, 0), (8, 28672, 4096, 8, 0), (200, 28672, 4096, 8, 0), (130, 2048, 768, 128, 0),
                                                       (700, 2560, 2048, 32, 0), (500, 2048, 1280, 24, 1), (3000, 2048, 768, 128, 1), (760, 256, 1024, 32, 1)])
def test_calls_of_few_rows_to_an_expert(rows, n, k, experts, backward):
    """They took blocks of 128 rows, which are up to 30 % slower there, and never faster."""
    assert plan(rows, n, k, experts, backward) in (1, 2, 4, 5)


def forward(rows, n, k, experts):
    """The call with pointers that are refused once the sizes have been taken."""
    return _lib.load().kiln_w4a16_gemm_experts(None, None, None, None, None, None, rows, rows, 1, n, k, experts, 128, 0, 0, None, None)


def gradient(rows, n, k, experts):
    return _lib.load().kiln_w4a16_gemm_experts_backward(None, None, None, None, None, rows, n, k, experts, 128, 0, None)


def test_sizes_that_a_call_refuses_have_no_plan():
    for rows, n, k, experts in ((1 << 24, 1 << 17, 128, 4), (1 << 23, 1 << 17, 128, 4), (1 << 22, 1 << 17, 128, 4), (1 << 20, 1 << 17, 128, 4), (1 << 24, 1 << 14, 128, 1024)):
        assert (plan(rows, n, k, experts, 0) == -1) == (forward(rows, n, k, experts) == _lib.ERR_KERN_SHAPE)
        assert (plan(rows, 256, n, experts, 1) == -1) == (gradient(rows, 256, n, experts) == _lib.ERR_KERN_SHAPE)
    assert plan(1 << 24, 1 << 17, 128, 4, 0) == plan(1 << 24, 256, 1 << 17, 4, 1) == -1


def test_sizes_up_to_the_documented_bound_are_taken():
    for experts, columns in itertools.product((1, 4, 63, 1024), (1, 2, 3, 10, 100, 512, 4096)):
        blocks = ((1 << 24) - 9) // columns                                            # rows / 32 + experts + 1 of them
        rows = (blocks - experts - 1) * 32 + 31
        if rows * 128 <= (1 << 35) - 2048:
            assert plan(rows, 256 * columns, 128, experts, 0) >= 0 and forward(rows, 256 * columns, 128, experts) == _lib.ERR_ARGUMENT
        assert plan(rows, 256, 256 * columns, experts, 1) >= 0 and gradient(rows, 256, 256 * columns, experts) == _lib.ERR_ARGUMENT
