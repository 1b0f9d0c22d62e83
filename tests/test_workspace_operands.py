"""Operands that a launch writes and reads itself begin on a cache line wherever in memory the caller's workspace lies, and end inside the
size that the library asks for.  CPU only: the workspace's address is never followed."""
import ctypes

import pytest

from kiln_amd import _lib

SIZES = [(1, 256, 128), (16, 2560, 9216), (16, 18432, 2560), (33, 2560, 2560), (77, 2560, 9216), (200, 5120, 13824), (515, 10240, 640), (777, 9216, 2560),
         (1031, 6144, 1152), (1503, 5888, 2176), (2045, 4096, 1280), (2048, 18432, 2560), (8192, 2560, 9216)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("rank", [0, 8, 40])
def test_operands_are_on_lines_inside_the_workspace(m, n, k, rank):
    L = _lib.load()
    size, prefix = L.kiln_w4a16_workspace_bytes(m, n, k), L.kiln_w4a16_workspace_zeroed_bytes()
    for base in range(1 << 30, (1 << 30) + 256, 16):
        out = (ctypes.c_size_t * 6)()
        assert L.kiln_w4a16_debug_workspace_operands(m, n, k, 256, rank, base, out) == 0
        *operands, end, slices, apart = out
        assert any(operands) and end <= base + size, base
        for at in operands:
            assert at == 0 or (at % 128 == 0 and base + prefix <= at <= end), (base, list(out))
        assert operands[2] + slices * apart <= end


def test_slices_of_a_projection_inside_the_launch_are_lines_apart():
    """... for every count of rows of a launch whose runs of 64 rows wait for their own rows of it alone."""
    L, seen = _lib.load(), 0
    for k, n in ((2560, 2560), (9216, 2560), (2560, 18432), (4096, 14336)):
        for m in range(17, 257):
            for rank in (8, 16, 24, 32, 40, 64):
                out = (ctypes.c_size_t * 6)()
                assert L.kiln_w4a16_debug_workspace_operands(m, n, k, 256, rank, 1 << 30, out) == 0
                slices, apart = out[4:]
                assert apart % 128 == 0 and apart >= slices and (slices == 0 or apart >= 32 * m), (m, n, k, rank)
                assert out[2] + slices * apart <= out[3]
                seen += slices > 1 and m > 64
    assert seen > 1000


def test_the_query_refuses():
    out = (ctypes.c_size_t * 6)()
    for m, n, k in ((0, 256, 128), (1, 128, 128), (1, 256, 64), (1, 300, 128)):
        assert _lib.load().kiln_w4a16_debug_workspace_operands(m, n, k, 256, 0, 1 << 30, out) == 1


@pytest.mark.parametrize("m", range(6445, 6454))
def test_row_sums_of_a_launch_in_front_take_their_rows_alone(m):
    """... which is what the static array has to hold: 6451 rows of 5120 -> 5120 fill it."""
    L, out = _lib.load(), (ctypes.c_size_t * 6)()
    assert L.kiln_w4a16_debug_prefill_rowsum_producers(m, 5120, 5120, 256) <= 0
    assert L.kiln_w4a16_debug_workspace_operands(m, 5120, 5120, 256, 0, 1 << 30, out) == 0
    assert (out[3] - (1 << 30) <= _lib.STATIC_SCRATCH_BYTES) == (m <= 6451)


def test_plain_calls_need_no_more_than_their_row_sums_and_partial_tiles():
    L, out = _lib.load(), (ctypes.c_size_t * 6)()
    for m, n, k in SIZES + [(m, n, k) for m in range(257, 4200, 131) for n, k in ((2560, 9216), (5120, 5120), (18432, 2560))]:
        assert L.kiln_w4a16_debug_workspace_operands(m, n, k, 256, 0, 1 << 30, out) == 0
        if out[0]:
            rows = -(-m // 8) * 8 if L.kiln_w4a16_debug_prefill_rowsum_producers(m, n, k, 256) > 0 else m
            assert out[1] <= out[0] and out[3] == out[0] + rows * (k // 128) * 16, (m, n, k)
