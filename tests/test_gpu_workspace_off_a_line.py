"""A workspace on any 16-byte boundary: the same bits as one on a cache line, call after call on two inputs in turn, and nothing behind the
size that the library asks for."""
import ctypes

import pytest
import torch

from kiln_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [0, 16])
@pytest.mark.parametrize("m,k,n", [(9, 9216, 2560), (70, 2560, 2560), (150, 2560, 5120), (515, 640, 10240), (777, 2560, 9216), (1503, 2176, 5888)])
@pytest.mark.parametrize("off", [16, 112])
def test_same_bits_as_on_a_line(m, k, n, rank, off):
    L = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    b = torch.randint(-2**31, 2**31, (k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    s = ((torch.rand(k // 128, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    x = [(torch.randn(m, k, device="cuda", generator=gen) + shift).bfloat16() for shift in (0.0, 40.0)]
    a_, b_ = (torch.randn(shape, device="cuda", generator=gen).bfloat16() for shape in ((16, k), (n, 16)))
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    size, prefix, stream = L.kiln_w4a16_workspace_bytes(m, n, k), L.kiln_w4a16_workspace_zeroed_bytes(), torch.cuda.current_stream().cuda_stream
    ranks, scales = (ctypes.c_int * 1)(16), (ctypes.c_float * 1)(0.5)

    def workspace(at):
        room = torch.full((size + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        first = -room.data_ptr() % 128 + at
        room[first:first + prefix] = 0
        return room, first

    def call(x, ws):
        room, first = ws
        args = (x.data_ptr(), b.data_ptr(), y.data_ptr(), s.data_ptr(), m, n, k, room.data_ptr() + first, 128, 0, stream)
        rc = L.kiln_w4a16_gemm_lora(*args, a_.data_ptr(), b_.data_ptr(), 16, 1, ranks, scales) if rank else L.kiln_marlin_w4a16_gemm(*args, -1, -1, -1, 16)
        assert rc == _lib.OK
        return y.view(torch.int16).clone()

    line, odd = workspace(0), workspace(off)
    want = [call(x_, line) for x_ in x]
    for i in range(8):
        assert torch.equal(call(x[i % 2], odd), want[i % 2]), i
    room, first = odd
    assert bool((room[:first] == 0xA5).all()) and bool((room[first + size:] == 0xA5).all())


def test_the_static_array_takes_the_rows_that_fill_it():
    L, m, k, n = _lib.load(), 6451, 5120, 5120
    gen = torch.Generator(device="cuda").manual_seed(5)
    b = torch.randint(-2**31, 2**31, (k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    s = ((torch.rand(k // 128, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    x = torch.randn(m, k, device="cuda", generator=gen).bfloat16()
    y, z = (torch.zeros(m, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ws, stream = torch.zeros(L.kiln_w4a16_workspace_bytes(m, n, k), dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
    assert L.kiln_marlin_w4a16_gemm(x.data_ptr(), b.data_ptr(), y.data_ptr(), s.data_ptr(), m, n, k, ws.data_ptr(), 128, 0, stream, -1, -1, -1, 16) == _lib.OK
    for _ in range(2):
        assert L.kiln_marlin_w4a16_gemm_static_scratch(x.data_ptr(), b.data_ptr(), z.data_ptr(), s.data_ptr(), m, n, k, 128, 0, stream) == _lib.OK
    assert bool(y.any()) and torch.equal(y.view(torch.int16), z.view(torch.int16))
    assert L.kiln_marlin_w4a16_gemm_static_scratch(x.data_ptr(), b.data_ptr(), z.data_ptr(), s.data_ptr(), m + 1, n, k, 128, 0, stream) == _lib.ERR_SCRATCH
