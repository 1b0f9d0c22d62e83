"""Calls on a bank whose contraction is longer than any model's here: what they write stays inside the scratch that the library asks for, and
the rows are the formula's."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, marlin_gemm
from tests.test_gpu_bank import check_forward, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", [
    (4, 32896, 256, 128, 4, 64, "any"), (1, 32896, 512, -1, 1, 16, "one"), (4, 43008, 256, 128, 2, 16, "runs"), (3, 75392, 256, 128, 3, 24, "any"),
    (16, 32896, 256, 128, 5, 8, "any"), (40, 33792, 256, -1, 3, 40, "any")])
def test_nothing_behind_the_scratch_is_written(m, k, n, g, count, rank, pattern):
    L, p = _lib.load(), problem(m, k, n, g, count, rank, pattern)
    size = L.kiln_w4a16_gemm_bank_scratch_bytes(m, n, k, count, rank)
    scratch = torch.full((size + 65536,), 0xA5, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    ws = marlin_gemm._workspace(p["x"].device, stream, L.kiln_w4a16_workspace_bytes(m, n, k))
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    bank = _lib.AdapterBank(p["a_"].data_ptr(), p["b_"].data_ptr(), p["sc"].data_ptr(), count, rank)
    assert L.kiln_w4a16_gemm_bank(p["x"].data_ptr(), p["b"].data_ptr(), y.data_ptr(), p["s"].data_ptr(), m, n, k, ws.data_ptr(), g, 0, stream,
                                  ctypes.byref(bank), p["of"].data_ptr(), scratch.data_ptr()) == _lib.OK
    check_forward(p, y)
    assert bool((scratch[size:] == 0xA5).all())
