"""What the calls from Python on sorted rows, their products and kept activations refuse: wrong shapes, types and ranges, before anything is launched."""
import pytest
import torch

from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def refused(call, match):
    with pytest.raises(mg.MarlinGemmError, match=match):
        call()


I32 = torch.int32


def test_sort():
    of = zeros(4, 2, dtype=I32)
    refused(lambda: mg.moe_sort(of, 0), "1 to 1024 experts")
    refused(lambda: mg.moe_sort(of, 1025), "1 to 1024 experts")
    refused(lambda: mg.moe_sort(of.long(), 4), "i32")
    refused(lambda: mg.moe_sort(of[0], 4), "i32")
    refused(lambda: mg.moe_sort(zeros(4, 17, dtype=I32), 4), "top_k")
    refused(lambda: mg.moe_sort(zeros(4, 0, dtype=I32), 4), "top_k")


def test_rows():
    of = zeros(4, 2, dtype=I32)
    _, first, place = mg.moe_sort(of, 3)
    x, rows, w = zeros(4, 64), zeros(8, 64), zeros(4, 2, dtype=torch.float32)
    refused(lambda: mg.moe_gather(zeros(4, 60), first, place), "multiple of 8")
    refused(lambda: mg.moe_gather(zeros(5, 64), first, place), "bf16")
    refused(lambda: mg.moe_gather(x.float(), first, place), "bf16")
    refused(lambda: mg.moe_gather(x, first.long(), place), "first")
    refused(lambda: mg.moe_gather(x, first, place.reshape(-1)), "place")
    refused(lambda: mg.moe_gather(x, first, place, out=zeros(4, 64)), "out")
    refused(lambda: mg.moe_combine(zeros(7, 64), w, first, place), "rows")
    refused(lambda: mg.moe_combine(rows, w.double(), first, place), "weights")
    refused(lambda: mg.moe_combine(rows, None, first, place), "weights")
    refused(lambda: mg.moe_combine(rows, w[:, :1], first, place), "weights")
    refused(lambda: mg.moe_combine_backward(zeros(4, 72), rows, w, first, place), "dy")
    refused(lambda: mg.moe_combine_backward(zeros(3, 64), rows, w, first, place), "dy")
    refused(lambda: mg.moe_gather_backward(zeros(7, 64), first, place), "rows")
    both = zeros(12, 64)                                   # a result over its operand
    refused(lambda: mg.moe_gather(both[:4], first, place, out=both[3:11]), "status 4")
    refused(lambda: mg.moe_combine(both[:8], w, first, place, out=both[7:11]), "status 4")


def test_products():
    b, s = zeros(3, 16, 1024, dtype=I32), zeros(3, 2, 512, dtype=torch.float16)
    first, x, dy = zeros(4, dtype=I32), zeros(6, 256), zeros(6, 512)
    f, g = mg.marlin_w4a16_gemm_experts, mg.marlin_w4a16_gemm_experts_backward
    refused(lambda: f(x, first, b, s, 64), "groupsize")
    refused(lambda: f(x, first[:3], b, s, 128), "first")
    refused(lambda: f(x.float(), first, b, s, 128), "bf16")
    refused(lambda: f(zeros(6, 128), first, b, s, 128), "k=256")
    refused(lambda: f(x, first, b[0], s[0], 128), "3-D")
    refused(lambda: f(x, first, b[:, :, :1000], s, 128), "b_packed")
    refused(lambda: f(x, first, b, s[:, :1], 128), "scales")
    refused(lambda: f(x, first, b, s.float(), 128), "scales")
    refused(lambda: f(x, first, b, s, 128, order=zeros(11, dtype=I32), top_k=2), "order")
    refused(lambda: f(x, first, b, s, 128, order=zeros(6, dtype=I32), top_k=0), "top_k")
    refused(lambda: f(x, first, b, s, 128, out=zeros(6, 256)), "out")
    refused(lambda: f(x, first, b, s, 128, swiglu=True, out=zeros(6, 512)), "out")
    refused(lambda: g(zeros(6, 256), first, b, s, 128), "dy")
    refused(lambda: g(dy[0], first, b, s, 128), "dy")
    refused(lambda: g(dy, first.long(), b, s, 128), "first")


def test_kept_activations():
    refused(lambda: mg.swiglu_keep(zeros(4, 128)), "multiple of 128")
    refused(lambda: mg.swiglu_keep(zeros(4, 256).float()), "bf16")
    h, whole, exponents = mg.swiglu_keep(zeros(4, 512))
    assert exponents.shape == (4, 8, 2)
    refused(lambda: mg.swiglu_keep_backward(zeros(4, 128), whole, exponents), "whole")
    refused(lambda: mg.swiglu_keep_backward(zeros(3, 256), whole, exponents), "whole")
    refused(lambda: mg.swiglu_keep_backward(h, whole.to(torch.int32), exponents), "whole")
    refused(lambda: mg.swiglu_keep_backward(h, whole, exponents[:, :4]), "exponents")
    refused(lambda: mg.swiglu_keep_backward(h.float(), whole, exponents), "bf16")
