"""What the C entry points of sorted rows, their products and kept activations refuse, before anything is launched (no GPU is touched), and what the
calls from Python do.  CPU only: the pointers handed over are never followed."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, marlin_gemm as mg

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)
ODD4 = ctypes.c_void_p((1 << 20) + 2)
R = [ctypes.c_void_p(i << 40) for i in range(1, 5)]      # results, which share no memory with operands


def at(base, bytes):
    return ctypes.c_void_p(base.value + bytes)


def sort(of=P, m=600, top=4, experts=8, order=R[0], first=R[1], place=R[2], scratch=R[3]):
    return _lib.load().kiln_w4a16_moe_sort(of, m, top, experts, order, first, place, 0, None, scratch)


def gather(x=P, first=P, place=P, rows=R[0], m=4, top=2, experts=8, width=64):
    return _lib.load().kiln_w4a16_moe_gather(x, first, place, rows, m, top, experts, width, 0, None)


def combine(rows=P, weights=P, first=P, place=P, y=R[0], m=4, top=2, experts=8, width=64):
    return _lib.load().kiln_w4a16_moe_combine(rows, weights, first, place, y, m, top, experts, width, 0, None)


def combine_backward(dy=P, rows=P, weights=P, first=P, place=P, d_rows=R[0], d_weights=R[1], m=4, top=2, experts=8, width=64):
    return _lib.load().kiln_w4a16_moe_combine_backward(dy, rows, weights, first, place, d_rows, d_weights, m, top, experts, width, 0, None)


def experts(x=P, first=P, order=None, b=P, s=P, y=R[0], rows=8, x_rows=8, top=1, n=512, k=256, count=4, g=128, swiglu=0, scratch=R[3]):
    return _lib.load().kiln_w4a16_gemm_experts(x, first, order, b, s, y, rows, x_rows, top, n, k, count, g, swiglu, 0, None, scratch)


def experts_backward(dy=P, first=P, b=P, s=P, dx=R[0], rows=8, n=512, k=256, count=4, g=128):
    return _lib.load().kiln_w4a16_gemm_experts_backward(dy, first, b, s, dx, rows, n, k, count, g, 0, None)


def keep(gate_up=P, h=R[0], whole=R[1], exponents=R[2], m=4, n=128):
    return _lib.load().kiln_w4a16_swiglu_keep(gate_up, h, whole, exponents, m, n, 0, None)


def keep_backward(dh=P, whole=P, exponents=P, d=R[0], h=R[1], m=4, n=128):
    return _lib.load().kiln_w4a16_swiglu_keep_backward(dh, whole, exponents, d, h, m, n, 0, None)


def refuses(call, shape, kernel, argument):
    for status, cases in ((_lib.ERR_PROB_SHAPE, shape), (_lib.ERR_KERN_SHAPE, kernel), (_lib.ERR_ARGUMENT, argument)):
        for kw in cases:
            assert call(**kw) == status, kw


ROUTED = (dict(top=0), dict(top=17), dict(experts=0), dict(experts=1025), dict(m=1 << 28, top=8), dict(m=2 ** 31 - 1, top=2))


def test_sort_refuses():
    refuses(sort, (dict(m=-1),), ROUTED,
            (*(dict([(name, bad)]) for name in ("of", "order", "first", "place", "scratch") for bad in (None, ODD4)),
             dict(order=P), dict(place=P), dict(first=P), dict(place=R[0]), dict(first=at(R[0], 600 * 4 * 4 - 4)), dict(first=at(R[2], 16)), dict(scratch=P), dict(scratch=R[0])))


def test_rows_refuse():
    shape = (dict(m=-1), dict(width=0), dict(width=60), dict(width=-8))
    for call, pointers, plain in ((gather, ("x", "rows"), ("first", "place")), (combine, ("rows", "y"), ("first", "place")),
                                  (combine_backward, ("dy", "rows", "d_rows"), ("first", "place", "weights", "d_weights"))):
        refuses(call, shape, ROUTED, (*(dict([(name, bad)]) for name in pointers for bad in (None, ODD)), *(dict([(name, None)]) for name in plain)))
    refuses(gather, (), (), (dict(place=R[0]), dict(first=R[0]), dict(rows=P), dict(rows=at(P, 4 * 64 * 2 - 16)), dict(x=at(R[0], 4 * 2 * 64 * 2 - 16))))
    refuses(combine, (), (), (dict(weights=R[0]), dict(place=R[0]), dict(weights=ODD4), dict(y=P), dict(rows=at(R[0], 16))))
    refuses(combine_backward, (), (), (dict(d_rows=P), dict(dy=at(R[0], 16)), dict(d_weights=P)))


def test_products_refuse():
    shape = (dict(n=300), dict(k=200), dict(g=64), dict(n=0), dict(k=0), dict(rows=-1))
    refuses(experts, shape, (dict(count=0), dict(count=1025), dict(x_rows=7), dict(order=P, x_rows=8, top=2), dict(order=P, x_rows=4, top=0), dict(x_rows=-1, rows=0)),
            (*(dict([(name, bad)]) for name in ("x", "b", "s", "y", "scratch") for bad in (None, ODD)), dict(first=None), dict(first=ODD4), dict(y=P), dict(x=at(R[0], 8 * 512 * 2 - 16)),
             dict(b=at(R[0], 16)), dict(s=R[0]), dict(first=R[0]), dict(order=R[0], x_rows=4, top=2), dict(scratch=R[0]), dict(order=ODD4, x_rows=4, top=2)))
    refuses(experts_backward, shape, (dict(count=0), dict(count=1025), dict(rows=2 ** 31 - 1, n=1 << 20)),
            (*(dict([(name, bad)]) for name in ("dy", "b", "s", "dx") for bad in (None, ODD)), dict(first=None), dict(dx=P), dict(dy=at(R[0], 16))))


def test_kept_activations_refuse():
    shape = (dict(m=-1), dict(n=0), dict(n=64), dict(n=192), dict(n=-128), dict(n=1 << 30))
    refuses(keep, shape, (), (*(dict([(name, bad)]) for name in ("gate_up", "h", "whole") for bad in (None, ODD)), dict(exponents=None), dict(exponents=at(R[2], 1)),
                              dict(h=P), dict(whole=P), dict(exponents=P), dict(whole=R[0]), dict(exponents=at(R[1], 16))))
    refuses(keep_backward, shape, (), (*(dict([(name, bad)]) for name in ("dh", "whole", "d") for bad in (None, ODD)), dict(exponents=None), dict(exponents=at(P, 1)),
                                       dict(h=ODD), dict(d=P), dict(h=P), dict(h=R[0])))


def test_calls_without_work_are_no_errors():
    assert gather(m=0) == combine(m=0) == combine_backward(m=0) == experts(rows=0, x_rows=0) == experts_backward(rows=0) == keep(m=0) == keep_backward(m=0) == _lib.OK


def test_scratch():
    L = _lib.load()
    assert L.kiln_w4a16_moe_sort_scratch_bytes(256, 8, 64) == 0 and L.kiln_w4a16_moe_sort_scratch_bytes(0, 8, 64) == 0
    for m, top, count in ((257, 8, 64), (8192, 8, 128), (1 << 26, 16, 1024)):
        assert L.kiln_w4a16_moe_sort_scratch_bytes(m, top, count) % (4 * (count + 1)) == 0
        assert 2 <= L.kiln_w4a16_moe_sort_scratch_bytes(m, top, count) // (4 * (count + 1)) <= 256
    assert L.kiln_w4a16_gemm_experts_scratch_bytes(1000, 2560) >= 1000 * 20 * 4 and L.kiln_w4a16_gemm_experts_scratch_bytes(0, 2560) == 256


def test_plans():
    plan = _lib.load().kiln_w4a16_debug_experts_plan
    assert plan(1, 2048, 2560, 8, 0, 256) == 0 and plan(16384, 2048, 2560, 64, 0, 256) == 3 == plan(16384, 2048, 2560, 64, 1, 256)
    assert plan(768, 2048, 2560, 64, 0, 256) in (1, 2, 3) and plan(0, 2048, 2560, 8, 0, 256) == -1 == plan(8, 2000, 2560, 8, 0, 256)
    for backward in (0, 1):                     # more rows never take smaller blocks again
        kinds = [plan(rows, 2048, 2560, 64, backward, 256) for rows in range(1, 40000, 37)]
        assert set(kinds) <= {0, 1, 2, 3, 4, 5} and kinds[-1] == 3


def test_calls_on_tensors_of_the_host_are_refused():
    of, x = torch.zeros((2, 3), dtype=torch.int32), torch.zeros((2, 256), dtype=torch.bfloat16)
    rows, weights, first = torch.zeros((6, 256), dtype=torch.bfloat16), torch.zeros((2, 3)), torch.zeros(5, dtype=torch.int32)
    b, s = torch.zeros((4, 16, 512), dtype=torch.int32), torch.zeros((4, 2, 256), dtype=torch.float16)
    whole, exponents = torch.zeros((2, 256), dtype=torch.int8), torch.zeros((2, 4, 2), dtype=torch.uint8)
    for call in (lambda: mg.moe_sort(of, 4), lambda: mg.moe_gather(x, first, of), lambda: mg.moe_gather_backward(rows, first, of),
                 lambda: mg.moe_combine(rows, weights, first, of), lambda: mg.moe_combine_backward(x, rows, weights, first, of),
                 lambda: mg.marlin_w4a16_gemm_experts(x, first, b, s, 128), lambda: mg.marlin_w4a16_gemm_experts_backward(x, first, b, s, 128),
                 lambda: mg.swiglu_keep(x), lambda: mg.swiglu_keep_backward(x[:, :128], whole, exponents)):
        with pytest.raises(mg.MarlinGemmError, match="on CUDA"):
            call()


def test_sizes_that_no_launch_has_work_items_for_are_refused():
    most = (1 << 24) - 1                        # blocks of 256
    assert gather(m=1 << 24, top=1, width=2048) == combine(m=1 << 24, top=1, width=2048) == _lib.ERR_KERN_SHAPE
    assert combine_backward(m=1 << 26, top=1, width=64) == combine_backward(m=1 << 23, top=8, width=64) == _lib.ERR_KERN_SHAPE
    assert keep(m=1 << 24, n=2048) == keep_backward(m=1 << 24, n=2048) == _lib.ERR_KERN_SHAPE
    assert experts(rows=1 << 24, x_rows=1 << 24, k=2048) == _lib.ERR_KERN_SHAPE                     # the rows' sums
    assert experts(rows=1 << 24, x_rows=1 << 24, k=128, n=1 << 17) == experts_backward(rows=1 << 24, k=1 << 17, n=256) == _lib.ERR_KERN_SHAPE
    # one less is asked for its pointers
    assert gather(m=most, top=1, width=2048, x=None) == combine(m=most, top=1, width=2048, y=None) == _lib.ERR_ARGUMENT
    assert combine_backward(m=4 * most, top=1, width=64, dy=None) == combine_backward(m=most // 2, top=8, width=64, dy=None) == _lib.ERR_ARGUMENT
    assert keep(m=most, n=2048, h=None) == experts(rows=most, x_rows=most, k=2048, x=None) == _lib.ERR_ARGUMENT
