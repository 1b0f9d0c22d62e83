"""Sorted rows, their products and kept activations where offsets pass 31 and 32 bits: the last rows and the last experts against 64 bits."""
import math

import pytest
import torch

from tests.expert_packs import weight
from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu
HALF, F32 = 2.0 ** -8, 2.0 ** -24


def bf16(*shape):
    return torch.randn(shape, dtype=torch.bfloat16, device="cuda")


def near(got, want, off):
    assert ((got.double() - want).abs() <= HALF * want.abs() + off).all()


def products(rows, counts, k, n, checked):
    """Experts with `counts` rows; `checked`: (expert, its rows)."""
    torch.manual_seed(rows)
    experts = len(counts)
    first = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    b = torch.empty((experts, k // 16, 2 * n), dtype=torch.int32, device="cuda").random_(-2 ** 31, 2 ** 31)
    s = (torch.rand((experts, k // 128, n), device="cuda") * 0.01 + 0.005).half()
    x, dy = bf16(rows, k), bf16(rows, n)
    y, dx = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128), mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, 128)
    for e, i, j in checked:
        w = weight(b[e], s[e])
        # partial sums of at most 144 times a random sum of 128 values, each of k additions off by 2^-24 of it, at random; four times that
        near(y[i:j], x[i:j].double() @ w, 4 * F32 * math.sqrt(k) * 144 * math.sqrt(128) * 5 * 0.015)
        w = w.float().bfloat16().double()
        near(dx[i:j], dy[i:j].double() @ w.t(), 4 * math.sqrt(n) * F32 * (dy[i:j].double().abs() @ w.abs().t()))
    assert not y[int(first[-1]):].any() and not dx[int(first[-1]):].any()


def test_packs_of_more_than_four_gigabytes():
    counts = [0] * 1024
    counts[0], counts[900], counts[1022], counts[1023] = 3, 64, 200, 40
    products(310, counts, 4096, 2304, [(0, 0, 3), (900, 3, 67), (1022, 67, 267), (1023, 267, 307)])


def test_rows_of_more_than_four_gigabytes():
    rows = 1100000
    products(rows, [500000, rows - 500100], 128, 2048, [(0, 0, 200), (0, 499900, 500000), (1, rows - 400, rows - 100)])


def test_sorted_rows_of_more_than_four_gigabytes():
    torch.manual_seed(0)
    m, top, experts, width = 270000, 8, 64, 1032
    of = torch.randint(0, experts, (m, top), dtype=torch.int32, device="cuda")
    order, first, place = mg.moe_sort(of, experts)
    assert int(first[-1]) == m * top and torch.equal(order[place.reshape(-1).long()], torch.arange(m * top, dtype=torch.int32, device="cuda"))
    x, weights = bf16(m, width), torch.rand((m, top), device="cuda")
    rows = mg.moe_gather(x, first, place)
    some = torch.cat((torch.arange(0, 100), torch.arange(m - 100, m))).cuda()
    at = place[some].long()
    assert torch.equal(rows[at], x[some][:, None].expand(-1, top, -1))
    rows.normal_()
    terms, w = rows[at].double(), weights[some].double()
    near(mg.moe_combine(rows, weights, first, place)[some], (terms * w[..., None]).sum(1), 2 * (top + 1) * F32 * (terms * w[..., None]).abs().sum(1))
    d_rows, d_weights = mg.moe_combine_backward(x, rows, weights, first, place)
    want = x[some].double()[:, None] * w[..., None]
    near(d_rows[at], want, F32 * want.abs())
    products = x[some].double()[:, None] * terms
    assert ((d_weights[some].double() - products.sum(2)).abs() <= width * F32 * products.abs().sum(2)).all()


def test_kept_activations_of_more_than_four_gigabytes():
    torch.manual_seed(0)
    m, n = 1100000, 1024
    gate_up, dh = bf16(m, 2 * n), bf16(m, n)
    h, whole, exponents = mg.swiglu_keep(gate_up)
    d, again = mg.swiglu_keep_backward(dh, whole, exponents, recompute=True)
    for i, j in ((0, 50), (m - 50, m)):         # the same rows alone
        few = mg.swiglu_keep(gate_up[i:j])
        assert all(torch.equal(a[i:j], f) for a, f in zip((h, whole, exponents), few))
        assert all(torch.equal(a[i:j], f) for a, f in zip((d, again), mg.swiglu_keep_backward(dh[i:j], few[1], few[2], recompute=True)))
