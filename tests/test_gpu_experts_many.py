"""Products of sorted rows with their experts' packs, and the gradient of the rows, against 64 bits (parity unpinned: the reference's model
family is dense; an expert's weight is what its packed GEMM multiplies with, crates/kiln-marlin-gemm/src/lib.rs:415-425)."""
import math

import pytest
import torch

from tests.expert_packs import choice, packs, silu_times, sorted_by_hand, weight
from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu
HALF, F32 = 2.0 ** -8, 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bf16(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).bfloat16()


def error_of_a_sum(x, s, k):
    """The sums run over x * (136 + d) in units of the scale with the surplus taken off first: a partial sum is at most of the size of 144 times a
    random sum of 128 values, and each of k additions is off by 2^-24 of it, at random; four times that."""
    return 4 * F32 * math.sqrt(k) * 144 * math.sqrt(128) * float(x.double().abs().max()) * float(s.double().max())


def check_forward(x, first, b, s, g, swiglu=False, order=None, top_k=1):
    y = mg.marlin_w4a16_gemm_experts(x, first, b, s, g, order=order, top_k=top_k, swiglu=swiglu)
    rows = x[(order.long() // top_k)] if order is not None else x
    bounds, k = first.tolist(), x.shape[1]
    assert y.shape == (len(rows), s.shape[2] // (2 if swiglu else 1)) and y.dtype == torch.bfloat16
    assert not y[bounds[-1]:].any()
    for e in range(len(b)):
        i, j = bounds[e], bounds[e + 1]
        if i == j:
            continue
        want = rows[i:j].double() @ weight(b[e], s[e])
        off = error_of_a_sum(rows[i:j], s[e], k)
        if swiglu:
            both = want.reshape(len(want), -1, 2, 8)
            gate, up = both[:, :, 0].reshape(len(want), -1).abs(), both[:, :, 1].reshape(len(want), -1).abs()
            want = silu_times(want)
            off = off * (1.1 * up + gate + off) + 2.0 ** -18 * want.abs()
        assert ((y[i:j].double() - want).abs() <= HALF * want.abs() + off).all(), (e, i, j)


def check_backward(dy, first, b, s, g):
    dx = mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, g)
    bounds = first.tolist()
    assert dx.shape == (len(dy), b.shape[1] * 16) and not dx[bounds[-1]:].any()
    for e in range(len(b)):
        i, j = bounds[e], bounds[e + 1]
        if i == j:
            continue
        w = weight(b[e], s[e]).float().bfloat16().double()   # what the product is documented to take
        want, size = dy[i:j].double() @ w.t(), dy[i:j].double().abs() @ w.abs().t()
        assert ((dx[i:j].double() - want).abs() <= HALF * want.abs() + 4 * math.sqrt(dy.shape[1]) * F32 * size).all(), (e, i, j)


def first_of(counts):
    return torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


# rows to each expert: none, one, around the tiles' 32, 64 and 128 and beyond; the last number: rows of no expert
COUNTS = [[1, 0], [0, 0, 1, 0], [31, 32, 33, 0, 1, 2], [64, 63, 65, 3], [128, 127, 129, 5], [0, 300, 0, 17, 9], [0, 0, 40], [500, 0], [7] * 40 + [0]]


@pytest.mark.parametrize("k,n,g", [(128, 256, 128), (384, 512, 128), (256, 768, -1), (1152, 256, 128)])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:6])))
def test_every_size_of_expert(counts, k, n, g):
    r = gen(sum(counts) + k + n)
    first = first_of(counts[:-1])
    rows = sum(counts)
    b, s = packs(r, len(counts) - 1, k, n, g)
    x, dy = bf16(r, rows, k), bf16(r, rows, n)
    for swiglu in (False, True):
        check_forward(x, first, b, s, g, swiglu)
    check_backward(dy, first, b, s, g)


@pytest.mark.parametrize("m,top,experts,away,k,n,g", [(1, 8, 64, 0, 512, 512, 128), (96, 8, 64, 0, 640, 256, 128), (100, 4, 16, 4, 256, 512, -1), (700, 3, 7, 1, 384, 1024, 128),
                                                      (9, 16, 1024, 24, 128, 256, 128), (2000, 2, 8, 0, 256, 256, 128)])
def test_straight_from_the_tokens(m, top, experts, away, k, n, g):
    r = gen(m + k)
    of = choice(r, m, top, experts, away)
    order, first, place = mg.moe_sort(of, experts)
    b, s = packs(r, experts, k, n, g)
    x = bf16(r, m, k)
    for swiglu in (False, True):
        check_forward(x, first, b, s, g, swiglu, order, top)
        gathered = mg.marlin_w4a16_gemm_experts(mg.moe_gather(x, first, place), first, b, s, g, swiglu=swiglu)
        assert torch.equal(mg.marlin_w4a16_gemm_experts(x, first, b, s, g, order=order, top_k=top, swiglu=swiglu), gathered)


@pytest.mark.parametrize("rows,experts,k,n", [(3000, 2, 2560, 2048), (700, 32, 2048, 2560), (100, 64, 2560, 2048), (4096, 8, 1024, 2560)])
def test_model_sizes(rows, experts, k, n):
    r = gen(rows)
    cuts = sorted(torch.randint(0, rows, (experts - 1,), generator=torch.Generator().manual_seed(rows)).tolist())
    first = torch.tensor([0] + cuts + [rows], dtype=torch.int32, device="cuda")
    b, s = packs(r, experts, k, n, 128)
    check_forward(bf16(r, rows, k), first, b, s, 128, swiglu=True)
    check_backward(bf16(r, rows, n), first, b, s, 128)


def test_one_expert_is_the_plain_product():
    r = gen(1)
    b, s = packs(r, 1, 512, 512, 128)
    x = bf16(r, 200, 512)
    first = first_of([200])
    y, plain = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128).double(), mg.marlin_w4a16_gemm(x, b[0], s[0], 128).double()
    assert ((y - plain).abs() <= 2 * HALF * plain.abs() + 2 * error_of_a_sum(x, s[0], 512)).all()


def test_scales_of_zero_small_and_large_and_codes_of_one_kind():
    r = gen(8)
    b, s = packs(r, 3, 512, 256, 128)
    s[0, 1], s[0, 3] = 0.0, 6e-8
    s[1, 0], s[1, 1:] = 100.0, 1e-3
    s[2, :, ::3] = 0.0
    b[2, :, : 128] = 0                        # -8 throughout
    first = first_of([40, 1, 77])
    x, dy = bf16(r, 118, 512), bf16(r, 118, 256)
    y = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128)
    for e, (i, j) in enumerate(((0, 40), (40, 41), (41, 118))):
        w = weight(b[e], s[e])
        want = x[i:j].double() @ w
        # a column's own scales: a group's sums are rounded in units of its own, and of the largest scale beside it when that comes later
        per_column = s[e].double().reshape(16, 4, 16).permute(1, 0, 2).reshape(4, 256).amax(0)
        off = 4 * F32 * math.sqrt(512) * 144 * math.sqrt(128) * float(x.double().abs().max()) * per_column
        assert ((y[i:j].double() - want).abs() <= HALF * want.abs() + off + 2.0 ** -26).all()   # (a zero scale is taken as 2^-40: 1088 of its units at most)
    check_backward(dy, first, b, s, 128)


def test_rows_without_numbers_stay_alone():
    r = gen(5)
    b, s = packs(r, 2, 256, 256, 128)
    first = first_of([50, 30])
    x, dy = bf16(r, 80, 256), bf16(r, 80, 256)
    for t, f in ((x, mg.marlin_w4a16_gemm_experts), (dy, mg.marlin_w4a16_gemm_experts_backward)):
        clean = f(t, first, b, s, 128)
        bad = t.clone()
        bad[13, 100], bad[60, 7] = float("nan"), float("inf")
        got = f(bad, first, b, s, 128)
        others = [i for i in range(80) if i not in (13, 60)]
        assert torch.equal(got[others], clean[others]) and torch.isnan(got[13]).all() and not torch.isfinite(got[60]).any()


def test_gradient_is_the_transpose():
    """<dy, experts(x)> = <experts_backward(dy), x>: the map is linear in its rows.  Weights that are bf16 values and small whole numbers as rows: every
    sum is exact in f32, and the results are rounded once."""
    r = gen(6)
    b, s = packs(r, 4, 256, 256, -1)
    s.fill_(1.0)
    first = first_of([33, 0, 70, 5])
    x, dy = (torch.randint(-2, 3, (108, 256), device="cuda", generator=r).bfloat16() for _ in range(2))
    y, dx = mg.marlin_w4a16_gemm_experts(x, first, b, s, -1).double(), mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, -1).double()
    left, right = (y * dy.double()).sum(), (dx * x.double()).sum()
    assert abs(left - right) <= HALF * ((y * dy.double()).abs().sum() + (dx * x.double()).abs().sum())
    for e, (i, j) in enumerate(((0, 33), (33, 33), (33, 103), (103, 108))):
        w = weight(b[e], s[e])
        assert torch.equal(y[i:j], (x[i:j].double() @ w).float().bfloat16().double())
        assert torch.equal(dx[i:j], (dy[i:j].double() @ w.t()).float().bfloat16().double())


def test_results_go_where_they_are_asked_for_and_operands_may_be_strided():
    r = gen(12)
    b, s = packs(r, 3, 256, 256, 128)
    first = first_of([5, 40, 9])
    x, dy = bf16(r, 60, 512)[:, ::2], bf16(r, 256, 60).t()
    out = torch.full((60, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    y = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128, out=out)
    assert y is out and torch.equal(y, mg.marlin_w4a16_gemm_experts(x.contiguous(), first, b, s, 128)) and not y[54:].any()
    assert torch.equal(mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, 128), mg.marlin_w4a16_gemm_experts_backward(dy.contiguous(), first, b, s, 128))
    assert mg.marlin_w4a16_gemm_experts(x[:0], first_of([0, 0, 0]), b, s, 128).shape == (0, 256)
    assert mg.marlin_w4a16_gemm_experts_backward(dy[:0], first_of([0, 0, 0]), b, s, 128).shape == (0, 256)


def test_the_same_bits_every_time():
    r = gen(14)
    of = choice(r, 500, 4, 16, 2)
    order, first, _ = mg.moe_sort(of, 16)
    assert all(torch.equal(a, b) for a, b in zip((order, first), sorted_by_hand(of, 16)[:2]))
    b, s = packs(r, 16, 512, 512, 128)
    x, dy = bf16(r, 500, 512), bf16(r, 2000, 512)
    y, dx = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128, order=order, top_k=4), mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, 128)
    for _ in range(10):
        assert torch.equal(y, mg.marlin_w4a16_gemm_experts(x, first, b, s, 128, order=order, top_k=4))
        assert torch.equal(dx, mg.marlin_w4a16_gemm_experts_backward(dy, first, b, s, 128))


@pytest.mark.parametrize("rows,k,n", [(5, 2560, 512), (90, 1152, 512), (300, 2560, 256), (600, 128, 256), (3000, 512, 1024)])
def test_rows_of_one_sign(rows, k, n):
    """The surplus of 136 times a row's sum is the largest there is: a partial sum is at most 144 * 128 times the largest value, each of k additions off by 2^-24
    of it, at random, and the row's own sum, 64 additions of pairs off by three times as much, times 136; four times that."""
    r = gen(rows)
    first = first_of([rows // 2, 0, rows - rows // 2])
    b, s = packs(r, 3, k, n, 128)
    x = (3 + torch.rand((rows, k), device="cuda", generator=r)).bfloat16()
    x[1::2] *= -1
    y, bounds = mg.marlin_w4a16_gemm_experts(x, first, b, s, 128), first.tolist()
    for e in (0, 2):
        i, j = bounds[e], bounds[e + 1]
        off = 4 * F32 * (math.sqrt(k) * 144 + 3 * math.sqrt(64) * 136) * 128 * 4 * float(s[e].double().max())
        want = x[i:j].double() @ weight(b[e], s[e])
        assert ((y[i:j].double() - want).abs() <= HALF * want.abs() + off).all(), e


@pytest.mark.parametrize("experts", [62, 63, 64, 200, 1024])
def test_more_experts_than_lanes(experts):
    r = gen(experts)
    counts = torch.randint(0, 5, (experts,), device="cuda", generator=r)
    counts[experts // 2], counts[experts - 1] = 150, 40
    first = first_of(counts.tolist())
    rows = int(first[-1]) + 33
    b, s = packs(r, experts, 128, 256, 128)
    x, dy = bf16(r, rows, 128), bf16(r, rows, 256)
    check_forward(x, first, b, s, 128)
    check_backward(dy, first, b, s, 128)
