"""moe_sort, moe_gather and moe_combine with their gradients, against their definitions in 64 bits (parity unpinned: the reference's model
family is dense).  A rounding to bf16 is off by at most 2^-8 of the value; sums in f32 of `count` terms by count * 2^-24 of the terms' sum."""
import pytest
import torch

from tests.expert_packs import choice, sorted_by_hand
from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu
HALF, F32 = 2.0 ** -8, 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


@pytest.mark.parametrize("m,top,experts,away", [(1, 1, 1, 0), (1, 8, 64, 0), (7, 3, 5, 2), (64, 16, 1024, 100), (300, 4, 32, 8), (256, 8, 64, 0), (257, 8, 64, 64),
                                                (2048, 2, 3, 1), (1025, 16, 17, 0), (8192, 8, 128, 16), (5000, 13, 1024, 3)])
def test_sort(m, top, experts, away):
    of = choice(gen(m), m, top, experts, away)
    for got, want in zip(mg.moe_sort(of, experts), sorted_by_hand(of, experts)):
        assert got.dtype == torch.int32 and torch.equal(got, want)


def test_sort_of_one_expert_of_none_and_of_odd_ids():
    for of in (torch.full((700, 4), 3), torch.full((700, 4), -1), torch.full((33, 2), 9), torch.tensor([[2 ** 31 - 1, -2 ** 31, 0, 5, 5, 5, 9, 10]] * 3),
               torch.tensor([[1, 1], [0, 1], [1, 0], [1, 1]])):
        of = of.to(torch.int32).cuda()
        for got, want in zip(mg.moe_sort(of, 9), sorted_by_hand(of, 9)):
            assert torch.equal(got, want)


def test_sort_is_the_same_every_time():
    of = choice(gen(5), 6000, 8, 64, 4)
    once = mg.moe_sort(of, 64)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(once, mg.moe_sort(of, 64)))


SHAPES = [(1, 8, 64, 0, 2560), (1, 1, 4, 0, 8), (5, 3, 4, 2, 24), (64, 8, 64, 0, 2560), (33, 16, 32, 8, 1032), (300, 2, 8, 2, 520), (100, 9, 10, 3, 512), (777, 4, 32, 32, 128),
          (1300, 8, 64, 8, 2560), (6200, 8, 64, 8, 512)]


@pytest.mark.parametrize("m,top,experts,away,width", SHAPES)
def test_rows_there_and_back(m, top, experts, away, width):
    g = gen(m + width)
    of = choice(g, m, top, experts, away)
    order, first, place = mg.moe_sort(of, experts)
    here = (of >= 0).reshape(-1)
    pairs = order[:int(here.sum())].long()                 # those with an expert, by position
    x = randn(g, m, width).bfloat16()
    rows = mg.moe_gather(x, first, place)
    want = torch.zeros_like(rows)
    want[:len(pairs)] = x[pairs // top]
    assert torch.equal(rows, want)

    rows, weights = randn(g, m * top, width).bfloat16(), torch.rand((m, top), device="cuda", generator=g)
    rows[len(pairs):] = float("nan")                       # rows of no expert are never read
    terms = rows[:len(pairs)].double()
    for w, got in ((weights, mg.moe_combine(rows, weights, first, place)), (torch.ones_like(weights), mg.moe_gather_backward(rows, first, place))):
        weighted = terms * w.reshape(-1)[pairs].double()[:, None]
        zero = torch.zeros((m, width), dtype=torch.float64, device="cuda")
        want, size = zero.index_add(0, pairs // top, weighted), zero.index_add(0, pairs // top, weighted.abs())
        assert ((got.double() - want).abs() <= HALF * want.abs() + 2 * (top + 1) * F32 * size).all()

    dy = randn(g, m, width).bfloat16()
    d_rows, d_weights = mg.moe_combine_backward(dy, rows, weights, first, place)
    want = torch.zeros((m * top, width), dtype=torch.float64, device="cuda")
    want[:len(pairs)] = dy.double()[pairs // top] * weights.reshape(-1)[pairs].double()[:, None]
    assert ((d_rows.double() - want).abs() <= (HALF + F32) * want.abs()).all()
    products = dy.double()[pairs // top] * terms
    want, size = (torch.zeros(m * top, dtype=torch.float64, device="cuda") for _ in range(2))
    want[pairs], size[pairs] = products.sum(1), products.abs().sum(1)
    assert ((d_weights.double().reshape(-1) - want).abs() <= width * F32 * size).all()


def test_gradients_are_the_transposes():
    """Both maps are linear: <gather(x), r> = <x, gather_backward(r)>; and differences of combine along each operand are its gradients."""
    g = gen(3)
    m, top, experts, width = 40, 4, 8, 256
    of = choice(g, m, top, experts, 2)
    _, first, place = mg.moe_sort(of, experts)
    whole = lambda *shape: torch.randint(-8, 9, shape, device="cuda", generator=g).float()  # small whole numbers: every sum is exact, in bf16 too
    x, r = whole(m, width).bfloat16(), whole(m * top, width).bfloat16()
    r[int(first[-1]):] = 0
    assert (mg.moe_gather(x, first, place).double() * r.double()).sum() == (x.double() * mg.moe_gather_backward(r, first, place).double()).sum()
    w, dy = whole(m, top), whole(m, width).bfloat16() / 8
    f = lambda r_, w_: (mg.moe_combine(r_, w_, first, place).double() * dy.double()).sum()
    rows = (whole(m * top, width) / 8).bfloat16()
    w = (w / 8).contiguous()
    d_rows, d_weights = mg.moe_combine_backward(dy, rows, w, first, place)
    base = mg.moe_combine(rows, w, first, place)
    for pair in (0, 17, 99):
        step = torch.zeros_like(w)
        step.view(-1)[pair] = 64.0                         # against which the rounding of y is small
        change = f(rows, w + step) - f(rows, w - step)
        size = ((base.double().abs() + 64 * 8) * dy.double().abs())[pair // top].sum()
        assert abs(change / 128 - d_weights.view(-1)[pair].double()) <= 2 * HALF * size / 128
        at = int(place.view(-1)[pair])
        bump = torch.zeros_like(rows)
        bump[at] = 16.0
        change, want = (f(rows + bump, w) - f(rows - bump, w)) / 32, (d_rows[at].double()).sum() if at < int(first[-1]) else torch.tensor(0.0)
        size = ((base.double().abs() + 17 * 8) * dy.double().abs())[pair // top].sum()
        assert abs(change - want) <= 2 * HALF * size / 32 + HALF * d_rows[at].double().abs().sum()


def test_results_go_where_they_are_asked_for_and_operands_may_be_strided():
    g = gen(11)
    m, top, experts, width = 21, 3, 6, 72
    of = choice(g, m, 2 * top, experts, 1)[:, ::2]         # not contiguous
    assert not of.is_contiguous()
    order, first, place = mg.moe_sort(of, experts)
    assert all(torch.equal(a, b) for a, b in zip((order, first, place), sorted_by_hand(of, experts)))
    wide = randn(g, m, 2 * width).bfloat16()
    x = wide[:, ::2]
    rows = torch.empty((m * top, width), dtype=torch.bfloat16, device="cuda")
    assert mg.moe_gather(x, first, place, out=rows) is rows and torch.equal(rows, mg.moe_gather(x.contiguous(), first, place))
    y = torch.empty((m, width), dtype=torch.bfloat16, device="cuda")
    weights = randn(g, top, m).t()
    assert mg.moe_combine(rows, weights, first, place, out=y) is y and torch.equal(y, mg.moe_combine(rows, weights.contiguous(), first, place))
    dy = randn(g, width, m).bfloat16().t()
    for a, b in zip(mg.moe_combine_backward(dy, rows, weights, first, place), mg.moe_combine_backward(dy.contiguous(), rows, weights.contiguous(), first, place)):
        assert torch.equal(a, b)


def test_no_rows():
    of = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    order, first, place = mg.moe_sort(of, 5)
    assert order.shape == (0,) and place.shape == (0, 4) and first.tolist() == [0] * 6
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda")
    assert mg.moe_gather(x, first, place).shape == (0, 64)
    w = torch.zeros((0, 4), device="cuda")
    assert mg.moe_combine(x, w, first, place).shape == (0, 64) and mg.moe_gather_backward(x, first, place).shape == (0, 64)
    assert [t.shape for t in mg.moe_combine_backward(x, x, w, first, place)] == [(0, 64), (0, 4)]


def test_infinities_stay_with_their_tokens():
    g = gen(2)
    of = torch.tensor([[0, 1], [1, 2], [2, 0]], dtype=torch.int32, device="cuda")
    _, first, place = mg.moe_sort(of, 3)
    rows = randn(g, 6, 64).bfloat16()
    rows[place[1, 0]] = float("inf")
    y = mg.moe_combine(rows, torch.ones((3, 2), device="cuda"), first, place)
    assert torch.isinf(y[1]).all() and torch.isfinite(y[[0, 2]]).all()
    x = randn(g, 3, 64).bfloat16()
    x[2] = float("nan")
    assert torch.isnan(mg.moe_gather(x, first, place)).sum() == 2 * 64
