"""The gradients of moe_combine against differences of moe_combine itself, pair by pair and exactly.  It is linear in either operand; with small whole numbers every
sum is a whole number of at most 256, exact in bf16 and f32, so nothing is rounded and the two have to be equal."""
import pytest
import torch

from tests.expert_packs import choice
from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu


def whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, device="cuda", generator=g).float()


@pytest.mark.parametrize("m,top,experts,away,width", [(12, 4, 8, 2, 256), (5, 3, 6, 0, 72), (20, 1, 4, 1, 8), (3, 16, 16, 3, 520)])
def test_gradients_are_the_differences(m, top, experts, away, width):
    g = torch.Generator(device="cuda").manual_seed(m)
    _, first, place = mg.moe_sort(choice(g, m, top, experts, away), experts)
    rows, w, dy = whole(g, 3, m * top, width).bfloat16(), whole(g, 3, m, top), whole(g, 3, m, width).bfloat16()   # sums of 16 * 4 * 4 at most, steps included
    d_rows, d_weights = mg.moe_combine_backward(dy, rows, w, first, place)
    f = lambda r, v: float((mg.moe_combine(r, v, first, place).double() * dy.double()).sum())
    base, weights_by, rows_by, rows_said = f(rows, w), [], [], []
    for pair in range(m * top):
        step = w.clone()
        step.view(-1)[pair] += 1
        weights_by.append(f(rows, step) - base)
        at, bump = int(place.view(-1)[pair]), whole(g, 1, width)
        moved = rows.clone()
        moved[at] += bump.bfloat16()
        rows_by.append(f(moved, w) - base)
        rows_said.append(float((d_rows[at].double() * bump.double()).sum()))
    assert d_weights.view(-1).tolist() == weights_by and rows_said == rows_by
    # (a gradient of zeros, or of the pair beside it, is another)
    placed = (place.view(-1) < int(first[-1])).sum()
    for by in (weights_by, rows_by):
        assert sum(v != 0 for v in by) > 0.5 * placed and sum(a != b for a, b in zip(by, by[1:] + by[:1])) > 0.5 * placed
