"""Rows of tokens in the order of their experts and back where a launch has more than 2^31 work-items."""
import pytest
import torch

from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu


def test_more_than_two_to_the_31_units():
    m, width = 8_400_000, 2048
    assert m * (width // 8) > 2 ** 31
    of = torch.randint(0, 5, (m, 1), dtype=torch.int32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    of[-3] = -1
    _, first, place = mg.moe_sort(of, 5)
    some = torch.cat((torch.arange(0, 50), torch.arange(m // 2, m // 2 + 50), torch.arange(m - 50, m))).cuda()
    at = place[some, 0].long()
    x = torch.empty((m, width), dtype=torch.bfloat16, device="cuda")
    x[some] = torch.randn((len(some), width), device="cuda").bfloat16()
    rows = mg.moe_gather(x, first, place)
    want = x[some].clone()
    want[-3] = 0
    assert torch.equal(rows[at], want)
    x.zero_()
    weights = torch.full((m, 1), 2.0, device="cuda")
    assert mg.moe_combine(rows, weights, first, place, out=x) is x and torch.equal(x[some], 2 * want)
