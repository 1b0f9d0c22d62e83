"""Rows with low-rank adapters of their own out of a bank, beside one packed projection: `marlin_w4a16_gemm_bank` and its gradients,
against the formulas in 64 bits.

Tolerances.  U = 2^-8 is the most that a rounding to bf16 changes a value by, relative to it; F = 2^-24 the same for f32.  A sum of n
products in f32 is off by at most n F times the sum of the products' magnitudes, whatever its order.
* forward: the result is the plain GEMM's bf16 row plus the low-rank term, rounded once: U |y| and, for the term, the projection's f32
  sum (k F), its two bf16 parts (2^-16: the second part is rounded by U of a part that is U of the value) and the second sum (2 rank F + a few),
  relative to the sum of magnitudes.
* dx: a weight is rounded to bf16 (U), so U times the sum of |dy| |W|, plus f32 sums (n F) and the low-rank term as above; U |dx| at the end.
* dA, dB: the inner product in f32 (K F), the sum over rows (rows F), U of the result.
"""
import pytest
import torch

from kiln_amd import marlin_gemm

pytestmark = pytest.mark.gpu
U, F = 2.0 ** -8, 2.0 ** -24


def packed(gen, k, n, g):
    words = torch.randint(-2**31, 2**31, (k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    scales = ((torch.rand(1 if g == -1 else k // g, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    return words, scales


def problem(m, k, n, g, count, rank, pattern, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + k + n + rank)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    b, s = packed(gen, k, n, g)
    if pattern == "any":
        of = torch.randint(-2, count + 2, (m,), device="cuda", generator=gen)
    elif pattern == "runs":
        of = torch.randint(0, count, (m,), device="cuda", generator=gen).sort().values
    elif pattern == "one":
        of = torch.full((m,), count - 1, device="cuda")
    else:
        of = torch.full((m,), {"none": -1, "beyond": 2**31 - 1, "below": -2**31}[pattern], device="cuda")
    return dict(x=rand(m, k).bfloat16(), b=b, s=s, g=g, a_=(rand(count, rank, k) / k ** 0.5).bfloat16(),
                b_=(rand(count, n, rank) / rank ** 0.5).bfloat16(), sc=torch.rand(count, device="cuda", generator=gen) * 2 - 0.5,
                of=of.to(torch.int32), dy=(rand(m, n) * 0.02).bfloat16())


def forward(p, **kw):
    return marlin_gemm.marlin_w4a16_gemm_bank(p["x"], p["b"], p["s"], p["g"], p["a_"], p["b_"], p["sc"], p["of"], **kw)


def backward(p):
    return marlin_gemm.marlin_w4a16_gemm_bank_backward(p["dy"], p["x"], p["b"], p["s"], p["g"], p["a_"], p["b_"], p["sc"], p["of"])


def check(got, want, bound):
    got = got.double()
    assert bool(torch.isfinite(got).all())
    excess = ((got - want).abs() - bound - U * want.abs()).max().item() if got.numel() else 0.0
    assert excess <= 0.0, (excess, (got - want).abs().max().item())


def check_forward(p, y):
    base = marlin_gemm.marlin_w4a16_gemm(p["x"], p["b"], p["s"], p["g"])
    rows_without = (p["of"] < 0) | (p["of"] >= len(p["sc"]))
    assert torch.equal(y[rows_without].view(torch.int16), base[rows_without].view(torch.int16))
    want, size = base.double(), torch.zeros_like(base, dtype=torch.float64)
    k, rank = p["x"].shape[1], p["a_"].shape[1]
    for j in range(len(p["sc"])):
        mine, s, a, b = p["of"] == j, p["sc"][j].double(), p["a_"][j].double(), p["b_"][j].double()
        x = p["x"][mine].double()
        want[mine] += s * ((x @ a.t()) @ b.t())
        size[mine] = s.abs() * ((x.abs() @ a.abs().t()) @ b.abs().t())
    check(y, want, size * ((k + 2 * rank + 64) * F + 2.0 ** -16) + base.double().abs() * 4 * F)


def check_backward(p, da, d_a, d_b):
    w = marlin_gemm.dequant_f32(p["b"], p["s"], p["g"]).double()
    dy, n, (m, k), rank = p["dy"].double(), p["dy"].shape[1], p["x"].shape, p["a_"].shape[1]
    want, bound = dy @ w.t(), (dy.abs() @ w.abs().t()) * (U + (n + 2 * rank) * F)
    for j in range(len(p["sc"])):
        mine, s, a, b = p["of"] == j, p["sc"][j].double(), p["a_"][j].double(), p["b_"][j].double()
        x, g = p["x"][mine].double(), dy[mine]
        u, t = g @ b, x @ a.t()
        u_size, t_size = g.abs() @ b.abs(), x.abs() @ a.abs().t()
        want[mine] += s * (u @ a)
        bound[mine] += s.abs() * (u_size @ a.abs()) * ((2 * n + 2 * rank + 64) * F + 2.0 ** -16)
        check(d_a[j], s * (u.t() @ x), s.abs() * (u_size.t() @ x.abs()) * ((n + m + 64) * F))
        check(d_b[j], s * (g.t() @ t), s.abs() * (g.abs().t() @ t_size) * ((k + m + 64) * F))
    check(da, want, bound)


SHAPES = [
    (1, 128, 256, 128, 1, 8, "one"), (1, 2560, 2560, 128, 4, 8, "any"), (2, 256, 256, -1, 3, 16, "any"), (5, 384, 512, 128, 7, 24, "any"),
    (16, 2560, 2560, 128, 16, 16, "any"), (17, 640, 768, 128, 40, 64, "any"), (33, 9216, 2560, -1, 5, 40, "runs"), (64, 1024, 256, 128, 64, 48, "any"),
    (65, 128, 1024, 128, 9, 56, "any"), (77, 4096, 512, -1, 3, 32, "runs"), (128, 256, 256, 128, 1, 64, "one"), (129, 896, 1792, 128, 200, 8, "any"),
    (300, 2560, 1024, 128, 6, 16, "runs"), (777, 384, 2560, -1, 11, 24, "any"), (1030, 256, 512, 128, 2, 32, "runs"),
    (9, 256, 256, 128, 3, 8, "none"), (90, 256, 256, 128, 3, 16, "beyond"), (70, 256, 256, -1, 3, 8, "below"),
]


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", SHAPES)
def test_forward(m, k, n, g, count, rank, pattern):
    p = problem(m, k, n, g, count, rank, pattern)
    check_forward(p, forward(p))


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", SHAPES)
def test_backward(m, k, n, g, count, rank, pattern):
    p = problem(m, k, n, g, count, rank, pattern, seed=1)
    check_backward(p, *backward(p))
