"""Rows with low-rank adapters of their own out of a bank, beside one packed projection: `marlin_w4a16_gemm_bank` and its gradients,
against the formulas in 64 bits.

Tolerances.  U = 2^-8 is the most that a rounding to bf16 changes a value by, relative to it; F = 2^-24 the same for f32.  A sum of n
products in f32 is off by at most n F times the sum of the products' magnitudes, whatever its order.
* forward: the base product in f32, where the kernels multiply 128 + code and take the rest off: (k + 8) F times the sum of |x| * 280 * scale
  (144 at most + 136); it may be rounded before the low-rank term is added (U of it: two steps of rounding instead of one), and the sum is
  rounded (U |y|) in every case.  For the term, the projection's f32 sum (k F), its two bf16 parts (2^-16: the second part is rounded by U of a part that
  is U of the value) and the second sum (2 rank F + a few), relative to the sum of magnitudes.
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


def check_forward(p, y, base=None):
    (m, k), rank = p["x"].shape, p["a_"].shape[1]
    if m > 16:                                    # a row without an adapter is the plain GEMM's of as many rows, to the bit
        base = base if base is not None else marlin_gemm.marlin_w4a16_gemm(p["x"], p["b"], p["s"], p["g"])
        without = (p["of"] < 0) | (p["of"] >= len(p["sc"]))
        assert torch.equal(y[without].view(torch.int16), base[without].view(torch.int16))
    w = marlin_gemm.dequant_f32(p["b"], p["s"], p["g"]).double()
    tiled = p["s"].reshape(-1, p["s"].shape[0], 16).transpose(0, 1).reshape(p["s"].shape)
    scale = tiled.double().repeat_interleave(k // tiled.shape[0], 0)
    want = p["x"].double() @ w
    bound = (p["x"].double().abs() @ scale) * 280 * (k + 8) * F + U * want.abs()
    for j in range(len(p["sc"])):
        mine, s, a, b = p["of"] == j, p["sc"][j].double(), p["a_"][j].double(), p["b_"][j].double()
        x = p["x"][mine].double()
        want[mine] += s * ((x @ a.t()) @ b.t())
        bound[mine] += s.abs() * ((x.abs() @ a.abs().t()) @ b.abs().t()) * ((k + 2 * rank + 64) * F + 2.0 ** -16)
    check(y, want, bound * (1 + U))


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
    (1, 640, 512, -1, 3, 64, "any"), (2, 384, 256, 128, 2, 40, "any"), (2, 128, 8192, 128, 5, 24, "runs"), (1, 5760, 256, 128, 3, 8, "one"), (2, 256, 8448, 128, 3, 16, "any"),
    (1, 5120, 512, 128, 2, 8, "below"), (11, 9216, 256, 128, 6, 16, "any"), (9, 256, 256, 128, 3, 8, "none"), (90, 256, 256, 128, 3, 16, "beyond"), (70, 256, 256, -1, 3, 8, "below"),
    # column tiles that no count of them to a block divides; rows of one adapter each
    (16, 256, 9472, 128, 20, 16, "any"), (7, 384, 18688, -1, 3, 40, "any"), (3, 256, 25600, 128, 4, 8, "any"), (13, 4224, 4352, 128, 13, 24, "any"),
    (16, 5120, 6912, 128, 40, 64, "any"), (6, 3200, 28160, 128, 2, 56, "runs"), (4, 7296, 1280, 128, 9, 16, "any"),
]


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", SHAPES)
def test_forward(m, k, n, g, count, rank, pattern):
    p = problem(m, k, n, g, count, rank, pattern)
    check_forward(p, forward(p))


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", SHAPES)
def test_backward(m, k, n, g, count, rank, pattern):
    p = problem(m, k, n, g, count, rank, pattern, seed=1)
    check_backward(p, *backward(p))


# from thousands of rows on, wide outputs: the product adds the term itself
MANY = [(2100, 2560, 8192, 128, 40, 24, "any"), (2048, 2560, 8192, -1, 3, 64, "runs"), (2177, 2560, 8192, 128, 300, 8, "any"), (2050, 2560, 8192, 128, 5, 40, "none")]


@pytest.mark.parametrize("m,k,n,g,count,rank,pattern", MANY)
def test_forward_of_many_rows(m, k, n, g, count, rank, pattern):
    p = problem(m, k, n, g, count, rank, pattern)
    y = forward(p)
    check_forward(p, y)
    assert torch.equal(bits(y)[0], bits(forward({**p, "x": p["x"].t().contiguous().t()}))[0])


def bits(ts):
    return [t.view(torch.int16).clone() for t in (ts if isinstance(ts, tuple) else (ts,))]


@pytest.mark.parametrize("m", [3, 40, 300])
def test_an_adapter_that_holds_no_numbers_stays_with_its_own_rows(m):
    """Infinities and NaN in one adapter, and in one row of the activations, reach the rows and gradients that the formula says and no other."""
    p = problem(m, 256, 512, 128, 5, 24, "any", seed=2)
    p["of"][0], p["of"][1] = 2, 3                 # both there
    bad = {**p, "a_": p["a_"].clone(), "b_": p["b_"].clone()}
    bad["a_"][2, 3, 17], bad["a_"][2, 5, 200], bad["b_"][2, 400, 1] = float("inf"), float("nan"), float("-inf")
    mine = p["of"] == 2
    y, z = forward(p), forward(bad)
    assert torch.equal(y[~mine].view(torch.int16), z[~mine].view(torch.int16))
    assert not bool(torch.isfinite(z[mine]).any())                        # T of such a row is NaN, and goes to every column
    (da, d_a, d_b), (ea, e_a, e_b) = backward(p), backward(bad)
    assert torch.equal(da[~mine].view(torch.int16), ea[~mine].view(torch.int16))
    others = [0, 1, 3, 4]
    assert torch.equal(d_a[others].view(torch.int16), e_a[others].view(torch.int16))
    assert torch.equal(d_b[others].view(torch.int16), e_b[others].view(torch.int16))
    # B's infinity makes U's column 1 of these rows infinite: with A finite there dx is infinite wherever A[1] is not zero, NaN elsewhere
    only_a = {**p, "a_": bad["a_"]}
    fa = backward(only_a)[0]
    odd = torch.zeros(256, dtype=torch.bool, device="cuda")
    odd[17] = odd[200] = True
    assert not bool(torch.isfinite(fa[mine][:, odd]).any()) and bool(torch.isfinite(fa[mine][:, ~odd]).all())
    assert bool(torch.isnan(fa[mine][:, 200]).all())
    assert torch.equal(fa[mine][:, ~odd].view(torch.int16), da[mine][:, ~odd].view(torch.int16))
    x = p["x"].clone()
    x[1, 7] = float("nan")                        # a row of adapter 3
    z = forward({**p, "x": x})
    keep = torch.arange(m, device="cuda") != 1
    assert torch.equal(y[keep].view(torch.int16), z[keep].view(torch.int16)) and bool(torch.isnan(z[1]).all())


def test_an_adapter_that_holds_no_numbers_stays_with_its_own_of_many_rows():
    p = problem(2100, 2560, 8192, 128, 37, 24, "any", seed=3)
    bad = {**p, "a_": p["a_"].clone(), "b_": p["b_"].clone(), "x": p["x"].clone()}
    bad["a_"][20, 3, 17], bad["b_"][2, 400, 1], bad["b_"][3, 8000, 20] = float("nan"), float("-inf"), float("nan")
    row = int((p["of"] == 5).nonzero()[0])
    bad["x"][row, 7] = float("inf")
    y, z = forward(p), forward(bad)
    odd = (p["of"] == 2) | (p["of"] == 3) | (p["of"] == 20)
    odd[row] = True
    assert torch.equal(bits(y[~odd])[0], bits(z[~odd])[0])
    assert not bool(torch.isfinite(z[p["of"] == 20]).any()) and not bool(torch.isfinite(z[p["of"] == 2][:, 400]).any())
    assert not bool(torch.isfinite(z[p["of"] == 3][:, 8000]).any()) and not bool(torch.isfinite(z[row]).all())


@pytest.mark.parametrize("m", [7, 130, 400])
def test_same_bits_again_on_views_other_streams_and_into_a_given_tensor(m):
    p = problem(m, 384, 512, 128, 6, 16, "any", seed=3)
    y, g = bits(forward(p)), bits(backward(p))
    wide = {**p, "x": torch.cat([p["x"], p["x"]], 1)[:, :384], "dy": torch.cat([p["dy"], p["dy"]], 1)[:, 512:],
            "of": torch.stack([p["of"], p["of"]], 1)[:, 0], "a_": p["a_"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert not any(wide[k].is_contiguous() for k in ("x", "dy", "a_")) and (m == 1 or not wide["of"].is_contiguous())
    out = torch.full((m, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        again = bits(forward(p, out=out)), bits(backward(p))
    stream.synchronize()
    for got in ((bits(forward(wide)), bits(backward(wide))), again, (bits(out), bits(backward(p)))):
        assert all(torch.equal(a, b) for a, b in zip(got[0] + got[1], y + g))


@pytest.mark.parametrize("m,k,n", [(5, 256, 512), (50, 256, 512), (300, 256, 512), (4200, 512, 8192)])
def test_replayed_from_a_graph(m, k, n):
    """Captured calls replayed with other contents in the same tensors, eager calls and synchronisations between the replays."""
    parts = [problem(m, k, n, 128, 4, 8, "any", seed=s) for s in (4, 5, 6)]
    live = {k: v.clone() if torch.is_tensor(v) else v for k, v in parts[0].items()}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        forward(live), backward(live)                 # the stream's workspace
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            made = (forward(live), *backward(live))
        for p in parts + parts:
            for k, v in p.items():
                if torch.is_tensor(v):
                    live[k].copy_(v)
            graph.replay()
            stream.synchronize()
            got = bits(made)
            want = bits((forward(p), *backward(p)))
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows_and_the_plain_gradient():
    p = problem(0, 256, 512, 128, 3, 8, "one", seed=7)
    assert forward(p).shape == (0, 512)
    da, d_a, d_b = backward(p)
    assert da.shape == (0, 256) and not bool(d_a.any()) and not bool(d_b.any())
    assert marlin_gemm.marlin_w4a16_gemm_backward(p["dy"], p["b"], p["s"], 128).shape == (0, 256)
    for m in (1, 50, 700):
        p = problem(m, 640, 512, -1, 3, 8, "none", seed=8)
        assert torch.equal(marlin_gemm.marlin_w4a16_gemm_backward(p["dy"], p["b"], p["s"], -1).view(torch.int16), backward(p)[0].view(torch.int16))


@pytest.mark.parametrize("m", [0, 6, 90])
def test_a_scale_that_is_no_number_stays_with_its_adapter(m):
    """An adapter without rows has gradients of zero, whatever its scale."""
    p = problem(m, 256, 512, 128, 4, 16, "one", seed=11)          # every row the last one's
    want_y, want = bits(forward(p)), bits(backward(p))
    p["sc"][0], p["sc"][1] = float("inf"), float("nan")
    assert all(torch.equal(a, b) for a, b in zip(want_y + want, bits(forward(p)) + bits(backward(p))))


def test_gradients_against_differences():
    """d(sum y * dy) along a direction of x, A and B, by the forward in steps either way, against the gradients."""
    p = problem(24, 256, 256, 128, 3, 8, "any", seed=9)
    da, d_a, d_b = (t.double() for t in backward(p))
    w = marlin_gemm.dequant_f32(p["b"], p["s"], 128).double()

    def loss(x, a, b):
        y = x @ w
        for j in range(3):
            mine = p["of"] == j
            y[mine] += p["sc"][j].double() * ((x[mine] @ a[j].t()) @ b[j].t())
        return (y * p["dy"].double()).sum()

    at = [p[k].double() for k in ("x", "a_", "b_")]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, grad in enumerate((da, d_a, d_b)):
        d = torch.randn(at[i].shape, dtype=torch.float64, device="cuda", generator=gen)
        step = [[t + sign * 1e-3 * d if j == i else t for j, t in enumerate(at)] for sign in (1, -1)]
        slope = (loss(*step[0]) - loss(*step[1])) / 2e-3                   # exact: the loss is linear in each of them
        bound = 4 * U * (grad * d).abs().sum() + 64 * U * grad.abs().max()
        assert abs((grad * d).sum() - slope) <= bound


def test_rows_behind_and_around_the_result_stay_as_they_were():
    p = problem(37, 256, 512, 128, 4, 16, "any", seed=10)
    room = torch.full((37 + 2, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    y = forward(p, out=room[1:38])
    assert y.data_ptr() == room[1:38].data_ptr() and bool((room[0] == 7).all()) and bool((room[38] == 7).all())
    assert torch.equal(bits(y)[0], bits(forward(p))[0])


def test_refusals():
    p = problem(6, 256, 512, 128, 3, 16, "any")
    for change, text in ((dict(a_=p["a_"][:, :, :128]), "bank shapes"), (dict(b_=p["b_"][:2]), "bank shapes"), (dict(sc=p["sc"][:2]), "bank shapes"),
                         (dict(of=p["of"][:5]), "adapter_of must be"), (dict(of=p["of"].long()), "adapter_of i32"), (dict(sc=p["sc"].double()), "bank_scales must be f32"),
                         (dict(a_=p["a_"].float()), "must be bf16"), (dict(a_=p["a_"][:, :12], b_=p["b_"][:, :, :12]), "multiple of 8"),
                         (dict(of=p["of"].cpu()), "must be on"), (dict(a_=p["a_"][0]), "a bank is"), (dict(x=p["x"].half()), "a must be bf16"), (dict(g=64), "groupsize")):
        for call in (forward, backward):
            with pytest.raises(marlin_gemm.MarlinGemmError, match=text):
                call({**p, **change})
    with pytest.raises(marlin_gemm.MarlinGemmError, match="dy must be"):
        backward({**p, "dy": p["dy"][:, :256]})
    with pytest.raises(marlin_gemm.MarlinGemmError, match="out must be"):
        forward(p, out=torch.empty(6, 256, dtype=torch.bfloat16, device="cuda"))


def test_more_rows_than_a_grid_is_high():
    """Over 65536 tiles of 16 rows: the rows sampled, at either end and where the count of tiles passes 16 bits."""
    m, k, n, count, rank = 16 * 65536 + 21, 128, 256, 3, 8
    gen = torch.Generator(device="cuda").manual_seed(11)
    b, s = packed(gen, k, n, 128)
    p = dict(x=torch.randn(m, k, device="cuda", generator=gen).bfloat16(), b=b, s=s, g=128, a_=(torch.randn(count, rank, k, device="cuda", generator=gen) / 11).bfloat16(),
             b_=(torch.randn(count, n, rank, device="cuda", generator=gen) / 3).bfloat16(), sc=torch.ones(count, device="cuda"),
             of=torch.randint(-1, count, (m,), device="cuda", generator=gen).to(torch.int32), dy=(torch.randn(m, n, device="cuda", generator=gen) * 0.02).bfloat16())
    y, (da, d_a, d_b) = forward(p), backward(p)
    at = torch.cat([torch.arange(40), torch.randint(0, m, (500,)), torch.arange(65536 * 16 - 20, m)]).cuda()
    few = {**p, "x": p["x"][at], "of": p["of"][at], "dy": p["dy"][at]}
    check_forward(few, y[at], marlin_gemm.marlin_w4a16_gemm(p["x"], b, s, 128)[at])
    want = few["dy"].double() @ marlin_gemm.dequant_f32(b, s, 128).double().t()
    bound = (few["dy"].double().abs() @ marlin_gemm.dequant_f32(b, s, 128).double().abs().t()) * (U + (n + 2 * rank) * F)
    for j in range(count):
        mine, a, bb = few["of"] == j, p["a_"][j].double(), p["b_"][j].double()
        g = few["dy"][mine].double()
        want[mine] += (g @ bb) @ a
        bound[mine] += (g.abs() @ bb.abs()) @ a.abs() * ((2 * n + 2 * rank + 64) * F + 2.0 ** -16)
        rows = p["of"] == j
        x, g = p["x"][rows].double(), p["dy"][rows].double()
        check(d_a[j], (g @ bb).t() @ x, ((g.abs() @ bb.abs()).t() @ x.abs()) * ((n + m + 64) * F))
        check(d_b[j], g.t() @ (x @ a.t()), (g.abs().t() @ (x.abs() @ a.abs().t())) * ((k + m + 64) * F))
    check(da[at], want, bound)


def test_a_step_of_many_requests_through_a_layer():
    """Requests with adapters of their own through a layer's packed projections and its experts, then the gradients of the adapters, each part
    held to its formula on what the part before it gave."""
    from kiln_amd import layer_pack, lora, moe
    from kiln_amd.layer_pack import LayerProjections, PackKind
    gen = torch.Generator(device="cuda").manual_seed(12)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    weight = lambda k, n: (rand(k, n) / k ** 0.5).bfloat16()
    layer = LayerProjections({PackKind.QProj: weight(256, 512), PackKind.OProj: weight(512, 256)})
    layer_pack.pack_layers([layer])
    adapters = lambda k, n: lora.make_bank([lora.LoraProjectionWeights((rand(r, k) / k ** 0.5).bfloat16(), (rand(n, r) / r ** 0.5).bfloat16()) for r in (8, 12, 3)], (0.5, 1.0, 2.0))
    bank_q, bank_o = adapters(256, 512), adapters(512, 256)
    of = torch.tensor([0, 0, 2, -1, 1, 1, 1, 0, 2, 3] * 3, dtype=torch.int32, device="cuda")

    def as_problem(x, kind, bank, dy=None):
        w = layer.packed[kind]
        return dict(x=x, b=w.b_packed, s=w.scales, g=w.groupsize, a_=bank.a, b_=bank.b, sc=bank.scales, of=of, dy=dy)

    x = rand(3, 10, 256).bfloat16()
    q = layer.forward_bank(PackKind.QProj, x, bank_q, of)
    assert q.shape == (3, 10, 512)
    check_forward(as_problem(x.reshape(30, 256), PackKind.QProj, bank_q), q.reshape(30, 512))
    o = lora.proj_forward_bank(q, layer.packed[PackKind.OProj], bank_o, of.reshape(3, 10))
    check_forward(as_problem(q.reshape(30, 512), PackKind.OProj, bank_o), o.reshape(30, 256))
    experts = moe.pack_experts(*(torch.stack([weight(k, n) for _ in range(4)]) for k, n in ((256, 256), (256, 256), (256, 256))))
    y = x + o + moe.moe_forward(x + o, weight(256, 4), experts, 2)
    assert bool(torch.isfinite(y).all())
    dy = (rand(3, 10, 256) * 0.1).bfloat16()
    dq, d_a, d_b = lora.proj_backward_bank(dy, q, layer.packed[PackKind.OProj], bank_o, of.reshape(3, 10))
    check_backward(as_problem(q.reshape(30, 512), PackKind.OProj, bank_o, dy.reshape(30, 256)), dq.reshape(30, 512), d_a, d_b)
    dx, e_a, e_b = lora.proj_backward_bank(dq, x, layer.packed[PackKind.QProj], bank_q, of)
    check_backward(as_problem(x.reshape(30, 256), PackKind.QProj, bank_q, dq.reshape(30, 512)), dx.reshape(30, 256), e_a, e_b)
    alone, none_a, none_b = lora.proj_backward_bank(dq, x, layer.packed[PackKind.QProj])
    assert alone.shape == x.shape and none_a is None and none_b is None
    # a projection that stayed on bf16 takes the same call
    plain = LayerProjections({PackKind.QProj: weight(256, 512)})
    z = plain.forward_bank(PackKind.QProj, x, bank_q, of).reshape(30, 512).double()
    w = plain.weights_t[PackKind.QProj].double()
    want = x.reshape(30, 256).double() @ w
    for j in range(3):
        mine = of == j
        want[mine] += bank_q.scales[j].double() * ((x.reshape(30, 256)[mine].double() @ bank_q.a[j].double().t()) @ bank_q.b[j].double().t())
    assert ((z - want).abs().max() / want.abs().max()).item() < 8 * U
