"""The experts of a mixture-of-experts MLP for a few tokens (`marlin_w4a16_moe`) and the router's choice (`moe_route`), against the
formulas in 64 bits.

Tolerances.  U = 2^-8 and F = 2^-24 are the most that a rounding to bf16 and to f32 changes a value by, relative to it.
* a product with codes in f32: the kernels multiply 128 + code and take the rest off, so n products are off by at most
  (n + 8) F times the sum of |x| * 280 * scale (144 at most + 136)
* h = silu(gate) * up: its rounding U |h|, exp and reciprocal a few F, and what gate's and up's errors make of it: silu's slope is at most 1.1
* y: down's sums as above over what h's errors make of it, its weights' f32 sum, and U |y|
* route: exp of differences up to d is off by at most (d + 4) F * 2 relative (the argument's rounding), sums of n by n F
"""
import math

import pytest
import torch

from kiln_amd import marlin_gemm, moe

pytestmark = pytest.mark.gpu
U, F = 2.0 ** -8, 2.0 ** -24


def packed(gen, experts, k, n, g):
    words = torch.randint(-2**31, 2**31, (experts, k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    scales = ((torch.rand(experts, 1 if g == -1 else k // g, n, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)).half()
    return words, scales


def layer(m, top, experts, hidden, n_out, n_down, g, pattern="any", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + experts + hidden + n_out)
    rand = lambda *shape: torch.rand(shape, device="cuda", generator=gen)
    if pattern == "any":                  # distinct experts, some of them elsewhere
        of = rand(m, experts).argsort(dim=1)[:, :top]
        of = torch.where(rand(m, top) < 0.1, torch.where(rand(m, top) < 0.5, -1, experts), of)
    elif pattern == "one":
        of = torch.full((m, top), -7, device="cuda")
        of[:, top // 2] = experts - 1
    elif pattern == "twice":              # the same expert in several places of a row
        of = torch.randint(0, min(2, experts), (m, top), device="cuda", generator=gen)
    else:
        of = torch.full((m, top), {"none": -1, "beyond": 2**31 - 1}[pattern], device="cuda")
    b_in, s_in = packed(gen, experts, hidden, 2 * n_out, g)
    b_out, s_out = packed(gen, experts, n_out, n_down, g)
    x = torch.randn(m, hidden, device="cuda", generator=gen).bfloat16()
    return x, of.to(torch.int32), rand(m, top) + 0.05, b_in, s_in, b_out, s_out, g


def check_layer(args, y):
    x, of, weights, b_in, s_in, b_out, s_out, g = args
    want = torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    hidden, n_out = x.shape[1], b_out.shape[1] * 16
    for e in range(b_in.shape[0]):
        rows, place = torch.nonzero(of == e, as_tuple=True)
        if not len(rows):
            continue
        w_in = marlin_gemm.dequant_f32(b_in[e], s_in[e], g).double()
        w_out = marlin_gemm.dequant_f32(b_out[e], s_out[e], g).double()

        def scale_of(s, k):
            s = s[e].reshape(-1, s.shape[1], 16).transpose(0, 1).reshape(s.shape[1], -1).double()     # tiled -> [groups, n]
            return s.repeat_interleave(k // s.shape[0], 0)

        xr, wt = x[rows].double(), weights[rows, place].double()[:, None]
        gu = (xr @ w_in).reshape(len(rows), -1, 2, 8)
        gu_off = ((xr.abs() @ scale_of(s_in, hidden)) * 280 * (hidden + 8) * F).reshape(len(rows), -1, 2, 8)
        gate, up, gate_off, up_off = (t.reshape(len(rows), n_out) for t in (gu[:, :, 0], gu[:, :, 1], gu_off[:, :, 0], gu_off[:, :, 1]))
        act = gate * torch.sigmoid(gate)
        h = act * up
        h_off = h.abs() * (U + 64 * F) + 1.1 * gate_off * up.abs() + (act.abs() + 1.1 * gate_off) * up_off
        out_off = h_off @ w_out.abs() + ((h.abs() + h_off) @ scale_of(s_out, n_out)) * 280 * (n_out + 8) * F
        want.index_add_(0, rows, wt * (h @ w_out))
        bound.index_add_(0, rows, wt * (out_off + (h @ w_out).abs() * (of.shape[1] + 16) * F))
    y = y.double()
    assert bool(torch.isfinite(y).all())
    excess = (y - want).abs() - bound * (1 + U) - U * want.abs()
    assert excess.max().item() <= 0.0, (excess.max().item(), (y - want).abs().max().item())


LAYERS = [
    (1, 8, 64, 2560, 1024, 2560, 128, "any"), (1, 1, 1, 128, 128, 256, -1, "any"), (2, 16, 16, 256, 256, 512, 128, "any"),
    (5, 2, 8, 384, 640, 768, -1, "any"), (3, 5, 9, 256, 768, 512, 128, "any"), (1, 16, 3, 256, 1152, 256, 128, "twice"), (8, 2, 2, 128, 640, 256, 128, "twice"),
    (16, 1, 1, 128, 1024, 256, -1, "any"), (2, 2, 4, 11008, 5504, 512, 128, "any"), (13, 4, 32, 2048, 1280, 2048, -1, "any"), (16, 8, 1024, 128, 128, 256, 128, "any"),
    (17, 3, 5, 640, 384, 256, 128, "any"), (33, 1, 4, 256, 256, 256, 128, "one"), (64, 8, 64, 1024, 256, 1024, 128, "any"),
    (65, 5, 7, 256, 128, 512, 128, "any"), (200, 2, 3, 384, 256, 256, -1, "one"), (9, 4, 6, 256, 128, 256, 128, "twice"),
    (64, 16, 24, 128, 128, 256, 128, "twice"), (4, 2, 8, 256, 128, 256, 128, "none"), (70, 3, 8, 256, 128, 256, 128, "beyond"),
]


@pytest.mark.parametrize("m,top,experts,hidden,n_out,n_down,g,pattern", LAYERS)
def test_experts(m, top, experts, hidden, n_out, n_down, g, pattern):
    args = layer(m, top, experts, hidden, n_out, n_down, g, pattern)
    check_layer(args, marlin_gemm.marlin_w4a16_moe(*args))


def check_route(logits, top, renormalise, of, weights):
    l = logits.double().cpu()
    value, order = torch.sort(l.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=1, descending=True, stable=True)
    value, order = value[:, :top], torch.where(value == -math.inf, -1, order)[:, :top]
    assert torch.equal(of.cpu(), order.to(torch.int32))
    best = value[:, :1]
    empty, bad = best[:, 0] == -math.inf, l.isnan().any(1) | (best[:, 0] == math.inf)
    share = torch.exp(value - best)
    share = share / (share.sum(1, keepdim=True) if renormalise else torch.exp(l - best).sum(1, keepdim=True))
    share[empty] = 0.0
    weights = weights.cpu().double()
    assert bool(weights[bad].isnan().all())
    far = (best - value).nan_to_num(nan=0.0).clamp(max=104)      # beyond that exp is 0 in f32; an empty row has no differences
    bound = share * ((far + 8) * 4 * F + 2 * l.shape[1] * F) + 2.0 ** -126
    assert bool(((weights - share).abs() <= bound)[~bad].all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,experts,top", [(1, 1, 1), (1, 64, 8), (3, 5, 5), (7, 63, 2), (9, 65, 16), (33, 128, 8), (130, 257, 7), (4097, 512, 4), (21, 1024, 16)])
def test_route(m, experts, top, dtype):
    gen = torch.Generator(device="cuda").manual_seed(m + experts)
    logits = (torch.randn(m, experts, device="cuda", generator=gen) * 3).to(dtype)
    for renormalise in (False, True):
        check_route(logits, top, renormalise, *marlin_gemm.moe_route(logits, top, renormalise))


def test_route_ties_masks_and_values_that_are_no_numbers():
    logits = torch.zeros(10, 70, device="cuda")
    logits[1, ::3] = 2.0                                  # ties beyond a wavefront's width
    logits[2] = -math.inf                                 # nothing left
    logits[3, 5:] = -math.inf                             # fewer than asked for
    logits[4] = torch.finfo(torch.float32).min            # a mask of the type's lowest value
    logits[4, 69] = 0.0
    logits[5, 17] = math.nan
    logits[6, 3], logits[6, 66] = math.inf, 1.0
    logits[7, 1::2] = -0.0                                # equal to the zeros beside them
    logits[8] = torch.finfo(torch.float32).max
    logits[9, :64] = -200.0
    for renormalise in (False, True):
        check_route(logits, 8, renormalise, *marlin_gemm.moe_route(logits, 8, renormalise))


def test_layer_from_bf16_weights():
    """The whole layer: router, choice and experts, the experts quantised here and packed as the MLP's projections are."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *shape: (torch.randn(shape, device="cuda", generator=gen) / shape[-2] ** 0.5).bfloat16()
    gate, up, down, router = rand(6, 256, 384), rand(6, 256, 384), rand(6, 384, 512), rand(256, 6)
    experts = moe.pack_experts(gate, up, down)
    x = torch.randn(2, 5, 256, device="cuda", generator=gen).bfloat16()
    y = moe.moe_forward(x, router, experts, 2)
    assert y.shape == (2, 5, 512)
    rows = x.reshape(10, 256)
    of, weights = marlin_gemm.moe_route(rows @ router, 2)
    args = (rows, of, weights, experts.b_gate_up, experts.s_gate_up, experts.b_down, experts.s_down, 128)
    check_layer(args, y.reshape(10, 512))
    # a token whose weight is all on one expert is that expert's MLP
    one = marlin_gemm.marlin_w4a16_moe(rows, torch.full((10, 1), 4, dtype=torch.int32, device="cuda"), torch.ones(10, 1, device="cuda"), *args[3:])
    mlp = marlin_gemm.marlin_w4a16_mlp(rows, experts.b_gate_up[4], experts.s_gate_up[4], experts.b_down[4], experts.s_down[4], 128)
    scale = mlp.double().abs().max()
    assert ((one.double() - mlp.double()).abs().max() / scale).item() < 4 * U


def bits(t):
    return t.view(torch.int16).clone()


@pytest.mark.parametrize("m,top,experts", [(1, 8, 16), (12, 4, 16), (40, 6, 16)])
def test_same_bits_again_on_views_other_streams_and_into_a_given_tensor(m, top, experts):
    args = layer(m, top, experts, 256, 256, 512, 128, seed=1)
    y = bits(marlin_gemm.marlin_w4a16_moe(*args))
    x, of, weights, *packs = args
    wide = (torch.cat([x, x], 1)[:, 256:], torch.stack([of, of], 2)[:, :, 1], torch.cat([weights, weights], 1)[:, :top], *packs)
    assert torch.equal(bits(marlin_gemm.marlin_w4a16_moe(*wide)), y)
    room = torch.full((m + 2, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        out = marlin_gemm.marlin_w4a16_moe(*args, out=room[1:m + 1])
    stream.synchronize()
    assert out.data_ptr() == room[1:].data_ptr() and torch.equal(bits(out), y)
    assert bool((room[0] == 7).all()) and bool((room[m + 1] == 7).all())
    logits = torch.randn(m, 2 * experts, device="cuda")
    a, b = marlin_gemm.moe_route(logits[:, ::2], top), marlin_gemm.moe_route(logits[:, ::2].contiguous(), top)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("m,top", [(1, 8), (12, 4), (70, 2)])
def test_a_layer_replayed_from_a_graph(m, top):
    parts = [layer(m, top, 12, 256, 256, 512, 128, seed=s) for s in (2, 3, 4)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = [torch.randn(m, 12, device="cuda", generator=gen) for _ in parts]
    live = [t.clone() if torch.is_tensor(t) else t for t in parts[0]]
    live_logits = logits[0].clone()

    def call(l, a):
        of, weights = marlin_gemm.moe_route(l, top)
        return of, weights, marlin_gemm.marlin_w4a16_moe(a[0], of, weights, *a[3:])

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(live_logits, live)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            made = call(live_logits, live)
        for l, a in zip(logits + logits, parts + parts):
            live_logits.copy_(l)
            for to, t in zip(live, a):
                if torch.is_tensor(t):
                    to.copy_(t)
            graph.replay()
            stream.synchronize()
            got = [t.clone() for t in made]
            want = call(l, a)
            stream.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(bits(got[2]), bits(want[2]))


def test_what_is_no_number_stays_with_its_token_and_its_expert():
    x, of, weights, b_in, s_in, b_out, s_out, g = layer(20, 2, 6, 256, 128, 256, 128, seed=6)
    of[:, 0], of[:, 1] = torch.arange(20, device="cuda") % 6, (torch.arange(20, device="cuda") + 1) % 6
    y = bits(marlin_gemm.marlin_w4a16_moe(x, of, weights, b_in, s_in, b_out, s_out, g))
    bad_x, bad_s, bad_w = x.clone(), s_in.clone(), weights.clone()
    bad_x[3, 5], bad_s[2, 1, 40], bad_w[7, 1] = math.nan, math.nan, math.inf
    z = marlin_gemm.marlin_w4a16_moe(bad_x, of, bad_w, b_in, bad_s, b_out, s_out, g)
    hit = (of == 2).any(1)
    hit[3] = hit[7] = True
    assert torch.equal(bits(z)[~hit], y[~hit]) and not bool(torch.isfinite(z[3]).any()) and not bool(torch.isfinite(z[7]).all())


def test_no_tokens_and_refusals():
    args = layer(4, 2, 3, 256, 128, 256, 128)
    x, of, weights, b_in, s_in, b_out, s_out, g = args
    assert marlin_gemm.marlin_w4a16_moe(x[:0], of[:0], weights[:0], *args[3:]).shape == (0, 256)
    of_none, w_none = marlin_gemm.moe_route(torch.empty(0, 5, device="cuda"), 2)
    assert of_none.shape == (0, 2) and w_none.shape == (0, 2)
    for change, text in (((x.half(), *args[1:]), "x must be bf16"), ((x, of[:3], *args[2:]), "must be \\[m=4"), ((x, of.long(), *args[2:]), "expert_of must be i32"),
                         ((x, of, weights.half(), *args[3:]), "weights f32"), ((x, of, weights, b_in[:2], *args[4:]), "s_gate_up must be"),
                         ((x[:, :128], *args[1:]), "b_gate_up must be"), ((x, of, weights, b_in, s_in, b_out, s_out, 64), "groupsize"),
                         ((x, of, weights, b_in, s_in, b_out.cpu(), s_out, g), "must be on"), ((x, of.repeat(1, 9), weights.repeat(1, 9), *args[3:]), "top_k must be")):
        with pytest.raises(marlin_gemm.MarlinGemmError, match=text):
            marlin_gemm.marlin_w4a16_moe(*change)
    logits = torch.zeros(3, 8, device="cuda")
    for call, text in (((logits, 0), "top_k"), ((logits, 9), "top_k"), ((logits.double(), 2), "f32, bf16 or f16"), ((logits[0], 2), "must be \\[m"),
                       ((torch.zeros(2, 1025, device="cuda"), 2), "1 to 1024"), ((logits.cpu(), 2), "on CUDA")):
        with pytest.raises(marlin_gemm.MarlinGemmError, match=text):
            marlin_gemm.moe_route(*call)
    with pytest.raises(moe.MarlinProjError, match="do not match"):
        moe.pack_experts(torch.zeros(2, 256, 128), torch.zeros(2, 256, 256), torch.zeros(2, 128, 256))
