"""A mixture of experts for many tokens as it is used: forward, forward in training and backward, on experts made by pack_experts; from several streams
and from a captured graph; and the dense MLP in training (parity unpinned: the reference trains neither on packed weights)."""
import pytest
import torch

from kiln_amd import _lib, marlin_gemm as mg, moe
from tests.expert_packs import choice, packs, silu_times, weight

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def experts_of(r, count, hidden, n_out, n_down, g):
    made = [(torch.randn((count, *shape), device="cuda", generator=r) / shape[0] ** 0.5).bfloat16() for shape in ((hidden, n_out), (hidden, n_out), (n_out, n_down))]
    return moe.pack_experts(*made, groupsize=g)


def exact(x, of, weights, e):
    """(y, gate, up by pair) in 64 bits."""
    m, top = of.shape
    y = torch.zeros((m, e.s_down.shape[2]), dtype=torch.float64, device="cuda")
    for i in range(len(e.b_down)):
        rows, place = torch.nonzero(of == i, as_tuple=True)
        h = silu_times(x[rows].double() @ weight(e.b_gate_up[i], e.s_gate_up[i]))
        y.index_add_(0, rows, (h @ weight(e.b_down[i], e.s_down[i])) * weights[rows, place].double()[:, None])
    return y


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("m,top,count,away,hidden,n_out,n_down,g", [(1, 2, 4, 0, 256, 128, 256, 128), (37, 4, 8, 2, 384, 256, 512, 128), (300, 8, 16, 0, 512, 384, 256, -1),
                                                                    (700, 2, 4, 1, 256, 256, 768, 128)])
def test_forward_and_backward(m, top, count, away, hidden, n_out, n_down, g):
    r = gen(m + hidden)
    e = experts_of(r, count, hidden, n_out, n_down, g)
    of = choice(r, m, top, count, away)
    if m > 10:
        of[3] = -1                                       # a token without experts here
        of[5, 1] = of[5, 0]                              # and one that names an expert twice
    weights = torch.rand((m, top), device="cuda", generator=r)
    x, dy = (torch.randn((m, w), device="cuda", generator=r).bfloat16() for w in (hidden, n_down))
    want = exact(x, of, weights, e)
    # roundings to bf16, 2^-8 of a value at most: h, the pairs' rows, y; in training gate and up as well, on which h depends with a slope of about one each
    y = moe.experts_many(x, of, weights, e)
    assert off(y, want) <= 3 * 2.0 ** -8
    trained, kept = moe.experts_keep(x, of, weights, e)
    assert off(trained, want) <= 5 * 2.0 ** -8
    if m > 10:
        assert not y[3].any() and not trained[3].any()

    # the backward pass from what was kept, in 64 bits: what is left are the roundings to bf16 of d_rows, dh, d_gate_up, their rows and dx and of two products'
    # weights, each 2^-8 of a value at most
    dx, d_weights = moe.experts_backward(dy, kept, e)
    bounds, order = kept.first.tolist(), kept.place.reshape(-1).argsort()
    scale = torch.exp2(kept.exponents.double() - 133).repeat_interleave(32, 1)                # [pairs, n_out, (gate, up)]
    whole = kept.whole.double().reshape(len(order), n_out // 8, 2, 8)
    gate, up = whole[:, :, 0].reshape(len(order), n_out) * scale[..., 0], whole[:, :, 1].reshape(len(order), n_out) * scale[..., 1]
    want_x, want_w = torch.zeros((m, hidden), dtype=torch.float64, device="cuda"), torch.zeros(m * top, dtype=torch.float64, device="cuda")
    for i in range(count):
        pairs = order[bounds[i]:bounds[i + 1]]
        at = slice(bounds[i], bounds[i + 1])
        d = dy.double()[pairs // top]
        want_w[pairs] = (d * kept.rows[at].double()).sum(1)
        dh = (d * weights.reshape(-1)[pairs].double()[:, None]) @ weight(e.b_down[i], e.s_down[i]).t()
        s = torch.sigmoid(gate[at])
        both = torch.stack(((dh * up[at] * s * (1 + gate[at] * (1 - s))).reshape(len(pairs), n_out // 8, 8), (dh * gate[at] * s).reshape(len(pairs), n_out // 8, 8)), 2)
        want_x.index_add_(0, pairs // top, both.reshape(len(pairs), 2 * n_out) @ weight(e.b_gate_up[i], e.s_gate_up[i]).t())
    assert off(dx, want_x) <= 7 * 2.0 ** -8 and off(d_weights.reshape(-1), want_w) <= 2.0 ** -18
    if m > 10:
        assert not dx[3].any() and not d_weights[3].any()


def test_the_whole_layer_beside_the_call_for_a_few_tokens():
    r = gen(4)
    e = experts_of(r, 8, 256, 256, 256, 128)
    x = torch.randn((3, 40, 256), device="cuda", generator=r).bfloat16()
    router = torch.randn((256, 8), device="cuda", generator=r).bfloat16()
    a, b = moe.moe_forward_many(x, router, e, 2), moe.moe_forward(x, router, e, 2)
    assert a.shape == b.shape == (3, 40, 256) and off(a, b) <= 4 * 2.0 ** -8    # h in both, the pairs' rows in one, y in both


def test_every_kind_of_block_is_taken_by_some_size():
    """The sizes that the tests of products and gradients run, on this part: each of the six kinds in both directions."""
    from tests import test_gpu_experts_many as t
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    plan = lambda *a: _lib.load().kiln_w4a16_debug_experts_plan(*a, cus)
    sizes = [(sum(c), n, k, len(c) - 1) for c in t.COUNTS for k, n in ((128, 256), (384, 512), (256, 768), (1152, 256))] + \
            [(3000, 2048, 2560, 2), (700, 2560, 2048, 32), (100, 2048, 2560, 64), (4096, 2560, 1024, 8)] + SIZES
    for backward in (0, 1):
        assert {plan(*s, backward) for s in sizes} == {0, 1, 2, 3, 4, 5}


SIZES = [(768, 2048, 512, 64), (1600, 512, 2048, 64), (3000, 2048, 512, 64), (3000, 512, 2048, 64), (6000, 1024, 1024, 32), (5000, 512, 512, 4),
         (360, 2560, 1024, 64), (400, 2048, 2560, 16), (800, 2048, 1280, 32), (1500, 2560, 1024, 64), (2331, 2048, 1280, 24),
         (850, 2560, 1280, 4), (2350, 1024, 1280, 16), (1350, 1024, 512, 16), (500, 512, 2560, 8), (1000, 512, 512, 8), (2000, 1024, 1024, 3)]


@pytest.mark.parametrize("rows,n,k,experts", SIZES)
def test_sizes_of_every_kind_of_block(rows, n, k, experts):
    from tests.test_gpu_experts_many import check_backward, check_forward
    r = gen(rows + n)
    cuts = torch.sort(torch.randint(0, rows + 1, (experts,), device="cuda", generator=r)).values
    first = torch.cat((cuts.new_zeros(1), cuts)).to(torch.int32)                              # ragged, and rows of no expert behind
    b, s = packs(r, experts, k, n, 128)
    x, dy = (torch.randn((rows, w), device="cuda", generator=r).bfloat16() for w in (k, n))
    for swiglu in (False, True):
        check_forward(x, first, b, s, 128, swiglu)
    check_backward(dy, first, b, s, 128)


def run_of(seed):
    r = gen(seed)
    e = experts_of(r, 8, 256, 256, 256, 128)
    calls = []
    for m in (1, 50, 900):
        of, weights = choice(r, m, 4, 8, 1), torch.rand((m, 4), device="cuda", generator=r)
        x, dy = (torch.randn((m, 256), device="cuda", generator=r).bfloat16() for _ in range(2))
        calls.append((x, of, weights, dy))

    def run():
        made = []
        for x, of, weights, dy in calls:
            y, kept = moe.experts_keep(x, of, weights, e)
            dx, d_weights = moe.experts_backward(dy, kept, e)
            order, first, place = mg.moe_sort(of, 8)
            made += [moe.experts_many(x, of, weights, e), y, dx, d_weights, mg.moe_gather(x, first, place), order]
            made += mg.swiglu_keep_backward(dy, kept.whole[:len(x)].contiguous(), kept.exponents[:len(x)].contiguous(), recompute=True)
        return made

    return run, calls


def test_streams_and_graphs_at_once():
    made = [run_of(seed) for seed in range(4)]
    runs = [m[0] for m in made]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs, captured = [], []
    for i in (2, 3):                                   # two graphs: each has its own scratch
        with torch.cuda.stream(streams[i]):
            runs[i]()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[i]):
            captured.append(runs[i]())
    for _ in range(4):
        for t in captured[0] + captured[1]:
            t.zero_()
        torch.cuda.synchronize()
        eager = [None, None]
        for i in range(2):
            with torch.cuda.stream(streams[2 + i]):
                graphs[i].replay()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                eager[i] = runs[i]()
        torch.cuda.synchronize()
        for got, expected in zip((*eager, *captured), want):
            assert len(got) == len(expected) and all(map(torch.equal, got, expected))
    # other choices, weights and rows in a graph's operands: what a replay gives is the eager call's
    x, of, weights, dy = made[2][1][2]
    r = gen(99)
    of.copy_(choice(r, *of.shape, 8, 3))
    x.copy_(torch.randn(x.shape, device="cuda", generator=r))
    with torch.cuda.stream(streams[2]):
        graphs[0].replay()
    torch.cuda.synchronize()
    assert all(map(torch.equal, captured[0], runs[2]()))


@pytest.mark.parametrize("m", [1, 45, 300])
def test_a_dense_mlp_in_training(m):
    r = gen(m)
    (gate_up, s_in), (down, s_out) = ((t[0] for t in packs(r, 1, 256, 512, 128)), (t[0] for t in packs(r, 1, 256, 256, 128)))
    x, dy = (torch.randn((m, 256), device="cuda", generator=r).bfloat16() for _ in range(2))
    y, whole, exponents = mg.marlin_w4a16_mlp_keep(x, gate_up, s_in, down, s_out, 128)
    w_in, w_out = weight(gate_up, s_in), weight(down, s_out)
    inner = x.double() @ w_in
    assert off(y, silu_times(inner) @ w_out) <= 4 * 2.0 ** -8
    assert off(y, mg.marlin_w4a16_mlp(x, gate_up, s_in, down, s_out, 128)) <= 6 * 2.0 ** -8
    dx = mg.marlin_w4a16_mlp_backward(dy, whole, exponents, gate_up, s_in, down, s_out, 128)
    scale = torch.exp2(exponents.double() - 133).repeat_interleave(32, 1)
    v = whole.double().reshape(m, 32, 2, 8)
    gate, up = v[:, :, 0].reshape(m, 256) * scale[..., 0], v[:, :, 1].reshape(m, 256) * scale[..., 1]
    dh, s = dy.double() @ w_out.t(), torch.sigmoid(gate)
    d = torch.stack(((dh * up * s * (1 + gate * (1 - s))).reshape(m, 32, 8), (dh * gate * s).reshape(m, 32, 8)), 2).reshape(m, 512)
    assert off(dx, d @ w_in.t()) <= 5 * 2.0 ** -8
    # against the gradient of the exact function: gate and up are off by 2^-7 of their block's largest, three times a typical value, at most
    both = inner.reshape(m, 32, 2, 8)
    gate, up = both[:, :, 0].reshape(m, 256), both[:, :, 1].reshape(m, 256)
    s = torch.sigmoid(gate)
    d = torch.stack(((dh * up * s * (1 + gate * (1 - s))).reshape(m, 32, 8), (dh * gate * s).reshape(m, 32, 8)), 2).reshape(m, 512)
    assert off(dx, d @ w_in.t()) <= 5 * 2.0 ** -8 + 2 * 3 * 2.0 ** -7
