"""swiglu_keep and swiglu_keep_backward against their definitions in 64 bits (parity unpinned: the reference keeps gate and up in bf16)."""
import pytest
import torch

from kiln_amd import marlin_gemm as mg

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8
FAST = 2.0 ** -18  # the reciprocal in f32, a few units, and the products around it


def off(gate):
    """Relative error of silu(gate) in f32.  exp(-gate) is 2^(gate * -log2 e): that product is rounded (2^-24) and so is its constant (2^-24 at most),
    each off by 2^-24 * 1.4427 |gate| in the exponent, which is 0.6931 times as much of the power: 2^-23 |gate| together."""
    return FAST + 2.0 ** -23 * gate.abs()


def near(got, want, relative, size):
    """size: what the reciprocal multiplies.  One below 2^-126 may be taken as zero; beyond what bf16 holds the result is infinite."""
    close = (got - want).abs() <= relative * want.abs() + 2.0 ** -126 * (1 + size.abs())
    return (close | ((want.abs() >= 2.0 ** 128 * (1 - 2.0 ** -9)) & (got == want.sign() * float("inf")))).all()


def split(v):
    both = v.reshape(len(v), -1, 2, 8)
    return both[:, :, 0].reshape(len(v), -1), both[:, :, 1].reshape(len(v), -1)


def joined(gate, up):
    m, n = gate.shape
    return torch.stack((gate.reshape(m, n // 8, 8), up.reshape(m, n // 8, 8)), 2).reshape(m, 2 * n)


def kept(v):
    """float64 values of gate or up [m, n] as they are kept, and (whole, exponent)."""
    blocks = v.double().reshape(len(v), -1, 32)
    most = blocks.abs().amax(2, keepdim=True)
    exponent = torch.where(most > 0, torch.floor(torch.log2(most.clamp_min(1e-45))), torch.full_like(most, -126.0)).clamp_min(-126) + 127
    exponent += (most >= torch.exp2(exponent - 126)).double() - (most < torch.exp2(exponent - 127)).double() * (exponent > 1)  # log2 next to a power of two
    whole = torch.round(blocks * torch.exp2(133 - exponent)).clamp(-127, 127)
    return (whole * torch.exp2(exponent - 133)).reshape(v.shape), whole.reshape(v.shape), exponent.squeeze(2)


def rows(seed, m, n):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, 2 * n), device="cuda", generator=g) * torch.exp(2 * torch.randn((m, 1), device="cuda", generator=g))
    return x.bfloat16(), (torch.randn((m, n), device="cuda", generator=g) * 0.01).bfloat16()


def check(gate_up, dh):
    h, whole, exponents = mg.swiglu_keep(gate_up)
    gate, up = (t.double() for t in split(gate_up))
    (kg, wg, eg), (ku, wu, eu) = kept(gate), kept(up)
    assert torch.equal(whole.double(), joined(wg, wu)) and torch.equal(exponents.double(), torch.stack((eg, eu), 2))
    want = gate * torch.sigmoid(gate) * up
    assert near(h.double(), want, HALF + off(gate), gate * up)
    d, again = mg.swiglu_keep_backward(dh, whole, exponents, recompute=True)
    assert torch.equal(d, mg.swiglu_keep_backward(dh, whole, exponents))
    s, g = torch.sigmoid(kg), dh.double()
    want = kg * s * ku
    assert near(again.double(), want, HALF + off(kg), kg * ku)
    d_gate, d_up = split(d.double())
    want = g * kg * s
    assert near(d_up, want, HALF + off(kg), g * kg)
    want, size = g * ku * s * (1 + kg * (1 - s)), (g * ku * s).abs() * (1 + kg.abs())
    assert ((d_gate - want).abs() <= HALF * want.abs() + off(kg) * size + 2.0 ** -126 * (1 + (g * ku).abs() * (1 + kg.abs()))).all()


@pytest.mark.parametrize("m,n", [(1, 128), (3, 256), (5, 1024), (17, 640), (100, 9216), (1000, 128)])
def test_against_the_definition(m, n):
    check(*rows(m + n, m, n))


def test_values_where_the_exponent_or_the_rounding_changes():
    n = 128
    special = [0.0, -0.0, 1.0, 1.0078125, 0.9921875, 2.0, 127.0, 127.5, 126.5, 63.5, 64.0, 0.5, 2.5, -2.5, 3.5, -127.5, 1e-38, 1.1754944e-38, 1e-40, 9.2e-41, 3.3e38, -3.3e38, 1e-20]
    g = torch.Generator(device="cuda").manual_seed(0)
    values = torch.tensor(special, device="cuda").bfloat16()
    x = values[torch.randint(0, len(special), (500, 2 * n), device="cuda", generator=g)]
    for i, v in enumerate(special):            # blocks of one magnitude, of zeros, and of one among small ones
        x[i] = v
        x[50 + i] = 0
        x[50 + i, :: 37] = v
        x[100 + i] = 0.25
        x[100 + i, 5::64] = v
    gate, up = split(x.double())
    (kg, wg, eg), (ku, wu, eu) = kept(gate), kept(up)
    _, whole, exponents = mg.swiglu_keep(x.contiguous())
    assert torch.equal(whole.double(), joined(wg, wu)) and torch.equal(exponents.double(), torch.stack((eg, eu), 2))
    for v, k in ((gate, kg), (up, ku)):        # the bound that the header gives, and that what is read back is a bf16 value
        most = v.abs().reshape(500, -1, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(v.shape)
        assert ((k - v).abs() <= 2.0 ** -7 * most + 2.0 ** -133).all() and torch.equal(k.float().bfloat16().double(), k)


def test_large_gates():
    x, dh = rows(7, 40, 256)
    x[:20] = (x[:20].float().sign() * 100).bfloat16()
    x[20:] = (x[20:].float().sign() * 1e30).bfloat16()
    x[20:, 1::2] = 1.0
    check(x, dh)


def test_blocks_without_numbers_are_nan_and_alone():
    x, dh = rows(9, 4, 128)
    x[1, 3], x[2, 64 + 9], x[3, 130] = float("nan"), float("inf"), -float("inf")   # gate of block 0, up of block 1, gate of block 2
    h, whole, exponents = mg.swiglu_keep(x)
    assert [tuple(i) for i in (exponents == 255).nonzero().tolist()] == [(1, 0, 0), (2, 1, 1), (3, 2, 0)]
    d, again = mg.swiglu_keep_backward(dh, whole, exponents, recompute=True)
    bad = torch.zeros((4, 128), dtype=torch.bool, device="cuda")
    bad[1, 0:32], bad[2, 32:64], bad[3, 64:96] = True, True, True
    assert torch.equal(torch.isnan(again), bad)
    d_gate, d_up = split(d)
    gate_bad = bad.clone()
    assert torch.equal(torch.isnan(d_gate), gate_bad)
    gate_bad[2] = False                        # d_up does not read up
    assert torch.equal(torch.isnan(d_up), gate_bad)


def test_gradient_against_differences():
    """d_gate_up is the derivative of sum(dh * h) where h is formed from the kept values: central differences in 64 bits."""
    x, dh = rows(21, 6, 128)
    _, whole, exponents = mg.swiglu_keep(x)
    d_gate, d_up = split(mg.swiglu_keep_backward(dh, whole, exponents).double())
    gate, up = split(x.double())
    kg, ku = kept(gate)[0], kept(up)[0]
    f = lambda a, b: dh.double() * a * torch.sigmoid(a) * b
    step = 1e-4 * (1 + kg.abs())
    want = (f(kg + step, ku) - f(kg - step, ku)) / (2 * step)
    assert ((d_gate - want).abs() <= 1.01 * HALF * want.abs() + 1e-6 * (dh.double() * ku).abs() * (1 + kg.abs())).all()
    want = (f(kg, ku + 1) - f(kg, ku - 1)) / 2
    assert ((d_up - want).abs() <= 1.01 * HALF * want.abs() + 1e-9 * dh.double().abs()).all()


def test_strided_rows_and_none():
    x, dh = rows(30, 8, 256)
    wide = torch.cat((x, x), 1)[:, :512]
    assert not wide.is_contiguous()
    for a, b in zip(mg.swiglu_keep(wide), mg.swiglu_keep(x)):
        assert torch.equal(a, b)
    h, whole, exponents = mg.swiglu_keep(x[:0])
    assert h.shape == (0, 256) and whole.shape == (0, 512) and exponents.shape == (0, 8, 2)
    assert mg.swiglu_keep_backward(dh[:0], whole, exponents).shape == (0, 512)
