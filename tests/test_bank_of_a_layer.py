"""A bank beside a layer's projection that stayed on bf16, and what makes a bank.  CPU only."""
import pytest
import torch

from kiln_amd import lora
from kiln_amd.layer_pack import LayerProjections, PackKind
from kiln_amd.marlin_proj import MarlinProjError


def layer_and_bank(k=96, n=40, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(0)
    rand = lambda *shape: torch.randn(shape, generator=gen)
    adapters = [lora.LoraProjectionWeights((rand(r, k) / k ** 0.5).bfloat16(), (rand(n, r) / r ** 0.5).bfloat16()) for r in (8, 3)]
    return LayerProjections({PackKind.QProj: (rand(k, n) / k ** 0.5).to(dtype)}), lora.make_bank(adapters, (0.5, 2.0)), rand


@pytest.mark.parametrize("shape", [(0,), (2, 0), (0, 3)])
def test_no_rows(shape):
    layer, bank, _ = layer_and_bank()
    y = layer.forward_bank(PackKind.QProj, torch.empty(*shape, 96, dtype=torch.bfloat16), bank, torch.empty(shape, dtype=torch.int32))
    assert y.shape == (*shape, 40) and y.dtype == torch.bfloat16


@pytest.mark.parametrize("rows", [0, 3, 5, 12])
def test_a_count_of_adapters_that_is_not_the_rows_is_refused(rows):
    layer, bank, rand = layer_and_bank()
    with pytest.raises(MarlinProjError, match="adapter_of"):
        layer.forward_bank(PackKind.QProj, rand(2, 3, 96).bfloat16(), bank, torch.zeros(rows, dtype=torch.int32))


def test_rows_of_several_adapters():
    """U = 2^-8 for each rounding to bf16: the base, the two products of the term, its scaled value and the sum; f32 sums beside it."""
    layer, bank, rand = layer_and_bank()
    x, of = rand(2, 5, 96).bfloat16(), torch.tensor([[0, 1, -1, 1, 2], [0, 0, 7, 1, -3]], dtype=torch.int32)
    y = layer.forward_bank(PackKind.QProj, x, bank, of).double().reshape(10, 40)
    rows, w = x.double().reshape(10, 96), layer.weights_t[PackKind.QProj].double()
    base = rows @ w
    want, bound = base.clone(), 2 ** -8 * base.abs() + 96 * 2 ** -24 * (rows.abs() @ w.abs())
    for j in range(2):
        mine, a, b, s = of.reshape(10) == j, bank.a[j].double(), bank.b[j].double(), bank.scales[j].double()
        want[mine] += s * (rows[mine] @ a.t()) @ b.t()
        bound[mine] += s * (rows[mine].abs() @ a.abs().t()) @ b.abs().t() * (3 * 2 ** -8 + (96 + 8) * 2 ** -24)
    assert bool(((y - want).abs() <= (bound + 2 ** -8 * want.abs()) * (1 + 2 ** -6)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_of_another_type_as_forward_takes_them(dtype):
    layer, bank, rand = layer_and_bank(dtype=dtype)
    x, of = rand(4, 96).to(dtype), torch.tensor([1, -1, 1, 1], dtype=torch.int32)
    y, alone = layer.forward_bank(PackKind.QProj, x, bank, of), layer.forward(PackKind.QProj, x, lora.LoraProjectionWeights(bank.a[1], bank.b[1]), 2.0)
    assert y.dtype == dtype and torch.equal(y[of == 1], alone[of == 1]) and torch.equal(y[1], layer.forward(PackKind.QProj, x)[1])


def test_ranks_that_no_call_takes_make_no_bank():
    adapter = lambda rank: lora.LoraProjectionWeights(torch.zeros(rank, 96, dtype=torch.bfloat16), torch.zeros(40, rank, dtype=torch.bfloat16))
    for ranks in ((65,), (8, 72), (0,), (0, 0)):
        with pytest.raises(MarlinProjError, match="rank"):
            lora.make_bank([adapter(r) for r in ranks], [1.0] * len(ranks))
    assert lora.make_bank([adapter(64), adapter(0)], [1.0, 1.0]).a.shape == (2, 64, 96)
