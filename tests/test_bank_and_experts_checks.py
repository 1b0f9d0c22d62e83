"""What the C entry points of banks, experts and routers refuse, before anything is launched (no GPU is touched), their scratch sizes, and
the host side of a bank.  CPU only: the pointers handed over are never followed."""
import ctypes

import pytest
import torch

from kiln_amd import _lib, lora, marlin_gemm
from kiln_amd.marlin_proj import MarlinPackedProj, MarlinProjError

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)
Y, Y2, Y3 = (ctypes.c_void_p(i << 40) for i in (1, 2, 3))      # results, which share no memory with operands


def bank(a=P, b=P, scales=P, count=3, rank=16):
    return ctypes.byref(_lib.AdapterBank(a, b, scales, count, rank))


def forward(m=4, n=512, k=256, g=128, x=P, w=P, y=Y, s=P, ws=P, bk=None, of=P, scratch=P):
    return _lib.load().kiln_w4a16_gemm_bank(x, w, y, s, m, n, k, ws, g, 0, None, bank() if bk is None else bk, of, scratch)


def backward(m=4, n=512, k=256, g=128, dy=P, x=P, w=P, s=P, bk=None, of=P, dx=Y, da=Y2, db=Y3, scratch=P):
    return _lib.load().kiln_w4a16_gemm_bank_backward(dy, x, w, s, m, n, k, g, 0, None, bank() if bk is None else bk, of, dx, da, db, scratch)


def experts(m=4, top=2, count=8, hidden=256, n_out=128, n_down=256, g=128, x=P, of=P, weights=P, packs=(P, P, P, P), y=Y, scratch=P):
    return _lib.load().kiln_w4a16_moe(x, of, weights, *packs, y, m, top, count, hidden, n_out, n_down, g, 0, None, scratch)


def route(m=4, count=8, top=2, dtype=0, logits=P, of=P, weights=P):
    return _lib.load().kiln_w4a16_moe_route(logits, dtype, m, count, top, 1, of, weights, 0, None)


@pytest.mark.parametrize("call", [forward, backward])
def test_a_bank_call_refuses(call):
    for m in (4, 40, 400):
        for kw in (dict(n=300), dict(k=200), dict(g=64), dict(m=-1), dict(n=-256), dict(k=-128)):
            assert call(**{"m": m, **kw}) == _lib.ERR_PROB_SHAPE, kw
        for rank in (0, 4, 12, 72, -8):
            assert call(m=m, bk=bank(rank=rank)) == _lib.ERR_KERN_SHAPE
        for count in (0, -1, 4097):
            assert call(m=m, bk=bank(count=count)) == _lib.ERR_KERN_SHAPE
        for kw in (dict(a=None), dict(b=None), dict(scales=None), dict(a=ODD), dict(b=ODD)):
            assert call(m=m, bk=bank(**kw)) == _lib.ERR_ARGUMENT, kw
        for kw in (dict(x=None), dict(w=None), dict(s=None), dict(of=None), dict(scratch=None), dict(x=ODD), dict(w=ODD), dict(s=ODD), dict(scratch=ODD)):
            assert call(m=m, **kw) == _lib.ERR_ARGUMENT, kw
        own = (dict(y=None), dict(ws=None), dict(y=ODD), dict(ws=ODD)) if call is forward else \
            (dict(dy=None), dict(dx=None), dict(da=None), dict(db=None), dict(dy=ODD), dict(dx=ODD), dict(da=ODD), dict(db=ODD))
        for kw in own:
            assert call(m=m, **kw) == _lib.ERR_ARGUMENT, kw


def test_results_that_share_memory_with_operands_are_refused():
    at = lambda base, bytes: ctypes.c_void_p(base.value + bytes)
    for m in (4, 40, 400):
        last = at(P, 2 * m * 256 - 16)                 # the last 16 bytes of x
        for kw in (dict(y=P), dict(y=last), dict(x=at(Y, 2 * m * 512 - 16)), dict(y=at(P, 2 * 3 * 16 * 512 - 16), x=Y2), dict(bk=bank(a=at(Y, 16)))):
            assert forward(m=m, **kw) == _lib.ERR_ARGUMENT, kw
        for kw in (dict(dx=P), dict(dx=last), dict(da=P), dict(db=P), dict(dy=at(Y, 16)), dict(dy=Y2), dict(x=Y3), dict(bk=bank(b=Y2)), dict(bk=bank(a=at(Y3, 32)))):
            assert backward(m=m, **kw) == _lib.ERR_ARGUMENT, kw
        for kw in (dict(y=P), dict(y=last), dict(x=at(Y, 2 * m * 256 - 16))):
            assert experts(m=m, **kw) == _lib.ERR_ARGUMENT, kw


def test_a_gradient_of_a_bank_needs_the_rows_adapters():
    x, dy = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, 512, dtype=torch.bfloat16)
    packed = MarlinPackedProj(torch.zeros(16, 1024, dtype=torch.int32), torch.zeros(2, 512, dtype=torch.float16), 128, 256, 512)
    made = lora.AdapterBank(torch.zeros(1, 8, 256, dtype=torch.bfloat16), torch.zeros(1, 512, 8, dtype=torch.bfloat16), torch.ones(1))
    with pytest.raises(MarlinProjError, match="adapter_of"):
        lora.proj_backward_bank(dy, x, packed, made)


def test_calls_without_work_are_no_errors():
    assert forward(m=0) == _lib.OK
    none = ctypes.POINTER(_lib.AdapterBank)()
    assert _lib.load().kiln_w4a16_gemm_bank_backward(None, None, None, None, 0, 512, 256, 128, 0, None, none, None, None, None, None, None) == _lib.OK
    assert experts(m=0) == _lib.OK and route(m=0) == _lib.OK


def test_a_backward_without_a_bank_needs_no_more_than_its_operands():
    L, none = _lib.load(), ctypes.POINTER(_lib.AdapterBank)()
    for missing in range(5):
        p = [P] * 5
        p[missing] = None
        assert L.kiln_w4a16_gemm_bank_backward(p[0], None, p[1], p[2], 4, 512, 256, 128, 0, None, none, None, p[3], None, None, p[4]) == _lib.ERR_ARGUMENT


def test_experts_and_routers_refuse():
    for kw in (dict(hidden=200), dict(n_out=64), dict(n_down=128), dict(g=32), dict(m=-1), dict(hidden=0), dict(n_out=0), dict(n_down=0), dict(n_out=1 << 30)):
        assert experts(**kw) == _lib.ERR_PROB_SHAPE, kw
    for kw in (dict(top=0), dict(top=17), dict(count=0), dict(count=1025)):
        assert experts(**kw) == _lib.ERR_KERN_SHAPE, kw
    for kw in (dict(x=None), dict(of=None), dict(weights=None), dict(y=None), dict(scratch=None), dict(x=ODD), dict(y=ODD), dict(scratch=ODD),
               *(dict(packs=tuple(bad if i == j else P for j in range(4))) for i in range(4) for bad in (None, ODD))):
        assert experts(**kw) == _lib.ERR_ARGUMENT, kw
    for kw in (dict(top=0), dict(top=17, count=64), dict(top=9), dict(count=0), dict(count=1025), dict(dtype=3), dict(dtype=-1)):
        assert route(**kw) == _lib.ERR_KERN_SHAPE, kw
    assert route(m=-1) == _lib.ERR_PROB_SHAPE
    for kw in (dict(logits=None), dict(of=None), dict(weights=None)):
        assert route(**kw) == _lib.ERR_ARGUMENT, kw


def test_scratch_of_a_forward_never_decreases_with_rows():
    L = _lib.load()
    for n, k, count, rank in ((2560, 2560, 4, 8), (18432, 2560, 64, 64), (2560, 9216, 1, 16), (256, 128, 4096, 64), (4096, 14336, 8, 32)):
        sizes = [L.kiln_w4a16_gemm_bank_scratch_bytes(m, n, k, count, rank) for m in range(1, 1200)]
        assert sizes == sorted(sizes)
        for m in (1, 16, 17, 256, 257, 1199):          # order, first and at least one slice of the projection
            assert sizes[m - 1] >= 4 * m + 4 * (count + 2) + 4 * m * rank
    assert L.kiln_w4a16_gemm_bank_backward_scratch_bytes(0, 512, 256, 3, 16) == L.kiln_w4a16_gemm_bank_backward_scratch_bytes(1, 512, 256, 3, 16)
    assert L.kiln_w4a16_moe_scratch_bytes(1000, 8, 1024, 2560) == L.kiln_w4a16_moe_scratch_bytes(64, 8, 1024, 2560) >= 64 * 8 * (2 * 1024 + 4 * 2560)


def test_a_bank_made_of_adapters_of_several_ranks():
    gen = torch.Generator().manual_seed(0)
    ads = [lora.LoraProjectionWeights(torch.randn(r, 96, generator=gen).bfloat16(), torch.randn(40, r, generator=gen).bfloat16()) for r in (3, 16, 9)]
    made = lora.make_bank(ads, [0.5, 1, 2.0])
    assert made.a.shape == (3, 16, 96) and made.b.shape == (3, 40, 16) and made.scales.tolist() == [0.5, 1.0, 2.0]
    for p, a, b in zip(ads, made.a, made.b):
        r = p.a.shape[0]
        assert torch.equal(a[:r], p.a) and torch.equal(b[:, :r], p.b) and not bool(a[r:].any()) and not bool(b[:, r:].any())
    for bad in (([], []), (ads, [1.0]), ([ads[0], lora.LoraProjectionWeights(ads[1].a[:, :95], ads[1].b)], [1, 1])):
        with pytest.raises(MarlinProjError):
            lora.make_bank(*bad)


def test_calls_on_tensors_of_the_host_are_refused():
    x, of = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    b, s = torch.zeros(16, 512, dtype=torch.int32), torch.zeros(2, 256, dtype=torch.float16)
    a_, b_, sc = torch.zeros(1, 8, 256, dtype=torch.bfloat16), torch.zeros(1, 256, 8, dtype=torch.bfloat16), torch.ones(1)
    for call in (lambda: marlin_gemm.marlin_w4a16_gemm_bank(x, b, s, 128, a_, b_, sc, of), lambda: marlin_gemm.marlin_w4a16_gemm_bank_backward(x, x, b, s, 128, a_, b_, sc, of),
                 lambda: marlin_gemm.marlin_w4a16_gemm_backward(x, b, s, 128), lambda: marlin_gemm.moe_route(torch.zeros(2, 4), 2),
                 lambda: marlin_gemm.marlin_w4a16_moe(x, of[:, None], torch.ones(2, 1), b[None], s[None], b[None], s[None], 128)):
        with pytest.raises(marlin_gemm.MarlinGemmError, match="on CUDA"):
            call()
