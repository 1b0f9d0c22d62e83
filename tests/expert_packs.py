"""What the tests of products with experts share: packs made from random codes, and what they stand for in 64 bits."""
import math

import torch

NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)


def packs(gen, experts, k, n, g):
    """(b int32 [experts, k/16, 2n], s f16 [experts, groups, n]) on the GPU: uniform codes, scales that give entries of about 1 / sqrt(k)."""
    b = torch.randint(-2 ** 31, 2 ** 31 - 1, (experts, k // 16, 2 * n), dtype=torch.int64, device="cuda", generator=gen).to(torch.int32)
    s = (torch.rand((experts, 1 if g == -1 else k // 128, n), device="cuda", generator=gen) + 0.5) / (4.6 * math.sqrt(k))
    return b, s.half()


def weight(b, s):
    """One pack as float64 [k, n] (kiln_amd/csrc/layout.h's definition)."""
    k, n, groups = b.shape[0] * 16, b.shape[1] // 2, s.shape[0]
    shifts = torch.tensor([4 * p for p in NIBBLE], dtype=torch.int32, device=b.device)
    codes = ((b.reshape(n // 16, k // 128, 4, 16, 4, 1) >> shifts) & 15).permute(1, 4, 2, 5, 0, 3).reshape(k, n)
    scale = s.reshape(n // 16, groups, 16).permute(1, 0, 2).reshape(groups, 1, n).double()
    return ((codes - 8).double().reshape(groups, k // groups, n) * scale).reshape(k, n)


def choice(gen, m, top, experts, away=0):
    """expert_of i32 [m, top]: different experts of a token, the last `away` experts as -1."""
    of = torch.rand((m, max(experts, top)), device="cuda", generator=gen).argsort(1)[:, :top]
    return torch.where(of >= experts - away, -1, of).to(torch.int32)


def sorted_by_hand(of, experts):
    """(order, first, place) of a choice, from the definition."""
    flat = of.reshape(-1).tolist()
    order = sorted(range(len(flat)), key=lambda p: (flat[p] if 0 <= flat[p] < experts else experts, p))
    first = [sum(1 for e in flat if 0 <= e < limit) for limit in range(experts + 1)]
    place = [0] * len(flat)
    for position, pair in enumerate(order):
        place[pair] = position
    return tuple(torch.tensor(v, dtype=torch.int32, device=of.device) for v in (order, first)) + (
        torch.tensor(place, dtype=torch.int32, device=of.device).reshape(of.shape),)


def silu_times(y):
    """silu(gate) * up of float64 columns in the packed order."""
    n = y.shape[1] // 2
    both = y.reshape(len(y), n // 8, 2, 8)
    gate, up = both[:, :, 0].reshape(len(y), n), both[:, :, 1].reshape(len(y), n)
    return gate * torch.sigmoid(gate) * up
