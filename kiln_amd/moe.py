"""A mixture-of-experts MLP on packed experts: the router's choice, the experts it names, their sum.

The reference's model family is dense (crates/kiln-core/src/config.rs:78-101): its MLP is `marlin_gemm.marlin_w4a16_mlp`
(crates/kiln-model/src/forward.rs:2723-2848), of which every expert here is one.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import marlin_gemm
from .marlin_proj import MarlinProjError


@dataclass
class MoeExperts:
    """The packs of a layer's experts, one after the other: `marlin_gemm.marlin_w4a16_moe`'s operands."""
    b_gate_up: torch.Tensor   # [experts, hidden/16, 4 n_out] int32
    s_gate_up: torch.Tensor   # [experts, hidden/groupsize, 2 n_out] f16
    b_down: torch.Tensor      # [experts, n_out/16, 2 n_down] int32
    s_down: torch.Tensor      # [experts, n_out/groupsize, n_down] f16
    groupsize: int


def pack_experts(gate_t: torch.Tensor, up_t: torch.Tensor, down_t: torch.Tensor, groupsize: int = 128) -> MoeExperts:
    """Quantise and pack the experts of a layer: `gate_t`, `up_t` bf16 `[experts, hidden, n_out]` and `down_t` `[experts, n_out, n_down]`
    on the GPU (`weight_t` of the other packing calls with the experts in front).  Gate and up are interleaved, 8 columns of one and 8 of
    the other, as `pack.interleave_gate_up` does with packed ones: a column's codes do not depend on its neighbours."""
    if gate_t.dim() != 3 or gate_t.shape != up_t.shape or down_t.dim() != 3 or down_t.shape[0] != gate_t.shape[0] or \
            down_t.shape[1] != gate_t.shape[2] or gate_t.shape[0] == 0:
        raise MarlinProjError(f"pack_experts: gate {tuple(gate_t.shape)}, up {tuple(up_t.shape)} and down {tuple(down_t.shape)} do not match "
                              "[experts, hidden, n_out] twice and [experts, n_out, n_down]")
    experts, hidden, n_out = gate_t.shape
    if hidden % 128 or n_out % 128 or down_t.shape[2] % 256:
        raise MarlinProjError(f"pack_experts: hidden={hidden} and n_out={n_out} must be multiples of 128, n_down={down_t.shape[2]} of 256")
    packs = []
    for e in range(experts):
        both = torch.stack((gate_t[e].reshape(hidden, n_out // 8, 8), up_t[e].reshape(hidden, n_out // 8, 8)), dim=2).reshape(hidden, 2 * n_out)
        packs.append((*marlin_gemm.pack.quantize_and_pack_device(both, groupsize), *marlin_gemm.pack.quantize_and_pack_device(down_t[e], groupsize)))
    return MoeExperts(*(torch.stack(part) for part in zip(*packs)), groupsize)


def moe_forward(x: torch.Tensor, router_t: torch.Tensor, experts: MoeExperts, top_k: int, renormalise: bool = True) -> torch.Tensor:
    """The whole layer: `x` bf16 `[..., hidden]`, `router_t` bf16 `[hidden, experts]` (its product stays on bf16, as the reference leaves every
    narrow projection: crates/kiln-model/src/marlin_proj.rs:53-55), then `moe_route` and `marlin_w4a16_moe`."""
    rows = x.reshape(-1, x.shape[-1])
    expert_of, weights = marlin_gemm.moe_route(rows @ router_t, top_k, renormalise)
    y = marlin_gemm.marlin_w4a16_moe(rows, expert_of, weights, experts.b_gate_up, experts.s_gate_up, experts.b_down, experts.s_down,
                                     experts.groupsize)
    return y.reshape(*x.shape[:-1], y.shape[-1])
