"""A mixture-of-experts MLP on packed experts: the router's choice, the experts it names, their sum; for a few tokens as one call, for many with their
rows in the order of the experts, and with its gradients.

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


def experts_many(x: torch.Tensor, expert_of: torch.Tensor, weights: torch.Tensor, experts: MoeExperts) -> torch.Tensor:
    """`marlin_w4a16_moe` for many tokens: the choices sorted by expert, gate, up and `silu(gate) * up` straight from the tokens, the down projection, and
    the rows back to their tokens with their weights.  `x` bf16 `[m, hidden]`, `expert_of` i32 and `weights` f32 `[m, top_k]`.  (`marlin_w4a16_moe` reads the
    packs of a run of 64 tokens' experts for every run; here they are read once.  A pair's row is rounded to bf16 before the sum.)"""
    order, first, place = marlin_gemm.moe_sort(expert_of, experts.b_down.shape[0])
    h = marlin_gemm.marlin_w4a16_gemm_experts(x, first, experts.b_gate_up, experts.s_gate_up, experts.groupsize, order=order, top_k=expert_of.shape[1],
                                              swiglu=True)
    rows = marlin_gemm.marlin_w4a16_gemm_experts(h, first, experts.b_down, experts.s_down, experts.groupsize)
    return marlin_gemm.moe_combine(rows, weights, first, place)


def moe_forward_many(x: torch.Tensor, router_t: torch.Tensor, experts: MoeExperts, top_k: int, renormalise: bool = True) -> torch.Tensor:
    """`moe_forward` for many tokens (`experts_many`): a prefill.  Worth it from 65 tokens on, where `marlin_w4a16_moe` reads packs a second time (64 experts, top 8,
    2560 -> 1024 -> 2560: 64 tokens 71 us here and 60 there, 96 tokens 71 and 113, 256 tokens 90 and 243)."""
    rows = x.reshape(-1, x.shape[-1])
    expert_of, weights = marlin_gemm.moe_route(rows @ router_t, top_k, renormalise)
    y = experts_many(rows, expert_of, weights, experts)
    return y.reshape(*x.shape[:-1], y.shape[-1])


@dataclass
class MoeKept:
    """What `experts_backward` needs of a forward pass: the order, the experts' rows (for the weights' gradient), and gate and up in 8 bits.  The rows stay
    in bf16: of a pair 2 n_down bytes beside the 2.0625 n_out of gate and up, 5120 beside 2112 at 1024 -> 2560, where gate and up in bf16 would be 4096."""
    first: torch.Tensor
    place: torch.Tensor
    weights: torch.Tensor
    rows: torch.Tensor        # bf16 [m * top_k, n_down]
    whole: torch.Tensor       # i8 [m * top_k, 2 n_out]
    exponents: torch.Tensor   # u8 [m * top_k, n_out / 32, 2]


def experts_keep(x: torch.Tensor, expert_of: torch.Tensor, weights: torch.Tensor, experts: MoeExperts):
    """`experts_many` in training: `(y, kept)`, `kept` for `experts_backward`.  Gate and up are rounded to bf16 before `silu(gate) * up` (they are a tensor
    here) and kept in 8 bits (`marlin_gemm.swiglu_keep`)."""
    order, first, place = marlin_gemm.moe_sort(expert_of, experts.b_down.shape[0])
    gate_up = marlin_gemm.marlin_w4a16_gemm_experts(x, first, experts.b_gate_up, experts.s_gate_up, experts.groupsize, order=order, top_k=expert_of.shape[1])
    h, whole, exponents = marlin_gemm.swiglu_keep(gate_up)
    rows = marlin_gemm.marlin_w4a16_gemm_experts(h, first, experts.b_down, experts.s_down, experts.groupsize)
    return marlin_gemm.moe_combine(rows, weights, first, place), MoeKept(first, place, weights, rows, whole, exponents)


def experts_backward(dy: torch.Tensor, kept: MoeKept, experts: MoeExperts):
    """The gradients of `experts_keep(x, ..., weights, ...)` from `dy` bf16 `[m, n_down]`, the packs frozen: `(dx bf16 [m, hidden], d_weights f32 [m, top_k])`."""
    d_rows, d_weights = marlin_gemm.moe_combine_backward(dy, kept.rows, kept.weights, kept.first, kept.place)
    dh = marlin_gemm.marlin_w4a16_gemm_experts_backward(d_rows, kept.first, experts.b_down, experts.s_down, experts.groupsize)
    d_gate_up = marlin_gemm.swiglu_keep_backward(dh, kept.whole, kept.exponents)
    d_rows = marlin_gemm.marlin_w4a16_gemm_experts_backward(d_gate_up, kept.first, experts.b_gate_up, experts.s_gate_up, experts.groupsize)
    return marlin_gemm.moe_gather_backward(d_rows, kept.first, kept.place), d_weights
