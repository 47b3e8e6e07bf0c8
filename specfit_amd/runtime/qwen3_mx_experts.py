"""Routed experts of one decoder layer held in HBM in microscaled 4 bits (K16).

Drop-in for transformers' ``Qwen3MoeExperts`` (tf:215-246): the same forward
arguments, every expert resident.  An expert of the Qwen3-30B-A3B shape takes
2.5 MB instead of 9.4, so the 48 layers of that model take 15.5 GB and the 94 of
Qwen3-235B-A22B 121 of a GPU's 288 GB (whose bf16 experts, 454 GB, do not fit:
``from_packed`` makes one layer at a time, ``install_mx_experts`` is for models that
are on the GPU).  ``Qwen3OffloadedExperts`` is for experts that have to stay exact
and stream.  A forward reads nothing back to the host and can be captured into a
graph.
"""
from __future__ import annotations

import torch
from torch import nn

from .. import ops


class Qwen3MXExperts(nn.Module):
    def __init__(self, records: torch.Tensor, *, hidden_size: int, intermediate_size: int) -> None:
        """``records``: uint8 [experts, ops.mx_expert_bytes(H, I)] on a GPU, as
        ``ops.mx_quantize_experts`` makes them."""
        super().__init__()
        nbytes = ops.mx_expert_bytes(hidden_size, intermediate_size)
        if records.dtype != torch.uint8 or records.dim() != 2 or records.shape[1] != nbytes \
                or not records.is_contiguous():
            raise ValueError(f"records must be contiguous uint8 [experts, {nbytes}]")
        if not 1 <= records.shape[0] <= 256:
            raise ValueError("a layer has 1 to 256 experts")
        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size
        self.register_buffer("records", records)

    @property
    def num_experts(self) -> int:
        return self.records.shape[0]

    @classmethod
    def from_packed(cls, packed: torch.Tensor, *, hidden_size: int,
                    intermediate_size: int) -> "Qwen3MXExperts":
        """From [gate | up | down] packed experts [experts, 3*H*I] on a GPU."""
        return cls(ops.mx_quantize_experts(packed, hidden_size, intermediate_size),
                   hidden_size=hidden_size, intermediate_size=intermediate_size)

    @classmethod
    def from_module(cls, experts: nn.Module) -> "Qwen3MXExperts":
        """From an HF ``Qwen3MoeExperts`` on a GPU (shares no storage)."""
        E, H, I = _checked(experts)
        gate_up, down = experts.gate_up_proj.detach(), experts.down_proj.detach()
        records = torch.empty((E, ops.mx_expert_bytes(H, I)), dtype=torch.uint8, device=down.device)
        for e in range(E):  # one expert's copy at a time, not the layer's
            packed = torch.cat([gate_up[e].reshape(-1), down[e].reshape(-1)])[None]
            ops.mx_quantize_experts(packed, H, I, out=records[e:e + 1])
        return cls(records, hidden_size=H, intermediate_size=I)

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                top_k_weights: torch.Tensor) -> torch.Tensor:
        """Sum over a token's experts of weight * expert(token), bf16 [tokens,
        H].  Routes to experts that the layer does not have count for nothing."""
        if top_k_weights.dtype != torch.bfloat16:
            top_k_weights = top_k_weights.to(torch.bfloat16)
        return ops.mx_experts(hidden_states, top_k_index.contiguous(), top_k_weights.contiguous(),
                              self.records, self.hidden_size, self.intermediate_size)


def _checked(experts: nn.Module) -> tuple[int, int, int]:
    """(experts, hidden size, intermediate size) of an HF ``Qwen3MoeExperts``
    that a ``Qwen3MXExperts`` can be made from."""
    if type(experts.act_fn).__name__ not in ("SiLUActivation", "SiLU"):
        raise ValueError("the experts' activation must be silu")
    gate_up, down = experts.gate_up_proj, experts.down_proj
    E, H, I = down.shape
    if gate_up.shape != (E, 2 * I, H) or not 1 <= E <= 256:
        raise ValueError("experts must be [1 to 256, 2 * intermediate, hidden] beside "
                         "[experts, hidden, intermediate]")
    if not (gate_up.is_cuda and down.is_cuda) or gate_up.device != down.device:
        raise ValueError("the experts' weights must be on a HIP device")
    if gate_up.dtype != down.dtype or down.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("the experts' weights must be bf16, fp16 or fp32")
    ops.mx_expert_bytes(H, I)
    return E, H, I


def install_mx_experts(model: nn.Module) -> int:
    """Replace the experts of every Qwen3-MoE layer of ``model`` that are
    transformers' own, on a GPU, with a ``Qwen3MXExperts`` of their weights in
    4 bits; returns how many.  Layers whose experts are offloaded stay.  All are
    looked over before the first is replaced, so a model that is refused is as it
    was; a layer's own weights go before the next one's are rounded."""
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeExperts

    places: dict[int, list[str]] = {}  # by module: layers may share one
    for name, mod in model.named_modules(remove_duplicate=False):
        if isinstance(mod, Qwen3MoeExperts):
            if mod is model:
                raise ValueError("the model is the experts themselves: Qwen3MXExperts.from_module")
            _checked(mod)
            places.setdefault(id(mod), []).append(name)
    for names in places.values():
        new = Qwen3MXExperts.from_module(model.get_submodule(names[0]))
        for name in names:
            parent, _, attr = name.rpartition(".")
            setattr(model.get_submodule(parent), attr, new)
    return len(places)
