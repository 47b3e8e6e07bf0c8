"""Routed experts of one decoder layer held in HBM in microscaled 4 bits (K16).

Drop-in for transformers' ``Qwen3MoeExperts`` (tf:215-246): the same forward
arguments, every expert resident.  An expert of the Qwen3-30B-A3B shape takes
2.5 MB instead of 9.4, so the 48 layers of that model take 15 GB and the 94 of
Qwen3-235B-A22B 117 of a GPU's 288 GB; ``Qwen3OffloadedExperts`` is for experts
that have to stay exact and stream.  A forward reads nothing back to the host
and can be captured into a graph.
"""
from __future__ import annotations

import functools

import torch
from torch import nn

from .. import ops

# Routes that read their experts for themselves save a dispatch, a combine and
# the launches of both: about 10 us on the device, and 20 on the host.  They
# read an expert again for each further route to it, with even routing
# routes - E (1 - (1 - 1/E)^routes) times; 10 us are 40 MB of such reads.
# us a call on the device, without dispatch and with it:
#   128 experts of 2048 x 768, 8 a token    1 token 12 / 21   4: 24 / 30   8: 42 / 42   12: 60 / 53
#   32 experts of 4096 x 1536, 8 a token    1 token 27 / 34   2: 40 / 45   3: 57 / 55   4: 71 / 67
#   100 experts of 1000 x 424, 2 a token    1 token 8 / 15    16: 14 / 19  32: 19 / 23
_READ_AGAIN = 40_000_000
_MOST_ROUTES = 128   # beyond, the products' idle rows would count


@functools.lru_cache(maxsize=1024)
def _without_dispatch(routes: int, experts: int, expert_bytes: int) -> bool:
    again = routes - experts * (1 - (1 - 1 / experts) ** routes)
    return routes <= _MOST_ROUTES and again * expert_bytes <= _READ_AGAIN


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
        if type(experts.act_fn).__name__ not in ("SiLUActivation", "SiLU"):
            raise ValueError("the experts' activation must be silu")
        gate_up, down = experts.gate_up_proj.detach(), experts.down_proj.detach()
        E, H, I = down.shape
        records = torch.empty((E, ops.mx_expert_bytes(H, I)), dtype=torch.uint8, device=down.device)
        for e in range(E):  # one expert's copy at a time, not the layer's
            packed = torch.cat([gate_up[e].reshape(-1), down[e].reshape(-1)])[None]
            ops.mx_quantize_experts(packed, H, I, out=records[e:e + 1])
        return cls(records, hidden_size=H, intermediate_size=I)

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                top_k_weights: torch.Tensor) -> torch.Tensor:
        """Sum over a token's experts of weight * expert(token), bf16 [tokens,
        H].  Routes to experts that the layer does not have count for nothing."""
        records = self.records
        if top_k_index.dim() != 2:
            raise ValueError("top_k_index must have shape [tokens, top_k]")
        if _without_dispatch(top_k_index.numel(), *records.shape):
            return ops.mx_routed_swiglu(hidden_states, top_k_index.contiguous(),
                                        top_k_weights.to(torch.bfloat16).contiguous(), records,
                                        self.hidden_size, self.intermediate_size)
        if hidden_states.shape != (top_k_index.shape[0], self.hidden_size):
            raise ValueError(f"hidden_states must have shape [tokens, {self.hidden_size}]")
        if top_k_weights.shape != top_k_index.shape:
            raise ValueError("top_k_weights must match top_k_index shape")
        for t in (hidden_states, top_k_index, top_k_weights):
            if t.device != records.device:
                raise ValueError("hidden_states and routes must be on the experts' device")
        if records.is_cuda and torch.cuda.current_device() != records.get_device():
            with torch.cuda.device(records.device):
                return self._dispatched(hidden_states, top_k_index, top_k_weights)
        return self._dispatched(hidden_states, top_k_index, top_k_weights)

    def _dispatched(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                    top_k_weights: torch.Tensor) -> torch.Tensor:
        plan = ops.dispatch(top_k_index, self.num_experts)
        rows = torch.empty((top_k_index.numel(), self.hidden_size), dtype=torch.bfloat16,
                           device=hidden_states.device)
        weights = top_k_weights.to(torch.bfloat16).contiguous().view(-1)
        ops.mx_grouped_swiglu(hidden_states, plan, weights, self.records, self.hidden_size,
                              self.intermediate_size, rows)
        return ops.combine(rows, top_k_index, plan, self.hidden_size, accumulate_fp32=True)


def install_mx_experts(model: nn.Module) -> int:
    """Replace the experts of every Qwen3-MoE layer of ``model`` that are
    transformers' own, on a GPU, with a ``Qwen3MXExperts`` of their weights in
    4 bits; returns how many.  Layers whose experts are offloaded stay."""
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeExperts

    targets = [(name, mod) for name, mod in model.named_modules()
               if isinstance(mod, Qwen3MoeExperts)]
    for name, mod in targets:
        parent_name, _, attr = name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        setattr(parent, attr, Qwen3MXExperts.from_module(mod))
    return len(targets)
