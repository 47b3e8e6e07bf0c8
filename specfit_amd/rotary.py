"""Frequencies of rotary positions.

``rotary_frequencies`` gives the turns per position of each rotated pair, in
64 bits, for the plain form and the ones scaled for long contexts (the
parameters are those of a Hugging Face config's ``rope_parameters``);
``ops.rotary_embed`` applies them.  Frequencies are kept in 64 bits where
transformers rounds them to 32: at position 10^6 that rounding moves the
fastest pair's angle by up to 0.06.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

ROPE_TYPES = ("default", "linear", "dynamic", "llama3", "yarn", "longrope")


@dataclass(frozen=True)
class RotaryTable:
    """What rotary_embed needs besides positions: ``turns`` (fp64
    [rotary_dim / 2], turns per position), the factor that the stretched forms
    put on both sine and cosine, and the layout."""

    head_dim: int
    rotary_dim: int
    interleaved: bool
    factor: float
    turns: torch.Tensor

    def __post_init__(self) -> None:
        # The kernel reads rotary_dim / 2 doubles one after another.
        t = self.turns
        if self.rotary_dim < 2 or self.rotary_dim % 2 or self.rotary_dim > self.head_dim:
            raise ValueError("rotary_dim must be even and at most head_dim")
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float64 \
                or t.shape != (self.rotary_dim // 2,) or not t.is_contiguous():
            raise ValueError(f"turns must be contiguous fp64 [{self.rotary_dim // 2}]")

    def to(self, device) -> "RotaryTable":
        return RotaryTable(self.head_dim, self.rotary_dim, self.interleaved, self.factor,
                           self.turns.to(device))

    @classmethod
    def from_config(cls, config, *, interleaved: bool = False, seq_len: int | None = None,
                    device=None) -> "RotaryTable":
        """The table of a Hugging Face config (``rope_parameters``, head_dim)."""
        parameters = dict(config.rope_parameters)
        head_dim = getattr(config, "head_dim", None) or \
            config.hidden_size // config.num_attention_heads
        return rotary_frequencies(
            head_dim, base=parameters["rope_theta"],
            rotary_dim=int(head_dim * parameters.get("partial_rotary_factor", 1.0)),
            scaling=parameters, interleaved=interleaved,
            max_position_embeddings=config.max_position_embeddings, seq_len=seq_len, device=device)


def _scale(factor: float, weight: float = 1.0) -> float:
    return 1.0 if factor <= 1 else 0.1 * weight * math.log(factor) + 1.0


def rotary_frequencies(head_dim: int, *, base: float = 10000.0, rotary_dim: int | None = None,
                       scaling: dict | None = None, interleaved: bool = False,
                       max_position_embeddings: int | None = None, seq_len: int | None = None,
                       device=None) -> RotaryTable:
    """The table of base^(-2 i / rotary_dim) radians per position, changed by
    ``scaling`` (a dict with ``rope_type`` one of ROPE_TYPES):

    linear    divided by ``factor``
    dynamic   the base grows with ``seq_len`` past ``max_position_embeddings``
    llama3    slow pairs divided by ``factor``, those between
              ``low_freq_factor`` and ``high_freq_factor`` turns over the
              original context in part
    yarn      the same with a ramp over the pairs between ``beta_slow`` and
              ``beta_fast`` turns, and sine and cosine times 0.1 ln(factor) + 1
              (or ``attention_factor``, or ``mscale`` and ``mscale_all_dim``)
    longrope  each pair divided by its entry of ``long_factor`` (or
              ``short_factor`` while ``seq_len`` is within the original context)
    """
    rot = head_dim if rotary_dim is None else int(rotary_dim)
    if rot < 2 or rot % 2 or rot > head_dim:
        raise ValueError("rotary_dim must be even and at most head_dim")
    if not base > 1:
        raise ValueError("the base must be above 1")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in ROPE_TYPES:
        raise ValueError(f"rope_type must be one of {ROPE_TYPES}, not {kind!r}")
    half = rot // 2
    pairs = torch.arange(half, dtype=torch.float64)
    attention = 1.0
    if kind == "dynamic":
        if max_position_embeddings is None:
            raise ValueError("dynamic scaling needs max_position_embeddings")
        if rot < 4:
            raise ValueError("dynamic scaling needs rotary_dim of at least 4")
        ratio = max(seq_len or 0, max_position_embeddings) / max_position_embeddings
        base = base * (scaling["factor"] * ratio - (scaling["factor"] - 1)) ** (rot / (rot - 2))
    radians = torch.exp(pairs * (-2.0 / rot * math.log(base)))
    if kind == "linear":
        radians = radians / scaling["factor"]
    elif kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = scaling["original_max_position_embeddings"] * radians / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        radians = radians * (keep + (1 - keep) / scaling["factor"])
    elif kind == "yarn":
        old = scaling.get("original_max_position_embeddings") or max_position_embeddings
        if old is None:
            raise ValueError("yarn scaling needs original_max_position_embeddings")
        factor = scaling["factor"]
        first, last = (half * math.log(old / (2 * math.pi * beta)) / math.log(base)
                       for beta in (scaling.get("beta_fast") or 32, scaling.get("beta_slow") or 1))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rot - 1)
        slow = ((pairs - first) / (last - first if last != first else 0.001)).clamp(0, 1)
        radians = radians * (1 - slow + slow / factor)
        attention = scaling.get("attention_factor")
        if attention is None:
            part, whole = scaling.get("mscale"), scaling.get("mscale_all_dim")
            attention = _scale(factor, part) / _scale(factor, whole) if part and whole \
                else _scale(factor)
    elif kind == "longrope":
        old = scaling["original_max_position_embeddings"]
        each = scaling["long_factor" if (seq_len or 0) > old else "short_factor"]
        if len(each) != half:
            raise ValueError(f"longrope needs {half} factors")
        radians = radians / torch.tensor(each, dtype=torch.float64)
        attention = scaling.get("attention_factor")
        if attention is None:
            factor = scaling.get("factor")
            if factor is None:
                if max_position_embeddings is None:
                    raise ValueError("longrope scaling needs factor or max_position_embeddings")
                factor = max_position_embeddings / old
            attention = 1.0 if factor <= 1 else math.sqrt(1 + math.log(factor) / math.log(old))
    return RotaryTable(int(head_dim), rot, bool(interleaved), float(attention),
                       (radians / (2 * math.pi)).to(device))
