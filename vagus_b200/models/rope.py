"""Rotary position embedding, interleaved-pair convention by default.

Pairs are channels (2i, 2i+1) of a head: ``y0 = x0 cos - x1 sin``,
``y1 = x0 sin + x1 cos`` with angle ``pos * base^(-i / (Dh/2))``.  The cos/sin
tables are built in fp32 and shared by every layer (one module per model);
``prepare_m(L)`` grows them.  The tables are non-persistent buffers.

Beyond that form a module may rotate only the first ``rotary_dim`` channels of a
head, pair channels (i, i + rotary_dim/2) (``layout="half"``), and scale its
frequencies for contexts longer than it was trained on (``scaling``, see
``rope_frequencies``).  Interleaved pairs over the whole head, scaled or not, keep
the table form, which the fused attention layer reads; the others rotate through
``ops.rotary``, whose angles come from the positions themselves.

Parity: reference ``infra/components/pos_embed.py:7-75``.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from .. import ops

SCALINGS = ("linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, base: float, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """(inv_freq (rotary_dim / 2,) float64, factor on the rotated channels).

    ``scaling``: ``{"type": "linear", "factor": f}`` divides every frequency by f;
    ``"ntk"`` raises the base so that the lowest frequency is divided by f and the
    highest is kept; ``"yarn"`` (with ``original_len``, and optionally
    ``beta_fast`` = 32 and ``beta_slow`` = 1) divides the frequencies that turn
    fewer than beta_slow times over the original length, keeps those that turn
    more than beta_fast times, blends between, and multiplies q and k by
    0.1 ln f + 1."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device="cpu")
    inv = float(base) ** (-2 * i / rotary_dim)
    if scaling is None:
        return inv, 1.0
    kind = scaling.get("type")
    known = {"type", "factor"} | ({"original_len", "beta_fast", "beta_slow"} if kind == "yarn" else set())
    if kind not in SCALINGS or set(scaling) - known:
        raise ValueError(f"rope scaling must be one of {SCALINGS} with keys {sorted(known)}, got {scaling}")
    f = float(scaling["factor"])
    if not f >= 1:
        raise ValueError(f"rope scaling factor must be at least 1, got {f}")
    if kind == "linear":
        return inv / f, 1.0
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        return (float(base) * f ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim), 1.0
    length = scaling["original_len"]

    def index(turns: float) -> float:                   # the pair that turns so often over the original length
        return rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))

    low = max(math.floor(index(scaling.get("beta_fast", 32))), 0)
    high = min(math.ceil(index(scaling.get("beta_slow", 1))), rotary_dim - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return inv * (1 - ramp) + inv / f * ramp, 0.1 * math.log(f) + 1.0


def rope_options(rope_dim: int | None, rope_layout: str, rope_scaling: dict | None) -> dict:
    """The config entries of a model's rotary options: only those that differ
    from the plain form, so plain configs keep their keys."""
    given = dict(rope_dim=rope_dim, rope_layout=rope_layout, rope_scaling=rope_scaling)
    return {k: v for k, v in given.items() if v not in (None, "interleaved")}


class RoPE(nn.Module):
    mcos: torch.Tensor
    msin: torch.Tensor

    def __init__(self, dim: int, head_dim: int, context_len: int, base: float = 10000.0,
                 rotary_dim: int | None = None, layout: str = "interleaved", scaling: dict | None = None):
        super().__init__()
        assert dim % head_dim == 0 and head_dim > 0 and head_dim % 2 == 0
        assert context_len > 0 and base > 1
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        assert 0 < rotary_dim <= head_dim and rotary_dim % 2 == 0 and layout in ("interleaved", "half")
        self.dim = dim
        self.head_dim = head_dim
        self.context_len = context_len
        self.base = base
        self.half = head_dim // 2
        self.rotary_dim = rotary_dim
        self.layout = layout
        self.scaling = scaling
        self._inv, self.scale = rope_frequencies(rotary_dim, base, scaling)
        self._inv_on: dict[torch.device, torch.Tensor] = {}
        self.prepared_L = 0
        self.register_buffer("mcos", torch.zeros(()), persistent=False)
        self.register_buffer("msin", torch.zeros(()), persistent=False)
        self.prepare_m(context_len)

    @property
    def table_form(self) -> bool:
        """Interleaved pairs over the whole head: what the fused kernels rotate from tables."""
        return self.layout == "interleaved" and self.rotary_dim == self.head_dim

    def inv_freq(self, device) -> torch.Tensor:
        """Angle per step of position, float64 whatever the module was cast to."""
        device = torch.device(device)
        if device not in self._inv_on:
            with torch.inference_mode(False):          # kept past the call: training may save it for its backward
                self._inv_on[device] = self._inv.to(device)
        return self._inv_on[device]

    def prepare_m(self, L: int) -> None:
        if L <= self.prepared_L:
            return
        if self.table_form:
            dev, dt = self.mcos.device, self.mcos.dtype
            if self.scaling is None:
                inv = torch.pow(self.base, -torch.arange(self.half, device=dev, dtype=torch.float32) / self.half)
                ang = torch.arange(L, device=dev, dtype=torch.float32)[:, None] * inv[None, :]
            else:
                ang = torch.arange(L, device=dev, dtype=torch.float64)[:, None] * self.inv_freq(dev)
            self.register_buffer("mcos", (torch.cos(ang) * self.scale).to(dt), persistent=False)
            self.register_buffer("msin", (torch.sin(ang) * self.scale).to(dt), persistent=False)
        self.prepared_L = L

    def _check(self, end: int) -> None:
        if end > self.prepared_L:
            raise ValueError("Context length exceeded. Please call RoPE.prepare_m to enlarge.")

    def tables(self, L: int, offset: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
        if not self.table_form:
            raise ValueError("this RoPE has no tables (half layout or part of the head): call rotate")
        self._check(offset + L)
        return self.mcos[offset:offset + L], self.msin[offset:offset + L]

    def rotate(self, q: torch.Tensor, k: torch.Tensor | None, offset: int = 0):
        """q (B, L, H, D) and k (B, L, Hk, D) at positions offset, offset + 1, ... (``ops.rotary``)."""
        self._check(offset + q.shape[1])
        return ops.rotary(q, k, offset, self.inv_freq(q.device), layout=self.layout, scale=self.scale)

    def forward(self, x: torch.Tensor, offset: int = 0) -> torch.Tensor:
        """x: (..., L, head_dim)."""
        assert x.shape[-1] == self.head_dim
        if not self.table_form:
            return self.rotate(x.reshape(-1, x.shape[-2], 1, self.head_dim), None, offset).view(x.shape)
        cos, sin = self.tables(x.shape[-2], offset)
        pairs = x.reshape(*x.shape[:-1], self.half, 2)
        x0, x1 = pairs[..., 0], pairs[..., 1]
        y = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1)
        return y.reshape(x.shape)
