"""Rotary position embedding (same class, arguments and results as
diffulex/layer/rotary_embedding.py), backed by the gfx950 kernel, plus the fused
form that also stores the rotated K and V into the paged cache.

``RotaryEmbedding.forward(positions, query, key)`` returns new tensors, as the
reference does.  ``forward_and_store`` additionally writes token t's rotated key
row and its value row to cache slot ``slot_mapping[t]`` (what
``store_kvcache_unified_layout`` would do in a launch of its own, reading K and V
a second time); the caller then runs attention with
``attn_metadata.need_kv_cache_store = False``.

Beyond the reference (which asserts ``rotary_dim == head_size`` and no scaling): pairs of neighbouring elements
(``is_neox_style=False``), a part of the head (``rotary_dim < head_size``), scaled frequencies (``rope_scaling``) and the
store into microscaled caches.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import _lib
from .kv_cache_kernels import (_call, _is_block_scale, _scales, store_kvcache_distinct_layout,
                               store_kvcache_unified_layout)


def _rows(x: torch.Tensor, head_size: int) -> Tuple[int, int, int]:
    """(tokens, heads, token stride in elements) of a [T, H * hd] or [T, H, hd] tensor."""
    assert x.is_cuda and x.dtype == torch.bfloat16, "rotary embedding runs on bf16 device tensors"
    assert x.dim() in (2, 3) and x.stride(-1) == 1
    if x.dim() == 3:
        assert x.shape[-1] == head_size and x.stride(1) == head_size
        return x.shape[0], x.shape[1], x.stride(0)
    assert x.shape[-1] % head_size == 0
    return x.shape[0], x.shape[-1] // head_size, x.stride(0)


def _scaled_frequencies(dim: int, max_position: int, base: float, scaling: Optional[dict]) -> Tuple[torch.Tensor, float]:
    """(angle per position of every pair in fp64, factor of cosines and sines).  ``scaling["rope_type"]`` (or ``"type"``):

    * ``"linear"``: positions divided by ``factor``;
    * ``"dynamic"``: the base grown for ``max_position`` from ``original_max_position_embeddings``, N = factor * max / original:
      base * (N - factor + 1) ** (dim / (dim - 2));
    * ``"yarn"``: pairs that turn fewer than ``beta_slow`` times over the original length are interpolated by ``factor``, pairs
      that turn more than ``beta_fast`` times are kept, a linear ramp between; cosines and sines times
      ``attention_factor`` (default 0.1 ln(factor) + 1)."""
    pair = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-pair / dim), 1.0
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in ("linear", "dynamic", "yarn"):
        raise ValueError(f"unknown rope_scaling {scaling!r}")
    known = {"rope_type", "type", "factor", "original_max_position_embeddings"}
    unknown = sorted(set(scaling) - known - ({"beta_fast", "beta_slow", "attention_factor"} if kind == "yarn" else set()))
    if unknown:  # (a setting left out would give other angles than the model was trained with)
        raise ValueError(f"rope_scaling {kind!r} has no {', '.join(unknown)}")
    factor = float(scaling["factor"])
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"rope_scaling factor {factor} is not a finite number >= 1")
    if kind == "linear":
        return base ** (-pair / dim) / factor, 1.0
    original = int(scaling.get("original_max_position_embeddings") or max_position)
    if original <= 0:
        raise ValueError(f"original_max_position_embeddings {original}")
    if kind == "dynamic":
        if dim <= 2:
            raise ValueError("dynamic scaling needs more than one pair")
        grown = base * max(1.0, factor * max_position / original - factor + 1.0) ** (dim / (dim - 2))
        return grown ** (-pair / dim), 1.0

    def place(turns):  # the pair that turns so many times over the original length
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(place(float(scaling.get("beta_fast") or 32))), 0)
    high = min(math.ceil(place(float(scaling.get("beta_slow") or 1))), dim - 1)
    ramp = ((pair / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    freq = base ** (-pair / dim)
    gain = scaling.get("attention_factor")
    gain = float(gain) if gain is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    return freq / factor * ramp + freq * (1 - ramp), gain


class RotaryEmbedding(nn.Module):
    """rotary_embedding.py:20-66 (neox-style halves, rotary_dim == head_size) and the other forms (module docstring).

    ``cos_sin_cache``: fp32 [max_position, rotary_dim], cosines then sines.  The reference's form has the reference's bits
    (angles in fp32); every other form's angles are computed in fp64 and its cosines and sines rounded once."""

    def __init__(self, head_size: int, rotary_dim: int, max_position_embeddings: int, base: float,
                 is_neox_style: bool = True, rope_scaling: Optional[dict] = None) -> None:
        super().__init__()
        self.head_size = head_size
        self.rotary_dim = rotary_dim
        self.is_neox_style = bool(is_neox_style)
        assert 0 < rotary_dim <= head_size and rotary_dim % 2 == 0
        self._plain = rotary_dim == head_size and self.is_neox_style
        if rope_scaling is not None and rope_scaling.get("rope_type", rope_scaling.get("type")) == "default":
            rope_scaling = None
        if self._plain and rope_scaling is None:
            inv_freq = 1.0 / (base ** (torch.arange(0, rotary_dim, 2, dtype=torch.float) / rotary_dim))
            t = torch.arange(max_position_embeddings, dtype=torch.float)
            freqs = torch.einsum("i,j -> ij", t, inv_freq)
            table = torch.cat((freqs.cos(), freqs.sin()), dim=-1)
        else:
            inv_freq, gain = _scaled_frequencies(rotary_dim, max_position_embeddings, float(base), rope_scaling)
            freqs = torch.arange(max_position_embeddings, dtype=torch.float64)[:, None] * inv_freq[None, :]
            table = torch.cat(((freqs.cos() * gain).float(), (freqs.sin() * gain).float()), dim=-1)
        self.register_buffer("cos_sin_cache", table, persistent=False)

    def _launch(self, positions, query, key, q_out, k_out, value=None, k_cache=None, v_cache=None,
                slot_mapping=None, attn_metadata=None, k_scale=None, v_scale=None) -> None:
        table = self.cos_sin_cache
        positions = positions.reshape(-1)
        if not positions.is_contiguous():
            positions = positions.contiguous()
        ks = vs = slots = None
        if slot_mapping is not None:
            slots = slot_mapping.reshape(-1)
            if not slots.is_contiguous():
                slots = slots.contiguous()
            if _is_block_scale(k_scale):
                ks, vs = k_scale, v_scale
            else:
                Hk = key.shape[1] if key.dim() == 3 else key.shape[-1] // self.head_size
                ks, vs = _scales(k_cache, attn_metadata, k_scale, v_scale, Hk)
        _call(_lib.ops().rope_kv_store, positions, query, key, q_out, k_out, table, self.head_size, value, k_cache,
              v_cache, slots, ks, vs, self.rotary_dim, not self.is_neox_style)

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor
                ) -> Tuple[torch.Tensor, torch.Tensor]:
        q_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        k_out = torch.empty(key.shape, dtype=key.dtype, device=key.device)
        self._launch(positions, query, key, q_out, k_out)
        return q_out, k_out

    def _stores(self, k_cache, k_scale) -> bool:
        """Whether one launch rotates and stores into this cache (dfx_rope_kv_store's supported shapes)."""
        if k_cache.dim() == 5:  # the distinct layout
            return self._plain
        if _is_block_scale(k_scale):
            return self.head_size % 64 == 0 and self.rotary_dim % (64 if self.is_neox_style else 32) == 0
        return True

    def forward_and_store(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                          value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          slot_mapping: torch.Tensor, attn_metadata=None,
                          k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
        """forward() and store_kvcache_unified_layout(rotated key, value, ...) in one launch -- or
        store_kvcache_distinct_layout(...) where the caches are in that layout (k_cache [pages, H_kv, hd / 8,
        page, 8], v_cache [pages, H_kv, hd, page], bf16).  Microscaled caches: ``k_scale`` / ``v_scale`` are their block
        scales, written as well.  (The distinct layout with one of the other forms, and microscaled caches whose blocks straddle
        the rotated halves, take the two launches.)"""
        if not self._stores(k_cache, k_scale):
            q_out, k_out = self.forward(positions, query, key)
            k3, v3 = (x if x.dim() == 3 else x.unflatten(-1, (-1, self.head_size)) for x in (k_out, value))
            if k_cache.dim() == 5:
                store_kvcache_distinct_layout(k3, v3, k_cache, v_cache, slot_mapping, attn_metadata)
            else:
                store_kvcache_unified_layout(k3, v3, k_cache, v_cache, slot_mapping, attn_metadata, k_scale, v_scale)
            return q_out, k_out
        q_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        k_out = torch.empty(key.shape, dtype=key.dtype, device=key.device)
        self._launch(positions, query, key, q_out, k_out, value, k_cache, v_cache, slot_mapping,
                     attn_metadata, k_scale, v_scale)
        return q_out, k_out


def _frozen(x):
    """A dict, list or tuple as nested tuples that a cache can be keyed with."""
    if isinstance(x, dict):
        return tuple(sorted((k, _frozen(v)) for k, v in x.items()))
    return tuple(_frozen(v) for v in x) if isinstance(x, (list, tuple)) else x


@lru_cache(1)
def _get_rope(head_size, rotary_dim, max_position, base, rope_scaling, is_neox_style):
    return RotaryEmbedding(head_size, rotary_dim, max_position, base, is_neox_style,
                           dict(rope_scaling) if rope_scaling is not None else None)


def get_rope(head_size: int, rotary_dim: int, max_position: int, base: float,
             rope_scaling: dict | None = None, is_neox_style: bool = True):
    """rotary_embedding.py:69-79 (one module, kept until other arguments are asked for)."""
    return _get_rope(head_size, rotary_dim, max_position, base,
                     _frozen(rope_scaling) if rope_scaling is not None else None, bool(is_neox_style))


# what the cached function of the reference offers besides the call
get_rope.cache_info, get_rope.cache_clear = _get_rope.cache_info, _get_rope.cache_clear
