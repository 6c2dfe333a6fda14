"""Rotary position embedding tables and the fused q/k-norm + RoPE + paged KV write."""
from __future__ import annotations

import math

import torch

from ._ext import ext
from .workspace import get_workspace


def rope_inv_freq(head_dim: int, theta: float, scaling: dict | None = None) -> torch.Tensor:
    """Inverse frequencies in float64, with optional Llama-3 style frequency scaling."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    if scaling and scaling.get("rope_type", scaling.get("type")) == "llama3":
        factor = float(scaling["factor"])
        low = float(scaling.get("low_freq_factor", 1.0))
        high = float(scaling.get("high_freq_factor", 4.0))
        old_ctx = float(scaling.get("original_max_position_embeddings", 8192))
        low_wl, high_wl = old_ctx / low, old_ctx / high
        wl = 2 * math.pi / inv
        scaled = torch.where(wl > low_wl, inv / factor, inv)
        smooth = (old_ctx / wl - low) / (high - low)
        mid = (1 - smooth) * scaled / factor + smooth * scaled
        is_mid = (wl >= high_wl) & (wl <= low_wl)
        inv = torch.where(is_mid, mid, scaled)
    return inv


def rope_cos_sin_table(max_pos: int, head_dim: int, theta: float, scaling: dict | None = None,
                       device=None) -> torch.Tensor:
    """``[max_pos, head_dim]`` fp32: first half cos, second half sin (rotate-half form)."""
    inv = rope_inv_freq(head_dim, theta, scaling)
    pos = torch.arange(max_pos, dtype=torch.float64)
    ang = torch.outer(pos, inv)
    tab = torch.cat([ang.cos(), ang.sin()], dim=-1).to(torch.float32)
    return tab.to(device) if device is not None else tab


def rope_kv_write(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                  cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  num_q_heads: int, num_kv_heads: int, q_norm: torch.Tensor | None = None,
                  k_norm: torch.Tensor | None = None, eps: float = 1e-6) -> None:
    """Rotate the q heads of ``qkv`` in place and write rotated k and raw v to the cache."""
    ext().rope_kv_write(qkv, positions, slots, cos_sin, q_norm, k_norm, float(eps), k_cache,
                        v_cache, num_q_heads, num_kv_heads)


def rope_kv_write_fp8(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                      cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      kv_scales: torch.Tensor, num_q_heads: int, num_kv_heads: int,
                      q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                      eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope_kv_write` for an e4m3 cache: norm, rotate and quantise in one pass.

    ``k_cache`` / ``v_cache`` are e4m3 ``[pages, Hkv, 64, 128]``, ``kv_scales`` uint8
    ``[pages, Hkv, 2, 64]`` (one power-of-two scale per token, head and side; see
    :mod:`.kv_fp8`).  Queries are computed in fp32 and rounded once; a key's norm is computed in fp64
    and its rotation keeps what it rounds off, so that its codes are those of the exact values (none
    wrong among 84 million in an emulation; rounding to fp32 first: 96).  The rotated
    queries go to ``q_out`` [T, Hq, 128], or back into ``qkv`` without it; returned either way.
    A negative slot skips the token's cache write (its queries are rotated all the same); the
    other slots must differ from one another.  A slot past the cache, or a position outside
    ``cos_sin``, raises the device status and writes nothing for that token."""
    ext().rope_kv_write_fp8(qkv, positions, slots, cos_sin, q_norm, k_norm, eps, k_cache,
                            v_cache, kv_scales, num_q_heads, num_kv_heads, q_out,
                            get_workspace(qkv.device).status)
    if q_out is not None:
        return q_out
    return qkv.as_strided((qkv.shape[0], num_q_heads, 128), (qkv.stride(0), 128, 1),
                          qkv.storage_offset())


def apply_rope_reference(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE in plain PyTorch.  x: [T, H, D]."""
    d = x.shape[-1]
    cs = cos_sin[positions.long()].to(x.device)
    cos, sin = cs[:, None, : d // 2], cs[:, None, d // 2:]
    xf = x.float()
    x1, x2 = xf[..., : d // 2], xf[..., d // 2:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)
