"""Byte format of a KV cache held in 4 bits, and its PyTorch implementation (the oracle and the CPU backend).

A cache is a uint8 tensor ``[num_blocks, kv_heads, block_size, row_bytes(head_dim)]``. Inside a page, 16 tokens of one
head are a *unit* of ``16 * row_bytes`` contiguous bytes: 16 rows of codes (``head_dim / 2`` bytes each), then 16 rows
of parameters (8 bytes each), so one unit is one aligned run whatever the page size.

* Codes: channel ``2 i`` is the low nibble of byte ``i``, channel ``2 i + 1`` the high one. Eight channels are one 32-bit
  word; a word's parity is its group (``(channel >> 3) & 1``). A rotary pair ``(i, i + head_dim / 2)`` lies in one group,
  so a large rotary pair coarsens only its own group.
* Parameters of a row: bf16 ``s0, c0, s1, c1``, steps never negative. A channel of group ``g`` stands for
  ``c_g + s_g * (code - 8)``.

``quantize`` fixes the numbers: with ``hi``/``lo`` a group's extremes (fp32 arithmetic on bf16 values)
``s = bf16((hi / 2 - lo / 2) / 7.5)``, ``c = bf16(hi / 2 + lo / 2 + s / 2)``, ``code = clamp(rint((x - c) / s) + 8, 0, 15)``.
A step below the smallest normal number counts as 0 (all codes 8: the group holds ``c``). A group with a NaN or an
infinity gets NaN parameters, so what was stored reads back as NaN instead of a plausible number.
"""

from __future__ import annotations

import torch

__all__ = ["UNIT", "row_bytes", "is_kv4", "check_caches", "quantize", "dequantize", "write_rows", "read_rows"]

UNIT = 16                      # tokens per unit
_MIN_NORMAL = 2.0 ** -126


def row_bytes(head_dim: int) -> int:
    """Bytes of one token of one KV head in one cache."""
    if head_dim % 16:
        raise ValueError(f"a 4-bit cache needs head_dim % 16 == 0, got {head_dim}")
    return head_dim // 2 + 8


def is_kv4(cache: torch.Tensor) -> bool:
    return cache.dtype == torch.uint8


def check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, head_dim: int, num_kv_heads: int | None = None) -> None:
    """Raises unless both tensors are 4-bit caches of one shape for this head size (and number of KV heads)."""
    if not (is_kv4(k_cache) and is_kv4(v_cache)):
        raise TypeError(f"a 4-bit cache is a pair of uint8 tensors, got {k_cache.dtype} and {v_cache.dtype}")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.device != v_cache.device:
        raise ValueError(f"4-bit caches need one 4-d shape and device, got {tuple(k_cache.shape)} on {k_cache.device} and "
                         f"{tuple(v_cache.shape)} on {v_cache.device}")
    _, heads, bs, row = k_cache.shape
    if bs <= 0 or bs % UNIT or row != row_bytes(head_dim) or (num_kv_heads is not None and heads != num_kv_heads):
        raise ValueError(f"4-bit cache of shape {tuple(k_cache.shape)}: expected [blocks, {num_kv_heads or 'kv_heads'}, a "
                         f"multiple of {UNIT}, {row_bytes(head_dim)}] for head_dim {head_dim}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("4-bit caches must be contiguous")


def _to_groups(x: torch.Tensor) -> torch.Tensor:
    """``[..., D]`` -> ``[..., 2, D/2]``, channels of even words first."""
    return x.unflatten(-1, (x.shape[-1] // 16, 2, 8)).transpose(-2, -3).flatten(-2)


def _from_groups(x: torch.Tensor) -> torch.Tensor:
    return x.unflatten(-1, (x.shape[-1] // 8, 8)).transpose(-2, -3).flatten(-3)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``[..., D]`` (uint8, 0..15) and parameters ``[..., 2, 2]`` (bf16, last axis ``s, c``) of ``x`` rounded to
    bf16."""
    g = _to_groups(x.to(torch.bfloat16).float())
    hi, lo = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    s = ((0.5 * hi - 0.5 * lo) / 7.5).to(torch.bfloat16).float()
    s = torch.where(s < _MIN_NORMAL, torch.zeros_like(s), s)
    c = (0.5 * hi + 0.5 * lo + 0.5 * s).to(torch.bfloat16).float()
    n = torch.where(s > 0, torch.round((g - c) / s) + 8, torch.full_like(g, 8.0)).clamp(0, 15)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    nan = torch.full_like(s, float("nan"))
    s, c, n = torch.where(bad, nan, s), torch.where(bad, nan, c), torch.where(bad, torch.full_like(n, 8.0), n)
    return _from_groups(n).to(torch.uint8), torch.cat([s, c], -1).to(torch.bfloat16)


def dequantize(codes: torch.Tensor, params: torch.Tensor) -> torch.Tensor:
    """fp32 values of ``codes [..., D]`` under ``params [..., 2, 2]``."""
    p = params.float()
    return _from_groups(p[..., 1:2] + p[..., 0:1] * (_to_groups(codes).float() - 8))


def _units(cache: torch.Tensor) -> torch.Tensor:
    nb, h, bs, row = cache.shape
    return cache.view(nb, h, bs // UNIT, UNIT * row)


def _places(cache: torch.Tensor, slots: torch.Tensor):
    """Index tensors of the code bytes and parameter bytes of ``slots`` inside ``_units(cache)``."""
    _, h, bs, row = cache.shape
    s = slots.long()
    blk, r = s // bs, s % bs
    heads = torch.arange(h, device=cache.device)[None, :, None]
    lead = (blk[:, None, None], heads, (r // UNIT)[:, None, None])
    i = (r % UNIT)[:, None, None]
    width = row - 8
    codes = i * width + torch.arange(width, device=cache.device)
    params = UNIT * width + i * 8 + torch.arange(8, device=cache.device)
    return lead, codes, params


def write_rows(cache: torch.Tensor, slots: torch.Tensor, x: torch.Tensor) -> None:
    """Stores ``x [T, kv_heads, D]`` at ``slots [T]`` (all non-negative and distinct)."""
    codes, params = quantize(x)
    lead, ci, pi = _places(cache, slots)
    u = _units(cache)
    u[(*lead, ci)] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    u[(*lead, pi)] = params.flatten(-2).contiguous().view(torch.uint8)


def read_rows(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """fp32 ``[T, kv_heads, D]`` at ``slots [T]`` (all non-negative)."""
    lead, ci, pi = _places(cache, slots)
    u = _units(cache)
    b = u[(*lead, ci)]
    codes = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    params = u[(*lead, pi)].contiguous().view(torch.bfloat16).unflatten(-1, (2, 2))
    return dequantize(codes, params)
