"""The 4-bit K/V cache in plain PyTorch (any device): how rows are quantised, stored and read.

The layout is in include/fdl.h. fdl.ops.kv4_append / kv4_read are the kernels; this module is for the
unfused driver (fdl.torch_path) and for programs that build or inspect a cache without a GPU. Both give
the same codes bit for bit.
"""
from __future__ import annotations

import torch

from .lib import KV4_CELL_BYTES

HEAD_DIM = 128
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of codes 0..7; 8..15: their negatives


def is_kv4(cache) -> bool:
    """Whether `cache` is a 4-bit K/V cache (fdl.ops.kv4_cache)."""
    return isinstance(cache, torch.Tensor) and cache.dtype == torch.uint8 and cache.dim() == 3 \
        and cache.shape[2] == KV4_CELL_BYTES


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (two per byte) [..., 64] and scale bytes [..., 4] of rows [..., 128]: per 32 channels the
    smallest power of two 2^e with max|x| <= 7 * 2^e (e in [-127, 125]; byte e + 127, 255 for a group
    with a NaN or an infinity), codes rounded to the nearest value, ties to the even code."""
    g = x.double().unflatten(-1, (4, 32))
    top = g.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    frac, e = torch.frexp(torch.where(bad, 1.0, top))  # top = frac * 2^e, frac in [0.5, 1)
    e = torch.where(top > 0, e - 3 + (frac > 0.875).int(), -127).clamp(-127, 125)
    # times 2^-e, by its bits: powers computed on a GPU (pow, ldexp) may be an ulp off, and a value half way
    # between two codes then gets the wrong one
    y = torch.where(bad, 0.0, g) * ((1023 - e.long()) << 52).view(torch.float64)
    m = y.abs()
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int()
            + (m > 2.5).int() + (m >= 3.5).int() + (m > 5.0).int())
    code = (code + 8 * torch.signbit(y).int()).flatten(-2)
    scale = torch.where(bad, 255, e + 127).squeeze(-1).to(torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), scale


def _regions(cache: torch.Tensor):
    """K codes [c, h, 16, 64], V codes [c, h, 4, 16, 4, 4], K and V scales [c, h, 4, 16] (views)."""
    return (cache[..., :1024].unflatten(-1, (16, 64)),
            cache[..., 1024:2048].unflatten(-1, (4, 16, 4, 4)),
            cache[..., 2048:2112].unflatten(-1, (4, 16)), cache[..., 2112:].unflatten(-1, (4, 16)))


def store_rows(cache: torch.Tensor, slot: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """Quantises K and V rows [n, n_kv_heads * 128] into cache slots slot [n] (distinct); rows with a slot
    outside the cache (padding: -1) are skipped."""
    kr, vr, ks, vs = _regions(cache)
    heads = cache.shape[1]
    inside = (slot >= 0) & (slot < 16 * cache.shape[0])
    slot, k, v = slot[inside], k[inside], v[inside]
    cell, s = slot // 16, slot % 16
    codes, scales = quantize_rows(k.reshape(-1, heads, HEAD_DIM))
    kr[cell, :, s] = codes
    ks[cell, :, :, s] = scales
    codes, scales = quantize_rows(v.reshape(-1, heads, HEAD_DIM))
    vr[cell, :, s // 4, :, s % 4] = codes.unflatten(-1, (16, 4))
    vs[cell, :, :, s] = scales


def _decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    lut = torch.tensor(VALUES + tuple(-x for x in VALUES), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127)).float()
    return (lut[c.long()].unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten(-3)


def load_rows(cache: torch.Tensor, slot: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows [n, n_kv_heads * 128] float32 of cache slots; zeros for a slot outside the cache."""
    kr, vr, ks, vs = _regions(cache)
    outside = (slot < 0) | (slot >= 16 * cache.shape[0])
    slot = torch.where(outside, 0, slot)
    cell, s = slot // 16, slot % 16
    rows = (_decode(kr[cell, :, s], ks[cell, :, :, s]),
            _decode(vr[cell, :, s // 4, :, s % 4].flatten(-2), vs[cell, :, :, s]))
    return tuple(x.masked_fill(outside[:, None], 0.0) for x in rows)
