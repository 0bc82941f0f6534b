"""A cache of E2M1 in plain 64-bit form on the CPU: what its bytes stand for, and how
values become bytes. With paged_oracle's attention over what is held, what the kernels for
4-bit pages are compared with."""

from __future__ import annotations

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BORDERS = (VALUES[1:] + VALUES[:-1]) / 2
LAST = 226        # the byte of the largest scale, 10240


def scale_of(byte: torch.Tensor) -> torch.Tensor:
    """5 bits of exponent (of 15), 3 of fraction, as FP16 has them; 255: NaN."""
    b = byte.long()
    e, f = b // 8, (b % 8).double()
    s = torch.where(e == 0, f * 2.0 ** -17, (1 + f / 8) * torch.exp2((e - 15).double()))
    return torch.where(b == 255, torch.full_like(s, float("nan")), s)


SCALES = scale_of(torch.arange(LAST + 1))
MIDDLES = (SCALES[1:] + SCALES[:-1]) / 2


def nearest(x: torch.Tensor, middles: torch.Tensor) -> torch.Tensor:
    """The index of the value nearest to x >= 0 among those with these middles; of two, the even one."""
    i = torch.bucketize(x, middles)
    at = i.clamp(max=len(middles) - 1)
    return torch.where((i < len(middles)) & (x == middles[at]) & (i % 2 == 1), i + 1, i)


def quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [.., d] float64: (codes as signed values [.., d], bytes [.., d / 32])."""
    g = x.double().unflatten(-1, (-1, 32))
    fine = torch.isfinite(g).all(-1)
    g = torch.where(fine[..., None], g, torch.zeros_like(g))
    byte = nearest(g.abs().amax(-1) / 6, MIDDLES)
    s = SCALES[byte][..., None]
    y = torch.where(s > 0, g / s.clamp(min=2.0 ** -17), torch.zeros_like(g))
    codes = VALUES[nearest(y.abs(), BORDERS)] * torch.sign(y)
    return codes.flatten(-2), torch.where(fine, byte, torch.full_like(byte, 255))


def values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    return (codes.unflatten(-1, (-1, 32)) * scale_of(byte)[..., None]).flatten(-2)


def codes_of(packed: torch.Tensor) -> torch.Tensor:
    """Packed bytes [.., n] as signed values [.., 2 n], float64."""
    p = packed.cpu().view(torch.uint8).long()
    c = torch.stack([p % 16, p // 16], -1).flatten(-2)
    return torch.where(c >= 8, -VALUES[c % 8], VALUES[c % 8])


def held_codes(c) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(k codes, v codes [pages, kv_heads, page, d], bytes of their scales [pages, kv_heads, page, d / 32])."""
    v = codes_of(c.v).transpose(-2, -1)             # [pages, kv_heads, page / 16, 16, d]
    return codes_of(c.k), v.flatten(-3, -2), c.k_scale.cpu().transpose(2, 3).long(), c.v_scale.cpu().transpose(2, 3).long()


def pools(c) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds as paged_oracle takes it: k [pages, kv_heads, page, d], v [.., d, page]."""
    k, v, ks, vs = held_codes(c)
    return values(k, ks), values(v, vs).transpose(2, 3).contiguous()


def turned(x: torch.Tensor, pos: int, inv_freq, interleaved=False, scale=1.0, w=None, eps=1e-6, offset=0.0) -> torch.Tensor:
    """x [heads, head_dim] of one token, normed and rotated to its position."""
    x = x.double().clone()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (offset + w.double().cpu())
    if inv_freq is None:
        return x
    h = inv_freq.numel()
    angle = pos * inv_freq.double().cpu()
    at = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    a, b = x[:, at[0]].clone(), x[:, at[1]].clone()
    x[:, at[0]] = scale * (a * angle.cos() - b * angle.sin())
    x[:, at[1]] = scale * (b * angle.cos() + a * angle.sin())
    return x
