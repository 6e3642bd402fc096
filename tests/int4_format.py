"""The 4-bit cache's format, restated in 64 bits for the tests: what the append stores of a
row, and what the bytes of a pool stand for."""

import torch


def quantise(x):
    """(codes, scales) of [..., D] values: 32 dims share a scale of 4 significant bits."""
    g = x.double().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    top = torch.maximum(-lo, hi)
    held = (top >= 2.0 ** -100) & (top < 2.0 ** 120)
    mantissa, exponent = torch.frexp(torch.where(held, top, torch.ones_like(top)) / 8)
    s = torch.ldexp((mantissa * 16).ceil() / 16, exponent)
    s = torch.where(-lo >= hi, s, -s)
    codes = ((g / s).round() + 8).clamp(0, 15)
    codes = torch.where(held, codes, torch.full_like(codes, 8.0)).nan_to_num(8.0)
    s = torch.where(held, s, torch.zeros_like(s))
    return codes.flatten(-2).to(torch.uint8), s.squeeze(-1)


def values(codes, scales):
    """The numbers that codes stand for, fp64 [..., D]."""
    return ((codes.double() - 8).unflatten(-1, (-1, 32)) * scales.double()[..., None]).flatten(-2)


def held(x):
    """What the cache holds of [..., D] values."""
    return values(*quantise(x))


def pack(codes, scales, fill=None):
    """[Hkv, NB, bs, D] codes and scales [Hkv, NB, bs, D / 32] as a pool (uint8)."""
    hkv, nb, bs, d = codes.shape
    words = codes.view(hkv, nb, bs, d // 8, 8).int()
    nibbles = torch.empty_like(words)
    for dim in range(8):
        nibbles[..., dim // 2 + 4 * (dim % 2)] = words[..., dim]
    data = (nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)).to(torch.uint8)
    data = data.reshape(hkv, nb, bs * d // 2)
    size = scales.to(torch.bfloat16).contiguous().view(torch.uint8).reshape(hkv, nb, bs * d // 16)
    return torch.cat([data, size], -1).view(hkv, nb, bs, d // 2 + d // 16)


def unpack(pool):
    """fp64 [Hkv, NB, bs, D] of a pool."""
    hkv, nb, bs, row = pool.shape
    d = row * 16 // 9
    flat = pool.reshape(hkv, nb, bs * row)
    data = flat[..., : bs * d // 2].reshape(hkv, nb, bs, d // 8, 4).int()
    nibbles = torch.stack([data & 15, data >> 4], -1).flatten(-2)
    codes = torch.stack([nibbles[..., dim // 2 + 4 * (dim % 2)] for dim in range(8)], -1)
    scales = flat[..., bs * d // 2:].contiguous().view(torch.bfloat16).view(hkv, nb, bs, d // 32)
    return values(codes.flatten(-2), scales)
