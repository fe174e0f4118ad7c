"""Microscaled FP4 in 64 bits on the CPU: encode, decode, the order of the block scales, and the product.

The reference has no such format (its 4-bit one is oracle.quant's int4 with groups of 64); the definitions are the library's own
(include/lyraq.h, lyraq_quant_fp4): e2m1 codes, a scale byte per block of 16 (e4m3, with a tensor scale) or 32 (e8m0).
"""

import torch

GROUP = {"nvfp4": 16, "mxfp4": 32}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E4M3 = torch.tensor([(f / 8 * 2.0 ** -6) if e == 0 else (1 + f / 8) * 2.0 ** (e - 7) for e in range(16) for f in range(8)][:127],
                    dtype=torch.float64)


def nearest(table, v):
    """Index of the entry of an ascending table that is nearest to v >= 0: ties to the even index, beyond the last entry the last."""
    border = (table[1:] + table[:-1]) / 2
    below = torch.searchsorted(border, v.contiguous())               # borders smaller than v
    tie = (below < border.numel()) & (border[below.clamp_max(border.numel() - 1)] == v) & (below % 2 == 1)
    return below + tie


def encode(x, fmt, g=1.0):
    """x [rows, k] -> (codes uint8 [rows, k] one per value, scale bytes uint8 [rows, k / group])."""
    b = x.double().reshape(x.shape[0], -1, GROUP[fmt])
    bad = ~torch.isfinite(b).all(dim=-1)
    b = torch.where(bad[..., None], 0.0, b)
    a = b.abs().amax(dim=-1)
    if fmt == "nvfp4":
        s = nearest(E4M3, a / (6 * g))
        t = E4M3[s] * g
    else:
        s = (torch.frexp(a).exponent.long() - 3 + 127).clamp(0, 254)
        s = torch.where(a == 0, 0, s)
        t = torch.ldexp(torch.ones_like(a), (s - 127).int())
    q = torch.where(t[..., None] > 0, b / torch.where(t > 0, t, 1.0)[..., None], 0.0)
    codes = nearest(E2M1, q.abs()) + 8 * (torch.signbit(b) & (t > 0)[..., None])
    codes = torch.where(bad[..., None], 0, codes)
    s = torch.where(bad, 0x7F if fmt == "nvfp4" else 0xFF, s)
    return codes.reshape(x.shape).to(torch.uint8), s.to(torch.uint8)


def pack(codes):
    """[rows, k] codes -> [rows, k / 2] bytes, the even element in the low nibble."""
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=-1).reshape(packed.shape[0], -1)


def scale_values(s, fmt):
    s = s.long()
    if fmt == "nvfp4":
        return torch.where(s == 0x7F, float("nan"), E4M3[s.clamp_max(126)])
    return torch.where(s == 0xFF, float("nan"), torch.ldexp(torch.ones(s.shape, dtype=torch.float64), (s - 127).int()))


def decode(codes, s, fmt, g=1.0):
    """The values that codes [rows, k] and scale bytes [rows, k / group] stand for, in 64 bits."""
    sign = 1 - 2 * (codes.long() >> 3)
    v = (E2M1[codes.long() & 7] * sign).reshape(codes.shape[0], -1, GROUP[fmt])
    return (v * scale_values(s, fmt)[..., None] * g).reshape(codes.shape)


def scale_offsets(rows, blocks):
    """Where the scale byte of (row, block) lies: [rows, blocks] byte offsets."""
    r, b = torch.arange(rows)[:, None], torch.arange(blocks)[None]
    atoms = (blocks + 3) // 4
    return ((r // 128) * atoms + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def scale_bytes(rows, k, fmt):
    blocks = k // GROUP[fmt]
    return (rows + 127) // 128 * ((blocks + 3) // 4) * 512


def tensor_scale(w):
    """The least power of two g with max|w| <= 6 * 448 * g over the finite values, 0 for zeros."""
    w = w.double()
    a = float(torch.where(torch.isfinite(w), w, 0.0).abs().max())
    if a == 0:
        return 0.0
    m, e = torch.frexp(torch.tensor(a / 2688, dtype=torch.float64))
    return max(2.0 ** (int(e) - (1 if float(m) == 0.5 else 0)), 2.0 ** -126)


def gelu_tanh(v):
    return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v ** 3)))
