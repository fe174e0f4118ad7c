"""FP8 with a scale for each block of 128 in 64 bits on the CPU: encode, decode and the product.

The reference has no such format (its FP8 has one scale per tensor); the definition is the library's own (include/lyraq.h,
lyraq_quant_fp8_block): s = max(fl(max|x| / 448), 2^-100), code = e4m3(fl(x / s)), fl rounding to fp32.
"""

import numpy as np
import torch

from . import e4m3

BLOCK = 128
LEAST = 2.0 ** -100


def spread(scales, rows, k, block_rows):
    """Scales [blocks of rows, blocks of k] -> [rows, k]."""
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :k]


def encode(x, block_rows=1):
    """x [rows, k] -> (codes uint8 [rows, k], scales fp32 [rows / block_rows, k / 128], rounded up)."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % BLOCK, 0, -rows % block_rows))
    b = v.reshape(-1, block_rows, v.shape[1] // BLOCK, BLOCK)
    bad = ~torch.isfinite(b).all(dim=3).all(dim=1)
    a = torch.where(torch.isfinite(b), b, 0.0).abs().amax(dim=(1, 3))
    s = (a / 448).float().clamp_min(LEAST)          # of a 64-bit quotient of two fp32 numbers: the fp32 quotient
    s = torch.where(bad, float("nan"), s)
    full = spread(s, rows, k, block_rows).double()
    q = (x.double() / full).float()
    codes = torch.from_numpy(e4m3.encode(q.nan_to_num(0.0).numpy()))
    return torch.where(full.isnan(), 0, codes).to(torch.uint8), s


def decode(codes, s, block_rows=1):
    rows, k = codes.shape
    return torch.from_numpy(e4m3.decode(codes.numpy()).astype(np.float64)) * spread(s, rows, k, block_rows).double()


def gelu_tanh(y):
    return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
