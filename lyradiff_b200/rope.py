"""Rotary-embedding table for the FLUX block ops (host side, runs once per image size).

The block classes take `rope_emb` as a [B, 1, S, head_dim/2, 2, 2] fp32 table whose last two axes hold the rotation
matrix [[cos, -sin], [sin, cos]] of each frequency; `lyraq_rmsnorm_rope` reads it in exactly that layout.  This is the
table the reference's Python wrapper builds before calling the ops (`rope` / `EmbedND`,
lyradiff/lyradiff_model/lyradiff_flux_transformer_model_v2.py:35-65): angles in float64, one block of frequencies per
position axis, concatenated along the frequency axis.

AxisRope is the plan of `lyraq_rope_axes` (ops.rope_axes), which needs no table: the frequency of every pair as a fraction of a turn, and the
position axis it follows.
"""

import decimal
import functools

import torch

_EXACT = decimal.Context(prec=60)
_TWO_PI = _EXACT.multiply(2, decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899"))
_TURN = _EXACT.divide(decimal.Decimal(2 ** 64), _TWO_PI)


def _turns(freq):
    """Frequency in radians per position, at least 0 and below a whole turn -> turns per position times 2^64, rounded, its bits as a signed
    64-bit number."""
    f = decimal.Decimal(freq)      # a float's value, exactly
    if not (f.is_finite() and 0 <= f < _TWO_PI):
        raise ValueError("rope: a frequency must be at least 0 and below 2 pi radians per position, got %s" % freq)
    t = min(int(_EXACT.multiply(f, _TURN).to_integral_value()), 2 ** 64 - 1)
    return t - 2 ** 64 if t >= 2 ** 63 else t


@functools.lru_cache(maxsize=256)
def _ladder(dim, theta):
    """theta^(-2 i / dim), i below dim / 2, to 60 digits, and their turns."""
    base = decimal.Decimal(theta)
    if not (base.is_finite() and base > 0):
        raise ValueError("rope: theta must be positive, got %s" % theta)
    step = _EXACT.power(base, _EXACT.divide(decimal.Decimal(-2), dim)) if dim else 0
    f, ladder = decimal.Decimal(1), []
    for _ in range(dim // 2):
        ladder.append(_turns(f))
        f = _EXACT.multiply(f, step)
    return tuple(ladder)


class AxisRope:
    """Which way each pair of a head turns: `turns` int64 [pairs] (turns per position, times 2^64), `axis` uint8 [pairs].

    AxisRope(axes_dim, theta): one block of pairs per axis, each with its own frequencies theta^(-2 i / dim) (theta: a number, or one per axis), as
    flux_rope_table lays them out.  AxisRope.sections: one ladder of frequencies over all pairs, cut into one section per axis.
    AxisRope.from_pairs: any frequency and axis per pair (scaled or learned frequencies, axes dealt in turn).  interleaved: pair i is (x[2 i],
    x[2 i + 1]), else (x[i], x[i + pairs]).  Elements of a head beyond 2 * pairs are left alone."""

    def __init__(self, axes_dim, theta=10000.0, interleaved=True, device="cuda"):
        thetas = list(theta) if isinstance(theta, (list, tuple)) else [theta] * len(axes_dim)
        if len(thetas) != len(axes_dim):
            raise ValueError("rope: %d axes and %d thetas" % (len(axes_dim), len(thetas)))
        turns, axis = [], []
        for a, (dim, th) in enumerate(zip(axes_dim, thetas)):
            if dim % 2 or dim < 0:
                raise ValueError("rope: the axis dimension must be even, got %d" % dim)
            turns += _ladder(dim, float(th))
            axis += [a] * (dim // 2)
        self._set(turns, axis, len(axes_dim), interleaved, device)

    def _set(self, turns, axis, axes, interleaved, device):
        if len(turns) != len(axis) or axes > 255 or any(not 0 <= a < axes for a in axis):
            raise ValueError("rope: one axis below %d for each of %d pairs" % (min(axes, 255), len(turns)))
        self.pairs, self.axes, self.interleaved = len(turns), axes, bool(interleaved)
        self.turns = torch.tensor(turns, dtype=torch.int64, device=device)
        self.axis = torch.tensor(axis, dtype=torch.uint8, device=device)

    @classmethod
    def sections(cls, sections, theta=10000.0, interleaved=False, device="cuda"):
        """sections: pairs per axis; pair i of all has frequency theta^(-i / pairs)."""
        plan = cls.__new__(cls)
        plan._set(list(_ladder(2 * sum(sections), float(theta))), [a for a, n in enumerate(sections) for _ in range(n)], len(sections), interleaved, device)
        return plan

    @classmethod
    def from_pairs(cls, freq, axis, axes, interleaved=False, device="cuda"):
        """freq: radians per position of each pair (floats), axis: its position axis, below `axes`."""
        plan = cls.__new__(cls)
        plan._set([_turns(float(f)) for f in freq], [int(a) for a in axis], axes, interleaved, device)
        return plan


def axis_table(pos, dim, theta):
    """pos [B, S] -> [B, S, dim/2, 2, 2] fp32 for one position axis with `dim` channels."""
    if dim % 2:
        raise ValueError("rope: the axis dimension must be even, got %d" % dim)
    freq = torch.pow(torch.tensor(float(theta), dtype=torch.float64, device=pos.device),
                     -torch.arange(0, dim, 2, dtype=torch.float64, device=pos.device) / dim)
    ang = pos.to(torch.float64).unsqueeze(-1) * freq
    c, s = torch.cos(ang), torch.sin(ang)
    rot = torch.stack([c, -s, s, c], dim=-1)
    return rot.reshape(pos.shape[0], -1, dim // 2, 2, 2).float()


def flux_rope_table(ids, axes_dim=(16, 56, 56), theta=10000):
    """ids [B, S, n_axes] (text rows all zero, image rows (0, y, x)) -> [B, 1, S, sum(axes_dim)/2, 2, 2] fp32."""
    if ids.shape[-1] != len(axes_dim):
        raise ValueError("rope: ids has %d axes, axes_dim %d" % (ids.shape[-1], len(axes_dim)))
    parts = [axis_table(ids[..., a], axes_dim[a], theta) for a in range(len(axes_dim))]
    return torch.cat(parts, dim=-3).unsqueeze(1)


def flux_position_ids(text_tokens, height, width, batch=1, device="cpu"):
    """Position ids of a FLUX sequence: `text_tokens` zero rows, then height x width image rows (0, y, x)."""
    ids = torch.zeros(batch, text_tokens + height * width, 3, device=device)
    ids[:, text_tokens:, 1] = torch.arange(height, device=device).repeat_interleave(width).float()
    ids[:, text_tokens:, 2] = torch.arange(width, device=device).repeat(height).float()
    return ids
