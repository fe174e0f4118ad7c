"""CPU checks of the rotary plan and of what the C entry points of the norm and the rotary embedding refuse."""

import ctypes
import math

import pytest
import torch

from lyradiff_b200 import _lib, build, rope


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def test_frequencies_are_fractions_of_a_turn():
    plan = rope.AxisRope((16, 56, 56), device="cpu")
    assert plan.pairs == 64 and plan.axes == 3 and plan.interleaved
    assert plan.axis.tolist() == [0] * 8 + [1] * 28 + [2] * 28
    turns = [int(t) % 2 ** 64 / 2.0 ** 64 for t in plan.turns]
    want = [10000.0 ** (-2 * i / d) / (2 * math.pi) for d in (16, 56, 56) for i in range(d // 2)]
    # the 64-bit ladder: its exponent is rounded (2^-53, times log theta = 9.2 in the result), then pow (2^-52), the division and 2 pi
    assert all(abs(a - b) <= (9.3 + 2 + 3) * 2.0 ** -53 * b for a, b in zip(turns, want))
    own = rope.AxisRope.sections((2, 2), theta=500000.0, device="cpu")
    assert [int(t) % 2 ** 64 for t in own.turns][0] == 2935890503282001226 and not own.interleaved


def test_far_positions_wrap_exactly():
    """pos * turns modulo 2^64 is the angle: against the same product in whole numbers of a 400-bit pi."""
    plan = rope.AxisRope((8,), device="cpu")
    for t, f in zip(plan.turns.tolist(), (1.0, 0.1, 0.01, 0.001)):
        for pos in (1, 10 ** 6 + 3, 2 ** 31 - 1, -12345):
            frac = (pos * t) % 2 ** 64 / 2.0 ** 64
            ang = math.fmod(pos * f, 2 * math.pi) / (2 * math.pi) % 1.0     # 64-bit: about pos * 2^-53 off
            d = abs(frac - ang)
            assert min(d, 1 - d) <= abs(pos) * 2.0 ** -50 + 2.0 ** -50


def test_plans_that_make_no_sense_are_refused():
    for bad in (lambda: rope.AxisRope((15,), device="cpu"), lambda: rope.AxisRope((16, 16), theta=[1e4], device="cpu"), lambda: rope.AxisRope((16,), theta=-1.0, device="cpu"),
                lambda: rope.AxisRope.from_pairs([1.0], [1], 1, device="cpu"), lambda: rope.AxisRope.from_pairs([1.0, 2.0], [0], 1, device="cpu"),
                lambda: rope.AxisRope.from_pairs([7.0], [0], 1, device="cpu"), lambda: rope.AxisRope.from_pairs([float("nan")], [0], 1, device="cpu"),
                lambda: rope.AxisRope.from_pairs([-0.5], [0], 1, device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_c_entry_points_refuse_without_a_device(lib):
    p, ok = 0x1000, 0
    INVALID, UNSUPPORTED = 1, 2

    def norm(**k):
        a = _lib.GatedNormArgs(**{**dict(y=p, x=p, x_out=p, h=2 * p, dtype=1, post=1, pre=2, batch=1, seq_len=4, dim=64, y_row=64, x_row=64, x_out_row=64, h_row=64), **k})
        return lib.lyraq_gated_residual_norm(ctypes.byref(a), None)
    assert lib.lyraq_gated_residual_norm(None, None) == INVALID
    assert norm(seq_len=0) == ok and norm(dim=60) == UNSUPPORTED and norm(dim=16392) == UNSUPPORTED and norm(dtype=2) == UNSUPPORTED
    assert norm(y=None) == INVALID and norm(x=p + 2) == INVALID and norm(pre=0) == INVALID and norm(post=3) == INVALID and norm(x_row=60) == INVALID
    assert norm(x_out=None, h=None) == INVALID and norm(qf8=p) == INVALID and norm(qf8=p + 4, f8_scale=p) == INVALID and norm(q4=p) == INVALID
    assert norm(q4=p, q4_scales=p, q4_format=5) == INVALID and norm(q4=p, q4_scales=p, dim=72) == UNSUPPORTED and norm(gate=p, gate_batch=4) == INVALID
    assert norm(post_weight=p + 8) == INVALID and norm(h=p) == INVALID

    def turn(**k):
        a = _lib.RopeAxesArgs(**{**dict(q=p, q_out=p, positions=p, turns=p, axis=p, pos_dtype=3, dtype=1, q_heads=2, head_dim=64, pairs=32, batch=1, seq_len=3), **k})
        return lib.lyraq_rope_axes(ctypes.byref(a), None)
    assert lib.lyraq_rope_axes(None, None) == INVALID
    assert turn(seq_len=0) == ok and turn(q_heads=0) == ok and turn(dtype=2) == UNSUPPORTED and turn(pos_dtype=1) == INVALID and turn(q=None) == INVALID
    assert turn(k_heads=1) == INVALID and turn(head_dim=258, pairs=4) == UNSUPPORTED and turn(head_dim=63, pairs=4) == UNSUPPORTED and turn(pairs=33) == UNSUPPORTED
    assert turn(turns=None) == INVALID and turn(positions=p + 2) == INVALID and turn(q=p + 1) == INVALID and turn(q_heads=-1) == INVALID
    assert turn(pos_dtype=5, positions=p + 4) == INVALID


def test_ctypes_structures_are_those_of_the_header(tmp_path):
    """Sizes and the place of every field, from the C compiler."""
    import os
    import shutil
    import subprocess
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "lyraq.h")
    pairs = (("lyraq_gated_norm_t", _lib.GatedNormArgs), ("lyraq_rope_axes_t", _lib.RopeAxesArgs))
    lines = ["printf(\"%%zu\\n\", sizeof(%s));" % c for c, _ in pairs]
    lines += ["printf(\"%%zu\\n\", offsetof(%s, %s));" % (c, f) for c, s in pairs for f, _ in s._fields_]
    src = tmp_path / "fields.cpp"
    src.write_text("#include \"%s\"\n#include <cstdio>\nint main() { %s }\n" % (header, " ".join(lines)))
    subprocess.run(["g++", str(src), "-o", str(tmp_path / "fields")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "fields")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(s) for _, s in pairs] + [getattr(s, f).offset for _, s in pairs for f, _ in s._fields_]
