"""CPU tests of the check that an output shares no memory with what a kernel still reads (csrc/views.h), and of the entry points that make it."""

import ctypes
import itertools
import os
import random
import shutil
import subprocess

import pytest
import torch

from lyradiff_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, CUDA = 0, 1, 2, 3
PROGRAM = """
#include "%s"
#include <cstdio>
using namespace lyraq;
int main()
{
    size_t v[18];
    for (;;) {
        for (size_t& x : v)
            if (std::scanf("%%zu", &x) != 1) return 0;
        const View a = view_of((const void*)v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]);
        const View b = view_of((const void*)v[9], v[10], v[11], v[12], v[13], v[14], v[15], v[16], v[17]);
        std::printf("%%d %%d %%d\\n", (int)views_meet(a, b), (int)views_meet(b, a), (int)views_same(a, b));
    }
}
"""


@pytest.fixture(scope="module")
def decide(tmp_path_factory):
    """[(a, b)] of views (base, element bytes, n0, s0, n1, s1, n2, s2, run) -> [(meet, meet the other way round, same)]."""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("views")
    (at / "views.cpp").write_text(PROGRAM % os.path.join(ROOT, "lyradiff_b200", "csrc", "views.h"))
    subprocess.run(["g++", "-std=c++17", "-O1", str(at / "views.cpp"), "-o", str(at / "views")], check=True)

    def run(pairs):
        text = "\n".join(" ".join(str(v) for v in a + b) for a, b in pairs)
        out = subprocess.run([str(at / "views")], input=text, check=True, capture_output=True, text=True).stdout
        return [tuple(int(v) for v in li.split()) for li in out.splitlines()]
    return run


def memory(v):
    base, e, n0, s0, n1, s1, n2, s2, run = v
    return {base + e * (i * s0 + j * s1 + k * s2) + r for i, j, k in itertools.product(range(n0), range(n1), range(n2)) for r in range(run * e)}


def test_against_every_byte(decide):
    rng = random.Random(3)
    pairs = []
    for _ in range(4000):
        e = rng.choice([1, 2])
        if rng.random() < 0.5:     # two parts of one packed tensor, as they lie or moved
            run, heads, parts = rng.randint(1, 4), rng.randint(1, 3), rng.randint(2, 3)
            seq, batch = rng.randint(1, 3), rng.randint(1, 2)
            row = run * heads * parts
            s = (batch, seq * row, seq, row, heads, run, run)
            a = (1000, e) + s
            b = (1000 + e * rng.choice([heads * run, run, run * (parts - 1) * heads, rng.randint(-2 * row, 2 * row)]), e) + s
        else:
            a, b = ((1000 + rng.randint(0, 40), e) + tuple(v for _ in range(3) for v in (rng.randint(1, 4), rng.randint(0, 30))) + (rng.randint(1, 4),)
                    for _ in range(2))
        pairs.append((a, b))
    got = decide(pairs)
    assert len(got) == len(pairs)
    met = 0
    for (a, b), (meet, back, same) in zip(pairs, got):
        want = not memory(a).isdisjoint(memory(b))
        assert meet == want and back == want, (a, b)
        met += want
    assert 500 < met < 3500


def test_sizes_of_real_tensors(decide):
    """Parts of a packed projection of 2^33 elements, heads before tokens, an expanded batch, two tensors with nothing between them; a dimension of one has any stride."""
    B, S, H, D = 8, 65536, 32, 128
    row = 3 * H * D
    q = (1 << 40, 2, B, S * row, S, row, H, D, D)
    k = (q[0] + 2 * H * D,) + q[1:]
    moved = (q[0] + 2 * D,) + q[1:]
    rows = (q[0] + 2 * row,) + q[1:]
    by_head = (q[0] + 2 * D, 2, B, S * row, S, D, H, S * D, D)
    behind = (q[0] + 2 * B * S * row, 2, B, S * H * D, S, H * D, H, D, D)
    one = (1 << 40, 2, 1, 12345, S, row, H, D, D)
    other = (1 << 40, 2, 1, 77, S, row, H, D, D)
    expanded = (k[0], 2, B, 0, S, row, H, D, D)
    got = decide([(q, k), (q, moved), (q, rows), (q, by_head), (q, behind), (q, q), (one, other), (q, expanded), (q, (0,) + q[1:])])
    assert [g[0] for g in got] == [0, 1, 1, 1, 0, 1, 1, 0, 0]
    assert [g[2] for g in got] == [0, 0, 0, 0, 0, 1, 1, 0, 0]


needs_no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nothing lies at: a call that is let through must find no device")


@needs_no_gpu
def test_rotary_embedding_refuses_outputs_on_what_it_reads():
    lib = _lib.lib()
    B, S, H, D = 2, 5, 4, 64
    p = 1 << 30
    packed = dict(zip(("batch", "token", "head"), (S * 3 * H * D, 3 * H * D, D)))

    def turn(**kw):
        a = dict(q=p, k=p + 2 * H * D, q_out=p + (1 << 24), k_out=p + (1 << 25), positions=p + (1 << 26), turns=p + (1 << 26), axis=p + (1 << 26), pos_dtype=3, dtype=1,
                 q_heads=H, k_heads=H, head_dim=D, pairs=D // 2, batch=B, seq_len=S)
        for t in ("q", "k", "q_out", "k_out"):
            a.update({t + "_" + n: v for n, v in packed.items()})
        return lib.lyraq_rope_axes(ctypes.byref(_lib.RopeAxesArgs(**{**a, **kw})), None)
    assert turn() == CUDA
    # in place, and on the part that neither reads
    assert turn(q_out=p, k_out=p + 2 * H * D) == CUDA and turn(q_out=p + 4 * H * D) == CUDA
    # one head on, one token on, on the other part, on part of it, on each other, other strides at the same place
    assert turn(q_out=p + 2 * D) == INVALID and turn(q_out=p + 6 * H * D) == INVALID
    assert turn(q_out=p + 2 * H * D) == INVALID and turn(k_out=p) == INVALID and turn(k_out=p + 2 * D) == INVALID
    assert turn(k_out=p + (1 << 24)) == INVALID and turn(k_out=p + (1 << 24) + 2 * D) == INVALID and turn(k_out=p + (1 << 24) + 2 * H * D) == CUDA
    assert turn(q_out=p, q_out_token=D, q_out_head=S * D) == INVALID and turn(k_out=p + 2 * H * D, k_out_batch=1024) == INVALID
    assert turn(q_out=p, batch=1, q_out_batch=7) == CUDA and turn(q_out=p, seq_len=1, q_out_token=7) == CUDA
    # without k its place is free
    assert turn(k=None, k_out=None, k_heads=0, q_out=p + 2 * H * D) == CUDA


@needs_no_gpu
def test_norms_refuse_outputs_on_what_they_read():
    lib = _lib.lib()
    B, S, D = 2, 5, 64
    p, far = 1 << 30, [p << 20 for p in range(1, 9)]
    joint = dict(zip(("batch", "row"), (8 * D, D)))       # 5 of 8 rows

    def norm(**kw):
        a = dict(y=p + far[0], x=p, x_out=p + far[1], h=p + far[2], batch=B, seq_len=S, dim=D, dtype=1, post=1, pre=2, residual_scale=1.0, eps=1e-6)
        for t in ("y", "x", "x_out", "h"):
            a.update({t + "_" + n: v for n, v in joint.items()})
        return lib.lyraq_gated_residual_norm(ctypes.byref(_lib.GatedNormArgs(**{**a, **kw})), None)
    assert norm() == CUDA
    # either output in either input's place, and on rows that nobody reads
    assert norm(x_out=p, h=p + far[0]) == CUDA and norm(x_out=p + far[0], h=p) == CUDA and norm(y=p, x_out=p) == CUDA
    assert norm(x_out=p, h=p + 2 * 5 * D, seq_len=3) == CUDA
    # a row on, within a row, with other strides, on each other, the two inputs a row apart
    assert norm(x_out=p + 2 * D) == INVALID and norm(h=p + 2 * D) == INVALID and norm(x_out=p + far[0] - 16) == INVALID and norm(x_out=p, x_out_batch=5 * D) == INVALID
    assert norm(x_out=p + far[2]) == INVALID and norm(x_out=p + far[2] + 2 * D) == INVALID and norm(y=p + 2 * D, x_out=p) == INVALID
    assert norm(x_out=p, batch=1, x_out_batch=5 * D) == CUDA
    # the quantized outputs: apart from everything
    q = dict(f8_scale=p + far[7], q4_format=0)
    for name, size in (("qf8", B * S * D), ("q4", B * S * D // 2)):
        more = dict(q, q4_scales=p + far[6]) if name == "q4" else q
        assert norm(**{name: p + far[3]}, **more) == CUDA
        for at in (p, p + 2 * D, p + far[0], p + far[1], p + far[2], p + far[2] - size + 16):
            assert norm(**{name: at}, **more) == INVALID
        assert norm(**{name: p + far[0] - size}, **more) == CUDA
    both = dict(q, qf8=p + far[3], q4=p + far[4], q4_scales=p + far[5])
    assert norm(**both) == CUDA
    for name, at in (("qf8", far[4]), ("q4", far[3]), ("q4_scales", far[3]), ("q4_scales", far[4]), ("q4_scales", 0), ("q4_scales", far[1])):
        assert norm(**{**both, name: p + at}) == INVALID


@needs_no_gpu
def test_fp4_products_refuse_a_result_on_what_they_read():
    lib = _lib.lib()
    m, n, k = 300, 256, 512
    p = [(i + 1) << 30 for i in range(9)]
    size = {"X": m * k // 2, "xs": lib.lyraq_fp4_scale_bytes(m, k, 0), "W": n * k // 2, "ws": lib.lyraq_fp4_scale_bytes(n, k, 0), "bias": 2 * n, "R": 2 * m * n}

    def gemm(Y=p[0], X=p[1], xs=p[2], W=p[3], ws=p[4], bias=p[5], R=p[6]):
        return lib.lyraq_gemm_fp4(X, xs, None, W, ws, None, 0, Y, 1, bias, R, 1.0, 0, m, n, k, None)

    need = lib.lyraq_workspace_bytes(8, m, n, k)

    def linear(Y=p[0], x=p[1], W=p[3], ws=p[4], bias=p[5], R=p[6], work=p[7]):
        return lib.lyraq_linear_fp4_forward(Y, x, 1, k, None, W, ws, None, 0, bias, R, 1.0, 0, m, n, k, work, need, None)
    assert gemm() == CUDA and linear() == CUDA and gemm(R=p[0]) == CUDA and linear(R=p[0]) == CUDA and gemm(bias=None, R=None) == CUDA
    assert linear(x=p[0]) == CUDA and linear(x=p[0] + 2 * n) == CUDA           # the rows are quantized before
    for call in (gemm, linear):
        for name in ("X", "xs", "W", "ws", "bias", "R"):
            if call is linear and name in ("X", "xs"):
                continue
            for at in (p[0] - size[name] + 16, p[0] + 16, p[0] + 2 * m * n - 16):
                assert call(**{name: at}) == INVALID, (call, name)
            assert call(**{name: p[0] - (size[name] + 15) // 16 * 16}) == CUDA and call(**{name: p[0] + 2 * m * n}) == CUDA
    assert linear(work=p[0] - 16) == INVALID and linear(work=p[6] + 32) == INVALID and linear(work=p[1] - need + 16) == INVALID
