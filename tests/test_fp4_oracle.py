"""CPU checks of the FP4 restatement that the GPU tests compare with: code tables, ties, saturation, the scale order, the tensor scale; and
of what the host side of the FP4 operators refuses."""

import pytest
import torch

from lyradiff_b200 import _lib, build, ops
from oracle import fp4


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def test_code_tables():
    assert fp4.E2M1.tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6]
    assert fp4.E4M3[-1] == 448 and fp4.E4M3[1] == 2.0 ** -9 and fp4.E4M3[8] == 2.0 ** -6 and len(fp4.E4M3) == 127


def test_ties_go_to_the_even_code():
    v = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, 100.0, 0.2499, 0.2501], dtype=torch.float64)
    assert fp4.nearest(fp4.E2M1, v).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7, 0, 1]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_round_trip_of_representable_values(fmt):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 16, (5, 96), generator=g).to(torch.uint8)
    codes[:, ::fp4.GROUP[fmt]] = 7                                    # each block reaches 6, so its scale comes back too
    s = torch.randint(100, 110, (5, 96 // fp4.GROUP[fmt]), generator=g).to(torch.uint8)
    x = fp4.decode(codes, s, fmt, 0.25 if fmt == "nvfp4" else 1.0)
    c2, s2 = fp4.encode(x, fmt, 0.25)
    assert torch.equal(s, s2)
    assert torch.equal(fp4.decode(c2, s2, fmt), fp4.decode(codes, s, fmt))
    assert torch.equal(fp4.unpack(fp4.pack(codes)), codes)


def test_blocks_that_hold_nan_or_infinity_read_back_as_nan():
    x = torch.ones(1, 64)
    x[0, 3], x[0, 40] = float("nan"), float("-inf")
    for fmt in ("nvfp4", "mxfp4"):
        bad = torch.isnan(fp4.decode(*fp4.encode(x, fmt), fmt))
        n = fp4.GROUP[fmt]
        want = torch.zeros(64, dtype=torch.bool)
        want[3 // n * n:3 // n * n + n] = True
        want[40 // n * n:40 // n * n + n] = True
        assert torch.equal(bad[0], want)


@pytest.mark.parametrize("rows,k", [(1, 32), (128, 64), (129, 160), (300, 4096)])
def test_scale_order_is_a_permutation_into_the_buffer(lib, rows, k):
    for fmt, code in ops.FP4_FORMATS.items():
        at = fp4.scale_offsets(rows, k // fp4.GROUP[fmt]).flatten()
        size = fp4.scale_bytes(rows, k, fmt)
        assert at.unique().numel() == at.numel() and int(at.max()) < size
        assert lib.lyraq_fp4_scale_bytes(rows, k, code) == size


def test_tensor_scale_is_the_least_power_of_two():
    assert fp4.tensor_scale(torch.tensor([2688.0])) == 1.0
    assert fp4.tensor_scale(torch.tensor([2688.5])) == 2.0
    assert fp4.tensor_scale(torch.tensor([-0.03, float("inf")])) == 2.0 ** -16
    assert fp4.tensor_scale(torch.zeros(3)) == 0.0


def test_c_entry_points_refuse_without_a_device(lib):
    INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 5
    p = 0x1000
    assert lib.lyraq_fp4_scale_bytes(4, 64, 7) == 0
    quant = lambda **k: lib.lyraq_quant_fp4(*[{**dict(q=p, s=p, x=p, dt=1, ld=64, g=p, f=0, r=4, k=64, st=None), **k}[n]   # noqa: E731
                                              for n in ("q", "s", "x", "dt", "ld", "g", "f", "r", "k", "st")])
    assert quant(f=2) == INVALID and quant(q=None) == INVALID and quant(x=p + 8) == INVALID and quant(s=p + 4) == INVALID
    assert quant(k=48) == UNSUPPORTED and quant(dt=3) == UNSUPPORTED and quant(ld=60) == INVALID and quant(ld=68) == INVALID
    assert quant(r=0) == 0
    weight = lambda **k: lib.lyraq_weight_quant_fp4(*[{**dict(q=p, s=p, g=p, w=p, dt=1, f=0, n=4, k=64, st=None), **k}[n]   # noqa: E731
                                                      for n in ("q", "s", "g", "w", "dt", "f", "n", "k", "st")])
    assert weight(g=None) == INVALID and weight(k=40) == UNSUPPORTED and weight(w=None) == INVALID and weight(n=0) == 0 and weight(f=-1) == INVALID
    gemm = lambda **k: lib.lyraq_gemm_fp4(*[{**dict(x=p, xs=p, xg=None, w=p, ws=p, wg=None, f=0, y=p, dt=1, b=None, r=None, beta=1.0, e=0, m=4,   # noqa: E731
                                                    n=8, k=64, st=None), **k}[n]
                                            for n in ("x", "xs", "xg", "w", "ws", "wg", "f", "y", "dt", "b", "r", "beta", "e", "m", "n", "k", "st")])
    assert gemm(f=3) == INVALID and gemm(e=2) == INVALID and gemm(dt=3) == INVALID and gemm(m=-1) == INVALID and gemm(y=None) == INVALID
    assert gemm(w=p + 1) == INVALID and gemm(b=p + 2) == INVALID and gemm(r=p + 8) == INVALID and gemm(k=16) == UNSUPPORTED and gemm(k=0) == UNSUPPORTED
    assert gemm(m=0) == 0 and gemm(n=0) == 0
    lin = lambda **k: lib.lyraq_linear_fp4_forward(*[{**dict(y=p, x=p, dt=1, ld=64, xg=None, w=p, ws=p, wg=None, f=0, b=None, r=None, beta=1.0,   # noqa: E731
                                                             e=0, m=4, n=8, k=64, wsp=p, wsb=1 << 20, st=None), **k}[n]
                                                     for n in ("y", "x", "dt", "ld", "xg", "w", "ws", "wg", "f", "b", "r", "beta", "e", "m", "n", "k",
                                                               "wsp", "wsb", "st")])
    assert lin(wsp=None) == WORKSPACE and lin(wsb=64) == WORKSPACE and lin(k=48) == UNSUPPORTED and lin(y=None) == INVALID and lin(m=0) == 0
    assert lin(x=None) == INVALID and lin(ld=32) == INVALID and lin(f=9) == INVALID and lin(e=4) == INVALID
    assert lib.lyraq_workspace_bytes(8, 200, 64, 96) == 200 * 48 // 256 * 256 + 256 + 2 * 2 * 512
    assert lib.lyraq_workspace_min_bytes(8, 200, 64, 96) == lib.lyraq_workspace_bytes(8, 200, 64, 96)


def test_python_side_refuses_parts_that_do_not_fit(lib):
    t = lambda *s: torch.empty(*s, dtype=torch.uint8)   # noqa: E731
    for bad in (ops.Fp4Tensor(4, 64, "nvfp4", t(4, 31), t(512)), ops.Fp4Tensor(4, 64, "nvfp4", t(4, 32), t(511)), ops.Fp4Tensor(4, 48, "mxfp4", t(4, 24), t(512)),
                ops.Fp4Tensor(4, 64, "fp4", t(4, 32), t(512)), ops.Fp4Tensor(4, 64, "nvfp4", t(4, 32), t(512), torch.ones(2))):
        with pytest.raises(ValueError):
            bad.check()
    with pytest.raises(ValueError):
        ops.Fp4Tensor.empty(4, 64, "int4", device="cpu")


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nothing lies at")
def test_sizes_next_to_31_bits_are_refused_by_linear_and_product_alike(lib):
    UNSUPPORTED, p = 2, [(i + 1) << 44 for i in range(5)]
    for m, n, k in ((1, 1, 0x7fffffe0), (1, 0x7fffffff, 32), (0x7fffffff, 1, 32)):
        assert lib.lyraq_gemm_fp4(p[0], p[1], None, p[2], p[3], None, 0, p[4], 1, None, None, 0.0, 0, m, n, k, None) == UNSUPPORTED
        need = lib.lyraq_workspace_bytes(8, m, n, k)
        assert lib.lyraq_linear_fp4_forward(p[0], p[1], 1, k, None, p[2], p[3], None, 0, None, None, 0.0, 0, m, n, k, p[4], need, None) == UNSUPPORTED


def test_input_scales_are_rounded_up_to_powers_of_two_of_fp32():
    from lyradiff_b200 import layers
    f = layers._power_of_two
    for s, want in ((1.0, 1.0), (0.011, 2.0 ** -6), (2.0 ** -7, 2.0 ** -7), (1.0000001, 2.0), (2.0 ** 127, 2.0 ** 127), (1e-40, 2.0 ** -126), (1e-300, 2.0 ** -126)):
        got = f(torch.tensor(s, dtype=torch.float64))
        assert got.dtype == torch.float32 and got.shape == (1,) and float(got) == want
    for s in (0.0, -1.0, float("nan"), float("inf"), 3e38, 1e300):
        with pytest.raises(ValueError):
            f(torch.tensor([s], dtype=torch.float64))


def test_mxfp4_has_no_tensor_scale():
    """Its quantizer reads none, so a product that multiplied by one would be off by it."""
    t, g = lambda *s: torch.empty(*s, dtype=torch.uint8), torch.ones(1)   # noqa: E731
    with pytest.raises(ValueError, match="mxfp4"):
        ops.Fp4Tensor(4, 64, "mxfp4", t(4, 32), t(512), g)
    with pytest.raises(ValueError, match="mxfp4"):
        ops.Fp4Tensor.empty(4, 64, "mxfp4", g, "cpu")
    with pytest.raises(ValueError, match="mxfp4"):
        ops.quant_fp4(torch.zeros(4, 64), g, "mxfp4")
    assert ops.Fp4Tensor(4, 64, "nvfp4", t(4, 32), t(512), g).tensor_scale is g
