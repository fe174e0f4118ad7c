"""CPU tests of the FP8 block format's restatement, and of what its calls refuse before they touch a device."""

import pytest
import torch

from lyradiff_b200 import _lib, build
from oracle import fp8_block


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("rows,k,block_rows", [(3, 128, 1), (5, 336, 1), (130, 272, 128), (128, 16, 128)])
def test_round_trip(rows, k, block_rows):
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g).bfloat16()
    codes, s = fp8_block.encode(x, block_rows)
    back = fp8_block.decode(codes, s, block_rows)
    full = fp8_block.spread(s, rows, k, block_rows).double()
    # half a step of e4m3 is 2^-4 of a normal number, 2^-10 scales of a subnormal one; 2^-22 for the roundings of scale and quotient
    assert bool(((back - x.double()).abs() <= x.double().abs() * (2.0 ** -4 + 2.0 ** -22) + full * 2.0 ** -10).all())
    again, s2 = fp8_block.encode(back.float(), block_rows)
    assert bool(((s2 - s).abs() <= s * 2.0 ** -22).all())
    sign = lambda c: torch.where(c == 128, 0, c.int())   # noqa: E731
    assert float((sign(again) != sign(codes)).float().mean()) < 0.01


def test_blocks_of_zeros_and_of_no_numbers():
    x = torch.zeros(2, 256)
    x[0, 130] = float("inf")
    x[1, 3] = float("nan")
    codes, s = fp8_block.encode(x)
    assert s.isnan().tolist() == [[False, True], [True, False]]
    assert float(s[0, 0]) == 2.0 ** -100 and not bool(codes.any())


def test_refusals(lib):
    INVALID, UNSUPPORTED, WORKSPACE, p = 1, 2, 5, 0x100000
    far = [p + (i << 32) for i in range(8)]
    quant = lambda q=far[0], s=far[1], sr=4, sb=1, x=far[2], t=1, ldx=512, rows=3, k=512: lib.lyraq_quant_fp8_block(q, s, sr, sb, x, t, ldx, rows, k, None)  # noqa: E731
    assert quant(rows=0) == 0 and quant(k=0) == 0
    assert quant(q=None) == quant(s=None) == quant(x=None) == quant(q=far[0] + 8) == quant(x=far[2] + 2) == quant(s=far[1] + 2) == INVALID
    assert quant(ldx=504) == quant(ldx=516) == INVALID
    assert quant(k=500) == quant(t=3) == UNSUPPORTED
    assert quant(sr=0) == quant(sr=3) == quant(sb=0) == quant(sr=2, sb=3) == INVALID          # two scales in one place
    assert quant(q=far[2]) == quant(s=far[0] + 512) == quant(s=far[2] + 1024) == INVALID      # memory in common
    weight = lambda q=far[0], s=far[1], w=far[2], t=1, n=256, k=256: lib.lyraq_weight_quant_fp8_block(q, s, w, t, n, k, None)  # noqa: E731
    assert weight(n=0) == 0 and weight(k=250) == UNSUPPORTED and weight(q=far[2]) == weight(s=far[0]) == weight(w=None) == INVALID
    def gemm(X=far[0], xs=far[1], sr=1, sb=4, W=far[2], ws=far[3], Y=far[4], t=1, b=None, r=None, epi=0, m=4, n=256, k=256):
        return lib.lyraq_gemm_fp8_block(X, xs, sr, sb, W, ws, Y, t, b, r, 1.0, epi, m, n, k, None)
    assert gemm(m=0) == gemm(n=0) == 0
    assert gemm(m=-1) == gemm(epi=2) == gemm(t=3) == gemm(X=None) == gemm(W=far[2] + 4) == gemm(b=far[5] + 2) == gemm(r=far[5] + 2) == INVALID
    assert gemm(k=0) == gemm(k=24) == gemm(n=0x7fffff80) == UNSUPPORTED
    for y in (far[0], far[1] + 12, far[2] + 16, far[3]):
        assert gemm(Y=y & ~15) == INVALID
    assert gemm(r=far[4] + 16) == INVALID                                                      # the residual, but not element for element
    need = lib.lyraq_workspace_bytes(9, 5, 256, 256)
    assert need >= 5 * 256 + 2 * 8 * 4
    def linear(Y=far[0], x=far[1], t=1, ldx=256, W=far[2], ws=far[3], b=None, r=None, epi=0, m=5, n=256, k=256, work=far[4], size=need):
        return lib.lyraq_linear_fp8_block_forward(Y, x, t, ldx, W, ws, b, r, 1.0, epi, m, n, k, work, size, None)
    assert linear(m=0) == 0
    assert linear(work=None) == linear(size=need - 1) == linear(work=far[4] + 8) == WORKSPACE
    assert linear(x=None) == linear(ldx=248) == linear(Y=far[2]) == linear(Y=far[4]) == linear(work=far[1]) == linear(work=far[2]) == linear(epi=7) == INVALID
    assert linear(k=100) == linear(t=4) == UNSUPPORTED
