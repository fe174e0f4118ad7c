"""GPU tests of the microscaled FP4 operators against the 64-bit restatement in oracle/fp4.py."""

import pytest
import torch

from oracle import fp4
from tests.util import check_status, cu

pytestmark = pytest.mark.gpu

FORMATS = ["nvfp4", "mxfp4"]


@pytest.fixture(scope="module")
def ops():
    from lyradiff_b200 import ops as _ops
    return _ops


@pytest.fixture
def tile():
    from lyradiff_b200 import _lib
    yield lambda code: _lib.check(_lib.lib().lyraq_debug_force_fp4_tile(code), "lyraq_debug_force_fp4_tile")
    _lib.lib().lyraq_debug_force_fp4_tile(0)


def assert_quantized(t, x, fmt, g=1.0):
    """Codes (as values: the sign of a zero does not matter) and scale bytes are exactly those of the definition, and blocks that a
    row does not have carry scale 0."""
    codes, s = fp4.encode(x, fmt, g)
    rows, k = x.shape
    got = fp4.unpack(t.codes.cpu())
    blocks = k // fp4.GROUP[fmt]
    sb = t.scales.cpu()
    assert torch.equal(sb[fp4.scale_offsets(rows, blocks)], s)
    pad = (blocks + 3) // 4 * 4
    assert not bool(sb[fp4.scale_offsets(rows, pad)][:, blocks:].any())
    sign = lambda c: torch.where(c == 8, 0, c)   # noqa: E731
    assert torch.equal(sign(got), sign(codes))


def inputs(rows, k, dtype, seed, spread=3.0):
    """Values over several binades, so that blocks differ in scale, with exact ties, zeros and a block of zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp2(spread * torch.randn(rows, k // 32, generator=g)).repeat_interleave(32, dim=1)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]) * torch.tensor([1.0, -1.0] * 4)
    x[::3, :8], x[1::4, 8:16] = ties, ties * 1.125 / 4
    x[::5, :32] = 0
    x[:, -1] = -x[:, -1]
    return x.clamp(-60000, 60000).to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (31, 160), (33, 64), (128, 256), (130, 1056), (300, 640)])
def test_quantize_is_exact(ops, fmt, dtype, rows, k):
    x = inputs(rows, k, dtype, rows + k)
    for g in ((1.0, 2.0 ** -5) if fmt == "nvfp4" else (None,)):
        t = ops.quant_fp4(cu(x), None if g is None else torch.tensor([g], device="cuda"), fmt)
        check_status()
        assert_quantized(t, x, fmt, g or 1.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_of_the_types_extremes(ops, fmt):
    """Subnormals, the largest numbers, infinities and NaN, a block scale that underflows, one that saturates."""
    x = torch.zeros(9, 64)
    x[0] = 1e-42
    x[1, 5] = 3.0e38
    x[1, 40] = -3.0e38
    x[2, 7], x[2, 50] = float("inf"), float("nan")
    x[3] = torch.linspace(-1e-3, 1e-3, 64)
    x[4] = 2.0 ** -126
    x[5, ::2] = -0.0
    x[6] = torch.tensor([448.0 * 6 * 4, 1.0] * 32)
    x[7, 63] = float("-inf")
    x[8] = torch.linspace(1e-38, 5e-38, 64)
    t = ops.quant_fp4(cu(x), None, fmt)
    check_status()
    assert_quantized(t, x, fmt)
    h = x.clamp(-3e38, 3e38).nan_to_num(0).bfloat16()
    assert_quantized(ops.quant_fp4(cu(h), None, fmt), h, fmt)


def test_tensor_scales_far_from_one(ops):
    """The division-free path gives way to divisions where a reciprocal would over- or underflow."""
    g = torch.Generator().manual_seed(4)
    base = torch.randn(4, 64, generator=g)
    for e, ge in ((-100, -108), (110, 104), (-30, 90), (100, -120), (0, -126), (0, 120)):
        x = base * 2.0 ** e
        t = ops.quant_fp4(cu(x), torch.tensor([2.0 ** ge], device="cuda"), "nvfp4")
        assert_quantized(t, x, "nvfp4", 2.0 ** ge)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_takes_rows_apart_and_leaves_absent_rows_alone(ops, fmt):
    x = inputs(70, 192, torch.bfloat16, 3)
    wide = torch.full((70, 448), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 128:320] = x.cuda()
    out = ops.Fp4Tensor.empty(70, 192, fmt)
    out.scales.fill_(0xAB)
    ops.quant_fp4(wide[:, 128:320], out=out)
    check_status()
    assert_quantized(out, x, fmt)
    wide[:, 136:328] = x.cuda()
    assert_quantized(ops.quant_fp4(wide[:, 136:328], None, fmt), x, fmt)      # rows on 16 bytes, not on 32
    odd = torch.empty(70, 200, dtype=torch.bfloat16, device="cuda")[:, :192]  # a pitch of 400 bytes
    odd.copy_(x)
    assert_quantized(ops.quant_fp4(odd, None, fmt), x, fmt)
    blocks = 192 // fp4.GROUP[fmt]
    rest = torch.ones(out.scales.numel(), dtype=torch.bool)
    rest[fp4.scale_offsets(70, (blocks + 3) // 4 * 4).flatten()] = False
    assert bool((out.scales.cpu()[rest] == 0xAB).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weight_quantize(ops, fmt, dtype):
    g = torch.Generator().manual_seed(9)
    w = (torch.randn(200, 352, generator=g) * 0.02).to(dtype)
    w[3, 7] = float("inf")
    for scale in (1.0, 0.0):
        t = ops.weight_quant_fp4(cu(w * scale if scale else torch.zeros_like(w)), fmt)
        check_status()
        ref = w if scale else torch.zeros_like(w)
        gs = fp4.tensor_scale(ref)
        if fmt == "nvfp4":
            assert float(t.tensor_scale) == gs
        assert_quantized(t, ref, fmt, gs or 1.0)


# ----------------------------------------------------------------------------- the product
def problem(m, n, k, fmt, dtype, seed, bias=True, residual=False, g=(0.5, 2.0 ** -7)):
    gen = torch.Generator().manual_seed(seed)
    xc, xs = fp4.encode(torch.randn(m, k, generator=gen) * 2, fmt, g[0])
    wc, ws = fp4.encode(torch.randn(n, k, generator=gen) * 0.05, fmt, g[1])
    b = torch.randn(n, generator=gen).to(dtype) if bias else None
    r = torch.randn(m, n, generator=gen).to(dtype) if residual else None
    return (xc, xs, g[0] if fmt == "nvfp4" else 1.0), (wc, ws, g[1] if fmt == "nvfp4" else 1.0), b, r


def to_device(ops, part, fmt, fill=0xAB):
    codes, s, g = part
    rows, k = codes.shape
    blocks = s.shape[1]
    t = ops.Fp4Tensor.empty(rows, k, fmt, torch.tensor([g], device="cuda") if fmt == "nvfp4" else None)
    t.codes.copy_(fp4.pack(codes))
    sb = torch.full((t.scales.numel(),), fill, dtype=torch.uint8)     # scales of absent rows: anything
    pad = fp4.scale_offsets(rows, (blocks + 3) // 4 * 4)
    sb[pad.flatten()] = 0
    sb[pad[:, :blocks].flatten()] = s.flatten()
    t.scales.copy_(sb)
    return t


def assert_product(got, x, w, fmt, bias=None, residual=None, beta=1.0, gelu=False):
    """Against 64 bits.  The products of two FP4 values and their scales are exact; the sum of K of them runs through the fp32 accumulator in
    K / 64 instructions, each of which may lose an ulp of what it adds up (2^-23 of the sum of magnitudes; 2 more for the sum inside it);
    the epilogue adds at most four fp32 roundings, tanh.approx has a relative error of 2^-10.9 (half of which reaches the result), and the
    result is rounded to its type: half a step."""
    xv, wv = fp4.decode(*x[:2], fmt, x[2]), fp4.decode(*w[:2], fmt, w[2])
    y, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    k = xv.shape[1]
    if residual is not None:
        y, mag = y + beta * residual.double(), mag + abs(beta) * residual.double().abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    tol = ((k + 63) // 64 + 2 + 4) * 2.0 ** -23 * mag
    if gelu:
        tol = 1.13 * tol + 0.5 * y.abs() * 2.0 ** -10.9 + 2.0 ** -21 * y.abs()
        y = fp4.gelu_tanh(y)
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * half * 2
    tol = tol * (1 + half) + half * y.abs() + tiny
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), "off by %g of the tolerance at %s" % (float((err / tol).max()), (err / tol).argmax())


SHAPES = [(1, 8, 32), (5, 24, 64), (128, 128, 256), (130, 200, 288), (257, 129, 512), (300, 520, 1056), (64, 100, 3200)]


@pytest.mark.parametrize("code", [1281, 2562])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_every_tile(ops, tile, code, fmt, m, n, k):
    tile(code)
    x, w, b, _ = problem(m, n, k, fmt, torch.bfloat16, m + n + k)
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp4(to_device(ops, w, fmt), to_device(ops, x, fmt), y, cu(b))
    check_status()
    assert_product(y, x, w, fmt, b)


@pytest.mark.parametrize("code", [0, 1281, 2562])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gelu,bias,residual", [(True, True, False), (False, False, True), (True, True, True)])
@pytest.mark.parametrize("m,n", [(3, 72), (140, 300), (260, 131)])
def test_epilogues_and_types(ops, tile, code, dtype, gelu, bias, residual, m, n):
    tile(code)
    x, w, b, r = problem(m, n, 320, "nvfp4", dtype, 5, bias, residual)
    y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    ops.gemm_fp4(to_device(ops, w, "nvfp4"), to_device(ops, x, "nvfp4"), y, cu(b), cu(r), 0.75, gelu)
    check_status()
    assert_product(y, x, w, "nvfp4", b, r, 0.75, gelu)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_of_every_row_and_block_reach_their_values(ops, tile, fmt):
    """One value in each (row, block), all scales different: a scale taken from another row or block shows."""
    for code, m, n, k in ((1281, 128, 128, 512), (2562, 256, 256, 512), (0, 16, 128, 512)):
        tile(code)
        blocks = k // fp4.GROUP[fmt]
        xc = torch.zeros(m, k, dtype=torch.uint8)
        wc = torch.zeros(n, k, dtype=torch.uint8)
        xc[:, ::fp4.GROUP[fmt]] = 2
        wc[:, ::fp4.GROUP[fmt]] = 2
        i, j, b = torch.arange(m)[:, None], torch.arange(n)[:, None], torch.arange(blocks)[None]
        xs = (48 + (i * 7 + b * 3) % 23 + (70 if fmt == "mxfp4" else 0)).to(torch.uint8)
        ws = (48 + (j * 5 + b * 11) % 19 + (70 if fmt == "mxfp4" else 0)).to(torch.uint8)
        x, w = (xc, xs, 1.0), (wc, ws, 1.0)
        y = torch.empty(m, n, dtype=torch.float32, device="cuda")
        ops.gemm_fp4(to_device(ops, w, fmt), to_device(ops, x, fmt), y)
        check_status()
        assert_product(y, x, w, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 129, 96), (2, 300, 1312), (7, 136, 2048), (16, 520, 4096), (11, 4224, 576)])
def test_few_rows(ops, tile, fmt, dtype, m, n, k):
    tile(16)
    x, w, b, r = problem(m, n, k, fmt, dtype, m * n + k, True, True)
    for gelu in (False, True):
        y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        ops.gemm_fp4(to_device(ops, w, fmt, 0xFF), to_device(ops, x, fmt, 0xFF), y, cu(b), cu(r), -0.5, gelu)
        check_status()
        assert_product(y, x, w, fmt, b, r, -0.5, gelu)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("n,k", [(264, 4096), (4224, 4096), (4352, 4096), (9088, 2048), (9216, 2048), (18944, 1024), (19072, 1024), (130, 32)])
def test_few_rows_with_every_split_of_k(ops, fmt, m, n, k):
    """One, two, four and eight CTAs along k, and both sides of the tile counts at which fewer are taken.  Codes of 0, 1, -1 and 2 under scales of
    one make every partial sum an integer below 2^24: exact in any order."""
    g = torch.Generator(device="cuda").manual_seed(n + m)
    codes = torch.tensor([0, 2, 10, 4], dtype=torch.uint8, device="cuda")
    values = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.float64, device="cuda")
    parts = []
    for rows in (n, m):
        i = torch.randint(0, 4, (rows, k), generator=g, device="cuda")
        t = ops.Fp4Tensor.empty(rows, k, fmt)
        c = codes[i]
        t.codes.copy_(c[:, 0::2] | (c[:, 1::2] << 4))
        t.scales.fill_(0x38 if fmt == "nvfp4" else 127)
        parts.append((t, values[i]))
    y = torch.empty(m, n, dtype=torch.float32, device="cuda")
    ops.gemm_fp4(parts[0][0], parts[1][0], y)
    check_status()
    assert torch.equal(y.double(), parts[1][1] @ parts[0][1].t())


def test_large_product_is_exact_and_the_same_with_every_tile(ops, tile):
    """All rounds of a persistent grid, both accumulator buffers, the tile order's last band: integer operands again."""
    g = torch.Generator(device="cuda").manual_seed(2)
    m, n, k = 2309, 4808, 1120
    codes = torch.tensor([0, 2, 10, 4], dtype=torch.uint8, device="cuda")
    values = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.float64, device="cuda")
    for fmt in FORMATS:
        parts = []
        for rows in (n, m):
            i = torch.randint(0, 4, (rows, k), generator=g, device="cuda")
            t = ops.Fp4Tensor.empty(rows, k, fmt)
            t.codes.copy_(codes[i][:, 0::2] | (codes[i][:, 1::2] << 4))
            t.scales.zero_()
            blocks = k // fp4.GROUP[fmt]
            t.scales[fp4.scale_offsets(rows, blocks).flatten().cuda()] = 0x38 if fmt == "nvfp4" else 127
            parts.append((t, values[i]))
        want = parts[1][1] @ parts[0][1].t()
        for code in (0, 1281, 2562):
            tile(code)
            y = torch.full((m, n), float("nan"), dtype=torch.float32, device="cuda")
            ops.gemm_fp4(parts[0][0], parts[1][0], y)
            check_status()
            assert torch.equal(y.double(), want), (fmt, code)
            h = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
            ops.gemm_fp4(parts[0][0], parts[1][0], h)
            assert torch.equal(h, want.bfloat16()), (fmt, code)


@pytest.mark.parametrize("code", [1281, 2562])
@pytest.mark.parametrize("m,n", [(60001, 32), (25000, 224), (30000, 72)])
def test_many_tiles_whose_last_columns_fill_one_store_box(ops, tile, code, m, n):
    """Tile after tile in which a warp stores an odd number of 32-column pieces, with a short K: integer operands, exact."""
    tile(code)
    g = torch.Generator(device="cuda").manual_seed(n)
    codes = torch.tensor([0, 2, 10, 4], dtype=torch.uint8, device="cuda")
    values = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.float32, device="cuda")
    parts = []
    for rows in (n, m):
        i = torch.randint(0, 4, (rows, 32), generator=g, device="cuda")
        t = ops.Fp4Tensor.empty(rows, 32)
        t.codes.copy_(codes[i][:, 0::2] | (codes[i][:, 1::2] << 4))
        t.scales.zero_()
        t.scales[fp4.scale_offsets(rows, 2).flatten().cuda()] = 0x38
        parts.append((t, values[i]))
    want = (parts[1][1].double() @ parts[0][1].double().t()).bfloat16()
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    r = torch.full((m, n), 3.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        ops.gemm_fp4(parts[0][0], parts[1][0], y)
        check_status()
        assert torch.equal(y, want)
    ops.gemm_fp4(parts[0][0], parts[1][0], r, residual=r, beta=2.0)   # |sum| + 6 <= 134: exact
    check_status()
    assert torch.equal(r, want + 6.0)


@pytest.mark.parametrize("code", [0, 1281, 2562])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(7, 72), (300, 264), (200, 131)])
def test_result_in_the_residuals_place(ops, tile, code, dtype, m, n):
    tile(code)
    x, w, b, r = problem(m, n, 320, "mxfp4", dtype, 21, True, True)
    y = cu(r).clone()
    ops.gemm_fp4(to_device(ops, w, "mxfp4"), to_device(ops, x, "mxfp4"), y, cu(b), y, -1.25)
    check_status()
    assert_product(y, x, w, "mxfp4", b, r, -1.25)


@pytest.mark.parametrize("stalled", [0, 1])
def test_few_rows_wait_that_runs_out_stores_nothing(ops, stalled):
    """One CTA of each cluster loads nothing (a debug switch, no fault): its wait ends with the status, and no CTA of the cluster stores."""
    from lyradiff_b200 import _lib
    lib = _lib.lib()
    x, w, _, _ = problem(4, 512, 2048, "nvfp4", torch.bfloat16, 8)
    X, W = to_device(ops, x, "nvfp4"), to_device(ops, w, "nvfp4")
    good, out = (torch.full((4, 512), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.gemm_fp4(W, X, good)
    check_status()
    assert lib.lyraq_debug_fp4_skinny_wait_test(stalled, 50) == 0
    try:
        ops.gemm_fp4(W, X, out)
        torch.cuda.synchronize()
        status, detail = ops.last_status()
    finally:
        assert lib.lyraq_debug_fp4_skinny_wait_test(-1, 0) == 0
    assert status == 4 and 0x6000 <= detail < 0x7000, (status, hex(detail))
    assert bool((out == 7.0).all())
    ops.gemm_fp4(W, X, out)
    check_status()
    assert torch.equal(out, good)


def test_blocks_of_nan_reach_their_outputs_and_no_others(ops):
    x = torch.randn(40, 256, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[7, 33] = float("nan")
    w = torch.randn(24, 256, generator=torch.Generator().manual_seed(2)).bfloat16()
    w[5, 100] = float("inf")
    for fmt in FORMATS:
        for rows in (40, 9):
            y = torch.zeros(rows, 24, dtype=torch.float32, device="cuda")
            ops.gemm_fp4(ops.weight_quant_fp4(cu(w), fmt), ops.quant_fp4(cu(x[:rows]), None, fmt), y)
            check_status()
            bad = torch.isnan(y).cpu()
            want = torch.zeros(rows, 24, dtype=torch.bool)
            want[7], want[:, 5] = True, True
            assert torch.equal(bad, want)


# ----------------------------------------------------------------------------- the layer
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead", [(1,), (2, 9), (3, 70)])
def test_layer_is_quantize_then_product(ops, fmt, dtype, lead):
    from lyradiff_b200 import layers
    g = torch.Generator().manual_seed(7)
    w, b = (torch.randn(160, 352, generator=g) * 0.05).to(dtype), torch.randn(160, generator=g).to(dtype)
    x, r = torch.randn(*lead, 352, generator=g).to(dtype), torch.randn(*lead, 160, generator=g).to(dtype)
    layer = layers.Fp4Linear(cu(w), cu(b), torch.tensor(0.011), gelu=True, fmt=fmt)
    if fmt == "nvfp4":
        assert float(layer.input_scale) == 2.0 ** -6 and layer.weight.tensor_scale is not None
    got = layer.forward(cu(x), residual=cu(r), beta=0.5)
    check_status()
    assert got.shape == (*lead, 160)
    rows = got.numel() // 160
    gx, gw = (2.0 ** -6, fp4.tensor_scale(w)) if fmt == "nvfp4" else (1.0, 1.0)
    assert_product(got.reshape(rows, 160), (*fp4.encode(x.reshape(rows, 352), fmt, gx), gx), (*fp4.encode(w, fmt, gw), gw), fmt, b, r.reshape(rows, 160), 0.5, True)
    q = layer.empty_input(rows)
    ops.quant_fp4(cu(x).reshape(rows, 352), out=q)
    again = layer.forward_quantized(q, dtype, cu(r), 0.5)
    assert torch.equal(again, got.reshape(rows, 160))
    with pytest.raises(ValueError):
        layer.forward(cu(x)[..., :320])
    with pytest.raises(ValueError):
        layer.forward(cu(x), residual=cu(r).float())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(136, 32), (520, 96), (264, 1312), (4224, 2048), (72, 12320), (9216, 3072)])
def test_few_rows_quantized_on_their_way(ops, tile, fmt, dtype, n, k):
    """The layer's one launch gives the bits of the quantizer and the product in turn, for every number of rows and way of dealing them to warps."""
    from lyradiff_b200 import layers
    g = torch.Generator().manual_seed(n + k)
    w, b = (torch.randn(n, k, generator=g) * 0.05).to(dtype), torch.randn(n, generator=g).to(dtype)
    layer = layers.Fp4Linear(cu(w), cu(b), torch.tensor(2.0 ** -7), fmt=fmt)
    wide = torch.full((16, k + 40), float("nan"), dtype=dtype, device="cuda")
    wide[:, :k] = torch.randn(16, k, generator=g).to(dtype).cuda()
    wide[3, k // 2] = float("inf")
    for m in (1, 2, 3, 4, 5, 8, 9, 16):
        x = wide[:m, :k]
        tile(1281)          # two launches
        q = layer.empty_input(m)
        ops.quant_fp4(x, out=q)
        tile(16)
        want = layer.forward_quantized(q, dtype)
        got = layer.forward(x)
        check_status()
        assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0)) and bool(torch.isnan(got).any()) == (m > 3)
        assert torch.equal(torch.isnan(got), torch.isnan(want))


def test_few_rows_with_the_result_in_their_place(ops):
    from lyradiff_b200 import layers
    g = torch.Generator().manual_seed(5)
    w, x = (torch.randn(2048, 2048, generator=g) * 0.05).bfloat16(), torch.randn(9, 2048, generator=g).bfloat16()
    layer = layers.Fp4Linear(cu(w), None, torch.tensor(2.0 ** -7))
    y = cu(x).clone()
    assert torch.equal(layer.forward(y, out=y), layer.forward(cu(x)))
    check_status()


@pytest.mark.parametrize("stalled", [0, 1])
def test_few_rows_quantized_on_their_way_wait_that_runs_out_stores_nothing(ops, stalled):
    from lyradiff_b200 import _lib, layers
    g = torch.Generator().manual_seed(6)
    layer = layers.Fp4Linear(cu((torch.randn(512, 2048, generator=g) * 0.05).bfloat16()), None, torch.tensor(2.0 ** -7))
    x, out = cu(torch.randn(4, 2048, generator=g).bfloat16()), torch.full((4, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    good = layer.forward(x)
    check_status()
    assert _lib.lib().lyraq_debug_fp4_skinny_wait_test(stalled, 50) == 0
    try:
        layer.forward(x, out=out)
        torch.cuda.synchronize()
        status, detail = ops.last_status()
    finally:
        assert _lib.lib().lyraq_debug_fp4_skinny_wait_test(-1, 0) == 0
    assert status == 4 and 0x6000 <= detail < 0x7000, (status, hex(detail))
    assert bool((out == 7.0).all())
    assert torch.equal(layer.forward(x, out=out), good)
    check_status()


def test_layer_in_two_captured_graphs_and_on_two_streams(ops):
    """Nothing is shared between calls: graphs captured from one layer replay at the same time and with new inputs."""
    from lyradiff_b200 import layers
    g = torch.Generator().manual_seed(8)
    layer = layers.Fp4Linear(cu((torch.randn(512, 1024, generator=g) * 0.05).bfloat16()), None, torch.tensor([0.01]))
    xs = [torch.randn(m, 1024, generator=g).bfloat16().cuda() for m in (3, 200)]
    graphs, outs = [], []
    side = [torch.cuda.Stream() for _ in xs]
    for x, s in zip(xs, side):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer.forward(x)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(layer.forward(x))
        graphs.append(gr)
    for x in xs:
        x.copy_(torch.randn(x.shape, generator=g))
    want = [layer.forward(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    check_status()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
