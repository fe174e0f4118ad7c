"""GPU tests of FP8 with a scale for each block of 128 against the 64-bit restatement in oracle/fp8_block.py."""

import pytest
import torch

from oracle import e4m3, fp8_block
from tests.util import check_status, cu

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    from lyradiff_b200 import ops as _ops
    return _ops


@pytest.fixture
def tile():
    from lyradiff_b200 import _lib
    yield lambda code: _lib.check(_lib.lib().lyraq_debug_force_fp8_block_tile(code), "lyraq_debug_force_fp8_block_tile")
    _lib.lib().lyraq_debug_force_fp8_block_tile(0)


def values(rows, k, dtype, seed):
    """Blocks of different size, quotients on ties of e4m3, zeros, a block of zeros, tiny and huge blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp2(3 * torch.randn(rows, (k + 127) // 128, generator=g)).repeat_interleave(128, 1)[:, :k]
    x[::3, :16] = torch.tensor([448.0, 17.0, -19.0, 26.0, 27.0, 2.0 ** -9, 3 * 2.0 ** -10, 2.0 ** -10, 0.0, -1.0625, 1.1875, 232.0, -248.0, 7.25, 6.75, 440.0])
    x[1::7] = 0
    if dtype != torch.float16:
        x[2::9] *= 2.0 ** -110
        x[4::9] *= 2.0 ** 100
    return x.clamp(-3e38, 3e38).to(dtype) if dtype != torch.float16 else x.clamp(-60000, 60000).to(dtype)


def assert_quantized(codes, s, x, block_rows=1):
    want, ws = fp8_block.encode(x, block_rows)
    got, gs = codes.cpu(), s.cpu()
    assert torch.equal(gs.isnan(), ws.isnan()) and torch.equal(gs.nan_to_num(), ws.nan_to_num())
    sign = lambda c: torch.where(c == 128, 0, c.int())   # noqa: E731
    assert torch.equal(sign(got), sign(want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 144), (31, 256), (130, 1040), (300, 4112), (5, 12304)])
def test_quantize_is_exact(ops, dtype, rows, k):
    x = values(rows, k, dtype, rows + k)
    assert_quantized(*ops.quant_fp8_block(cu(x)), x)
    check_status()


def test_quantize_of_views_into_scales_of_any_steps(ops):
    x = values(70, 400, torch.bfloat16, 1)
    for pitch, at in ((1024, 128), (1024, 136), (408, 0)):      # rows on 32 bytes, on 16, a pitch that is a multiple of 16 only
        wide = torch.zeros(70, pitch, dtype=torch.bfloat16, device="cuda")
        wide[:, at:at + 400] = x.cuda()
        assert_quantized(*ops.quant_fp8_block(wide[:, at:at + 400]), x)
    s = torch.full((75, 9), 7.0, device="cuda")
    codes, view = ops.quant_fp8_block(cu(x), scales=s[2:72, 1:8:2])
    assert_quantized(codes, view, x)
    s[2:72, 1:8:2] = 7.0
    assert bool((s == 7.0).all())                               # nothing beside them was written
    check_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_that_hold_no_number(ops, dtype):
    x = values(9, 400, dtype, 3)
    x[2, 130], x[4, 399], x[5, 0], x[5, 1] = float("inf"), float("nan"), float("-inf"), float("nan")
    codes, s = ops.quant_fp8_block(cu(x))
    assert_quantized(codes, s, x)
    w = values(200, 400, dtype, 4)
    w[150, 300] = float("nan")
    codes, s = ops.weight_quant_fp8_block(cu(w))
    assert_quantized(codes, s, w, 128)
    check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 272), (300, 1040)])
def test_weight_quantize_is_exact(ops, dtype, n, k):
    w = values(n, k, dtype, n)
    assert_quantized(*ops.weight_quant_fp8_block(cu(w)), w, 128)
    check_status()


# ----------------------------------------------------------------------------- the product
def problem(m, n, k, dtype, seed, bias=True, residual=False):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp2(2 * torch.randn(m, (k + 127) // 128, generator=g)).repeat_interleave(128, 1)[:, :k]
    x = fp8_block.encode(torch.randn(m, k, generator=g) * size)
    wsize = torch.exp2(2 * torch.randn((n + 127) // 128, (k + 127) // 128, generator=g)).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    w = fp8_block.encode(torch.randn(n, k, generator=g) * 0.05 * wsize, 128)
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    return x, w, b, r


def assert_product(got, x, w, bias=None, residual=None, beta=1.0, gelu=False):
    """Against 64 bits.  Products of two e4m3 numbers are exact; the sum of a block runs through the fp32 accumulator in at most four
    instructions, each of which may lose an ulp of what it adds up (2^-23 of the sum of magnitudes; 2 more for the sum inside it); its factor is rounded
    once (2^-24) and its addition to the sum of the blocks once (2^-24 of all magnitudes, for each block; a few-row kernel adds the parts of up to 16
    warps as well); the epilogue adds at most four fp32 roundings, tanh.approx has a relative error of 2^-10.9 (half of which reaches the result), and
    the result is rounded to its type: half a step."""
    xv, wv = fp8_block.decode(*x), fp8_block.decode(*w, 128)
    y, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    k = xv.shape[1]
    if residual is not None:
        y, mag = y + beta * residual.double(), mag + abs(beta) * residual.double().abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    tol = ((4 + 2) * 2.0 ** -23 + ((k + 127) // 128 + 1 + 16 + 4) * 2.0 ** -24) * mag
    if gelu:
        tol = 1.13 * tol + 0.5 * y.abs() * 2.0 ** -10.9 + 2.0 ** -21 * y.abs()
        y = fp8_block.gelu_tanh(y)
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * half * 2
    tol = tol * (1 + half) + half * y.abs() + tiny
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), "off by %g of the tolerance at %s" % (float((err / tol).max()), (err / tol).argmax())


SHAPES = [(1, 8, 16), (5, 24, 64), (128, 128, 256), (130, 200, 304), (257, 129, 512), (300, 520, 1040), (64, 100, 3200), (2, 260, 1664), (16, 40, 128)]


@pytest.mark.parametrize("code", [0, 16, 1281, 2562])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_every_kernel(ops, tile, code, m, n, k):
    tile(code)
    x, w, b, _ = problem(m, n, k, torch.bfloat16, m + n + k)
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_block(cu(w[0]), cu(w[1]), cu(x[0]), cu(x[1]), y, cu(b))
    check_status()
    assert_product(y, x, w, b)


@pytest.mark.parametrize("code", [0, 16, 1281, 2562])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gelu,bias,residual", [(True, True, False), (False, False, True), (True, True, True)])
@pytest.mark.parametrize("m,n", [(3, 72), (140, 300), (260, 131)])
def test_epilogues_and_types(ops, tile, code, dtype, gelu, bias, residual, m, n):
    tile(code)
    x, w, b, r = problem(m, n, 336, dtype, 5, bias, residual)
    y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    ops.gemm_fp8_block(cu(w[0]), cu(w[1]), cu(x[0]), cu(x[1]), y, cu(b), cu(r), 0.75, gelu)
    check_status()
    assert_product(y, x, w, b, r, 0.75, gelu)
    z = cu(r).clone() if residual else None
    if residual:                                               # the result in the residual's place
        ops.gemm_fp8_block(cu(w[0]), cu(w[1]), cu(x[0]), cu(x[1]), z, cu(b), z, 0.75, gelu)
        check_status()
        assert torch.equal(z, y)


@pytest.mark.parametrize("code,m", [(16, 1), (16, 8), (16, 9), (16, 16), (1281, 300), (2562, 600)])
def test_scales_of_every_row_and_block_reach_their_values(ops, tile, code, m):
    """One value in each block, every scale another power of two or three times one: a scale of another row or block shows, and so does a lost block."""
    tile(code)
    n, k = 400, 1040
    kb = (k + 127) // 128
    xc, wc = torch.zeros(m, k, dtype=torch.uint8), torch.zeros(n, k, dtype=torch.uint8)
    xc[:, 5::128] = 0x38
    wc[:, 5::128] = 0x38
    i, b = torch.arange(m)[:, None], torch.arange(kb)[None]
    xs = torch.exp2(((i * 7 + b * 3) % 11).float()) * (1 + 2 * ((i + b) % 2))
    ws = torch.exp2(((torch.arange((n + 127) // 128)[:, None] * 5 + b * 2) % 7).float())
    want = (xs.double() @ fp8_block.spread(ws, n, k, 128)[:, 5::128].double().t()).float()      # integers below 2^24
    for strided in (False, True):
        s = cu(xs)
        if strided:                                             # rows of a block beside each other, with a gap
            s = torch.zeros(kb, m + 3, device="cuda")
            s[:, :m] = cu(xs).t()
            s = s.t()[:m]
        y = torch.empty(m, n, dtype=torch.float32, device="cuda")
        ops.gemm_fp8_block(cu(wc), cu(ws), cu(xc), s, y)
        check_status()
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("code,m,n,k", [(0, 2309, 4808, 1136), (1281, 2309, 4808, 1136), (2562, 2309, 4808, 1136), (16, 16, 20000, 1040), (16, 7, 4104, 9232),
                                        (0, 3, 33, 40000), (16, 1, 5000, 13824)])
def test_large_products_are_exact(ops, tile, code, m, n, k):
    """All rounds of a persistent grid: integer operands and scales, exact in any order."""
    tile(code)
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.tensor([0, 0x38, 0xB8, 0x40], dtype=torch.uint8, device="cuda")
    value = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.float64, device="cuda")
    i, j = (torch.randint(0, 4, (rows, k), generator=g, device="cuda") for rows in (m, n))
    kb = (k + 127) // 128
    xs = torch.randint(1, 3, (m, kb), generator=g, device="cuda").float()
    ws = torch.randint(1, 3, ((n + 127) // 128, kb), generator=g, device="cuda").float()
    want = (value[i] * fp8_block.spread(xs, m, k, 1)) @ (value[j] * fp8_block.spread(ws, n, k, 128)).t()
    for dtype in (torch.float32, torch.bfloat16):
        y = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        ops.gemm_fp8_block(table[j], ws, table[i], xs, y)
        check_status()
        assert torch.equal(y, want.to(dtype))


SPLIT = [1282, 1284, 1288]      # CTAs along K


@pytest.mark.parametrize("code", SPLIT)
@pytest.mark.parametrize("m,n,k", SHAPES + [(20, 136, 144), (77, 1300, 5136)])
def test_product_with_k_over_a_cluster(ops, tile, code, m, n, k):
    test_product_of_every_kernel(ops, tile, code, m, n, k)


@pytest.mark.parametrize("code", SPLIT)
@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
@pytest.mark.parametrize("gelu,bias,residual", [(True, True, False), (True, True, True)])
@pytest.mark.parametrize("m,n", [(33, 72), (140, 300), (260, 131)])
def test_epilogues_with_k_over_a_cluster(ops, tile, code, dtype, gelu, bias, residual, m, n):
    test_epilogues_and_types(ops, tile, code, dtype, gelu, bias, residual, m, n)


@pytest.mark.parametrize("code,m", [(code, m) for code in SPLIT for m in (17, 300)])
def test_scales_with_k_over_a_cluster(ops, tile, code, m):
    test_scales_of_every_row_and_block_reach_their_values(ops, tile, code, m)


@pytest.mark.parametrize("code,m,n,k", [(0, 64, 5120, 13824), (0, 17, 33, 40000), (1282, 700, 3000, 1136), (1284, 300, 2100, 9232), (1288, 129, 1111, 13824)])
def test_large_products_with_k_over_a_cluster_are_exact(ops, tile, code, m, n, k):
    """More clusters than run at once, and the automatic choice."""
    test_large_products_are_exact(ops, tile, code, m, n, k)


def test_k_over_a_cluster_gives_the_same_bits_again_and_captured(ops, tile):
    x, w, b, r = (cu(t) if torch.is_tensor(t) else tuple(cu(u) for u in t) for t in problem(40, 300, 9232, torch.bfloat16, 11, True, True))
    first = torch.empty(40, 300, dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_block(*w, *x, first, b, r)
    check_status()
    again = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_fp8_block(*w, *x, again, b, r)
    for _ in range(3):
        again.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, first)


def test_a_scale_that_is_no_number_spoils_its_rows_and_no_others(ops, tile):
    for code, m in ((0, 3), (1281, 200), (2562, 300)):
        tile(code)
        x, w, _, _ = problem(m, 300, 400, torch.bfloat16, 9, bias=False)
        x[1][1, 2] = float("nan")
        w[1][2, 0] = float("nan")
        y = ops.gemm_fp8_block(cu(w[0]), cu(w[1]), cu(x[0]), cu(x[1]), torch.bfloat16)
        check_status()
        bad = torch.zeros(m, 300, dtype=torch.bool)
        bad[1], bad[:, 256:] = True, True
        assert torch.equal(y.isnan().cpu(), bad)


# ----------------------------------------------------------------------------- the layer
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 5, 16, 33, 150])
def test_layer_is_quantize_and_product(ops, dtype, m):
    from lyradiff_b200.layers import Fp8BlockLinear
    g = torch.Generator().manual_seed(m)
    w, b = (torch.randn(264, 1552, generator=g) * 0.02).to(dtype), torch.randn(264, generator=g).to(dtype)
    x = values(m, 1552, dtype, m).clamp(-1000, 1000)
    r = torch.randn(m, 264, generator=g).to(dtype)
    layer = Fp8BlockLinear.from_float(cu(w), cu(b), gelu=True)
    qx, qw = fp8_block.encode(x), fp8_block.encode(w, 128)
    y = layer.forward(cu(x), residual=cu(r), beta=0.5)
    check_status()
    assert_product(y, qx, qw, b, r, 0.5, True)
    three = layer.forward(cu(x)[None], residual=cu(r)[None], beta=0.5)
    assert three.shape == (1, m, 264) and torch.equal(three[0], y)
    wide = torch.zeros(m, 1600, dtype=dtype, device="cuda")
    wide[:, 16:1568] = cu(x)
    assert torch.equal(layer.forward(wide[:, 16:1568], residual=cu(r), beta=0.5), y)
    out = torch.empty(m, 264, dtype=dtype, device="cuda")
    assert layer.forward(cu(x), residual=cu(r), beta=0.5, out=out) is out and torch.equal(out, y)


def test_layer_result_in_its_inputs_place_and_empty_calls(ops):
    from lyradiff_b200.layers import Fp8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = Fp8BlockLinear.from_float(torch.randn(512, 512, generator=g, device="cuda").bfloat16())
    for m in (1, 7, 200):
        x = torch.randn(m, 512, generator=g, device="cuda").bfloat16()
        want = layer.forward(x)
        assert layer.forward(x, out=x) is x and torch.equal(x, want)
    assert layer.forward(torch.empty(0, 512, dtype=torch.bfloat16, device="cuda")).shape == (0, 512)
    with pytest.raises(ValueError):
        layer.forward(torch.empty(3, 500, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        layer.forward(torch.empty(3, 512, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        layer.forward(torch.empty(3, 512, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        Fp8BlockLinear(layer.codes, layer.scales[:3])
    with pytest.raises(ValueError):
        ops.gemm_fp8_block(layer.codes, layer.scales, layer.codes[:4], layer.scales[:3], torch.bfloat16)


def test_layer_on_streams_and_in_graphs(ops):
    from lyradiff_b200.layers import Fp8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = Fp8BlockLinear.from_float(torch.randn(640, 768, generator=g, device="cuda").bfloat16() * 0.03)
    xs = [torch.randn(m, 768, generator=g, device="cuda").bfloat16() for m in (1, 300, 16, 129)]
    want = [layer.forward(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(5):
        for s, x, o in zip(streams, xs, got):
            with torch.cuda.stream(s):
                o.append(layer.forward(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for o, w in zip(got, want) for y in o)
    graphs = []
    for x in xs:                                                # two graphs and more, replayed in any order
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward(x)
        graphs.append((graph, x, y))
    for step in range(3):
        for graph, x, _ in graphs:
            x.mul_(-1)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, y), w in zip(graphs, want):
            assert torch.equal(y, w if step % 2 else -w)


def test_encode_matches_torch(ops):
    """The conversion itself, at every tie of e4m3 and next to it."""
    v = torch.arange(127, dtype=torch.uint8)
    table = torch.from_numpy(e4m3.decode(v.numpy()).copy())
    mid = (table[1:] + table[:-1]) / 2
    q = torch.cat([mid, torch.nextafter(mid, mid * 2), torch.nextafter(mid, mid * 0)])
    q = torch.cat([q, torch.full((-q.numel() % 128,), 448.0)])
    x = q.reshape(-1, 128).clone()
    x[:, -1] = 448.0                                            # the scale of every block is one
    codes, s = ops.quant_fp8_block(cu(x))
    assert bool((s == 1).all())
    assert torch.equal(codes.cpu(), x.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("m", [1, 3, 8, 16])
@pytest.mark.parametrize("n,k", [(264, 4096), (4224, 2560), (9088, 1024), (9216, 2048), (18944, 512), (19072, 1152), (130, 16), (33000, 400), (200, 33008)])
def test_few_rows_with_every_split_of_k(ops, tile, m, n, k):
    """One, two, four and eight CTAs along K, both sides of the tile counts at which fewer are taken, more K blocks than tensor memory has buffers: integers, exact."""
    tile(16)
    g = torch.Generator(device="cuda").manual_seed(n + m)
    table = torch.tensor([0, 0x38, 0xB8, 0x40], dtype=torch.uint8, device="cuda")
    value = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.float64, device="cuda")
    i, j = (torch.randint(0, 4, (rows, k), generator=g, device="cuda") for rows in (m, n))
    xs, ws = torch.ones(m, (k + 127) // 128, device="cuda"), torch.ones((n + 127) // 128, (k + 127) // 128, device="cuda")
    y = torch.full((m, n), float("nan"), dtype=torch.float32, device="cuda")
    ops.gemm_fp8_block(table[j], ws, table[i], xs, y)
    check_status()
    assert torch.equal(y.double(), value[i] @ value[j].t())


@pytest.mark.parametrize("m", [1, 2, 7, 16])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_quantized_in_the_product_are_the_same(ops, tile, m, dtype):
    """The few-row kernel's own quantize against the quantizer and the product on its codes: the same bits."""
    from lyradiff_b200.layers import Fp8BlockLinear
    g = torch.Generator().manual_seed(m)
    for n, k in ((200, 1040), (1300, 336), (264, 6416)):
        x = values(m, k, dtype, m + k).clamp(-1e4, 1e4)
        layer = Fp8BlockLinear.from_float(cu((torch.randn(n, k, generator=g) * 0.02).to(dtype)))
        tile(16)
        y = layer.forward(cu(x))
        codes, s = ops.quant_fp8_block(cu(x))
        assert torch.equal(ops.gemm_fp8_block(layer.codes, layer.scales, codes, s, dtype), y)
        tile(0)
        assert torch.equal(layer.forward(cu(x)), y) or m > 6 and k <= 7 * 128
        check_status()


def test_a_wait_that_runs_out_is_reported(ops):
    from lyradiff_b200 import _lib
    from lyradiff_b200.layers import Fp8BlockLinear
    layer = Fp8BlockLinear.from_float(torch.randn(640, 4096, device="cuda").bfloat16())
    x = torch.randn(3, 4096, device="cuda").bfloat16()
    want = layer.forward(x)
    check_status()
    _lib.check(_lib.lib().lyraq_debug_fp8_block_rows_wait_test(1, 200), "hook")
    try:
        y = torch.zeros(3, 640, dtype=torch.bfloat16, device="cuda")
        layer.forward(x, out=y)
        from lyradiff_b200 import ops as _ops
        status, detail = _ops.last_status()
        assert status == 4 and detail >> 12 == 10
        assert not bool(y.any())                                 # none of a cluster stores anything
    finally:
        _lib.lib().lyraq_debug_fp8_block_rows_wait_test(-1, 0)
    assert torch.equal(layer.forward(x), want)                   # tensor memory was given back
    check_status()
