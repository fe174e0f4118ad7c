"""GPU tests of FP4 linears of few rows whose CTAs go through the ring of stages several times (csrc/fp4_deal.h): the rows quantized on their way."""

import pytest
import torch

from tests.util import check_status

pytestmark = pytest.mark.gpu

# (n, k): one, two, four and eight CTAs along K; 8 to 33 K blocks each, 12, 9, 8 or 9, 10, 13 or 14, 8 or 9, 32, 33, 33 and, with a part of one, 8 or 9
SHAPES = [(21504, 3072), (19072, 2304), (9216, 4352), (13824, 5120), (5120, 13824), (4096, 16896), (28672, 8192), (19072, 8448), (72, 67584), (9216, 4384)]
ROWS = (1, 2, 3, 4, 8, 16)


@pytest.fixture(scope="module")
def layers():
    from lyradiff_b200 import layers as _layers
    return _layers


@pytest.fixture
def tile():
    from lyradiff_b200 import _lib
    yield lambda code: _lib.check(_lib.lib().lyraq_debug_force_fp4_tile(code), "lyraq_debug_force_fp4_tile")
    _lib.lib().lyraq_debug_force_fp4_tile(0)


def whole(rows, k, g):
    """Values of 0, 1, -1 and 2 with a 6 in front of every 16: scale 1 (times powers of two) in either format, so FP4 holds them as they are and every
    partial sum is an integer below 36 * 67584 < 2^24: exact in any order."""
    v = torch.tensor([0.0, 1.0, -1.0, 2.0], dtype=torch.bfloat16, device="cuda")[torch.randint(0, 4, (rows, k), generator=g, device="cuda")]
    v[:, ::16] = 6
    return v


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("n,k", SHAPES)
def test_products_of_whole_numbers_are_exact(layers, tile, fmt, n, k):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    w, x = whole(n, k, g), whole(16, k, g)
    layer = layers.Fp4Linear(w, None, torch.tensor(1.0), fmt=fmt)
    want = x.double() @ w.double().t()
    for code in (0, 16):        # the automatic choice, and the few-row kernel wherever it can
        tile(code)
        for m in ROWS:
            for dtype in (torch.float32, torch.bfloat16):
                got = layer.forward(x[:m].to(dtype))
                check_status()
                assert torch.equal(got, want[:m].to(dtype)), (code, m, dtype)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", SHAPES)
def test_bits_of_quantize_then_product(layers, tile, fmt, dtype, n, k):
    from lyradiff_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(n + k)
    w = (torch.randn(n, k, generator=g, device="cuda") * 0.05).bfloat16()
    x = torch.randn(16, k, generator=g, device="cuda").to(dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype)
    layer = layers.Fp4Linear(w, bias, torch.tensor(2.0 ** -7), fmt=fmt)
    tile(16)
    for m in ROWS:
        q = layer.empty_input(m)
        ops.quant_fp4(x[:m], out=q)
        want = layer.forward_quantized(q, dtype)
        for _ in range(3):
            got = layer.forward(x[:m])
            check_status()
            assert torch.equal(got, want), m


@pytest.mark.parametrize("m", [1, 2])
def test_a_captured_chain_of_one_and_two_rows(layers, m):
    """The width of a block's projections and back, several times over, replayed with new rows."""
    g = torch.Generator(device="cuda").manual_seed(m)
    up, down = (layers.Fp4Linear((torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).bfloat16(), None, torch.tensor(2.0 ** -7))
                for n, k in ((21504, 3072), (3072, 21504)))
    x = torch.randn(m, 3072, generator=g, device="cuda").bfloat16()

    def chain(v):
        for _ in range(4):
            v = down.forward(up.forward(v))
        return v
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = chain(x)
    for _ in range(5):
        x.copy_(torch.randn(m, 3072, generator=g, device="cuda"))
        want = chain(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_status()
        assert torch.equal(out, want) and bool(torch.isfinite(out).all())


@pytest.mark.parametrize("m", [2, 100])
def test_a_result_on_the_weight_or_partly_on_the_residual_is_refused(layers, m):
    from lyradiff_b200._lib import LyraqError
    g = torch.Generator(device="cuda").manual_seed(4)
    layer = layers.Fp4Linear((torch.randn(512, 512, generator=g, device="cuda") * 0.05).bfloat16(), None, torch.tensor(2.0 ** -7))
    x = torch.randn(m, 512, generator=g, device="cuda").bfloat16()
    both = torch.randn((m + 1) * 512, generator=g, device="cuda").bfloat16()
    r, moved, before = both[:m * 512].view(m, 512), both[512:].view(m, 512), both.clone()
    want = layer.forward(x, residual=r.clone())
    with pytest.raises(LyraqError):
        layer.forward(x, residual=r, out=moved)
    with pytest.raises(LyraqError):
        layer.forward(x, out=layer.weight.codes.view(-1).view(torch.bfloat16)[:m * 512].view(m, 512))
    torch.cuda.synchronize()
    assert torch.equal(both, before)
    layer.forward(x, residual=r, out=r)
    check_status()
    assert torch.equal(r, want)
