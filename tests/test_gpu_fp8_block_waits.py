"""GPU test of the tiled block-scaled FP8 product when a wait runs out: a CTA that issues no loads, and waits of 200 ms."""

import pytest
import torch

from tests.util import check_status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,rank", [(1281, 0), (2562, 1), (1282, 1), (1284, 0), (1288, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_wait_that_runs_out_is_reported(code, rank, dtype):
    """The status tells, tiles of the stalled CTA (with K over a cluster: of any of its CTAs) are not stored, and the next call has its tensor memory again."""
    from lyradiff_b200 import _lib, ops
    g = torch.Generator(device="cuda").manual_seed(code)
    w, x = torch.randn(200, 2320, generator=g, device="cuda"), torch.randn(100, 2320, generator=g, device="cuda")
    operands = *ops.weight_quant_fp8_block(w), *ops.quant_fp8_block(x)
    lib = _lib.lib()
    try:
        _lib.check(lib.lyraq_debug_force_fp8_block_tile(code), "tile")
        want = ops.gemm_fp8_block(*operands, dtype)
        check_status()
        _lib.check(lib.lyraq_debug_fp8_block_wait_test(rank, 200), "hook")
        y = torch.full_like(want, 7.0)
        ops.gemm_fp8_block(*operands, y)
        status, detail = ops.last_status()
        assert status == 4 and detail >> 12 == 7
        assert bool((y == 7.0).all())
        lib.lyraq_debug_fp8_block_wait_test(-1, 0)
        ops.gemm_fp8_block(*operands, y)
        check_status()
        assert torch.equal(y, want)
    finally:
        lib.lyraq_debug_fp8_block_wait_test(-1, 0)
        lib.lyraq_debug_force_fp8_block_tile(0)
