"""Fp8BlockLinear from what a block-scaled checkpoint holds: codes as torch.float8_e4m3fn and fp32 scales."""

import pytest
import torch

from oracle import fp8_block


def held(n, k):
    codes, scales = fp8_block.encode(torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * 0.05, 128)
    return codes.view(torch.float8_e4m3fn), scales


def test_codes_of_either_type_are_the_same_weight():
    from lyradiff_b200.layers import Fp8BlockLinear
    codes, scales = held(200, 272)
    a, b = Fp8BlockLinear(codes, scales), Fp8BlockLinear(codes.view(torch.uint8), scales)
    assert a.codes.dtype == torch.uint8 and torch.equal(a.codes, b.codes) and (a.n, a.k) == (200, 272)
    assert torch.equal(Fp8BlockLinear(codes.t().contiguous().t(), scales).codes, b.codes)
    for bad in (codes.view(torch.int8), codes.float(), codes.float().to(torch.float8_e5m2)):
        with pytest.raises(ValueError):
            Fp8BlockLinear(bad, scales)
    with pytest.raises(ValueError):
        Fp8BlockLinear(codes, scales.half())


@pytest.mark.gpu
def test_forward():
    from lyradiff_b200.layers import Fp8BlockLinear
    from tests.test_gpu_fp8_block import assert_product
    from tests.util import check_status
    codes, scales = held(200, 272)
    x = torch.randn(40, 272, generator=torch.Generator().manual_seed(1)).bfloat16()
    y = Fp8BlockLinear(codes.cuda(), scales.cuda()).forward(x.cuda())
    check_status()
    assert_product(y, fp8_block.encode(x), (codes.view(torch.uint8), scales))
