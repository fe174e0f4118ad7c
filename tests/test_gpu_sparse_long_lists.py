"""GPU tests of few queries against lists of thousands of key blocks: the first keys of a list weigh as much as the last."""

import pytest
import torch

from tests.util import check_status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,block,queries", [(64, 64, 1), (128, 64, 1), (128, 128, 3)])
def test_equal_keys_weigh_the_same_however_long_the_list(dtype, dim, block, queries):
    """All keys of a head are alike, so its maximum stands from the first key on, and lists are too many to be split: each is one run of 4096 half blocks.  The values
    are 1 in the first half of a list and -1 in the second, so a query's result is 0.  Exactly: with |score * log2(e)| below 2^11 the exponent's rounding is
    at most 2^-14, which leaves every weight within 5e-5 of one, nearer than half a step of either type (2^-12, 2^-9 below one), so it is rounded to one; sums of up to
    2^18 ones are exact in 32 bits, in any order.  A weight that drifted by 2^-24 for each half block would show as 2^-24 * 2048 / 2 = 6e-5."""
    from lyradiff_b200 import ops
    heads = torch.cuda.get_device_properties(0).multi_processor_count + 12
    count = 4096 * 64 // block
    g = torch.Generator().manual_seed(dim + block)
    k = torch.randn(1, 1, heads, dim, generator=g).to(dtype)
    scale = 900.0 / dim
    score = (k.double() ** 2).sum(-1) * scale * 1.4426950408889634
    assert bool((score > 500).all()) and bool((score < 2048).all())
    q, keys = k.expand(1, queries, heads, dim).contiguous(), k.expand(1, 2 * block, heads, dim).contiguous()
    v = torch.ones(1, 2 * block, heads, dim).to(dtype)
    v[:, block:] = -1
    index = torch.zeros(1, heads, 1, count, dtype=torch.int32)
    index[..., count // 2:] = 1
    counts = torch.full((1, heads, 1), count, dtype=torch.int32)
    got = ops.sparse_attention(q.cuda(), keys.cuda(), v.cuda(), index.cuda(), counts.cuda(), block, softmax_scale=scale)
    check_status()
    assert bool((got == 0).all()), "off by %g" % float(got.abs().max())
