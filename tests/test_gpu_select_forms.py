"""GPU tests of the selection's and the block means' forms for many rows: one warp a row and several, each with its own range of key blocks."""

import pytest
import torch

from oracle import sparse
from tests.util import check_status

pytestmark = pytest.mark.gpu

Q_BLOCKS, BATCH, HEADS = 23, 3, 3          # 207 rows: more than the SMs, no multiple of four


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def assert_selected(qm, km, count, **k):
    from lyradiff_b200 import ops
    want = sparse.select(qm, km, count, **k)
    k = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in k.items()}
    got = ops.select_blocks(qm.cuda(), km.cuda(), count, **k)
    check_status()
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


def means(kb, seed):
    """Products that are often equal, zeros of either sign, infinities and a key block that is no number."""
    g = torch.Generator().manual_seed(seed)
    qm, km = torch.randint(-1, 2, (BATCH, HEADS, Q_BLOCKS, 8), generator=g).float(), torch.randint(-2, 3, (BATCH, HEADS, kb, 8), generator=g).float()
    # queries that keep away from the infinities' channel in one head, whose products there are no numbers then
    qm[:, :2, :, 0], km[:, :, :, 0] = 1, 0
    km[0, :, kb // 3] = float("nan")
    km[:, :, kb // 2, 0], km[:, :, kb // 4, 0] = float("inf"), float("-inf")
    return qm, km


@pytest.mark.parametrize("kb", [1, 31, 70, 128, 129, 511, 512, 513, 1025, 2048, 2049])
def test_rows_of_every_length(kb):
    block, queries = 64, 128 * Q_BLOCKS - 50
    keys = kb * block - 3
    qm, km = means(kb, kb)
    args = dict(queries=queries, keys=keys, block=block)
    lens = ints([0, keys - keys // 3, keys])
    start = ints([5, keys // 2 - queries, keys - queries])
    for count in sorted({1, max(1, kb // 7), max(1, kb - 1), kb + 2}):
        assert_selected(qm, km, count, **args)
    assert_selected(qm, km, max(1, kb // 5), **args, k_lens=lens, q_start=start, causal=True, window=2, sink=1)
    assert_selected(qm, km, 4, **args, k_lens=lens, sink=9)              # more than there is room for
    assert_selected(qm, km, 9, **args, k_lens=lens, sink=kb, shared=True, causal=True)


@pytest.mark.parametrize("kb", [70, 500, 1000, 1025])
def test_random_scores(kb):
    g = torch.Generator().manual_seed(kb)
    qm, km = torch.randn(BATCH, HEADS, Q_BLOCKS, 128, generator=g), torch.randn(BATCH, HEADS, kb, 128, generator=g)
    assert_selected(qm, km, 17, queries=128 * Q_BLOCKS, keys=64 * kb, block=64, window=1)


def test_few_rows_of_more_than_1024_key_blocks():
    g = torch.Generator().manual_seed(1)
    for kb in (1024, 1025):
        qm, km = torch.randint(-2, 3, (1, 2, 2, 8), generator=g).float(), torch.randint(-2, 3, (1, 2, kb, 8), generator=g).float()
        for count in (1, 33, kb - 1):
            assert_selected(qm, km, count, queries=200, keys=64 * kb, block=64, causal=True)


def test_places_far_from_blocks_of_any_length():
    g = torch.Generator().manual_seed(4)
    qm, km = torch.randn(4, 2, 2, 16, generator=g), torch.randn(4, 1, 1, 16, generator=g)
    for block in (570, 2 ** 29 + 1, 2 ** 30):
        for causal in (False, True):
            for window in (0, 1, 2 ** 31 - 1):
                assert_selected(qm, km, 2, queries=200, keys=570, block=block, q_start=ints([-2 ** 30, -2 ** 31, 2 ** 31 - 1, -200]), causal=causal, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 72, 128, 256])
@pytest.mark.parametrize("block", [64, 128, 50])
def test_means_of_many_blocks(dtype, dim, block):
    """More blocks than a thread block each would be given to, an odd number of them, some of several exponents (the way in 64 bits), sequences that end early."""
    from lyradiff_b200 import ops
    n, heads = block * 100 + 7, 7
    g = torch.Generator().manual_seed(dim + block)
    x = torch.randn(2, n, heads, dim, generator=g)
    x[:, ::97] *= 2.0 ** 13
    x[:, 5::89] *= 2.0 ** -13
    x = x.to(dtype)
    y = x.clone()
    lens = ints([n - n // 3, n])
    y[0, int(lens[0]):] = float("nan")
    got = ops.block_means(y.cuda(), block, lens.cuda()).cpu()
    check_status()
    want, size = sparse.means(x, block, lens).double(), sparse.means(x.abs().double(), block, lens).double()
    # sums in 64 bits in two orders, 2^-46 of the magnitudes apart at most (128 additions), then half a step of fp32 each
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -23 + size * 2.0 ** -45).all())
    assert bool((got[0, :, (int(lens[0]) + block - 1) // block:] == 0).all())
