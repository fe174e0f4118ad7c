"""GPU tests of attention over selected key blocks in a padded batch: what lies behind a sequence reaches neither a list nor a result."""

import pytest
import torch

from oracle import sparse
from tests.test_gpu_sparse import assert_attention, ints, lists, tokens
from tests.util import check_status

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def behind(x, lens, fill):
    x = x.clone()
    for b, n in enumerate(lens):
        x[b, n:] = fill
    return x


@pytest.mark.parametrize("dtype,dim,block", [(BF16, 128, 64), (F16, 64, 128)])
@pytest.mark.parametrize("options", [{}, {"shared": True, "window": 1}, {"causal": True, "sink": 1, "window": 2}])
def test_a_padded_batch_is_its_sequences_one_by_one(dtype, dim, block, options):
    from lyradiff_b200.layers import SparseAttention
    lens, n, heads, k_heads, count = [520, 700, 0, 384, 257, 1], 700, 4, 2, 3
    q, k, v = tokens(1, 6, n, heads, dim, dtype), tokens(2, 6, n, k_heads, dim, dtype), tokens(3, 6, n, k_heads, dim, dtype)
    layer = SparseAttention(block, count, **options)
    at = ints(lens)
    args = {"k_lens": at, "q_lens": at}
    first = None
    for fill in (0.0, 7.0, float("nan"), float("inf")):
        out, index, counts = layer.forward(*(behind(x, lens, fill).cuda() for x in (q, k, v)), k_lens=at.cuda(), q_lens=at.cuda(), with_selection=True)
        check_status()
        first = first or (out, index, counts)
        assert all(torch.equal(a, b) for a, b in zip(first, (out, index, counts)))
    want = sparse.select(sparse.means(q, 128, at), sparse.means(k, block, at), count, n, n, block, **args, **options)
    assert torch.equal(index.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    assert_attention(out, q, k, v, *want, block, causal=options.get("causal", False), **args)
    for b, m in enumerate(lens):
        assert bool((out[b, m:] == 0).all()) and bool((counts[b, :, (m + 127) // 128:] == 0).all())
        if m > 16:                                                # few queries alone go to another kernel, whose sums run in another order
            alone = layer.forward(*(x[b:b + 1, :m].cuda() for x in (q, k, v)), with_selection=True)
            blocks = (m + 127) // 128
            assert torch.equal(alone[0][0], out[b, :m])
            assert torch.equal(alone[1][0], index[b, :, :blocks]) and torch.equal(alone[2][0], counts[b, :, :blocks])
    check_status()


@pytest.mark.parametrize("queries,heads", [(300, 2), (3000, 4)])      # several warps a row, and one
@pytest.mark.parametrize("shared", [False, True])
def test_selection_for_the_queries_that_exist(queries, heads, shared):
    from lyradiff_b200 import ops
    g = torch.Generator().manual_seed(queries)
    qm, km = torch.randn(6, heads, sparse.blocks(queries, 128), 64, generator=g), torch.randn(6, 2, 15, 64, generator=g)
    q_lens, start = ints([0, 1, 128, 129, -5, 2 ** 31 - 1]), ints([3, 800, -70, 500, 0, -200])
    for options in ({}, {"causal": True}, {"window": 1}, {"causal": True, "window": 2, "sink": 1}):
        want = sparse.select(qm, km, 4, queries, 900, 64, q_start=start, q_lens=q_lens, shared=shared, **options)
        got = ops.select_blocks(qm.cuda(), km.cuda(), 4, queries, 900, 64, q_start=start.cuda(), q_lens=q_lens.cuda(), shared=shared, **options)
        check_status()
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])
        assert bool((got[1][0] == 0).all())


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("nq", [1, 4, 40, 300])
def test_rows_behind_the_queries_get_zeros(dtype, dim, nq):
    from lyradiff_b200 import ops
    heads, k_heads, nk = 4, 2, 640
    q, k, v = tokens(1, 6, nq, heads, dim, dtype), tokens(2, 6, nk, k_heads, dim, dtype), tokens(3, 6, nk, k_heads, dim, dtype)
    q_lens, start = ints([0, 1, nq // 2, nq, -3, 2 ** 31 - 1]), ints([3, 500, 129 - nq, 70, -nq // 2, 640 - nq])
    index, counts = lists(nq, 6, heads, nq, nk, 64, 5)
    ends = [min(max(n, 0), nq) for n in q_lens.tolist()]
    qd = behind(q, ends, float("nan"))
    for causal in (False, True):
        out = torch.full_like(q, float("nan")).cuda()
        got = ops.sparse_attention(qd.cuda(), k.cuda(), v.cuda(), index.cuda(), counts.cuda(), 64, q_start=start.cuda(), causal=causal, out=out, q_lens=q_lens.cuda())
        check_status()
        assert_attention(got, q, k, v, index, counts, 64, q_start=start, causal=causal, q_lens=q_lens)
        for b, n in enumerate(ends):
            assert bool((got[b, n:] == 0).all())


def test_captured_with_lengths_that_change():
    """The lengths are read on the device: one graph serves any of them."""
    from lyradiff_b200.layers import SparseAttention
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = torch.randn(3, 2, 500, 4, 64, generator=g, device="cuda").bfloat16()
    layer, lens = SparseAttention(64, 3, window=1), torch.tensor([500, 500], dtype=torch.int32, device="cuda")
    layer.forward(q, k, v, k_lens=lens, q_lens=lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.forward(q, k, v, k_lens=lens, q_lens=lens)
    for values in ([400, 17], [0, 500], [129, 128]):
        lens.copy_(torch.tensor(values, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer.forward(q, k, v, k_lens=lens, q_lens=lens))
        assert all(bool((y[b, n:] == 0).all()) for b, n in enumerate(values))
    check_status()


def test_refusals():
    from lyradiff_b200 import ops
    from lyradiff_b200.layers import SparseAttention
    q = torch.zeros(2, 300, 2, 64, dtype=F16, device="cuda")
    for bad in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32, device="cuda")):
        with pytest.raises((ValueError, TypeError)):
            SparseAttention(64, 2).forward(q, q, q, q_lens=bad)
        with pytest.raises((ValueError, TypeError)):
            ops.select_blocks(ops.block_means(q, 128), ops.block_means(q, 64), 2, 300, 300, 64, q_lens=bad)
