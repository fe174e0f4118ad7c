"""GPU tests of attention over selected key blocks against the 64-bit restatement in oracle/sparse.py."""

import math

import pytest
import torch

from oracle import sparse
from tests.util import check_status

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from lyradiff_b200 import ops as _ops
    return _ops


def tokens(seed, batch, n, heads, dim, dtype, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(batch, n, heads, dim, generator=g) * size + 0.5 * torch.randn(batch, 1, heads, dim, generator=g)).to(dtype)


def dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


def ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32)


# ----------------------------------------------------------------------------- means
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,block,heads,dim", [(1, 64, 1, 8), (64, 64, 2, 64), (65, 64, 3, 128), (1000, 128, 2, 128), (777, 100, 2, 72), (300, 7, 1, 256)])
def test_means(ops, dtype, n, block, heads, dim):
    x = tokens(n, 2, n, heads, dim, dtype)
    x[0, n // 2] *= 1000
    x[1, :, :, 0] = 0
    lens = ints([n - n // 3, n])
    for l in (None, lens):
        y = x.clone()
        if l is not None:
            y[0, int(l[0]):] = float("nan")                     # tokens that do not exist are not read
        got = ops.block_means(y.cuda(), block, None if l is None else l.cuda())
        check_status()
        assert torch.equal(got.cpu(), sparse.means(x, block, l))


def test_means_of_views_and_of_the_newest_tokens(ops):
    x = tokens(3, 3, 500, 12, 64, BF16).unflatten(2, (3, 4))
    packed = x.cuda()
    want = sparse.means(x[:, :, 1], 64)
    assert torch.equal(ops.block_means(packed[:, :, 1], 64).cpu(), want)
    heads_first = packed[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.block_means(heads_first, 64).cpu(), want)
    lens = ints([1, 320, 0])
    for newest in (1, 2, 64, 65, 600):
        m = torch.full((3, 4, 8, 64), 9.0, device="cuda")
        assert ops.block_means(packed[:, :, 1], 64, lens.cuda(), m, newest) is m
        full = sparse.means(x[:, :, 1], 64, lens)
        for b, n in enumerate(lens.tolist()):
            for j in range(8):
                fresh = j * 64 < n and (j + 1) * 64 > n - newest
                assert torch.equal(m[b, :, j].cpu(), full[b, :, j] if fresh else torch.full((4, 64), 9.0)), (newest, b, j)
    check_status()
    with pytest.raises(ValueError):
        ops.block_means(packed[:, :, 1], 64, newest=1)
    with pytest.raises(ValueError):
        ops.block_means(packed[:, :, 1], 64, lens=lens)          # on the host


def test_means_of_numbers_at_the_ends_of_the_type(ops):
    for dtype in (BF16, F16):
        info = torch.finfo(dtype)
        x = torch.zeros(1, 256, 1, 8, dtype=dtype)
        x[0, :64, 0, 0], x[0, 64:128, 0, 1], x[0, 128, 0, 2], x[0, 192, 0, 3] = info.smallest_normal / 4, info.max, float("inf"), float("nan")
        x[0, :64, 0, 4] = -0.0
        x[0, :2, 0, 5] = torch.tensor([info.max, -info.max], dtype=dtype)
        x[0, 2, 0, 5] = info.eps
        got = ops.block_means(x.cuda(), 64).cpu()
        want = sparse.means(x, 64)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,block", [(128, 128), (640, 64), (50000, 64)])
def test_means_of_values_far_apart(ops, dtype, n, block):
    """Exponents on both sides of what sums in fp32 with their errors hold exactly, cancellation, and blocks that need 64 bits beside others: the means are
    those of exact sums."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, n, 2, 128, generator=g)
    low, high = (-126, 126) if dtype == BF16 else (-14, 15)
    for i, spread in enumerate((0, 10, 28, 29, 30, 31, 32, 33, 34, 40, 100, 250)):
        c = slice(i * 8, i * 8 + 8)
        at = torch.randint(0, spread + 1, (n, 2, 8), generator=g) + low
        x[0, :, :, c] = torch.ldexp(1 + torch.rand(n, 2, 8, generator=g), at.clamp(low, high - 1)) * (1 - 2 * torch.randint(0, 2, (n, 2, 8), generator=g))
    x[0, 1::2, :, 100:104] = -x[0, ::2, :, 100:104]                    # sums of 0
    x[0, ::3, :, 104] = 2.0 ** high * 1.5                             # sums beyond fp32's largest on the way, for bf16
    x[0, 1::3, :, 104] = -2.0 ** high * 1.5
    x = x.to(dtype)
    got = ops.block_means(x.cuda(), block).cpu()
    check_status()
    m = torch.zeros(1, 2, sparse.blocks(n, block), 128, dtype=torch.float64)
    for j in range(m.shape[2] if n < 10000 else 3):
        part = x[0, j * block:(j + 1) * block].double()
        for h in range(2):
            for c in range(128):
                m[0, h, j, c] = math.fsum(part[:, h, c].tolist()) / part.shape[0]
        want = m[0, :, j]
        # an exact sum, against one in 64 bits: 2^-50 of the magnitudes before it is rounded
        slack = part.abs().sum(0) / part.shape[0] * 2.0 ** -50
        half = torch.maximum(want.abs() * 2.0 ** -24, torch.tensor(2.0 ** -150, dtype=torch.float64))
        assert bool(((got[0, :, j].double() - want).abs() <= half + slack).all())
    # every block against the restatement: either side is half a step of fp32 and 2^-50 of the magnitudes from the exact mean
    size = sparse.means(x.double().abs(), block).double()
    want = sparse.means(x, block).double()
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -23 + size * 2.0 ** -48 + 2.0 ** -149).all())


# ----------------------------------------------------------------------------- selection
def assert_selected(ops, qm, km, count, **k):
    want = sparse.select(qm, km, count, **k)
    k = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in k.items()}
    got = ops.select_blocks(qm.cuda(), km.cuda(), count, **k)
    check_status()
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("queries,keys,block,count", [(1, 1, 64, 1), (1, 64, 64, 3), (130, 700, 64, 4), (1100, 1100, 128, 5), (300, 9000, 64, 17), (5, 33000, 64, 64),
                                                      (1, 140000, 64, 100), (140, 530000, 64, 33)])
@pytest.mark.parametrize("shared", [False, True])
def test_selection(ops, queries, keys, block, count, shared):
    g = torch.Generator().manual_seed(queries + keys)
    dim = 40 if keys > 100000 else 128
    qm = torch.randn(2, 4, sparse.blocks(queries, 128), dim, generator=g)
    km = torch.randn(2, 2, sparse.blocks(keys, block), dim, generator=g)
    lens, start = ints([keys - keys // 3, keys]), ints([keys // 2 - queries, keys - queries])
    for k in ({}, {"k_lens": lens, "q_start": start, "causal": True, "window": 1}, {"k_lens": lens, "sink": 2, "window": 2}, {"causal": True, "sink": 1}):
        assert_selected(ops, qm, km, count, queries=queries, keys=keys, block=block, shared=shared, **k)


def test_equal_scores_go_to_the_lowest_and_what_is_no_number_last(ops):
    g = torch.Generator().manual_seed(3)
    for keys in (1280, 64 * 700, 64 * 3000):
        kb = keys // 64
        km = torch.randint(-2, 3, (1, 1, kb, 8), generator=g).float()                # many equal products, zeros of either sign
        qm = torch.randint(-1, 2, (1, 1, 3, 8), generator=g).float()
        km[0, 0, 7] = float("nan")
        km[0, 0, 3, 0] = float("-inf")
        km[0, 0, 4, 0] = float("inf")
        qm[0, 0, :, 0] = 1
        for count in (1, 2, 5, kb // 2, kb - 1, kb, kb + 3):
            assert_selected(ops, qm, km, count, queries=300, keys=keys, block=64)
        assert_selected(ops, qm, km, 4, queries=300, keys=keys, block=64, sink=9)     # more than there is room for
        assert_selected(ops, qm, km, 9, queries=300, keys=keys, block=64, sink=kb, causal=True, q_start=ints([1]))


def test_places_outside_the_keys(ops):
    g = torch.Generator().manual_seed(4)
    qm, km = torch.randn(4, 2, 2, 16, generator=g), torch.randn(4, 1, 9, 16, generator=g)
    for causal in (False, True):
        for window in (0, 1, 3):
            assert_selected(ops, qm, km, 4, queries=200, keys=570, block=64, k_lens=ints([570, 0, 3, 570]), q_start=ints([-300, 5, -2 ** 31, 2 ** 31 - 1]), causal=causal,
                            window=window, sink=1)
    index, counts = ops.select_blocks(torch.zeros(1, 2, 1, 16, device="cuda"), torch.zeros(1, 2, 0, 16, device="cuda"), 3, 1, 0, 64)
    assert counts.flatten().tolist() == [0, 0] and bool((index == -1).all())


def test_means_and_selection_of_tokens(ops):
    q, k = tokens(1, 2, 900, 4, 128, BF16), tokens(2, 2, 2900, 2, 128, BF16)
    for shared in (False, True):
        args = dict(queries=900, keys=2900, block=64, causal=True, window=1, shared=shared)
        want = sparse.select(sparse.means(q, 128), sparse.means(k, 64), 9, **args)
        got = ops.select_blocks(ops.block_means(q.cuda(), 128), ops.block_means(k.cuda(), 64), 9, **args)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# ----------------------------------------------------------------------------- attention
def assert_attention(got, q, k, v, index, counts, block, **args):
    """Against 64 bits.  A score is a sum of head_dim products in head_dim / 16 instructions, each of which may lose an ulp (2^-23) of the sum of
    magnitudes, and the product with the scale, its exponent and exp2 lose another 2^-22 of that and of the result; a weight is off by twice the absolute error of
    its score and by half a step of its type (for fp16, whose small weights are subnormal, by 2^-25 of the row's sum if that is more); the sum of the
    products with v loses 2^-23 of the magnitudes in every 16 keys; the result is rounded to its type: half a step."""
    y, mag = sparse.attend(q, k, v, index, counts, block, **args)
    dim = q.shape[-1]
    scale = args.get("scale") or dim ** -0.5
    n = index.shape[3] * block
    finite_k, finite_v = k.float().nan_to_num(0, 0, 0).abs(), v.double().nan_to_num(0, 0, 0).abs()
    top = float(q.float().abs().flatten(0, 2).norm(dim=-1).max() * finite_k.flatten(0, 2).norm(dim=-1).max()) * scale
    half = torch.finfo(q.dtype).eps / 2
    rel = 2 * top * (dim // 16 + 3) * 2.0 ** -23 + 2.0 ** -20 + half + (n // 16 + 8) * 2.0 ** -23
    tol = rel * mag * (1 + half) + half * y.abs() + torch.finfo(q.dtype).tiny
    if q.dtype == F16:
        tol = tol + n * 2.0 ** -25 * float(finite_v.max())
    err = (got.cpu().double() - y).abs()
    bad = ~(err <= tol) & ~(got.cpu().isnan() & y.isnan())
    assert not bool(bad.any()), "off by %g of the tolerance at %s" % (float((err / tol).nan_to_num(1e9).max()), bad.nonzero()[0].tolist())


def lists(seed, batch, heads, nq, nk, block, count, fill=None):
    """Random lists of random lengths, ascending, with -1 (or anything else) behind."""
    g = torch.Generator().manual_seed(seed)
    qb, kb = sparse.blocks(nq, 128), sparse.blocks(nk, block)
    index = torch.full((batch, heads, qb, count), -1 if fill is None else fill, dtype=torch.int32)
    counts = torch.randint(0, min(count, kb) + 1, (batch, heads, qb), generator=g, dtype=torch.int32)
    counts[0, 0, 0] = min(count, kb)
    for b in range(batch):
        for h in range(heads):
            for i in range(qb):
                n = int(counts[b, h, i])
                index[b, h, i, :n] = torch.randperm(kb, generator=g)[:n].sort().values.to(torch.int32)
    return index, counts


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 64, 2, 1, 1), (1, 1, 1000, 8, 8, 4), (2, 3, 700, 8, 2, 5), (2, 128, 128, 2, 2, 2), (1, 129, 300, 4, 1, 3), (2, 300, 1111, 4, 2, 9),
          (1, 700, 700, 3, 3, 4), (1, 17, 5000, 16, 1, 20)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("batch,nq,nk,heads,k_heads,count", SHAPES)
def test_attention(ops, dtype, dim, block, batch, nq, nk, heads, k_heads, count):
    q, k, v = tokens(1, batch, nq, heads, dim, dtype), tokens(2, batch, nk, k_heads, dim, dtype), tokens(3, batch, nk, k_heads, dim, dtype)
    for shared in ([False, True] if heads != k_heads else [False]):
        index, counts = lists(nq + nk, batch, k_heads if shared else heads, nq, nk, block, count)
        for causal in (False, True):
            out = torch.full_like(q, float("nan")).cuda()
            got = ops.sparse_attention(*dev(q, k, v, index, counts), block, causal=causal, out=out)
            check_status()
            assert got is out
            assert_attention(got, q, k, v, index, counts, block, causal=causal)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("nq", [1, 4, 40, 300])
def test_lengths_places_and_what_lies_beyond(ops, dtype, dim, block, nq):
    """Keys and values beyond a sequence's length are NaN and infinities, lengths end inside a block and on its edges, a sequence has no keys; causal order
    with rows that see nothing."""
    batch, nk, heads, k_heads = 6, 640, 4, 2
    q, k, v = tokens(1, batch, nq, heads, dim, dtype), tokens(2, batch, nk, k_heads, dim, dtype), tokens(3, batch, nk, k_heads, dim, dtype)
    lens = ints([0, 1, 129, 256, 511, 640])
    start = ints([3, -5, 129 - nq, 70, -nq // 2, 640 - nq])
    kd, vd = k.clone(), v.clone()
    for b, n in enumerate(lens.tolist()):
        kd[b, n:], vd[b, n:] = float("nan"), float("inf")
        vd[b, n + 1::2] = float("nan")
    index, counts = lists(nq, batch, heads, nq, nk, block, 5)
    index[:, :, :, 0], counts = 0, counts.clamp_min(1)                  # the first block is in every list
    for args in ({}, {"q_start": start, "causal": True}):
        got = ops.sparse_attention(*dev(q, kd, vd, index, counts), block, k_lens=lens.cuda(), **{n: a.cuda() if isinstance(a, torch.Tensor) else a for n, a in args.items()})
        check_status()
        assert_attention(got, q, k, v, index, counts, block, k_lens=lens, **args)
        assert bool((got[0] == 0).all())


@pytest.mark.parametrize("nq", [1, 200])
def test_lists_as_they_come(ops, nq):
    """Indices outside the keys add nothing, a block listed twice counts twice, order does not matter, counts beyond the list or below 0 are taken as its ends."""
    q, k, v = tokens(1, 2, nq, 4, 128, BF16), tokens(2, 2, 500, 4, 128, BF16), tokens(3, 2, 500, 4, 128, BF16)
    qb = sparse.blocks(nq, 128)
    index = torch.tensor([7, 3, -1, 8, 3, 2 ** 31 - 1, -2 ** 31, 0, 1000], dtype=torch.int32).expand(2, 4, qb, 9).contiguous()
    counts = torch.tensor([9, 100, -4, 5], dtype=torch.int32)[None, :, None].expand(2, 4, qb).contiguous()
    got = ops.sparse_attention(*dev(q, k, v, index, counts), 64)
    check_status()
    assert_attention(got, q, k, v, index, counts, 64)
    assert bool((got[:, :, 2] == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq", [1, 260])
def test_strides(ops, nq, dim):
    """q, k and v inside one packed projection, a cache with heads before tokens, a result inside a wider tensor, a cache that all sequences share."""
    packed = tokens(1, 2, 260, 12, dim, F16).unflatten(2, (3, 4))
    q, k, v = packed[:, :nq, 0], packed[:, :, 1], packed[:, :, 2]
    index, counts = lists(5, 2, 4, nq, 260, 64, 4)
    pd = packed.cuda()
    wide = torch.full((2, nq + 3, 5, dim + 8), 7.0, dtype=F16, device="cuda")
    out = wide[:, 1:nq + 1, 1:, :dim]
    ops.sparse_attention(pd[:, :nq, 0], pd[:, :, 1], pd[:, :, 2], *dev(index, counts), 64, out=out)
    check_status()
    assert_attention(out, q, k, v, index, counts, 64)
    out.fill_(7.0)
    assert bool((wide == 7.0).all())                              # rows beside and behind: as they were
    cache = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v)]
    got = ops.sparse_attention(pd[:, :nq, 0], *cache, *dev(index, counts), 64)
    assert_attention(got, q, k, v, index, counts, 64)
    one = [t[:1].expand(2, -1, -1, -1) for t in cache]
    got = ops.sparse_attention(pd[:, :nq, 0], *one, *dev(index, counts), 64)
    check_status()
    assert_attention(got, q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), index, counts, 64)


@pytest.mark.parametrize("nq", [1, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_grow_and_that_are_no_numbers(ops, dtype, nq):
    """Maxima that rise from block to block (by much and by little), large scores, and queries whose scores are infinite or no number: NaN in that row alone."""
    q, k, v = tokens(1, 1, nq, 2, 128, dtype), tokens(2, 1, 1000, 2, 128, dtype), tokens(3, 1, 1000, 2, 128, dtype)
    k = k * torch.linspace(0.1, 6, 1000)[None, :, None, None].to(dtype)
    index, counts = lists(1, 1, 2, nq, 1000, 64, 16)
    counts.fill_(16)
    index[:] = torch.arange(16, dtype=torch.int32)
    got = ops.sparse_attention(*dev(q, k, v, index, counts), 64, softmax_scale=0.3)
    assert_attention(got, q, k, v, index, counts, 64, scale=0.3)
    got = ops.sparse_attention(*dev(q, k, v, index.flip(-1).contiguous(), counts), 64, softmax_scale=0.3)
    assert_attention(got, q, k, v, index, counts, 64, scale=0.3)
    if nq > 1:
        q[0, 5, 0, 3], q[0, 200, 1, 0] = float("nan"), float("inf")
        got = ops.sparse_attention(*dev(q, k, v, index, counts), 64)
        bad = torch.zeros(1, nq, 2, dtype=torch.bool)
        bad[0, 5, 0] = bad[0, 200, 1] = True
        assert torch.equal(got.isnan().all(-1).cpu(), bad) and torch.equal(got.isnan().any(-1).cpu(), bad)
    check_status()


@pytest.mark.parametrize("nq", [1, 130])
def test_a_cache_beyond_31_bits(ops, nq):
    """2^31 elements and more in k, and lists at its end."""
    n = 2 ** 24 + 2 ** 16
    k = torch.empty(1, n, 2, 64, dtype=BF16, device="cuda")
    tail = tokens(2, 1, 2 ** 10, 2, 64, BF16)
    k[:, -2 ** 10:] = tail.cuda()
    k[:, :64] = tail[:, :64].cuda()
    q = tokens(1, 1, nq, 2, 64, BF16)
    qb = sparse.blocks(nq, 128)
    index = torch.tensor([0, n // 64 - 16, n // 64 - 9, n // 64 - 1], dtype=torch.int32).expand(1, 2, qb, 4).contiguous()
    counts = torch.full((1, 2, qb), 4, dtype=torch.int32)
    got = ops.sparse_attention(q.cuda(), k, k, *dev(index, counts), 64)
    check_status()
    short = torch.cat([tail[:, :64], tail], dim=1)
    assert_attention(got, q, short, short, torch.tensor([0, 1, 8, 16], dtype=torch.int32).expand(1, 2, qb, 4).contiguous(), counts, 64)


def test_many_items_and_long_lists(ops):
    """Several rounds of the persistent grid, lists of very different length next to each other, against attention in torch on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = torch.randn(3, 1, 5000, 12, 128, generator=g, device="cuda").bfloat16()
    index, counts = lists(2, 1, 12, 5000, 5000, 64, 79)
    got = ops.sparse_attention(q, k, v, *dev(index, counts), 64)
    check_status()
    for h in (0, 5, 11):
        mask = torch.zeros(40, 79, dtype=torch.bool)
        for i in range(40):
            mask[i, index[0, h, i, :int(counts[0, h, i])].long()] = True
        see = mask.repeat_interleave(128, 0)[:5000].repeat_interleave(64, 1)[:, :5000].cuda()
        s = (q[0, :, h].double() @ k[0, :, h].double().t() * 128 ** -0.5).masked_fill(~see, float("-inf"))
        w = torch.softmax(s, -1).nan_to_num(0)
        y, mag = w @ v[0, :, h].double(), w @ v[0, :, h].double().abs()
        # half a step of the weights and of the result, 2^-11 for the rest (scores below 32: 2 * 32 * 11 * 2^-23 and the sums' 320 * 2^-23)
        assert bool(((got[0, :, h].double() - y).abs() <= mag * (2.0 ** -8 * 1.01 + 2.0 ** -11) + y.abs() * 2.0 ** -8).all())


def test_the_same_bits_every_time_on_streams_and_in_graphs(ops):
    from lyradiff_b200.layers import SparseAttention
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = SparseAttention(64, 6, sink=1, window=1)
    calls = []
    for nq, nk, hq, hk in ((700, 700, 4, 4), (1, 2000, 8, 2), (1, 300, 2, 2), (300, 1500, 4, 1)):
        calls.append([torch.randn(2, n, h, 128, generator=g, device="cuda").bfloat16() for n, h in ((nq, hq), (nk, hk), (nk, hk))])
    want = [layer.forward(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for s, c, o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(layer.forward(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for o, w in zip(got, want) for y in o)
    graphs = []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward(*c)
        graphs.append((graph, y))
    for step in range(3):
        for (graph, _), c in zip(graphs, calls):
            c[2].mul_(-1)
            graph.replay()
        torch.cuda.synchronize()
        for (_, y), w in zip(graphs, want):
            assert torch.equal(y, w if step % 2 else -w)
    check_status()


def test_layer_is_means_selection_and_attention(ops):
    from lyradiff_b200.layers import SparseAttention
    q, k, v = (t.cuda() for t in (tokens(1, 2, 300, 4, 64, F16), tokens(2, 2, 900, 2, 64, F16), tokens(3, 2, 900, 2, 64, F16)))
    lens, start = ints([800, 900]).cuda(), ints([500, 600]).cuda()
    for shared in (False, True):
        layer = SparseAttention(128, 3, sink=1, window=1, shared=shared, causal=True, softmax_scale=0.2)
        out, index, counts = layer.forward(q, k, v, k_lens=lens, q_start=start, with_selection=True)
        km = ops.block_means(k, 128, lens)
        i2, c2 = ops.select_blocks(ops.block_means(q, 128), km, 3, 300, 900, 128, lens, start, True, 1, 1, shared)
        assert torch.equal(index, i2) and torch.equal(counts, c2)
        assert torch.equal(out, ops.sparse_attention(q, k, v, i2, c2, 128, lens, start, True, 0.2))
        again = torch.empty_like(q)
        assert layer.forward(q, k, v, k_lens=lens, q_start=start, k_means=km, out=again) is again and torch.equal(again, out)
    check_status()


def test_refusals(ops):
    from lyradiff_b200 import _lib
    from lyradiff_b200.layers import SparseAttention
    q, k = torch.zeros(1, 5, 2, 64, dtype=F16, device="cuda"), torch.zeros(1, 300, 2, 64, dtype=F16, device="cuda")
    index, counts = torch.zeros(1, 2, 1, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, 1, dtype=torch.int32, device="cuda")
    good = dict(q=q, k=k, v=k, index=index, counts=counts, block=64)
    assert bool((ops.sparse_attention(**good) == 0).all())
    for change in (dict(q=q.bfloat16()), dict(v=k[:, :200]), dict(k=k[:, :, :, :32]), dict(index=index.long()), dict(counts=counts[:, :1]), dict(index=index[:, :1]),
                   dict(k_lens=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(k_lens=torch.zeros(1, device="cuda")), dict(q=q.cpu()), dict(q=q[0]),
                   dict(out=torch.empty(1, 6, 2, 64, dtype=F16, device="cuda")), dict(out=q.expand(1, 5, 2, 64)[:, :1].expand(1, 5, 2, 64))):
        with pytest.raises((ValueError, TypeError)):
            ops.sparse_attention(**{**good, **change})
    for change in (dict(out=q), dict(softmax_scale=-1.0), dict(block=32), dict(q=q[..., :32].contiguous(), k=k[..., :32].contiguous(), v=k[..., :32].contiguous())):
        with pytest.raises(_lib.LyraqError):
            ops.sparse_attention(**{**good, **change})
    for bad in ((32, 1), (64, 0), (64, 1, -1)):
        with pytest.raises(ValueError):
            SparseAttention(*bad)
    empty = torch.zeros(1, 0, 2, 64, dtype=F16, device="cuda")
    assert bool((SparseAttention(64, 2).forward(q, empty, empty) == 0).all())
    assert SparseAttention(64, 2).forward(empty, k, k).shape == empty.shape
    check_status()


@pytest.mark.parametrize("nq,kernel", [(300, 8), (1, 9)])
def test_a_wait_that_runs_out_is_reported(ops, nq, kernel):
    from lyradiff_b200 import _lib
    q, k = torch.randn(1, nq, 2, 128, device="cuda").bfloat16(), torch.randn(1, 600, 2, 128, device="cuda").bfloat16()
    qb = sparse.blocks(nq, 128)
    index, counts = torch.arange(5, dtype=torch.int32, device="cuda").expand(1, 2, qb, 5).contiguous(), torch.full((1, 2, qb), 5, dtype=torch.int32, device="cuda")
    want = ops.sparse_attention(q, k, k, index, counts, 64)
    check_status()
    _lib.check(_lib.lib().lyraq_debug_sparse_attention_wait_test(1, 200), "hook")
    try:
        ops.sparse_attention(q, k, k, index, counts, 64)
        status, detail = ops.last_status()
        assert status == 4 and detail >> 12 == kernel
    finally:
        _lib.lib().lyraq_debug_sparse_attention_wait_test(0, 0)
    assert torch.equal(ops.sparse_attention(q, k, k, index, counts, 64), want)     # tensor memory was given back
    check_status()
