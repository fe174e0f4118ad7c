"""GPU tests of a block's attention over a long sequence as it is run: FP8 block linears around QK norm and rotary embedding, selection and block-sparse
attention, eager, captured, and token by token over a cache."""

import pytest
import torch

from oracle import fp8_block, sparse
from tests.test_gpu_fp8_block import assert_product
from tests.test_gpu_sparse import assert_attention
from tests.util import check_status

pytestmark = pytest.mark.gpu

HEADS, K_HEADS, DIM, WIDTH = 4, 2, 128, 512


def parts(seed, dtype):
    from lyradiff_b200.layers import Fp8BlockLinear, SparseAttention
    from lyradiff_b200.rope import AxisRope
    g = torch.Generator().manual_seed(seed)
    qkv_w = (torch.randn((HEADS + 2 * K_HEADS) * DIM, WIDTH, generator=g) * 0.06).to(dtype)
    out_w = (torch.randn(WIDTH, HEADS * DIM, generator=g) * 0.05).to(dtype)
    norms = [(1 + 0.1 * torch.randn(DIM, generator=g)).to(dtype).cuda() for _ in range(2)]
    return qkv_w, out_w, Fp8BlockLinear.from_float(qkv_w.cuda()), Fp8BlockLinear.from_float(out_w.cuda()), norms, AxisRope((DIM,)), SparseAttention


def project(x, qkv, norms, plan, first):
    from lyradiff_b200 import ops
    b, n = x.shape[:2]
    heads = qkv.forward(x).view(b, n, HEADS + 2 * K_HEADS, DIM)
    q, k, v = heads.split([HEADS, K_HEADS, K_HEADS], dim=2)
    pos = (first.reshape(-1, 1) + torch.arange(n, device="cuda")).expand(b, n)[..., None].int()
    q, k = ops.rope_axes(plan, pos, q, k, q_norm=norms[0], k_norm=norms[1])
    return q, k, v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,n,causal", [(1, 700, False), (2, 301, True)])
def test_step_by_step_and_captured(dtype, batch, n, causal):
    qkv_w, out_w, qkv, out, norms, plan, attention = parts(n, dtype)
    attend = attention(64, 4, sink=1, window=1, causal=causal)
    x = torch.randn(batch, n, WIDTH, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()

    zero = torch.zeros(1, dtype=torch.int32, device="cuda")

    def block():
        q, k, v = project(x, qkv, norms, plan, zero)
        a, index, counts = attend.forward(q, k, v, with_selection=True)
        return q, k, v, a, index, counts, out.forward(a.flatten(2), residual=x)

    q, k, v, a, index, counts, y = block()
    check_status()
    heads = qkv.forward(x).view(batch * n, -1)
    assert_product(heads, fp8_block.encode(x.cpu().flatten(0, 1)), fp8_block.encode(qkv_w, 128))
    want = sparse.select(sparse.means(q.cpu(), 128), sparse.means(k.cpu(), 64), 4, n, n, 64, causal=causal, sink=1, window=1)
    assert torch.equal(index.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    assert_attention(a, q.cpu(), k.cpu(), v.cpu(), *want, 64, causal=causal)
    assert_product(y.flatten(0, 1), fp8_block.encode(a.cpu().flatten(2).flatten(0, 1)), fp8_block.encode(out_w, 128), residual=x.cpu().flatten(0, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    x.copy_(x.flip(1))
    graph.replay()
    for c, e in zip(captured, block()):
        assert torch.equal(c, e)
    check_status()


@pytest.mark.parametrize("shared", [False, True])
def test_token_by_token_over_a_cache(shared):
    """Sequences of different length grow by a token a step, captured once; the means of the newest blocks are renewed.  Each step against the operators on the
    whole cache, and the attention against 64 bits."""
    from lyradiff_b200 import ops
    dtype, batch, room = torch.bfloat16, 3, 400
    qkv_w, out_w, qkv, out, norms, plan, attention = parts(7, dtype)
    attend = attention(64, 3, sink=1, window=1, shared=shared, causal=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = [torch.full((batch, K_HEADS, room, DIM), float("nan"), dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2)]   # what is not there yet: NaN
    lens = torch.tensor([63, 250, 128], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens.tolist()):
        for c in cache:
            c[b, :n] = torch.randn(n, K_HEADS, DIM, generator=g, device="cuda").to(dtype)
    means = ops.block_means(cache[0], 64, lens)
    x = torch.randn(batch, 1, WIDTH, generator=g, device="cuda").to(dtype)
    rows = torch.arange(batch, device="cuda")

    def step():
        q, k, v = project(x, qkv, norms, plan, lens)
        cache[0][rows, lens.long()] = k[:, 0]
        cache[1][rows, lens.long()] = v[:, 0]
        lens.add_(1)
        ops.block_means(cache[0], 64, lens, means, newest=1)
        a, index, counts = attend.forward(q, *cache, k_lens=lens, q_start=lens - 1, k_means=means, with_selection=True)
        return q, a, index, counts, out.forward(a.flatten(2), residual=x)

    kept = [t.clone() for t in (*cache, lens, means)]
    step()                                                            # warm-up, then everything back
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, a, index, counts, y = step()
    for t, old in zip((*cache, lens, means), kept):
        t.copy_(old)
    for _ in range(4):                                                # across the edges of blocks
        x.copy_(torch.randn(batch, 1, WIDTH, generator=g, device="cuda"))
        graph.replay()
        check_status()
        assert torch.equal(means, ops.block_means(cache[0], 64, lens))
        n = lens.cpu()
        want = sparse.select(sparse.means(q.cpu(), 128), sparse.means(cache[0].cpu(), 64, n), 3, 1, room, 64, n, n - 1, True, 1, 1, shared)
        assert torch.equal(index.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
        k, v = (c.cpu().nan_to_num(0.0) for c in cache)
        assert_attention(a, q.cpu(), k, v, *want, 64, k_lens=n, q_start=n - 1, causal=True)
        assert torch.equal(y, out.forward(a.flatten(2), residual=x))
