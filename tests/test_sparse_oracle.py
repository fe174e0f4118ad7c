"""CPU tests of block-sparse attention's restatement, and of what its calls refuse before they touch a device."""

import ctypes
import math

import pytest
import torch

from lyradiff_b200 import _lib, build
from oracle import sparse

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 5
P = [0x100000 + (i << 34) for i in range(12)]


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("causal", [False, True])
def test_all_blocks_are_dense_attention(causal):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, n, h, 16, generator=g) for n, h in ((150, 4), (300, 2), (300, 2)))
    qm, km = sparse.means(q, 128), sparse.means(k, 64)
    index, counts = sparse.select(qm, km, 7, 150, 300, 64, causal=causal)
    assert counts.tolist() == [[[5 if not causal or i else (150 + 127) // 64 + 1 for i in range(2)]] * 4] * 2
    got, _ = sparse.attend(q, k, v, index, counts, 64, causal=causal)
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double().repeat_interleave(2, 2)) / 4
    if causal:
        s = s.masked_fill(torch.arange(300)[None] > 150 + torch.arange(150)[:, None], -math.inf)
    want = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v.double().repeat_interleave(2, 2))
    assert float((got - want).abs().max()) < 1e-12


def test_selection_by_hand():
    km = torch.tensor([3.0, 1.0, 3.0, float("nan"), 2.0, 3.0]).reshape(1, 1, 6, 1)
    qm = torch.ones(1, 1, 1, 1)
    pick = lambda count, **k: [t.flatten().tolist() for t in sparse.select(qm, km, count, 1, 384, 64, **k)]   # noqa: E731
    assert pick(2) == [[0, 2], [2]] and pick(4) == [[0, 2, 4, 5], [4]] and pick(7) == [[0, 1, 2, 3, 4, 5, -1], [6]]
    assert pick(2, k_lens=[130]) == [[0, 2], [2]] and pick(2, k_lens=[0]) == [[-1, -1], [0]]
    assert pick(2, sink=1, window=1, q_start=[200]) == [[0, 3], [2]] and pick(3, window=2, q_start=[70]) == [[0, 1, 2], [3]]
    assert pick(3, causal=True, q_start=[127]) == [[0, 1, -1], [2]] and pick(1, causal=True, q_start=[-1]) == [[-1], [0]]


def test_means_refusals(lib):
    def means(m=P[0], x=P[1], t=1, sb=4096, st=64, sh=32, lens=None, block=64, newest=0, batch=2, tokens=60, heads=2, dim=32):
        return lib.lyraq_block_means(m, x, t, sb, st, sh, lens, block, newest, batch, tokens, heads, dim, None)
    assert means(batch=0) == means(tokens=0) == means(heads=0) == 0
    assert means(block=0) == means(newest=-1) == means(m=None) == means(x=None) == means(x=P[1] + 2) == means(st=60) == means(lens=P[2] + 2) == INVALID
    assert means(t=2) == means(dim=36) == means(dim=264) == means(tokens=1 << 31) == UNSUPPORTED
    assert means(m=P[1] + 4096) == means(lens=P[0]) == INVALID


def test_select_refusals(lib):
    def select(size=None, work=P[6], **k):
        f = dict(q_means=P[0], k_means=P[1], index=P[2], counts=P[3], k_lens=P[4], q_start=P[5], batch=2, queries=300, keys=1000, q_heads=4, k_heads=2, lists=2,
                 head_dim=64, block=64, count=5, sink=0, window=0, causal=0)
        f.update(k)
        a = _lib.SelectBlocksArgs(**f)
        need = lib.lyraq_select_blocks_workspace(f["batch"], f["lists"], f["queries"], f["keys"], f["block"])
        return lib.lyraq_select_blocks(ctypes.byref(a), work, need if size is None else size, None)
    assert lib.lyraq_select_blocks_workspace(2, 2, 300, 1000, 64) == 2 * 2 * 3 * 16 * 4 and lib.lyraq_select_blocks(None, None, 0, None) == INVALID
    assert select(batch=0) == select(queries=0) == select(q_heads=0) == 0
    assert select(block=0) == select(count=0) == select(sink=-1) == select(window=-1) == select(k_heads=3) == select(lists=3) == select(k_heads=0) == INVALID
    assert select(head_dim=60) == select(head_dim=0) == select(keys=64 * 32769) == select(count=40000) == UNSUPPORTED
    assert select(q_means=None) == select(index=None) == select(counts=P[3] + 2) == select(k_means=P[1] + 4) == INVALID
    assert select(work=None) == select(size=100) == select(work=P[6] + 4) == WORKSPACE
    assert select(index=P[1]) == select(counts=P[2] + 8) == select(work=P[0]) == select(counts=P[6]) == select(k_lens=P[3]) == INVALID


def test_attention_refusals(lib):
    def attend(**k):
        f = dict(q=P[0], k=P[1], v=P[2], out=P[3], index=P[4], counts=P[5], k_lens=P[6], q_start=P[7], batch=2, queries=300, keys=1000, q_heads=4, k_heads=2, lists=4,
                 head_dim=64, block=64, count=5, causal=0, softmax_scale=0.125, dtype=1)
        for a, n, h in (("q", 300, 4), ("k", 1000, 2), ("v", 1000, 2), ("o", 300, 4)):
            f.update({a + "_batch": n * h * 64, a + "_token": h * 64, a + "_head": 64})
        f.update(k)
        return lib.lyraq_sparse_attention(ctypes.byref(_lib.SparseAttentionArgs(**f)), None)
    assert lib.lyraq_sparse_attention(None, None) == INVALID
    assert attend(batch=0) == attend(queries=0) == attend(q_heads=0) == 0
    assert attend(o_batch=0) == attend(o_token=0) == attend(o_head=0) == INVALID
    for scale in (0.0, -1.0, float("inf"), float("nan"), 3e38):
        assert attend(softmax_scale=scale) == INVALID
    assert attend(k_heads=3) == attend(lists=1) == attend(count=-1) == attend(q=None) == attend(k=None) == attend(index=None) == attend(counts=None) == INVALID
    assert attend(q=P[0] + 2) == attend(out=P[3] + 8) == attend(k_token=130) == attend(v_head=1 << 40) == attend(counts=P[5] + 1) == INVALID
    assert attend(dtype=2) == attend(head_dim=80) == attend(block=32) == attend(keys=1 << 31) == attend(k_token=0) == attend(q_head=0) == UNSUPPORTED
    for at in (P[0], P[1] + 128, P[2] + 2 * 1000 * 128 * 2 - 128, P[4], P[5], P[6], P[7]):
        assert attend(out=at & ~15) == INVALID
