"""CPU tests of what the calls of block-sparse attention refuse before they touch a device: lengths and places."""

import ctypes

import pytest
import torch

from lyradiff_b200 import _lib, build
from oracle import sparse

INVALID, UNSUPPORTED = 1, 2
P = [0x100000 + (i << 34) for i in range(10)]


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def select_args(**k):
    return {**dict(q_means=P[0], k_means=P[1], index=P[2], counts=P[3], k_lens=P[4], q_lens=P[5], q_start=P[6], batch=2, queries=300, keys=1000, q_heads=4, k_heads=2, lists=2,
                   head_dim=64, block=64, count=5, sink=0, window=0, causal=0), **k}


def test_query_lengths(lib):
    def select(**k):
        return lib.lyraq_select_blocks(ctypes.byref(_lib.SelectBlocksArgs(**select_args(**k))), P[7], 1 << 20, None)

    def attend(**k):
        f = dict(q=P[0], k=P[1], v=P[2], out=P[3], index=P[4], counts=P[5], k_lens=P[6], q_lens=P[7], q_start=P[8], batch=2, queries=300, keys=1000, q_heads=4, k_heads=2,
                 lists=4, head_dim=64, block=64, count=5, causal=0, softmax_scale=0.125, dtype=1)
        for a, n, h in (("q", 300, 4), ("k", 1000, 2), ("v", 1000, 2), ("o", 300, 4)):
            f.update({a + "_batch": n * h * 64, a + "_token": h * 64, a + "_head": 64})
        return lib.lyraq_sparse_attention(ctypes.byref(_lib.SparseAttentionArgs(**{**f, **k})), None)
    assert select(q_lens=P[5] + 2) == select(counts=P[5]) == select(q_lens=P[7] + 64) == select(q_lens=P[2] + 4) == INVALID
    assert attend(q_lens=P[7] + 1) == attend(out=P[7]) == INVALID


def test_blocks_beyond_30_bits(lib):
    """As the means: the distance of a place 2^30 in front of the keys to the end of a longer block does not fit 32 bits."""
    def select(**k):
        return lib.lyraq_select_blocks(ctypes.byref(_lib.SelectBlocksArgs(**select_args(**k))), P[7], 1 << 20, None)
    assert select(block=2 ** 31 - 1, causal=1) == select(block=2 ** 30 + 1) == UNSUPPORTED
    assert lib.lyraq_block_means(P[0], P[1], 1, 4096, 64, 32, None, 2 ** 30 + 1, 0, 2, 60, 2, 32, None) == UNSUPPORTED


def test_rows_behind_a_sequence_choose_nothing_and_for_no_one():
    """Two sequences of 520 and 700 tokens: the restatement's lists are those of each alone, whatever the rows behind hold."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 700, 2, 16, generator=g), torch.randn(2, 700, 2, 16, generator=g)
    lens = [520, 700]
    want = [sparse.select(sparse.means(q[b:b + 1, :n], 128), sparse.means(k[b:b + 1, :n], 64), 3, n, n, 64) for b, n in enumerate(lens)]
    for fill in (0.0, 9.0, float("nan")):
        q[0, 520:], k[0, 520:] = fill, fill
        index, counts = sparse.select(sparse.means(q, 128, lens), sparse.means(k, 64, lens), 3, 700, 700, 64, k_lens=lens, q_lens=lens)
        for b, n in enumerate(lens):
            blocks = sparse.blocks(n, 128)
            assert torch.equal(index[b, :, :blocks], want[b][0][0]) and torch.equal(counts[b, :, :blocks], want[b][1][0])
            assert bool((counts[b, :, blocks:] == 0).all()) and bool((index[b, :, blocks:] == -1).all())
