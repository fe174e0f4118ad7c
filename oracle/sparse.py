"""Attention over selected key blocks in 64 bits on the CPU: block means, selection, and the attention itself.

The reference's attention is dense; the definitions are the library's own (include/lyraq.h, lyraq_block_means, lyraq_select_blocks,
lyraq_sparse_attention).
"""

import math

import torch

QUERY_BLOCK = 128


def blocks(n, block):
    return (n + block - 1) // block


def means(x, block, lens=None):
    """x [batch, tokens, heads, dim] -> fp32 [batch, heads, blocks, dim]."""
    batch, n, heads, dim = x.shape
    out = torch.zeros(batch, heads, blocks(n, block), dim)
    for b in range(batch):
        end = n if lens is None else min(max(int(lens[b]), 0), n)
        for j in range(blocks(end, block)):
            out[b, :, j] = x[b, j * block:min(end, (j + 1) * block)].double().mean(0).float()
    return out


def select(q_means, k_means, count, queries, keys, block, k_lens=None, q_start=None, causal=False, sink=0, window=0, shared=False, q_lens=None):
    """One query block after the other, by sorting (score, -index)."""
    batch, heads, qb, _ = q_means.shape
    k_heads, kb = k_means.shape[1:3]
    lists, group = (k_heads if shared else heads), heads // k_heads
    index = torch.full((batch, lists, qb, count), -1, dtype=torch.int32)
    counts = torch.zeros(batch, lists, qb, dtype=torch.int32)
    for b in range(batch):
        n = keys if k_lens is None else min(max(int(k_lens[b]), 0), keys)
        start = keys - queries if q_start is None else int(q_start[b])
        nq = queries if q_lens is None else min(max(int(q_lens[b]), 0), queries)
        for h in range(lists):
            if shared:
                q, k = q_means[b, h * group:(h + 1) * group].double().sum(0), k_means[b, h].double()
            else:
                q, k = q_means[b, h].double(), k_means[b, h // group].double()
            scores = (q @ k.t()).float()
            for i in range(blocks(nq, QUERY_BLOCK)):
                first = start + i * QUERY_BLOCK
                last = first + min(QUERY_BLOCK, nq - i * QUERY_BLOCK) - 1
                rank = []
                for j in range(kb):
                    if j * block >= n or (causal and j * block > last):
                        continue
                    forced = j < sink or (window > 0 and first // block - (window - 1) <= j <= last // block + (window - 1))
                    s = float(scores[i, j])
                    rank.append((not forced, 0.0 if forced else math.inf if math.isnan(s) else -s, j))
                got = sorted(j for *_, j in sorted(rank)[:count])
                counts[b, h, i] = len(got)
                index[b, h, i, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return index, counts


def attend(q, k, v, index, counts, block, k_lens=None, q_start=None, causal=False, scale=None, q_lens=None):
    """Key by key as the lists name them (a block listed twice counts twice); also returns what bounds the rounding of the weights: the sum of |weight * value|."""
    batch, nq, heads, dim = q.shape
    nk, k_heads = k.shape[1:3]
    scale = dim ** -0.5 if scale is None else scale
    per, group = heads // index.shape[1], heads // k_heads
    out = torch.zeros(batch, nq, heads, dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(batch):
        n = nk if k_lens is None else min(max(int(k_lens[b]), 0), nk)
        start = nk - nq if q_start is None else int(q_start[b])
        end = nq if q_lens is None else min(max(int(q_lens[b]), 0), nq)
        for h in range(heads):
            for i in range(index.shape[2]):
                lists = index[b, h // per, i, :max(0, min(int(counts[b, h // per, i]), index.shape[3]))].tolist()
                pos = [p for j in lists if 0 <= j < blocks(nk, block) for p in range(j * block, min((j + 1) * block, n))]
                rows = torch.arange(min(end, i * QUERY_BLOCK), min(end, (i + 1) * QUERY_BLOCK))
                if not pos or not len(rows):
                    continue
                at = torch.tensor(pos)
                s = q[b, rows, h].double() @ k[b, at, h // group].double().t() * scale
                if causal:
                    s = s.masked_fill(at[None] > start + rows[:, None], -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                den = p.sum(-1, keepdim=True)
                w = p / torch.where(den == 0, 1.0, den)
                out[b, rows, h] = w @ v[b, at, h // group].double()
                mag[b, rows, h] = w @ v[b, at, h // group].double().abs()
    return out, mag
