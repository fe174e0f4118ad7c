"""Operators of transformer blocks over long sequences, as measurable cases: the FP8 linear with a scale for each block of 128, and attention
over the key blocks that a cheap score selects, with the selection itself.

A case is a dict of plain values; "kind" picks the operator, the rest are sizes and options:

  linear   quantize of x [m, k] (a scale for 128 values of a row) and product with a quantized weight [n, k] (a scale for 128 x 128 values)
                                                                          m, n, k, gelu, residual, dtype
  select   means of query and key blocks, their products, the `count` key blocks with the largest for each 128 queries
           cached: the key means are at hand but for the last block, which the newest token has changed
  attend   attention of q over selected key blocks of `block` tokens
  sparse   select and attend in one call
                                                                          batch, nq, nk, q_heads, k_heads, head_dim, block, count, sink, window,
                                                                          shared (one list for the query heads of a key head), causal, lens
                                                                          (sequences of unequal length), packed (q, k, v in one tensor), dtype

Where `own` is false run() computes the plain form with elementary torch operations in 32 bits (scores that decide a selection: in 64); where it
is true it makes the calls that a user of this library makes.  exact() restates the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROWS = 128          # queries that share a list of key blocks
LEAST = 2.0 ** -100   # the smallest scale of an FP8 block


def _attn(name, kind, batch, nq, nk, q_heads, k_heads, head_dim, block, count, sink=0, window=0, shared=False, causal=False, lens=False, packed=False,
          cached=False, dtype="bf16"):
    case = {"kind": kind, "batch": batch, "nq": nq, "nk": nk, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim, "block": block,
            "count": count, "sink": sink, "window": window, "shared": shared, "causal": causal, "lens": lens, "packed": packed, "cached": cached,
            "dtype": dtype}
    return case if name is None else {"name": name, **case}


def _linear(name, m, n, k, gelu=False, residual=False, dtype="bf16"):
    case = {"kind": "linear", "m": m, "n": n, "k": k, "gelu": gelu, "residual": residual, "dtype": dtype}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The modulation linear of a block, or one new token: a single row against 26 million weights.  The weight stream and latency.
        _linear("fp8b_one_row", 1, 5120, 5120),
        # Key/value projection of the text in cross attention: 2 x 77 tokens, a small matrix.
        _linear("fp8b_text", 154, 1280, 2048, dtype="fp16"),
        # Feed-forward output linear over an odd number of tokens with its residual.
        _linear("fp8b_ragged", 1317, 1280, 5120, residual=True, dtype="fp16"),
        # The feed-forward's first linear over the tokens of a short clip: the largest linear.
        _linear("fp8b_mlp", 4680, 13824, 5120, gelu=True),
        # Selection for a video clip of 21 latent frames of 30 x 52 patches: 256 query blocks against 512 key blocks in each of 12 heads.
        _attn("select_video", "select", 1, 32760, 32760, 12, 12, 128, 64, 64, window=1, packed=True),
        # The next token of four long sequences: the newest key's block mean, one query against 512 key blocks, a list for each key head.
        _attn("select_decode", "select", 4, 1, 32768, 32, 8, 128, 64, 64, sink=1, window=2, shared=True, lens=True, cached=True),
        # One query over a short memory: nothing but latency.
        _attn("attend_one", "attend", 1, 1, 1000, 8, 8, 64, 64, 4, dtype="fp16"),
        # The next token of eight long sequences, four query heads to a key head: a gather of keys and values.
        _attn("attend_decode", "attend", 8, 1, 32768, 32, 8, 128, 64, 64, sink=1, window=2, shared=True, lens=True),
        # A chunk of new tokens behind a long prefix, causal.
        _attn("attend_chunk", "attend", 1, 1024, 17408, 32, 8, 128, 128, 32, sink=1, window=2, causal=True),
        # Two images of unequal odd size in one padded batch, heads of 64.
        _attn("attend_ragged", "attend", 2, 4429, 4429, 20, 20, 64, 128, 12, lens=True, packed=True, dtype="fp16"),
        # The attention of the video clip, an eighth of the keys: the largest.
        _attn("attend_video", "attend", 1, 32760, 32760, 12, 12, 128, 64, 64, window=1, packed=True),
        # A block over 512 text and 4096 image tokens, q, k and v as the projection writes them, a quarter of the keys: selection and attention together.
        _attn("sparse_image", "sparse", 1, 4608, 4608, 24, 24, 128, 64, 18, sink=8, window=1, packed=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges; costs no more than the largest listed one."""
    dtype = rng.choice(["bf16", "fp16"])
    kind = rng.choice(["linear", "linear", "select", "attend", "attend", "sparse"])
    if kind == "linear":
        while True:
            m, n, k = _log(rng, 1, 4680), _log(rng, 64, 13824), 16 * _log(rng, 8, 864)
            n = n if rng.random() < 0.3 else (n + 7) // 8 * 8
            if m * n * k <= 4680 * 13824 * 5120:
                return _linear(None, m, n, k, rng.random() < 0.4, rng.random() < 0.4, dtype)
    head_dim, block = rng.choice([64, 128, 128]), rng.choice([64, 64, 128])
    lens, shared = rng.random() < 0.4, rng.random() < 0.5
    sink, window = rng.choice([0, 1, 3]), rng.choice([0, 1, 2])
    if rng.random() < 0.4:   # new tokens over a cache
        batch, k_heads = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 8])
        q_heads = k_heads * rng.choice([1, 4, 8])
        nk = _log(rng, 1, 32768)
        nq = min(nk, rng.choice([1, 1, 1, 2, _log(rng, 3, 1024)]))
        cached = kind == "select" and nq == 1
        count = _log(rng, 1, min(64, max(1, 4096 // block)))
        return _attn(None, kind, batch, nq, nk, q_heads, k_heads, head_dim, block, count, sink, window, shared, not lens and rng.random() < 0.5, lens,
                     False, cached, dtype)
    batch, heads = rng.choice([1, 1, 2]), rng.choice([4, 10, 12, 20, 24])
    n = _log(rng, 100, 32760 * 12 // (batch * max(heads, 12)))
    count = _log(rng, 1, 4096 // block)
    return _attn(None, kind, batch, n, n, heads, heads, head_dim, block, count, sink, window, shared, rng.random() < 0.3, lens, rng.random() < 0.7, False,
                 dtype)


# ----------------------------------------------------------------------------- inputs
def _activations(g, shape, dtype):
    """N(0, 1) with some channels several times as large, as the streams of a transformer have them."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 1 + 5 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.02).float()
    return x.to(dtype)


def _tokens(g, batch, n, heads, dim, dtype):
    """[batch, n, heads, dim]: noise over a walk that neighbouring tokens share, so that blocks differ and near ones are alike."""
    x = torch.randn(batch, n, heads, dim, generator=g, device="cuda", dtype=dtype)
    steps = (n + 31) // 32
    walk = torch.randn(batch, steps, heads, dim, generator=g, device="cuda").cumsum(1) / math.sqrt(steps)
    return x + walk.to(dtype).repeat_interleave(32, dim=1)[:, :n]


def _blocks(n, block):
    return (n + block - 1) // block


def _allowed(case, k_lens):
    """[batch, query blocks, key blocks]: key blocks that hold a key that some query of the block may see; and those taken in any case."""
    nq, nk, block = case["nq"], case["nk"], case["block"]
    lens = torch.full((case["batch"],), nk, device="cuda") if k_lens is None else k_lens.long()
    start = nk - nq if k_lens is None or nq == nk else lens - nq
    i, j = torch.arange(_blocks(nq, ROWS), device="cuda"), torch.arange(_blocks(nk, block), device="cuda")
    first = torch.zeros_like(lens)[:, None] + (start if isinstance(start, int) else start[:, None]) + i * ROWS
    last = first + (nq - i * ROWS).clamp_max(ROWS) - 1
    ok = (j * block < lens[:, None])[:, None, :]
    if case["causal"]:
        ok = ok & (j * block <= last[:, :, None])
    forced = j[None, None, :].expand(ok.shape[0], last.shape[1], -1) < case["sink"]
    if case["window"]:
        w = case["window"] - 1
        low, high = torch.div(first, block, rounding_mode="floor") - w, torch.div(last, block, rounding_mode="floor") + w
        forced = forced | ((j >= low[:, :, None]) & (j <= high[:, :, None]))
    ok = ok.expand(-1, last.shape[1], -1)
    return ok, forced & ok


def _pick(scores, ok, forced, count):
    """scores [batch, heads, query blocks, key blocks] fp32: the largest `count` of the allowed, ties to the lowest, in ascending order."""
    s = torch.where(forced[:, None], math.inf, scores)
    s = torch.where(ok[:, None], s, -math.inf)
    count_in = min(count, s.shape[-1])
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :count_in]
    have = ok.sum(-1, dtype=torch.int32).clamp_max(count_in)[:, None].expand(s.shape[:3])
    slot = torch.arange(count_in, device=s.device)
    big = s.shape[-1]
    index = torch.sort(torch.where(slot < have[..., None], order, big), dim=-1).values
    index = torch.where(index == big, -1, index).to(torch.int32)
    if count_in < count:
        index = torch.cat([index, index.new_full((*index.shape[:3], count - count_in), -1)], dim=-1)
    return index.contiguous(), have.contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 54321)
    T = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _activations(g, (m, k), T)
        # rows of a weight matrix differ in size
        s["w"] = (torch.randn(n, k, generator=g, device="cuda") * 0.02 * (0.5 + torch.rand(n, 1, generator=g, device="cuda"))).to(T)
        s["bias"] = (torch.randn(n, generator=g, device="cuda") * 0.02).to(T)
        s["residual"] = torch.randn(m, n, generator=g, device="cuda").to(T) if case["residual"] else None
        return s
    batch, nq, nk, hq, hk, dim = (case[key] for key in ("batch", "nq", "nk", "q_heads", "k_heads", "head_dim"))
    if case["packed"]:   # as one projection writes them
        s["q"], s["k"], s["v"] = _tokens(g, batch, nq, 3 * hq, dim, T).unflatten(2, (3, hq)).unbind(2)
    else:                # a cache keeps the tokens of a head together
        s["q"] = _tokens(g, batch, nq, hq, dim, T)
        s["k"] = _tokens(g, batch, nk, hk, dim, T).transpose(1, 2).contiguous().transpose(1, 2)
        s["v"] = _tokens(g, batch, nk, hk, dim, T).transpose(1, 2).contiguous().transpose(1, 2)
    s["k_lens"] = None
    if case["lens"]:
        least = max(1, nk * 3 // 4, nq if case["causal"] else 1)
        s["k_lens"] = torch.randint(least, nk + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
        s["k_lens"][-1] = nk
    # where the queries stand: behind the cache, or each at its own key
    s["q_start"] = None if s["k_lens"] is None or nq == nk else (s["k_lens"] - nq)
    if case["cached"]:
        s["k_means"] = _means(s["k"], case["block"], s["k_lens"])
    if case["kind"] == "attend":
        heads = hk if case["shared"] else hq
        scores = torch.randn(batch, heads, _blocks(nq, ROWS), _blocks(nk, case["block"]), generator=g, device="cuda")
        s["index"], s["counts"] = _pick(scores, *_allowed(case, s["k_lens"]), case["count"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from lyradiff_b200.layers import Fp8BlockLinear, SparseAttention
        if "k_means" in s:
            s["k_means"] = s["k_means"].contiguous()   # as ops.block_means returns them
        if case["kind"] == "linear":
            s["layer"] = Fp8BlockLinear.from_float(s["w"], s["bias"], gelu=case["gelu"])
        elif case["kind"] == "sparse":
            s["layer"] = SparseAttention(case["block"], case["count"], sink=case["sink"], window=case["window"], shared=case["shared"],
                                         causal=case["causal"])
    elif case["kind"] == "linear":
        w = s["w"].float()
        n, k = w.shape
        pad = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).unflatten(1, (-1, 128)).unflatten(0, (-1, 128))
        s["w_plain"] = _plain_fp8(pad, (1, 3)).flatten(2, 3).flatten(0, 1)[:n, :k].contiguous()
    return s


# ----------------------------------------------------------------------------- the plain form
def _plain_fp8(b, dims):
    """Blocks over `dims` through FP8: the scale is the largest magnitude over 448, a code the e4m3 number next to the value over the scale, both
    quotients rounded to 32 bits (a quotient by a tensor: one by a number is a product with its reciprocal)."""
    scale = (b.abs().amax(dim=dims, keepdim=True) / torch.full((1,), 448.0, device=b.device)).clamp_min(LEAST)
    return (b / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * scale


def _plain_linear(s):
    x = s["x"].float()
    k = x.shape[1]
    x = _plain_fp8(torch.nn.functional.pad(x, (0, -k % 128)).unflatten(1, (-1, 128)), -1).flatten(1)[:, :k]
    y = torch.matmul(x, s["w_plain"].t())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y + s["bias"].float()
    if s["case"]["gelu"]:
        y = y * torch.sigmoid(1.5957691216057308 * (y + 0.044715 * y * y * y))   # 0.5 y (1 + tanh) without the cancellation of its sum
    return y.to(s["x"].dtype)


def _means(x, block, lens=None):
    """[batch, heads, blocks, dim] fp32: means of the tokens of a block that exist, 0 where none does; sums in 64 bits, next to a border they decide."""
    n = x.shape[1]
    pos = torch.arange(_blocks(n, block) * block, device=x.device)
    there = pos < (torch.full((x.shape[0], 1), n, device=x.device) if lens is None else lens[:, None])
    y = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -n % block))
    y = torch.where(there[:, :, None, None], y, 0.0).unflatten(1, (-1, block)).sum(2, dtype=torch.float64)
    return (y / there.unflatten(1, (-1, block)).sum(2).clamp_min(1)[:, :, None, None]).float().transpose(1, 2)


def _plain_select(s):
    case = s["case"]
    qm = _means(s["q"], ROWS).double()
    if case["cached"]:
        km = s["k_means"]
        at = torch.arange(case["batch"], device=km.device)
        n = torch.full_like(at, case["nk"]) if s["k_lens"] is None else s["k_lens"].long()
        j = (n - 1) // case["block"]   # the block of the newest token
        pos = j[:, None] * case["block"] + torch.arange(case["block"], device=km.device)
        there = pos < n[:, None]
        last = s["k"][at[:, None], pos.clamp_max(case["nk"] - 1)].double()
        km[at, :, j] = (torch.where(there[..., None, None], last, 0.0).sum(1) / there.sum(1)[:, None, None]).float()
    else:
        km = _means(s["k"], case["block"], s["k_lens"])
    group = case["q_heads"] // case["k_heads"]
    q = qm.unflatten(1, (case["k_heads"], group))
    if case["shared"]:
        scores = torch.matmul(q.sum(2), km.double().transpose(-1, -2))
    else:
        scores = torch.matmul(q, km.double().transpose(-1, -2)[:, :, None]).flatten(1, 2)
    return (*_pick(scores.float(), *_allowed(case, s["k_lens"]), case["count"]), km)


def _plain_attend(s, index):
    case = s["case"]
    q, k, v, block = s["q"], s["k"], s["v"], case["block"]
    batch, nq, hq, dim = q.shape
    nk, group, per = case["nk"], case["q_heads"] // case["k_heads"], case["q_heads"] // index.shape[1]
    qb, rows = index.shape[2], min(nq, ROWS)
    lens = torch.full((batch,), nk, device=q.device) if s["k_lens"] is None else s["k_lens"]
    start = torch.full((batch,), nk - nq, device=q.device) if s["q_start"] is None else s["q_start"]
    pad = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, qb * rows - nq))
    out = torch.empty(batch * hq, qb * rows, dim, dtype=q.dtype, device=q.device)
    # as many heads at a time as 2^28 gathered values hold
    for part in torch.arange(batch * hq, device=q.device).split(max(1, 2 ** 28 // (qb * case["count"] * block * dim))):
        b, h = part // hq, part % hq
        idx = index[b, h // per].long()                                                              # [heads, query blocks, count]
        pos = (idx.clamp_min(0)[..., None] * block + torch.arange(block, device=q.device)).flatten(2)   # [heads, query blocks, keys]
        there = (idx >= 0)[..., None].expand(-1, -1, -1, block).flatten(2) & (pos < lens[b][:, None, None])
        at = (b[:, None, None], pos.clamp_max(nk - 1), (h // group)[:, None, None])
        kk = torch.where(there[..., None], k[at].float(), 0.0)
        sc = torch.matmul(pad[b, :, h].float().unflatten(1, (qb, rows)), kk.transpose(-1, -2)) * dim ** -0.5
        del kk
        see = there[:, :, None]
        if case["causal"]:
            i = start[b][:, None] + torch.arange(qb * rows, device=q.device)
            see = see & (pos[:, :, None] <= i.unflatten(1, (qb, rows))[..., None])
        sc = torch.where(see, sc, -math.inf)
        top = sc.amax(-1, keepdim=True)
        sc = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
        den = sc.sum(-1, keepdim=True)
        o = torch.matmul(sc, torch.where(there[..., None], v[at].float(), 0.0)) / torch.where(den > 0, den, 1.0)
        out[part] = o.flatten(1, 2).to(q.dtype)
    return out.unflatten(0, (batch, hq))[:, :, :nq].transpose(1, 2)


# ----------------------------------------------------------------------------- one pass
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        return _own(s, s["case"], kind)
    if kind == "linear":
        return _plain_linear(s)
    if kind == "select":
        return _plain_select(s)
    if kind == "attend":
        return _plain_attend(s, s["index"])
    index, counts, _ = _plain_select(s)
    return _plain_attend(s, index), index, counts


def _own(s, case, kind):
    from lyradiff_b200 import ops
    if kind == "linear":
        return s["layer"].forward(s["x"], residual=s["residual"])
    if kind == "sparse":
        out, index, counts = s["layer"].forward(s["q"], s["k"], s["v"], k_lens=s["k_lens"], q_start=s["q_start"], with_selection=True)
        return out, index, counts
    if kind == "select":
        q_means = ops.block_means(s["q"], ROWS)
        if case["cached"]:
            k_means = ops.block_means(s["k"], case["block"], lens=s["k_lens"], out=s["k_means"], newest=1)
        else:
            k_means = ops.block_means(s["k"], case["block"], lens=s["k_lens"])
        index, counts = ops.select_blocks(q_means, k_means, case["count"], queries=case["nq"], keys=case["nk"], block=case["block"],
                                          k_lens=s["k_lens"], q_start=s["q_start"], causal=case["causal"], sink=case["sink"],
                                          window=case["window"], shared=case["shared"])
        return index, counts, k_means
    return ops.sparse_attention(s["q"], s["k"], s["v"], s["index"], s["counts"], case["block"], k_lens=s["k_lens"], q_start=s["q_start"],
                                causal=case["causal"])


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        weight = n * k + 4 * _blocks(n, 128) * _blocks(k, 128)
        return {"bytes": 2 * m * k + weight + 2 * n + 2 * m * n * (2 if case["residual"] else 1), "flops": 2 * m * n * k}
    batch, nq, nk, hq, hk, dim, block = (case[key] for key in ("batch", "nq", "nk", "q_heads", "k_heads", "head_dim", "block"))
    qb, kb = _blocks(nq, ROWS), _blocks(nk, block)
    lists = hk if case["shared"] else hq
    take = min(case["count"], kb)
    listed_bytes = 4 * batch * lists * qb * (case["count"] + 1)
    means = 4 * batch * hk * kb * dim
    total = {"bytes": 0, "flops": 0}
    if case["kind"] in ("select", "sparse"):
        keys = block if case["cached"] else nk
        total["bytes"] += 2 * batch * nq * hq * dim + 2 * batch * keys * hk * dim + listed_bytes
        if case["kind"] == "select":
            total["bytes"] += means
        total["flops"] += batch * (nq * hq + keys * hk) * dim + 2 * batch * lists * qb * kb * dim
    if case["kind"] in ("attend", "sparse"):
        # each key head's tokens once, but no more than the lists can name
        tokens = min(nk, qb * (lists // hk) * take * block)
        if case["kind"] == "attend":
            total["bytes"] += 2 * batch * nq * hq * dim + 2 * batch * tokens * hk * dim + listed_bytes
        total["bytes"] += 2 * batch * nq * hq * dim + 2 * batch * tokens * hk * dim
        total["flops"] += 4 * batch * nq * hq * dim * min(nk, take * block)
    return total


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _exact_e4m3(t):
    """Nearest e4m3 value, ties to the even code; |t| up to 448 and a rounding of it."""
    a = t.abs().clamp_max(448.0)
    # of a number in [2^e, 2^(e + 1)) the codes lie 2^(e - 3) apart, of all below 2^-6 as there
    step = torch.exp2(torch.frexp(a).exponent.clamp_min(-5).double() - 4)
    return torch.round(a / step) * step * torch.sign(t)


def _exact_fp8(x, rows, cols):
    """x [n, k] in blocks of rows x cols; scales and quotients are rounded to 32 bits, as the format is defined."""
    out = torch.empty_like(x)
    n, k = x.shape
    for c in range(0, k, cols):
        part = x[:, c:c + cols]
        top = part.abs().amax(dim=1)
        if rows > 1:
            top = torch.stack([t.max() for t in top.split(rows)]).repeat_interleave(rows)[:n]
        scale = (top / 448).float().double().clamp_min(LEAST)[:, None]
        out[:, c:c + cols] = _exact_e4m3((part / scale).float().double()) * scale
    return out


def _exact_mean(x, block, lens):
    """[batch, heads, blocks, dim]"""
    batch, n, heads, dim = x.shape
    out = torch.zeros(batch, heads, _blocks(n, block), dim, dtype=torch.float64, device=x.device)
    for b in range(batch):
        end = n if lens is None else int(lens[b])
        whole = end // block
        if whole:
            out[b, :, :whole] = x[b, :whole * block].double().reshape(whole, block, heads, dim).mean(1).permute(1, 0, 2)
        if end % block:
            out[b, :, whole] = x[b, whole * block:end].double().mean(0)
    return out.float().double()


def _exact_select(s):
    case = s["case"]
    qm, km = _exact_mean(s["q"], ROWS, None), _exact_mean(s["k"], case["block"], s["k_lens"])
    group = case["q_heads"] // case["k_heads"]
    if case["shared"]:
        qm = qm.reshape(case["batch"], case["k_heads"], group, -1, case["head_dim"]).sum(2)
    else:
        km = km.repeat_interleave(group, dim=1)
    scores = torch.einsum("bhqd,bhkd->bhqk", qm, km).float()
    if not case["shared"]:
        km = km[:, ::group]
    ok, forced = _allowed(case, s["k_lens"])
    # rank of every block: how many come before it
    scores = scores.masked_fill(forced[:, None], math.inf)
    batch, heads, qb, kb = scores.shape
    index = torch.full((batch, heads, qb, case["count"]), -1, dtype=torch.int32, device=scores.device)
    counts = torch.zeros(batch, heads, qb, dtype=torch.int32, device=scores.device)
    place = torch.arange(kb, device=scores.device)
    for b in range(batch):
        for h in range(heads):
            v = scores[b, h].masked_fill(~ok[b], -math.inf)
            rank = torch.argsort(torch.argsort(v, dim=-1, descending=True, stable=True), dim=-1, stable=True)
            taken = ok[b] & (rank < case["count"])
            counts[b, h] = taken.sum(-1)
            nth = torch.cumsum(taken, -1) - 1
            r, c = taken.nonzero(as_tuple=True)
            index[b, h, r, nth[r, c]] = place[c].to(torch.int32)
    return index, counts, km.float() if case["kind"] == "select" else None


def _exact_attend(s, index):
    """Softmax over all keys with the mask that the lists, the lengths and the order leave."""
    case = s["case"]
    batch, nq, hq, dim = s["q"].shape
    nk, block = case["nk"], case["block"]
    kb, per, group = _blocks(nk, block), hq // index.shape[1], hq // case["k_heads"]
    out = torch.empty(batch, nq, hq, dim, dtype=torch.float64, device=s["q"].device)
    key = torch.arange(nk, device=s["q"].device)
    for b in range(batch):
        end = nk if s["k_lens"] is None else int(s["k_lens"][b])
        start = nk - nq if s["q_start"] is None else int(s["q_start"][b])
        for h in range(hq):
            lists = index[b, h // per].long()
            marks = torch.zeros(lists.shape[0], kb + 1, dtype=torch.bool, device=lists.device)
            marks.scatter_(1, torch.where(lists < 0, kb, lists), True)
            k, v = s["k"][b, :, h // group].double(), s["v"][b, :, h // group].double()
            v = v.masked_fill((key >= end)[:, None], 0.0)
            for r in range(0, nq, 4096):
                i = torch.arange(r, min(nq, r + 4096), device=lists.device)
                see = marks[i // ROWS][:, key // block] & (key < end)
                if case["causal"]:
                    see &= key <= start + i[:, None]
                z = (s["q"][b, i, h].double() @ k.T / math.sqrt(dim)).masked_fill_(~see, -math.inf)
                out[b, i, h] = torch.softmax(z, dim=-1).nan_to_num(0.0) @ v
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "linear":
        y = _exact_fp8(s["x"].double(), 1, 128) @ _exact_fp8(s["w"].double(), 128, 128).T + s["bias"].double()
        if s["residual"] is not None:
            y += s["residual"].double()
        return y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))) if case["gelu"] else y
    if case["kind"] == "select":
        return _exact_select(s)
    if case["kind"] == "attend":
        return _exact_attend(s, s["index"])
    index, counts, _ = _exact_select(s)
    return _exact_attend(s, index), index, counts
