"""GPU tests of lyraq_rope_axes against its formula in 64 bits."""

import math

import pytest
import torch

from tests.util import check_status, cu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from lyradiff_b200 import ops as _ops
    return _ops


@pytest.fixture(scope="module")
def rope():
    from lyradiff_b200 import rope as _rope
    return _rope


def reference(x, pos, freq, axis, interleaved, norm, eps):
    """(rotated x, bound of what fp32 loses before the rounding): the norm's sum has at most 8 chained squares a lane (16 for 2 * VEC = 16) and
    5 levels, rsqrt 2 ulp: 32 * 2^-24 relative; cosine and sine are within 4 * 2^-24 + 2 pi 2^-26 of the angle's; three more roundings."""
    x = x.double()
    rel = 0.0
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
        rel = 32 * 2.0 ** -24
    ang = pos.double()[..., torch.tensor(axis, dtype=torch.long)] * torch.tensor(freq, dtype=torch.float64)
    c, s = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]
    n = len(freq)
    y, err = x.clone(), (rel + 2.0 ** -24) * x.abs()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    e = (rel + (4 + 2 * math.pi / 4 + 3) * 2.0 ** -24) * (a.abs() + b.abs())
    for o, v in ((0, a * c - b * s), (1, a * s + b * c)):
        at = slice(o, 2 * n, 2) if interleaved else slice(o * n, (o + 1) * n)
        y[..., at] = v
        err[..., at] = e
    return y, err


def assert_close(got, want, err):
    half = torch.finfo(got.dtype).eps / 2
    tol = err * (1 + half) + half * want.abs() + torch.finfo(got.dtype).tiny * half * 2
    d = (got.cpu().double() - want).abs()
    assert bool((d <= tol).all()), "off by %g of the tolerance" % float((d / tol).max())


def ladder(dims, theta=10000.0):
    return [theta ** (-2 * i / d) for d in dims for i in range(d // 2)], [a for a, d in enumerate(dims) for _ in range(d // 2)]


def positions(batch, seq, axes, dtype, start=0):
    g = torch.Generator().manual_seed(seq + axes)
    p = torch.randint(0, 100, (batch, seq, axes), generator=g) + start
    return p.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("batch,seq,hq,hk,d,dims", [(1, 1, 1, 1, 64, (64,)), (2, 7, 24, 24, 128, (16, 56, 56)), (1, 33, 24, 8, 128, (16, 24, 24)), (3, 5, 5, 2, 72, (24, 24, 24)),
                                                    (1, 9, 3, 3, 80, (80,)), (1, 300, 12, 12, 128, (44, 42, 42)), (1, 4, 40, 1, 256, (128, 128)), (2, 3, 2, 1, 72, (36,)),
                                                    (1, 2, 3, 2, 34, (10, 6)), (1, 5, 2, 2, 254, (84, 84, 84)), (1, 3, 2, 0, 128, ()), (1, 4800, 2, 1, 64, (32, 32)),
                                                    # few heads: tokens beside each other, the last block's in part
                                                    (3, 401, 1, 1, 128, (64,)), (1, 700, 3, 1, 80, (80,)), (1, 2503, 1, 0, 256, (128, 128)), (1, 4801, 1, 1, 2, (2,)),
                                                    (2, 5001, 1, 1, 72, (36,))])
def test_against_the_formula(ops, rope, dtype, interleaved, norm, batch, seq, hq, hk, d, dims):
    g = torch.Generator().manual_seed(d + seq)
    q, k = (torch.randn(batch, seq, h, d, generator=g).to(dtype) for h in (hq, hk))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype) if norm else None for _ in range(2))
    freq, axis = ladder(dims)
    pos = positions(batch, seq, len(dims), torch.int64)
    plan = rope.AxisRope(dims, interleaved=interleaved)
    kk = cu(k) if hk else None
    qo, ko = ops.rope_axes(plan, cu(pos), cu(q), kk, cu(wq), cu(wk) if hk else None, eps=1e-6)
    check_status()
    assert_close(qo, *reference(q, pos, freq, axis, interleaved, wq, 1e-6))
    if hk:
        assert_close(ko, *reference(k, pos, freq, axis, interleaved, wk, 1e-6))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_far_negative_and_fractional_positions(ops, rope, kind):
    dims = (32, 32)
    freq, axis = ladder(dims)
    at = [0, 1, -1, 3, 1000003, -77777, 2 ** 24 - 1, -(2 ** 23)]
    if kind == torch.float32:
        at += [0.5, -0.25, 1e-3, 7.75, 123456.5, 2.0 ** 30, 1e-30]
    elif kind == torch.int64:
        at += [2 ** 31 + 5, -(2 ** 33)]
    pos = torch.tensor(at, dtype=torch.float64).to(kind).reshape(1, -1, 1).expand(1, len(at), 2)
    q = torch.randn(1, len(at), 3, 64, generator=torch.Generator().manual_seed(1)).half()
    # the ladder itself in 64 bits: 2^-53 of the angle, at most 2^33 rad, in the reference
    got, _ = ops.rope_axes(rope.AxisRope(dims), pos.cuda(), cu(q))
    check_status()
    y, err = reference(q, pos, freq, axis, True, None, 1e-6)
    far = 2.0 ** -52 * pos.double().abs().amax(-1)[..., None, None] * 8
    assert_close(got, y, err + far * q.double().abs().amax())


def test_a_position_that_is_no_number_gives_nan_and_only_there(ops, rope):
    pos = torch.tensor([0.0, float("nan"), 2.0, float("inf")]).reshape(1, 4, 1).cuda()
    q = torch.ones(1, 4, 2, 96, dtype=torch.bfloat16, device="cuda")
    got, _ = ops.rope_axes(rope.AxisRope((64,)), pos, q)
    assert torch.isnan(got[0, [1, 3], :, :64]).all() and torch.isfinite(got[0, [0, 2]]).all() and (got[..., 64:] == 1).all()


@pytest.mark.parametrize("d,dims", [(128, (16, 56, 56)), (72, (36,))])
def test_layouts_and_in_place(ops, rope, d, dims):
    """Views of a packed projection, heads before tokens, rows that share nothing with 16 bytes, q and k turned where they lie."""
    g = torch.Generator().manual_seed(2)
    plan = rope.AxisRope(dims)
    pos = positions(2, 11, len(dims), torch.int32).cuda()
    qkv = torch.randn(2, 11, 3, 4, d, generator=g).bfloat16().cuda()
    q, k, v = qkv.unbind(2)
    want = ops.rope_axes(plan, pos, q.contiguous(), k.contiguous())
    split = ops.rope_axes(plan, pos, q, k)
    assert torch.equal(split[0], want[0]) and torch.equal(split[1], want[1])
    t = ops.rope_axes(plan, pos, q.transpose(1, 2).contiguous().transpose(1, 2), k)
    assert torch.equal(t[0], want[0])
    odd = torch.empty(2, 11, 4, d + 3, dtype=torch.bfloat16, device="cuda")[..., 1:d + 1]
    odd.copy_(q)
    assert torch.equal(ops.rope_axes(plan, pos, odd)[0], want[0])
    by_16 = torch.empty(2, 11, 4, d + 8, dtype=torch.bfloat16, device="cuda")[..., 8:]          # on 16 bytes, not on 32
    by_16.copy_(q)
    assert torch.equal(ops.rope_axes(plan, pos, by_16)[0], want[0])
    assert torch.equal(ops.rope_axes(plan, pos, q, q_out=q.new_zeros(2, 11, 4, d + 8)[..., 8:])[0], want[0])
    out = torch.zeros(2, 4, 11, d, dtype=torch.bfloat16, device="cuda")
    ops.rope_axes(plan, pos, q, q_out=out.transpose(1, 2))
    assert torch.equal(out.transpose(1, 2), want[0])
    v0 = v.clone()
    ops.rope_axes(plan, pos, q, k, q_out=q, k_out=k)
    check_status()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, v0)
    shared = ops.rope_axes(plan, pos[0], want[0], want[1])
    again = ops.rope_axes(plan, pos[:1].expand(2, -1, -1), want[0], want[1])
    assert torch.equal(shared[0], again[0]) and torch.equal(shared[1], again[1])
    by_axis = pos.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(ops.rope_axes(plan, by_axis, want[0])[0], ops.rope_axes(plan, pos, want[0])[0])


def test_agrees_with_the_table_form(ops, rope):
    """The packed FLUX call with its table in the tensors' type, three roundings more: within two ulp at the head's amplitude."""
    ids = rope.flux_position_ids(5, 4, 6)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(29, 3 * 4 * 128, generator=g).half().cuda()
    w = (1 + 0.2 * torch.randn(2, 128, generator=g)).half().cuda()
    table = rope.flux_rope_table(ids)[0, 0].half().cuda()
    old = torch.empty_like(qkv)
    ops.invoke_fused_rmsnorm_and_rope(old, qkv, w, table, 1e-6, 1, 29, 4, 128)
    x = qkv.reshape(1, 29, 3, 4, 128)
    q, k = ops.rope_axes(rope.AxisRope((16, 56, 56)), ids.cuda(), x[:, :, 0], x[:, :, 1], w[0], w[1])
    check_status()
    o = old.reshape(1, 29, 3, 4, 128)
    for a, b in ((q, o[:, :, 0]), (k, o[:, :, 1])):
        assert float((a.float() - b.float()).abs().max()) <= 4 * torch.finfo(torch.float16).eps * float(b.float().abs().max())


def test_sections_and_free_pairs(ops, rope):
    q = torch.randn(1, 6, 2, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    pos = positions(1, 6, 3, torch.int32)
    freq = [10000.0 ** (-i / 32) for i in range(32)]
    got, _ = ops.rope_axes(rope.AxisRope.sections((8, 12, 12)), cu(pos), cu(q))
    assert_close(got, *reference(q, pos, freq, [0] * 8 + [1] * 12 + [2] * 12, False, None, 1e-6))
    axis = [i % 3 for i in range(32)]
    got, _ = ops.rope_axes(rope.AxisRope.from_pairs([f / 4 for f in freq], axis, 3, interleaved=True), cu(pos), cu(q))
    assert_close(got, *reference(q, pos, [f / 4 for f in freq], axis, True, None, 1e-6))


def test_refusals(ops, rope):
    plan = rope.AxisRope((64,))
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(1, 4, 1, dtype=torch.int32, device="cuda")
    from lyradiff_b200._lib import LyraqError
    for args, kw in (((plan, pos.double(), q), {}), ((plan, pos[:, :3], q), {}), ((plan, pos.cpu(), q), {}), ((plan, pos, q[..., ::2]), {}), ((plan, pos, q.float()), {}),
                     ((plan, pos, q, q[:, :2]), {}), ((plan, pos, q), {"q_norm": q[0, 0, 0, :32]}), ((plan, pos, q), {"k_norm": q[0, 0, 0]}),
                     ((plan, pos, q), {"q_out": q[:, :, :1].expand(1, 4, 2, 64)}), ((plan, pos, q[0]), {}), ((rope.AxisRope((32, 32)), pos, q), {})):
        with pytest.raises((ValueError, TypeError, LyraqError)):
            ops.rope_axes(*args, **kw)
    with pytest.raises(LyraqError):
        ops.rope_axes(rope.AxisRope((66,)), pos, q)                   # more pairs than the head has
    with pytest.raises(LyraqError):
        ops.rope_axes(plan, pos, torch.zeros(1, 4, 1, 258, dtype=torch.bfloat16, device="cuda"))
    k = torch.zeros_like(q)
    for kw in ({"q_out": k}, {"k_out": q}, {"q_out": torch.empty_like(q)}):
        kw.setdefault("k_out", kw.get("q_out") if kw.get("q_out") is not k else None)
        with pytest.raises(LyraqError):
            ops.rope_axes(plan, pos, q, k, **kw)


def test_empty_calls(ops, rope):
    plan = rope.AxisRope((64,))
    q = torch.zeros(1, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    out, _ = ops.rope_axes(plan, torch.zeros(1, 0, 1, dtype=torch.int32, device="cuda"), q)
    assert out.shape == q.shape
    check_status()


def test_outputs_that_share_memory_with_what_is_read_are_refused(ops, rope):
    """Views one head or one token on, the other part of a packed projection, other strides at the same place; parts that nobody reads are taken."""
    from lyradiff_b200._lib import LyraqError
    g = torch.Generator().manual_seed(6)
    plan = rope.AxisRope((64,))
    pos = torch.arange(9, device="cuda").reshape(9, 1)
    buf = torch.randn(2 * 10 * 4 * 4 * 64, generator=g).bfloat16().cuda()
    qkv = buf[:2 * 9 * 4 * 4 * 64].view(2, 9, 4, 4, 64)        # q, k, v and a place
    q, k, v, place = qkv.unbind(2)
    want = ops.rope_axes(plan, pos, q.contiguous(), k.contiguous())
    before = buf.clone()
    by_head = qkv.view(-1)[:2 * 4 * 9 * 64].view(2, 4, 9, 64).transpose(1, 2)
    moved = lambda n: buf.as_strided(q.shape, q.stride(), n)   # noqa: E731
    for kw in ({"q_out": moved(64)}, {"q_out": moved(16 * 64)}, {"q_out": k}, {"k_out": q}, {"k_out": moved(5 * 64)}, {"q_out": by_head}, {"q_out": v, "k_out": v},
               {"q_out": v, "k_out": moved(9 * 64)}):
        with pytest.raises(LyraqError):
            ops.rope_axes(plan, pos, q, k, **kw)
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    got = ops.rope_axes(plan, pos, q, k, q_out=place, k_out=v)
    check_status()
    assert torch.equal(got[0], want[0]) and torch.equal(v, want[1]) and torch.equal(qkv[:, :, :2], before[:qkv.numel()].view_as(qkv)[:, :, :2])
    ops.rope_axes(plan, pos, q, q_out=q)
    ops.rope_axes(plan, pos, k, q_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
