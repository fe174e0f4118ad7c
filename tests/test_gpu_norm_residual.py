"""GPU tests of lyraq_gated_residual_norm against its formula in 64 bits."""

import pytest
import torch

from tests.util import check_status, cu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from lyradiff_b200 import ops as _ops
    return _ops


def make(batch, seq, dim, dtype, seed, mod=True, weights=True, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    t = {"y": torch.randn(batch, seq, dim, generator=g) * 2 + mean, "x": torch.randn(batch, seq, dim, generator=g) * 3 - mean}
    if mod:
        for n in ("gate", "scale", "shift"):
            t[n] = torch.randn(batch, dim, generator=g) * 0.5
    if weights:
        for n in ("post_weight", "pre_weight"):
            t[n] = 1 + 0.3 * torch.randn(dim, generator=g)
    return {k: v.to(dtype) for k, v in t.items()}


def reference(t, post, pre, r, eps):
    """(v, h) in 64 bits and bounds of what fp32 may lose before the one rounding of each.  Every sum of a row has at most 8 * 4 terms a thread
    in a chain, 5 levels of a warp and 16 warps: 53 roundings, taken as 64 with those of the elementwise steps, each 2^-24 of the sum of
    magnitudes; rsqrt adds 2 ulp."""
    d = {k: v.double() for k, v in t.items()}
    u = 64 * 2.0 ** -24

    def normed(v, err, kind):
        if kind == "none":
            return v, err
        m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
        dm = err.mean(-1, keepdim=True) + u * v.abs().mean(-1, keepdim=True) if kind == "layer" else m
        c, dc = v - m, err + dm
        inv = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
        rel = (c.abs() * dc).mean(-1, keepdim=True) * inv ** 2 + u
        return c * inv, dc * inv + (c * inv).abs() * rel
    n, dn = normed(d["y"], torch.zeros_like(d["y"]), post)
    f = d.get("post_weight", torch.ones(1).double()) * (d["gate"].unsqueeze(1) if "gate" in d else 1.0)
    v = r * d["x"] + n * f
    dv = dn * f.abs() + 4 * 2.0 ** -24 * ((r * d["x"]).abs() + (n * f).abs())
    n2, dn2 = normed(v, dv, pre)
    f2 = d.get("pre_weight", torch.ones(1).double()) * (1 + d["scale"].unsqueeze(1) if "scale" in d else 1.0)
    s = d["shift"].unsqueeze(1) if "shift" in d else 0.0
    h = n2 * f2 + s
    dh = dn2 * f2.abs() + 6 * 2.0 ** -24 * ((n2 * f2).abs() + (s.abs() if "shift" in d else 0.0))
    return v, dv, h, dh


def assert_close(got, want, err):
    half = torch.finfo(got.dtype).eps / 2
    tol = err * (1 + half) + half * want.abs() + torch.finfo(got.dtype).tiny * half * 2
    d = (got.cpu().double() - want).abs()
    assert bool((d <= tol).all()), "off by %g of the tolerance" % float((d / tol).max())


CASES = [("none", "rms"), ("rms", "rms"), ("layer", "layer"), ("rms", "layer"), ("layer", "rms"), ("none", "layer")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("post,pre", CASES)
@pytest.mark.parametrize("batch,seq,dim", [(1, 1, 8), (2, 3, 64), (3, 5, 264), (1, 400, 256), (2, 200, 640), (1, 333, 1024), (1, 2, 1280), (2, 170, 1288),
                                           (1, 3, 3072), (1, 310, 3072), (2, 2, 8192), (1, 300, 8200), (1, 2, 16384), (1, 301, 16384)])
def test_against_the_formula(ops, dtype, post, pre, batch, seq, dim):
    t = make(batch, seq, dim, dtype, batch + seq + dim)
    v, dv, h, dh = reference(t, post, pre, 0.75, 1e-5)
    xo, ho = ops.gated_residual_norm(post=post, pre=pre, residual_scale=0.75, eps=1e-5, **{k: cu(a) for k, a in t.items()})
    check_status()
    assert_close(xo, v, dv)
    assert_close(ho, h, dh)


@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms")])
@pytest.mark.parametrize("rows,dim", [(889, 768), (901, 1000), (890, 1280), (1201, 1096), (9473, 1280), (3, 1536), (320, 1536), (1200, 2048),
                                      (1200, 4096), (300, 2560)])
def test_every_way_of_dealing_a_row_to_threads(ops, post, pre, rows, dim):
    """Three, four and five vectors a lane of a warp, whole and in part, a block where there are more rows than warps with five pay for, blocks of one to
    four vectors a thread without absent ones; the quantized outputs are those of the separate calls."""
    t = make(1, rows, dim, torch.bfloat16, rows)
    v, dv, h, dh = reference(t, post, pre, 0.75, 1e-5)
    dev = {k: cu(a) for k, a in t.items()}
    xo, ho = ops.gated_residual_norm(post=post, pre=pre, residual_scale=0.75, eps=1e-5, **dev)
    check_status()
    assert_close(xo, v, dv)
    assert_close(ho, h, dh)
    if dim % 32 == 0:
        for fmt in ("nvfp4", "mxfp4"):
            q = ops.Fp4Tensor.empty(rows, dim, fmt)
            ops.gated_residual_norm(post=post, pre=pre, residual_scale=0.75, eps=1e-5, q4=q, **dev)
            want = ops.quant_fp4(ho[0], None, fmt, ops.Fp4Tensor(rows, dim, fmt, torch.empty_like(q.codes), q.scales.clone()))
            assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)


@pytest.mark.parametrize("post,pre", CASES)
def test_without_modulation_and_weights(ops, post, pre):
    t = make(2, 9, 320, torch.float16, 1, mod=False, weights=False)
    v, dv, h, dh = reference(t, post, pre, 1.0, 1e-6)
    xo, ho = ops.gated_residual_norm(cu(t["y"]), cu(t["x"]), post=post, pre=pre)
    check_status()
    assert_close(xo, v, dv)
    assert_close(ho, h, dh)


def test_a_mean_far_above_the_spread(ops):
    """A difference of sums of squares would have nothing left."""
    t = make(1, 40, 1280, torch.float16, 2, mean=500.0)
    v, dv, h, dh = reference(t, "layer", "layer", 1.0, 1e-6)
    xo, ho = ops.gated_residual_norm(post="layer", pre="layer", **{k: cu(a) for k, a in t.items()})
    assert_close(xo, v, dv)
    assert_close(ho, h, dh)


def test_rows_of_zeros_and_rows_of_nan(ops):
    t = make(1, 5, 640, torch.bfloat16, 3, mod=False)
    t["y"][0, 1], t["x"][0, 1] = 0, 0
    t["x"][0, 3, 7] = float("nan")
    t["y"][0, 4, 2] = float("inf")
    xo, ho = ops.gated_residual_norm(post="rms", pre="layer", **{k: cu(a) for k, a in t.items()})
    check_status()
    assert not bool(ho[0, 1].any()) and not bool(xo[0, 1].any())
    assert bool(torch.isnan(ho[0, 3]).all()) and bool(torch.isnan(ho[0, 4]).all()) and bool(torch.isfinite(ho[0, [0, 2]]).all())


def test_views_in_place_and_chunks_of_one_modulation(ops):
    """Text and image part of a joint sequence, thirds of one modulation tensor, x_out in place of x and h in place of y."""
    g = torch.Generator().manual_seed(4)
    joint_y, joint_x = (torch.randn(2, 50, 640, generator=g).bfloat16().cuda() for _ in range(2))
    mod = torch.randn(2, 3 * 640, generator=g).bfloat16().cuda()
    gate, scale, shift = mod.chunk(3, dim=-1)
    y, x = joint_y[:, 20:], joint_x[:, 20:]
    keep = joint_y[:, :20].clone(), joint_x[:, :20].clone()
    want = ops.gated_residual_norm(y.contiguous(), x.contiguous(), gate.contiguous(), scale.contiguous(), shift.contiguous(), pre="layer")
    got = ops.gated_residual_norm(y, x, gate, scale, shift, pre="layer", x_out=x, h=y)
    check_status()
    assert got[0] is x and got[1] is y and torch.equal(x, want[0]) and torch.equal(y, want[1])
    assert torch.equal(joint_y[:, :20], keep[0]) and torch.equal(joint_x[:, :20], keep[1])
    one = ops.gated_residual_norm(want[0], want[1], gate[0])
    two = ops.gated_residual_norm(want[0], want[1], gate[:1].expand(2, 640))
    assert torch.equal(one[1], two[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,seq,dim", [(1, 3, 96), (2, 150, 640), (1, 5, 3072), (1, 300, 3104), (1, 2, 32), (1, 299, 16384)])
def test_quantized_outputs_are_those_of_the_separate_calls(ops, dtype, batch, seq, dim):
    t = {k: cu(a) for k, a in make(batch, seq, dim, dtype, dim + seq).items()}
    xo, h = ops.gated_residual_norm(post="rms", pre="layer", **t)
    s8 = torch.tensor([0.031], device="cuda")
    q8, want8 = torch.empty(batch, seq, dim, dtype=torch.uint8, device="cuda"), torch.empty(batch, seq, dim, dtype=torch.uint8, device="cuda")
    ops.invoke_cuda_d2d_scale_cpy_convert(want8, h, s8)
    for fmt in ("nvfp4", "mxfp4"):
        g4 = torch.tensor([2.0 ** -5], device="cuda") if fmt == "nvfp4" else None
        q4, want4 = (ops.Fp4Tensor.empty(batch * seq, dim, fmt, g4) for _ in range(2))
        q4.scales.zero_()
        want4.scales.zero_()
        ops.quant_fp4(h.reshape(batch * seq, dim), out=want4)
        x2, h2 = ops.gated_residual_norm(post="rms", pre="layer", qf8=q8, f8_scale=s8, q4=q4, **t)
        check_status()
        assert h2 is None and torch.equal(x2, xo) and torch.equal(q8, want8)
        assert torch.equal(q4.codes, want4.codes) and torch.equal(q4.scales, want4.scales)
        h3 = torch.empty_like(h)
        ops.gated_residual_norm(post="rms", pre="layer", h=h3, q4=q4, **t)
        assert torch.equal(h3, h) and torch.equal(q4.codes, want4.codes)


def test_python_side_refuses(ops):
    t = {k: cu(a) for k, a in make(2, 4, 64, torch.bfloat16, 5).items()}
    bad = [dict(t, x=t["x"][:, :3]), dict(t, gate=t["gate"].float()), dict(t, post_weight=t["post_weight"][:32]), dict(t, post="l2"), dict(t, pre="none"),
           dict(t, qf8=torch.empty(2, 4, 64, dtype=torch.uint8, device="cuda")), dict(t, q4=ops.Fp4Tensor.empty(7, 64)), dict(t, y=t["y"].cpu()),
           dict(t, x_out=t["x"][:1].expand(2, 4, 64)), dict(t, y=t["y"].transpose(1, 2)),
           dict(t, h=torch.zeros(512, dtype=torch.bfloat16, device="cuda").as_strided((2, 4, 64), (64, 64, 1)))]
    for b in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.gated_residual_norm(**b)
    from lyradiff_b200._lib import LyraqError
    wide = torch.zeros(1, 2, 72, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(LyraqError):
        ops.gated_residual_norm(wide[..., 4:68], wide[..., :64])      # not on 16 bytes
    with pytest.raises(LyraqError):
        ops.gated_residual_norm(wide[..., :60].contiguous(), wide[..., :60].contiguous())
    with pytest.raises(LyraqError):
        ops.gated_residual_norm(wide.float(), wide.float())
    both = torch.zeros_like(wide)
    with pytest.raises(LyraqError):
        ops.gated_residual_norm(wide, wide, x_out=both, h=both)


@pytest.mark.parametrize("dim", [640, 1288, 1536])
def test_outputs_in_the_inputs_places(ops, dim):
    t = {k: cu(a) for k, a in make(2, 200, dim, torch.bfloat16, 11).items()}
    want = ops.gated_residual_norm(post="layer", pre="rms", **t)
    for first, second in (("x", "y"), ("y", "x")):
        own = dict(t, x=t["x"].clone(), y=t["y"].clone())
        ops.gated_residual_norm(post="layer", pre="rms", x_out=own[first], h=own[second], **own)
        check_status()
        assert torch.equal(own[first], want[0]) and torch.equal(own[second], want[1])


def test_outputs_that_share_memory_with_what_is_read_are_refused(ops):
    """A row on, other strides at the same place, on another output, the quantized outputs on x; rows of a joint sequence that nobody reads are taken."""
    from lyradiff_b200._lib import LyraqError
    g = torch.Generator().manual_seed(9)
    joint_y, joint_x = (torch.randn(2, 16, 640, generator=g).bfloat16().cuda() for _ in range(2))
    y, x, below = joint_y[:, :7], joint_x[:, :7], joint_x[:, 8:15]
    want = ops.gated_residual_norm(y.contiguous(), x.contiguous(), pre="layer")
    before = joint_y.clone(), joint_x.clone()
    dense = joint_x.flatten()[:14 * 640].view(2, 7, 640)                 # x's first row, other rows
    fresh = torch.empty(2, 7, 640, dtype=torch.bfloat16, device="cuda")
    s8, bytes_of_x = torch.ones(1, device="cuda"), joint_x.view(-1).view(torch.uint8)[:14 * 640].view(2, 7, 640)
    q4 = ops.Fp4Tensor.empty(14, 640)
    on_x = ops.Fp4Tensor(14, 640, "nvfp4", joint_x.view(-1).view(torch.uint8)[:14 * 320].view(14, 320), q4.scales)
    scales_on_y = ops.Fp4Tensor(14, 640, "nvfp4", q4.codes, joint_y.view(-1).view(torch.uint8)[:q4.scales.numel()])
    for kw in ({"x_out": joint_x[:, 1:8]}, {"h": joint_y[:, 1:8]}, {"x_out": dense}, {"x_out": fresh, "h": fresh}, {"x_out": below, "h": joint_x[:, 9:16]},
               {"qf8": bytes_of_x, "f8_scale": s8}, {"q4": on_x}, {"q4": scales_on_y}):
        with pytest.raises(LyraqError):
            ops.gated_residual_norm(y, x, pre="layer", **kw)
    torch.cuda.synchronize()
    assert torch.equal(joint_y, before[0]) and torch.equal(joint_x, before[1])
    got = ops.gated_residual_norm(y, x, pre="layer", x_out=below, h=joint_y[:, 8:15])
    check_status()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(joint_y[:, :8], before[0][:, :8]) and torch.equal(joint_x[:, :8], before[1][:, :8])
    # one stream with itself, the result in its place
    twice = ops.gated_residual_norm(x.contiguous(), x.contiguous(), pre="layer")
    own = x.contiguous().clone()
    again = ops.gated_residual_norm(own, own, pre="layer", x_out=own)
    assert torch.equal(own, twice[0]) and torch.equal(again[1], twice[1])
