"""The FP4 linear, the fused norms and the rotary embedding over axes as they follow one another in a transformer block, with this library's attention
between them; captured in a graph; and where their offsets pass 32 bits."""

import threading

import pytest
import torch

from oracle import blocks, fp4
from tests.test_gpu_fp4 import assert_product
from tests.test_gpu_norm_residual import assert_close as norm_close, reference as norm_reference
from tests.test_gpu_rope_axes import assert_close as rope_close, ladder, reference as rope_reference
from tests.util import check_status, cu

pytestmark = pytest.mark.gpu

HEADS, HEAD_DIM, DIM = 3, 128, 384
AXES = (16, 56, 56)


@pytest.fixture(scope="module")
def lib():
    from lyradiff_b200 import layers, ops, rope
    return layers, ops, rope


class Block:
    """norm -> QKV linear -> rotary embedding with QK norm -> attention -> output linear -> norm, in one type."""

    def __init__(self, lib, fmt, dtype, seed):
        layers, self.ops, rope = lib
        g = torch.Generator().manual_seed(seed)
        self.w = {n: (torch.randn(o, i, generator=g) * 0.05).to(dtype) for n, o, i in (("qkv", 3 * DIM, DIM), ("out", DIM, DIM))}
        self.b = {n: (torch.randn(v.shape[0], generator=g) * 0.1).to(dtype) for n, v in self.w.items()}
        self.layer = {n: layers.Fp4Linear(cu(v), cu(self.b[n]), torch.tensor(2.0 ** -6), fmt=fmt) for n, v in self.w.items()}
        self.p = {n: (1 + 0.2 * torch.randn(DIM, generator=g)).to(dtype) for n in ("post", "pre")}
        self.qk = [(1 + 0.2 * torch.randn(HEAD_DIM, generator=g)).to(dtype) for _ in range(2)]
        self.plan = rope.AxisRope(AXES)
        self.dev = {n: cu(v) for n, v in self.p.items()}
        self.dqk = [cu(v) for v in self.qk]

    def run(self, y, x, mod, pos):
        """(x1, q4, qkv before the rotation, qkv after it, attention, out, x2, h2)"""
        b, s, _ = y.shape
        gate, scale, shift = mod.chunk(3, dim=-1)
        kw = dict(scale=scale, shift=shift, post_weight=self.dev["post"], pre_weight=self.dev["pre"], post="rms", pre="layer")
        q4 = self.layer["qkv"].empty_input(b * s)
        x1, _ = self.ops.gated_residual_norm(y, x, gate, q4=q4, **kw)
        qkv = self.layer["qkv"].forward_quantized(q4, y.dtype)
        raw = qkv.clone()
        heads = qkv.view(b, s, 3, HEADS, HEAD_DIM)
        q, k = heads[:, :, 0], heads[:, :, 1]
        self.ops.rope_axes(self.plan, pos, q, k, *self.dqk, q_out=q, k_out=k)
        att = self.ops.flash_attention(qkv, b, s, HEADS, HEAD_DIM)
        out = self.layer["out"].forward(att)
        x2, h2 = self.ops.gated_residual_norm(out.view(b, s, DIM), x1, gate, **kw)
        return x1, q4, raw, qkv, att, out, x2, h2


def inputs(dtype, b, s, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(b, s, DIM, generator=g).to(dtype), torch.randn(b, s, DIM, generator=g).to(dtype),
            (torch.randn(b, 3 * DIM, generator=g) * 0.4).to(dtype), torch.randint(0, 60, (b, s, 3), generator=g))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,s", [(1, 1), (2, 75), (1, 300)])
def test_every_step_of_a_block_against_64_bits(lib, fmt, dtype, b, s):
    """Each step is held to its own formula over what the step before it left, so its tolerance is its own."""
    blk = Block(lib, fmt, dtype, 3)
    y, x, mod, pos = inputs(dtype, b, s, s)
    x1, q4, raw, qkv, att, out, x2, h2 = blk.run(cu(y), cu(x), cu(mod), cu(pos))
    check_status()
    t = dict(zip(("gate", "scale", "shift"), mod.chunk(3, dim=-1)), y=y, x=x, post_weight=blk.p["post"], pre_weight=blk.p["pre"])
    v, dv, _, _ = norm_reference(t, "rms", "layer", 1.0, 1e-6)
    norm_close(x1, v, dv)
    gx = 2.0 ** -6 if fmt == "nvfp4" else 1.0

    def weight(n):
        g = fp4.tensor_scale(blk.w[n]) if fmt == "nvfp4" else 1.0
        return (*fp4.encode(blk.w[n], fmt, g), g)
    codes = fp4.unpack(q4.codes.cpu())
    scales = q4.scales.cpu()[fp4.scale_offsets(b * s, DIM // fp4.GROUP[fmt])]
    assert_product(raw, (codes, scales, gx), weight("qkv"), fmt, blk.b["qkv"])
    r, q = raw.cpu().view(b, s, 3, HEADS, HEAD_DIM), qkv.view(b, s, 3, HEADS, HEAD_DIM)
    freq, axis = ladder(AXES)
    for i in range(2):
        rope_close(q[:, :, i], *rope_reference(r[:, :, i], pos, freq, axis, True, blk.qk[i], 1e-6))
    assert torch.equal(q[:, :, 2].cpu(), r[:, :, 2])
    z = q.cpu().permute(2, 0, 3, 1, 4)
    want = blocks.attention(z[0], z[1], z[2]).permute(0, 2, 1, 3).reshape(b * s, DIM)
    eps = torch.finfo(dtype).eps
    assert float((att.cpu().double() - want).abs().max()) <= 2.5 * eps * float(want.abs().max())     # as tests/test_gpu_attention.py has it
    assert_product(out, (*fp4.encode(att.cpu(), fmt, gx), gx), weight("out"), fmt, blk.b["out"])
    t.update(y=out.cpu().view(b, s, DIM), x=x1.cpu())
    v, dv, h, dh = norm_reference(t, "rms", "layer", 1.0, 1e-6)
    norm_close(x2, v, dv)
    norm_close(h2, h, dh)


def test_a_captured_block_replays_with_new_inputs_beside_an_eager_one(lib):
    blk = Block(lib, "nvfp4", torch.bfloat16, 4)
    ins = [cu(t) for t in inputs(torch.bfloat16, 2, 40, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        blk.run(*ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = blk.run(*ins)
    other = [cu(t) for t in inputs(torch.bfloat16, 2, 40, 2)]
    want = blk.run(*other)
    for a, b in zip(ins, other):
        a.copy_(b)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    again = blk.run(*other)                                             # at the same time, on the current stream
    torch.cuda.synchronize()
    check_status()
    for a, b, c in zip(got, want, again):
        if isinstance(a, torch.Tensor):
            assert torch.equal(a, b) and torch.equal(c, b)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 6])
def test_a_chain_of_few_row_linears_replays(lib, fmt, rows):
    """Launches that begin before their predecessors end, each of which reads what the one before wrote."""
    layers, ops, _ = lib
    g = torch.Generator().manual_seed(rows)
    chain = [layers.Fp4Linear(cu((torch.randn(1024, 1024, generator=g) * 0.06).bfloat16()), None, torch.tensor(2.0 ** -6), fmt=fmt) for _ in range(6)]

    def by_steps(x):
        for layer in chain:
            q = layer.empty_input(x.shape[0])
            ops.quant_fp4(x, out=q)
            torch.cuda.synchronize()
            x = layer.forward_quantized(q, x.dtype)
            torch.cuda.synchronize()
        return x

    def run(x):
        for layer in chain:
            x = layer.forward(x)
        return x
    x = torch.randn(rows, 1024, generator=g).bfloat16().cuda()
    run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x)
    for seed in range(8):
        x.copy_(torch.randn(rows, 1024, generator=g).bfloat16())
        want = by_steps(x)
        graph.replay()
        assert torch.equal(run(x), want) and torch.equal(got, want)
    check_status()


def test_calls_from_several_threads(lib):
    """Each thread on a stream of its own; the calls leave the interpreter lock while they launch."""
    layers, ops, rope = lib
    g = torch.Generator().manual_seed(9)
    layer = layers.Fp4Linear(cu((torch.randn(512, 512, generator=g) * 0.05).bfloat16()), None, torch.tensor(2.0 ** -6))
    plan, pos = rope.AxisRope((16, 24, 24)), torch.randint(0, 50, (40, 3), generator=g).cuda()
    xs = [torch.randn(1, n, 512, generator=g).bfloat16().cuda() for n in (1, 40, 7, 40)]

    def once(x):
        y = layer.forward(x)
        x1, h = ops.gated_residual_norm(y, x, post="layer")
        n = x.shape[1]
        return y, x1, h, ops.rope_axes(plan, pos[:n], h.view(1, n, 8, 64))[0]
    want = [once(x) for x in xs]
    torch.cuda.synchronize()
    wrong, streams = [], [torch.cuda.Stream() for _ in xs]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(60):
                if not all(torch.equal(a, b) for a, b in zip(once(xs[i]), want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    check_status()
    assert not wrong


def test_offsets_beyond_32_bits(lib):
    """Rows that lie more than 2^31 elements (4 GB) apart."""
    layers, ops, rope = lib
    far = 2 ** 31 + 64
    big = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(6)
    data = torch.randn(2, 512, generator=g).bfloat16().cuda()

    def rows(width):
        return big.as_strided((2, width), (far, 1))
    rows(512).copy_(data)
    for fmt in ("nvfp4", "mxfp4"):
        a, b = ops.quant_fp4(rows(512), None, fmt), ops.quant_fp4(data, None, fmt)
        assert torch.equal(a.codes, b.codes)
    layer = layers.Fp4Linear(torch.randn(64, 512, generator=g).bfloat16().cuda())
    assert torch.equal(layer.forward(rows(512)), layer.forward(data))
    x = data.view(1, 2, 512)
    want = ops.gated_residual_norm(x, x)
    apart = rows(512).unsqueeze(0)
    got = ops.gated_residual_norm(apart, apart)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    plan, pos = rope.AxisRope((64, 64)), torch.tensor([[3, 5], [1000, 7]], device="cuda")
    want = ops.rope_axes(plan, pos, data.view(1, 2, 4, 128))[0]
    q = apart.unflatten(-1, (4, 128))
    assert torch.equal(ops.rope_axes(plan, pos, q)[0], want)
    ops.rope_axes(plan, pos, q, q_out=q)
    check_status()
    assert torch.equal(rows(512).view(1, 2, 4, 128), want)
