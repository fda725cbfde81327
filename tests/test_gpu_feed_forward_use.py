"""The feed-forward operators as programs use them: recorded into graphs, on another stream than the default one, side by side in one launch or
apart, on rows that begin at odd elements and on more rows than a grid's second side has, and all together in the example."""
import numpy as np
import pytest

import ffn_reference as ref
from reference_model_amd import Context, TmiError, capi
from test_gpu_gated_ffn import KINDS, Rows, backward, forward, near, operands

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


# rows, d, f, gap, lead: rows of whole 256-byte steps and more, of which all, the odd ones or the even ones begin inside a word
ODD = [(1, 129, 40, 0, 0), (1, 257, 16, 1, 1), (4, 400, 33, 1, 0), (16, 385, 50, 0, 1), (9, 256, 20, 0, 1), (17, 131, 40, 0, 0), (32, 513, 18, 2, 3), (20, 1150, 35, 1, 0)]


@pytest.mark.parametrize("shape", ODD, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_few_rows_at_odd_elements(ctx, kind, shape):
    kind, (m, d, f, gap, lead) = KINDS[kind], shape
    x, gate, up = operands(kind, m, d, f, m + d)
    got = forward(ctx, kind, "silu", x, gate, up, gap=gap, lead=lead)
    assert ctx.last_kernel == "ffn_rows"
    for v, want in zip(got, ref.gated(kind, "silu", x, gate, up)):
        near(kind.wide(v), want)


@pytest.mark.parametrize("shape", ODD + [(33, 300, 70, 1, 1), (64, 2100, 40, 0, 1)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("kind", list(KINDS))
def test_4_bit_weights_and_x_at_odd_elements(ctx, kind, group, shape):
    kind, (m, k, n, gap, lead) = KINDS[kind], shape
    rng = np.random.default_rng(m + k)
    x, w, _ = operands(kind, m, k, n, m + k)
    v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.normal(0, 0.02, (n, -(-k // group))))
    held, dev, out = ctx.upload(ref.packed(kind, v, scales, group)), Rows(ctx, kind, (m, k), x, gap, lead), Rows(ctx, kind, (m, n), None, gap, lead)
    ctx.matvec_int4(ctx.int4_desc(kind.dtype, group, n, k), m, dev.at, k + gap, held, out.at, n + gap)
    assert ctx.sync() == capi.VALID
    near(out.values(), ref.product(kind, x, ref.weights(kind, v, scales, group)))
    for t in (held, dev, out):
        t.free()


@pytest.mark.parametrize("n,k", [(40, 513), (17, 1030), (129, 135)])
@pytest.mark.parametrize("kind", list(KINDS))
def test_quantisation_of_several_column_tiles_at_odd_elements(ctx, kind, n, k):
    kind, group = KINDS[kind], 64
    w = operands(kind, 1, k, n, n + k)[1]
    v, scales = ref.quantized(kind, w, group)
    want = ref.packed(kind, v, scales, group)
    desc = ctx.int4_desc(kind.dtype, group, n, k)
    for gap, lead in ((0, 0), (1, 0), (0, 1), (3, 1)):
        dev, to, back = Rows(ctx, kind, (n, k), w, gap, lead), ctx.upload(np.full(want.size, 0xA5, np.uint8)), Rows(ctx, kind, (n, k), None, gap, lead)
        ctx.quantize_int4(desc, dev.at, k + gap, to)
        ctx.dequantize_int4(desc, to, back.at, k + gap)
        assert ctx.sync() == capi.VALID
        assert np.array_equal(to.numpy().view(np.uint8), want)
        assert np.array_equal(back.stored().view(np.uint16), kind.narrow(ref.weights(kind, v, scales, group)).view(np.uint16))
        for t in (dev, to, back):
            t.free()


@pytest.mark.parametrize("shape", [(70, 129, 65), (200, 256, 300), (40, 64, 1200), (1100, 72, 40), (5, 720, 500), (300, 1500, 40)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_gradients_together_and_alone(ctx, kind, shape):
    """one call for all of them, which may put both products into one launch, and a call for each"""
    kind, (m, d, f) = KINDS[kind], shape
    x, gate, up = operands(kind, m, d, f, m + d + f)
    rng = np.random.default_rng(7)
    g, u, dh = (kind.wide(kind.narrow(v)) for v in (x @ gate.T, x @ up.T, rng.normal(0, 0.5, (m, f))))
    want = ref.gated_gradients(kind, "silu", x, gate, up, g, u, dh)
    both = backward(ctx, kind, "silu", x, gate, up, g, u, dh)
    of_x = backward(ctx, kind, "silu", x, gate, up, g, u, dh, dw=False)
    of_w = backward(ctx, kind, "silu", x, gate, up, g, u, dh, dx=False)
    for got in (both, [of_x[0], of_w[1], of_w[2]]):
        for v, w in zip(got, want):
            near(kind.wide(v), w)


def test_more_rows_than_a_grids_second_side(ctx):
    """66000 rows whose sums are long enough to be split; compared over rows from both ends and between"""
    kind, (m, d, f) = KINDS["bf16"], (66000, 1024, 40)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, gate, up = (torch.randn(n, d, device="cuda", generator=gen).mul_(s).to(torch.bfloat16) for n, s in ((m, 1), (f, d ** -0.5), (f, d ** -0.5)))
    h = torch.full((m, f), float("nan"), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ctx.gated_ffn(ctx.gated_ffn_desc(kind.dtype, capi.ACT_SILU, m, d, f), x, gate, up, h)
    assert ctx.sync() == capi.VALID and not torch.isnan(h).any()
    rows = [0, 1, 127, 128, 32767, 65534, 65535, 65536, 65537, 65999]
    wide = lambda t: t.double().cpu().numpy()  # noqa: E731
    near(wide(h[rows]), ref.gated(kind, "silu", wide(x[rows]), wide(gate), wide(up))[0])


class Block:
    """tensors of every feed-forward operator, and one pass through all of them"""

    def __init__(self, ctx, name, rows=70, d=200, f=136, group=64):
        self.ctx, kind, t = ctx, KINDS[name], TYPES[name]
        new = lambda *s: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
        self.x, self.gate, self.up, self.dh = new(rows, d), new(f, d), new(f, d), new(rows, f)
        self.desc, self.int4 = ctx.gated_ffn_desc(kind.dtype, capi.ACT_GELU, rows, d, f), ctx.int4_desc(kind.dtype, group, f, d)
        self.few = ctx.gated_ffn_desc(kind.dtype, capi.ACT_GELU, 3, d, f)
        packed = [torch.empty(ctx.int4_packed_bytes(self.int4), device="cuda", dtype=torch.uint8) for _ in range(2)]
        self.out = [new(rows, f), new(rows, f), new(rows, f), new(rows, d), new(f, d), new(f, d), *packed, new(f, d), new(3, f), new(3, f), new(rows, f), new(rows, f)]

    def fill(self, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for v, std in ((self.x, 1.0), (self.gate, 0.07), (self.up, 0.07), (self.dh, 0.5)):
            v.copy_(torch.randn(v.shape, device="cuda", generator=gen) * std)

    def step(self):
        c, (h, g, u, dx, dg, du, pg, pu, back, h3, q3, y, q) = self.ctx, self.out
        rows, d = self.x.shape
        f = self.gate.shape[0]
        c.gated_ffn(self.desc, self.x, self.gate, self.up, h, g, u)
        c.gated_ffn_backward(self.desc, self.x, self.gate, self.up, g, u, self.dh, dx, dg, du)
        c.quantize_int4(self.int4, self.gate, d, pg)
        c.quantize_int4(self.int4, self.up, d, pu)
        c.dequantize_int4(self.int4, pg, back, d)
        c.gated_ffn(self.few, self.x, self.gate, self.up, h3)
        c.gated_ffn_int4(self.int4, capi.ACT_GELU, 3, self.x, d, pg, pu, q3, f)
        c.matvec_int4(self.int4, rows, self.x, d, pg, y, f)
        c.gated_ffn_int4(self.int4, capi.ACT_GELU, rows, self.x, d, pg, pu, q, f)

    def spoil(self):
        for t in self.out:
            t.fill_(77)


@pytest.mark.parametrize("name", list(KINDS))
@pytest.mark.parametrize("sizes", [dict(), dict(rows=300, d=201, f=135), dict(rows=40, d=1030, f=100)], ids=["whole", "odd", "split"])
def test_graph_of_all_of_them_matches_eager_on_every_replay(name, sizes):
    ctx = Context(0)
    try:
        stream = torch.cuda.current_stream()
        ctx.set_stream(stream.cuda_stream)
        block = Block(ctx, name, **sizes)
        block.fill(0)
        block.step()    # scratch buffer and kernel attributes
        assert ctx.sync() == capi.VALID
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(stream)
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            block.step()
        ctx.set_stream(stream.cuda_stream)
        for seed in (1, 2, 3, 4):
            block.fill(seed)
            block.step()
            assert ctx.sync() == capi.VALID
            want = [t.clone() for t in block.out]
            block.spoil()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert ctx.sync() == capi.VALID
            for got, ref_ in zip(block.out, want):
                assert torch.equal(got, ref_)
    finally:
        ctx.close()


def test_scratch_is_not_grown_inside_a_capture():
    """the gradients need a scratch buffer and say so; the forward pass goes on without one"""
    ctx = Context(0)
    try:
        block = Block(ctx, "bf16", rows=64, d=1030, f=96)
        block.fill(5)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        c, o = ctx, block.out
        few = ctx.gated_ffn_desc(capi.BF16, capi.ACT_GELU, 64, 64, 64)
        c.gated_ffn(few, block.x, block.gate, block.up, o[0])    # kernels' attributes
        assert ctx.sync() == capi.VALID
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            c.gated_ffn(block.desc, block.x, block.gate, block.up, o[0], o[1], o[2])
            with pytest.raises(TmiError) as e:
                c.gated_ffn_backward(block.desc, block.x, block.gate, block.up, o[1], o[2], block.dh, o[3], o[4], o[5])
        assert e.value.status == capi.ERROR
        graph.replay()
        torch.cuda.synchronize()
        got = o[0].clone()
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        c.gated_ffn(block.desc, block.x, block.gate, block.up, o[0], o[1], o[2])
        assert ctx.sync() == capi.VALID
        wide = lambda t: t.double().cpu().numpy()  # noqa: E731
        want = ref.gated(KINDS["bf16"], "gelu", wide(block.x), wide(block.gate), wide(block.up))[0]
        near(wide(got), want)
        near(wide(o[0]), want)
    finally:
        ctx.close()


@pytest.mark.parametrize("name", list(KINDS))
def test_another_stream(name):
    """operands that another stream writes just before, results that it reads just behind"""
    ctx = Context(0)
    try:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        block = Block(ctx, name, rows=90, d=333)
        block.fill(8)
        block.step()
        assert ctx.sync() == capi.VALID
        want = [t.clone() for t in block.out]
        block.spoil()
        for v in (block.x, block.gate, block.up, block.dh):
            v.zero_()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            ctx.set_stream(side.cuda_stream)
            block.fill(8)
            block.step()
            got = [t.clone() for t in block.out]
        side.synchronize()
        assert ctx.sync() == capi.VALID
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    finally:
        ctx.close()


def test_example():
    from reference_model_amd import feed_forward

    got = feed_forward.run(rows=130, width=200, hidden=296, steps=40, tokens=20)
    losses = got["losses"]
    assert all(b < a for a, b in zip(losses[:10], losses[1:11])) and losses[-1] < losses[0] / 2
    # a group's largest weight is 7 steps, so a rounding is off by a fourteenth of it at most, 2.9 / 14 / sqrt(3) of a normal number's deviation at 32 a group and about
    # half of that in the mean; three such matrices make an answer
    assert 0.02 < got["weights_off"] < 0.12 and got["answers_off"] < 0.35


# few results from long rows, whose columns workgroups share; the last rows of tiles and the last column tiles empty, one column past a tile, one short of it
LONG = [(1, 6001, 40), (14, 8193, 17), (16, 2111, 100), (5, 4095, 16), (31, 5000, 9), (60, 3001, 33)]


@pytest.mark.parametrize("shape", LONG, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_few_results_of_long_rows(ctx, kind, shape):
    kind, (m, k, n), group = KINDS[kind], shape, 64
    rng = np.random.default_rng(k)
    x, gate, up = operands(kind, m, k, n, k)
    for v, want in zip(forward(ctx, kind, "gelu", x, gate, up), ref.gated(kind, "gelu", x, gate, up)):
        near(kind.wide(v), want)
    desc, held, packed = ctx.int4_desc(kind.dtype, group, n, k), [], []
    for _ in range(2):
        v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.normal(0, 0.2 / np.sqrt(k), (n, -(-k // group))))
        packed.append(ref.weights(kind, v, scales, group))
        held.append(ctx.upload(ref.packed(kind, v, scales, group)))
    dev, y, h = Rows(ctx, kind, (m, k), x, 1, 0), Rows(ctx, kind, (m, n), None, 3, 0), Rows(ctx, kind, (m, n), None, 3, 0)
    ctx.matvec_int4(desc, m, dev.at, k + 1, held[0], y.at, n + 3)
    ctx.gated_ffn_int4(desc, capi.ACT_SILU, m, dev.at, k + 1, *held, h.at, n + 3)
    assert ctx.sync() == capi.VALID
    near(y.values(), ref.product(kind, x, packed[0]))
    near(h.values(), ref.gated(kind, "silu", x, *packed)[0])
    for t in held + [dev, y, h]:
        t.free()
