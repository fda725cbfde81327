"""The norm, its gradients, rows in 8 bits and the linear layer on them as programs use them: one after the other in a layer, recorded into graphs, on other
streams, in two contexts at once, and on tensors that reach beyond 32 bits."""
import pytest

torch = pytest.importorskip("torch")

import projection_reference as ref  # noqa: E402
from projection_plan import plan  # noqa: E402
from projection_reference import KINDS, near  # noqa: E402
from reference_model_amd import Context, TmiError, capi  # noqa: E402

pytestmark = pytest.mark.gpu

# rows, out_features, in_features of every kernel of the linear layer: rows (0: the one of few rows) and features of its tiles, and whether the sum is split
KINDS_OF_FORMS = [((1, 1000, 700), 0, 16, False), ((9, 200, 16400), 0, 16, True), ((20, 300, 500), 0, 16, False), ((40, 300, 500), 0, 16, False),
                  ((60, 300, 500), 0, 16, False), ((30, 100, 9000), 0, 16, True), ((300, 500, 200), 64, 64, False), ((200, 300, 12000), 64, 64, True),
                  ((300, 5003, 1111), 128, 64, False), ((500, 4000, 1000), 128, 64, False), ((900, 4000, 1000), 128, 128, False),
                  ((2000, 4090, 1000), 128, 256, False), ((3600, 3700, 700), 256, 256, False)]
FORMS = [f[0] for f in KINDS_OF_FORMS]


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def on_the_current_stream(ctx):
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    assert ctx.sync() == capi.VALID


def pitch(width):
    return -(-width // 16) * 16


class Layer:
    """a layer whose norms lead into projections: trained in dtype, and answering with 8-bit weights"""

    def __init__(self, ctx, name, rows=70, width=200, hidden=136, out=90):
        self.ctx, self.kind, t = ctx, KINDS[name], KINDS[name].t
        self.sizes = rows, width, hidden, out
        new = lambda *s, dtype=t: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        self.x, self.residual, self.weight, self.dh, self.ds = new(rows, width), new(rows, width), new(width), new(rows, hidden), new(rows, width)
        self.gate, self.up, self.w, self.bias = new(hidden, width), new(hidden, width), new(out, width), new(out)
        d = self.kind.dtype
        self.norm = ctx.rms_norm_desc(d, rows, width, 1e-5, 1.0)
        self.ffn = None if name == "fp32" else ctx.gated_ffn_desc(d, capi.ACT_SILU, rows, width, hidden)
        self.linear = ctx.linear_int8_desc(d, rows, width, out)
        bytes_, f32 = dict(dtype=torch.int8), dict(dtype=torch.float32)
        self.sum, self.y, self.r, self.h, self.g, self.u = new(rows, width), new(rows, width), new(rows, **f32), new(rows, hidden), new(rows, hidden), new(rows, hidden)
        self.dy, self.dx, self.dweight, self.dgate, self.dup = new(rows, width), new(rows, width), new(width), new(hidden, width), new(hidden, width)
        self.q, self.scales = new(rows, pitch(width), **bytes_), new(rows, **f32)
        self.qw, self.wscales, self.wback = new(out, pitch(width), **bytes_), new(out, **f32), new(out, width)
        self.answer = new(rows, out)
        self.out = [v for k, v in vars(self).items() if k in ("sum y r dx dweight q scales qw wscales wback answer".split() + ("h g u dy dgate dup".split() if self.ffn else []))]

    def fill(self, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for v, std in ((self.x, 1.0), (self.residual, 1.0), (self.weight, 0.2), (self.dh, 0.5), (self.ds, 0.3), (self.gate, 0.07), (self.up, 0.07), (self.w, 0.1),
                       (self.bias, 0.1)) + (() if self.ffn else ((self.dy, 0.5),)):
            v.copy_(torch.randn(v.shape, device="cuda", generator=gen) * std)

    def step(self):
        c, (rows, width, hidden, out), d = self.ctx, self.sizes, self.kind.dtype
        c.rms_norm(self.norm, self.x, self.residual, self.weight, self.sum, self.y, self.r)
        if self.ffn:
            c.gated_ffn(self.ffn, self.y, self.gate, self.up, self.h, self.g, self.u)
            c.gated_ffn_backward(self.ffn, self.y, self.gate, self.up, self.g, self.u, self.dh, self.dy, self.dgate, self.dup)
        c.rms_norm_backward(self.norm, self.sum, self.weight, self.r, self.dy, self.ds, self.dx, self.dweight)
        c.quantize_int8(d, out, width, self.w, width, self.qw, pitch(width), self.wscales)
        c.dequantize_int8(d, out, width, self.qw, pitch(width), self.wscales, self.wback, width)
        c.rms_norm_int8(self.norm, self.x, self.residual, self.weight, None, self.q, self.scales)
        c.linear_int8(self.linear, self.q, self.scales, self.qw, self.wscales, self.bias, self.answer)

    def spoil(self):
        for t in self.out:
            t.fill_(77)


SIZES = [dict(), dict(rows=301, width=1111, hidden=65, out=33), dict(rows=3, width=4100, hidden=20, out=1000), dict(rows=1000, width=600, hidden=200, out=2000)]


@pytest.mark.parametrize("sizes", SIZES, ids=["whole", "odd", "few", "many"])
@pytest.mark.parametrize("name", list(KINDS))
def test_a_layer(ctx, name, sizes):
    """each result against the formula, from what the operator before it left"""
    layer, wide = Layer(ctx, name, **sizes), lambda t: t.double().cpu()
    layer.fill(11)
    layer.step()
    assert ctx.sync() == capi.VALID
    kind, (rows, width, hidden, out) = layer.kind, layer.sizes
    (s, off_s), (y, off_y), (r, off_r) = ref.norm(kind, wide(layer.x), wide(layer.residual), wide(layer.weight), 1e-5, 1.0)
    near(wide(layer.sum), s, off_s)
    near(wide(layer.y), y, off_y + kind.rounding(y, off_y))
    near(wide(layer.r), r, off_r)
    (dx, off_x), (dw, off_w) = ref.norm_gradients(kind, wide(layer.sum), wide(layer.weight), wide(layer.r), wide(layer.dy), wide(layer.ds), 1.0)
    near(wide(layer.dx), dx, off_x)
    near(wide(layer.dweight), dw, off_w)
    ref.check_int8(wide(layer.qw), wide(layer.wscales), wide(layer.w), 0.0, width, kind.t != torch.float32)
    back = wide(layer.qw)[:, :width] * wide(layer.wscales)[:, None]
    near(wide(layer.wback), back, kind.rounding(back))
    ref.check_int8(wide(layer.q), wide(layer.scales), y, (ref.depth(width) / 2 + 10) * ref.EPS, width)
    near(wide(layer.answer), *ref.linear(kind, wide(layer.q), wide(layer.scales), wide(layer.qw), wide(layer.wscales), wide(layer.bias)))
    # and the projection beside the one that was not rounded: each product is off by half a step of either operand
    want = y @ wide(layer.w).T + wide(layer.bias)
    step = wide(layer.scales)[:, None] / 2 * wide(layer.w).abs().sum(1) + wide(layer.wscales) / 2 * y.abs().sum(1, keepdim=True) + \
        width * wide(layer.scales)[:, None] * wide(layer.wscales) / 4
    near(wide(layer.answer), want, 1.01 * step + kind.rounding(want, step))


@pytest.mark.parametrize("sizes", SIZES, ids=["whole", "odd", "few", "many"])
@pytest.mark.parametrize("name", list(KINDS))
def test_a_graph_of_the_layer_gives_the_eager_bits_on_every_replay(ctx, name, sizes):
    stream, layer = torch.cuda.current_stream(), Layer(ctx, name, **sizes)
    layer.fill(0)
    layer.step()    # scratch buffer and kernel attributes
    assert ctx.sync() == capi.VALID
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(stream)
    with torch.cuda.graph(graph, stream=side):
        ctx.set_stream(side.cuda_stream)
        layer.step()
    ctx.set_stream(stream.cuda_stream)
    for seed in (1, 2, 3, 4):
        layer.fill(seed)
        layer.step()
        assert ctx.sync() == capi.VALID
        want = [t.clone() for t in layer.out]
        layer.spoil()
        if not layer.ffn:
            layer.fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(layer.out, want):
            assert torch.equal(got, eager)


class Product:
    """a call of the linear layer"""

    def __init__(self, ctx, shape, seed, name="fp32"):
        (m, n, k), kind = shape, KINDS[name]
        gen = torch.Generator(device="cuda").manual_seed(seed)
        of = lambda rows: torch.nn.functional.pad(torch.randint(-127, 128, (rows, k), generator=gen, device="cuda"), (0, pitch(k) - k)).to(torch.int8)  # noqa: E731
        self.x, self.w, self.sx, self.sw = of(m), of(n), torch.rand(m, generator=gen, device="cuda"), torch.rand(n, generator=gen, device="cuda")
        self.y, self.desc, self.ctx, self.kind = torch.full((m, n), 77.0, device="cuda").to(kind.t), ctx.linear_int8_desc(kind.dtype, m, k, n), ctx, kind

    def call(self):
        self.ctx.linear_int8(self.desc, self.x, self.sx, self.w, self.sw, None, self.y)

    def check(self):
        wide = lambda t: t.double().cpu()  # noqa: E731
        near(wide(self.y), *ref.linear(self.kind, wide(self.x), wide(self.sx), wide(self.w), wide(self.sw), None))


@pytest.mark.parametrize("shape", FORMS, ids=lambda s: "x".join(map(str, s)))
def test_every_form_into_two_graphs_that_take_turns(ctx, shape):
    """they name the same scratch buffer, and run one after the other"""
    a, b = Product(ctx, shape, 1), Product(ctx, shape, 2)
    a.call(), b.call()
    torch.cuda.synchronize()
    a.check(), b.check()
    want, graphs, stream = [a.y.clone(), b.y.clone()], [], torch.cuda.current_stream()
    for p in (a, b):
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(stream)
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            p.call()
        ctx.set_stream(stream.cuda_stream)
        graphs.append(graph)
    for _ in range(3):
        a.y.fill_(77), b.y.fill_(77)
        for i in (0, 1, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(a.y, want[0]) and torch.equal(b.y, want[1])
        a.call()
        torch.cuda.synchronize()
        assert torch.equal(a.y, want[0])


@pytest.mark.parametrize("shape", [f[0] for f in KINDS_OF_FORMS if f[3]], ids=lambda s: "x".join(map(str, s)))
def test_sums_in_one_piece_where_the_scratch_buffer_cannot_grow(shape):
    c = Context(0)
    try:
        stream = torch.cuda.current_stream()
        c.set_stream(stream.cuda_stream)
        p = Product(c, shape, 3)
        few = Product(c, (shape[0], 3, 16), 4)
        few.call()
        assert c.sync() == capi.VALID and c.workspace_bytes()[0] == 0
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(stream)
        with torch.cuda.graph(graph, stream=side):
            c.set_stream(side.cuda_stream)
            p.call()
        c.set_stream(stream.cuda_stream)
        assert c.workspace_bytes()[0] == 0
        graph.replay()
        torch.cuda.synchronize()
        got = p.y.clone()
        p.check()
        p.call()
        assert c.sync() == capi.VALID and c.workspace_bytes()[0] > 0
        assert torch.equal(p.y, got)
    finally:
        c.close()


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 63, 1023, 1025])
@pytest.mark.parametrize("m", [1, 9, 70])
def test_split_sums_of_any_width(ctx, m, n):
    """joined in fours, of which a row's last begin inside its neighbour's"""
    for k in (20000, 60000):
        assert plan(m, n, k).splits > 1
        p = Product(ctx, (m, n, k), n + k, "bf16")
        p.call()
        assert ctx.sync() == capi.VALID
        p.check()


def test_gradients_that_need_scratch_are_refused_where_it_cannot_grow():
    c = Context(0)
    try:
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        for width, dw in ((100, True), (17000, False)):
            new = lambda *s: torch.ones(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
            s, w, dy, dx, d_w, r = new(5, width), new(width), new(5, width), new(5, width), new(width), torch.ones(5, device="cuda")
            desc = c.rms_norm_desc(capi.BF16, 5, width, 1e-5)
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                c.set_stream(side.cuda_stream)
                dx.zero_()
                with pytest.raises(TmiError) as e:
                    c.rms_norm_backward(desc, s, w, r, dy, None, dx, d_w if dw else None)
                if width == 100:
                    c.rms_norm_backward(desc, s, w, r, dy, None, dx, None)    # no sums over rows
            assert e.value.status == capi.ERROR and "scratch" in e.value.message
            graph.replay()
            torch.cuda.synchronize()
            assert (d_w == 1).all() and (dx == 0).all()    # g - n mean(g n) of ones
            c.set_stream(torch.cuda.current_stream().cuda_stream)
    finally:
        c.close()


def test_two_contexts_at_once():
    """on streams of their own, each with its scratch buffer"""
    streams, layers, want = [torch.cuda.Stream() for _ in range(2)], [], []
    contexts = [Context(0), Context(0)]
    try:
        for i, (c, s) in enumerate(zip(contexts, streams)):
            c.set_stream(s.cuda_stream)
            layers.append(Layer(c, "bf16", rows=700, width=1000, hidden=300, out=500))
            layers[i].fill(20 + i)
        torch.cuda.synchronize()
        for layer in layers:
            layer.step()
            assert layer.ctx.sync() == capi.VALID
            want.append([t.clone() for t in layer.out])
            layer.spoil()
        torch.cuda.synchronize()
        for _ in range(4):
            for layer in layers:
                layer.step()
        for layer, kept in zip(layers, want):
            assert layer.ctx.sync() == capi.VALID
            for got, alone in zip(layer.out, kept):
                assert torch.equal(got, alone)
    finally:
        for c in contexts:
            c.close()


def test_gradients_of_equal_calls_have_equal_bits(ctx):
    for rows, width in ((5000, 40), (3000, 1000), (700, 3000), (300, 20000)):
        layer = Layer(ctx, "fp32", rows=rows, width=width, hidden=1, out=1)
        layer.fill(30)
        ctx.rms_norm(layer.norm, layer.x, layer.residual, layer.weight, layer.sum, layer.y, layer.r)
        kept = None
        for _ in range(4):
            layer.dx.fill_(77), layer.dweight.fill_(77)
            ctx.rms_norm_backward(layer.norm, layer.sum, layer.weight, layer.r, layer.dy, layer.ds, layer.dx, layer.dweight)
            torch.cuda.synchronize()
            if kept:
                assert torch.equal(layer.dx, kept[0]) and torch.equal(layer.dweight, kept[1])
            kept = layer.dx.clone(), layer.dweight.clone()


def far(rows, width, ld, t):
    """rows so far apart that the last begins beyond 32 bits; what lies between them is left as it is"""
    return torch.empty((rows - 1) * ld + width + 64, dtype=t, device="cuda").as_strided((rows, width), (ld, 1))


@pytest.mark.parametrize("width", [40, 1000, 3000, 17000])
def test_norm_and_gradients_beyond_32_bits(ctx, width):
    kind, rows, ld = KINDS["bf16"], 3, (1 << 31) + 24
    gen = torch.Generator().manual_seed(width)
    values = [torch.randn(rows, width, generator=gen).to(kind.t) for _ in range(2)]
    weight = torch.randn(width, generator=gen).to(kind.t)
    x, y, dy = far(rows, width, ld, kind.t), far(rows, width, ld, kind.t), far(rows, width, ld, kind.t)
    r, dw, w = torch.empty(rows, device="cuda"), torch.empty(width, device="cuda", dtype=kind.t), weight.cuda()
    x.copy_(values[0]), dy.copy_(values[1])
    desc = ctx.rms_norm_desc(kind.dtype, rows, width, 1e-5)
    desc.ld_x = desc.ld_y = desc.ld_sum = ld
    ctx.rms_norm(desc, x, None, w, None, y, r)
    torch.cuda.synchronize()
    wide = lambda t: t.double().cpu()  # noqa: E731
    _, (want, off), (want_r, off_r) = ref.norm(kind, wide(values[0]), None, wide(weight), 1e-5, 0.0)
    near(wide(y), want, off + kind.rounding(want, off))
    near(wide(r), want_r, off_r)
    ctx.rms_norm_backward(desc, x, w, r, dy, None, y, dw)
    torch.cuda.synchronize()
    (dx, off_x), (want_w, off_w) = ref.norm_gradients(kind, wide(values[0]), wide(weight), wide(r), wide(values[1]), None, 0.0)
    near(wide(y), dx, off_x)
    near(wide(dw), want_w, off_w)


def test_8_bits_beyond_32_bits(ctx):
    kind, rows, width, ld = KINDS["fp16"], 3, 1000, (1 << 31) + 32
    v = torch.randn(rows, width, generator=torch.Generator().manual_seed(9)).to(kind.t)
    x, q, back, scales = far(rows, width, ld, kind.t), far(rows, pitch(width), ld, torch.int8), far(rows, width, ld, kind.t), torch.empty(rows, device="cuda")
    x.copy_(v)
    ctx.quantize_int8(kind.dtype, rows, width, x, ld, q, ld, scales)
    ctx.dequantize_int8(kind.dtype, rows, width, q, ld, scales, back, ld)
    torch.cuda.synchronize()
    wide = lambda t: t.double().cpu()  # noqa: E731
    ref.check_int8(wide(q), wide(scales), v.double(), 0.0, width, True)
    want = wide(q)[:, :width] * wide(scales)[:, None]
    near(wide(back), want, kind.rounding(want))


@pytest.mark.parametrize("shape,ld_x,ld_w,ld_y", [
    ((3, 50, 40), 1 << 31, 1 << 27, 1 << 31), ((300, 300, 96), (1 << 23) - 16, (1 << 23) - 16, 1 << 24), ((200, 300, 12000), (1 << 23) - 16, 1 << 14, 1 << 25),
    ((500, 4000, 1000), 9 << 20, 1 << 12, 9 << 20), ((900, 4000, 1000), 5 << 20, 1 << 12, 5 << 20),
    ((2000, 4090, 1000), 5 << 19, 1 << 12, 5 << 19), ((3600, 3700, 192), 5 << 18, 5 << 18, 5 << 18)],
    ids=["few", "64", "split", "128x64", "128", "128x256", "256"])
def test_linear_beyond_32_bits(ctx, shape, ld_x, ld_w, ld_y):
    """tensors of more than 4 GiB each but the weights of some"""
    kind, (m, n, k) = KINDS["bf16"], shape
    gen = torch.Generator().manual_seed(m)
    ops = [torch.randint(-127, 128, (rows, k), generator=gen).to(torch.int8) for rows in (m, n)]
    x, w, y = far(m, pitch(k), ld_x, torch.int8), far(n, pitch(k), ld_w, torch.int8), far(m, n, ld_y, kind.t)
    for to, v in ((x, ops[0]), (w, ops[1])):
        to.copy_(torch.nn.functional.pad(v, (0, pitch(k) - k)))
    sx, sw = torch.rand(m, generator=gen), torch.rand(n, generator=gen)
    ctx.linear_int8(ctx.linear_int8_desc(kind.dtype, m, k, n, ld_x, ld_w, ld_y), x, sx.cuda(), w, sw.cuda(), None, y)
    torch.cuda.synchronize()
    near(y.double().cpu(), *ref.linear(kind, ops[0].double(), sx.double(), ops[1].double(), sw.double(), None))
