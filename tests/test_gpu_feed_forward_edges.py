"""The feed-forward operators at the ends of their ranges: rows that lie gigabytes apart, pre-activations far out, gradients whose
factors fp16 does not hold."""
import math

import numpy as np
import pytest

import ffn_reference as ref
from reference_model_amd import Context, capi
from test_gpu_gated_ffn import KINDS, Rows, backward, forward, near

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def test_gradients_of_rows_that_lie_4_gib_apart_over_a_tile(ctx):
    """128 rows of 2 x 8500096 features of dg and du: the last lies 2^32 bytes behind the first.  Small whole numbers in a few features, so that every sum is exact."""
    m, d, f, t = 128, 8, 8_500_000, torch.float16
    features = torch.cat((torch.arange(40), torch.arange(f // 2, f // 2 + 40), torch.arange(f - 40, f))).cuda()
    gen = torch.Generator(device="cuda").manual_seed(4)
    whole = lambda *s: torch.randint(-2, 3, s, device="cuda", generator=gen).to(t)  # noqa: E731
    gate, up, x, ones, dh = whole(f, d), whole(f, d), whole(m, d), torch.ones(m, f, device="cuda", dtype=t), torch.zeros(m, f, device="cuda", dtype=t)
    dh[:, features] = whole(m, len(features))
    dx, d_gate, d_up = torch.full_like(x, float("nan")), torch.full_like(gate, float("nan")), torch.full_like(up, float("nan"))
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    ctx.gated_ffn_backward(ctx.gated_ffn_desc(capi.FP16, capi.ACT_RELU, m, d, f), x, gate, up, ones, ones, dh, dx, d_gate, d_up)
    assert ctx.sync() == capi.VALID
    # g = u = 1: dg = du = dh
    few = dh[:, features].double()
    assert torch.equal(dx.double(), torch.mm(few, (gate.double() + up.double())[features]))
    want = torch.zeros(f, d, device="cuda", dtype=torch.float64)
    want[features] = torch.mm(few.t().contiguous(), x.double())
    assert torch.equal(d_gate.double(), want) and torch.equal(d_up.double(), want)


def slope_off(name, g, slope):
    """How far act'(g) may be off in 32 bits: 32 units in 2^24 of what it is summed from, of which every factor has all its digits; an exponent z multiplies the
    rounding of its argument by |z|, taken four times (GELU: z = g^2 / 2; its tanh form: z = 2 sqrt(2 / pi) (g + 0.044715 g^3))."""
    with np.errstate(over="ignore", under="ignore"):
        if name == "relu":
            return 0 * g
        if name == "gelu":
            z, parts = g * g / 2, ref.act(name, -np.abs(g))[0] / -np.maximum(np.abs(g), 1e-30) + np.abs(g) * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
            return ref.EPS * ((32 + 4 * z) * parts + 32 * np.abs(slope))
        z, factor = g, 1.0
        if name == "gelu_tanh":
            z, factor = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3), 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
        p, q = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
        if name == "sigmoid":
            return ref.EPS * 32 * slope
        return ref.EPS * (32 + (4 * np.abs(z) if name == "gelu_tanh" else 0)) * (np.minimum(p, q) + np.abs(g) * p * q * factor) + ref.EPS * 32 * np.abs(slope)


@pytest.mark.parametrize("name", list(ref.ACTS))
@pytest.mark.parametrize("kind", list(KINDS))
def test_slopes_over_their_range(ctx, kind, name):
    """g from -30 to 30; one row whose first element is 1, u = dh = 1: the gradients of the weights are act'(g) and act(g) themselves, one term each"""
    kind = KINDS[kind]
    g = kind.wide(kind.narrow(np.r_[np.linspace(-30, 30, 601), np.linspace(9, 20, 100)]))[None]
    f, one, w = g.shape[1], np.eye(1, 8), np.zeros((g.shape[1], 8))
    _, d_gate, d_up = (kind.wide(v) for v in backward(ctx, kind, name, one, w, w, g, np.ones((1, f)), np.ones((1, f))))
    value, slope = (v[0] for v in ref.act(name, g))
    off = slope_off(name, g[0], slope)
    near(d_gate[:, 0], (slope, off + kind.rounding(slope, off)))
    off = ref.value_off(name, g[0], value)
    near(d_up[:, 0], (value, off + kind.rounding(value, off)))
    assert not d_gate[:, 1:].any() and not d_up[:, 1:].any()


# rows, d, f: both gradients in one launch with d_x's or the weights' sums split, through registers, on copies, and one after the other with d_x in parts
RANGE_SHAPES = {"split_dx": (40, 64, 1200), "split_dw": (1100, 72, 40), "registers": (70, 129, 65), "copies": (300, 7, 9), "apart": (2048, 1024, 4096)}


def fp16_operands(shape, about, seed=3):
    """dg and du beyond fp16's range on either side, or one of them beyond it and the others ordinary; the gradients are numbers that it holds"""
    kind, rng = KINDS["fp16"], np.random.default_rng(seed)
    m, d, f = shape
    of_x, of_w, of_g, of_u, of_dh = {"large": (3e-4, 1e-4, 1, 100, 3000), "tiny": (300, 300, 1e-2, 3e-3, 3e-6), "ordinary": (1, d ** -0.5, 1, 1, 0.1),
                                     "outlier": (0.05, 0.05, 1, 1, 10)}[about]
    made = lambda std, *s: kind.wide(kind.narrow(rng.normal(0, std, s)))  # noqa: E731
    x, gate, up, g, u, dh = made(of_x, m, d), made(of_w, f, d), made(of_w, f, d), made(of_g, m, f), made(of_u, m, f), made(of_dh, m, f)
    if about == "outlier":
        g[3, 5], u[3, 5], dh[3, 5] = 1, 65, 2000
    return x, gate, up, g, u, dh


def held_gradients(x, gate, up, g, u, dh, most):
    """the reference where dg and du lose, besides their rounding, at most 2^-25 of the largest of them"""
    kind = ref.Kind("fp16")
    kind.tiny = 2.0 ** -25 * most
    return [(w, off + KINDS["fp16"].tiny) for w, off in ref.gated_gradients(kind, "silu", x, gate, up, g, u, dh)]


def largest(g, u, dh):
    value, slope = ref.act("silu", g)
    return max(np.abs(dh * value).max(), np.abs(dh * u * slope).max())


@pytest.mark.parametrize("about", ["large", "tiny", "outlier"])
@pytest.mark.parametrize("where", list(RANGE_SHAPES))
def test_fp16_gradients_of_products_beyond_its_range(ctx, where, about):
    shape = RANGE_SHAPES[where]
    x, gate, up, g, u, dh = fp16_operands(shape, about)
    most = largest(g, u, dh)
    assert most > 65504 if about != "tiny" else most < 2.0 ** -22
    got = [KINDS["fp16"].wide(v) for v in backward(ctx, KINDS["fp16"], "silu", x, gate, up, g, u, dh)]
    # a sample of rows and of features
    rows, features = (np.unique(np.r_[0:min(n, 40), max(n - 40, 0):n]) for n in (shape[0], shape[2]))
    want = [held_gradients(x[rows], gate, up, g[rows], u[rows], dh[rows], most)[0], *held_gradients(x, gate[features], up[features], g[:, features], u[:, features],
                                                                                                        dh[:, features], most)[1:]]
    for v, w, pick in zip(got, want, (rows, features, features)):
        near(v[pick], w)
        assert (np.abs(w[0]) > 4 * w[1]).mean() > 0.5    # the comparison says something
    of_x = backward(ctx, KINDS["fp16"], "silu", x, gate, up, g, u, dh, dw=False)[0]
    assert np.isfinite(KINDS["fp16"].wide(of_x)).all()


def test_fp16_gradients_of_nothing_and_of_infinities(ctx):
    kind, shape = KINDS["fp16"], (40, 64, 200)
    x, gate, up, g, u, dh = fp16_operands(shape, "large")
    for v in backward(ctx, kind, "silu", x, gate, up, g, u, 0 * dh):
        assert not kind.wide(v).any()
    dh[2, 4], dh[7, 9] = np.inf, np.nan
    got = [kind.wide(v) for v in backward(ctx, kind, "silu", x, gate, up, g, u, dh)]
    dh[2, 4], dh[7, 9] = 0, 0
    want = held_gradients(x, gate, up, g, u, dh, largest(g, u, dh))
    for v, w, spoilt in zip(got, want, ((2, 7), (4, 9), (4, 9))):
        fine = np.setdiff1d(np.arange(len(v)), spoilt)
        assert not np.isfinite(v[list(spoilt)]).any()
        near(v[fine], (w[0][fine], w[1][fine]))


def test_graph_of_fp16_gradients_finds_the_range_of_every_replay():
    kind, (m, d, f) = KINDS["fp16"], (90, 200, 136)
    ctx, new = Context(0), lambda *s: torch.empty(*s, device="cuda", dtype=torch.float16)
    try:
        stream = torch.cuda.current_stream()
        ctx.set_stream(stream.cuda_stream)
        held, out = [new(m, d), new(f, d), new(f, d), new(m, f), new(m, f), new(m, f)], [new(m, d), new(f, d), new(f, d)]
        desc = ctx.gated_ffn_desc(kind.dtype, capi.ACT_SILU, m, d, f)
        fill = lambda about, seed: [t.copy_(torch.from_numpy(v)) for t, v in zip(held, fp16_operands((m, d, f), about, seed))]  # noqa: E731
        fill("ordinary", 0)
        ctx.gated_ffn_backward(desc, *held, *out)
        assert ctx.sync() == capi.VALID
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(stream)
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            ctx.gated_ffn_backward(desc, *held, *out)
        ctx.set_stream(stream.cuda_stream)
        for seed, about in enumerate(("large", "ordinary", "tiny", "outlier", "ordinary", "tiny", "large")):
            fill(about, seed)
            ctx.gated_ffn_backward(desc, *held, *out)
            assert ctx.sync() == capi.VALID
            want = [t.clone() for t in out]
            for t in out:
                t.fill_(77)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.isfinite(b).all() and torch.equal(a, b)
    finally:
        ctx.close()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", list(KINDS))
def test_pack_given_values_of_both_types(ctx, kind, group):
    """rows that lie apart and side by side, infinite and NaN scales as they are, one row and column past whole tiles"""
    kind, rng = KINDS[kind], np.random.default_rng(group)
    for (n, k), gap in (((33, 257), 7), ((16, 128), 0), ((1, 1), 3)):
        v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.normal(0, 1, (n, -(-k // group))))
        scales[0, 0] = kind.narrow([np.inf])[0]
        scales[-1, -1] = kind.narrow([np.nan])[0]
        wide = np.full((n, k + gap), 99, np.int8)
        wide[:, :k] = v
        held, stored = ctx.upload(wide), ctx.upload(scales, kind.dtype)
        want = ref.packed(kind, v, scales, group)
        to = ctx.upload(np.full(want.size + 16, 0xA5, np.uint8))
        ctx.pack_int4(ctx.int4_desc(kind.dtype, group, n, k), held, k + gap if gap else 0, stored, to)
        assert ctx.sync() == capi.VALID
        got = to.numpy().view(np.uint8)
        assert np.array_equal(got[:want.size], want) and (got[want.size:] == 0xA5).all()
        for t in (held, stored, to):
            t.free()


@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("kind", list(KINDS))
def test_products_of_no_columns_and_of_no_rows(ctx, kind, rows):
    """sums of nothing with 4-bit weights are 0 on the kernels of few and of more rows"""
    kind, out = KINDS[kind], Rows(ctx, KINDS[kind], (rows, 40))
    desc = ctx.int4_desc(kind.dtype, 64, 40, 0)
    ctx.matvec_int4(desc, rows, None, 0, None, out.at, 0)
    assert ctx.sync() == capi.VALID and not out.values().any()
    again = Rows(ctx, kind, (rows, 40))
    ctx.gated_ffn_int4(desc, capi.ACT_SIGMOID, rows, None, 0, None, None, again.at, 0)
    assert ctx.sync() == capi.VALID and not again.values().any()


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("kind", list(KINDS))
def test_subnormal_operands_count(ctx, kind, rows):
    """x below the least normal number of its type, weights that bring the sums back"""
    kind, rng = KINDS[kind], np.random.default_rng(rows)
    least, k, n = (2.0 ** -133, 72, 24) if kind.bf16 else (2.0 ** -24, 72, 24)
    x = rng.integers(-60, 61, (rows, k)) * least    # exact
    gate, up = (kind.wide(kind.narrow(rng.normal(0, 2.0 ** 60 if kind.bf16 else 100, (n, k)))) for _ in range(2))
    for v, want in zip(forward(ctx, kind, "relu", x, gate, up)[1:], ref.gated(kind, "relu", x, gate, up)[1:]):
        near(kind.wide(v), want)
        assert (np.abs(want[0]) > 4 * want[1]).mean() > 0.9
    v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.uniform(0.5, 1, (n, 3)) * (2.0 ** 60 if kind.bf16 else 100))
    dev, held, out = Rows(ctx, kind, (rows, k), x), ctx.upload(ref.packed(kind, v, scales, 32)), Rows(ctx, kind, (rows, n))
    ctx.matvec_int4(ctx.int4_desc(kind.dtype, 32, n, k), rows, dev.at, 0, held, out.at, 0)
    assert ctx.sync() == capi.VALID
    near(out.values(), ref.product(kind, x, ref.weights(kind, v, scales, 32)))
