"""The gated feed-forward block in 16 bits and its gradients against the same in 64 bits: one row to several tiles of them, sizes that end inside
tiles and pieces, rows that begin at any element, lengths of zero, sums that are split, numbers that are none, and what is refused."""
import numpy as np
import pytest

import ffn_reference as ref
from reference_model_amd import Context, TmiError, capi

pytestmark = pytest.mark.gpu
KINDS = {k: ref.Kind(k) for k in ("fp16", "bf16")}


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class Rows:
    """a matrix on the GPU whose rows lie `gap` elements further apart than they are long, the first of them `lead` elements into its buffer; what lies
    around them is no number, and stays as it is"""

    def __init__(self, ctx, kind, shape, values=None, gap=0, lead=0):
        self.ctx, self.kind, self.shape, self.ld, self.lead = ctx, kind, shape, shape[1] + gap, lead
        self.host = kind.narrow(np.full(lead + shape[0] * self.ld + 8, np.nan))
        if values is not None:
            self.inside(self.host)[:] = kind.narrow(values)
        self.dev = ctx.upload(self.host, kind.dtype)
        self.at = self.dev.ptr + 2 * lead

    def inside(self, buf):
        return buf[self.lead:self.lead + self.shape[0] * self.ld].reshape(self.shape[0], self.ld)[:, :self.shape[1]]

    def stored(self):
        """the matrix now; nothing beside it was written"""
        now = self.dev.numpy().astype(self.host.dtype, copy=False).copy()
        got = self.inside(now).copy()
        self.inside(now)[:] = self.inside(self.host)
        assert np.array_equal(now.view(np.uint16), self.host.view(np.uint16)), "written outside the tensor"
        return got

    def values(self):
        return self.kind.wide(self.stored())

    def free(self):
        self.dev.free()


def near(got, want_and_off):
    want, off = want_and_off
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]} +- {off[bad][0]}"


def operands(kind, m, d, f, seed):
    rng = np.random.default_rng(seed)
    back = lambda v: kind.wide(kind.narrow(v))  # noqa: E731
    return back(rng.normal(0, 1, (m, d))), back(rng.normal(0, 1 / np.sqrt(max(d, 1)), (f, d))), back(rng.normal(0, 1 / np.sqrt(max(d, 1)), (f, d)))


def forward(ctx, kind, name, x, gate, up, save=True, gap=0, lead=0):
    m, d, f = x.shape[0], x.shape[1], gate.shape[0]
    dev = [Rows(ctx, kind, v.shape, v, gap, lead) for v in (x, gate, up)]
    out = [Rows(ctx, kind, (m, f), None, gap, lead) for _ in range(3 if save else 1)]
    desc = ctx.gated_ffn_desc(kind.dtype, ref.ACTS[name], m, d, f, d + gap, d + gap, f + gap)
    ctx.gated_ffn(desc, *(t.at for t in dev), *(t.at for t in out))
    assert ctx.sync() == capi.VALID
    got = [t.stored() for t in out]
    for t in dev + out:
        t.free()
    return got


def backward(ctx, kind, name, x, gate, up, g, u, dh, gap=0, lead=0, dx=True, dw=True):
    m, d, f = x.shape[0], x.shape[1], gate.shape[0]
    dev = [Rows(ctx, kind, v.shape, v, gap, lead) for v in (x, gate, up, g, u, dh)]
    out = [Rows(ctx, kind, s, None, gap, lead) for s in ((m, d), (f, d), (f, d))]
    desc = ctx.gated_ffn_desc(kind.dtype, ref.ACTS[name], m, d, f, d + gap, d + gap, f + gap)
    ctx.gated_ffn_backward(desc, *(t.at for t in dev), out[0].at if dx else None, *(t.at if dw else None for t in out[1:]))
    assert ctx.sync() == capi.VALID
    got = [t.stored() for t in out]
    for t in dev + out:
        t.free()
    return got


# rows, d, f, gap, lead: whole tiles, then everything that ends inside one
SHAPES = [(1, 64, 64, 0, 0), (1, 1, 1, 0, 0), (1, 130, 33, 0, 0), (3, 200, 129, 8, 8), (16, 256, 48, 0, 0), (17, 8, 100, 3, 1), (40, 777, 65, 0, 0), (64, 128, 7, 1, 0),
          (65, 64, 64, 0, 0), (128, 192, 130, 0, 0), (100, 65, 66, 0, 0), (129, 72, 200, 8, 8), (257, 40, 136, 1, 3), (300, 7, 9, 0, 0), (66, 520, 24, 16, 0)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_forward(ctx, kind, shape):
    kind, (m, d, f, gap, lead) = KINDS[kind], shape
    x, gate, up = operands(kind, m, d, f, m + d)
    for name in ("silu", "gelu_tanh") if m > 64 else ref.ACTS:
        got = forward(ctx, kind, name, x, gate, up, gap=gap, lead=lead)
        for v, want in zip(got, ref.gated(kind, name, x, gate, up)):
            near(kind.wide(v), want)
    alone = forward(ctx, kind, name, x, gate, up, save=False, gap=gap, lead=lead)
    assert np.array_equal(alone[0].view(np.uint16), got[0].view(np.uint16))


@pytest.mark.parametrize("name", list(ref.ACTS))
@pytest.mark.parametrize("kind", list(KINDS))
def test_every_activation_over_its_range(ctx, kind, name):
    """g from -30 to 30 in steps of the type, and far out, on the kernel of many rows; u = 1"""
    kind = KINDS[kind]
    g = np.concatenate([np.linspace(-30, 30, 501), [-6e4, -300, 300, 6e4, 0, -0.0]])
    x = np.zeros((80, 8))
    x[:, 0] = 1
    gate, up = np.zeros((len(g), 8)), np.zeros((len(g), 8))
    gate[:, 0], up[:, 0] = kind.wide(kind.narrow(g)), 1
    for rows in (1, 80):
        got = forward(ctx, kind, name, x[:rows], gate, up)
        for v, want in zip(got, ref.gated(kind, name, x[:rows], gate, up)):
            near(kind.wide(v), want)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] != 40] + [(1, 300, 200, 0, 0), (700, 64, 64, 0, 0), (1100, 24, 40, 0, 0)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_gradients(ctx, kind, shape):
    kind, (m, d, f, gap, lead) = KINDS[kind], shape
    x, gate, up = operands(kind, m, d, f, m + f)
    rng = np.random.default_rng(m)
    g, u, dh = (kind.wide(kind.narrow(v)) for v in (x @ gate.T, x @ up.T, rng.normal(0, 0.5, (m, f))))
    for name in ("silu", "gelu") if m > 64 else ref.ACTS:
        got = backward(ctx, kind, name, x, gate, up, g, u, dh, gap, lead)
        for v, want in zip(got, ref.gated_gradients(kind, name, x, gate, up, g, u, dh)):
            near(kind.wide(v), want)
    bits = [v.view(np.uint16) for v in got]
    only_x = backward(ctx, kind, name, x, gate, up, g, u, dh, gap, lead, dw=False)
    only_w = backward(ctx, kind, name, x, gate, up, g, u, dh, gap, lead, dx=False)
    assert np.array_equal(only_x[0].view(np.uint16), bits[0]) and all(np.array_equal(w.view(np.uint16), b) for w, b in zip(only_w[1:], bits[1:]))
    assert np.isnan(kind.wide(only_x[1])).all() and np.isnan(kind.wide(only_w[0])).all()


@pytest.mark.parametrize("name", list(ref.ACTS))
@pytest.mark.parametrize("kind", list(KINDS))
def test_gradients_against_differences(ctx, kind, name):
    """the change of sum(dh h) along a direction.  x of -1, 0, 1 and weights in eighths up to 1 make pre-activations that both types hold, so the
    gradients are those of the formula at these operands but for their own roundings; the step of the differences leaves 1e-7 of them."""
    kind, (m, d, f) = KINDS[kind], (70, 16, 40)
    rng = np.random.default_rng(7)
    x = rng.integers(-1, 2, (m, d)).astype(np.float64)
    gate, up = (rng.integers(-8, 9, (f, d)) / 8.0 for _ in range(2))
    gate[:, 0], x[:, 0] = 1 / 8, 1    # no pre-activation is 0, where relu has no derivative: an odd number of eighths
    gate[:, 1:] = np.round(gate[:, 1:] * 4) / 4
    dh = kind.wide(kind.narrow(rng.normal(0, 0.5, (m, f))))
    g, u = x @ gate.T, x @ up.T
    assert np.array_equal(kind.wide(kind.narrow(g)), g) and np.array_equal(kind.wide(kind.narrow(u)), u) and (g != 0).all()
    got = [kind.wide(v) for v in backward(ctx, kind, name, x, gate, up, g, u, dh)]
    offs = [off for _, off in ref.gated_gradients(kind, name, x, gate, up, g, u, dh)]

    def loss(a, b, c):
        return (dh * ref.act(name, a @ b.T)[0] * (a @ c.T)).sum()

    step = 1e-5
    for i, shape in enumerate(((m, d), (f, d), (f, d))):
        for _ in range(4):
            v = rng.normal(0, 1, shape)
            at = [[x, gate, up], [x, gate, up]]
            at[0][i], at[1][i] = at[0][i] + step * v, at[1][i] - step * v
            slope = (loss(*at[0]) - loss(*at[1])) / (2 * step)
            assert abs((got[i] * v).sum() - slope) <= (offs[i] * np.abs(v)).sum() + 1e-6 * np.abs(got[i] * v).sum()


@pytest.mark.parametrize("kind", list(KINDS))
def test_long_sums_of_few_tiles_are_split(ctx, kind):
    """65 rows and 70 features over 4100, and gradients over 2 x 2500 features and over 3000 rows"""
    kind = KINDS[kind]
    x, gate, up = operands(kind, 65, 4104, 70, 3)
    for v, want in zip(forward(ctx, kind, "silu", x, gate, up), ref.gated(kind, "silu", x, gate, up)):
        near(kind.wide(v), want)
    for m, d, f in ((70, 72, 2500), (2900, 64, 30)):
        x, gate, up = operands(kind, m, d, f, 4)
        rng = np.random.default_rng(5)
        g, u, dh = (kind.wide(kind.narrow(v)) for v in (x @ gate.T, x @ up.T, rng.normal(0, 0.5, (m, f))))
        got = backward(ctx, kind, "silu", x, gate, up, g, u, dh)
        for v, want in zip(got, ref.gated_gradients(kind, "silu", x, gate, up, g, u, dh)):
            near(kind.wide(v), want)
        again = backward(ctx, kind, "silu", x, gate, up, g, u, dh)
        assert all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(got, again))


@pytest.mark.parametrize("kind", list(KINDS))
def test_large_tiles(ctx, kind):
    """enough tiles of 256 x 256, none of them whole at the edges; a sample of the results"""
    kind, (m, d, f) = KINDS[kind], (2600, 72, 2568)
    x, gate, up = operands(kind, m, d, f, 8)
    pick_m, pick_f = np.r_[0:40, 250:262, 2550:2600], np.r_[0:40, 120:136, 2540:2568]
    got = forward(ctx, kind, "gelu", x, gate, up)
    for v, want in zip(got, ref.gated(kind, "gelu", x[pick_m], gate[pick_f], up[pick_f])):
        near(kind.wide(v[np.ix_(pick_m, pick_f)]), want)
    # gradients: many rows and features in turn, so that each product has its large tiles
    for m, d, f in ((4100, 2600, 40), (72, 2600, 2100)):
        x, gate, up = operands(kind, m, d, f, 9)
        rng = np.random.default_rng(6)
        g, u, dh = (kind.wide(kind.narrow(v)) for v in (x @ gate.T, x @ up.T, rng.normal(0, 0.5, (m, f))))
        got = backward(ctx, kind, "silu", x, gate, up, g, u, dh)
        for v, want in zip(got, ref.gated_gradients(kind, "silu", x, gate, up, g, u, dh)):
            near(kind.wide(v), want)


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("kind", list(KINDS))
def test_infinite_and_nan_operands_stay_in_their_rows(ctx, kind, rows):
    kind = KINDS[kind]
    x, gate, up = operands(kind, rows, 72, 40, 11)
    x[0, 3], gate[7, 5], up[9, 71] = np.inf, np.nan, -np.inf
    with np.errstate(invalid="ignore"):
        g, u = x @ gate.T, x @ up.T
        h = ref.act("silu", g)[0] * u
    got_h, got_g, got_u = (kind.wide(v) for v in forward(ctx, kind, "silu", x, gate, up))
    for got, want in ((got_g, g), (got_u, u)):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        inf = np.isinf(want)
        assert inf.any() and np.array_equal(got[inf], want[inf])
    fine = np.isfinite(h)
    assert fine.sum() > 1 and np.array_equal(np.isfinite(got_h), fine)


@pytest.mark.parametrize("kind", list(KINDS))
def test_lengths_of_zero(ctx, kind):
    kind = KINDS[kind]
    for rows in (3, 80):    # a sum of nothing is 0, and act(0) * 0
        for v in forward(ctx, kind, "sigmoid", np.zeros((rows, 0)), np.zeros((5, 0)), np.zeros((5, 0))):
            assert not kind.wide(v).any()
    forward(ctx, kind, "silu", np.zeros((0, 8)), np.zeros((5, 8)), np.zeros((5, 8)))
    forward(ctx, kind, "silu", np.zeros((4, 8)), np.zeros((0, 8)), np.zeros((0, 8)))
    assert ctx.last_kernel == "empty"
    none = np.zeros((0, 5))
    got = backward(ctx, kind, "silu", np.zeros((0, 8)), np.ones((5, 8)), np.ones((5, 8)), none, none, none)
    assert not kind.wide(got[1]).any() and not kind.wide(got[2]).any()
    none = np.zeros((4, 0))
    got = backward(ctx, kind, "silu", np.ones((4, 8)), np.zeros((0, 8)), np.zeros((0, 8)), none, none, none)
    assert not kind.wide(got[0]).any()


def test_what_is_refused(ctx):
    buf = ctx.upload(np.zeros(4096, np.float16))
    p = buf.ptr
    ok = (capi.FP16, capi.ACT_SILU, 4, 16, 8)

    def refused(say, desc, args, fn=ctx.gated_ffn):
        with pytest.raises(TmiError) as e:
            fn(desc, *args)
        assert e.value.status == capi.ERROR and say in e.value.message

    fine, back = (p,) * 4, (p,) * 9
    for fn, args in ((ctx.gated_ffn, fine), (ctx.gated_ffn_backward, back)):
        refused("data type", ctx.gated_ffn_desc(capi.FP32, *ok[1:]), args, fn)
        refused("activation", ctx.gated_ffn_desc(capi.FP16, 0, *ok[2:]), args, fn)
        refused("activation", ctx.gated_ffn_desc(capi.FP16, 6, *ok[2:]), args, fn)
        for bad in ((-1, 16, 8), (4, -1, 8), (4, 16, -1)):
            refused("negative", ctx.gated_ffn_desc(*ok[:2], *bad), args, fn)
        for ld in ((15, 16, 8), (16, 15, 8), (16, 16, 7), (-16, 16, 8)):
            refused("apart", ctx.gated_ffn_desc(*ok, *ld), args, fn)
        refused("more than", ctx.gated_ffn_desc(*ok[:2], 1 << 30, 16, 8), args, fn)
        refused("null tensor", ctx.gated_ffn_desc(*ok), (None,) + args[1:], fn)
        refused("aligned", ctx.gated_ffn_desc(*ok), (p + 1,) + args[1:], fn)
    refused("without the other", ctx.gated_ffn_desc(*ok), fine + (p, None))
    refused("without the other", ctx.gated_ffn_desc(*ok), back[:7] + (p, None), ctx.gated_ffn_backward)
    refused("null tensor", ctx.gated_ffn_desc(*ok), back[:5] + (None,) + back[6:], ctx.gated_ffn_backward)
    ctx.gated_ffn_backward(ctx.gated_ffn_desc(*ok), *back[:6], None, None, None)
    assert ctx.last_kernel == "empty" and ctx.sync() == capi.VALID
