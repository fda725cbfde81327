"""Gradients of the root-mean-square norm against the formula's in 64 bits, and against differences: widths of one element to rows that are read twice, rows
that begin at any element, more rows than there are workgroups, each gradient alone, and results in place of operands."""
import pytest

torch = pytest.importorskip("torch")

import projection_reference as ref  # noqa: E402
from projection_reference import KINDS, Held, near  # noqa: E402
from reference_model_amd import Context, TmiError, capi  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def operands(kind, rows, width, seed, past=True):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=gen).to(kind.t).double()  # noqa: E731
    s, dy = new(rows, width), new(rows, width)
    r = (1 / (s.square().mean(1) + 1e-5).sqrt()).float().double() if width else torch.ones(rows).double()
    return s, (1 + 0.3 * torch.randn(width, generator=gen)).to(kind.t).double(), r, dy, new(rows, width) if past else None


class Call:
    def __init__(self, ctx, kind, s, weight, r, dy, d_sum, offset=0.0, gap=0, lead=0):
        self.ctx, self.kind, shape = ctx, kind, s.shape
        hold = lambda v: None if v is None else Held(shape, kind.t, gap, lead, v)  # noqa: E731
        self.s, self.dy, self.d_sum = hold(s), hold(dy), hold(d_sum)
        self.weight, self.rstd = Held((1, shape[1]), kind.t, 0, lead, weight[None]), Held((1, shape[0]), torch.float32, 0, 0, r[None])
        self.dx, self.dw = Held(shape, kind.t, gap, lead), Held((1, shape[1]), kind.t, 0, lead)
        ld = shape[1] + gap
        self.desc = ctx.rms_norm_desc(kind.dtype, shape[0], shape[1], 1e-5, offset, ld, 0, ld, ld)

    def run(self, dx=True, dw=True):
        self.ctx.rms_norm_backward(self.desc, self.s.at, self.weight.at, self.rstd.at, self.dy.at, self.d_sum and self.d_sum.at, self.dx.at if dx else None,
                                   self.dw.at if dw else None)
        assert self.ctx.sync() == capi.VALID and self.ctx.last_kernel == "rms_norm_backward"


SIZES = [(1, 1), (3, 2), (2, 5), (70, 8), (33, 64), (17, 127), (300, 128), (19, 130), (3, 257), (6, 512), (50, 514), (9, 1000), (2, 1024), (3, 1030), (4, 2047),
         (5, 2056), (1, 4096), (3, 4111), (2, 8200), (3, 12001), (2, 16384), (2, 16391), (5, 20000), (1, 40003)]


@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_gradients(ctx, name, shape):
    kind = KINDS[name]
    for i, (gap, lead) in enumerate(((0, 0), (1, 0), (0, 1), (8, 8)) if shape[1] < 4096 else ((0, 0), (3, 1))):
        ops, offset = operands(kind, *shape, i, past=i % 2 == 0), float(i % 3 == 1)
        call = Call(ctx, kind, *ops, offset, gap, lead)
        call.run()
        for got, want in zip((call.dx.values(), call.dw.values()[0]), ref.norm_gradients(kind, *ops, offset)):
            near(got, *want)
        # each alone, and again: the same bits
        both = call.dx.m.clone(), call.dw.m.clone()
        for dx, dw in ((True, False), (False, True)):
            one = Call(ctx, kind, *ops, offset, gap, lead)
            one.run(dx, dw)
            assert torch.equal(one.dx.m, both[0]) if dx else (one.dx.values() == ref.CANARY).all()
            assert torch.equal(one.dw.m, both[1]) if dw else (one.dw.values() == ref.CANARY).all()


@pytest.mark.parametrize("shape", [(20000, 24), (3000, 200), (2100, 1030), (1500, 4104), (1100, 9000), (700, 17000)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_more_rows_than_workgroups(ctx, name, shape):
    kind = KINDS[name]
    ops = operands(kind, *shape, 5)
    call = Call(ctx, kind, *ops)
    call.run()
    for got, want in zip((call.dx.values(), call.dw.values()[0]), ref.norm_gradients(kind, *ops, 0.0)):
        near(got, *want)


@pytest.mark.parametrize("shape", [(4, 100), (3, 1001), (2, 4097), (3, 20001)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_results_in_place_of_operands(ctx, name, shape):
    kind = KINDS[name]
    ops = operands(kind, *shape, 6)
    want = Call(ctx, kind, *ops, gap=1)
    want.run()
    for where in ("s", "dy", "d_sum"):
        call = Call(ctx, kind, *ops, gap=1)
        call.dx = getattr(call, where)
        call.run()
        assert torch.equal(call.dx.m, want.dx.m) and torch.equal(call.dw.m, want.dw.m)


@pytest.mark.parametrize("shape", [(9000, 24), (5000, 61), (5000, 200), (2000, 255)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_short_rows_that_share_a_wave(ctx, name, shape):
    test_gradients(ctx, name, shape)
    test_results_in_place_of_operands(ctx, name, shape)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(5, 24), (3, 300)], ids=lambda s: "x".join(map(str, s)))
def test_against_differences(ctx, shape, residual):
    """the loss a . y + b . sum of the forward operator: d(loss) along a direction is the difference of its values, (f(+h) - f(-h)) / 2h.  In 32 bits a value
    is off by about 2^-21 of the sum of its terms' sizes, and the third derivative adds h^2 / 6 of itself: h = 2^-7 leaves 2^-13 of the sizes."""
    kind, (rows, width) = KINDS["fp32"], shape
    gen = torch.Generator().manual_seed(2)
    new = lambda *s: torch.randn(*s, generator=gen).float().double()  # noqa: E731
    x, other, w, a, b = new(*shape), new(*shape), 1 + 0.3 * new(width), new(*shape), new(*shape)
    desc = ctx.rms_norm_desc(kind.dtype, rows, width, 1e-5)

    def forward(x, w):
        dev = [Held(shape, kind.t, 0, 0, v) for v in (x, other)] + [Held((1, width), kind.t, 0, 0, w[None])]
        s, y, r = Held(shape, kind.t), Held(shape, kind.t), Held((1, rows), torch.float32)
        ctx.rms_norm(desc, dev[0].at, dev[1].at if residual else None, dev[2].at, s.at, y.at, r.at)
        assert ctx.sync() == capi.VALID
        return s, y, r

    def loss(x, w):
        s, y, _ = forward(x, w)
        terms = torch.cat(((a * y.values()).reshape(-1), (b * s.values()).reshape(-1) if residual else torch.zeros(0).double()))
        return terms.sum(), terms.abs().sum()

    s, _, r = forward(x, w)
    call = Call(ctx, kind, s.values(), w, r.values()[0], a, b if residual else None)
    call.run()
    dx, dw, h = call.dx.values(), call.dw.values()[0], 2.0 ** -7
    for seed in range(3):
        vx, vw = new(*shape), new(width)
        ahead, size = loss(x + h * vx, w + h * vw)
        behind, _ = loss(x - h * vx, w - h * vw)
        want = (ahead - behind) / (2 * h)
        assert abs(float((dx * vx).sum() + (dw * vw).sum() - want)) <= 2.0 ** -12 * float(size + (dx * vx).abs().sum() + (dw * vw).abs().sum())


def test_numbers_that_are_none(ctx):
    """NaN stays in its row of d_x, and in its column of d_weight"""
    kind = KINDS["bf16"]
    ops = operands(kind, 4, 600, 3)
    clean = Call(ctx, kind, *ops)
    clean.run()
    ops[3][2, 17] = float("nan")
    call = Call(ctx, kind, *ops)
    call.run()
    dx, dw, was = call.dx.values(), call.dw.values()[0], clean.dw.values()[0]
    assert dx[2].isnan().all() and torch.equal(dx[[0, 1, 3]], clean.dx.values()[[0, 1, 3]])
    assert dw[17].isnan() and torch.equal(dw[:17], was[:17]) and torch.equal(dw[18:], was[18:])


def test_no_rows_leave_zeros(ctx):
    kind = KINDS["fp16"]
    dw = Held((1, 70), kind.t)
    ctx.rms_norm_backward(ctx.rms_norm_desc(kind.dtype, 0, 70, 0.0), None, None, None, None, None, None, dw.at)
    assert ctx.sync() == capi.VALID and (dw.values() == 0).all()
    ctx.rms_norm_backward(ctx.rms_norm_desc(kind.dtype, 3, 0, 0.0), None, None, None, None, None, None, dw.at)
    assert ctx.last_kernel == "empty"
    ctx.rms_norm_backward(ctx.rms_norm_desc(kind.dtype, 3, 8, 0.0), None, None, None, None, None, None, None)
    assert ctx.last_kernel == "empty" and ctx.sync() == capi.VALID


def test_refusals(ctx):
    kind = KINDS["fp16"]
    ops = operands(kind, 4, 24, 1)
    call = Call(ctx, kind, *ops)
    good = [call.s.at, call.weight.at, call.rstd.at, call.dy.at, call.d_sum.at, call.dx.at, call.dw.at]

    def refused(args=good, **changed):
        d = ctx.rms_norm_desc(kind.dtype, 4, 24, 1e-5)
        for k, v in changed.items():
            setattr(d, k, v)
        with pytest.raises(TmiError) as e:
            ctx.rms_norm_backward(d, *args)
        assert e.value.status == capi.ERROR
        return e.value.message

    assert "data type" in refused(dtype=capi.INT16) and "negative" in refused(rows=-1) and "negative" in refused(width=-2)
    for name in ("ld_x", "ld_sum", "ld_y"):
        assert "apart" in refused(**{name: 23})
    odd = call.s.buf.view(torch.uint8)[1:]
    for at in range(7):
        assert "aligned" in refused([odd if i == at else v for i, v in enumerate(good)])
    for at in range(4):
        assert "null" in refused([None if i == at else v for i, v in enumerate(good)])
    assert ctx.sync() == capi.VALID and (call.dx.values() == ref.CANARY).all() and (call.dw.values() == ref.CANARY).all()
