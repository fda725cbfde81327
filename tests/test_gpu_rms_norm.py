"""The root-mean-square norm with the residual's addition, in 16 and 32 bits and in 8, and rows into 8 bits and back, against 64 bits: widths of one
element to rows that no workgroup's registers hold, rows that begin at any element, numbers whose squares leave the range, and numbers that are none."""
import pytest

torch = pytest.importorskip("torch")

import projection_reference as ref  # noqa: E402
from projection_reference import KINDS, Held, held8, near  # noqa: E402
from reference_model_amd import Context, TmiError, capi  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def operands(kind, rows, width, seed, residual=True):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=gen).to(kind.t).double()  # noqa: E731
    return new(rows, width), new(rows, width) * 2 if residual else None, (1 + 0.3 * torch.randn(width, generator=gen)).to(kind.t).double()


class Call:
    """one call's tensors on the GPU"""

    def __init__(self, ctx, kind, x, residual, weight, eps=EPS, offset=0.0, gap=0, lead=0):
        self.ctx, self.kind, self.shape, self.width = ctx, kind, x.shape, x.shape[1]
        hold = lambda v: None if v is None else Held(self.shape, kind.t, gap, lead, v)  # noqa: E731
        self.x, self.residual, self.weight = hold(x), hold(residual), Held((1, self.width), kind.t, 0, lead, weight[None])
        self.sum, self.y = (Held(self.shape, kind.t, gap, lead) for _ in range(2))
        self.rstd = Held((1, x.shape[0]), torch.float32)
        ld = self.width + gap
        self.desc = ctx.rms_norm_desc(kind.dtype, x.shape[0], self.width, eps, offset, ld, ld, ld, ld)
        self.desc8 = ctx.rms_norm_desc(kind.dtype, x.shape[0], self.width, eps, offset, ld, ld, ld, 0)

    def norm(self, keep=True):
        self.ctx.rms_norm(self.desc, self.x.at, self.residual and self.residual.at, self.weight.at, self.sum.at if keep else None, self.y.at,
                          self.rstd.at if keep else None)
        assert self.ctx.sync() == capi.VALID and self.ctx.last_kernel == "rms_norm"

    def norm8(self, more=0, keep=True):
        self.q, self.scales = held8(self.shape[0], self.width, more), Held((1, self.shape[0]), torch.float32)
        self.desc8.ld_y = self.q.ld
        self.ctx.rms_norm_int8(self.desc8, self.x.at, self.residual and self.residual.at, self.weight.at, self.sum.at if keep else None, self.q.at,
                               self.scales.at)
        assert self.ctx.sync() == capi.VALID and self.ctx.last_kernel == "rms_norm_int8"


SIZES = [(1, 1), (3, 2), (2, 3), (5, 7), (4, 8), (7, 9), (33, 64), (17, 127), (40, 128), (19, 130), (3, 257), (6, 512), (5, 514), (9, 1000), (2, 1024), (3, 1030),
         (4, 2047), (3, 2048), (2, 2056), (1, 4096), (3, 4111), (2, 8192), (2, 8200), (1, 12001), (2, 16384), (1, 16385), (2, 20008), (1, 40003)]
PLACES = [(0, 0), (1, 0), (0, 1), (3, 1), (8, 8), (2, 2)]


@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_norm(ctx, name, shape):
    kind = KINDS[name]
    places = PLACES if shape[1] < 4096 else PLACES[:4:3]
    for i, (gap, lead) in enumerate(places):
        x, residual, weight = operands(kind, *shape, i, residual=i % 3 != 1)
        offset = 1.0 if i % 2 else 0.0
        call = Call(ctx, kind, x, residual, weight, EPS, offset, gap, lead)
        call.norm()
        (s, off_s), (y, off_y), (r, off_r) = ref.norm(kind, x, residual, weight, EPS, offset)
        near(call.sum.values(), s, off_s)
        near(call.y.values(), y, off_y + kind.rounding(y, off_y))
        near(call.rstd.values()[0], r, off_r)
        first = call.y.m.clone()
        call.norm(keep=False)
        assert torch.equal(call.y.m, first)
        assert torch.equal(call.x.values(), x) and torch.equal(call.weight.values()[0], weight)


@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_norm_in_8_bits(ctx, name, shape):
    kind, (rows, width) = KINDS[name], shape
    places = PLACES if width < 4096 else PLACES[:4:3]
    for i, (gap, lead) in enumerate(places):
        x, residual, weight = operands(kind, *shape, i + 9, residual=i % 3 != 1)
        if rows > 2:
            x[1] = 0
            if residual is not None:
                residual[1] = 0
        call = Call(ctx, kind, x, residual, weight, EPS, 0.0, gap, lead)
        call.norm8(more=16 * (i % 3))
        (s, off_s), (y, _), _ = ref.norm(kind, x, residual, weight, EPS, 0.0)
        near(call.sum.values(), s, off_s)
        q, scales = call.q.values(), call.scales.values()[0]
        ref.check_int8(q, scales, y, (ref.depth(width) / 2 + 10) * ref.EPS, width)
        # and what these stand for
        back = Held(shape, kind.t, gap, lead)
        ctx.dequantize_int8(kind.dtype, rows, width, call.q.at, call.q.ld, call.scales.at, back.at, width + gap)
        assert ctx.sync() == capi.VALID and ctx.last_kernel == "dequantize_int8"
        # (a product rounded to 32 bits and then to the type, or at once)
        want = scales[:, None] * q[:, :width]
        near(back.values(), want, ref.EPS * want.abs() + kind.rounding(want, ref.EPS * want.abs()))


@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_rows_into_8_bits(ctx, name, shape):
    kind, (rows, width) = KINDS[name], shape
    for i, (gap, lead) in enumerate(PLACES if width < 4096 else PLACES[:4:3]):
        x, _, _ = operands(kind, *shape, i + 20, residual=False)
        if rows > 2:
            x[2] = 0
        dev, q, scales = Held(shape, kind.t, gap, lead, x), held8(rows, width, 16 * (i % 2)), Held((1, rows), torch.float32)
        ctx.quantize_int8(kind.dtype, rows, width, dev.at, dev.ld, q.at, q.ld, scales.at)
        assert ctx.sync() == capi.VALID and ctx.last_kernel == "quantize_int8"
        ref.check_int8(q.values(), scales.values()[0], x, 0.0, width, ties=name != "fp32")


@pytest.mark.parametrize("name", ["fp16", "bf16"])
def test_halves_go_to_even(ctx, name):
    """every quotient of a largest number and the numbers up to it: of an even one the number half as large gives 63.5, of a multiple of 254 every odd multiple
    of its 254th gives one"""
    kind = KINDS[name]
    digits = 11 if name == "fp16" else 8
    most = torch.cat((torch.arange(2, 2 ** digits, 2), torch.arange(254, 2 ** digits, 254))).double()
    shape = len(most), 2 ** digits
    x = torch.arange(2 ** digits).double()[None].minimum(most[:, None]) * 2.0 ** -7
    x[:, ::2] *= -1
    dev, q, scales = Held(shape, kind.t, 0, 0, x), held8(*shape), Held((1, shape[0]), torch.float32)
    ctx.quantize_int8(kind.dtype, *shape, dev.at, 0, q.at, 0, scales.at)
    assert ctx.sync() == capi.VALID
    assert ref.check_int8(q.values(), scales.values()[0], x, 0.0, shape[1], ties=True) >= len(most)


@pytest.mark.parametrize("rows,width", [(70001, 8), (40000, 128), (9000, 200), (5000, 1030), (3000, 4100)])
def test_more_rows_than_places(ctx, rows, width):
    kind = KINDS["bf16"]
    x, residual, weight = operands(kind, rows, width, 3)
    call = Call(ctx, kind, x, residual, weight)
    call.norm()
    (s, off_s), (y, off_y), (r, off_r) = ref.norm(kind, x, residual, weight, EPS, 0.0)
    near(call.sum.values(), s, off_s)
    near(call.y.values(), y, off_y + kind.rounding(y, off_y))
    near(call.rstd.values()[0], r, off_r)
    call.norm8()
    ref.check_int8(call.q.values(), call.scales.values()[0], y, (ref.depth(width) / 2 + 10) * ref.EPS, width)


@pytest.mark.parametrize("shape", [(4, 100), (3, 1000), (2, 4097), (2, 20001)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_results_in_place_of_operands(ctx, name, shape):
    kind = KINDS[name]
    x, residual, weight = operands(kind, *shape, 5)
    want = Call(ctx, kind, x, residual, weight, gap=1)
    want.norm()
    for sum_in, y_in in (("x", "residual"), ("residual", "x"), ("residual", None), (None, "x")):
        call = Call(ctx, kind, x, residual, weight, gap=1)
        to = lambda where, own: own if where is None else getattr(call, where)  # noqa: E731, B023
        call.sum, call.y = to(sum_in, call.sum), to(y_in, call.y)
        call.norm()
        assert torch.equal(call.sum.m, want.sum.m) and torch.equal(call.y.m, want.y.m) and torch.equal(call.rstd.m, want.rstd.m)
    want.norm8()
    call = Call(ctx, kind, x, residual, weight, gap=1)
    call.sum = call.x
    call.norm8()
    assert torch.equal(call.q.m, want.q.m) and torch.equal(call.scales.m, want.scales.m) and torch.equal(call.sum.m, want.sum.m)


@pytest.mark.parametrize("shape", [(600, 24), (600, 61), (300, 200), (300, 255), (300, 1030), (257, 1101), (300, 1536), (260, 520), (270, 767)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_rows_that_share_a_wave_or_have_three_pieces_a_lane(ctx, name, shape):
    """enough of them for every workgroup to have several"""
    test_norm(ctx, name, shape)
    test_norm_in_8_bits(ctx, name, shape)
    test_rows_into_8_bits(ctx, name, shape)
    test_results_in_place_of_operands(ctx, name, shape)


@pytest.mark.parametrize("width", [48, 1000, 4096, 20000])
@pytest.mark.parametrize("size", [2.0 ** 120, 2.0 ** 70, 2.0 ** -70, 2.0 ** -110])
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_squares_beyond_the_range(ctx, name, size, width):
    """rows whose squares overflow or vanish in 32 bits, among others that are as usual"""
    kind = KINDS[name]
    x, residual, weight = operands(kind, 6, width, 8)
    x[::2] *= size
    residual[::2] *= size
    for eps in (0.0, EPS):
        call = Call(ctx, kind, x, residual, weight, eps)
        call.norm()
        (s, off_s), (y, off_y), (r, off_r) = ref.norm(kind, x, residual, weight, eps, 0.0)
        near(call.sum.values(), s, off_s)
        near(call.y.values(), y, off_y + kind.rounding(y, off_y) + 2.0 ** -140)
        near(call.rstd.values()[0], r, off_r + 2.0 ** -149)
        call.norm8()
        ref.check_int8(call.q.values(), call.scales.values()[0], y, (ref.depth(width) / 2 + 10) * ref.EPS, width)


@pytest.mark.parametrize("width", [48, 4096, 20000])
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_tiny_rows_and_weights_into_8_bits(ctx, name, width):
    kind = KINDS[name]
    x, residual, weight = operands(kind, 4, width, 8)
    small = (x * 2.0 ** -115).to(kind.t).double()
    dev, q, scales = Held(x.shape, kind.t, 0, 0, small), held8(4, width), Held((1, 4), torch.float32)
    ctx.quantize_int8(kind.dtype, 4, width, dev.at, 0, q.at, 0, scales.at)
    assert ctx.sync() == capi.VALID
    ref.check_int8(q.values(), scales.values()[0], small, 0.0, width, ties=name == "bf16")
    # weights so small that the products lose their digits, weights of zero, and products that leave the range where the results do not
    for factor, of_x in ((2.0 ** -110, 1.0), (0.0, 1.0), (2.0 ** 100, 2.0 ** 60), (2.0 ** 60, 2.0 ** 100)):
        w, big = (weight * factor).to(kind.t).double(), (x * of_x).to(kind.t).double()
        call = Call(ctx, kind, big, None, w)
        call.norm8()
        y = ref.norm(kind, big, None, w, EPS, 0.0)[1][0]
        ref.check_int8(call.q.values(), call.scales.values()[0], y, (ref.depth(width) / 2 + 10) * ref.EPS, width)
    # squares that vanish beside weights that do not
    w, little = (weight * 2.0 ** 90).to(kind.t).double(), (x * 2.0 ** -60).to(kind.t).double()
    call = Call(ctx, kind, little, None, w, 0.0)
    call.norm8()
    ref.check_int8(call.q.values(), call.scales.values()[0], ref.norm(kind, little, None, w, 0.0, 0.0)[1][0], (ref.depth(width) / 2 + 10) * ref.EPS, width)


@pytest.mark.parametrize("width", [40, 700, 3000, 17000])
@pytest.mark.parametrize("name", list(KINDS))
def test_numbers_that_are_none(ctx, name, width):
    """they stay in their rows; a row of zeros is zeros"""
    kind = KINDS[name]
    x, residual, weight = operands(kind, 5, width, 4)
    clean = Call(ctx, kind, x, residual, weight)
    clean.norm()
    clean.norm8()
    x[1, width // 2], x[2, 3], residual[3, width - 1] = float("nan"), float("inf"), float("-inf")
    x[4], residual[4] = 0, 0
    call = Call(ctx, kind, x, residual, weight)
    call.norm()
    y = call.y.values()
    assert torch.equal(y[0], clean.y.values()[0]) and (y[4] == 0).all()
    assert y[1].isnan().all() and y[2, 3].isnan() and y[3, width - 1].isnan() and (y[2, 4:] == 0).all() and (y[3, :-1] == 0).all()
    call.norm8()
    q, scales = call.q.values(), call.scales.values()[0]
    assert torch.equal(q[0], clean.q.values()[0]) and scales[0] == clean.scales.values()[0, 0]
    assert (q[1:] == 0).all() and not scales[1:4].isfinite().any() and scales[4] == 0
    dev, q, scales = Held(x.shape, kind.t, 0, 0, x), held8(5, width), Held((1, 5), torch.float32)
    ctx.quantize_int8(kind.dtype, 5, width, dev.at, 0, q.at, 0, scales.at)
    assert ctx.sync() == capi.VALID
    q, scales = q.values(), scales.values()[0]
    assert (q[[1, 2, 4]] == 0).all() and scales[1].isnan() and scales[2].isinf() and scales[4] == 0 and (q[[0, 3]].abs().amax(1) == 127).all()


def test_calls_with_nothing_to_do(ctx):
    kind = KINDS["bf16"]
    x, residual, weight = operands(kind, 3, 16, 1)
    call = Call(ctx, kind, x, residual, weight)
    none = ctx.rms_norm_desc(kind.dtype, 0, 16, EPS)
    ctx.rms_norm(none, None, None, None, None, None)
    ctx.rms_norm_int8(none, None, None, None, None, None, None)
    ctx.rms_norm(ctx.rms_norm_desc(kind.dtype, 3, 0, EPS), None, None, None, None, None)
    ctx.quantize_int8(kind.dtype, 0, 16, None, 0, None, 0, None)
    ctx.dequantize_int8(kind.dtype, 3, 0, None, 0, call.rstd.at, None, 0)
    assert ctx.last_kernel == "empty"
    # rows of no elements have scales all the same
    for name in KINDS:
        for fill in (lambda: ctx.quantize_int8(KINDS[name].dtype, 3, 0, None, 0, None, 0, call.rstd.at),  # noqa: B023
                     lambda: ctx.rms_norm_int8(ctx.rms_norm_desc(KINDS[name].dtype, 3, 0, EPS), None, None, None, None, None, call.rstd.at)):  # noqa: B023
            call.rstd.m.fill_(5)
            fill()
            assert ctx.sync() == capi.VALID and (call.rstd.values() == 0).all()
    assert (call.y.values() == ref.CANARY).all()


def refused(fn, *args):
    with pytest.raises(TmiError) as e:
        fn(*args)
    assert e.value.status == capi.ERROR
    return e.value.message


def test_refusals(ctx):
    kind = KINDS["fp16"]
    x, residual, weight = operands(kind, 4, 24, 1)
    call = Call(ctx, kind, x, residual, weight)
    q, scales = held8(4, 24), Held((1, 4), torch.float32)

    def desc(**changed):
        d = ctx.rms_norm_desc(kind.dtype, 4, 24, EPS)
        for k, v in changed.items():
            setattr(d, k, v)
        return d

    norm = lambda d, *a: refused(ctx.rms_norm, d, *(a or (call.x.at, None, call.weight.at, None, call.y.at, None)))  # noqa: E731
    norm8 = lambda d, *a: refused(ctx.rms_norm_int8, d, *(a or (call.x.at, None, call.weight.at, None, q.at, scales.at)))  # noqa: E731
    for both in (norm, norm8):
        assert "data type" in both(desc(dtype=capi.INT8))
        assert "negative" in both(desc(rows=-1)) and "negative" in both(desc(width=-1))
        assert "more than one call" in both(desc(width=(1 << 28) + 1))
        assert "eps" in both(desc(eps=-1e-6)) and "eps" in both(desc(eps=float("nan"))) and "eps" in both(desc(eps=float("inf")))
        assert "weight_offset" in both(desc(weight_offset=float("inf")))
        for name in ("ld_x", "ld_residual", "ld_sum"):
            assert "apart" in both(desc(**{name: 23})) and "apart" in both(desc(**{name: -24}))
    assert "apart" in norm(desc(ld_y=23)) and "apart" in norm8(desc(ld_y=24)) and "apart" in norm8(desc(ld_y=16)) and "apart" in norm8(desc(ld_y=40))
    odd = call.x.buf.view(torch.uint8)[1:]
    for at in range(5):
        args = [call.x.at, None, call.weight.at, None, call.y.at, None]
        args[at] = odd
        assert "aligned" in norm(desc(), *args)
    assert "aligned" in norm(desc(), call.x.at, None, call.weight.at, None, call.y.at, call.x.at[1:])
    assert "16 bytes" in norm8(desc(), call.x.at, None, call.weight.at, None, q.buf[8:], scales.at)
    for at in (0, 2, 4):
        args = [call.x.at, None, call.weight.at, None, call.y.at, None]
        args[at] = None
        assert "null" in norm(desc(), *args)
    assert "null" in norm8(desc(), call.x.at, None, call.weight.at, None, q.at, None)
    into = lambda *a: refused(ctx.quantize_int8, *a)  # noqa: E731
    back = lambda *a: refused(ctx.dequantize_int8, *a)  # noqa: E731
    h = kind.dtype
    assert "data type" in into(capi.INT32, 4, 24, call.x.at, 0, q.at, 0, scales.at) and "data type" in back(capi.INT32, 4, 24, q.at, 0, scales.at, call.y.at, 0)
    assert "negative" in into(h, -4, 24, call.x.at, 0, q.at, 0, scales.at) and "negative" in back(h, 4, -24, q.at, 0, scales.at, call.y.at, 0)
    assert "apart" in into(h, 4, 24, call.x.at, 20, q.at, 0, scales.at) and "apart" in into(h, 4, 24, call.x.at, 0, q.at, 24, scales.at)
    assert "apart" in back(h, 4, 24, q.at, 33, scales.at, call.y.at, 0) and "apart" in back(h, 4, 24, q.at, 0, scales.at, call.y.at, 1)
    assert "null" in into(h, 4, 24, None, 0, q.at, 0, scales.at) and "null" in into(h, 4, 24, call.x.at, 0, q.at, 0, None)
    assert "null" in back(h, 4, 24, q.at, 0, None, call.y.at, 0) and "null" in back(h, 4, 24, None, 0, scales.at, call.y.at, 0)
    assert "aligned" in into(h, 4, 24, odd, 0, q.at, 0, scales.at) and "16 bytes" in into(h, 4, 24, call.x.at, 0, q.buf[1:], 0, scales.at)
    assert "aligned" in back(h, 4, 24, q.at, 0, call.x.at[1:], call.y.at, 0) and "16 bytes" in back(h, 4, 24, q.buf[4:], 0, scales.at, call.y.at, 0)
    assert ctx.sync() == capi.VALID and (call.y.values() == ref.CANARY).all() and (q.values() == ref.CANARY).all()
