"""Where the operators on the way into a projection can go wrong and a bound on roundings would not show it: halves on the way into 8 bits, products beyond
the range of 32 bits there, scales that 32 bits hardly hold, the widest rows, and gradients that are whole numbers, so that no row may be lost."""
import pytest

torch = pytest.importorskip("torch")

import projection_reference as ref  # noqa: E402
from projection_reference import KINDS, Held, held8, near  # noqa: E402
from reference_model_amd import Context, capi  # noqa: E402
from test_gpu_rms_norm import Call, operands  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


@pytest.mark.parametrize("width", [128, 500, 1000, 4096, 20000])
@pytest.mark.parametrize("name", list(KINDS))
def test_halves_out_of_the_norm_go_to_even(ctx, name, width):
    """a row of s = a and weights 1, 3, 5 .. 253 with 254 the largest: every quotient 127 a w / (254 a) is half an odd number, whatever a"""
    kind = KINDS[name]
    odd = 2.0 * (torch.arange(width) % 127).double() + 1
    odd[5] = 254
    a = torch.cat((torch.arange(1, 256), torch.arange(1, 256) * 2.0 ** -9)).double()
    sign = torch.where(torch.arange(width) % 3 == 0, -1.0, 1.0).double()
    want = 2 * torch.round(odd / 4) * sign    # w / 2 to the nearest even number
    want[5] = 127 * sign[5]
    for offset, residual in ((0.0, False), (1.0, True)):
        x = a[:, None] * sign
        call = Call(ctx, kind, x / 2 if residual else x, x / 2 if residual else None, odd - offset, 0.0, offset)
        call.norm8()
        assert torch.equal(call.q.values()[:, :width], want.expand(len(a), width))


@pytest.mark.parametrize("shape", [(3000, 40), (800, 1000), (200, 4096), (100, 4111), (40, 20000)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_halves_of_any_maximum_go_to_even(ctx, name, shape):
    """v = s (offset + weight) as 32 bits hold it, in rows that hold their maximum's half many times: 254 v and whole multiples of the maximum are exact in 64 bits"""
    kind, (rows, width), seen = KINDS[name], shape, 0
    for seed, offset in ((1, 0.0), (2, 1.0)):
        x, residual, weight = operands(kind, rows, width, seed, residual=bool(offset))
        weight[::3] = 1 - offset
        x[:, 0] = 1 + x[:, 1].abs() * 4
        x = x.to(kind.t).double()
        x[:, 3::6] = x[:, :1] * torch.where(torch.arange(3, width, 6) % 4 == 3, 0.5, -0.5)
        if residual is not None:
            residual[:, 3::6] = residual[:, :1] * torch.where(torch.arange(3, width, 6) % 4 == 3, 0.5, -0.5)
        call = Call(ctx, kind, x, residual, weight, offset=offset)
        call.norm8()
        s = x.float() if residual is None else x.float() + residual.float()
        v = (s * (offset + weight.float())).double()
        most, q = v.abs().amax(1, keepdim=True), call.q.values()[:, :width]
        k = torch.round(v * 254 / most)
        half = (k * most == v * 254) & (k % 2 != 0)
        seen += int(half.sum())
        assert torch.equal(q[half], 2 * torch.round(k / 4)[half])
        # (v and the maximum are as they stand: what is left is the reciprocal's last place, two halves of one)
        assert ((q - v * 127 / most).abs() <= 0.5 + 127 * 2 * ref.EPS).all()
    assert seen > 0


def check_norm8(ctx, kind, x, weight, eps):
    call = Call(ctx, kind, x, None, weight, eps)
    call.norm8()
    y = ref.norm(kind, x, None, weight, eps, 0.0)[1][0]
    ref.check_int8(call.q.values(), call.scales.values()[0], y, (ref.depth(x.shape[1]) / 2 + 10) * ref.EPS, x.shape[1])


# x and weights times these: squares that leave the range beside products that do not, both, products alone at either end, and rows that are next to nothing
FACTORS = [(2.0 ** 70, 2.0 ** 50), (2.0 ** 110, 2.0 ** 100), (2.0 ** 120, 2.0 ** 120), (2.0 ** 100, 2.0 ** -110), (2.0 ** 40, 2.0 ** 110), (2.0 ** -30, 2.0 ** -80),
           (2.0 ** -60, 2.0 ** 100), (2.0 ** -122, 2.0 ** -60), (2.0 ** -120, 2.0 ** -100), (2.0 ** -122, 2.0 ** 110)]


@pytest.mark.parametrize("width", [48, 1000, 4096, 20000])
@pytest.mark.parametrize("factors", FACTORS, ids=lambda f: f"{f[0]:.0e}-{f[1]:.0e}")
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_products_beyond_the_range_into_8_bits(ctx, name, factors, width):
    """the scale is a number wherever y is; every other row is of the usual size"""
    kind = KINDS[name]
    x, _, weight = operands(kind, 6, width, 12, residual=False)
    x[::2] *= factors[0]
    weight = (weight * factors[1]).to(kind.t).double()
    for eps in (0.0, 1e-5):
        if eps and factors[0] < 2.0 ** -100:
            continue    # (y of those rows is nothing beside eps)
        check_norm8(ctx, kind, x.to(kind.t).double(), weight, eps)


@pytest.mark.parametrize("width", [48, 1000, 4096, 20000])
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_rows_that_span_the_range_into_8_bits(ctx, name, width):
    """one element makes the squares leave the range, and the others, of every size, make the row's maximum"""
    kind = KINDS[name]
    for first, of_first, others, of_others in ((2.0 ** 66, 0.0, 2.0 ** -69, 2.0 ** 100), (2.0 ** 127, 2.0 ** -10, 8.0, 2.0 ** 125), (2.0 ** 127, 0.0, 2.0 ** -40, 2.0 ** 40),
                                               (2.0 ** -42, 0.0, 2.0 ** -100, 2.0 ** -20), (2.0 ** -10, 0.0, 2.0 ** -90, 2.0 ** -10)):
        x, _, weight = operands(kind, 5, width, 13, residual=False)
        x, weight = x * others, weight * of_others
        x[:, 7], weight[7] = first, of_first
        check_norm8(ctx, kind, x.to(kind.t).double(), weight.to(kind.t).double(), 0.0)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_gradients_of_the_widest_rows(ctx, name):
    """more columns than 2^32 threads have at 32 threads a column; whole numbers and halves, exact in every type"""
    kind, rows, width = KINDS[name], 2, (1 << 27) + 40
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = lambda: torch.randint(-3, 4, (rows, width), generator=gen, device="cuda", dtype=torch.int8).to(kind.t)  # noqa: E731
    s, dy, w = new(), new(), torch.ones(width, device="cuda", dtype=kind.t)
    r = torch.tensor([0.5, 2.0], device="cuda")
    dw = torch.full((width + 8,), ref.CANARY, device="cuda", dtype=kind.t)
    ctx.rms_norm_backward(ctx.rms_norm_desc(kind.dtype, rows, width, 1e-5), s, w, r, dy, None, None, dw)
    assert ctx.sync() == capi.VALID and (dw[width:] == ref.CANARY).all()
    want = s[0] * dy[0] * 0.5 + s[1] * dy[1] * 2    # (at most 22.5 in halves)
    assert torch.equal(dw[:width], want)


@pytest.mark.parametrize("shape", [(1, 24), (31, 24), (20000, 24), (9000, 24), (9001, 64), (5000, 61), (5000, 200), (4999, 255), (3000, 300), (2100, 1030), (1500, 4104),
                                   (1025, 2048), (1100, 9000), (700, 17000), (65, 17000), (300, 40003)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_every_row_counts_once_in_the_weights_gradient(ctx, name, shape):
    """terms of +-1 and +-2: their sums are whole numbers that 32 bits hold exactly whatever their order, and a result is the sum rounded once.  A lost or repeated
    row is off by one or two in every column, in fp32 and fp16 always (sums below 2048), in bf16 where a sum is below 256, as most are."""
    kind, (rows, width) = KINDS[name], shape
    gen = torch.Generator().manual_seed(rows + width)
    one = lambda: torch.randint(0, 2, shape, generator=gen) * 2.0 - 1  # noqa: E731
    s, dy, r = one() * 4, one() * (torch.randint(0, 2, (rows, 1), generator=gen) + 1), torch.full((rows,), 0.25)
    want = (s * dy).double().sum(0) / 4
    assert want.abs().max() < 2048 and (want.abs() < 256).any()
    for gap, lead in ((0, 0), (3, 1)):
        hold = lambda v: Held(shape, kind.t, gap, lead, v)  # noqa: E731, B023
        ds, ddy, dx = hold(s), hold(dy), hold(torch.zeros(shape))
        w, dw = Held((1, width), kind.t, 0, lead, torch.ones(1, width)), Held((1, width), kind.t, 0, lead)
        ld = width + gap
        desc = ctx.rms_norm_desc(kind.dtype, rows, width, 1e-5, 0.0, ld, 0, ld, ld)
        for to in (dx.at, None):
            dw.m.fill_(ref.CANARY)
            ctx.rms_norm_backward(desc, ds.at, w.at, r.cuda(), ddy.at, None, to, dw.at)
            assert ctx.sync() == capi.VALID and torch.equal(dw.values()[0], want.to(kind.t).double())
        # and in d_x: dy / 4 - s / 16 mean(dy s / 4), whose mean is a whole number over width
        mean = (s * dy).double().sum(1, keepdim=True) / 4 / width
        dx_want = (dy.double() - s.double() / 4 * mean) / 4
        off = 4 * ref.EPS * (dy.double().abs() + mean.abs())
        near(dx.values(), dx_want, off + kind.rounding(dx_want, off))


@pytest.mark.parametrize("width", [7, 48, 4096, 20000])
@pytest.mark.parametrize("size", [2.0 ** -118, 2.0 ** -125, 2.0 ** -130, 2.0 ** -140, 2.0 ** -149])
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_scales_that_32_bits_hardly_hold(ctx, name, size, width):
    """a scale is the nearest number that 32 bits hold, below 2^-126 a multiple of 2^-149; where that is 0 so is q, else q is as of any row"""
    kind = KINDS[name]
    x, _, weight = operands(kind, 5, width, 14, residual=False)

    def check(q, scales, v, rel, off_q):
        most = v.abs().amax(1)
        assert ((scales - most / 127).abs() <= rel * most / 127 + 2.0 ** -150 * (1 + 2.0 ** -20)).all()
        assert (q[scales == 0] == 0).all() and (q[:, width:] == 0).all()
        live = scales > 0
        t = v[live] * 127 / most[live][:, None]
        assert ((q[live][:, :width] - t).abs() <= 0.5 + off_q).all() and (q[live].abs().amax(1) == 127).all()

    small = (x * size).to(kind.t).double()
    dev, q, scales = Held(x.shape, kind.t, 0, 0, small), held8(5, width), Held((1, 5), torch.float32)
    ctx.quantize_int8(kind.dtype, 5, width, dev.at, 0, q.at, 0, scales.at)
    assert ctx.sync() == capi.VALID
    # (127 over the maximum is rounded, and the product joins its rounding to a whole number: 2^-17 of 127)
    check(q.values(), scales.values()[0], small, 2 * ref.EPS, 0.0 if name == "bf16" else 2.0 ** -17)
    # the same sizes out of the norm: weights that small
    w = (weight * size).to(kind.t).double()
    call = Call(ctx, kind, x, None, w)
    call.norm8()
    check(call.q.values(), call.scales.values()[0], ref.norm(kind, x, None, w, 1e-5, 0.0)[1][0], (ref.depth(width) / 2 + 10) * ref.EPS, 127 * 8 * ref.EPS)
