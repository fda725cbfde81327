"""Where the operators on the way into a projection can go wrong and a bound on roundings would not show it: halves on the way into 8 bits, products beyond
the range of 32 bits there, and the widest rows."""
import pytest

torch = pytest.importorskip("torch")

import projection_reference as ref  # noqa: E402
from projection_reference import KINDS  # noqa: E402
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
