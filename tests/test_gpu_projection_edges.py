"""Where the operators on the way into a projection can go wrong and a bound on roundings would not show it: halves on the way into 8 bits."""
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
