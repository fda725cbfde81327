"""The feed-forward operators at the ends of their ranges: rows that lie gigabytes apart, pre-activations far out."""
import math

import numpy as np
import pytest

import ffn_reference as ref
from reference_model_amd import Context, capi
from test_gpu_gated_ffn import KINDS, backward, near

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
