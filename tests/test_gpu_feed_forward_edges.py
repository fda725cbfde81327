"""The feed-forward operators at the ends of their ranges: rows that lie gigabytes apart."""
import pytest

from reference_model_amd import Context, capi

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
