"""Every form that the products of the gated block and of its gradients have: tiles, waves, operands straight into LDS, through registers or on copies, split
sums, both gradients in one launch.  The library says which form a size takes, so a size that moves to another one is found out.  All results are
compared with 64 bits."""
import pytest

import ffn_reference as ref
from ffn_plan import D_W, D_X, FORWARD, plan
from reference_model_amd import Context, capi
from test_gpu_gated_ffn import KINDS

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

REGISTERS, STRAIGHT, COPIED, COPIED_REGISTERS = (0, 0), (1, 0), (1, 1), (0, 1)    # (straight into LDS, on copies)
# product, (rows, columns, waves of a tile), operands, one launch, split sum, (rows, d, f)
FORMS = [
    (FORWARD, (128, 128, 4), REGISTERS, 0, False, (130, 129, 8200)),
    (FORWARD, (128, 128, 4), REGISTERS, 0, True, (130, 2057, 4100)),
    (FORWARD, (128, 128, 8), REGISTERS, 0, True, (70, 1030, 40)),
    (FORWARD, (128, 128, 8), STRAIGHT, 0, True, (70, 1032, 40)),
    (FORWARD, (128, 128, 8), COPIED, 0, False, (3100, 129, 2570)),
    (FORWARD, (256, 128, 8), STRAIGHT, 0, False, (130, 200, 8200)),
    (FORWARD, (256, 128, 8), STRAIGHT, 0, True, (130, 2056, 4100)),
    (FORWARD, (256, 128, 8), COPIED, 0, False, (2600, 1030, 777)),
    (FORWARD, (256, 256, 8), STRAIGHT, 0, False, (400, 16, 8200)),
    (FORWARD, (256, 256, 8), COPIED, 0, False, (4100, 129, 1000)),
    (D_X, (128, 128, 4), REGISTERS, 0, True, (400, 2057, 4100)),
    (D_X, (128, 128, 8), REGISTERS, 0, False, (2600, 777, 777)),
    (D_X, (128, 128, 8), REGISTERS, 0, True, (130, 391, 8200)),
    (D_X, (128, 128, 8), REGISTERS, 1, True, (70, 129, 520)),
    (D_X, (128, 128, 8), STRAIGHT, 0, False, (1300, 2056, 1400)),
    (D_X, (128, 128, 8), STRAIGHT, 0, True, (400, 1032, 3100)),
    (D_X, (128, 128, 8), COPIED, 0, False, (4100, 391, 777)),
    (D_X, (128, 128, 8), COPIED, 0, True, (3100, 391, 777)),
    (D_X, (256, 128, 8), STRAIGHT, 0, False, (3100, 2056, 301)),
    (D_X, (256, 128, 8), STRAIGHT, 0, True, (130, 2056, 5200)),
    (D_X, (256, 128, 8), COPIED, 0, False, (4100, 1030, 301)),
    (D_X, (256, 128, 8), COPIED, 0, True, (4100, 129, 2050)),
    (D_X, (256, 256, 8), STRAIGHT, 0, False, (4100, 2056, 520)),
    (D_X, (256, 256, 8), STRAIGHT, 0, True, (2050, 2056, 3100)),
    (D_X, (256, 256, 8), COPIED, 0, False, (4100, 2057, 40)),
    (D_X, (256, 256, 8), COPIED, 0, True, (2050, 2057, 3100)),
    (D_W, (128, 128, 4), REGISTERS, 0, False, (1, 9, 16400)),
    (D_W, (128, 128, 4), REGISTERS, 0, True, (4100, 4099, 301)),
    (D_W, (128, 128, 8), REGISTERS, 0, False, (1300, 1030, 1400)),
    (D_W, (128, 128, 8), REGISTERS, 0, True, (4100, 2057, 40)),
    (D_W, (128, 128, 8), REGISTERS, 1, True, (1000, 129, 40)),
    (D_W, (128, 128, 8), STRAIGHT, 0, False, (70, 2056, 4100)),
    (D_W, (128, 128, 8), STRAIGHT, 0, True, (3100, 2056, 301)),
    (D_W, (128, 128, 8), COPIED, 0, False, (1700, 391, 2050)),
    (D_W, (128, 128, 8), COPIED, 0, True, (1700, 257, 2050)),
    (D_W, (256, 128, 8), STRAIGHT, 0, False, (400, 1032, 3100)),
    (D_W, (256, 128, 8), STRAIGHT, 0, True, (4100, 2056, 520)),
    (D_W, (256, 128, 8), COPIED, 0, False, (777, 2057, 1000)),
    (D_W, (256, 128, 8), COPIED, 0, True, (2600, 129, 3100)),
    (D_W, (256, 256, 8), STRAIGHT, 0, False, (130, 2056, 3100)),
    (D_W, (256, 256, 8), COPIED, 0, False, (130, 391, 8200)),
    (D_W, (256, 256, 8), COPIED, 0, True, (4100, 129, 8200)),
    # rows of dg and du too far apart for the offsets of loads straight into LDS
    (D_X, (128, 128, 8), REGISTERS, 0, True, (20, 16, 2_100_000)),
    (D_X, (128, 128, 8), COPIED_REGISTERS, 0, True, (40, 3, 2_100_000)),
    (D_W, (128, 128, 4), COPIED_REGISTERS, 0, False, (40, 3, 2_100_000)),
]


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def near(got, want, off):
    bad = ~((got.double() - want).abs() <= off)
    at = bad.nonzero()
    assert not len(at), f"{len(at)} of {bad.numel()}, first at {at[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- {off[bad][0]}"


def rounding(kind, want, off):
    return off + kind.unit * (want.abs() + off) + kind.tiny


def times(a, b):
    """a b^T in 64 bits"""
    return torch.mm(a.double(), b.double().t().contiguous())


@pytest.mark.parametrize("form", FORMS, ids=lambda c: "-".join(map(str, (("forward", "d_x", "d_w")[c[0]], *c[1], *c[2], c[3], int(c[4]), *c[5]))))
@pytest.mark.parametrize("name", list(KINDS))
def test_form(ctx, name, form):
    product, tile, operands, together, split, (m, d, f) = form
    kind, t = KINDS[name], TYPES[name]
    p = plan(product, m, d, f, dtype=kind.dtype)
    assert (p[:3], (p.direct, p.copies), p.together, p.splits > 1) == (tile, operands, together, split)
    gen = torch.Generator(device="cuda").manual_seed(m + d + f)
    made = lambda std, *s: (torch.randn(*s, device="cuda", generator=gen) * std).to(t)  # noqa: E731
    none = lambda *s: torch.full(s, float("nan"), device="cuda", dtype=t)  # noqa: E731
    x, gate, up = made(1, m, d), made(d ** -0.5, f, d), made(d ** -0.5, f, d)
    assert all(v.data_ptr() % 16 == 0 for v in (x, gate, up))
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    desc, terms = ctx.gated_ffn_desc(kind.dtype, capi.ACT_SILU, m, d, f), lambda n: (n + 2) * ref.EPS  # noqa: E731
    if product == FORWARD:
        h, g, u = none(m, f), none(m, f), none(m, f)
        ctx.gated_ffn(desc, x, gate, up, h, g, u)
        assert ctx.sync() == capi.VALID and ctx.last_kernel == "gated_ffn"
        wg, wu = times(x, gate), times(x, up)
        og, ou = (terms(d) * times(x.abs(), w.abs()) for w in (gate, up))
        value = wg * torch.sigmoid(wg)
        wh, oh = value * wu, (1.13 * og + 16 * ref.EPS * value.abs()) * (wu.abs() + ou) + value.abs() * ou
        for got, want, off in ((h, wh, oh + ref.EPS * wh.abs()), (g, wg, og), (u, wu, ou)):
            near(got, want, rounding(kind, want, off))
        alone = none(m, f)
        ctx.gated_ffn(desc, x, gate, up, alone)
        assert ctx.sync() == capi.VALID and torch.equal(alone, h)
        return
    g, u, dh, out = made(1, m, f), made(1, m, f), made(0.5, m, f), [none(m, d), none(f, d), none(f, d)]
    ctx.gated_ffn_backward(desc, x, gate, up, g, u, dh, *out)
    assert ctx.sync() == capi.VALID
    s = torch.sigmoid(g.double())
    du, dg = dh.double() * g.double() * s, dh.double() * u.double() * s * (1 + g.double() * (1 - s))
    odu, odg = 17 * ref.EPS * du.abs(), 16 * ref.EPS * (dh.double() * u.double()).abs() * (1 + g.double().abs())
    odu, odg = rounding(kind, du, odu), rounding(kind, dg, odg)
    if product == D_X:
        gate_t, up_t = gate.t().contiguous(), up.t().contiguous()
        want = times(dg, gate_t) + times(du, up_t)
        off = times(odg, gate_t.abs()) + times(odu, up_t.abs()) + terms(2 * f) * (times(dg.abs() + odg, gate_t.abs()) + times(du.abs() + odu, up_t.abs()))
        near(out[0], want, rounding(kind, want, off))
    else:
        x_t = x.t().contiguous()
        for got, v, ov in ((out[1], dg, odg), (out[2], du, odu)):
            v_t, ov_t = v.t().contiguous(), ov.t().contiguous()
            want = times(v_t, x_t)
            off = times(ov_t, x_t.abs()) + terms(m) * times(v_t.abs() + ov_t, x_t.abs())
            near(got, want, rounding(kind, want, off))
