"""The linear layer on 8-bit activations and weights against exact sums: few rows and many, sizes that end inside tiles and blocks, sums that are split,
rows that lie apart, all results' types, the largest sums that 32 bits hold, and scales that are no numbers."""
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


def whole(v, more=0):
    """rows in 8 bits on the GPU, filled up with zeros to whole 16 bytes and `more`, which is no part of the rows"""
    rows, width = v.shape
    pitch = -(-width // 16) * 16
    h = Held((rows, pitch), torch.int8, more, 0, torch.nn.functional.pad(v, (0, pitch - width)))
    return h


def operands(m, n, k, seed, lowest=-127):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randint(lowest, 128, (m, k), generator=gen).to(torch.int8), torch.rand(m, generator=gen) * 0.05 + 0.001,
            torch.randint(lowest, 128, (n, k), generator=gen).to(torch.int8), torch.rand(n, generator=gen) * 0.01 + 0.0001)


def run(ctx, kind, x, x_scales, w, w_scales, bias=None, more=0, gap=0, lead=0):
    dx, dw, out = whole(x, more), whole(w, 2 * more), Held((x.shape[0], w.shape[0]), kind.t, gap, lead)
    sx, sw = Held((1, x.shape[0]), torch.float32, 0, 1, x_scales[None]), Held((1, w.shape[0]), torch.float32, 0, 3, w_scales[None])
    b = None if bias is None else Held((1, w.shape[0]), kind.t, 0, lead, bias[None])
    desc = ctx.linear_int8_desc(kind.dtype, x.shape[0], x.shape[1], w.shape[0], dx.ld, dw.ld, out.ld)
    ctx.linear_int8(desc, dx.at, sx.at, dw.at, sw.at, b and b.at, out.at)
    assert ctx.sync() == capi.VALID and ctx.last_kernel == "linear_int8"
    return out.values()


def check(ctx, kind, m, n, k, seed, bias=False, **place):
    x, sx, w, sw = operands(m, n, k, seed)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(kind.t) if bias else None
    got = run(ctx, kind, x, sx, w, sw, b, **place)
    near(got, *ref.linear(kind, x.double(), sx.double(), w.double(), sw.double(), None if b is None else b.double()))


FEW = [(1, 1, 1), (1, 16, 16), (1, 17, 15), (2, 5, 64), (1, 100, 65), (3, 33, 127), (1, 64, 128), (16, 48, 129), (1, 300, 1000), (1, 40, 4111), (17, 31, 200), (32, 70, 777),
       (33, 65, 1111), (48, 20, 500), (64, 16, 2048), (5, 2000, 300), (64, 1000, 96)]
MANY = [(65, 1, 1), (65, 64, 64), (128, 128, 63), (100, 130, 65), (129, 127, 128), (200, 300, 1111), (777, 260, 320), (300, 1000, 4000), (1000, 96, 700), (70, 3000, 2500),
        (513, 514, 48), (2000, 2000, 100)]


@pytest.mark.parametrize("shape", FEW + MANY, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(KINDS))
def test_sizes(ctx, name, shape):
    kind = KINDS[name]
    check(ctx, kind, *shape, 1)
    check(ctx, kind, *shape, 2, bias=True, more=16, gap=3, lead=1)


@pytest.mark.parametrize("shape", [(3600, 3700, 192), (3585, 3600, 64), (4000, 3601, 80), (5000, 5100, 130)], ids=lambda s: "x".join(map(str, s)))
def test_large_tiles(ctx, shape):
    """more tiles of the largest kind than there are workgroups' places, of one block of columns to a few, ended anywhere"""
    check(ctx, KINDS["bf16"], *shape, 3, bias=True)
    check(ctx, KINDS["fp32"], *shape, 4, gap=1)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_the_largest_sums(ctx, m):
    """-128 times -128 over as many columns as 32 bits hold"""
    k, n, kind = 131071, 48, KINDS["fp32"]
    x, w = torch.full((m, k), -128, dtype=torch.int8), torch.full((n, k), -128, dtype=torch.int8)
    w[1] = 127
    sx, sw = torch.full((m,), 0.5), torch.full((n,), 0.25)
    got = run(ctx, kind, x, sx, w, sw)
    want = torch.full((n,), 128.0 * 128 * k / 8).double()
    want[1] = -128.0 * 127 * k / 8
    near(got, want.expand(m, n), 2 * ref.EPS * want.abs().expand(m, n))


@pytest.mark.parametrize("m", [3, 130])
def test_rows_far_apart(ctx, m):
    """strides beyond what a lane's 32-bit offset reaches over a tile (8 MiB), of which only a few bytes are there"""
    k, n, kind = 40, 20, KINDS["bf16"]
    x, sx, w, sw = operands(m, n, k, 5)
    ld = (1 << 23) + 16
    far = torch.zeros((m - 1) * ld + 48, dtype=torch.int8, device="cuda")
    far.as_strided((m, k), (ld, 1)).copy_(x)
    dw, out = whole(w), Held((m, n), kind.t)
    ctx.linear_int8(ctx.linear_int8_desc(kind.dtype, m, k, n, ld, dw.ld, 0), far, sx.cuda(), dw.at, sw.cuda(), None, out.at)
    torch.cuda.synchronize()
    near(out.values(), *ref.linear(kind, x.double(), sx.double(), w.double(), sw.double(), None))


@pytest.mark.parametrize("m", [2, 70, 300])
def test_scales_that_are_no_numbers(ctx, m):
    """they stay in their rows and columns"""
    kind, n, k = KINDS["fp16"], 80, 96
    x, sx, w, sw = operands(m, n, k, 6)
    clean = run(ctx, kind, x, sx, w, sw)
    sx[1], sw[7], sw[8] = float("nan"), float("inf"), 0.0
    got = run(ctx, kind, x, sx, w, sw)
    rows, cols = [i for i in range(m) if i != 1], [i for i in range(n) if i not in (7, 8)]
    assert got[1].isnan().all() and not got[:, 7].isfinite().any() and (got[rows, 8] == 0).all()
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("m", [1, 50, 260])
def test_no_columns(ctx, m):
    """sums of nothing are zeros, and the bias stays"""
    kind, n = KINDS["bf16"], 70
    out, ones = Held((m, n), kind.t), torch.ones(max(m, n), device="cuda")
    bias = torch.randn(n, device="cuda").to(kind.t)
    desc = ctx.linear_int8_desc(kind.dtype, m, 0, n)
    ctx.linear_int8(desc, None, ones, None, ones, None, out.at)
    assert ctx.sync() == capi.VALID and (out.values() == 0).all()
    ctx.linear_int8(desc, None, ones, None, ones, bias, out.at)
    assert ctx.sync() == capi.VALID and torch.equal(out.values(), bias.double().cpu().expand(m, n))
    ctx.linear_int8(ctx.linear_int8_desc(kind.dtype, 0, 5, n), None, None, None, None, None, None)
    assert ctx.last_kernel == "empty"
    ctx.linear_int8(ctx.linear_int8_desc(kind.dtype, m, 5, 0), None, None, None, None, None, None)
    assert ctx.last_kernel == "empty" and ctx.sync() == capi.VALID


def test_the_same_bits_again(ctx):
    for m, n, k in ((9, 100, 700), (150, 200, 3000), (3600, 3650, 200)):
        ops = operands(m, n, k, 7)
        first = run(ctx, KINDS["fp32"], *ops)
        for _ in range(3):
            assert torch.equal(run(ctx, KINDS["fp32"], *ops), first)


def test_refusals(ctx):
    kind, m, n, k = KINDS["fp16"], 4, 20, 40
    x, sx, w, sw = operands(m, n, k, 8)
    dx, dw, out = whole(x), whole(w), Held((m, n), kind.t)
    sx, sw, bias = sx.cuda(), sw.cuda(), torch.zeros(n + 1, dtype=kind.t, device="cuda")
    good = [dx.at, sx, dw.at, sw, bias, out.at]

    def refused(args=good, **changed):
        d = ctx.linear_int8_desc(kind.dtype, m, k, n)
        for key, v in changed.items():
            setattr(d, key, v)
        with pytest.raises(TmiError) as e:
            ctx.linear_int8(d, *args)
        assert e.value.status == capi.ERROR
        return e.value.message

    assert "data type" in refused(dtype=capi.INT8)
    for name in ("rows", "in_features", "out_features"):
        assert "negative" in refused(**{name: -1})
    assert "131071" in refused(in_features=131072)
    assert "more than one call" in refused(rows=(1 << 22) + 1) and "more than one call" in refused(rows=1 << 20, out_features=1 << 24)
    for name in ("ld_x", "ld_w"):
        assert "apart" in refused(**{name: 40}) and "apart" in refused(**{name: 32}) and "apart" in refused(**{name: 56})
    assert "apart" in refused(ld_y=19)
    swap = lambda at, v: [v if i == at else g for i, g in enumerate(good)]  # noqa: E731
    for at in (0, 1, 2, 3, 5):
        assert "null" in refused(swap(at, None))
    assert "16 bytes" in refused(swap(0, dx.buf[8:])) and "16 bytes" in refused(swap(2, dw.buf[1:]))
    odd = bias.view(torch.uint8)[1:]
    for at in (1, 3, 4, 5):
        assert "aligned" in refused(swap(at, odd))
    assert ctx.sync() == capi.VALID and (out.values() == ref.CANARY).all()
