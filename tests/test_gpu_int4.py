"""4-bit weights: the packed form byte by byte, products of a few rows with it and the gated block on it against 64 bits, over sizes that end
inside tiles and groups, rows that begin at any element, all three groups, and numbers that are none."""
import numpy as np
import pytest

import ffn_reference as ref
from reference_model_amd import Context, TmiError, capi
from test_gpu_gated_ffn import KINDS, Rows, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def weights(kind, n, k, seed):
    rng = np.random.default_rng(seed)
    return kind.wide(kind.narrow(rng.normal(0, 1 / np.sqrt(max(k, 1)), (n, k))))


def held(ctx, kind, group, v, scales):
    """the packed form on the GPU, made on the host"""
    return ctx.upload(ref.packed(kind, v, scales, group))


SIZES = [(1, 1), (16, 128), (5, 32), (17, 129), (33, 200), (130, 520), (3, 1000), (64, 127)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", list(KINDS))
def test_quantize_pack_and_back(ctx, kind, group, size):
    kind, (n, k) = KINDS[kind], size
    w = weights(kind, n, k, n + k)
    w[n // 2] = 0    # a row of zeros: scale 0
    v, scales = ref.quantized(kind, w, group)
    want = ref.packed(kind, v, scales, group)
    desc = ctx.int4_desc(kind.dtype, group, n, k)
    assert ctx.int4_packed_bytes(desc) == want.size
    for gap, lead in ((0, 0), (3, 1), (8, 8)):
        dev, to = Rows(ctx, kind, (n, k), w, gap, lead), ctx.upload(np.full(want.size + 16, 0xA5, np.uint8))
        ctx.quantize_int4(desc, dev.at, k + gap, to)
        assert ctx.sync() == capi.VALID
        got = to.numpy().view(np.uint8)
        assert np.array_equal(got[:want.size], want) and (got[want.size:] == 0xA5).all()
        back = Rows(ctx, kind, (n, k), None, gap, lead)
        ctx.dequantize_int4(desc, to, back.at, k + gap)
        assert ctx.sync() == capi.VALID
        assert np.array_equal(back.stored().view(np.uint16), kind.narrow(ref.weights(kind, v, scales, group)).view(np.uint16))
        for t in (dev, to, back):
            t.free()


@pytest.mark.parametrize("group", [32, 128])
def test_pack_given_values(ctx, group):
    kind, (n, k) = KINDS["fp16"], (35, 300)
    rng = np.random.default_rng(group)
    v = rng.integers(-8, 8, (n, k))
    scales = kind.narrow(rng.normal(0, 1, (n, -(-k // group))))
    wide = np.full((n, k + 5), 99, np.int8)
    wide[:, :k] = v
    wide[0, 0], wide[1, 1] = 127, -128    # kept to the range
    v[0, 0], v[1, 1] = 7, -8
    dev, sc = ctx.upload(wide), ctx.upload(scales)
    want = ref.packed(kind, v, scales, group)
    to = ctx.upload(np.zeros(want.size, np.uint8))
    ctx.pack_int4(ctx.int4_desc(kind.dtype, group, n, k), dev, k + 5, sc, to)
    assert ctx.sync() == capi.VALID and np.array_equal(to.numpy().view(np.uint8), want)


@pytest.mark.parametrize("kind", list(KINDS))
def test_weights_that_are_no_numbers_and_tiny_ones(ctx, kind):
    kind, (n, k, group) = KINDS[kind], (4, 96, 32)
    w = weights(kind, n, k, 1)
    w[0, 5], w[1, 40], w[2, 70] = np.nan, np.inf, -np.inf
    w[3, :32] = np.arange(32) * 2.0 ** -24    # a scale that is subnormal, and no division by it
    w[3, 32:64] = 0
    w[3, 40] = 2.0 ** -24
    v, scales = ref.quantized(kind, w, group)
    dev, desc = ctx.upload(kind.narrow(w), kind.dtype), ctx.int4_desc(kind.dtype, group, n, k)
    to = ctx.upload(np.zeros(ctx.int4_packed_bytes(desc), np.uint8))
    ctx.quantize_int4(desc, dev, 0, to)
    back = Rows(ctx, kind, (n, k))
    ctx.dequantize_int4(desc, to, back.at, 0)
    assert ctx.sync() == capi.VALID
    with np.errstate(invalid="ignore"):
        want = kind.wide(kind.narrow(ref.weights(kind, v, scales, group)))
    assert np.array_equal(back.values(), want, equal_nan=True) and np.isnan(want[0, :32]).all() and np.isnan(want[1, 32:64]).all()


PRODUCTS = [(1, 64, 64, 0, 0), (1, 1, 1, 0, 0), (2, 16, 128, 0, 0), (1, 33, 4100, 0, 0), (5, 299, 1111, 9, 1), (16, 48, 1024, 0, 0), (17, 40, 160, 8, 8), (33, 70, 257, 1, 3),
            (64, 16, 96, 0, 0), (150, 20, 130, 3, 0)]


@pytest.mark.parametrize("shape", PRODUCTS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", list(KINDS))
def test_products(ctx, kind, group, shape):
    kind, (m, n, k, gap, lead) = KINDS[kind], shape
    rng = np.random.default_rng(n)
    x = kind.wide(kind.narrow(rng.normal(0, 1, (m, k))))
    v = [rng.integers(-8, 8, (n, k)) for _ in range(2)]
    scales = [kind.narrow(rng.uniform(0.01, 0.1, (n, -(-k // group)))) for _ in range(2)]
    dev, packs = Rows(ctx, kind, (m, k), x, gap, lead), [held(ctx, kind, group, *p) for p in zip(v, scales)]
    out = Rows(ctx, kind, (m, n), None, gap, lead)
    desc = ctx.int4_desc(kind.dtype, group, n, k)
    ctx.matvec_int4(desc, m, dev.at, k + gap, packs[0], out.at, n + gap)
    assert ctx.sync() == capi.VALID
    w = [ref.weights(kind, *p, group) for p in zip(v, scales)]
    near(out.values(), ref.product(kind, x, w[0]))
    for name in ref.ACTS if m == 5 else ("silu",):
        ctx.gated_ffn_int4(desc, ref.ACTS[name], m, dev.at, k + gap, *packs, out.at, n + gap)
        assert ctx.sync() == capi.VALID
        near(out.values(), ref.gated(kind, name, x, *w)[0])
    for t in [dev, out] + packs:
        t.free()


@pytest.mark.parametrize("rows", [1, 20, 40])
@pytest.mark.parametrize("kind", list(KINDS))
def test_wide_matrices(ctx, kind, rows):
    """so many weight rows that a wave takes two tiles of them; the last workgroup has one"""
    kind, (n, k, group) = KINDS[kind], (16 * 2049, 130, 64)
    rng = np.random.default_rng(rows)
    x = kind.wide(kind.narrow(rng.normal(0, 1, (rows, k))))
    v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.uniform(0.01, 0.1, (n, 3)))
    pick = np.r_[0:40, n - 40:n]
    w = ref.weights(kind, v, scales, group)
    pack, dev, out = held(ctx, kind, group, v, scales), Rows(ctx, kind, (rows, k), x), Rows(ctx, kind, (rows, n))
    desc = ctx.int4_desc(kind.dtype, group, n, k)
    ctx.matvec_int4(desc, rows, dev.at, 0, pack, out.at, 0)
    assert ctx.sync() == capi.VALID
    near(out.values(), ref.product(kind, x, w))
    ctx.gated_ffn_int4(desc, capi.ACT_SILU, rows, dev.at, 0, pack, pack, out.at, 0)
    assert ctx.sync() == capi.VALID
    near(out.values()[:, pick], ref.gated(kind, "silu", x, w[pick], w[pick])[0])


@pytest.mark.parametrize("kind", list(KINDS))
def test_infinite_and_nan_rows(ctx, kind):
    """an infinite x times a weight of 0 is no number, times another infinite; a NaN stays in its row"""
    kind, (n, k, group) = KINDS[kind], (40, 200, 64)
    rng = np.random.default_rng(2)
    x = kind.wide(kind.narrow(rng.normal(0, 1, (3, k))))
    x[0, 7], x[1, 150] = np.inf, np.nan
    v, scales = rng.integers(-8, 8, (n, k)), kind.narrow(rng.uniform(0.01, 0.1, (n, 4)))
    v[3, 7], v[4, 7], v[5, 7] = 0, 7, -8
    with np.errstate(invalid="ignore"):
        want = x @ ref.weights(kind, v, scales, group).T
    out, desc = Rows(ctx, kind, (3, n)), ctx.int4_desc(kind.dtype, group, n, k)
    ctx.matvec_int4(desc, 3, ctx.upload(kind.narrow(x), kind.dtype), 0, held(ctx, kind, group, v, scales), out.at, 0)
    assert ctx.sync() == capi.VALID
    got = out.values()
    assert np.isnan(got[0, 3]) and got[0, 4] == np.inf and got[0, 5] == -np.inf and np.isnan(got[1]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want)) and np.isfinite(got[2]).all()


def test_lengths_of_zero(ctx):
    kind = KINDS["fp16"]
    out = Rows(ctx, kind, (3, 8))
    desc = ctx.int4_desc(kind.dtype, 32, 8, 0)
    ctx.matvec_int4(desc, 3, None, 0, None, out.at, 0)
    assert ctx.sync() == capi.VALID and not out.values().any()
    assert ctx.int4_packed_bytes(desc) == 0
    ctx.matvec_int4(ctx.int4_desc(kind.dtype, 32, 0, 64), 3, None, 0, None, None, 0)
    assert ctx.last_kernel == "empty"
    ctx.matvec_int4(ctx.int4_desc(kind.dtype, 32, 8, 64), 0, None, 0, None, None, 0)
    ctx.quantize_int4(ctx.int4_desc(kind.dtype, 32, 0, 64), None, 0, None)
    assert ctx.last_kernel == "empty" and ctx.sync() == capi.VALID


def test_what_is_refused(ctx):
    buf = ctx.upload(np.zeros(1 << 16, np.uint8))
    p, ok = buf.ptr, (capi.BF16, 64, 16, 128)
    calls = [lambda d, a=p, b=p, ld=0: ctx.matvec_int4(d, 1, a, ld, b, p, 0), lambda d, a=p, b=p, ld=0: ctx.gated_ffn_int4(d, capi.ACT_SILU, 1, a, ld, b, p, p, 0),
             lambda d, a=p, b=p, ld=0: ctx.quantize_int4(d, a, ld, b), lambda d, a=p, b=p, ld=0: ctx.dequantize_int4(d, b, a, ld),
             lambda d, a=p, b=p, ld=0: ctx.pack_int4(d, a, ld, p, b)]

    def refused(say, call, *args, **kw):
        with pytest.raises(TmiError) as e:
            call(*args, **kw)
        assert e.value.status == capi.ERROR and say in e.value.message

    for call in calls:
        refused("data type", call, ctx.int4_desc(capi.INT8, *ok[1:]))
        for group in (0, 16, 48, 256, -32):
            refused("groups", call, ctx.int4_desc(capi.BF16, group, 16, 128))
        refused("negative", call, ctx.int4_desc(capi.BF16, 64, -1, 128))
        refused("negative", call, ctx.int4_desc(capi.BF16, 64, 16, -1))
        refused("more than", call, ctx.int4_desc(capi.BF16, 64, 1 << 30, 1 << 20))
        refused("apart", call, ctx.int4_desc(*ok), ld=127)
        refused("apart", call, ctx.int4_desc(*ok), ld=-128)
        refused("null tensor", call, ctx.int4_desc(*ok), a=None)
        refused("null tensor", call, ctx.int4_desc(*ok), b=None)
        refused("16 bytes", call, ctx.int4_desc(*ok), b=p + 8)
    for call in calls[:4]:
        refused("aligned to its elements", call, ctx.int4_desc(*ok), a=p + 1)
    refused("data type", ctx.int4_packed_bytes, ctx.int4_desc(capi.FP32, *ok[1:]))
    refused("activation", ctx.gated_ffn_int4, ctx.int4_desc(*ok), 9, 1, p, 0, p, p, p, 0)
    refused("negative", ctx.matvec_int4, ctx.int4_desc(*ok), -1, p, 0, p, p, 0)
    refused("null tensor", ctx.pack_int4, ctx.int4_desc(*ok), p, 0, None, p)
    assert ctx.sync() == capi.VALID


@pytest.mark.parametrize("shape", [(1, 16 * 1030, 4100, 128), (3, 16 * 1030, 4100, 32), (16, 16 * 600 + 5, 2050, 64), (13, 4099, 4111, 64), (9, 200, 33000, 128), (33, 5500, 2048, 32),
                                   (64, 4099, 4100, 128), (50, 2000, 1111, 64), (64, 40, 9000, 32)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(KINDS))
def test_large_matrices(ctx, kind, shape):
    """blocks of weight rows one after the other, columns of x a part at a time, row tiles of x in one or several workgroups; some of the results"""
    kind, (m, n, k, group) = KINDS[kind], shape
    rng = np.random.default_rng(n)
    x = kind.wide(kind.narrow(rng.normal(0, 1, (m, k))))
    desc = ctx.int4_desc(kind.dtype, group, n, k)
    pick = np.unique(np.r_[0:20, rng.integers(0, n, 40), n - 20:n])
    packs, w = [], []
    for _ in range(2):
        v, scales = rng.integers(-8, 8, (n, k), np.int8), kind.narrow(rng.uniform(0.01, 0.1, (n, -(-k // group))))
        dv, ds = ctx.upload(v), ctx.upload(scales, kind.dtype)
        to = ctx.upload(np.zeros(ctx.int4_packed_bytes(desc), np.uint8))
        ctx.pack_int4(desc, dv, 0, ds, to)
        assert ctx.sync() == capi.VALID
        dv.free(), ds.free()
        packs.append(to)
        w.append(ref.weights(kind, v[pick].astype(np.int64), scales[pick], group))
    dev, out = Rows(ctx, kind, (m, k), x, 3, 1), Rows(ctx, kind, (m, n), None, 8, 0)
    ctx.matvec_int4(desc, m, dev.at, k + 3, packs[0], out.at, n + 8)
    assert ctx.sync() == capi.VALID
    got = out.values()
    near(got[:, pick], ref.product(kind, x, w[0]))
    ctx.matvec_int4(desc, m, dev.at, k + 3, packs[0], out.at, n + 8)
    assert ctx.sync() == capi.VALID and np.array_equal(out.values(), got)
    ctx.gated_ffn_int4(desc, capi.ACT_GELU_TANH, m, dev.at, k + 3, *packs, out.at, n + 8)
    assert ctx.sync() == capi.VALID
    near(out.values()[:, pick], ref.gated(kind, "gelu_tanh", x, *w)[0])
    for t in [dev, out] + packs:
        t.free()
