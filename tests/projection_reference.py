"""The root-mean-square norm, rows in 8 bits and the linear layer on them in 64 bits, with how far a result may be off.

Numbers in 32 bits are off by EPS = 2^-24 of themselves for each operation; a rounding to fp16 by 2^-11 (2^-25 where that is subnormal), to bf16 by
2^-8, to fp32 by 2^-24.  A sum over a row is made of at most 16 terms a piece of a lane, 4 pieces, 6 steps over a wave and 16 waves, or for rows beyond
16384 elements of one more for every 4096: DEPTH roundings on the way of each term."""
import torch

from reference_model_amd import capi

EPS = 2.0 ** -24


class Kind:
    def __init__(self, torch_type, dtype, unit, tiny):
        self.t, self.dtype, self.unit, self.tiny = torch_type, dtype, unit, tiny

    def rounding(self, want, off=0.0):
        """of a number that is `want` but for `off`"""
        return self.unit * (want.abs() + off) + self.tiny


KINDS = {"fp16": Kind(torch.float16, capi.FP16, 2.0 ** -11, 2.0 ** -25), "bf16": Kind(torch.bfloat16, capi.BF16, 2.0 ** -8, 2.0 ** -134),
         "fp32": Kind(torch.float32, capi.FP32, 2.0 ** -24, 2.0 ** -150)}
CANARY = 77.0


def depth(width):
    return 42 + width // 4096


class Held:
    """a matrix on the GPU whose rows lie `gap` elements further apart than they are long, the first of them `lead` elements into its buffer; what lies
    around them stays as it is"""

    def __init__(self, shape, t, gap=0, lead=0, values=None):
        rows, width = shape
        self.ld = width + gap
        self.buf = torch.full((lead + rows * self.ld + 8,), CANARY, dtype=t, device="cuda")
        self.at = self.buf[lead:]    # what a call is given
        self.m = self.buf.as_strided((rows, width), (self.ld, 1), lead)
        if values is not None:
            self.m.copy_(values)
        self.was = self.buf.clone()

    def values(self):
        """the matrix now, in 64 bits; nothing beside it was written"""
        got = self.m.clone()
        beside = self.buf.clone()
        beside.as_strided(self.m.shape, self.m.stride(), self.m.storage_offset()).copy_(
            self.was.as_strided(self.m.shape, self.m.stride(), self.m.storage_offset()))
        width = beside.element_size()
        whole = {1: torch.int8, 2: torch.int16, 4: torch.int32}[width]
        assert torch.equal(beside.view(whole), self.was.view(whole)), "written outside the tensor"
        return got.double().cpu()


def held8(rows, width, more=0, fill=0):
    """rows in 8 bits: a matrix of whole 16 bytes (and `more`) a row"""
    return Held((rows, -(-width // 16) * 16), torch.int8, more)


def near(got, want, off):
    bad = ~((got - want).abs() <= off)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} "
                           f"+- {off[bad][0]}")


def norm(kind, x, residual, weight, eps, offset):
    """(sum, off), (y before its rounding, off), (r, off)"""
    s = x if residual is None else x + residual
    w = offset + weight
    r = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    y = s * r * w
    off = (depth(x.shape[1]) / 2 + 10) * EPS    # of r: half of the squares' sum; s, its square, the mean, eps, root and reciprocal; and the products
    off_s = EPS * s.abs() + kind.rounding(s, EPS * s.abs())
    return (s, off_s), (y, off * y.abs()), (r[:, 0], off * r[:, 0])


def check_int8(q, scales, v, off, width, ties=False):
    """q [rows][whole 16s] and scales of rows whose values are v [rows][width] but for a part `off` of each.  With `ties` v are operands, and halves go to even."""
    most = v.abs().amax(1)
    want = most / 127
    assert ((scales - want).abs() <= (off + 4 * EPS) * want + 2.0 ** -149).all()
    assert (q[:, width:] == 0).all()
    t = torch.where(most[:, None] > 0, v * 127 / most[:, None].clamp_min(1e-300), 0.0)
    # s (offset + weight): four roundings, the reciprocal's two and the last one; of a number up to 127
    assert ((q[:, :width] - t).abs() <= 0.5 + 127 * 8 * EPS).all()
    assert (q.abs() <= 127).all() and (q.abs().amax(1)[most > 0] == 127).all()
    if ties:
        # v * 254 / most is odd where v is a half: in whole numbers, of both times a power of two
        ratio = v * 254
        k = torch.round(ratio / most[:, None].clamp_min(1e-300))
        half = (k * most[:, None] == ratio) & (k.abs() % 2 == 1) & (most[:, None] > 0)
        even = 2 * torch.round(k / 4)    # k / 2 to the nearest even number
        assert torch.equal(q[:, :width][half], even[half])
        return int(half.sum())
    return 0


def norm_gradients(kind, s, weight, r, dy, d_sum, offset):
    """(d_x, off), (d_weight, off)"""
    width, rows = s.shape[1], s.shape[0]
    r = r[:, None]
    w = offset + weight
    n, g = s * r, dy * w
    mean = (g * n).mean(1, keepdim=True)
    off_mean = (depth(width) + 8) * EPS * (g * n).abs().mean(1, keepdim=True)
    dx = r * (g - n * mean)
    off = r * (n.abs() * (off_mean + 4 * EPS * mean.abs()) + 4 * EPS * (g.abs() + (n * mean).abs())) + EPS * dx.abs()
    if d_sum is not None:
        dx = dx + d_sum
        off = off + EPS * dx.abs()
    dw = (dy * n).sum(0)
    off_w = (rows + 4) * EPS * (dy * n).abs().sum(0)
    return (dx, off + kind.rounding(dx, off)), (dw, off_w + kind.rounding(dw, off_w))


def linear(kind, x, x_scales, w, w_scales, bias):
    """x, w: whole numbers; the sum is exact, its rounding, two products and a sum follow"""
    p = (x @ w.T) * x_scales[:, None] * w_scales
    y = p if bias is None else p + bias
    off = 4 * EPS * (p.abs() + y.abs()) + 2.0 ** -148
    return y, off + kind.rounding(y, off)
