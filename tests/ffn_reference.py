"""The gated feed-forward block and 4-bit weights in 64 bits, with how far a result in 16 bits may be off.

A product summed in 32 bits in any order is off by at most (terms + 2) 2^-24 times the sum of the absolute products; a rounding to fp16 by 2^-11 of the
value (2^-25 where that is subnormal), to bf16 by 2^-8; the functions of 32 bits by a few 2^-24, taken as 16."""
import math

import numpy as np

import cases
from reference_model_amd import capi

EPS = 2.0 ** -24
ACTS = {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH, "relu": capi.ACT_RELU, "sigmoid": capi.ACT_SIGMOID}
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


class Kind:
    """one of the two 16-bit types"""

    def __init__(self, name):
        self.name, self.bf16 = name, name == "bf16"
        self.dtype = capi.BF16 if self.bf16 else capi.FP16
        self.np = np.uint16 if self.bf16 else np.float16
        self.unit = 2.0 ** -8 if self.bf16 else 2.0 ** -11
        self.tiny = 2.0 ** -133 if self.bf16 else 2.0 ** -25

    def narrow(self, v):
        """stored values of an array"""
        v = np.asarray(v, np.float32)
        return cases.float_to_bf16_bits(v) if self.bf16 else v.astype(np.float16)

    def wide(self, stored):
        return (cases.bf16_bits_to_float(stored) if self.bf16 else stored).astype(np.float64)

    def rounding(self, want, off=0.0):
        """of a number that is `want` but for `off`"""
        return self.unit * (np.abs(want) + off) + self.tiny


def act(name, g):
    """act(g) and its derivative"""
    with np.errstate(over="ignore"):
        if name == "relu":
            return np.maximum(g, 0), (g > 0).astype(np.float64)
        if name == "gelu":
            cdf = 0.5 * _erfc(-g / math.sqrt(2))
            return g * cdf, cdf + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        z, slope = g, 1.0
        if name == "gelu_tanh":
            c = 2 * math.sqrt(2 / math.pi)
            z, slope = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
        p, q = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
        return (p, p * q) if name == "sigmoid" else (g * p, p + g * p * q * slope)


def value_off(name, g, value):
    """how far act(g) may be off in 32 bits for an exact g: a GELU whose cdf lies far out multiplies the rounding of its argument by twice the square of it
    (erfc) or four times it (exp)"""
    with np.errstate(over="ignore"):
        far = 0.0
        if name == "gelu":
            far = 2 * g * g * 0.5 * _erfc(g / math.sqrt(2))
        if name == "gelu_tanh":
            z = np.clip(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3), -700, 700)
            far = 4 * np.abs(z) / (1 + np.exp(z))
    return (16 + far) * EPS * np.abs(value)


def gated(kind, name, x, gate, up):
    """h, g, u and how far each may be off"""
    g, u = x @ gate.T, x @ up.T
    value, _ = act(name, g)
    terms = (x.shape[1] + 2) * EPS
    off_g, off_u = terms * (np.abs(x) @ np.abs(gate).T), terms * (np.abs(x) @ np.abs(up).T)
    h = value * u
    # no activation is steeper than 1.13
    off_h = (1.13 * off_g + value_off(name, g, value)) * (np.abs(u) + off_u) + np.abs(value) * off_u + EPS * np.abs(h)
    return tuple((v, off + kind.rounding(v, off)) for v, off in ((h, off_h), (g, off_g), (u, off_u)))


def gated_gradients(kind, name, x, gate, up, g, u, dh):
    """dx, d_gate and d_up, and how far each may be off: dg and du are rounded before the products"""
    value, slope = act(name, g)
    du, dg = dh * value, dh * u * slope
    # the slopes are sums of terms up to 1 + |g|, each off by a few units in 32 bits
    off_du, off_dg = value_off(name, g, value) * np.abs(dh) + EPS * np.abs(du), 16 * EPS * np.abs(dh * u) * (1 + np.abs(g))
    off_du, off_dg = off_du + kind.rounding(du, off_du), off_dg + kind.rounding(dg, off_dg)
    terms = lambda n: (n + 2) * EPS  # noqa: E731
    f, m = g.shape[1], x.shape[0]
    dx = dg @ gate + du @ up
    off = off_dg @ np.abs(gate) + off_du @ np.abs(up) + terms(2 * f) * ((np.abs(dg) + off_dg) @ np.abs(gate) + (np.abs(du) + off_du) @ np.abs(up))
    out = [(dx, off + kind.rounding(dx, off))]
    for d, od in ((dg, off_dg), (du, off_du)):
        w = d.T @ x
        off = od.T @ np.abs(x) + terms(m) * ((np.abs(d) + od).T @ np.abs(x))
        out.append((w, off + kind.rounding(w, off)))
    return out


# ---- 4-bit weights ------------------------------------------------------------------------------------------------------------------

def quantized(kind, w, group):
    """values [n][k] and stored scales [n][groups] of weights (64 bits, of numbers that the type holds)"""
    n, k = w.shape
    groups = -(-k // group)
    v, scales = np.zeros((n, k), np.int64), np.zeros((n, groups), kind.np)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        for j in range(groups):
            part = w[:, j * group:(j + 1) * group]
            scales[:, j] = kind.narrow((np.abs(part).max(1) / 7).astype(np.float32))
            v[:, j * group:(j + 1) * group] = np.nan_to_num(np.rint(part / kind.wide(scales[:, j])[:, None]), nan=0.0, posinf=0.0,
                                                            neginf=0.0).clip(-7, 7)
    return v, scales


def packed(kind, v, scales, group):
    """the packed form, byte by byte as the header describes it"""
    n, k = v.shape
    tn, tk, per = -(-n // 16), -(-k // 128), 128 // group
    words = np.zeros((tn, tk, 64, 4), np.uint32)
    full = np.zeros((tn * 16, tk * 128), np.int64)
    full[:n, :k] = v
    for col in range(tk * 128):
        e = col % 8
        word = words[:, col // 128, 16 * (col % 32 // 8):16 * (col % 32 // 8) + 16, col % 128 // 32]
        word |= ((full[:, col].reshape(tn, 16) + 8) << (4 * (e // 2) + 16 * (e % 2))).astype(np.uint32)
    s = np.zeros((tn * 16, tk * per), kind.np)
    s[:n, :scales.shape[1]] = scales
    s = s.reshape(tn, 16, tk, per).transpose(0, 2, 1, 3)
    return np.concatenate([words.reshape(-1).view(np.uint8), np.ascontiguousarray(s).reshape(-1).view(np.uint8)])


def weights(kind, v, scales, group):
    """the weights that values and scales stand for, 64 bits"""
    return v * np.repeat(kind.wide(scales), group, 1)[:, :v.shape[1]]


def product(kind, x, w):
    """x w^T and how far it may be off: sums of exact products, one more multiplication by the scale"""
    y = x @ w.T
    off = (x.shape[1] + 4) * EPS * (np.abs(x) @ np.abs(w).T)
    return y, off + kind.rounding(y, off)
