"""What the library says a call of the gated block would launch (host arithmetic, no GPU): the tests choose their sizes by it."""
import collections
import ctypes

from reference_model_amd import capi

Plan = collections.namedtuple("Plan", "rows cols waves splits direct copies together span")
FORWARD, D_X, D_W = 0, 1, 2


def plan(product, rows, d, f, ld=(0, 0, 0), dtype=capi.BF16, at=4096):
    """`at`: the address of x, gate and up, of which nothing is read"""
    lib, out = capi.load_library(), (ctypes.c_int64 * 8)()
    desc = capi.Context.gated_ffn_desc(dtype, capi.ACT_SILU, rows, d, f, *ld)
    if lib.tmi_debug_gated_ffn_plan(ctypes.byref(desc), at, at, at, product, out) != capi.VALID:
        return None
    return Plan(*out)
