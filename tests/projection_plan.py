"""What the library says a call of the linear layer in 8 bits would launch (host arithmetic, no GPU): the tests choose their sizes by it."""
import collections
import ctypes

from reference_model_amd import capi

Plan = collections.namedtuple("Plan", "tile features splits")


def plan(rows, out_features, in_features, dtype=capi.BF16, ld_x=0, ld_w=0):
    lib, out = capi.load_library(), (ctypes.c_int64 * 3)()
    desc = capi.Context.linear_int8_desc(dtype, rows, in_features, out_features, ld_x, ld_w)
    if lib.tmi_debug_linear_int8_plan(ctypes.byref(desc), out) != capi.VALID:
        return None
    return Plan(*out)
