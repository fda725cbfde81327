"""The feed-forward operators' calls, ctypes and native: the same names, arguments, results and errors, and the structures' sizes (no GPU needed: a
context that does not exist refuses every call with the library's own message)."""
import ctypes
import inspect
import subprocess
import sys

import pytest

from reference_model_amd import TmiError, build, capi

pytest.importorskip("torch")    # first: the library then shares its HIP runtime; loaded behind the library it would bring a second one, which finds no GPU
capi.load_library()
NATIVE = {name: vars(capi.Context)[name] for name in capi.PLAIN_FEED_FORWARD}
FFN, INT4 = capi.GatedFfnDesc(), capi.Int4Desc()
CALLS = {"gated_ffn": (FFN, 0, 0, 0, 0), "gated_ffn_backward": (FFN,) + (0,) * 9, "quantize_int4": (INT4, 0, 0, 0), "dequantize_int4": (INT4, 0, 0, 0),
         "matvec_int4": (INT4, 1, 0, 0, 0, 0, 0), "gated_ffn_int4": (INT4, 1, 1, 0, 0, 0, 0, 0, 0)}


@pytest.fixture
def nothing():
    """a Context whose library is loaded and whose handle is none"""
    c = object.__new__(capi.Context)
    c.lib, c.handle = capi.load_library(), None
    return c


def test_native_calls_are_the_ones_in_use():
    assert set(NATIVE) == set(CALLS) and all(NATIVE[n] is not capi.PLAIN_FEED_FORWARD[n] for n in NATIVE)
    for name, plain in capi.PLAIN_FEED_FORWARD.items():
        assert list(inspect.signature(NATIVE[name]).parameters) == list(inspect.signature(plain).parameters)
        for a, b in zip(inspect.signature(NATIVE[name]).parameters.values(), inspect.signature(plain).parameters.values()):
            assert a.default is b.default


@pytest.mark.parametrize("form", ["native", "plain"])
@pytest.mark.parametrize("name", list(CALLS))
def test_arguments_and_errors_of_both_forms(nothing, form, name):
    fn, args = (NATIVE if form == "native" else capi.PLAIN_FEED_FORWARD)[name], CALLS[name]
    call = lambda *a, **k: fn.__get__(nothing, capi.Context)(*a, **k)  # noqa: E731
    with pytest.raises(TmiError) as e:
        call(*args)
    assert e.value.status == capi.ERROR and "null context" in e.value.message
    names = list(inspect.signature(capi.PLAIN_FEED_FORWARD[name]).parameters)[1:]
    with pytest.raises(TmiError):
        call(**dict(zip(names, args)))
    if name == "gated_ffn":
        with pytest.raises(TmiError):
            call(*args, None, None)
        with pytest.raises(TmiError):
            call(*args, pre_up=0)
    with pytest.raises(TypeError):
        call(*args[:-1])
    with pytest.raises(TypeError):
        call(*args, no_such_argument=1)
    with pytest.raises((TypeError, ctypes.ArgumentError)):
        call(capi.PoolDesc(), *args[1:])
    with pytest.raises((TypeError, ctypes.ArgumentError)):
        call(args[0], "no tensor", *args[2:])


def test_the_binding_works_without_the_extension():
    code = ("import sys; sys.modules['reference_model_amd._calls'] = None\n"
            "from reference_model_amd import capi\n"
            "capi.load_library()\n"
            "assert all(vars(capi.Context)[n] is f for n, f in capi.PLAIN_FEED_FORWARD.items())\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=build.HERE + "/..")
    assert r.returncode == 0, r.stderr


def test_structs_match_header_sizes():
    assert ctypes.sizeof(capi.GatedFfnDesc) == 3 * 8 + 5 * 4 + 4    # and what rounds it up to eight bytes
    assert ctypes.sizeof(capi.Int4Desc) == 4 * 4


def test_a_context_that_is_none():
    lib, size = capi.load_library(), ctypes.c_size_t(0)
    assert lib.tmi_int4_packed_bytes(None, ctypes.byref(INT4), ctypes.byref(size)) == capi.ERROR
    assert lib.tmi_pack_int4(None, ctypes.byref(INT4), None, 0, None, None) == capi.ERROR
