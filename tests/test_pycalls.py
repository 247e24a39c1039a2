"""Calls of a serving step from Python: the module of csrc/pycalls.c beside ctypes.  No GPU needed: the
calls are refused, by the library itself."""
import ctypes as C

import numpy as np
import pytest

COUNTS = {"llmx_adapters_project": 9, "llmx_verify_drafts": 19, "llmx_token_logprobs": 15, "llmx_paged_append": 17, "llmx_paged_attention": 16}


@pytest.fixture(scope="module")
def calls(llmx):
    llmx.lib()
    return llmx._calls


@pytest.mark.parametrize("name", list(COUNTS))
def test_same_answers_as_ctypes(llmx, calls, name):
    """None, numbers, numpy's numbers, numbers wider than their parameter, ctypes' own pointers."""
    slow, n = getattr(llmx.lib(), name), COUNTS[name]
    for args in ([None if t in (C.c_void_p,) else 0 for t in slow.argtypes], [0] * n):
        assert slow(*args) == calls[name](*args)
        detail = llmx.last_error()
        slow(*args)
        assert llmx.last_error() == detail
    null = [C.c_void_p(0) if t is C.c_void_p else 0 for t in slow.argtypes]
    assert calls[name](*null) == slow(*null)
    assert calls[name](*[np.int64(0)] * n) == slow(*[0] * n)
    assert calls[name](*[0 if t is C.c_void_p else 1 << 40 for t in slow.argtypes]) == slow(*[0 if t is C.c_void_p else 1 << 40 for t in slow.argtypes])


@pytest.mark.parametrize("name", list(COUNTS))
def test_wrong_arguments(llmx, calls, name):
    n = COUNTS[name]
    with pytest.raises((TypeError, C.ArgumentError)):
        calls[name](*[0] * (n - 1))
    with pytest.raises((TypeError, C.ArgumentError)):
        calls[name](*["a"] * n)
    with pytest.raises((TypeError, C.ArgumentError)):
        calls[name](*[1.5] * n)


def test_arguments_arrive_in_their_places(llmx, calls):
    """What the library says of each argument in turn."""
    def said(name, args):
        assert calls[name](*args) == llmx.ERR_ARG
        return llmx.last_error()

    good = [256, 0, 100, 2, 256, 256, 3, 256, 256, 256, 256, 256, 256, llmx.logprobs_workspace_bytes(2, 100, 3), None]
    for at, value, text in ((1, 99, "stride"), (2, 0, "vocab must"), (3, 1 << 21, "rows must"), (6, 33, "top must"), (0, None, "null"),
                            (7, None, "null pointer with tokens"), (10, None, "null pointer with top"), (12, 128, "256-byte"),
                            (13, 1, "too small")):
        bad = list(good)
        bad[at] = value
        assert text in said("llmx_token_logprobs", bad), at
    good = [256, 0, 256, 0, 1000, 256, 256, 2, 4, 3, 256, 256, 256, 256, 256, 256, 256, 1 << 20, None]
    for at, value, text in ((1, 999, "stride"), (3, 999, "stride"), (4, 0, "vocab must"), (7, 0, "requests must"), (8, 7, "exceeds"),
                            (9, 1024, "max_drafts must"), (16, 128, "256-byte"), (17, 1, "too small"), (12, None, "null"), (15, 252, "aligned")):
        bad = list(good)
        bad[at] = value
        assert text in said("llmx_verify_drafts", bad), at
    for name in ("llmx_paged_append", "llmx_paged_attention", "llmx_adapters_project"):
        assert "null handle" in said(name, [None] + [1] * (COUNTS[name] - 1))


@pytest.mark.parametrize("name", list(COUNTS))
def test_none_is_no_number(llmx, calls, name):
    """None is a NULL pointer, and an error in the place of a number (where it would be 0: no rows, say, and a call that
    does nothing)."""
    slow = getattr(llmx.lib(), name)
    good = [None if t is C.c_void_p else 0 for t in slow.argtypes]
    for i, t in enumerate(slow.argtypes):
        args = list(good)
        args[i] = None
        if t is C.c_void_p:
            assert calls[name](*args) == slow(*args)
        else:
            with pytest.raises((TypeError, C.ArgumentError)):
                calls[name](*args)


class Index:
    """Something that can stand for a whole number without being one, as a tensor of one element can."""

    def __index__(self):
        return 0


@pytest.mark.parametrize("name", list(COUNTS))
def test_arrays_are_no_addresses(llmx, calls, name):
    """An array of one element in the place of its address: its value is not taken for that.  In a number's place it is
    one, as for ctypes."""
    slow = getattr(llmx.lib(), name)
    good = [None if t is C.c_void_p else 0 for t in slow.argtypes]
    wrong = [Index(), np.array(0), np.zeros(1, np.int32)]
    try:
        import torch
        wrong += [torch.zeros(1, dtype=torch.int32), torch.tensor(0)]
    except ImportError:
        pass
    for i, t in enumerate(slow.argtypes):
        for x in wrong:
            args = [*good[:i], x, *good[i + 1:]]
            if t is C.c_void_p or getattr(x, "ndim", 0) == 1 and isinstance(x, np.ndarray):
                with pytest.raises((TypeError, C.ArgumentError)):
                    calls[name](*args)
            else:
                assert calls[name](*args) == slow(*args)
        calls[name](*good[:i], np.int32(0), *good[i + 1:])  # (a whole number)


def compiled(folder, source, names):
    """The module made of `source`, under each of the names in `folder`."""
    import os
    import shutil
    import subprocess
    import sysconfig
    inc = sysconfig.get_paths()["include"]
    gcc = os.environ.get("CC", "gcc")
    if not os.path.exists(os.path.join(inc, "Python.h")) or shutil.which(gcc) is None:
        pytest.skip("no headers of Python, or no compiler")
    (folder / "calls.c").write_text(source)
    include = os.path.join(os.path.dirname(__file__), "..", "include")
    for name in names:
        subprocess.run([gcc, "-O1", "-shared", "-fPIC", "-I", inc, "-I", include, str(folder / "calls.c"), "-o", str(folder / name)], check=True)


def source_of_calls():
    import os
    with open(os.path.join(os.path.dirname(__file__), "..", "llm-accel_b200", "csrc", "pycalls.c")) as f:
        return f.read()


@pytest.fixture
def elsewhere(llmx, tmp_path, monkeypatch):
    """The binding as it looks for its module in an empty folder; afterwards as it was."""
    L = llmx.lib()
    monkeypatch.setattr(llmx, "HERE", str(tmp_path))
    yield lambda: llmx._bind_calls(L)
    monkeypatch.undo()
    llmx._bind_calls(L)


def test_module_of_an_older_source(llmx, elsewhere, tmp_path):
    """A module that lacks a function: that one goes through ctypes, the others through the module."""
    import re
    import sysconfig
    source = source_of_calls()
    source = re.sub(r"\n    BIND\(llmx_paged_attention\)", "", source)
    source = re.sub(r"ENTRY\(llmx_paged_attention\),", "", source)
    compiled(tmp_path, source, ["_llmxcalls.so", "_llmxcalls" + sysconfig.get_config_var("EXT_SUFFIX")])
    elsewhere()
    for name in COUNTS:
        through_ctypes = llmx._calls[name] is getattr(llmx.lib(), name)
        assert through_ctypes == (name == "llmx_paged_attention")
        assert llmx._calls[name](*[None if t is C.c_void_p else 0 for t in getattr(llmx.lib(), name).argtypes]) == llmx.ERR_ARG


def test_module_of_another_interpreter(llmx, elsewhere, tmp_path):
    """Only a module whose file name says that it is for this interpreter is loaded: one for another may load as well, and
    run with that one's reference counting."""
    import sysconfig
    compiled(tmp_path, source_of_calls(), ["_llmxcalls.so", "_llmxcalls.cpython-3999-x86_64-linux-gnu.so"])
    elsewhere()
    assert all(llmx._calls[name] is getattr(llmx.lib(), name) for name in COUNTS)
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    assert suffix not in (None, ".so")
    (tmp_path / "_llmxcalls.so").rename(tmp_path / ("_llmxcalls" + suffix))
    elsewhere()
    assert all(llmx._calls[name] is not getattr(llmx.lib(), name) for name in COUNTS)


@pytest.fixture
def module(llmx, calls):
    """The module itself; afterwards bound to the library again.  Without it the tests above compare ctypes with itself."""
    import os
    import sysconfig
    import types
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        pytest.skip("no headers of Python: the module is not built")
    assert all(isinstance(calls[name], types.BuiltinFunctionType) for name in COUNTS)
    yield calls["llmx_paged_append"].__self__
    llmx._bind_calls(llmx.lib())


@pytest.mark.parametrize("name", list(COUNTS))
def test_every_argument_in_its_place(llmx, module, name):
    """A function that writes down what it gets, in the library's place: other values in every place, as wide as
    the parameters are, and wider ones."""
    slow, got = getattr(llmx.lib(), name), []
    fake = C.CFUNCTYPE(C.c_int, *slow.argtypes)(lambda *a: got.append(a) or 42)
    module.bind(name, C.cast(fake, C.c_void_p).value, slow)
    width = [8 * C.sizeof(t) for t in slow.argtypes]
    assert len(width) == COUNTS[name]
    for values in ([3 + i for i in range(len(width))], [(0x7123456789abcdef - (i << 33) - (i << 3)) % 2**(w - 1) for i, w in enumerate(width)],
                   [(0xfedcba9876543210 + (i << 32) + i) for i in range(len(width))]):
        assert getattr(module, name)(*values) == 42
        kept = [v % 2**w for v, w in zip(values, width)]
        kept = [v - 2**w if t is C.c_int and v >= 2**(w - 1) else v for v, w, t in zip(kept, width, slow.argtypes)]
        assert list(got.pop()) == kept and not got
    nothing = [None if t is C.c_void_p else 0 for t in slow.argtypes]
    assert getattr(module, name)(*nothing) == 42 and list(got.pop()) == nothing
