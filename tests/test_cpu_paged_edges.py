"""Calls of the paged-cache operators at the borders of what their documentation allows: no GPU is used.

Every call names a device that is not there, so one that passes the checks of its arguments is refused for the device and launches
nothing, on a machine with a GPU too."""
import pytest

import ptts_lib
import ptts_paged
from ptts_paged import DeviceArray

PTR = 1 << 20      # never read
GONE = 99


def arr(shape, dtype="int32", strides=None, ptr=PTR):
    return DeviceArray(ptr, shape, dtype, strides, GONE)


def passes_checks(call, *args, **kw):
    with pytest.raises(ptts_lib.PttsError, match="device"):
        call(*args, **kw)


@pytest.mark.parametrize("parts", ["q", "kv", "qkv"])
def test_a_step_without_rows(parts):
    """Nothing arrives: the same calls with no rows."""
    x = arr((0, 4, 64), "bfloat16")
    pages = arr((9, 16, 2, 64), "bfloat16")
    q = x if "q" in parts else None
    more = dict(slot_map=arr((0,)), k_pages=pages, v_pages=pages) if "kv" in parts else {}
    k = arr((0, 2, 64), "bfloat16") if "kv" in parts else None
    passes_checks(ptts_paged.rotary_append, q, k, k, arr((0,)), arr((32,), "float64"), **more)
    passes_checks(ptts_paged.attention, x, pages, pages, arr((3, 5)), arr((4,)), arr((3,)), out=x)


def test_workspace_query_with_an_explicit_none():
    """out=None is the documented default of the query."""
    x, pages = arr((5, 4, 64), "bfloat16"), arr((9, 16, 2, 64), "bfloat16")
    lead = (x, pages, pages, arr((3, 5)), arr((4,)), arr((3,)))
    passes_checks(ptts_paged.attention_workspace, *lead)
    passes_checks(ptts_paged.attention_workspace, *lead, out=None)
    with pytest.raises(ptts_lib.PttsError, match="must not be q"):
        ptts_paged.attention_workspace(*lead, out=x)


@pytest.mark.parametrize("name,dtype", [("cached", "int32"), ("free_pages", "int32"), ("block_table", "int32"), ("counts", "int32"), ("status", "int32")])
def test_plan_refuses_what_is_not_aligned(name, dtype):
    """Arrays off their type's alignment: an atomic on such an address faults."""
    shapes = dict(cached=(3,), arriving=(3,), free_pages=(9,), block_table=(3, 5), slot_map=(7,), positions=(7,), cu_rows=(4,), kv_len=(3,), counts=(4,), status=(1,))
    a = {k: arr(s, ptr=PTR + 2 * (k == name)) for k, s in shapes.items()}
    with pytest.raises(ptts_lib.PttsError, match="aligned"):
        ptts_paged.plan(a.pop("cached"), a.pop("arriving"), a.pop("free_pages"), a.pop("block_table"), 16, **a)


@pytest.mark.parametrize("name", ["positions", "slot_map", "freq", "status"])
def test_rotary_refuses_what_is_not_aligned(name):
    x, kv, pages = arr((5, 4, 64), "bfloat16"), arr((5, 2, 64), "bfloat16"), arr((9, 16, 2, 64), "bfloat16")
    a = {k: arr(s, t, ptr=PTR + (4 if t == "float64" else 2) * (k == name)) for k, s, t in (("positions", (5,), "int32"), ("slot_map", (5,), "int32"),
                                                                                       ("freq", (32,), "float64"), ("status", (1,), "int32"))}
    with pytest.raises(ptts_lib.PttsError, match="aligned"):
        ptts_paged.rotary_append(x, kv, kv, a.pop("positions"), a.pop("freq"), k_pages=pages, v_pages=pages, **a)


@pytest.mark.parametrize("name", ["block_table", "cu_rows", "kv_len", "lse", "status"])
def test_attention_refuses_what_is_not_aligned(name):
    x, out, pages = arr((5, 4, 64), "bfloat16"), arr((5, 4, 64), "bfloat16", ptr=2 * PTR), arr((9, 16, 2, 64), "bfloat16")
    a = {k: arr(s, t, ptr=PTR + 2 * (k == name)) for k, s, t in (("block_table", (3, 5), "int32"), ("cu_rows", (4,), "int32"), ("kv_len", (3,), "int32"),
                                                                 ("lse", (5, 4), "float32"), ("status", (1,), "int32"))}
    with pytest.raises(ptts_lib.PttsError, match="aligned"):
        ptts_paged.attention(x, pages, pages, a.pop("block_table"), a.pop("cu_rows"), a.pop("kv_len"), out=out, **a)


def test_make_without_python_headers():
    """The library and the programs are made where Python's headers are missing; with them the binding is made, too."""
    import os
    import subprocess
    for inc, there in (("/nowhere", False), (None, True)):
        cmd = ["make", "-n", "-C", ptts_lib.PKG, "all", f"OBJDIR={ptts_lib.PKG}/no_such_build"] + ([f"PYINC={inc}"] if inc else [])
        r = subprocess.run(cmd + ["-W", os.path.join(ptts_lib.PKG, "csrc", "py_paged.cpp")], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        assert ("py_paged.cpp" in r.stdout) == there and "c_api.cpp" in r.stdout
        assert ("no Python headers" in r.stdout) != there
