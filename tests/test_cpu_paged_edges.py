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
