"""Refusals of the paged-cache operators, their argument layout and the rotary frequencies: no GPU is used."""
import ctypes as C

import numpy as np
import pytest

import ptts_lib
import ptts_paged
from ptts_paged import DeviceArray

PTR = 1 << 20      # never read: every call below is refused before anything is launched


def arr(shape, dtype="int32", strides=None, ptr=PTR, device=0):
    return DeviceArray(ptr, shape, dtype, strides, device)


def test_frequencies():
    f, m = ptts_paged.frequencies(64)
    np.testing.assert_allclose(f, 10000.0 ** (-2.0 * np.arange(32) / 64), rtol=1e-14)
    assert m == 1.0
    lin, _ = ptts_paged.frequencies(64, scaling="linear", factor=4.0)
    np.testing.assert_allclose(lin, f / 4, rtol=1e-14)
    base, _ = ptts_paged.frequencies(64, scaling="base", factor=4.0)
    np.testing.assert_allclose([base[0] / f[0], base[-1] / f[-1]], [1.0, 0.25], rtol=1e-12)
    parts, m = ptts_paged.frequencies(64, scaling="parts", factor=8.0, trained=4096.0)
    turns = 4096 * f / (2 * np.pi)
    np.testing.assert_allclose(parts[turns >= 32], f[turns >= 32], rtol=1e-14)
    np.testing.assert_allclose(parts[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 32)
    keep = (turns[between] - 1) / 31
    np.testing.assert_allclose(parts[between], f[between] * keep + f[between] / 8 * (1 - keep), rtol=1e-12)
    assert m == pytest.approx(0.1 * np.log(8) + 1, rel=1e-6)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, scaling="linear", factor=0.5),
                dict(rot_dim=8, scaling="parts", factor=2.0), dict(rot_dim=8, scaling="other"), dict(rot_dim=8, base=float("nan"))):
        with pytest.raises(ptts_lib.PttsError):
            ptts_paged.frequencies(**bad)


def _plan(page=16, **over):
    a = dict(cached=arr((3,)), arriving=arr((3,)), free_pages=arr((9,)), block_table=arr((3, 5)), slot_map=arr((7,)), positions=arr((7,)),
             cu_rows=arr((4,)), kv_len=arr((3,)), counts=arr((4,)))
    a.update(over)
    ptts_paged.plan(a.pop("cached"), a.pop("arriving"), a.pop("free_pages"), a.pop("block_table"), page, **a)


@pytest.mark.parametrize("over,text", [
    (dict(arriving=arr((2,))), "arriving"), (dict(cu_rows=arr((3,))), "cu_rows"), (dict(counts=arr((3,))), "counts"),
    (dict(positions=arr((6,))), "positions"), (dict(block_table=arr((2, 5))), "block_table"), (dict(block_table=arr((15,))), "axes"),
    (dict(cached=arr((3,), "float32")), "int32"), (dict(cached=arr((3,), strides=(2,))), "contiguous"), (dict(page=0), "page_size"),
    (dict(page=1 << 30), "page_size"), (dict(block_table=arr((3, 5), strides=(4, 1))), "table_stride"), (dict(status=arr((0,))), "status"),
    (dict(kv_len=arr((3,), device=1)), "one device"), (dict(cached=arr((3,), ptr=0)), "required"), (dict(cached=np.zeros(3, np.int32)), "DeviceArray"),
])
def test_plan_refusals(over, text):
    with pytest.raises(ptts_lib.PttsError, match=text):
        _plan(**over)


def _rotary(**over):
    a = dict(q=arr((5, 4, 64), "bfloat16"), k=arr((5, 2, 64), "bfloat16"), v=arr((5, 2, 64), "bfloat16"), positions=arr((5,)),
             freq=arr((32,), "float64"), q_out=arr((5, 4, 64), "bfloat16", ptr=2 * PTR), slot_map=arr((5,)), k_pages=arr((9, 16, 2, 64), "bfloat16"),
             v_pages=arr((9, 16, 2, 64), "bfloat16"))
    a.update(over)
    ptts_paged.rotary_append(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("positions"), a.pop("freq"), **a)


@pytest.mark.parametrize("over,text", [
    (dict(q=None, q_out=None, k=None, v=None, slot_map=None, k_pages=None, v_pages=None), "nothing"), (dict(v=None), "together"),
    (dict(slot_map=None), "together"), (dict(q_out=arr((5, 4, 64), "float16")), "type"), (dict(v=arr((5, 2, 64), "float32")), "one type"),
    (dict(freq=arr((33,), "float64")), "rot_dim"), (dict(freq=arr((0,), "float64")), "rot_dim"), (dict(freq=arr((32,), "float32")), "float64"),
    (dict(positions=arr((4,))), "positions"), (dict(k_pages=arr((9, 16, 3, 64), "bfloat16")), "shape"),
    (dict(k_pages=arr((9, 16, 2, 64), "float16"), v_pages=arr((9, 16, 2, 64), "float16")), "rows' type"),
    (dict(k_pages=arr((9, 16, 2, 64), "bfloat16", ptr=PTR + 8)), "16 bytes"), (dict(magnitude=float("inf")), "magnitude"),
    (dict(k_pages=arr((1 << 20, 1 << 10, 2, 64), "bfloat16"), v_pages=arr((1 << 20, 1 << 10, 2, 64), "bfloat16")), "2\\^30"),
    (dict(q=arr((5, 4, 64), "bfloat16", ptr=PTR + 1)), "aligned"), (dict(v_pages=arr((9, 16, 2, 64), "bfloat16", strides=(4096, 128, 64, 1))), "strides"),
    (dict(q=arr((5, 4, 64), "bfloat16", ptr=2 * PTR, strides=(512, 64, 1))), "same strides"), (dict(q=arr((5, 4, 64), "bfloat16", strides=(256, 0, 1))), "positive"),
])
def test_rotary_refusals(over, text):
    with pytest.raises(ptts_lib.PttsError, match=text):
        _rotary(**over)


def _attention(call=ptts_paged.attention, **over):
    a = dict(q=arr((5, 4, 64), "bfloat16"), k_pages=arr((9, 16, 2, 64), "bfloat16"), v_pages=arr((9, 16, 2, 64), "bfloat16"), block_table=arr((3, 5)),
             cu_rows=arr((4,)), kv_len=arr((3,)), out=arr((5, 4, 64), "bfloat16", ptr=2 * PTR))
    a.update(over)
    lead = [a.pop(n) for n in ("q", "k_pages", "v_pages", "block_table", "cu_rows", "kv_len")]
    call(*lead, **a)


@pytest.mark.parametrize("over,text", [
    (dict(out=arr((5, 4, 32), "bfloat16")), "out"), (dict(out=arr((5, 4, 64), "float32")), "type"), (dict(out=arr((5, 4, 64), "bfloat16")), "must not be q"),
    (dict(q=arr((5, 3, 64), "bfloat16"), out=arr((5, 3, 64), "bfloat16", ptr=2 * PTR)), "multiple of kv_heads"),
    (dict(q=arr((5, 4, 64), "float16"), out=arr((5, 4, 64), "float16", ptr=2 * PTR)), "rows' type"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(sinks=-1), "sinks"), (dict(max_kv=-1), "max_kv"),
    (dict(cu_rows=arr((3,))), "cu_rows"), (dict(block_table=arr((2, 5))), "block_table"), (dict(lse=arr((5, 3), "float32")), "lse"),
    (dict(q=arr((5, 4, 64), "bfloat16", ptr=PTR + 2)), "16 bytes"), (dict(q=arr((5, 4, 64), "bfloat16", strides=(260, 64, 1))), "16 bytes"),
    (dict(block_table=arr((3, 1 << 27))), "2\\^30"), (dict(block_table=arr((3, 5), strides=(4, 1))), "table_stride"),
    (dict(q=arr((5, 4, 12), "bfloat16"), out=arr((5, 4, 12), "bfloat16", ptr=2 * PTR), k_pages=arr((9, 16, 2, 12), "bfloat16"), v_pages=arr((9, 16, 2, 12), "bfloat16")), "head_dim"),
    (dict(q=arr((5, 4, 264), "bfloat16"), out=arr((5, 4, 264), "bfloat16", ptr=2 * PTR), k_pages=arr((9, 16, 2, 264), "bfloat16"), v_pages=arr((9, 16, 2, 264), "bfloat16")), "head_dim"),
])
def test_attention_refusals(over, text):
    with pytest.raises(ptts_lib.PttsError, match=text):
        _attention(**over)
    if not any(k in over for k in ("lse",)):
        with pytest.raises(ptts_lib.PttsError, match=text):
            _attention(ptts_paged.attention_workspace, **over)


def test_attention_refuses_what_passes_31_bits():
    many = dict(q=arr((1 << 20, 2048, 64), "bfloat16"), out=arr((1 << 20, 2048, 64), "bfloat16", ptr=2 * PTR))
    with pytest.raises(ptts_lib.PttsError, match="below 2\\^30"):
        _attention(**many)


def test_rotary_refuses_more_threads_than_a_launch_holds():
    n = 1 << 24
    with pytest.raises(ptts_lib.PttsError, match="2\\^24"):
        ptts_paged.rotary_append(arr((n, 1, 8), "float32"), None, None, arr((n,)), arr((4,), "float64"))


def test_null_arguments():
    L = ptts_lib.load()
    assert L.ptts_paged_plan(None, 0, None) == -1
    assert L.ptts_rotary_append(None, 0, None) == -1
    assert L.ptts_paged_attention(None, 0, None) == -1
    assert L.ptts_paged_attention_workspace(None, 0) == -1


def test_second_runtime_is_refused():
    ptts_lib.load()
    if ptts_lib.runtime == "system":
        with pytest.raises(ptts_lib.PttsError, match="system's HIP runtime"):
            ptts_lib.load_with_torch()
    assert C.sizeof(C.c_void_p) == 8
