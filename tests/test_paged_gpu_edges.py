"""The paged-cache operators at the borders of what their documentation allows, through the public bindings."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def test_plan_counts_rows_of_a_held_page_that_is_missing():
    """A page that an earlier plan could not give: rows that still fall into it have no page, and are counted."""
    from test_paged_gpu import _run_plan
    table = np.array([[4, -1, -1, -1], [2, 3, -1, -1], [-1, -1, -1, -1]])
    for cached, arriving in (([5, 6, 0], [2, 1, 3]), ([5, 6, 0], [9, 0, 0]), ([4, 8, 4], [1, 1, 0]), ([7, 3, 3], [1, 1, 1])):
        free = np.arange(10, 20)
        rows = sum(arriving)
        want = ref.plan(cached, arriving, free, table, 4, rows)
        got, status = _run_plan(cached, arriving, 4, table, free, rows)
        for name, g, w in zip(("table", "slots", "positions", "cu", "kv_len", "counts"), got, want):
            np.testing.assert_array_equal(g, w, err_msg=f"{name} {cached} {arriving}")
        assert status == 0
    many = 300                                             # the form for many requests
    table = np.where(np.arange(many)[:, None] % 3 == 0, -1, np.arange(2 * many).reshape(many, 2))
    cached, arriving = np.full(many, 2), np.arange(many) % 5
    want = ref.plan(cached, arriving, np.arange(1000, 1500), table, 4, int(arriving.sum()))
    got, _ = _run_plan(cached, arriving, 4, table, np.arange(1000, 1500), int(arriving.sum()))
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)


def test_plan_reports_free_pages_that_are_none():
    """An id below 0 in the free list: the rows that fall into it get no slot and the status says so; one that no row needs does not matter."""
    from test_paged_gpu import _run_plan
    got, status = _run_plan([0, 0], [5, 3], 4, np.full((2, 3), -1), np.array([7, -3, 9, -1]), 8)
    assert status == 1 and got[1].tolist() == [28, 29, 30, 31, -1, 36, 37, 38]
    got, status = _run_plan([0, 0], [4, 3], 4, np.full((2, 3), -1), np.array([7, 9, -1]), 7)
    assert status == 0 and got[1].tolist() == [28, 29, 30, 31, 36, 37, 38]


def test_a_step_without_rows():
    """Nothing arrives: all three calls run and leave everything as it was."""
    import ptts_paged
    from ptts_paged import DeviceArray
    d = {k: ref.Dev(np.asarray(v), "int32") for k, v in dict(cached=[5, 0], arriving=[0, 0], free=[3], table=[[1, -1], [-1, -1]], cu=[9, 9, 9], kv_len=[9, 9],
                                                             counts=np.full(4, 9), status=[0]).items()}
    none = lambda dtype, *shape: DeviceArray(0, shape, dtype)
    ptts_paged.plan(d["cached"].a, d["arriving"].a, d["free"].a, d["table"].a, 4, slot_map=none("int32", 0), positions=none("int32", 0), cu_rows=d["cu"].a,
                    kv_len=d["kv_len"].a, counts=d["counts"].a, status=d["status"].a)
    assert d["cu"].host().tolist() == [0, 0, 0] and d["kv_len"].host().tolist() == [5, 0] and d["counts"].host().tolist() == [0, 0, 0, 0]
    assert d["table"].host().tolist() == [[1, -1], [-1, -1]]
    k0 = np.random.default_rng(0).standard_normal((4, 4, 2, 64)).astype(np.float32)
    pages, freq = ref.floats(k0, "float32"), ref.Dev(np.ones(32), "float64")
    q, k = none("float32", 0, 4, 64), none("float32", 0, 2, 64)
    ptts_paged.rotary_append(q, k, k, none("int32", 0), freq.a, slot_map=none("int32", 0), k_pages=pages.a, v_pages=pages.a, status=d["status"].a)
    ptts_paged.attention(q, pages.a, pages.a, d["table"].a, d["cu"].a, d["kv_len"].a, out=q, lse=none("float32", 0, 4), status=d["status"].a)
    np.testing.assert_array_equal(pages.host(), k0)
    assert d["status"].host()[0] == 0


def test_an_error_from_before_the_call_is_not_the_calls():
    """The thread's last error belongs to whoever made it: a call that launches reports its own launches alone and leaves it."""
    import ctypes as C

    from test_paged_gpu_use import Loop, _clear_slots, _hip
    h = _hip()
    h.hipSetDevice.argtypes, h.hipGetLastError.argtypes = [C.c_int], []
    loop, rng = Loop(), np.random.default_rng(0)
    for arriving in ((3, 1, 20), (1, 1, 1)):
        loop.feed(arriving, rng)
        _clear_slots(loop)
        bad = h.hipSetDevice(99)
        assert bad != 0
        loop.launch()
        assert h.hipGetLastError() == bad
        loop.check()


@pytest.mark.parametrize("kind", ["float16", "float32"])
def test_attention_beyond_one_launch(kind):
    """More workgroups than one launch holds (2^24): 65536 requests of one row and one key, 256 heads of 8."""
    import ptts_paged
    n, heads, dim, pages = 65536, 256, 8, 64
    rng = np.random.default_rng(1)
    v = ref.rounded(rng.standard_normal((pages, 1, heads, dim)), kind)
    page_of = rng.integers(0, pages, n)
    page_of[:2] = 0, 1
    row = rng.standard_normal((heads, dim))
    d = [ref.floats(np.broadcast_to(row, (n, heads, dim)), kind), ref.floats(rng.standard_normal((pages, 1, heads, dim)), kind), ref.floats(v, kind),
         ref.floats(np.zeros((n, heads, dim)), kind)]
    ints = [ref.Dev(x, "int32") for x in (page_of[:, None], np.arange(n + 1), np.ones(n), np.zeros(1))]
    a = [x.a for x in d[:3]] + [x.a for x in ints[:3]]
    assert ptts_paged.attention_workspace(*a, out=d[3].a, max_rows=1, max_kv=1) == 0
    ptts_paged.attention(*a, out=d[3].a, status=ints[3].a, max_rows=1, max_kv=1)
    # One key: its value.  The kernel forms v w / w with a weight w near 1: a product, a reciprocal and a product in float32, each off by at most
    # 2^-24 of its result, so 3.01 2^-24 in all.  Half a step of float16 is 2^-11: there it rounds back to v.
    off = np.abs(ref.from_bits(d[3].host(), kind) - v[page_of, 0])
    assert (off <= (3.01 * 2.0 ** -24 * np.abs(v[page_of, 0]) if kind == "float32" else 0.0)).all(), off.max()
    assert ints[3].host()[0] == 0


@pytest.mark.parametrize("hints", [(1, 1), (1, 1 << 30), (1 << 30, 1), (5, 64)])
@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
def test_hints_that_are_wrong_change_no_results(kind, hints):
    """max_rows and max_kv far from the truth: other forms and splits, the same results within the bounds."""
    import ptts_paged
    from test_paged_gpu import _attend, _compare
    real, query = ptts_paged.attention, ptts_paged.attention_workspace
    over = dict(max_rows=hints[0], max_kv=hints[1])
    try:
        ptts_paged.attention = lambda *a, **k: real(*a, **{**k, **over})
        ptts_paged.attention_workspace = lambda *a, **k: query(*a, **{**k, **over})
        for lens in ([(300, 70), (0, 1), (900, 2)], [(2500, 1), (40, 1)]):
            for window, sinks in ((0, 0), (130, 9)):
                _compare(*_attend(lens, 4, 2, 64, 16, kind, kind, window, sinks), kind, 64)
    finally:
        ptts_paged.attention, ptts_paged.attention_workspace = real, query


@pytest.mark.parametrize("window,sinks", [(50, 2 ** 31 - 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1 << 30, 5), ((1 << 30) + 1, 3), (-5, 7), (1, 0)])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_windows_and_sinks_at_their_limits(kind, window, sinks):
    from test_paged_gpu import _attend, _compare
    _compare(*_attend([(300, 70), (0, 1), (900, 2)], 4, 2, 64, 16, kind, kind, window, sinks), kind, 64)
