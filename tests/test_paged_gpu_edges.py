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
