"""The paged-cache operators against float64, through the public bindings: the block-table plan, rotary positions with the append,
and attention over the pages."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def _table(total, page, rng, spare=3, width=None):
    """(block table, page count) with the pages of a pool dealt out at random."""
    need = [-(-int(t) // page) for t in total]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.full((len(total), max(max(need, default=0), 1) if width is None else width), -1, np.int64)
    k = 0
    for i, n in enumerate(need):
        table[i, :n] = order[k:k + n]
        k += n
    return table, pages, order[k:]


# ---------------------------------------------------------------- plan

PLANS = [
    # cached, arriving, page, table width beyond need, free pages beyond need, rows beyond need
    ([0], [1], 16, 0, 0, 0),
    ([5, 16, 17, 0], [1, 1, 1, 1], 16, 2, 3, 2),
    ([0, 0, 0], [0, 0, 0], 7, 1, 1, 3),
    ([100, 3, 0, 64, 31], [1, 0, 300, 64, 2], 32, 0, 0, 5),
    ([7, 7, 7], [50, 60, 70], 1, 0, 2, 0),
    ([10, 20, 30], [100, 200, 300], 24, 1, -5, 0),          # the free list runs out
    ([10, 20, 30], [100, 200, 300], 24, -4, 0, 0),          # table rows too short
    ([10, 20, 30], [100, 200, 300], 16, 0, 0, -57),         # more rows than room for them
    ([3, -2, 9], [5, 4, -6], 8, 1, 1, 1),                   # negative lengths count as 0
]


def _run_plan(cached, arriving, page, table, free, rows):
    import ptts_paged
    n = len(cached)
    d = {k: ref.Dev(np.asarray(v), "int32") for k, v in dict(cached=cached, arriving=arriving, free=free, table=table, slots=np.full(rows, -7),
         positions=np.full(rows, -7), cu=np.zeros(n + 1), kv_len=np.zeros(n), counts=np.zeros(4), status=np.zeros(1)).items()}
    ptts_paged.plan(d["cached"].a, d["arriving"].a, d["free"].a, d["table"].a, page, slot_map=d["slots"].a, positions=d["positions"].a,
                    cu_rows=d["cu"].a, kv_len=d["kv_len"].a, counts=d["counts"].a, status=d["status"].a)
    return [d[k].host() for k in ("table", "slots", "positions", "cu", "kv_len", "counts")], int(d["status"].host()[0])


@pytest.mark.parametrize("cached,arriving,page,wider,more_free,more_rows", PLANS)
def test_plan(cached, arriving, page, wider, more_free, more_rows):
    rng = np.random.default_rng(page)
    c, a = np.maximum(cached, 0), np.maximum(arriving, 0)
    have, end = -(-c // page), -(-(c + a) // page)
    width = max(int(end.max()) + wider, 1)
    order = rng.permutation(int(end.sum()) + max(more_free, 0) + 1)
    table = np.full((len(c), width), -1)
    k = 0
    for i in range(len(c)):
        m = min(int(have[i]), width)
        table[i, :m] = order[k:k + m]
        k += m
    free = order[k:k + max(int((end - have).sum()) + more_free, 0)]
    rows = max(int(a.sum()) + more_rows, 0)
    want = ref.plan(cached, arriving, free, table, page, rows)
    got, status = _run_plan(cached, arriving, page, table, free, rows)
    for name, g, w in zip(("table", "slots", "positions", "cu", "kv_len", "counts"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)
    assert bool(status & 4) == (min(cached) < 0 or min(arriving) < 0)


@pytest.mark.parametrize("n,most,page", [(64, 1, 16), (1024, 9, 16), (1025, 40, 5), (5000, 3, 1)])
def test_plan_many_requests(n, most, page):
    rng = np.random.default_rng(n)
    cached, arriving = rng.integers(0, 60, n), rng.integers(0, most + 1, n)
    have, end = -(-cached // page), -(-(cached + arriving) // page)
    order = rng.permutation(int(end.sum()) + 4)
    table = np.full((n, int(end.max()) + 1), -1)
    table[np.arange(table.shape[1]) < have[:, None]] = order[:int(have.sum())]
    rows = int(arriving.sum()) + 2
    want = ref.plan(cached, arriving, order[int(have.sum()):], table, page, rows)
    got, status = _run_plan(cached, arriving, page, table, order[int(have.sum()):], rows)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    assert status == 0


# ---------------------------------------------------------------- rotary positions and append

ROTARY = [
    # rows, heads, kv_heads, dim, rot, interleaved, type, cache, page, first position, magnitude
    (1, 16, 16, 64, 64, True, "float32", "float32", 16, 0, 1.0),
    (64, 16, 16, 64, 64, True, "float32", "bfloat16", 16, 531, 1.0),
    (67, 4, 2, 128, 128, False, "bfloat16", "bfloat16", 24, 1048000, 1.0),
    (33, 6, 3, 96, 32, False, "float16", "float16", 7, 1 << 20, 1.2079),
    (19, 5, 1, 80, 40, True, "bfloat16", "bfloat16", 1, 77, 1.0),
    (19, 5, 5, 80, 40, False, "float32", "float32", 64, 3, 1.0),          # half = 20: a multiple of 4, wide in f32
    (9, 2, 2, 80, 40, False, "float16", "float16", 16, 100000, 0.5),      # half = 20: no multiple of 8, value by value
    (1030, 3, 1, 32, 32, True, "float16", "float16", 16, 9, 1.0),
    (2050, 2, 1, 256, 6, False, "bfloat16", "bfloat16", 100, 9, 1.0),
    (5, 1, 1, 8, 2, True, "float32", "float32", 3, 2, 1.0),
]


def _rotary_bound(x, want, rot, cache):
    """Two products and a sum in float32 around cosine and sine that are off by at most 3e-7 (angle reduction 2^-52 of the turns,
    fraction rounded to float32, a few units of the functions), then one rounding to the stored type."""
    big = np.abs(x).max(-1, keepdims=True) * 2 * 6e-7
    return big + ref.EPS[cache] * np.abs(want) + 1e-30


@pytest.mark.parametrize("case", ROTARY)
@pytest.mark.parametrize("layout", ["plain", "fused", "odd"])
def test_rotary_append(case, layout):
    import ptts_paged
    rows, heads, kvh, dim, rot, inter, kind, cache, page, first, mag = case
    rng = np.random.default_rng(rows + dim)
    x = rng.standard_normal((rows, heads + 2 * kvh, dim)).astype(np.float32)
    x = ref.rounded(x, kind)
    pages = -(-rows // page) + 2
    slots = rng.permutation(pages * page)[:rows]
    slots[rows // 2] = -1                                              # one row is not stored
    positions = first + np.arange(rows)
    freq = ptts_paged.frequencies(rot)[0]
    k0 = ref.rounded(rng.standard_normal((pages, page, kvh, dim)), cache)
    v0 = ref.rounded(rng.standard_normal((pages, page, kvh, dim)), cache)
    dk, dv = ref.floats(k0, cache), ref.floats(v0, cache)
    dq = ref.floats(np.zeros((rows, heads, dim)), kind)
    args = [ref.Dev(positions, "int32"), ref.Dev(freq, "float64"), ref.Dev(slots, "int32")]
    if layout == "plain":
        t = [ref.floats(x[:, a:b], kind) for a, b in ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh))]
        q, k, v = (d.a for d in t)
    else:
        # one row after the other, q, k and v side by side; "odd": rows start at no multiple of 16 bytes
        extra = 1 if layout == "odd" else 0
        flat = np.zeros((rows, (heads + 2 * kvh) * dim + extra), np.float32)
        flat[:, extra:] = x.reshape(rows, -1)
        t = [ref.floats(flat, kind)]
        w = flat.shape[1]
        q = t[0].view(extra, (rows, heads, dim), (w, dim, 1))
        k = t[0].view(extra + heads * dim, (rows, kvh, dim), (w, dim, 1))
        v = t[0].view(extra + (heads + kvh) * dim, (rows, kvh, dim), (w, dim, 1))
    status = ref.Dev(np.zeros(1), "int32")
    ptts_paged.rotary_append(q, k, v, args[0].a, args[1].a, interleaved=inter, magnitude=mag, q_out=dq.a, slot_map=args[2].a,
                             k_pages=dk.a, v_pages=dv.a, status=status.a)
    xq, xk, xv = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
    want = ref.rotate(xq.astype(np.float64), positions, freq, inter, np.float32(mag))
    got = ref.from_bits(dq.host(), kind)
    assert (np.abs(got - want) <= _rotary_bound(xq, want, rot, kind)).all()
    wk, wv = k0.astype(np.float64), v0.copy()
    turned = ref.rotate(xk.astype(np.float64), positions, freq, inter, np.float32(mag))
    for r, s in enumerate(slots):
        if s >= 0:
            wk[s // page, s % page], wv[s // page, s % page] = turned[r], ref.rounded(xv[r], cache)
    gk, gv = ref.from_bits(dk.host(), cache), ref.from_bits(dv.host(), cache)
    hit = np.zeros((pages * page,), bool)
    hit[slots[slots >= 0]] = True
    hit = hit.reshape(pages, page)
    np.testing.assert_array_equal(gk[~hit], k0[~hit])                   # slots that nobody names stay as they were
    np.testing.assert_array_equal(gv, wv)
    assert (np.abs(gk[hit] - wk[hit]) <= _rotary_bound(wk[hit], wk[hit], rot, cache)).all()
    assert status.host()[0] == 0


def test_rotary_in_place_and_parts():
    import ptts_paged
    rng = np.random.default_rng(0)
    x = ref.rounded(rng.standard_normal((37, 3, 64)), "bfloat16")
    freq, mag = ptts_paged.frequencies(64, scaling="parts", factor=8.0, trained=4096)
    pos = np.arange(37) * 900
    d, p, f = ref.floats(x, "bfloat16"), ref.Dev(pos, "int32"), ref.Dev(freq, "float64")
    ptts_paged.rotary_append(d.a, None, None, p.a, f.a, magnitude=mag)
    want = ref.rotate(x.astype(np.float64), pos, freq, False, np.float32(mag))
    assert (np.abs(ref.from_bits(d.host(), "bfloat16") - want) <= _rotary_bound(x, want, 64, "bfloat16")).all()


def test_rotary_bad_slots_are_skipped_and_reported():
    import ptts_paged
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 4, 1, 64)).astype(np.float32)
    slots = np.array([3, 32, -5, 1])                                    # 2 pages of 16: 32 is outside, -5 is no slot
    pages = [ref.floats(np.zeros((2, 16, 1, 64)), "float32") for _ in range(2)]
    d = [ref.floats(k, "float32"), ref.floats(v, "float32"), ref.Dev(np.arange(4), "int32"), ref.Dev(np.ones(32), "float64"),
         ref.Dev(slots, "int32"), ref.Dev(np.zeros(1), "int32")]
    ptts_paged.rotary_append(None, d[0].a, d[1].a, d[2].a, d[3].a, slot_map=d[4].a, k_pages=pages[0].a, v_pages=pages[1].a, status=d[5].a)
    got = pages[1].host().reshape(32, 64)
    np.testing.assert_array_equal(got[3], v[0, 0])
    np.testing.assert_array_equal(got[1], v[3, 0])
    assert d[5].host()[0] == 1 and not got[[0] + list(range(4, 32))].any()


# ---------------------------------------------------------------- attention

ATTEND = [
    # name, (cached, new) of each request, heads, kv_heads, dim, page, type, cache, window, sinks
    ("first row", [(0, 1)], 2, 2, 64, 16, "bfloat16", "bfloat16", 0, 0),
    ("decode", [(0, 1), (15, 1), (16, 1), (63, 1), (64, 1), (200, 1), (333, 1)], 4, 4, 64, 16, "bfloat16", "bfloat16", 0, 0),
    ("decode grouped", [(7, 1), (130, 1), (1000, 1)], 16, 2, 128, 24, "float16", "float16", 0, 0),
    ("decode one key head", [(257, 1), (90, 1)], 20, 1, 64, 7, "bfloat16", "bfloat16", 0, 0),
    ("decode f32", [(0, 1), (218, 1), (37, 1)], 4, 4, 64, 16, "float32", "float32", 0, 0),
    ("decode f32 rows, bf16 pages", [(100, 1), (31, 1)], 4, 2, 64, 16, "float32", "bfloat16", 0, 0),
    ("chunk", [(0, 70)], 3, 3, 64, 16, "bfloat16", "bfloat16", 0, 0),
    ("chunk after context", [(129, 100), (40, 33), (0, 64)], 4, 2, 64, 32, "float16", "float16", 0, 0),
    ("chunk of 128 wide heads", [(70, 150)], 4, 1, 128, 16, "bfloat16", "bfloat16", 0, 0),
    ("chunk of 256 wide heads", [(33, 40), (3, 1)], 2, 1, 256, 16, "bfloat16", "bfloat16", 0, 0),
    ("odd head", [(33, 40), (50, 1)], 6, 3, 80, 5, "bfloat16", "bfloat16", 0, 0),
    ("narrow head", [(10, 20), (50, 1)], 4, 2, 8, 16, "float16", "float16", 0, 0),
    ("head of 96 in f32", [(30, 20), (50, 1)], 4, 2, 96, 16, "float32", "float32", 0, 0),
    ("head of 192", [(30, 40), (50, 1)], 2, 2, 192, 16, "float16", "float16", 0, 0),
    ("chunk f32", [(90, 50), (0, 17)], 4, 2, 64, 16, "float32", "float32", 0, 0),
    ("chunk f32 over bf16", [(90, 50), (0, 17)], 4, 4, 128, 16, "float32", "bfloat16", 0, 0),
    ("mixed", [(100, 1), (0, 130), (64, 0), (300, 1), (10, 90)], 4, 2, 64, 24, "bfloat16", "bfloat16", 0, 0),
    ("pages of one row", [(20, 30), (77, 1)], 2, 2, 64, 1, "bfloat16", "bfloat16", 0, 0),
    ("large pages", [(20, 30), (77, 1)], 2, 2, 64, 4096, "float16", "float16", 0, 0),
    ("window", [(300, 1), (40, 1), (200, 90)], 4, 2, 64, 16, "bfloat16", "bfloat16", 50, 0),
    ("window of one", [(30, 1), (10, 20)], 2, 2, 64, 16, "bfloat16", "bfloat16", 1, 0),
    ("window and sinks", [(400, 1), (3, 1), (250, 150)], 4, 2, 64, 16, "float16", "float16", 70, 5),
    ("sinks meet the window", [(100, 1), (90, 60)], 2, 1, 128, 8, "bfloat16", "bfloat16", 64, 60),
    ("window and sinks f32", [(400, 1), (3, 1), (150, 60)], 2, 2, 64, 16, "float32", "float32", 33, 3),
    ("wide window", [(100, 50)], 2, 2, 64, 16, "bfloat16", "bfloat16", 100000, 9),
]


def _attend(lens, heads, kvh, dim, page, kind, cache, window, sinks, *, layout="nhd", poison=None, behind=3, hints=True, scale=None, seed=0,
            spread=1.0, workspace=True):
    """Runs a case; returns what the call wrote and what float64 says."""
    import ptts_paged
    rng = np.random.default_rng(seed + dim + len(lens))
    cached, new = np.array([c for c, _ in lens]), np.array([n for _, n in lens])
    total = cached + new
    table, pages, _ = _table(total, page, rng)
    pool = rng.standard_normal((2, pages, page, kvh, dim))
    k, v = ref.rounded(pool[0] * spread, cache), ref.rounded(pool[1], cache)
    used = np.zeros((pages, page), bool)
    for i, t in enumerate(total):
        j = np.arange(t)
        used[table[i, j // page], j % page] = True
    k[~used], v[~used] = np.nan, np.nan                     # rows that no request holds must not matter
    if poison is not None:
        poison(k, v, table, page, total)
    cu = np.concatenate([[0], np.cumsum(new)])
    rows = int(cu[-1]) + behind
    q = ref.rounded(rng.standard_normal((rows, heads, dim)) * spread, kind)
    if layout == "hnd":
        kd, vd = (ref.floats(np.transpose(x, (0, 2, 1, 3)), cache) for x in (k, v))
        ka, va = (d.view(0, k.shape, (kvh * page * dim, dim, page * dim, 1)) for d in (kd, vd))
    elif layout == "joint":                                 # keys and values of a page side by side
        kd = vd = ref.floats(np.stack([k, v], 1), cache)
        n = page * kvh * dim
        ka, va = (kd.view(o, k.shape, (2 * n, kvh * dim, dim, 1)) for o in (0, n))
    else:
        kd, vd = ref.floats(k, cache), ref.floats(v, cache)
        ka, va = kd.a, vd.a
    if layout == "nhd":
        qd = ref.floats(q, kind)
        qa = qd.a
    else:                                                   # rows of a wider buffer
        wide = np.zeros((rows, heads + 2, dim), np.float32)
        wide[:, 1:-1] = q
        qd = ref.floats(wide, kind)
        qa = qd.view(dim, q.shape, ((heads + 2) * dim, dim, 1))
    before = np.full(q.shape, 7.0)
    od, ld = ref.floats(before, kind), ref.floats(np.full((rows, heads), 7.0), "float32")
    ints = [ref.Dev(x, "int32") for x in (table, cu, total, np.zeros(1))]
    more = dict(window=window, sinks=sinks, scale=scale, max_rows=int(new.max()) if hints else 0, max_kv=int(total.max()) if hints else 0)
    need = ptts_paged.attention_workspace(qa, ka, va, *(d.a for d in ints[:3]), out=od.a, **more)
    ws = ref.Dev(np.full(max(need, 16), 255), "uint8")      # NaN patterns: nothing may be taken from it
    from ptts_paged import DeviceArray
    wa = DeviceArray(ws.ptr, (max(need, 16) // 4,), "int32")
    ptts_paged.attention(qa, ka, va, *(d.a for d in ints[:3]), out=od.a, lse=ld.a, workspace=wa, status=ints[3].a, **more)
    out, lse = ref.from_bits(od.host(), kind), ld.host()

    def rows_of(x):
        def pick(i):
            j = np.arange(total[i])
            return x[table[i, j // page], j % page]
        return pick

    want = ref.attention(q, rows_of(k), rows_of(v), cu, total, dim ** -0.5 if scale is None else scale, window, sinks)
    return out, lse, want, int(cu[-1]), int(ints[3].host()[0]), int(total.max())


def _compare(out, lse, want, live, status, longest, kind, dim):
    w_out, w_lse, size, logit = want
    assert status == 0
    assert (out[live:] == 7.0).all() and (lse[live:] == 7.0).all()       # rows behind the last request
    out, lse, w_out, w_lse, size, logit = (x[:live] for x in (out, lse, w_out, w_lse, size, logit))
    fine = np.isfinite(w_out)
    np.testing.assert_array_equal(np.isnan(out), np.isnan(w_out))
    np.testing.assert_array_equal(out[~fine & ~np.isnan(w_out)], w_out[~fine & ~np.isnan(w_out)])
    b_out, b_lse = ref.attention_bounds(w_out, size, logit, np.where(np.isfinite(w_lse), w_lse, 0), kind, dim, longest)
    off = np.abs(out - w_out)[fine] / b_out[fine]
    assert off.max(initial=0.0) <= 1.0, off.max()
    shown = np.isfinite(w_lse)
    np.testing.assert_array_equal(lse[~shown & ~np.isnan(w_lse)], w_lse[~shown & ~np.isnan(w_lse)])
    off = np.abs(lse - w_lse)[shown] / b_lse[shown]
    assert off.max(initial=0.0) <= 1.0, off.max()


@pytest.mark.parametrize("case", ATTEND, ids=[c[0] for c in ATTEND])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "joint"])
def test_attention(case, layout):
    _, lens, heads, kvh, dim, page, kind, cache, window, sinks = case
    got = _attend(lens, heads, kvh, dim, page, kind, cache, window, sinks, layout=layout)
    _compare(*got, kind, dim)


@pytest.mark.parametrize("case", [c for c in ATTEND if c[0] in ("decode", "mixed", "chunk after context", "chunk f32", "window and sinks")], ids=lambda c: c[0])
def test_attention_without_hints(case):
    _, lens, heads, kvh, dim, page, kind, cache, window, sinks = case
    _compare(*_attend(lens, heads, kvh, dim, page, kind, cache, window, sinks, hints=False), kind, dim)


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("lens", [[(0, 0), (5, 0), (0, 3), (0, 0)], [(-3, 5), (-2, 2), (4, 1)], [(-90, 170), (60, 1)]])
def test_attention_rows_that_see_nothing(kind, lens):
    # more rows than the length: the first of them lie before position 0
    _compare(*_attend(lens, 4, 2, 64, 16, kind, kind, 0, 0), kind, 64)


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("lens", [[(100, 60), (30, 1)], [(20, 3), (64, 4)], [(0, 200)]])
def test_attention_unseen_nan_and_infinity(kind, window, sinks, lens):
    """A key that is NaN or infinite reaches the rows that see it and no other."""
    def poison(k, v, table, page, total):
        j = total[0] - 2                       # seen by the last two rows of request 0 at most
        at = table[0, j // page], j % page
        v[at][0, 3], v[at][0, 5], v[at][1, 7] = np.nan, np.inf, -np.inf
        j = total[0] - 1
        at = table[0, j // page], j % page
        k[at][0, 1] = np.nan
        v[at][1, 9] = np.inf
        if window:
            at = table[0, 5 // page], 5 % page  # behind the window of most rows
            v[at][0, 2], v[at][1, 2] = np.nan, np.inf

    _compare(*_attend(lens, 4, 2, 64, 16, kind, kind, window, sinks, poison=poison), kind, 64)


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_attention_large_logits_and_scale(kind):
    _compare(*_attend([(300, 70), (150, 1)], 4, 2, 64, 16, kind, kind, 0, 0, spread=6.0), kind, 64)
    _compare(*_attend([(300, 70), (150, 1)], 4, 2, 64, 16, kind, kind, 0, 0, scale=3.0), kind, 64)


@pytest.mark.parametrize("lens,heads,kvh,dim,kind", [([(9000, 1)], 2, 1, 128, "bfloat16"), ([(5000, 1), (20, 1), (0, 1)], 4, 2, 64, "float32"),
                                                     ([(4000, 40), (100, 5)], 2, 2, 64, "float16")])
def test_attention_split_over_long_contexts(lens, heads, kvh, dim, kind):
    for window, sinks in ((0, 0), (3000, 10)):
        _compare(*_attend(lens, heads, kvh, dim, 16, kind, kind, window, sinks), kind, dim)


def test_attention_many_requests():
    rng = np.random.default_rng(3)
    lens = [(int(c), int(n)) for c, n in zip(rng.integers(0, 40, 300), rng.integers(0, 3, 300))]
    _compare(*_attend(lens, 2, 2, 64, 16, "bfloat16", "bfloat16", 0, 0), "bfloat16", 64)


def test_attention_bad_pages_and_lengths_are_reported():
    """Page ids outside the pool are not read: their keys count as rows of zeros, and the status says so."""
    import ptts_paged
    from ptts_paged import DeviceArray
    rng = np.random.default_rng(5)
    for kind, new in (("bfloat16", 1), ("bfloat16", 40), ("float32", 3)):
        pages, page, dim = 6, 16, 64
        k, v = (ref.rounded(rng.standard_normal((pages, page, 1, dim)), kind) for _ in range(2))
        table = np.array([[0, 99, 2, -4], [3, 4, 5, 1]])
        total, cu = np.array([60, 500]), np.array([0, new, new + 1])   # the second length passes its table: 64 rows
        q = ref.rounded(rng.standard_normal((new + 1, 2, dim)), kind)
        d = [ref.floats(x, kind) for x in (q, k, v, np.zeros_like(q))]
        ints = [ref.Dev(x, "int32") for x in (table, cu, total, np.zeros(1))]
        need = ptts_paged.attention_workspace(d[0].a, d[1].a, d[2].a, *(x.a for x in ints[:3]), out=d[3].a)
        ws = ref.Dev(np.zeros(max(need, 16)), "uint8")
        ptts_paged.attention(d[0].a, d[1].a, d[2].a, *(x.a for x in ints[:3]), out=d[3].a, workspace=DeviceArray(ws.ptr, (max(need, 16) // 4,), "int32"),
                             status=ints[3].a)

        def rows_of(x):
            def pick(i):
                n = min(int(total[i]), 64)
                j = np.arange(n)
                ids = table[i, j // page]
                return np.where(((ids >= 0) & (ids < pages))[:, None, None], x[np.clip(ids, 0, pages - 1), j % page], 0.0)
            return pick

        want = ref.attention(q, rows_of(k), rows_of(v), cu, [60, 64], dim ** -0.5)
        got = ref.from_bits(d[3].host(), kind)
        bound, _ = ref.attention_bounds(want[0], want[2], want[3], want[1], kind, dim, 64)
        assert (np.abs(got - want[0]) <= bound).all()
        assert ints[3].host()[0] == 1 | 4
