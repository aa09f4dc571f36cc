"""Paged LM states with a window and sinks against a float64 model that keeps every row, in pools that are exactly large enough, and
what calls that are refused leave behind."""
import threading

import numpy as np
import pytest

from lm_ref import Lm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(packs):
    import ptts_lib
    e = ptts_lib.Engine(packs["small"][0], precision="fp32", temperature=0.0, lsd_steps=2, max_frames=64)
    yield e
    e.close()


def _rows(rng, n, d):
    return (rng.standard_normal((n, d)) * 0.5).astype(np.float32)


def _held(length, page, window, sinks):
    """Pages of a slot of `length` rows after its last row went in alone: those of the sinks and those that this row's window touches."""
    return sum(p * page < sinks or (p + 1) * page > length - window for p in range(-(-length // page))) if window else -(-length // page)


@pytest.mark.parametrize("page,window,sinks", [(8, 40, 11), (8, 40, 16), (7, 33, 0), (1, 20, 3), (16, 16, 17), (5, 1, 0)])
def test_window_in_a_pool_without_a_spare_page(eng, packs, page, window, sinks):
    """Pages that fall behind the window are taken by the other slot in the same step, so a page given back too early, or a row of the sinks
    lost, changes the results; the free pages say whether one is given back too late."""
    _, spec, w = packs["small"]
    rng = np.random.default_rng(page)
    start, steps = (23, 9, 1), 90
    length = np.array(start)
    pool = max(sum(_held(n + k, page, window, sinks) for n in start) for k in range(1, steps + 1))
    pool = max(pool, sum(-(-n // page) for n in start))
    st, refs = eng.paged_state(3, pages=pool, page_size=page, max_context=200, window=window, sinks=sinks), [Lm(spec, w, window, sinks) for _ in start]
    for i, n in enumerate(start):
        x = _rows(rng, n, eng.d_model)
        eng.lm_prefill(st, i, x)
        refs[i].rows(x)
    assert st.free_pages() == pool - sum(-(-n // page) for n in start)
    seq = np.full((3, eng.latent), np.nan, np.float32)
    for k in range(steps):
        cond, eos = eng.lm_step(st, seq)
        length += 1
        assert st.free_pages() == pool - sum(_held(n, page, window, sinks) for n in length), k
        for i, r in enumerate(refs):
            want, want_eos = r.latent(seq[i])
            # float32 sums of a few hundred terms in two layers, as against the oracle
            assert np.abs(cond[i] - want).max() < 1e-3 and abs(eos[i] - want_eos) < 1e-3, (k, i)
        seq = (rng.standard_normal((3, eng.latent)) * 0.7).astype(np.float32)
    st.close()


def test_window_over_prompts_in_chunks(eng, packs):
    """Prompts longer than the window, in passes of 128 rows and in pieces, then steps."""
    _, spec, w = packs["small"]
    rng = np.random.default_rng(3)
    st, ref = eng.paged_state(1, pages=22, page_size=16, max_context=600, window=100, sinks=20), Lm(spec, w, 100, 20)
    for n in (300, 1, 77):
        x = _rows(rng, n, eng.d_model)
        eng.lm_prefill(st, 0, x)
        ref.rows(x)
    for k in range(4):
        z = (rng.standard_normal((1, eng.latent)) * 0.7).astype(np.float32)
        cond, eos = eng.lm_step(st, z)
        want, want_eos = ref.latent(z[0])
        assert np.abs(cond[0] - want).max() < 1e-3 and abs(eos[0] - want_eos) < 1e-3, k
    st.close()


@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 200])
def test_sinks_that_cover_everything(eng, packs, sinks):
    """With all rows sinks a window hides nothing and no page comes back."""
    _, spec, w = packs["small"]
    rng = np.random.default_rng(5)
    st, ref = eng.paged_state(1, pages=9, page_size=8, max_context=72, window=5, sinks=sinks), Lm(spec, w)
    x = _rows(rng, 30, eng.d_model)
    eng.lm_prefill(st, 0, x)
    ref.rows(x)
    for k in range(40):
        z = (rng.standard_normal((1, eng.latent)) * 0.7).astype(np.float32)
        cond, _ = eng.lm_step(st, z)
        assert np.abs(cond[0] - ref.latent(z[0])[0]).max() < 1e-3, k
        assert st.free_pages() == 9 - -(-(31 + k) // 8)
    st.close()


def test_refused_step_gives_no_page_back(eng):
    """Three slots need a page each and one could give one back: the step is refused and the first rows can still be shared."""
    import ptts_lib
    rng = np.random.default_rng(6)
    st = eng.paged_state(3, pages=4, page_size=8, max_context=64, window=8)
    for i, n in enumerate((16, 8, 8)):
        eng.lm_prefill(st, i, _rows(rng, n, eng.d_model))
    assert st.free_pages() == 0
    seq = np.zeros((3, eng.latent), np.float32)
    with pytest.raises(ptts_lib.PttsError, match="free pages"):
        eng.lm_step(st, seq)
    assert st.free_pages() == 0
    st.share(0, 1, 8)                       # page 0 of slot 0 is still there; slot 1's comes back
    assert st.free_pages() == 1
    st.close()
    # the limit of the context is met by the second slot only
    st = eng.paged_state(2, pages=20, page_size=8, max_context=24, window=8)
    for i, n in enumerate((17, 24)):
        eng.lm_prefill(st, i, _rows(rng, n, eng.d_model))
    free = st.free_pages()
    with pytest.raises(ptts_lib.PttsError, match="max_context"):
        eng.lm_step(st, np.zeros((2, eng.latent), np.float32))
    assert st.free_pages() == free
    st.close()


def test_step_that_fits_through_pages_shared_behind_the_window(eng):
    """Two slots share the pages that both leave behind in one step: they come back once, and the step takes them."""
    rng = np.random.default_rng(7)
    st = eng.paged_state(2, pages=3, page_size=8, max_context=64, window=8)
    eng.lm_prefill(st, 0, _rows(rng, 16, eng.d_model))
    st.share(0, 1, 16)
    assert st.free_pages() == 1             # 2 pages, both in both slots
    seq = np.zeros((2, eng.latent), np.float32)
    out = eng.lm_step(st, seq)[0]           # both give page 0 back and need one each
    assert st.free_pages() == 0
    np.testing.assert_array_equal(out[0], out[1])
    st.close()


def test_share_into_a_slot_of_a_full_pool(eng, packs):
    """A finished utterance's slot begins anew with the voice though no page is free: its own pages serve."""
    import ptts_lib
    _, spec, w = packs["small"]
    rng = np.random.default_rng(8)
    voice, other = _rows(rng, 11, eng.d_model), _rows(rng, 16, eng.d_model)
    st, ref = eng.paged_state(2, pages=4, page_size=8, max_context=32), Lm(spec, w)
    eng.lm_prefill(st, 0, voice)
    eng.lm_prefill(st, 1, other)
    assert st.free_pages() == 0
    st.share(0, 1, 11)
    assert st.free_pages() == 1             # the whole page is shared, the three rows of the second are copied
    eng.lm_prefill(st, 1, other[:5])
    ref.rows(voice)
    ref.rows(other[:5])
    z = np.zeros((2, eng.latent), np.float32)
    cond, _ = eng.lm_step(st, z)
    assert np.abs(cond[1] - ref.latent(z[1])[0]).max() < 1e-3
    st.close()
    # pages that are shared with the source do not serve
    st = eng.paged_state(2, pages=2, page_size=8, max_context=32)
    eng.lm_prefill(st, 0, _rows(rng, 11, eng.d_model))
    st.share(0, 1, 8)
    with pytest.raises(ptts_lib.PttsError, match="no free page"):
        st.share(0, 1, 9)
    assert st.free_pages() == 0
    st.close()


def test_free_pages_and_reset_beside_steps(eng):
    """Another thread asks for the free pages, and resets a state of its own, while steps run."""
    a, b = (eng.paged_state(2, pages=40, page_size=2, max_context=40) for _ in range(2))
    seen, stop, errors = set(), threading.Event(), []

    def ask():
        try:
            while not stop.is_set():
                seen.add(a.free_pages())
                b.reset()
        except BaseException as e:
            errors.append(e)

    t = threading.Thread(target=ask)
    t.start()
    try:
        for _ in range(40):
            eng.lm_step(a, np.zeros((2, eng.latent), np.float32))
    finally:
        stop.set()
        t.join()
    assert not errors and seen <= set(range(0, 41, 2)) and a.free_pages() == 0 and b.free_pages() == 40
    a.close()
    b.close()


def test_the_codec_beside_a_paged_lm(eng):
    """A paged state decodes as a fixed one does."""
    rng = np.random.default_rng(9)
    fixed, paged = eng.state(1), eng.paged_state(1, pages=4)
    z = (rng.standard_normal((6, eng.latent)) * 0.7).astype(np.float32)
    for part in (z[:2], z[2:]):
        np.testing.assert_array_equal(eng.mimi_decode(paged, part[None]), eng.mimi_decode(fixed, part[None]))
    fixed.close()
    paged.close()
