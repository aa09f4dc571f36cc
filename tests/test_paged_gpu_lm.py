"""The LM on a paged state (ptts_state_new_paged) against the fixed cache and the oracle: prompts in chunks, a shared voice, windows with
sinks in a bounded pool."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engines(packs):
    import ptts_lib
    made = {}

    def get(precision, pack="small"):
        if (precision, pack) not in made:
            made[precision, pack] = ptts_lib.Engine(packs[pack][0], precision=precision, temperature=0.0, lsd_steps=2, max_frames=64)
        return made[precision, pack]

    yield get
    for e in made.values():
        e.close()


def _rows(rng, n, d):
    return (rng.standard_normal((n, d)) * 0.5).astype(np.float32)


def _steps(eng, st, n, seed):
    rng = np.random.default_rng(seed)
    out = []
    seq = np.full((st.batch, eng.latent), np.nan, np.float32)
    for _ in range(n):
        out.append(eng.lm_step(st, seq))
        seq = (rng.standard_normal((st.batch, eng.latent)) * 0.7).astype(np.float32)
    return np.array([c for c, _ in out]), np.array([e for _, e in out])


# float32: two orders of the same float32 sums (24 bits, a few thousand terms).  bf16: keys and values are rounded to bf16 in both caches
# from rotations that agree to float32, so a few of them round the other way (one part in 256 of one value each).
@pytest.mark.parametrize("precision,tol", [("fp32", 2e-4), ("bf16", 1e-2)])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_paged_state_matches_fixed_cache(engines, precision, tol, page):
    eng = engines(precision)
    rng = np.random.default_rng(page)
    prompts = [_rows(rng, n, eng.d_model) for n in (37, 150, 5)]
    fixed, paged = eng.state(3), eng.paged_state(3, pages=600 // page + 6, page_size=page, max_context=400)
    for i, p in enumerate(prompts):
        eng.lm_prefill(fixed, i, p)
        cut = [0, len(p) // 3, len(p) // 3 + 1, len(p)]         # in chunks, one of them a single row
        for a, b in zip(cut, cut[1:]):
            if b > a:
                eng.lm_prefill(paged, i, p[a:b])
    want, got = _steps(eng, fixed, 20, 1), _steps(eng, paged, 20, 1)
    for w, g in zip(want, got):
        np.testing.assert_allclose(g, w, rtol=0, atol=tol * max(1.0, np.abs(w).max()))
    paged.reset()
    fixed.reset()
    assert paged.free_pages() == 600 // page + 6
    want, got = _steps(eng, fixed, 3, 2), _steps(eng, paged, 3, 2)
    np.testing.assert_allclose(got[0], want[0], rtol=0, atol=tol * max(1.0, np.abs(want[0]).max()))
    fixed.close()
    paged.close()


def test_paged_state_matches_oracle(engines, packs, oracle_mod):
    path, spec, _ = packs["small"]
    eng, o = engines("fp32"), oracle_mod.Oracle(path)
    rng = np.random.default_rng(4)
    voice, ids = _rows(rng, 21, spec.d_model), rng.integers(0, spec.vocab, 9).astype(np.int64)
    st, ref = eng.paged_state(1, pages=8, page_size=16), o.lm_state(128)
    eng.lm_prefill(st, 0, voice)
    eng.lm_prefill(st, 0, eng.text_conditioner(ids))
    o.lm_main(ref, None, voice)
    o.lm_main(ref, None, o.text_conditioner(ids))
    cur = np.full((1, spec.latent_dim), np.nan, np.float32)
    for k in range(12):
        cond, eos = eng.lm_step(st, cur)
        want, want_eos = o.lm_main(ref, cur, None)
        assert np.abs(cond[0] - want).max() < 1e-3 and abs(eos[0] - want_eos) < 1e-3, k
        cur = (rng.standard_normal((1, spec.latent_dim)) * 0.7).astype(np.float32)
    st.close()


def test_int8_engine_runs_on_pages(engines):
    # the int8 scheme is discontinuous (two correct engines agree to about 1e-1, see the int8 tests); a wrong page would be off by the signal
    eng = engines("int8", "small")
    rng = np.random.default_rng(8)
    p = _rows(rng, 40, eng.d_model)
    fixed, paged = eng.state(2), eng.paged_state(2, pages=12, page_size=16)
    for s in (fixed, paged):
        for i in range(2):
            eng.lm_prefill(s, i, p)
    want, got = _steps(eng, fixed, 6, 3)[0], _steps(eng, paged, 6, 3)[0]
    assert np.linalg.norm(got - want) < 0.2 * np.linalg.norm(want)
    fixed.close()
    paged.close()


@pytest.mark.parametrize("page", [16, 7])
def test_shared_voice(engines, page):
    """One voice's rows in one slot, shared by the others: the same results as a prefill of each, with fewer pages."""
    eng = engines("fp32")
    rng = np.random.default_rng(page)
    voice, texts = _rows(rng, 62, eng.d_model), [_rows(rng, n, eng.d_model) for n in (9, 20, 1)]
    alone, shared = (eng.paged_state(3, pages=60, page_size=page, max_context=140) for _ in range(2))
    for i in range(3):
        eng.lm_prefill(alone, i, voice)
    eng.lm_prefill(shared, 0, voice)
    for i in (1, 2):
        shared.share(0, i, 62)
    assert shared.free_pages() == 60 - (-(-62 // page)) - 2 * (62 % page != 0)
    for s in (alone, shared):
        for i, t in enumerate(texts):
            eng.lm_prefill(s, i, t)
    want, got = _steps(eng, alone, 10, 5), _steps(eng, shared, 10, 5)
    np.testing.assert_array_equal(got[0], want[0])           # the same kernels on the same rows
    np.testing.assert_array_equal(got[1], want[1])
    # the shared slot may be given up and taken again while the others go on
    shared.share(1, 0, 62)
    alone.share(1, 0, 62)
    eng.lm_prefill(shared, 0, texts[2])
    eng.lm_prefill(alone, 0, texts[2])
    np.testing.assert_array_equal(_steps(eng, shared, 3, 6)[0], _steps(eng, alone, 3, 6)[0])
    alone.close()
    shared.close()


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_window_runs_in_a_bounded_pool(engines, precision):
    """A long stream whose pages behind the window return to the pool sees what a stream that keeps them all sees."""
    eng = engines(precision)
    rng = np.random.default_rng(2)
    voice = _rows(rng, 20, eng.d_model)
    kw = dict(page_size=8, max_context=400, window=40, sinks=11)
    small, large = eng.paged_state(2, pages=2 * 10, **kw), eng.paged_state(2, pages=110, **kw)
    for s in (small, large):
        for i in range(2):
            eng.lm_prefill(s, i, voice)
    got, want = _steps(eng, small, 150, 9), _steps(eng, large, 150, 9)
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    # held: the pages of the sinks (2) and those that the window of 40 touches (6 at most), for each slot
    assert small.free_pages() >= 20 - 2 * 8
    # while nothing has fallen out of the window, it changes nothing
    plain, window = eng.paged_state(1, pages=10, page_size=8), eng.paged_state(1, pages=10, page_size=8, window=60)
    for s in (plain, window):
        eng.lm_prefill(s, 0, voice)
    np.testing.assert_array_equal(_steps(eng, window, 30, 3)[0], _steps(eng, plain, 30, 3)[0])
    for s in (small, large, plain, window):
        s.close()


def test_refusals(engines):
    import ptts_lib
    eng = engines("fp32")
    rng = np.random.default_rng(0)
    st = eng.paged_state(2, pages=4, page_size=16, max_context=64)
    with pytest.raises(ptts_lib.PttsError, match="free pages"):
        eng.lm_prefill(st, 0, _rows(rng, 65 - 1, eng.d_model)) or eng.lm_prefill(st, 1, _rows(rng, 1, eng.d_model))
    st.reset()
    eng.lm_prefill(st, 0, _rows(rng, 40, eng.d_model))       # 3 pages
    with pytest.raises(ptts_lib.PttsError, match="free pages"):
        eng.lm_prefill(st, 1, _rows(rng, 17, eng.d_model))
    assert st.free_pages() == 1                               # nothing was taken
    eng.lm_prefill(st, 1, _rows(rng, 16, eng.d_model))
    with pytest.raises(ptts_lib.PttsError, match="free pages"):
        eng.lm_step(st, np.zeros((2, eng.latent), np.float32))
    with pytest.raises(ptts_lib.PttsError, match="max_context"):
        eng.lm_prefill(st, 0, _rows(rng, 25, eng.d_model))
    for a, b, n in ((0, 0, 1), (0, 2, 1), (-1, 0, 1), (0, 1, 41), (0, 1, -1)):
        with pytest.raises(ptts_lib.PttsError):
            st.share(a, b, n)
    with pytest.raises(ptts_lib.PttsError, match="not created with pages"):
        eng.state(1).free_pages()
    for bad in (dict(pages=4, page_size=0), dict(pages=4, window=-1), dict(pages=4, sinks=-1), dict(pages=1 << 20, page_size=1 << 12), dict(pages=0)):
        with pytest.raises(ptts_lib.PttsError):
            eng.paged_state(1, **bad)
    st.close()
