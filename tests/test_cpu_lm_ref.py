"""The float64 language model that the paged state's tests compare with, against the oracle."""
import numpy as np
import pytest

from lm_ref import Lm


def test_lm_ref_matches_oracle(packs, oracle_mod):
    path, spec, w = packs["small"]
    o, ref, rng = oracle_mod.Oracle(path), Lm(spec, w), np.random.default_rng(0)
    st = o.lm_state(64)
    voice = (rng.standard_normal((9, spec.d_model)) * 0.5).astype(np.float32)
    o.lm_main(st, None, voice)
    ref.rows(voice)
    cur = np.full((1, spec.latent_dim), np.nan, np.float32)
    for k in range(20):
        cond, eos = o.lm_main(st, cur, None)
        want, want_eos = ref.latent(cur[0])
        # float32 sums of a few hundred terms in two layers
        assert np.abs(cond - want).max() < 1e-4 and abs(eos - want_eos) < 1e-4, k
        cur = (rng.standard_normal((1, spec.latent_dim)) * 0.7).astype(np.float32)


@pytest.mark.parametrize("window,sinks", [(6, 0), (6, 3), (1, 2), (50, 0)])
def test_lm_ref_window(packs, window, sinks):
    """Rows that fell out of the window do not matter, whatever they hold; those of the sinks do."""
    _, spec, w = packs["tiny"]
    rng = np.random.default_rng(1)
    x = rng.standard_normal((30, spec.d_model))
    a, b = (Lm(spec, w, window, sinks) for _ in range(2))
    a.rows(x)
    b.rows(x)
    gone = slice(sinks, max(sinks, 31 - window))     # the next row, at position 30, sees from 31 - window on
    for m in (b.keys, b.values):
        for i in range(spec.lm_layers):
            m[i][gone] = rng.standard_normal(m[i][gone].shape)
    y = rng.standard_normal((1, spec.d_model))
    np.testing.assert_array_equal(a.rows(y)[0], b.rows(y)[0])
    if sinks:
        for i in range(spec.lm_layers):
            b.values[i][:sinks] += 1.0
        assert np.abs(a.rows(y)[0] - b.rows(y)[0]).max() > 1e-3
