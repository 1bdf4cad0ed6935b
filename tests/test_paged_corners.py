"""Corners of the paged cache's operators and of the selection: scores out of range, scales far apart, sequences beyond the first 64, shared pages that are
cut back, equal rows at odd places, handles and streams.

The plain restatements, the inputs' helpers and the tolerances' derivation are tests/test_paged.py's."""

import numpy as np
import pytest

from calm_amd import paged
from test_paged import TYPES, U, Cache, Rig, attention, check_select, dev, from_type, ints, to_type


# ---- scores and queries out of range --------------------------------------------------------------------------------------------------


def marked(rows, heads, dim, dtype="float32"):
    return dev(to_type(np.full((rows, heads, dim), 77.0), dtype), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 45])
@pytest.mark.parametrize("tokens", [90, 4100])
def test_rows_whose_scores_overflow_are_nan(hiplib, rows, tokens):
    """numbers near 1e20 in q and K: scores beyond 2^128 on both sides of zero, in contexts walked by one workgroup and by several.  (The softmax of +inf is NaN in
    32 bits; what must not happen is that the row keeps what its memory held.)"""
    r = Rig(1, tokens, 1, 64, np.random.default_rng(31))
    r.add([tokens], "float32", k=to_type(r.rng.standard_normal((tokens, 1, 64)) * 1e20, "float32"))
    q = to_type(r.rng.standard_normal((rows, 2, 64)) * 1e20, "float32")
    out = marked(rows, 2, 64)
    paged.attend(r.pool, r.batch([rows]), dev(q), out=out)
    assert np.isnan(out.numpy()).all()
    r.pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 45])
@pytest.mark.parametrize("tokens", [90, 4100])
def test_a_row_with_an_infinity_is_nan(hiplib, dtype, rows, tokens):
    """whatever its sign and the keys' signs; the other rows are what they are without it"""
    r = Rig(1, tokens, 1, 64, np.random.default_rng(32))
    k = r.rng.standard_normal((tokens, 1, 64))
    k[:, :, 5] = np.abs(k[:, :, 5]) + 0.5  # (-inf times these: a row whose scores are all -inf)
    r.add([tokens], "float32", k=to_type(k, "float32"))
    q = to_type(r.rng.standard_normal((rows, 4, 64)), dtype)
    clean = paged.attend(r.pool, r.batch([rows]), dev(q, dtype)).numpy()
    bad = np.array(q)
    for h, x in ((1, np.inf), (2, -np.inf), (3, np.nan)):
        bad[rows // 2, h, 5] = to_type(np.full(1, x), dtype)[0]
    out = marked(rows, 4, 64, dtype)
    paged.attend(r.pool, r.batch([rows]), dev(bad, dtype), out=out)
    got = from_type(out.numpy(), dtype)
    assert np.isnan(got[rows // 2, 1:]).all()
    keep = np.ones((rows, 4), dtype=bool)
    keep[rows // 2, 1:] = False
    np.testing.assert_array_equal(got[keep], from_type(clean, dtype)[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 45])
@pytest.mark.parametrize("tokens", [90, 4100])
def test_a_row_whose_scores_are_all_beyond_range_below_is_nan(hiplib, rows, tokens):
    """it sees tokens, so zeros -- the answer of a row that sees none -- would pass for a result"""
    r = Rig(2, tokens, 1, 64, np.random.default_rng(33))
    k = to_type((np.abs(r.rng.standard_normal((tokens, 1, 64))) + 0.1) * 1e20, "float32")
    r.add([tokens, 0], "float32", k=k)
    q = to_type((np.abs(r.rng.standard_normal((2 * rows, 2, 64))) + 0.1) * -1e20, "float32")
    out = marked(2 * rows, 2, 64)
    paged.attend(r.pool, r.batch([rows, rows]), dev(q), out=out)
    got = out.numpy()
    assert np.isnan(got[:rows]).all() and not got[rows:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30])
@pytest.mark.parametrize("rows", [12, 50])
def test_the_widest_windows_beside_rows_before_position_0(hiplib, rows, window):
    """a sequence of fewer tokens than rows, under a window that ends beyond 32 bits before its first rows: the rows at positions see what they see without a window"""
    r = Rig(2, 100, 2, 64, np.random.default_rng(36))
    r.add([rows - 7, 90], "float32")
    q = dev(to_type(r.rng.standard_normal((2 * rows, 4, 64)), "float32"))
    want = paged.attend(r.pool, r.batch([rows, rows]), q).numpy()
    got = paged.attend(r.pool, r.batch([rows, rows]), q, window=window).numpy()
    np.testing.assert_array_equal(got, want)
    got = paged.attend(r.pool, r.batch([rows, rows]), q, window=window, sinks=2 ** 31 - 1).numpy()
    np.testing.assert_array_equal(got, want)
    assert not got[:7].any() and got[7:].any(axis=(1, 2)).all()


# ---- selection ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("beams,vocab", [(2, 9000), (8, 128256), (1, 20000), (32, 9000)])
def test_select_a_finished_beam_beside_dead_ones(hiplib, beams, vocab):
    """as many chunks of the vocabulary as beams, or more: behind the finished beam's end token come its other tokens, at -inf, the lowest first"""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((2 * beams, vocab))
    scores = np.full((2, beams), -np.inf)
    done = np.zeros((2, beams))
    scores[0, 0], done[0, 0] = -3.0, 1
    scores[1, -1], done[1, -1] = -2.0, 1
    for eos in (0, 1, vocab - 1):
        check_select(x, scores, done, eos)
