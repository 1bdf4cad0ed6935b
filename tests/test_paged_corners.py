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
