"""Corners of the paged cache's operators and of the selection: scores out of range, scales far apart, sequences beyond the first 64, shared pages that are
cut back, equal rows at odd places, handles and streams.

The plain restatements, the inputs' helpers and the tolerances' derivation are tests/test_paged.py's."""

import os
import subprocess
import sys

import numpy as np
import pytest

from calm_amd import paged
from conftest import ROOT
from test_paged import TYPES, U, Book, Cache, Fake, Rig, attention, check_select, dev, from_type, ints, to_type


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


# ---- queries with one large element -----------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [1, 45])
def test_an_outlier_in_a_row_costs_the_others_nothing(hiplib, dtype, dim, rows):
    """one element of q 4000 times the others, where K is zero: the scores are those of the other elements.  What a row leaves out of them is 6e-8 (2^-24) of its
    largest element and 2^-25 in chunks, so a score is off by sqrt(dim) * 2^-24 * 4000 * max|K| * dim ** -0.5 < 1e-3 at the very worst and a weight by twice that
    share: inside the 2^-9 of tests/test_paged.py, which stands for this."""
    r = Rig(1, 300, 1, dim, np.random.default_rng(dim))
    k = r.rng.standard_normal((300, 1, dim))
    k[:, :, 3] = 0
    r.add([300], "float32", k=to_type(k, "float32"))
    q = r.rng.standard_normal((rows, 2, dim))
    q[:, :, 3] = 4000 * np.sign(q[:, :, 3])
    q = to_type(q, dtype)
    got = from_type(paged.attend(r.pool, r.batch([rows]), dev(q, dtype)).numpy(), dtype)
    want = attention(from_type(q, dtype), r.k.values(0), r.v.values(0), dim ** -0.5, 0, 0)
    assert np.abs(got - want).max() <= (2.0 ** -9 + U[dtype]) * np.abs(r.v.values(0)).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens", [(1, 300), (45, 300), (1, 4100), (45, 4100)])
def test_a_row_that_weighs_one_token_returns_its_value(hiplib, dtype, rows, tokens):
    """one token's score 30 to 60 above all others (0): their weights, e^-30 in sum at most 4100 * 1e-13 = 4e-10, are nothing, so the output is that token's V -- exactly
    for 16-bit rows, whose sum of weights is that of the weights as they go into the product (V, a code of 7 bits times a power of two, is a number of the type), and
    to 2^-21 for fp32 ones: the weight as two halves (2^-22), the reciprocal, one product"""
    r = Rig(1, tokens, 1, 64, np.random.default_rng(37))
    k = np.zeros((tokens, 1, 64))
    at = tokens // 3
    k[at, 0] = np.where(r.rng.random(64) < 0.5, 1.0, -1.0)
    r.add([tokens], "float32", k=to_type(k, "float32"))
    q = k[at, 0] * (30 + 30 * r.rng.random((rows, 4, 1))) * 8 / 64  # q . K * 64 ** -0.5 = 30 .. 60
    got = from_type(paged.attend(r.pool, r.batch([rows]), dev(to_type(q, dtype), dtype)).numpy(), dtype)
    want = np.broadcast_to(r.v.values(0)[at, 0], got.shape)
    if dtype == "float32":
        np.testing.assert_allclose(got, want, rtol=2.0 ** -21, atol=1e-9 * np.abs(r.v.values(0)).max())
    else:
        np.testing.assert_allclose(got, want, rtol=0, atol=1e-7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens", [(1, 300), (45, 300), (1, 4100), (45, 4100)])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 22, 2.0 ** 26, 2.0 ** 60, 2.0 ** 110])
def test_huge_scores_pick_their_token_whatever_the_scales(hiplib, dtype, rows, tokens, size):
    """one token's score `size` above the others', among V's of very different scales, up to where fp32 ends: the output is that token's V (as above); where K is turned
    round, at -size, the output is that of the sequence without it"""
    if dtype == "float16" and size > 2.0 ** 22:
        pytest.skip("queries of fp16 and keys of int8 do not reach that far")
    r = Rig(1, tokens, 1, 64, np.random.default_rng(39))
    at = tokens // 3
    k = np.zeros((tokens, 1, 64))
    k[at, 0] = np.where(r.rng.random(64) < 0.5, 1.0, -1.0) * size ** 0.5
    v = r.rng.standard_normal((tokens, 1, 64)) * np.repeat(2.0 ** r.rng.integers(-9, 10, -(-tokens // 16)), 16)[:tokens, None, None]
    r.add([tokens], "float32", k=to_type(k, "float32"), v=to_type(v, "float32"))
    q = to_type(np.sign(k[at, 0]) * np.ones((rows, 4, 1)) * size ** 0.5 / 8, dtype)
    vv = r.v.values(0)[:, 0]
    got = from_type(paged.attend(r.pool, r.batch([rows]), dev(q, dtype)).numpy(), dtype)
    np.testing.assert_allclose(got, np.broadcast_to(vv[at], got.shape), rtol=2.0 ** -21 if dtype == "float32" else 0, atol=1e-9 * np.abs(vv[at]).max())
    got = from_type(paged.attend(r.pool, r.batch([rows]), dev(to_type(-from_type(q, dtype), dtype), dtype)).numpy(), dtype)
    left = np.arange(tokens) != at
    for t in range(rows):
        want = vv[left & (np.arange(tokens) <= tokens - rows + t)].mean(axis=0)
        assert np.abs(got[t] - want).max() <= (2.0 ** -9 + U[dtype]) * np.abs(vv).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_what_lies_behind_the_tokens_does_not_matter(hiplib, dtype, rows):
    """the same bits whatever the pages hold behind a sequence's tokens, in rows and blocks of one tile that some rows do not see, and in pages of nobody"""
    got = []
    for junk in (0x00, 0x01, 0x3F, 0x7F, 0xFF):
        r = Rig(2, 1000, 2, 64, np.random.default_rng(38))
        for a in (r.pool.k, r.pool.v, r.pool.k_scale, r.pool.v_scale):
            b = np.full(a.nbytes, junk, dtype=np.uint8)
            a._lib.copy_hip(a.data_ptr(), b.ctypes.data, b.nbytes)
        r.add([993, 70], "float32")
        q = to_type(r.rng.standard_normal((2 * rows, 8, 64)), dtype)
        b = r.batch([rows, rows])
        got.append([paged.attend(r.pool, b, dev(q, dtype), window=w).numpy() for w in (0, 37)])
        r.pool.check()
    for x in got[1:]:
        for a, b in zip(x, got[0]):
            np.testing.assert_array_equal(a, b)


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


# ---- V's scales -----------------------------------------------------------------------------------------------------------------------


def weighted_size(q, k, v, scale, window, sinks):
    """sum_j p_j max_d |V_j|: what an output is made of, [rows, heads]"""
    return attention(q, k, np.broadcast_to(np.abs(v).max(axis=2, keepdims=True), v.shape), scale, window, sinks)[..., 0]


def weighted_blocks(q, k, cache, scale, window, sinks):
    """sum_j p_j 127 s_j, s_j the scale of the token's block: what the same output could be made of, by the codes' range.  A row's reference is the largest
    p_j s_j it sees, whichever codes those tokens hold (small ones beside a large one are held in its steps already): with two binary16 halves up to
    2^15 and the largest at 2^6 or more, a term is off by 2^-31 of the reference times its code, n of them by n 2^-31 of this size: 3e-7 for 600."""
    s = np.repeat(np.stack([cache.scale[0, b] for b in range(-(-len(k) // 16))]), 16, axis=0)[:len(k)]
    return attention(q, k, np.broadcast_to(127 * s[:, :, None], k.shape), scale, window, sinks)[..., 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens", [(14, 408), (50, 408), (14, 4104), (50, 4104)])
@pytest.mark.parametrize("ratio", [12, 20, 60])
def test_large_values_that_a_row_does_not_weigh_cost_it_nothing(hiplib, dtype, rows, tokens, ratio):
    """V blocks 2^ratio larger: among the last tokens, which the earlier rows do not see, and one in the middle that every row sees and gives a weight of next
    to nothing.  The error is held against what the row's own output is made of, by the bounds of tests/test_paged.py."""
    dim, rng = 64, np.random.default_rng(ratio + rows)
    r = Rig(1, tokens, 1, dim, rng)
    u = rng.standard_normal(dim)
    k = rng.standard_normal((tokens, 1, dim))
    v = rng.standard_normal((tokens, 1, dim))
    far = slice(160, 176)
    k[far] = u * (-40 * dim ** 0.5 / (u @ u) * (1 + 0.02 * rng.standard_normal((16, 1, 1))))  # scores near -40
    if ratio == 60:
        k[far] *= 2  # ... of -80: e^-80 2^60 is nothing either
    v[far] *= 2.0 ** ratio
    last = (tokens - 1) // 16 * 16  # (the last block: later rows of a tile alone see it)
    v[last:] *= 2.0 ** ratio
    r.add([tokens], "float32", k=to_type(k, "float32"), v=to_type(v, "float32"))
    q = to_type(u + 0.05 * rng.standard_normal((rows, 2, dim)), dtype)
    got = from_type(paged.attend(r.pool, r.batch([rows]), dev(q, dtype)).numpy(), dtype)
    x, kv, vv = from_type(q, dtype), r.k.values(0), r.v.values(0)
    want = attention(x, kv, vv, dim ** -0.5, 0, 0)
    size = weighted_size(x, kv, vv, dim ** -0.5, 0, 0)
    before = tokens - rows + np.arange(rows) < last
    assert before.any() and not before.all()
    if dtype == "float16":  # (a result beyond the type's range is an infinity)
        over = np.abs(want) >= 65520
        np.testing.assert_array_equal(got[over], np.sign(want[over]) * np.inf)
        got[over] = want[over]
    err = np.abs(got - want) / size[..., None]
    assert err.max() <= 2.0 ** -9 + U[dtype], (err.max(), np.unravel_index(err.argmax(), err.shape))
    if dtype == "float32":
        assert ((err ** 2).mean(axis=(1, 2)) ** 0.5).max() <= 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 50])
def test_zeros_and_the_smallest_and_largest_scales(hiplib, rows):
    """blocks of zeros (the least scale there is), of 1e-36 and of 1e30 in one sequence, weighted alike or not"""
    rng = np.random.default_rng(35)
    r = Rig(1, 600, 1, 64, rng)
    v = rng.standard_normal((600, 1, 64))
    v[:100], v[200:300], v[400:450] = 0, v[200:300] * 1e-36, v[400:450] * 1e30
    r.add([600], "float32", v=to_type(v, "float32"))
    q = to_type(rng.standard_normal((rows, 2, 64)), "float32")
    for window in (0, 100, 170):
        got = paged.attend(r.pool, r.batch([rows]), dev(q), window=window).numpy().astype(np.float64)
        want = attention(q.astype(np.float64), r.k.values(0), r.v.values(0), 0.125, window, 0)
        size = weighted_blocks(q.astype(np.float64), r.k.values(0), r.v, 0.125, window, 0)
        err = np.abs(got - want) / size[..., None]
        assert err.max() <= 2.0 ** -9 + U["float32"] and (err ** 2).mean() ** 0.5 <= 2e-5, (window, err.max())
    # nothing but zeros, and nothing but the smallest
    for lo, hi in ((0, 100), (200, 300)):
        one = Rig(1, 100, 1, 64, rng)
        one.add([100], "float32", v=to_type(v[lo:hi], "float32"))
        got = paged.attend(one.pool, one.batch([rows]), dev(q)).numpy().astype(np.float64)
        want = attention(q.astype(np.float64), one.k.values(0), one.v.values(0), 0.125, 0, 0)
        err = np.abs(got - want) / max(np.abs(v[lo:hi]).max(), 1e-37)
        assert err.max() <= 2.0 ** -9 and (err ** 2).mean() ** 0.5 <= 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 50])
def test_values_beyond_any_weight(hiplib, rows):
    """V's 2^122 apart, the large ones under a weight of 2^-115: the output is made of both"""
    dim, rng = 64, np.random.default_rng(42)
    r = Rig(1, 300, 1, dim, rng)
    u = np.where(rng.random(dim) < 0.5, 1.0, -1.0)
    k, v = np.zeros((300, 1, dim)), rng.standard_normal((300, 1, dim)) * 2.0 ** -20
    k[64:80] = u * -(115 * np.log(2) / 8)  # q . K * dim ** -0.5 = -115 ln 2 for q = u
    v[64:80] *= 2.0 ** 122
    r.add([300], "float32", k=to_type(k, "float32"), v=to_type(v, "float32"))
    q = to_type(np.broadcast_to(u, (rows, 2, dim)), "float32")
    got = paged.attend(r.pool, r.batch([rows]), dev(q)).numpy().astype(np.float64)
    x, kv, vv = q.astype(np.float64), r.k.values(0), r.v.values(0)
    want, size = attention(x, kv, vv, dim ** -0.5, 0, 0), weighted_size(x, kv, vv, dim ** -0.5, 0, 0)
    err = np.abs(got - want) / size[..., None]
    # (a score of 80 is off by 80 * 2^-24 times a few: 1e-5 of its weight)
    assert err.max() <= 2.0 ** -9 + U["float32"] and (err ** 2).mean() ** 0.5 <= 2e-5, err.max()


# ---- batches that do not add up -------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,bad", [(70, 69), (70, 66), (64, 63), (200, 130)])
def test_append_reports_starts_of_any_sequence(hiplib, seqs, bad):
    """one token each for `seqs` sequences, one of them with starts outside its rows: it is not stored, and the pool says so"""
    r = Rig(seqs, 3, 1, 64, np.random.default_rng(seqs))
    starts = list(range(seqs + 1))
    if bad == seqs - 1:
        starts[-1] = seqs + 5
    else:
        starts[bad + 1] = starts[bad] - 3  # (the sequence behind it begins inside other rows: still within its bounds)
    x = dev(np.ones((seqs, 1, 64), dtype=np.float32))
    b = paged.KvBatch(r.dtable, ints([5] * seqs), ints(starts), rows=seqs, max_rows=seqs, max_len=5)
    paged.append(r.pool, b, x, x)
    with pytest.raises(RuntimeError, match="max_rows"):
        r.pool.check()
    good = paged.KvBatch(r.dtable, ints([1] * seqs), ints(list(range(seqs + 1))), rows=seqs, max_rows=1, max_len=1)
    paged.append(r.pool, good, x, x)
    r.pool.check()


# ---- pages that rows share ------------------------------------------------------------------------------------------------------------


def fill(pool, rng):
    """random bytes in every page; the host's copy"""
    want = []
    for x in (pool.k, pool.v, pool.k_scale, pool.v_scale):
        junk = rng.integers(-128, 128, x.shape).astype(np.int8) if x.dtype == "int8" else rng.standard_normal(x.shape).astype(np.float32)
        x._lib.copy_hip(x.data_ptr(), junk.ctypes.data, junk.nbytes)
        want.append(junk)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,layers", [(1, 64, 1), (3, 96, 2)])
def test_a_row_cut_back_into_a_shared_page_gets_its_own(hiplib, heads, dim, layers):
    """rows that share full pages are cut back into them (drafts given up behind a fork): before new tokens go in, reserve gives each writer a page of its own
    with the old one's bytes; the rows that keep the page keep its bytes"""
    rng = np.random.default_rng(heads)
    pool = paged.KvPool(layers, 20, heads, dim)
    want = fill(pool, rng)
    # rows 0 .. 2 list pages 0, 1, 2 (192 tokens); row 3 lists 0, 1 and owns 3; row 4 owns 4
    t0 = [[0, 1, 2, -1], [0, 1, 2, -1], [0, 1, 2, -1], [0, 1, 3, -1], [4, -1, -1, -1]]
    r0 = [4, 4, 3, 1, 1] + [0] * 15
    table, refs = dev(np.array(t0, dtype=np.int32)), dev(np.array(r0, dtype=np.int32))
    # row 0 goes back to 100 tokens (inside page 1), row 1 to 128 (a border), row 2 keeps 192, row 3 goes back to 70, row 4 to 10
    lens = [100, 128, 192, 70, 10]
    paged.trim(pool, table, refs, ints(lens))
    np.testing.assert_array_equal(refs.numpy(), [4, 4, 1, 0, 1] + [0] * 15)
    new = [101, 130, 192, 70, 12]
    paged.reserve(pool, table, refs, ints(lens), ints(new))
    # pages in rows' order, the lowest free one each: row 0 a copy of page 1, row 1 a new page; row 3 adds no token and copies nothing, row 4 owns its page
    np.testing.assert_array_equal(table.numpy(), [[0, 3, -1, -1], [0, 1, 5, -1], [0, 1, 2, -1], [0, 1, -1, -1], [4, -1, -1, -1]])
    np.testing.assert_array_equal(refs.numpy(), [4, 3, 1, 1, 1, 1] + [0] * 14)
    for x in want:
        x[:, 3] = x[:, 1]
    for got, x in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), want):
        np.testing.assert_array_equal(got.numpy(), x)
    # every row that lists page 1 goes on inside it: each gets a copy, and the page itself is free
    lens = [101, 100, 100, 100, 12]
    paged.trim(pool, table, refs, ints(lens))
    paged.reserve(pool, table, refs, ints(lens), ints([n + 1 for n in lens]))
    t, n = table.numpy(), refs.numpy()
    assert len({t[1, 1], t[2, 1], t[3, 1], t[0, 1], t[4, 0], 0}) == 6 and (t[:4, 0] == 0).all()
    counts = np.bincount(t[t >= 0], minlength=20)
    np.testing.assert_array_equal(n, counts)
    for row in (1, 2, 3):
        for x, got in zip(want, (pool.k, pool.v, pool.k_scale, pool.v_scale)):
            np.testing.assert_array_equal(got.numpy()[:, t[row, 1]], x[:, 1])
    pool.check()


@pytest.mark.gpu
def test_no_page_for_a_row_cut_back_into_a_shared_one(hiplib):
    """no free page: the row loses the entry rather than write into the others' page, and the pool says so"""
    pool = paged.KvPool(1, 2, 1, 64)
    table, refs = dev(np.array([[0, 1], [0, 1]], dtype=np.int32)), dev(np.array([2, 2], dtype=np.int32))
    paged.reserve(pool, table, refs, ints([100, 128]), ints([101, 128]))
    np.testing.assert_array_equal(table.numpy(), [[0, -1], [0, 1]])
    np.testing.assert_array_equal(refs.numpy(), [2, 1])
    with pytest.raises(RuntimeError, match="no page was free"):
        pool.check()


@pytest.mark.gpu
def test_drafts_given_up_behind_a_fork(hiplib):
    """two rows of one prompt, full pages shared; one is cut back into them and goes on: the other's values stay"""
    rng = np.random.default_rng(41)
    pool = paged.KvPool(1, 12, 2, 64)
    table, refs = dev(np.full((2, 4), -1, dtype=np.int32)), dev(np.zeros(12, dtype=np.int32))
    k, v = Cache(2, 64), Cache(2, 64)

    def add(lens, new, rows):
        paged.reserve(pool, table, refs, ints(lens), ints(new))
        starts = np.concatenate([[0], np.cumsum([b - a for a, b in zip(lens, new)])])
        batch = paged.KvBatch(table, ints(new), ints(starts), rows=int(starts[-1]), max_rows=int(np.diff(starts).max()), max_len=max(new))
        paged.append(pool, batch, dev(rows), dev(-rows))

    rows = rng.standard_normal((128, 2, 64)).astype(np.float32)
    add([0, 0], [128, 0], rows)
    k.append(0, rows.astype(np.float64)), v.append(0, -rows.astype(np.float64))
    table, refs = paged.fork(pool, table, ints([128, 0]), refs, ints([0, 0]))
    paged.trim(pool, table, refs, ints([80, 128]))  # (80: a block's border, so that the first row's old blocks keep their scales)
    add([80, 128], [90, 128], rng.standard_normal((10, 2, 64)).astype(np.float32) * 50)
    gk, gv = paged.read(pool, table, ints([90, 128]), ints([0, 0]), 128)
    for got, want in ((gk, k), (gv, v)):
        np.testing.assert_array_equal(got.numpy()[1], want.values(0).astype(np.float32))
        np.testing.assert_array_equal(got.numpy()[0, :80], want.values(0)[:80].astype(np.float32))
        assert np.abs(got.numpy()[0, 80:90]).max() > 50
    pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,pages", [(9, 80), (300, 1500), (1500, 4000)])
def test_rounds_of_sharing_and_cutting_back(hiplib, rows, pages):
    """fork, cut back to any length, go on: table, counts and bytes follow the plain bookkeeping, more rows than the workgroup has threads among them"""
    rng = np.random.default_rng(rows)
    mp = 4
    pool = paged.KvPool(1, pages, 1, 64)
    want = fill(pool, rng)
    book = Book(pages, rows, mp)
    table, refs = dev(np.array(book.table, dtype=np.int32)), dev(np.array(book.refs, dtype=np.int32))
    lens = [0] * rows
    for step in range(6):
        new = [min(n + int(x), 64 * mp) for n, x in zip(lens, rng.integers(0, 60, rows))]
        live = sum(x > 0 for x in book.refs)
        if live + sum(-(-m // 64) - n // 64 for n, m in zip(lens, new)) > pages:
            new = lens
        paged.reserve(pool, table, refs, ints(lens), ints(new))
        given, held = [], list(book.refs)
        for row, a, b in zip(book.table, lens, new):
            for c in range(a // 64, -(-b // 64) if b > a else a // 64):
                if a % 64 and c == a // 64 and row[c] >= 0 and held[row[c]] > 1:
                    given.append(row[c])
                    row[c] = book.take()
                    for x in want:
                        x[:, row[c]] = x[:, given[-1]]
                elif row[c] < 0:
                    row[c] = book.take()
        for p in given:
            book.refs[p] -= 1
        book.same(table.numpy(), refs.numpy())
        lens = new
        # most rows continue one of a few
        parents = [int(p) for p in np.where(rng.random(rows) < 0.8, rng.integers(0, max(rows // 6, 1), rows), np.arange(rows))]
        free = sum(x == 0 for x in book.refs)
        if sum(lens[p] % 64 > 0 for p in parents) > free:
            parents = list(range(rows))
        table, refs = paged.fork(pool, table, ints(lens), refs, ints(parents))
        for src, to in book.fork(lens, parents):
            for x in want:
                x[:, to] = x[:, src]
        book.same(table.numpy(), refs.numpy())
        lens = [lens[p] for p in parents]
        lens = [int(rng.integers(0, n + 1)) if rng.random() < 0.4 else n for n in lens]
        paged.trim(pool, table, refs, ints(lens))
        book.trim(lens)
        book.same(table.numpy(), refs.numpy())
        live = [p for p in range(pages) if book.refs[p]]
        for got, x in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), want):
            np.testing.assert_array_equal(got.numpy()[:, live], x[:, live])
    pool.check()
    assert max(book.refs) > 1


@pytest.mark.gpu
def test_reserve_does_not_make_up_a_page_that_is_lost(hiplib):
    """a row whose last tokens' page is missing: the entry stays -1 (whatever a free page holds would be read as those tokens), the pages behind it are given"""
    pool = paged.KvPool(1, 6, 1, 64)
    table, refs = dev(np.array([[0, -1, -1], [1, -1, -1]], dtype=np.int32)), dev(np.array([1, 1, 0, 0, 0, 0], dtype=np.int32))
    paged.reserve(pool, table, refs, ints([100, 64]), ints([130, 65]))
    np.testing.assert_array_equal(table.numpy(), [[0, -1, 2], [1, 3, -1]])
    np.testing.assert_array_equal(refs.numpy(), [1, 1, 1, 1, 0, 0])
    with pytest.raises(RuntimeError, match="missing"):
        pool.check()


@pytest.mark.gpu
def test_every_page_that_a_row_goes_on_in_is_its_own(hiplib):
    """a row that was cut back without giving its pages up: those behind its tokens are the others', too, and are not written"""
    rng = np.random.default_rng(43)
    pool = paged.KvPool(2, 12, 1, 64)
    want = fill(pool, rng)
    # three rows of four shared pages (256 tokens)
    table, refs = dev(np.array([[0, 1, 2, 3, -1]] * 3, dtype=np.int32)), dev(np.array([3, 3, 3, 3] + [0] * 8, dtype=np.int32))
    # row 0 goes on from 70 to 200 tokens, row 1 from 128 to 129, row 2 stays
    paged.reserve(pool, table, refs, ints([70, 128, 256]), ints([200, 129, 256]))
    np.testing.assert_array_equal(table.numpy(), [[0, 4, 5, 6, -1], [0, 1, 7, 3, -1], [0, 1, 2, 3, -1]])
    np.testing.assert_array_equal(refs.numpy(), [3, 2, 1, 2, 1, 1, 1, 1, 0, 0, 0, 0])
    for x in want:
        x[:, 4] = x[:, 1]  # (tokens 64 .. 69 of row 0; nothing of the other pages is a token of it)
    for got, x in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), want):
        np.testing.assert_array_equal(got.numpy(), x)
    # the last two that list page 3 both go on in it: both give it up, and the lower row takes it as the lowest free page
    paged.reserve(pool, table, refs, ints([192, 192, 192]), ints([192, 200, 193]))
    np.testing.assert_array_equal(table.numpy(), [[0, 4, 5, 6, -1], [0, 1, 7, 3, -1], [0, 1, 2, 8, -1]])
    np.testing.assert_array_equal(refs.numpy(), [3, 2, 1, 1, 1, 1, 1, 1, 1, 0, 0, 0])
    pool.check()


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("beams,vocab", [(4, 20011), (3, 8193), (8, 32001), (16, 1001), (2, 128257)])
def test_select_equal_beams_at_any_alignment(hiplib, dtype, beams, vocab):
    """hypotheses with the same logits and the same score: their totals are equal, so the lowest beam's tokens come first, wherever a row begins"""
    rng = np.random.default_rng(vocab)
    x = np.repeat(rng.standard_normal((2, 1, vocab)) * 3, beams, axis=1).reshape(2 * beams, vocab)
    check_select(x, np.zeros((2, beams)), None, -1, dtype)
    check_select(x, np.full((2, beams), -1.5), None, -1, dtype, strided=3)


def test_select_refuses_vocabularies_beyond_its_indexes(hiplib):
    assert hiplib.beam_workspace_hip(1, 1, 1 << 30) > 0
    assert hiplib.beam_workspace_hip(1, 1, (1 << 30) + 1) == -1 and b"2^30 tokens" in hiplib.calm_hip_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("beams,vocab", [(8, 500), (5, 9001)])
def test_select_beams_whose_logits_differ_by_a_constant(hiplib, dtype, beams, vocab):
    """a constant on all of a row's logits changes no log softmax: the totals are equal still, and the lowest beam comes first"""
    rng = np.random.default_rng(beams)
    x = np.repeat(rng.integers(-8, 9, (6, 1, vocab)).astype(np.float64), beams, axis=1).reshape(6 * beams, vocab)
    scores = np.repeat(-3 * rng.random((6, 1)), beams, axis=1)
    shifted = to_type(x + np.tile(rng.permutation(np.arange(beams)), 6)[:, None] * 16, dtype)  # (whole numbers below 256: exact in every type)
    want = paged.beam_select(dev(to_type(x, dtype), dtype), dev(scores.astype(np.float32)))
    got = paged.beam_select(dev(shifted, dtype), dev(scores.astype(np.float32)))
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), b.numpy())
    check_select(x, scores, None, -1, dtype)


# ---- handles and streams --------------------------------------------------------------------------------------------------------------


def test_handles_are_not_changed():
    """a pool's and a batch's arrays and bounds went to the library when they were made: a change would be seen by the checks here and not by the kernels"""
    k, v, s = Fake((2, 10, 2, 64, 64), "int8"), Fake((2, 10, 2, 4, 64, 16), "int8"), Fake((2, 10, 2, 4), "float32")
    t, n, st = Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32")
    b = paged.KvBatch(t, n, st, 2, 1, 10)
    for name, x in (("table", t), ("lens", n), ("starts", st), ("rows", 1), ("max_rows", 1), ("max_len", 5), ("n_seqs", 1)):
        with pytest.raises(AttributeError, match="make another"):
            setattr(b, name, x)
    with pytest.raises(AttributeError, match="make another"):
        del b.table
    assert (b.table, b.rows) == (t, 2)
    pool = paged.KvPool.__new__(paged.KvPool)
    for name, x in (("k", k), ("v", v), ("k_scale", s), ("v_scale", s), ("n_layers", 2), ("_c", None)):  # (as its constructor does, without memory)
        setattr(pool, name, x)
    with pytest.raises(AttributeError, match="make another"):
        pool.k = k


@pytest.mark.gpu
def test_paged_operators_on_torch_tensors_corners():
    """streams and gradients of torch tensors, in a process of its own: torch has to come before the library"""
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "tests", "paged_corners_child.py")], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("ALL OK"), r.stdout[-2000:] + r.stderr[-3000:]
