"""The paged 8-bit cache and the beam selection (calm_amd/paged.py, include/calm_hip.h) against plain 64-bit restatements.

Tolerances, from the types alone.  u(t) = torch.finfo(t).eps / 2: fp32 2^-24, fp16 2^-11, bf16 2^-8 -- one rounding.
  codes, scales, values read back as fp32, tables, counts, selected tokens: equal.  (Scales are powers of two, so x / scale is exact and the one
      rounding, to a code, is the same in 32 and 64 bits; rows are given in the type they are stored in.)
  attention, max |out - ref| over max |V| of the row's visible values (an output is an average of them, so that is its scale):
      scores: q . K in fp32 over at most 256 dims, |error| <= 256 * 2^-24 * sum |q K|; with |scale * sum |q K|| <= S_MAX = 32 in these tests (checked
      below) a score is off by less than 32 * 256 * 2^-24 = 4.9e-4 at the very worst, sqrt(256) instead of 256 in practice; for fp32 rows q's
      second half adds 2^-22 * 32.  (Few rows: q is held as base-254 digits, off by at most 0.5 / (127 * 254) = 1.55e-5 of the row's largest magnitude for 16-bit
      rows, by 6e-8 for fp32 ones, and the products are exact.  D such errors, evenly spread, move a score by a standard deviation of
      1.55e-5 / sqrt(3) * max|q| * |K| * scale; with max|q| <= 5 and |K| about sqrt(D) for normal rows and scale = D ** -0.5 that is 4.5e-5, four of them 1.8e-4,
      inside the 4.9e-4 above; rows whose largest element is 8 times as large still meet 2^-9 by 2 * 1.4e-3 + averaging, and have u(t) besides.)  A score error e changes a weight by a factor within 1 +- e.  2 e = 9.8e-4 bounds the output's error from scores
      (numerator and denominator).  The weight's own rounding: 2^-12 for 16-bit outputs (to binary16), 2^-22 for fp32.  exp2, sums: n * 2^-24 with
      n <= 4100 tokens at the very worst 2.4e-4.  Bounds below: 2^-9 = 2e-3 + u(t) covers all of these for every type; the typical error is far below,
      so fp32 has to meet 2e-5 in the root mean square besides (sums of n random errors of 2^-24 .. 2^-22, weights of 16 .. 4100 tokens)."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from calm_amd import paged
from conftest import ROOT

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TYPES = ["float32", "float16", "bfloat16"]


# ---- host copies of the types ---------------------------------------------------------------------------------------------------------


def to_type(x: np.ndarray, dtype: str) -> np.ndarray:
    """x rounded to `dtype`, as DeviceArray.of takes it (bfloat16: uint16)"""
    x = np.asarray(x, dtype=np.float32)
    if dtype != "bfloat16":
        with np.errstate(over="ignore"):
            return x.astype(dtype)
    b = x.view(np.uint32).astype(np.uint64)
    r = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def from_type(x: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "bfloat16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def dev(x, dtype=None):
    return paged.DeviceArray.of(np.ascontiguousarray(x), dtype)


def ints(v):
    return dev(np.array(v, dtype=np.int32))


# ---- the plain cache ------------------------------------------------------------------------------------------------------------------


class Cache:
    """sequences of quantised values, token by token, from the definition in include/calm_hip.h"""

    def __init__(self, heads, dim):
        self.heads, self.dim = heads, dim
        self.codes, self.scale, self.n = {}, {}, {}  # by (sequence, block): [16, heads, dim] and [heads]

    def append(self, s, rows):
        """rows [n, heads, dim] float64"""
        n = self.n.get(s, 0)
        for b in range(n // 16, (n + len(rows) + 15) // 16 if len(rows) else 0):
            old = min(max(n - 16 * b, 0), 16)
            new = rows[max(16 * b - n, 0):16 * b + 16 - n]
            top = np.abs(new).max(axis=(0, 2)) if len(new) else np.zeros(self.heads)
            codes = self.codes.setdefault((s, b), np.zeros((16, self.heads, self.dim)))
            scale = self.scale.setdefault((s, b), np.zeros(self.heads))
            for h in range(self.heads):
                if not np.isfinite(top[h]) or (old and np.isnan(scale[h])):
                    scale[h] = np.nan
                    codes[old:old + len(new), h] = 0
                    continue
                e = -126
                while 127 * 2.0 ** e < top[h]:
                    e += 1
                step = max(2.0 ** e, scale[h]) if old else 2.0 ** e
                if old:
                    codes[:old, h] = np.rint(codes[:old, h] * (scale[h] / step))
                codes[old:old + len(new), h] = np.rint(new[:, h] / step)
                scale[h] = step
        self.n[s] = n + len(rows)

    def values(self, s):
        n = self.n.get(s, 0)
        if n == 0:
            return np.zeros((0, self.heads, self.dim))
        out = [self.codes[s, b] * self.scale[s, b][None, :, None] for b in range((n + 15) // 16)]
        return np.concatenate(out)[:n]


def attention(q, k, v, scale, window, sinks):
    """q [n, heads, dim] are the last n of len(k) tokens; zeros for a row that sees nothing"""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = np.zeros_like(q)
    for t in range(n):
        p = len(k) - n + t
        j = np.arange(len(k))
        seen = (j <= p) & ((window <= 0) | (j > p - window) | (j < sinks))
        if not seen.any():
            continue
        for h in range(heads):
            x = k[seen, h // group] @ q[t, h] * scale
            w = np.exp(x - x.max())
            out[t, h] = (w / w.sum()) @ v[seen, h // group]
    return out


class Rig:
    """a pool, a table in scattered pages, and the plain cache beside it"""

    def __init__(self, seqs, tokens, heads, dim, rng, layers=1, layer=0):
        self.seqs, self.heads, self.dim, self.layer, self.rng = seqs, heads, dim, layer, rng
        self.mp = -(-tokens // 64) + 1
        self.pages = seqs * self.mp + 3
        self.pool = paged.KvPool(layers, self.pages, heads, dim)
        # memory that nobody initialised: every bit pattern a kernel may meet behind the tokens
        for a in (self.pool.k, self.pool.v, self.pool.k_scale, self.pool.v_scale):
            junk = np.full(a.nbytes, 0xFF, dtype=np.uint8)
            a._lib.copy_hip(a.data_ptr(), junk.ctypes.data, junk.nbytes)
        order = rng.permutation(self.pages)[: seqs * self.mp]
        self.table = order.reshape(seqs, self.mp).astype(np.int32)
        self.dtable = dev(self.table)
        self.k, self.v = Cache(heads, dim), Cache(heads, dim)
        self.lens = [0] * seqs

    def batch(self, rows, spare=0):
        starts = np.concatenate([[0], np.cumsum(rows)])
        return paged.KvBatch(self.dtable, ints(self.lens), ints(starts), rows=int(starts[-1]) + spare, max_rows=max(max(rows), 0), max_len=max(max(self.lens), 1))

    def add(self, rows, dtype, scale=1.0, strided=False, k=None, v=None):
        """append rows[s] tokens to every sequence"""
        total = sum(rows)
        k = to_type(self.rng.standard_normal((total, self.heads, self.dim)) * scale, dtype) if k is None else k
        v = to_type(self.rng.standard_normal((total, self.heads, self.dim)) * scale, dtype) if v is None else v
        at = 0
        for s, n in enumerate(rows):
            self.k.append(s, from_type(k[at:at + n], dtype))
            self.v.append(s, from_type(v[at:at + n], dtype))
            self.lens[s] += n
            at += n
        b = self.batch(rows)
        if strided:  # one packed array of k and v heads, as a fused projection leaves it
            both = dev(np.concatenate([k, v], axis=1), dtype)
            paged.append(self.pool, b, View(both, 0, (total, self.heads, self.dim)), View(both, self.heads * self.dim, (total, self.heads, self.dim)), layer=self.layer)
        else:
            paged.append(self.pool, b, dev(k, dtype), dev(v, dtype), layer=self.layer)

    def read(self, start, count, dtype="float32"):
        k, v = paged.read(self.pool, self.dtable, ints(self.lens), ints(start), count, layer=self.layer, dtype=dtype)
        return k.numpy(), v.numpy()

    def check_values(self):
        n = max(self.lens)
        k, v = self.read([0] * self.seqs, n + 5)
        for s in range(self.seqs):
            for got, want in ((k[s], self.k.values(s)), (v[s], self.v.values(s))):
                np.testing.assert_array_equal(got[:len(want)], want.astype(np.float32))
                assert not got[len(want):].any()


class View(paged.DeviceArray):
    """heads of a packed array, strided rows"""

    def __init__(self, base, offset, shape):
        self.base, self.shape, self.dtype = base, shape, base.dtype
        self._view = base.data_ptr() + offset * paged._SIZES[base.dtype]
        self._stride = base.stride()

    def data_ptr(self):
        return self._view

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return False


# ---- append, read ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dim", paged.HEAD_DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_append_then_read_is_the_definition(hiplib, dim, dtype):
    """prompts, single tokens, tokens that raise a block's scale, sequences without rows, across block and page borders"""
    r = Rig(4, 210, 3, dim, np.random.default_rng(dim), layers=2, layer=1)
    r.add([1, 63, 17, 0], dtype)
    r.check_values()
    for step, rows in enumerate(([1, 1, 1, 1], [1, 1, 0, 15], [64, 1, 2, 1], [3, 70, 129, 16], [1, 1, 1, 1])):
        r.add(rows, dtype, scale=[1.0, 9.0, 0.01, 30.0, 1e-3][step], strided=step % 2 == 0)
        r.check_values()
    r.pool.check()


@pytest.mark.gpu
def test_append_scale_borders_and_extremes(hiplib):
    """maxima at, just below and just above 127 * 2^e; zeros; the largest and the smallest numbers; ties to even"""
    r = Rig(1, 200, 1, 64, np.random.default_rng(5))
    tops = [127.0, np.nextafter(np.float32(127), np.float32(128)), 128.0, 63.5, 0.0, 3.0e38, 1e-38, 1e-44, 2.5, 1.984375, 1.9843751]
    for t in tops:  # one block each
        x = np.zeros((16, 1, 64), dtype=np.float32)
        x[:, 0] = np.float32(t) * np.linspace(-1, 1, 64, dtype=np.float32)
        x[3, 0, 0] = t
        r.add([16], "float32", k=x, v=np.ascontiguousarray(x[::-1]))
    r.check_values()


@pytest.mark.gpu
def test_append_infinity_and_nan_poison_their_block_alone(hiplib):
    r = Rig(2, 120, 2, 64, np.random.default_rng(6))
    k = to_type(r.rng.standard_normal((100, 2, 64)), "float32")
    v = k.copy()
    k[20, 1, 3], v[50, 0, 7] = np.inf, np.nan
    r.add([60, 40], "float32", k=k, v=v)
    r.check_values()
    r.add([9, 1], "float32")  # into the blocks behind, and beside
    r.check_values()
    # a row that sees the block is NaN in its heads; one whose mask leaves the block out is not
    q = to_type(r.rng.standard_normal((2, 2, 64)), "float32")
    out = paged.attend(r.pool, r.batch([1, 1]), dev(q)).numpy()
    assert np.isnan(out[0]).all() and np.isfinite(out[1]).all()  # sequence 0: head 1 by K, head 0 by V
    out = paged.attend(r.pool, r.batch([1, 1]), dev(q), window=5).numpy()
    assert np.isfinite(out).all()
    # rows of one tile on both sides of the mask: the last 16 tokens see block 1 (tokens 16 .. 31) or not
    q = to_type(r.rng.standard_normal((31, 2, 64)), "float32")
    out = paged.attend(r.pool, r.batch([30, 1]), dev(q), window=32).numpy()
    p = r.lens[0] - 30 + np.arange(30)
    sees = p - 32 < 31
    assert np.isnan(out[:30][sees, 1]).all() and np.isfinite(out[:30][~sees, 1]).all() and sees.any() and (~sees).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_read_any_range(hiplib, dtype):
    r = Rig(3, 150, 2, 96, np.random.default_rng(7))
    r.add([150, 3, 77], dtype)
    start = [-7, 1, 60]
    k, v = r.read(start, 41, dtype)
    for s in range(3):
        want_k, want_v = r.k.values(s), r.v.values(s)
        for i in range(41):
            p = start[s] + i
            inside = 0 <= p < r.lens[s]
            for got, want in ((k, want_k), (v, want_v)):
                # a code has 7 bits beside its sign, so the value is a number of every type unless fp16 runs out of range (not here)
                np.testing.assert_array_equal(from_type(got[s, i], dtype), want[p] if inside else np.zeros((2, 96)))


# ---- attention ------------------------------------------------------------------------------------------------------------------------


def check_attend(r, rows, q_heads, dtype, window=0, sinks=0, scale=None, max_rows=None, spare=2):
    total = sum(rows)
    q = to_type(r.rng.standard_normal((total + spare, q_heads, r.dim)) * 1.5, dtype)
    b = r.batch(rows, spare)
    if max_rows is not None:
        b = paged.KvBatch(b.table, b.lens, b.starts, rows=b.rows, max_rows=max_rows, max_len=b.max_len)
    mark = to_type(np.full((total + spare, q_heads, r.dim), 77.0), dtype)
    out = dev(mark, dtype)
    assert paged.attend(r.pool, b, dev(q, dtype), layer=r.layer, window=window, sinks=sinks, scale=scale, out=out) is out
    got = from_type(out.numpy(), dtype)
    assert (got[total:] == 77.0).all(), "rows behind the last sequence are left as they were"
    at, worst, sq, n_sq = 0, 0.0, 0.0, 0
    sc = r.dim ** -0.5 if scale is None else scale
    for s, n in enumerate(rows):
        k, v = r.k.values(s), r.v.values(s)
        x = from_type(q[at:at + n], dtype)
        if n:
            if len(k):  # what the bounds assume of the scores
                assert max((np.abs(x[:, h]) @ np.abs(k[:, h // (q_heads // r.heads)]).T).max() for h in range(q_heads)) * abs(sc) <= 32
            want = attention(x, k, v, sc, window, sinks)
            top = np.abs(v).max() if len(v) else 1.0
            err = np.abs(got[at:at + n] - want) / top
            worst = max(worst, err.max())
            sq, n_sq = sq + (err ** 2).sum(), n_sq + err.size
        at += n
    assert worst <= 2.0 ** -9 + U[dtype], worst
    if dtype == "float32" and n_sq:
        assert (sq / n_sq) ** 0.5 <= 2e-5, (sq / n_sq) ** 0.5
    r.pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", paged.HEAD_DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_one_token(hiplib, dim, dtype):
    """lengths from one token, around block and page borders, to several pages; groups of 1, 4 and 7 heads"""
    r = Rig(7, 420, 2, dim, np.random.default_rng(dim + 1), layers=2, layer=1)
    r.add([1, 15, 16, 63, 64, 65, 400], dtype)
    for group in (1, 4, 7):
        check_attend(r, [1] * 7, 2 * group, dtype)
    check_attend(r, [1, 0, 1, 0, 0, 1, 1], 2, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group,rows", [(64, 1, 17), (64, 8, 5), (128, 4, 3), (128, 4, 8), (96, 2, 16), (256, 3, 7), (128, 20, 1), (64, 33, 1), (128, 1, 33), (64, 4, 70),
                                            (96, 5, 40), (256, 2, 40), (128, 6, 61)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_several_rows(hiplib, dim, group, rows, dtype):
    """every kernel form (16 and 32 rows a tile, 128 rows a workgroup), ragged"""
    r = Rig(3, 230, 2, dim, np.random.default_rng(rows))
    r.add([rows, 200, 131], dtype)
    check_attend(r, [rows, max(rows - 3, 1), 1], 2 * group, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (64, 4), (65, 70), (100, 64), (100, 200), (1000, 3), (31, 16)])
@pytest.mark.parametrize("rows,group", [(1, 4), (6, 4), (50, 2)])
def test_attend_window_and_first_tokens(hiplib, window, sinks, rows, group):
    r = Rig(3, 330, 2, 64, np.random.default_rng(window + sinks))
    r.add([rows, 300, 191], "float16")
    check_attend(r, [rows] * 3, 2 * group, "float16", window, sinks)
    check_attend(r, [rows, 1, 0], 2 * group, "float32", window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(128, "float32"), (64, "bfloat16"), (256, "float16")])
@pytest.mark.parametrize("rows", [1, 5, 45])
def test_attend_long_context_is_cut_and_joined(hiplib, dim, dtype, rows):
    """a context whose pages are walked by many workgroups, beside short ones that are not; also under a window"""
    r = Rig(3, 4100, 1, dim, np.random.default_rng(11))
    r.add([4090, 70, rows], dtype)
    check_attend(r, [rows, rows, rows], 2, dtype)
    check_attend(r, [rows, rows, rows], 2, dtype, window=2000, sinks=5)


@pytest.mark.gpu
def test_attend_scales_of_blocks_far_apart(hiplib):
    """V blocks 2^20 apart: a row that sees only the small ones keeps their precision; the sum follows the large ones where they are seen"""
    r = Rig(1, 200, 1, 128, np.random.default_rng(12))
    for i in range(10):
        k = to_type(r.rng.standard_normal((16, 1, 128)), "float32")
        r.add([16], "float32", k=k, v=to_type(r.rng.standard_normal((16, 1, 128)) * (2.0 ** 20 if i < 2 else 1.0), "float32"))
    q = to_type(r.rng.standard_normal((1, 2, 128)), "float32")
    for window in (0, 100):
        got = paged.attend(r.pool, r.batch([1]), dev(q), window=window).numpy()
        want = attention(q.astype(np.float64), r.k.values(0), r.v.values(0), 128 ** -0.5, window, 0)
        assert np.abs(got - want).max() <= 1e-5 * np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_rows_that_see_nothing(hiplib, rows):
    """a sequence of length zero, and rows before position 0 (more rows than tokens): zeros"""
    r = Rig(2, 100, 2, 64, np.random.default_rng(13))
    r.add([0, 20], "float32")
    q = to_type(r.rng.standard_normal((rows + rows, 4, 64)), "float32")
    out = paged.attend(r.pool, r.batch([rows, rows]), dev(q)).numpy()
    assert not out[:rows].any()
    if rows > 20:
        assert not out[rows:2 * rows - 20].any() and out[2 * rows - 20:].any(axis=(1, 2)).all()


@pytest.mark.gpu
def test_attend_extreme_queries(hiplib):
    """rows of zeros, tiny and huge rows, and large scores: a row's power of two keeps them inside binary16"""
    r = Rig(1, 100, 1, 64, np.random.default_rng(14))
    r.add([90], "float32")
    q = np.stack([np.zeros((1, 64)), r.rng.standard_normal((1, 64)) * 1e-30, r.rng.standard_normal((1, 64)) * 1e4, r.rng.standard_normal((1, 64)) * 1e6]).astype(np.float32)
    got = paged.attend(r.pool, r.batch([4]), dev(q)).numpy()
    want = attention(q.astype(np.float64), r.k.values(0), r.v.values(0), 0.125, 0, 0)
    # the two large rows pick one token each: their scores are 1e3 apart, far beyond their error
    np.testing.assert_allclose(got, want, rtol=0, atol=2e-5 * np.abs(want).max())
    bad = np.array(q)
    bad[1, 0, 5] = np.nan
    got = paged.attend(r.pool, r.batch([4]), dev(bad)).numpy()
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2, 3]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_missing_pages(hiplib, rows):
    """-1 for a page that no row sees is fine; for one that rows see, or a number outside the pool, those rows are NaN and the pool says so"""
    r = Rig(2, 300, 1, 64, np.random.default_rng(15))
    r.add([290, 290], "float16")
    t = r.table.copy()
    t[0, 1:3] = -1
    r.dtable = dev(t)
    check_attend(r, [rows, rows], 2, "float16", window=50, sinks=3)
    t[0, 0] = r.pages
    r.dtable = dev(t)
    q = to_type(r.rng.standard_normal((2 * rows, 2, 64)), "float16")
    out = paged.attend(r.pool, r.batch([rows, rows]), dev(q), window=50, sinks=3).numpy()
    assert np.isnan(out[:rows]).all() and np.isfinite(out[rows:]).all()
    with pytest.raises(RuntimeError, match="outside the pool"):
        r.pool.check()
    r.pool.check()


@pytest.mark.gpu
def test_batches_that_lie_are_reported(hiplib):
    r = Rig(2, 100, 1, 64, np.random.default_rng(16))
    r.add([60, 60], "float32")
    q = dev(to_type(r.rng.standard_normal((50, 2, 64)), "float32"))
    b = r.batch([40, 10])
    b = paged.KvBatch(b.table, b.lens, b.starts, rows=50, max_rows=2, max_len=60)
    paged.attend(r.pool, b, q)
    with pytest.raises(RuntimeError, match="max_rows"):
        r.pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 50])
def test_bounds_that_are_too_small_only_shape_the_launch(hiplib, rows):
    """a max_len far below the longest sequence: it is attended in full, cut or not"""
    r = Rig(2, 3000, 2, 64, np.random.default_rng(18))
    r.add([2990, 700], "float32")
    q = dev(to_type(r.rng.standard_normal((2 * rows, 4, 64)), "float32"))
    b = r.batch([rows, rows])
    want = paged.attend(r.pool, b, q).numpy()
    for most in (1, 500, 1100):
        got = paged.attend(r.pool, paged.KvBatch(b.table, b.lens, b.starts, rows=2 * rows, max_rows=rows, max_len=most), q).numpy()
        np.testing.assert_allclose(got, want, rtol=0, atol=1e-5)
    r.pool.check()


@pytest.mark.gpu
def test_rows_outside_the_sequences_are_left_alone(hiplib):
    """starts that begin behind row 0 and end before the last; starts that do not add up are reported"""
    r = Rig(2, 2100, 1, 64, np.random.default_rng(19))
    r.add([2050, 300], "float32")
    q = dev(to_type(r.rng.standard_normal((8, 2, 64)), "float32"))
    want = paged.attend(r.pool, r.batch([2, 3]), View(q, 2 * 128, (5, 2, 64))).numpy()
    out = dev(np.full((8, 2, 64), 5.0, dtype=np.float32))
    paged.attend(r.pool, paged.KvBatch(r.dtable, ints(r.lens), ints([2, 4, 7]), rows=8, max_rows=3, max_len=2100), q, out=out)
    got = out.numpy()
    np.testing.assert_array_equal(got[2:7], want)
    assert (got[:2] == 5).all() and (got[7:] == 5).all()
    r.pool.check()
    for starts in ([0, 9, 9], [0, 5, 3], [-1, 2, 4]):
        paged.attend(r.pool, paged.KvBatch(r.dtable, ints(r.lens), ints(starts), rows=8, max_rows=8, max_len=2100), q)
        with pytest.raises(RuntimeError, match="max_rows"):
            r.pool.check()
        x = dev(np.zeros((8, 1, 64), dtype=np.float32))
        paged.append(r.pool, paged.KvBatch(r.dtable, ints([0, 0]), ints(starts), rows=8, max_rows=8, max_len=2100), x, x)
        with pytest.raises(RuntimeError, match="max_rows"):
            r.pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [12, 60])
def test_a_missing_page_spares_the_rows_that_do_not_see_it(hiplib, rows):
    """rows of one tile on both sides of a window's end inside a missing page, with infinities where its stand-in's scales would be"""
    r = Rig(1, 400, 1, 64, np.random.default_rng(20))
    r.add([400], "float32")
    t = r.table.copy()
    spare = [p for p in range(r.pages) if p not in set(t[0])]
    if 0 not in spare:  # page 0 out of use
        t[0, list(t[0]).index(0)] = spare[0]
        r.table = t
        r.dtable = dev(t)
        r.k, r.v, r.lens = Cache(1, 64), Cache(1, 64), [0]
        r.add([400], "float32")
    for x in (r.pool.k_scale, r.pool.v_scale):
        one = np.full(4, np.inf, dtype=np.float32)
        x._lib.copy_hip(x.data_ptr(), one.ctypes.data, 16)
    t = r.table.copy()
    t[0, 3] = -1  # tokens 192 .. 255
    window = 400 - 255 - rows // 2  # the later half of the rows does not see them
    q = to_type(r.rng.standard_normal((rows, 2, 64)), "float32")
    b = r.batch([rows])
    got = paged.attend(r.pool, paged.KvBatch(dev(t), b.lens, b.starts, rows=rows, max_rows=rows, max_len=400), dev(q), window=window).numpy()
    want = attention(q.astype(np.float64), r.k.values(0), r.v.values(0), 0.125, window, 0)
    p = 400 - rows + np.arange(rows)
    sees = p - window < 255
    assert sees.any() and (~sees).any() and np.isnan(got[sees]).all()
    np.testing.assert_allclose(got[~sees], want[~sees], rtol=0, atol=2e-5 * np.abs(want).max())


@pytest.mark.gpu
def test_attend_is_the_same_twice(hiplib):
    r = Rig(2, 2000, 2, 128, np.random.default_rng(17))
    r.add([2000, 1500], "bfloat16")
    q = dev(to_type(r.rng.standard_normal((2, 8, 128)), "bfloat16"), "bfloat16")
    a, b = (paged.attend(r.pool, r.batch([1, 1]), q).numpy() for _ in range(2))
    np.testing.assert_array_equal(a, b)


# ---- pages ----------------------------------------------------------------------------------------------------------------------------


class Book:
    """the plain bookkeeping"""

    def __init__(self, pages, rows, mp):
        self.refs = [0] * pages
        self.table = [[-1] * mp for _ in range(rows)]

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, lens, new):
        for row, a, b in zip(self.table, lens, new):
            for c in range(a // 64, -(-b // 64) if b > a else a // 64):
                if row[c] < 0:
                    row[c] = self.take()

    def trim(self, lens, window=0, sinks=0):
        for row, n in zip(self.table, lens):
            for c in range(len(row)):
                dead = 64 * c >= n or (window > 0 and 64 * c + 63 <= n - window and 64 * c >= sinks)
                if dead and row[c] >= 0:
                    self.refs[row[c]] -= 1
                    row[c] = -1

    def fork(self, lens, parents):
        """-> copies (from, to)"""
        old, copies = [list(r) for r in self.table], []
        first = {}
        for i, p in enumerate(parents):
            first.setdefault(p, i)
        want = []
        self.refs = [0] * len(self.refs)
        for i, p in enumerate(parents):
            full = lens[p] // 64
            row = list(old[p]) if first[p] == i else [x if c < full else -1 for c, x in enumerate(old[p])]
            if first[p] != i and lens[p] % 64 and old[p][full] >= 0:
                want.append((i, full, old[p][full]))
            self.table[i] = row
            for x in row:
                if x >= 0:
                    self.refs[x] += 1
        for i, c, src in want:
            self.table[i][c] = self.take()
            copies.append((src, self.table[i][c]))
        return copies

    def same(self, table, refs):
        np.testing.assert_array_equal(table, np.array(self.table))
        np.testing.assert_array_equal(refs, np.array(self.refs))


def pool_bytes(pool):
    return [x.numpy() for x in (pool.k, pool.v, pool.k_scale, pool.v_scale)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,pages", [(6, 90), (40, 400), (1, 12)])
def test_pages_reserve_fork_trim(hiplib, rows, pages):
    """rounds of growing, reordering, trimming: table, counts and every byte of the pool follow the plain bookkeeping"""
    rng = np.random.default_rng(rows)
    mp = 8
    pool = paged.KvPool(2, pages, 3, 64)
    for x in (pool.k, pool.v):
        junk = rng.integers(-128, 128, x.shape).astype(np.int8)
        x._lib.copy_hip(x.data_ptr(), junk.ctypes.data, junk.nbytes)
    for x in (pool.k_scale, pool.v_scale):
        junk = rng.standard_normal(x.shape).astype(np.float32)
        x._lib.copy_hip(x.data_ptr(), junk.ctypes.data, junk.nbytes)
    want = pool_bytes(pool)
    book = Book(pages, rows, mp)
    table, refs = dev(np.array(book.table, dtype=np.int32)), dev(np.array(book.refs, dtype=np.int32))
    lens = [0] * rows
    for step in range(9):
        new = [min(n + int(x), 64 * mp) for n, x in zip(lens, rng.integers(0, [30, 70, 1, 90][step % 4] + 1, rows))]
        if sum(max(-(-m // 64), 1) for m in new) + rows > pages:
            new = lens
        paged.reserve(pool, table, refs, ints(lens), ints(new))
        book.reserve(lens, new)
        book.same(table.numpy(), refs.numpy())
        lens = new
        parents = np.sort(rng.integers(0, rows, rows)) if step % 2 else rng.permutation(rng.integers(0, rows, rows))
        table, refs = paged.fork(pool, table, ints(lens), refs, ints(parents))
        for src, to in book.fork(lens, [int(p) for p in parents]):
            for x in want:
                x[:, to] = x[:, src]
        book.same(table.numpy(), refs.numpy())
        for a, b in zip(pool_bytes(pool), want):
            np.testing.assert_array_equal(a, b)
        lens = [lens[p] for p in parents]
        if step % 3 == 2:  # some rows end, others keep a window
            lens = [0 if rng.random() < 0.3 else n for n in lens]
            paged.trim(pool, table, refs, ints(lens), window=70, sinks=2)
            book.trim(lens, 70, 2)
            book.same(table.numpy(), refs.numpy())
        pool.check()
    paged.trim(pool, table, refs, ints([0] * rows))
    assert not refs.numpy().any() and (table.numpy() == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [24576, 24577])
def test_fork_in_a_large_pool(hiplib, pages):
    """counts in LDS, and one page too many for that; most pages are in other hands, the free ones lie at the end"""
    rng = np.random.default_rng(pages)
    rows, mp = 30, 7
    pool = paged.KvPool(1, pages, 1, 64)
    book = Book(pages, rows, mp)
    book.refs = [1] * (pages - 600) + [0] * 600
    lens = [int(n) for n in rng.integers(0, 64 * mp + 1, rows)]
    book.reserve([0] * rows, lens)
    codes = rng.integers(-128, 128, (pages, 4096)).astype(np.int8)
    pool.k._lib.copy_hip(pool.k.data_ptr(), codes.ctypes.data, codes.nbytes)
    table, refs = dev(np.array(book.table, dtype=np.int32)), dev(np.array(book.refs, dtype=np.int32))
    held = np.array(book.refs)
    parents = [int(p) for p in rng.integers(0, rows, rows)]
    table, refs = paged.fork(pool, table, ints(lens), refs, ints(parents))
    for n in range(pages - 600):  # (the plain bookkeeping counts the table's rows alone)
        held[n] = 1
    held[pages - 600:] = 0
    before = [list(r) for r in book.table]
    first, want = {}, []
    for i, p in enumerate(parents):
        first.setdefault(p, i)
    for i, p in enumerate(parents):
        full = lens[p] // 64
        book.table[i] = [x if first[p] == i or c < full else -1 for c, x in enumerate(before[p])]
        if first[p] != i and lens[p] % 64:
            want.append((i, full, before[p][full]))
        for x in book.table[i]:
            if x >= 0:
                held[x] += 1
    for i, c, src in want:
        to = int(np.argmin(held))
        held[to] = 1
        book.table[i][c] = to
        codes[to] = codes[src]
    np.testing.assert_array_equal(table.numpy(), np.array(book.table))
    np.testing.assert_array_equal(refs.numpy(), held)
    np.testing.assert_array_equal(pool.k.numpy().reshape(pages, 4096), codes)
    pool.check()


@pytest.mark.gpu
def test_pages_run_out(hiplib):
    """no free page: the entries stay -1, the pool says so, nothing else changes"""
    pool = paged.KvPool(1, 3, 1, 64)
    table, refs = dev(np.full((2, 4), -1, dtype=np.int32)), dev(np.zeros(3, dtype=np.int32))
    paged.reserve(pool, table, refs, ints([0, 0]), ints([130, 65]))
    np.testing.assert_array_equal(table.numpy(), [[0, 1, 2, -1], [-1, -1, -1, -1]])
    with pytest.raises(RuntimeError, match="no page was free"):
        pool.check()
    t, r = paged.fork(pool, table, ints([130, 0]), refs, ints([0, 0]))
    np.testing.assert_array_equal(t.numpy(), [[0, 1, 2, -1], [0, 1, -1, -1]])
    np.testing.assert_array_equal(r.numpy(), [2, 2, 1])
    with pytest.raises(RuntimeError, match="no page was free"):
        pool.check()
    t, r = paged.fork(pool, table, ints([130, 0]), refs, ints([0, 5]))
    np.testing.assert_array_equal(t.numpy(), [[0, 1, 2, -1], [-1, -1, -1, -1]])
    with pytest.raises(RuntimeError, match="a parent"):
        pool.check()


@pytest.mark.gpu
@pytest.mark.parametrize("pages,live", [(1, 1), (2, 1), (7, 0), (7, 7), (64, 20), (2100, 1300), (12288, 9001), (12289, 9001)])
def test_compact(hiplib, pages, live):
    rng = np.random.default_rng(pages)
    heads = 1 if pages > 100 else 3
    pool = paged.KvPool(2, pages, heads, 64)
    want = []
    for x in (pool.k, pool.v, pool.k_scale, pool.v_scale):
        junk = rng.integers(-128, 128, x.shape).astype(np.int8) if x.dtype == "int8" else rng.standard_normal(x.shape).astype(np.float32)
        x._lib.copy_hip(x.data_ptr(), junk.ctypes.data, junk.nbytes)
        want.append(junk)
    kept = rng.permutation(pages)[:live]
    refs = np.zeros(pages, dtype=np.int32)
    refs[kept] = rng.integers(1, 4, live)
    table = np.full((2, max(live, 1) + 1), -1, dtype=np.int32)
    table[0, :live] = kept
    table[1, 1:1 + live // 2] = kept[:live // 2]
    t, r, n = paged.compact(pool, dev(table), dev(refs))
    assert n.numpy()[0] == live
    to = np.arange(pages)
    to[[p for p in range(live, pages) if refs[p]]] = [p for p in range(live) if not refs[p]]
    np.testing.assert_array_equal(t.numpy(), np.where(table >= 0, to[np.maximum(table, 0)], -1))
    now = np.zeros(pages, dtype=np.int32)
    now[to[kept]] = refs[kept]
    np.testing.assert_array_equal(r.numpy(), now)
    for got, was in zip(pool_bytes(pool), want):
        np.testing.assert_array_equal(got[:, to[kept]], was[:, kept])
    pool.check()


# ---- selection ------------------------------------------------------------------------------------------------------------------------


def select(logits, scores, done, eos):
    """the definition: logits [groups * beams, vocab] float64"""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    out = []
    for g in range(groups):
        total = np.full((beams, vocab), -np.inf)
        for w in range(beams):
            x, s = logits[g * beams + w], float(scores[g, w])
            if eos >= 0 and done[g, w]:
                total[w, eos] = s
                continue
            if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf or s == -np.inf:
                continue
            total[w] = s + (x - (x.max() + np.log(np.exp(x - x.max()).sum())))
        order = np.argsort(-total.ravel(), kind="stable")[:beams]
        p, t = order // vocab, order % vocab
        d = [int(eos >= 0 and (done[g, a] or b == eos)) for a, b in zip(p, t)]
        out.append((total.ravel()[order], p, t, d))
    return [np.stack(x) for x in zip(*out)]


def check_select(logits, scores, done, eos, dtype="float32", strided=None):
    stored = to_type(logits, dtype)
    arr = dev(stored, dtype)
    if strided:
        wide = np.zeros((stored.shape[0], stored.shape[1] + strided), dtype=stored.dtype)
        wide[:, :stored.shape[1]] = stored
        base = dev(wide, dtype)
        arr = View(base, 0, stored.shape)
    got = paged.beam_select(arr, dev(scores.astype(np.float32)), None if done is None else dev(done.astype(np.uint8)), eos=eos)
    want = select(from_type(stored, dtype), scores.astype(np.float32), np.zeros_like(scores) if done is None else done, eos)
    for i, name in ((1, "parents"), (2, "tokens"), (3, "done")):
        np.testing.assert_array_equal(got[i].numpy(), want[i], err_msg=name)
    # the sum is 64 bits wide with 32-bit exponentials (2^-22 each, about), the score is rounded once to fp32
    g = got[0].numpy().astype(np.float64)
    fin = np.isfinite(want[0])
    np.testing.assert_array_equal(np.isneginf(g), ~fin)
    assert (np.abs(g[fin] - want[0][fin]) <= 2.0 ** -22 + np.abs(want[0][fin]) * 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (2, 3, 2), (1, 4, 320), (3, 8, 8191), (2, 5, 8192), (1, 32, 8185), (2, 16, 20011), (1, 2, 128256)])
def test_select(hiplib, groups, beams, vocab, dtype):
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((groups * beams, vocab)) * 2.5
    scores = -5 * rng.random((groups, beams))
    check_select(logits, scores, None, -1, dtype)
    done = rng.random((groups, beams)) < 0.4
    check_select(logits, scores, done, vocab // 2, dtype, strided=3)
    check_select(logits, np.where(np.arange(beams) == 0, 0.0, -np.inf) + np.zeros((groups, 1)), None, 0, dtype, strided=1)


@pytest.mark.gpu
def test_select_ties_go_to_the_lowest_index(hiplib):
    x = np.zeros((4, 50))
    check_select(x, np.zeros((1, 4)), None, -1)
    x = np.tile(np.repeat([3.0, 5.0, 5.0, 1.0], 10000), (6, 1))  # equal values across chunks, equal beams
    check_select(x, np.zeros((2, 3)), None, -1)
    x[1] = 0
    x[:, 7] = -0.0
    check_select(x, np.zeros((2, 3)), None, -1)


@pytest.mark.gpu
def test_select_infinities_and_nan(hiplib):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 9000))
    x[0] = -np.inf          # no finite logit
    x[1, 100] = np.nan
    x[2, 8999] = np.inf
    x[3, 5:] = -np.inf      # five tokens allowed
    x[4, :8998] = -np.inf
    scores = np.array([[0, 0, 0, -1.0], [-2.0, -np.inf, -3.0, -1.0]])
    check_select(x, scores, None, -1)
    check_select(x, scores, np.array([[1, 0, 0, 0], [0, 1, 0, 1]]), 8999)
    check_select(np.full((4, 6), -np.inf), np.zeros((1, 4)), None, 2)
    check_select(rng.standard_normal((3, 2)), np.zeros((1, 3)), np.ones((1, 3)), 1)


# ---- a search, with all of them -------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_a_search_with_all_operators(hiplib):
    """Two prompts, four beams each, a window: reserve, append, attend, select, fork, trim, compact -- the steps of a decoder with one attention layer
    whose 'model' is random matrices -- against the plain cache and mask, step by step on the same selections."""
    rng = np.random.default_rng(21)
    groups, beams, heads, q_heads, dim, vocab, window, sinks = 2, 4, 2, 4, 64, 500, 90, 4
    rows, mp, pages = groups * beams, 6, 60
    pool = paged.KvPool(1, pages, heads, dim)
    table, refs = dev(np.full((rows, mp), -1, dtype=np.int32)), dev(np.zeros(pages, dtype=np.int32))
    prompts = [130, 61]
    mk, mv, mq, mo = (rng.standard_normal(s).astype(np.float32) for s in ((vocab, heads, dim), (vocab, heads, dim), (vocab, q_heads, dim), (q_heads * dim, vocab)))
    words = [rng.integers(0, vocab, n) for n in prompts]
    # the prompt goes into every group's first beam, and forks from there
    lens = [0] * rows
    new = [prompts[i // beams] if i % beams == 0 else 0 for i in range(rows)]
    paged.reserve(pool, table, refs, ints(lens), ints(new))
    starts = np.concatenate([[0], np.cumsum(new)])
    tok = np.concatenate(words)
    lens = new
    paged.append(pool, paged.KvBatch(table, ints(lens), ints(starts), rows=len(tok), max_rows=max(new), max_len=max(new)), dev(mk[tok]), dev(mv[tok]))
    parents = [i // beams * beams for i in range(rows)]
    table, refs = paged.fork(pool, table, ints(lens), refs, ints(parents))
    lens = [lens[p] for p in parents]
    cache_k, cache_v = {}, {}
    for i in range(rows):
        cache_k[i], cache_v[i] = Cache(heads, dim), Cache(heads, dim)
        w = words[i // beams]
        cache_k[i].append(0, mk[w].astype(np.float64)), cache_v[i].append(0, mv[w].astype(np.float64))
    scores = np.where(np.arange(beams) == 0, 0.0, -np.inf) + np.zeros((groups, 1))
    scores, done = dev(scores.astype(np.float32)), dev(np.zeros((groups, beams), dtype=np.uint8))
    tok = np.array([w[-1] for w in words for _ in range(beams)])
    import copy

    for step in range(12):
        new = [n + 1 for n in lens]
        paged.reserve(pool, table, refs, ints(lens), ints(new))
        lens = new
        b = paged.KvBatch(table, ints(lens), ints(np.arange(rows + 1)), rows=rows, max_rows=1, max_len=max(lens))
        paged.append(pool, b, dev(mk[tok]), dev(mv[tok]))
        att = paged.attend(pool, b, dev(mq[tok]), window=window, sinks=sinks).numpy()
        for i in range(rows):
            cache_k[i].append(0, mk[tok[i]][None].astype(np.float64)), cache_v[i].append(0, mv[tok[i]][None].astype(np.float64))
            want = attention(mq[tok[i]][None].astype(np.float64), cache_k[i].values(0), cache_v[i].values(0), dim ** -0.5, window, sinks)
            np.testing.assert_allclose(att[i], want[0], rtol=0, atol=2e-5 * np.abs(cache_v[i].values(0)).max())
        logits = (att.reshape(rows, -1) @ mo * 0.1).astype(np.float32)
        was = scores.numpy()
        scores, par, t, done_new = paged.beam_select(dev(logits), scores, done, eos=3)
        want = select(logits.astype(np.float64), was, done.numpy(), 3)
        np.testing.assert_array_equal(par.numpy(), want[1])
        np.testing.assert_array_equal(t.numpy(), want[2])
        done = done_new
        parents = (par.numpy() + np.arange(groups)[:, None] * beams).ravel()
        table, refs = paged.fork(pool, table, ints(lens), refs, ints(parents))
        lens = [lens[p] for p in parents]
        cache_k, cache_v = ({i: copy.deepcopy(c[p]) for i, p in enumerate(parents)} for c in (cache_k, cache_v))
        tok = t.numpy().ravel()
        paged.trim(pool, table, refs, ints(lens), window=window, sinks=sinks)
        if step % 4 == 3:
            table, refs, live = paged.compact(pool, table, refs)
            assert not refs.numpy()[live.numpy()[0]:].any()
    pool.check()


# ---- refusals (no GPU) ----------------------------------------------------------------------------------------------------------------


class Fake:
    """an array's outside, with no memory behind it: a call that gets past its checks would have nothing to launch on"""

    def __init__(self, shape, dtype, stride=None, ptr=4096, dense=True, device="cuda:0"):
        self.device = device
        self.shape, self.dtype, self._ptr, self._dense = shape, dtype, ptr, dense
        s, out = 1, []
        for n in reversed(shape):
            out.append(s)
            s *= n
        self._stride = stride or tuple(reversed(out))

    def data_ptr(self):
        return self._ptr

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._dense


def c_pool(**kw):
    f = dict(k=4096, v=8192, k_scale=4096, v_scale=4096, status=4096, n_layers=2, n_pages=10, n_kv_heads=2, head_dim=64)
    f.update(kw)
    return paged._Pool(*[f[n] for n, _ in paged._Pool._fields_])


def c_batch(**kw):
    f = dict(table=4096, lens=4096, starts=4096, n_seqs=2, max_pages=4, n_rows=2, max_rows=1, max_len=100)
    f.update(kw)
    return paged._Batch(*[f[n] for n, _ in paged._Batch._fields_])


def refused(rc, lib, words):
    assert rc == -1
    assert words in lib.calm_hip_error().decode(), lib.calm_hip_error()


def test_entries_refuse_bad_pools_and_batches(hiplib):
    b = c_batch()
    for kw, words in [(dict(k=0), "missing"), (dict(status=0), "missing"), (dict(head_dim=80), "head sizes"), (dict(n_pages=0), "no layers"), (dict(n_kv_heads=2000), "1024 heads"),
                      (dict(k=4100), "16-byte")]:
        p = c_pool(**kw)
        refused(hiplib.kv_append_hip(C.byref(p), C.byref(b), 0, 4096, 4096, 0, 128, 64, 128, 64, None), hiplib, words)
        refused(hiplib.kv_attend_hip(C.byref(p), C.byref(b), 0, 4096, 4096, 0, 4, 256, 64, 0.1, 0, 0, None, 0, None), hiplib, words)
        refused(hiplib.kv_read_hip(C.byref(p), 0, 4096, 4096, 4096, 2, 4, 5, 4096, 4096, 0, None), hiplib, words)
        refused(hiplib.kv_fork_hip(C.byref(p), 4096, 4096, 4096, 4096, 2, 4, 8192, 8192, 4096, 64, None), hiplib, words)
        refused(hiplib.kv_compact_hip(C.byref(p), 4096, 4096, 2, 4, 8192, 8192, 4096, 4096, 80, None), hiplib, words)
    refused(hiplib.kv_append_hip(None, C.byref(b), 0, 4096, 4096, 0, 128, 64, 128, 64, None), hiplib, "missing")
    p = c_pool()
    for kw, words in [(dict(table=0), "missing"), (dict(n_seqs=0), "65535 sequences"), (dict(n_seqs=70000), "65535"), (dict(max_pages=0), "page column"), (dict(n_rows=-1), "negative"),
                      (dict(n_seqs=60000, max_pages=60000), "2^30")]:
        bb = c_batch(**kw)
        refused(hiplib.kv_append_hip(C.byref(p), C.byref(bb), 0, 4096, 4096, 0, 128, 64, 128, 64, None), hiplib, words)
        refused(hiplib.kv_attend_workspace_hip(C.byref(p), C.byref(bb), 0, 4, 0, 0), hiplib, words)
    # no rows: nothing to do
    assert hiplib.kv_append_hip(C.byref(p), C.byref(c_batch(n_rows=0)), 0, None, None, 0, 0, 0, 0, 0, None) == 0


def test_entries_refuse_bad_arguments(hiplib):
    p, b = c_pool(), c_batch()
    P, B = C.byref(p), C.byref(b)
    app = lambda **k: hiplib.kv_append_hip(P, B, *[dict(dict(layer=0, k=4096, v=4096, t=0, kr=128, kh=64, vr=128, vh=64), **k)[n] for n in ("layer", "k", "v", "t", "kr", "kh", "vr", "vh")], None)  # noqa: E731
    for kw, words in [(dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(t=3), "types"), (dict(k=0), "missing"), (dict(k=4104), "multiples of four"), (dict(kr=126), "multiples of four"),
                      (dict(vh=62), "multiples of four")]:
        refused(app(**kw), hiplib, words)
    att = lambda **k: hiplib.kv_attend_hip(P, B, *[dict(dict(layer=0, q=4096, o=4096, t=0, nh=4, qr=256, qh=64, sc=0.1, w=0, s=0, ws=None, n=0), **k)[n]  # noqa: E731
                                                   for n in ("layer", "q", "o", "t", "nh", "qr", "qh", "sc", "w", "s", "ws", "n")], None)
    for kw, words in [(dict(layer=9), "layer"), (dict(t=-1), "types"), (dict(nh=3), "multiple"), (dict(nh=0), "multiple"), (dict(w=-1), "negative"), (dict(s=-2), "negative"),
                      (dict(sc=float("nan")), "finite"), (dict(sc=float("inf")), "finite"), (dict(q=0), "missing"), (dict(o=4100), "multiples of four"), (dict(qr=2), "multiples of four")]:
        refused(att(**kw), hiplib, words)
    long = c_batch(max_len=100000, n_seqs=1)
    need = hiplib.kv_attend_workspace_hip(P, C.byref(long), 0, 4, 0, 0)
    assert need > 0
    for ws, n in ((None, need), (4096, need - 1), (4104, need)):
        refused(hiplib.kv_attend_hip(P, C.byref(long), 0, 4096, 4096, 0, 4, 256, 64, 0.1, 0, 0, ws, n, None), hiplib, "workspace")
    # two rows of 4 heads of 64 fp32 values: 2048 bytes
    for kw in (dict(), dict(o=4096 + 2032), dict(o=4096 - 2032), dict(qr=512, o=4096 + 2048), dict(qr=-256, o=4096 - 2048)):
        refused(att(**kw), hiplib, "overlaps")
    refused(hiplib.kv_read_hip(P, 0, 4096, 4096, 4096, 2, 4, -1, 4096, 4096, 0, None), hiplib, "negative")
    refused(hiplib.kv_read_hip(P, 0, 4096, 0, 4096, 2, 4, 1, 4096, 4096, 0, None), hiplib, "missing")
    refused(hiplib.kv_read_hip(P, 0, 4096, 4096, 4096, 2, 4, 1, 4098, 4096, 1, None), hiplib, "aligned")
    refused(hiplib.kv_reserve_hip(P, 4096, 4096, 4096, None, 2, 4, None), hiplib, "missing")
    refused(hiplib.kv_reserve_hip(P, 4096, 4096, 4096, 4096, 5000, 4, None), hiplib, "2048 table rows")
    refused(hiplib.kv_trim_hip(P, 4096, 4096, 4096, 2, 4, -1, 0, None), hiplib, "negative")
    refused(hiplib.kv_fork_hip(P, 4096, 4096, 4096, 4096, 2, 4, 4096, 8192, 4096, 64, None), hiplib, "beside")
    refused(hiplib.kv_fork_hip(P, 4096, 4096, 4096, 4096, 2, 4, 8192, 8192, 4096, 15, None), hiplib, "workspace")
    refused(hiplib.kv_compact_hip(P, 4096, 4096, 2, 4, 8192, 4096, 4096, 4096, 80, None), hiplib, "beside")
    refused(hiplib.kv_compact_hip(P, 4096, 4096, 2, 4, 8192, 8192, 4096, 4096, 79, None), hiplib, "workspace")


def test_select_refuses(hiplib):
    need = hiplib.beam_workspace_hip(2, 4, 1000)
    assert need > 0
    for args in ((0, 4, 1000), (2, 0, 1000), (2, 33, 1000), (2, 4, 0), (20000, 4, 10)):
        refused(hiplib.beam_workspace_hip(*args), hiplib, "beams")
    call = lambda **k: hiplib.beam_select_hip(*[dict(dict(l=4096, t=0, row=1000, g=2, b=4, v=1000, s=4096, d=None, e=2, so=8192, p=8192, tk=8192, do=8192, w=4096, n=need), **k)[x]  # noqa: E731
                                                for x in ("l", "t", "row", "g", "b", "v", "s", "d", "e", "so", "p", "tk", "do", "w", "n")], None)
    for kw, words in [(dict(b=33), "beams"), (dict(t=5), "types"), (dict(l=0), "missing"), (dict(do=0), "missing"), (dict(l=4098), "aligned"), (dict(row=999), "overlap"), (dict(e=1000), "vocabulary"),
                      (dict(w=None), "workspace"), (dict(n=need - 1), "workspace"), (dict(so=4096), "beside"), (dict(d=8192), "beside")]:
        refused(call(**kw), hiplib, words)


def test_python_checks():
    k, v, s = Fake((2, 10, 2, 64, 64), "int8"), Fake((2, 10, 2, 4, 64, 16), "int8"), Fake((2, 10, 2, 4), "float32")
    with pytest.raises(ValueError, match="head size"):
        paged.KvPool(1, 1, 1, 80)
    with pytest.raises(ValueError, match="without"):
        paged.KvPool(0, 1, 1, 64)
    for bad in (dict(k=Fake((2, 10, 2, 32, 64), "int8")), dict(k=Fake((2, 10, 2, 64, 64), "uint8")), dict(v=Fake((2, 10, 2, 64, 64), "int8")), dict(s=Fake((2, 10, 2, 8), "float32")),
                dict(v=Fake((2, 10, 2, 4, 64, 16), "int8", dense=False))):
        a = dict(dict(k=k, v=v, s=s), **bad)
        with pytest.raises(ValueError):
            paged.KvPool.over(a["k"], a["v"], a["s"], a["s"])
    t, n, st = Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32")
    with pytest.raises(ValueError, match="int32"):
        paged.KvBatch(Fake((2, 4), "int64"), n, st, 2, 1, 10)
    with pytest.raises(ValueError, match="shape"):
        paged.KvBatch(t, Fake((3,), "int32"), st, 2, 1, 10)
    with pytest.raises(ValueError, match="shape"):
        paged.KvBatch(t, n, n, 2, 1, 10)
    with pytest.raises(ValueError, match="max_rows"):
        paged.KvBatch(t, n, st, 2, 3, 10)
    with pytest.raises(ValueError, match="contiguous"):
        paged.KvBatch(Fake((2, 4), "int32", dense=False), n, st, 2, 1, 10)
    far = Fake((2,), "int32", device="cuda:1")
    with pytest.raises(ValueError, match="cuda:1"):
        paged.KvBatch(t, far, st, 2, 1, 10)
    with pytest.raises(ValueError, match="cuda:1"):
        paged.KvPool.over(k, v, s, Fake((2, 10, 2, 4), "float32", device="cuda:1"))
    with pytest.raises(ValueError, match="at most"):
        paged.KvBatch(t, n, st, 2, 1, 1 << 32)
    pool = paged.KvPool.__new__(paged.KvPool)
    pool.n_layers, pool.n_pages, pool.n_kv_heads, pool.head_dim = 2, 10, 2, 64
    b = paged.KvBatch(t, n, st, 2, 1, 10)
    row = Fake((2, 2, 64), "float16")
    for bad in (Fake((1, 2, 64), "float16"), Fake((2, 3, 64), "float16"), Fake((2, 2, 32), "float16"), Fake((2, 2, 64), "int8"), Fake((2, 2, 64), "float16", stride=(256, 128, 2)),
                Fake((2, 2, 64), "float16", stride=(130, 64, 1)), Fake((2, 2, 64), "float32")):
        with pytest.raises(ValueError):
            paged.append(pool, b, row, bad)
    for kw in (dict(window=1 << 32), dict(sinks=1 << 31), dict(window=-1), dict(layer=2), dict(layer=(1 << 32) + 1), dict(layer=-1)):
        with pytest.raises(ValueError, match="window|layer"):
            paged.attend(pool, b, row, **kw)
    with pytest.raises(ValueError, match="layer"):
        paged.append(pool, b, row, row, layer=1 << 32)
    with pytest.raises(ValueError, match="tokens"):
        paged.read(pool, t, n, n, 1 << 32)
    with pytest.raises(ValueError, match="out"):
        paged.attend(pool, b, row, out=Fake((2, 2, 64), "float32"))
    with pytest.raises(ValueError, match="beams"):
        paged.beam_select(Fake((66, 10), "float32"), Fake((2, 33), "float32"))
    with pytest.raises(ValueError, match="logits"):
        paged.beam_select(Fake((7, 10), "float32"), Fake((2, 4), "float32"))
    with pytest.raises(ValueError, match="done"):
        paged.beam_select(Fake((8, 10), "float32"), Fake((2, 4), "float32"), Fake((2, 4), "int32"), eos=1)


def test_parameters_and_structs_match_the_header(tmp_path):
    """the ctypes mirrors of struct KvPool / KvBatch have the header's layout"""
    src = tmp_path / "o.c"
    fields = [("KvPool", paged._Pool), ("KvBatch", paged._Batch)]
    lines = [f'printf("%zu\\n", offsetof(struct {n}, {f}));' for n, c in fields for f, _ in c._fields_] + [f'printf("%zu\\n", sizeof(struct {n}));' for n, _ in fields]
    src.write_text(f'#include <stdio.h>\n#include "{os.path.join(ROOT, "include", "calm_hip.h")}"\nint main(void) {{ {" ".join(lines)} return 0; }}')
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "o")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "o")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(c, f).offset for _, c in fields for f, _ in c._fields_] + [C.sizeof(c) for _, c in fields]
