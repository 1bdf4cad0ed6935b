"""A paged 8-bit cache for several sequences, attention over it, and the selection of a beam search (include/calm_hip.h, libcalm_hip.so).

    pool  = KvPool(n_layers, n_pages, n_kv_heads, head_dim)       pages of 64 tokens: int8 codes, a power-of-two scale per 16 tokens and head
    batch = KvBatch(table, lens, starts, rows=.., max_rows=.., max_len=..)   which rows of a call belong to which sequence
    reserve / append / attend / read                             pages for new tokens, their K and V in, attention, values back
    fork / trim / compact                                        rows continue others (shared full pages), give pages up, move together
    beam_select                                                  the W best continuations of W hypotheses

Arrays are torch tensors on the GPU -- the calls run on torch's current stream of their device -- or `DeviceArray`s (memory of this
library, for programs without torch), which run on the backend's own stream, the one forward_hip is ordered on.  All arrays of a call are
of one kind and on one device.  Nothing here synchronises but `KvPool.check`, `DeviceArray.numpy` and the creation of DeviceArrays; with
tensors every call can be captured into a graph.  A call that cannot be right raises ValueError before anything is launched.  There is no
backward pass: tensors that require gradients are refused unless gradients are switched off, and tensors with forward-mode tangents always.

torch has to be imported before the library is loaded in a process that uses both (host.require_torch_first).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import sys
from typing import Optional

import numpy as np

from . import host

PAGE, BLOCK = 64, 16
HEAD_DIMS = (64, 96, 128, 256)
MAX_BEAMS = 32
_TYPES = {"float32": 0, "float16": 1, "bfloat16": 2}
_DTYPES = {}  # a name -> torch's dtype
_NAMES = {}  # a dtype object -> its name (str(torch.float16) costs a microsecond)
_SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int8": 1, "uint8": 1, "bool": 1}


class _Pool(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("status", C.c_void_p),
                ("n_layers", C.c_int), ("n_pages", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int)]


class _Batch(C.Structure):
    _fields_ = [("table", C.c_void_p), ("lens", C.c_void_p), ("starts", C.c_void_p), ("n_seqs", C.c_int), ("max_pages", C.c_int), ("n_rows", C.c_int),
                ("max_rows", C.c_int), ("max_len", C.c_int)]


class DeviceArray:
    """a dense array in device memory of this library; bfloat16 is held as uint16 on the host's side.  Its memory goes back when it is dropped: that waits
    for the device, so calls that still use it are through by then"""

    def __init__(self, shape, dtype="float32"):
        self.shape = tuple(int(n) for n in shape)
        self.dtype = str(dtype)
        self.nbytes = int(np.prod(self.shape, dtype=np.int64)) * _SIZES[self.dtype]
        self._lib = host.load_lib()
        self._ptr = self._lib.alloc_hip(max(self.nbytes, 16))

    @classmethod
    def of(cls, a: np.ndarray, dtype: Optional[str] = None) -> "DeviceArray":
        a = np.ascontiguousarray(a)
        d = cls(a.shape, dtype or str(a.dtype))
        if a.nbytes != d.nbytes:
            raise ValueError(f"{a.dtype} values for an array of {d.dtype}")
        if d.nbytes:
            d._lib.copy_hip(d._ptr, a.ctypes.data, d.nbytes)
        return d

    def numpy(self) -> np.ndarray:
        out = np.empty(self.shape, dtype=np.uint16 if self.dtype == "bfloat16" else self.dtype)
        if self.nbytes:
            self._lib.download_hip(out.ctypes.data, self._ptr, self.nbytes)
        return out

    def data_ptr(self) -> int:
        return self._ptr

    def stride(self):
        s, out = 1, []
        for n in reversed(self.shape):
            out.append(s)
            s *= n
        return tuple(reversed(out))

    def is_contiguous(self) -> bool:
        return True

    def __del__(self):
        if getattr(self, "_ptr", None):
            self._lib.free_hip(self._ptr)
            self._ptr = None


_lib_ready = None


def _lib():
    """the library, bound to the one HIP runtime of the process"""
    global _lib_ready
    if _lib_ready is None:
        lib = host.load_lib()
        if "torch" in sys.modules:
            with open("/proc/self/maps") as f:
                runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
            if len(runtimes) > 1:
                raise RuntimeError("libcalm_hip.so was loaded before torch, and each has its own HIP runtime: import torch first (" + ", ".join(sorted(runtimes)) + ")")
        _lib_ready = lib
    return _lib_ready


def _name(x) -> str:
    d = x.dtype
    n = _NAMES.get(d)
    if n is None:
        n = str(d)
        n = _NAMES[d] = n[6:] if n.startswith("torch.") else n
    return n


_nothing = contextlib.nullcontext()
_INT = 2 ** 31 - 1
_torch = None  # torch and the functions that every call asks, once it is known to be there


def _torch_calls():
    global _torch
    if _torch is None:
        import torch
        import torch.autograd.forward_ad as forward

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle alone, without a Stream object around it
        _torch = (torch, torch.Tensor, raw or (lambda i: torch.cuda.current_stream(i).cuda_stream), getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device), forward)
    return _torch


def _on(arrays):
    """(stream, guard) of a call's arrays: a hipStream_t, and None or a context that makes their device current"""
    first = arrays[0]
    if isinstance(first, DeviceArray):
        for a in arrays:
            if not isinstance(a, DeviceArray):
                raise ValueError("tensors and DeviceArrays in one call")
        return _lib().calm_hip_stream(), None
    torch, tensor, raw_stream, current, forward = _torch or _torch_calls()
    dev = first.device
    if dev.type != "cuda":
        raise ValueError(f"arrays on {dev}: these operators run on the GPU only")
    grads, tangents = torch.is_grad_enabled(), forward._current_level >= 0
    for a in arrays:
        if not isinstance(a, tensor):
            raise ValueError("tensors and DeviceArrays in one call")
        if a.device != dev:
            raise ValueError(f"arrays on {dev} and on {a.device} in one call")
        if grads and a.requires_grad:
            raise ValueError("there is no backward pass: call under torch.no_grad()")
        if tangents and forward.unpack_dual(a).tangent is not None:
            raise ValueError("there is no derivative: a tensor has a forward-mode tangent")
    index = dev.index
    return raw_stream(index), None if index == current() else torch.cuda.device(dev)


def _call(guard, entry, *args) -> None:
    """the C entry, on the arrays' device; ValueError if it refuses"""
    if guard is None:
        rc = entry(*args)
    else:
        with guard:
            rc = entry(*args)
    if rc:
        raise ValueError(_lib().calm_hip_error().decode())


def _empty(like, shape, dtype: str):
    if isinstance(like, DeviceArray):
        return DeviceArray(shape, dtype)
    kind = _DTYPES.get(dtype)
    if kind is None:
        kind = _DTYPES[dtype] = getattr((_torch or _torch_calls())[0], dtype)
    return like.new_empty(shape, dtype=kind)


def _need(cond, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _together(arrays) -> None:
    """arrays that are kept for later calls: of one kind, on one device"""
    first = arrays[0]
    for a in arrays:
        if isinstance(a, DeviceArray) != isinstance(first, DeviceArray):
            raise ValueError("tensors and DeviceArrays in one call")
        if getattr(a, "requires_grad", False):
            raise ValueError("there is no backward pass, and the arrays of a pool or batch are written in place: detach() them")
        if getattr(a, "device", None) != getattr(first, "device", None):
            raise ValueError(f"arrays on {first.device} and on {a.device} in one call")


def _sees(layer: int, layers: int, window: int, sinks: int) -> None:
    if not 0 <= layer < layers:
        raise ValueError(f"no such layer: {layer} of {layers}")
    if not (0 <= window <= _INT and 0 <= sinks <= _INT):
        raise ValueError(f"window {window} and first tokens {sinks}: 0 to {_INT}")


def _array(x, name: str, dtypes, shape) -> None:
    """x is a dense array of one of `dtypes` and of `shape` (None: any size)"""
    if _name(x) not in dtypes:
        raise ValueError(f"{name}: {_name(x)} where {' or '.join(dtypes)} is wanted")
    got = x.shape
    if got != shape and (len(got) != len(shape) or any(w is not None and w != n for n, w in zip(got, shape))):
        got = tuple(got)
        raise ValueError(f"{name}: shape {got} where {tuple('any' if w is None else w for w in shape)} is wanted")
    if not x.is_contiguous():
        raise ValueError(f"{name} is not contiguous")


def _sizes(table):
    """rows and columns of a table"""
    if len(table.shape) != 2:
        raise ValueError(f"table: shape {tuple(table.shape)} where [rows][pages] is wanted")
    _array(table, "table", ("int32",), table.shape)
    n, mp = table.shape
    return n, mp


def _rows(x, name: str, rows: int, heads: Optional[int], dim: int):
    """x is [rows][heads][dim] with dense dims; its row and head strides"""
    if _name(x) not in _TYPES:
        raise ValueError(f"{name}: {_name(x)} where float32, float16 or bfloat16 is wanted")
    shape = x.shape
    if len(shape) != 3 or shape[0] < rows or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name}: shape {tuple(shape)} where ({rows}, {heads or 'heads'}, {dim}) is wanted")
    r, h, d = x.stride()
    if d != 1:
        raise ValueError(f"{name}: the dims of a head are not contiguous")
    if r % 4 or h % 4:
        raise ValueError(f"{name}: row and head strides {r}, {h} are not multiples of four elements")
    return r, h


class _Fixed:
    """attributes that are set once: the library has the arrays' addresses and the bounds from then on (`_c`)"""

    def __setattr__(self, name, value):
        if "_c" in self.__dict__:
            raise AttributeError(f"{type(self).__name__}.{name} is not changed behind its making: make another")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} is not taken away: make another")


class KvPool(_Fixed):
    """pages of a cache, for every layer of a model"""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, device=None):
        """device: a torch device for tensors, None for memory of the library"""
        _need(head_dim in HEAD_DIMS, f"head size {head_dim}: {HEAD_DIMS} are there")
        _need(n_layers > 0 and n_pages > 0 and n_kv_heads > 0, "a pool without layers, pages or heads")
        shape = (n_layers, n_pages, n_kv_heads)

        def new(tail, dtype):
            if device is None:
                return DeviceArray(shape + tail, dtype)
            import torch

            return torch.empty(shape + tail, dtype=getattr(torch, dtype), device=device)

        self._set(new((PAGE, head_dim), "int8"), new((4, head_dim, 16), "int8"), new((4,), "float32"), new((4,), "float32"))

    @classmethod
    def over(cls, k, v, k_scale, v_scale) -> "KvPool":
        """a pool in arrays that the caller has: k int8 [layers][pages][heads][64][dim], v int8 [layers][pages][heads][4][dim][16] (byte
        4 b + i of quad g: token 16 b + 4 g + i), scales float32 [layers][pages][heads][4], positive powers of two or NaN"""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        _need(len(k.shape) == 5, "k: [layers][pages][heads][64][dim]")
        layers, pages, heads, _, dim = (int(n) for n in k.shape)
        _need(dim in HEAD_DIMS, f"head size {dim}: {HEAD_DIMS} are there")
        _array(k, "k", ("int8",), (layers, pages, heads, PAGE, dim))
        _array(v, "v", ("int8",), (layers, pages, heads, 4, dim, 16))
        for x, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _array(x, name, ("float32",), (layers, pages, heads, 4))
        _together((k, v, k_scale, v_scale))
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_layers, self.n_pages, self.n_kv_heads, self.head_dim = layers, pages, heads, dim
        if isinstance(k, DeviceArray):
            self.status = DeviceArray.of(np.zeros(1, dtype=np.int32))
        else:
            import torch

            self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        c = _Pool(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.status.data_ptr(), layers, pages, heads, dim)
        self._ref = C.byref(c)
        self._c = c

    def check(self) -> None:
        """waits for the calls so far, on any stream, and raises RuntimeError if one of them found its pages or batch wanting"""
        if isinstance(self.status, DeviceArray):
            found = int(self.status.numpy()[0])
            if found:  # (in place: a captured graph has the word's address)
                none = np.zeros(1, dtype=np.int32)
                self.status._lib.copy_hip(self.status.data_ptr(), none.ctypes.data, none.nbytes)
        else:
            import torch

            torch.cuda.synchronize(self.status.device)  # (.item() waits for the current stream alone)
            found = int(self.status.item())
            if found:
                self.status.zero_()
                torch.cuda.synchronize(self.status.device)  # (before a call on another stream finds something new)
        words = [(1, "a page that was needed is missing from the table or outside the pool"), (2, "no page was free"),
                 (4, "a sequence has more new rows than max_rows, or row starts that do not fit the rows"), (8, "a parent outside the table")]
        if found:
            raise RuntimeError("paged cache: " + "; ".join(w for bit, w in words if found & bit))


class KvBatch(_Fixed):
    """Which rows of a call belong to which sequence: rows starts[s] .. starts[s + 1] - 1 are the last tokens of sequence s, which has lens[s]
    tokens with them.  The arrays are read when a call runs, so a program may change their values between calls (other arrays -- the table of a
    fork, say -- make another batch); rows, max_rows and max_len are the host's bounds (rows: what the packed row arrays hold; max_rows: of one sequence; max_len: tokens of a sequence)."""

    def __init__(self, table, lens, starts, rows: int, max_rows: int, max_len: int):
        n, mp = _sizes(table)
        _array(lens, "lens", ("int32",), (n,))
        _array(starts, "starts", ("int32",), (n + 1,))
        _together((table, lens, starts))
        _need(n > 0 and mp > 0, "a table without rows or columns")
        _need(rows <= _INT and max_len <= _INT, f"rows and max_len are at most {_INT}")
        _need(rows >= 0 and 0 <= max_rows <= rows and max_len >= 0, "rows, max_rows and max_len are not negative, max_rows is at most rows")
        self.table, self.lens, self.starts = table, lens, starts
        self.n_seqs, self.rows, self.max_rows, self.max_len = n, rows, max_rows, max_len
        self._work = {}  # workspace sizes of attention
        c = _Batch(table.data_ptr(), lens.data_ptr(), starts.data_ptr(), n, mp, rows, max_rows, max_len)
        self._ref = C.byref(c)
        self._c = c


def append(pool: KvPool, batch: KvBatch, k, v, layer: int = 0) -> None:
    """K and V rows [rows][kv heads][dim] (strided rows and heads) into the pages of their sequences"""
    kr, kh = _rows(k, "k", batch.rows, pool.n_kv_heads, pool.head_dim)
    vr, vh = _rows(v, "v", batch.rows, pool.n_kv_heads, pool.head_dim)
    _need(_name(k) == _name(v), "k and v of different types")
    _sees(layer, pool.n_layers, 0, 0)
    stream, guard = _on((k, v, pool.k, batch.table))
    _call(guard, _lib().kv_append_hip, pool._ref, batch._ref, layer, k.data_ptr(), v.data_ptr(), _TYPES[_name(k)], kr, kh, vr, vh, stream)


def attend(pool: KvPool, batch: KvBatch, q, layer: int = 0, window: int = 0, sinks: int = 0, scale: Optional[float] = None, out=None):
    """softmax(scale q . K) . V for query rows [rows][query heads][dim]: a row at position p sees tokens j <= p, with a window > 0 those of them
    with j > p - window or j < sinks; zeros where it sees none.  scale: dim ** -0.5 if not given; out does not overlap q.  Rows behind the last sequence's
    are not written: of a result that was not given as `out` they are whatever its memory held"""
    dim = pool.head_dim
    _sees(layer, pool.n_layers, window, sinks)
    qr, qh = _rows(q, "q", batch.rows, None, dim)
    heads = int(q.shape[1])
    if out is None:
        out = _empty(q, (int(q.shape[0]), heads, dim), _name(q))
    else:
        _array(out, "out", (_name(q),), tuple(q.shape))
    lib, kind = _lib(), _TYPES[_name(q)]
    stream, guard = _on((q, out, pool.k, batch.table))
    # (the workspace's size follows from shapes and bounds alone)
    key = (kind, heads, window, sinks, pool.n_kv_heads, dim)
    need = batch._work.get(key)
    if need is None:
        with guard or _nothing:
            need = lib.kv_attend_workspace_hip(pool._ref, batch._ref, kind, heads, window, sinks)
        if need < 0:
            raise ValueError(lib.calm_hip_error().decode())
        batch._work[key] = need
    work = _empty(q, (need // 4,), "float32") if need else None
    _call(guard, lib.kv_attend_hip, pool._ref, batch._ref, layer, q.data_ptr(), out.data_ptr(), kind, heads, qr, qh, dim ** -0.5 if scale is None else scale, window, sinks,
          work.data_ptr() if need else None, need, stream)
    return out


def read(pool: KvPool, table, lens, start, count: int, layer: int = 0, dtype: str = "float32"):
    """(K, V), [seqs][count][kv heads][dim]: the values of tokens start[s] .. start[s] + count - 1, zeros where sequence s has no such token"""
    n, mp = _sizes(table)
    _array(lens, "lens", ("int32",), (n,))
    _array(start, "start", ("int32",), (n,))
    _need(dtype in _TYPES, f"{dtype} where float32, float16 or bfloat16 is wanted")
    _need(0 <= count <= _INT, f"{count} tokens")
    _sees(layer, pool.n_layers, 0, 0)
    stream, guard = _on((pool.k, table, lens, start))
    k, v = (_empty(pool.k, (n, count, pool.n_kv_heads, pool.head_dim), dtype) for _ in range(2))
    _call(guard, _lib().kv_read_hip, pool._ref, layer, table.data_ptr(), lens.data_ptr(), start.data_ptr(), n, mp, count, k.data_ptr(), v.data_ptr(), _TYPES[dtype], stream)
    return k, v


def _table(pool, table, refs):
    _array(refs, "refs", ("int32",), (pool.n_pages,))
    return _sizes(table)


def reserve(pool: KvPool, table, refs, lens, lens_new) -> None:
    """pages for tokens lens[r] .. lens_new[r] - 1 of every row of the table, in place; refs[p] counts the rows that list page p.  These pages are the row's own
    then: one that was cut back gives up pages that other rows list, too, for others, with the tokens that it keeps"""
    n, mp = _table(pool, table, refs)
    _array(lens, "lens", ("int32",), (n,))
    _array(lens_new, "lens_new", ("int32",), (n,))
    stream, guard = _on((table, refs, lens, lens_new, pool.k))
    _call(guard, _lib().kv_reserve_hip, pool._ref, table.data_ptr(), refs.data_ptr(), lens.data_ptr(), lens_new.data_ptr(), n, mp, stream)


def trim(pool: KvPool, table, refs, lens, window: int = 0, sinks: int = 0) -> None:
    """gives up, in place, the pages behind lens[r] (0: the whole row) and, with a window > 0, those that no later token of the row sees"""
    n, mp = _table(pool, table, refs)
    _array(lens, "lens", ("int32",), (n,))
    _sees(0, 1, window, sinks)
    stream, guard = _on((table, refs, lens, pool.k))
    _call(guard, _lib().kv_trim_hip, pool._ref, table.data_ptr(), refs.data_ptr(), lens.data_ptr(), n, mp, window, sinks, stream)


def fork(pool: KvPool, table, lens, refs, parents):
    """(table, refs) in which row r continues row parents[r]: full pages are shared, a page that is not full is copied for every child but its
    row's first.  (Lengths follow as lens[parents].)"""
    n, mp = _table(pool, table, refs)
    _array(lens, "lens", ("int32",), (n,))
    _array(parents, "parents", ("int32",), (n,))
    stream, guard = _on((table, refs, lens, parents, pool.k))
    new, now, work = _empty(table, (n, mp), "int32"), _empty(table, (pool.n_pages,), "int32"), _empty(table, (2 * n,), "int32")
    _call(guard, _lib().kv_fork_hip, pool._ref, table.data_ptr(), lens.data_ptr(), refs.data_ptr(), parents.data_ptr(), n, mp, new.data_ptr(), now.data_ptr(),
          work.data_ptr(), 8 * n, stream)
    return new, now


def compact(pool: KvPool, table, refs):
    """(table, refs, number of live pages) after the live pages at or behind that number have moved into the free ones before it"""
    n, mp = _table(pool, table, refs)
    stream, guard = _on((table, refs, pool.k))
    new, now, live = _empty(table, (n, mp), "int32"), _empty(table, (pool.n_pages,), "int32"), _empty(table, (1,), "int32")
    work = _empty(table, (2 * pool.n_pages,), "int32")
    _call(guard, _lib().kv_compact_hip, pool._ref, table.data_ptr(), refs.data_ptr(), n, mp, new.data_ptr(), now.data_ptr(), live.data_ptr(), work.data_ptr(),
          8 * pool.n_pages, stream)
    return new, now, live


def beam_select(logits, scores, done=None, eos: int = -1):
    """(scores, parents, tokens, done), [groups][beams] each: the best continuations of every group's beams by score + log softmax(logits), best first,
    equal ones by beam, then token.  logits [groups * beams][vocab] (strided rows), scores float32 [groups][beams], done uint8 [groups][beams]: a hypothesis that
    is done continues with `eos` alone, its score unchanged; eos < 0: there is none"""
    _array(scores, "scores", ("float32",), (None, None))
    groups, beams = (int(x) for x in scores.shape)
    _need(1 <= beams <= MAX_BEAMS and groups >= 1, f"1 to {MAX_BEAMS} beams")
    _need(_name(logits) in _TYPES, f"logits: {_name(logits)} where float32, float16 or bfloat16 is wanted")
    _need(len(logits.shape) == 2 and logits.shape[0] == groups * beams and logits.shape[1] >= 1, "logits: [groups * beams][vocab]")
    row, one = logits.stride()
    vocab = int(logits.shape[1])
    _need(one == 1 or vocab == 1, "the logits of a row are not contiguous")
    arrays = [logits, scores]
    if done is not None:
        _array(done, "done", ("uint8", "bool"), (groups, beams))
        arrays.append(done)
    _need(-_INT <= eos <= _INT, f"eos {eos}")
    lib = _lib()
    stream, guard = _on(arrays)
    need = lib.beam_workspace_hip(groups, beams, vocab)
    if need < 0:
        raise ValueError(lib.calm_hip_error().decode())
    best, parents, tokens, ended = (_empty(scores, (groups, beams), d) for d in ("float32", "int32", "int32", "uint8"))
    work = _empty(scores, (-(-need // 4),), "float32")
    _call(guard, lib.beam_select_hip, logits.data_ptr(), _TYPES[_name(logits)], row if groups * beams > 1 else max(row, vocab), groups, beams, vocab, scores.data_ptr(),
          done.data_ptr() if done is not None else None, eos, best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ended.data_ptr(), work.data_ptr(), need, stream)
    return best, parents, tokens, ended
