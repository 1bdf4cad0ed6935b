"""Corners of calm_amd/paged.py on torch tensors: run by tests/test_paged_corners.py in a process of its own (torch has to come before the library).

Prints one line per check, then ALL OK."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from calm_amd import paged  # noqa: E402


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def refused(f, words, kind=ValueError):
    try:
        f()
    except kind as e:
        assert words in str(e), e
    else:
        raise AssertionError(words)


pool = paged.KvPool(1, 8, 2, 64, device="cuda")
table, lens = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), ints([200, 130])
paged.append(pool, paged.KvBatch(table, lens, ints([0, 200, 330]), rows=330, max_rows=200, max_len=200), *(torch.randn((330, 2, 64), device="cuda") for _ in range(2)))
batch = paged.KvBatch(table, lens, ints([0, 1, 2]), rows=2, max_rows=1, max_len=200)
q = torch.randn((2, 4, 64), device="cuda")
want = paged.attend(pool, batch, q)
pool.check()

# check() waits for calls on every stream, not on the current one alone; what it found is cleared for good
side = torch.cuda.Stream()
big = torch.randn((8192, 8192), device="cuda")
torch.cuda.synchronize()
bad = paged.KvBatch(ints([[0, 1, 2, -1], [-1, -1, -1, -1]]), lens, ints([0, 1, 2]), rows=2, max_rows=1, max_len=200)
torch.cuda.synchronize()
for rep in range(3):
    with torch.cuda.stream(side):
        for _ in range(20):
            torch.mm(big, big)
        paged.attend(pool, bad, q)
    refused(pool.check, "missing", RuntimeError)
    pool.check()
with torch.cuda.stream(side):
    paged.attend(pool, bad, q)
refused(pool.check, "missing", RuntimeError)
assert torch.equal(paged.attend(pool, batch, q), want)
pool.check()
print("check", flush=True)

# no derivative is dropped silently: forward-mode tangents and arrays of a pool that require gradients are refused as reverse-mode ones are
import torch.autograd.forward_ad as fwd  # noqa: E402

with fwd.dual_level():
    refused(lambda: paged.attend(pool, batch, fwd.make_dual(q, torch.ones_like(q))), "no derivative")
    rows = torch.randn((2, 2, 64), device="cuda")
    refused(lambda: paged.append(pool, batch, rows, fwd.make_dual(rows, rows)), "no derivative")
    x = torch.randn((2, 50), device="cuda")
    refused(lambda: paged.beam_select(fwd.make_dual(x, x), torch.zeros((1, 2), device="cuda")), "no derivative")
    assert torch.equal(paged.attend(pool, batch, q), want)  # (tensors without tangents)
assert torch.equal(paged.attend(pool, batch, q), want)
refused(lambda: paged.KvPool.over(pool.k, pool.v, pool.k_scale.clone().requires_grad_(), pool.v_scale), "no backward")
print("forward mode", flush=True)

# from a selection to a fork: the beams of a group as rows of the table
groups, width = 2, 3
table6 = torch.arange(12, dtype=torch.int32, device="cuda").view(6, 2)
pool6 = paged.KvPool(1, 12, 1, 64, device="cuda")
refs6, lens6 = torch.ones(12, dtype=torch.int32, device="cuda"), ints([128] * 6)
logits = torch.full((6, 10), -5.0, device="cuda")
for row, tok in ((2, 4), (2, 5), (0, 6), (4, 1), (4, 2), (4, 3)):
    logits[row, tok] = 9.0 - tok
best, beams, tokens, done = paged.beam_select(logits, torch.zeros((groups, width), device="cuda"))
parents = (beams + torch.arange(0, groups * width, width, dtype=torch.int32, device="cuda")[:, None]).view(-1)
t2, r2 = paged.fork(pool6, table6, lens6, refs6, parents)
# (row 0: one token at 3, -0.0; row 2: 5 and 4, -0.3 and -1.3; row 4: 8, 7 and 6, -0.4, -1.4 and -2.4; the even rows: -log 10 = -2.3 each)
assert parents.tolist() == [0, 2, 2, 4, 4, 3]
assert torch.equal(t2, table6[parents.long()])
assert torch.equal(r2, torch.bincount(t2.flatten().long(), minlength=12).to(torch.int32))
pool6.check()
print("selection to fork", flush=True)
print("ALL OK")
