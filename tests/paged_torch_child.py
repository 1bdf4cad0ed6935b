"""The paged operators on torch tensors: run by tests/test_paged_torch.py in a process of its own (torch has to come before the library).

Prints one line per check, then ALL OK."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from calm_amd import paged  # noqa: E402


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def case(seed, seqs=3, length=900, heads=2, dim=64, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mp = -(-length // 64)
    pool = paged.KvPool(1, seqs * mp, heads, dim, device="cuda")
    table = torch.randperm(seqs * mp, device="cuda", generator=g).to(torch.int32).view(seqs, mp)
    lens = ints([length] * seqs)
    kv = torch.randn((2, seqs * length, heads, dim), device="cuda", generator=g).to(dtype)
    paged.append(pool, paged.KvBatch(table, lens, ints([i * length for i in range(seqs + 1)]), rows=seqs * length, max_rows=length, max_len=length), kv[0], kv[1])
    batch = paged.KvBatch(table, lens, ints(range(seqs + 1)), rows=seqs, max_rows=1, max_len=length)
    q = torch.randn((seqs, 4 * heads, dim), device="cuda", generator=g).to(dtype)
    return pool, batch, q, kv


def values(pool, batch, length):
    return paged.read(pool, batch.table, batch.lens, ints([0] * batch.n_seqs), length)


def plain(pool, batch, q, length):
    k, v = (x.double() for x in values(pool, batch, length))
    group = q.shape[1] // k.shape[2]
    k, v = (x.repeat_interleave(group, 2).permute(0, 2, 1, 3).contiguous() for x in (k, v))
    p = (torch.matmul(k, q.double().unsqueeze(-1))[..., 0] * q.shape[2] ** -0.5).softmax(-1)
    return torch.matmul(p.unsqueeze(-2), v)[..., 0, :]


def near(a, b, tol):
    assert float((a.double() - b.double()).abs().max()) <= tol * float(b.abs().max()), float((a.double() - b.double()).abs().max())


# fp32: sums of 900 weights and 64 products, each 2^-24 .. 2^-22 off, all alike at the very worst: 900 * 2^-24 = 5e-5.  bf16: its rounding, 2^-8, beside it
pool, batch, q, kv = case(1)
want = plain(pool, batch, q, 900)
near(paged.attend(pool, batch, q), want, 1e-4)
print("default stream", flush=True)

for dtype, tol in ((torch.float16, 2.0 ** -10), (torch.bfloat16, 2.0 ** -7)):
    p2, b2, q2, _ = case(2, dtype=dtype, dim=128)
    near(paged.attend(p2, b2, q2), plain(p2, b2, q2, 900), tol)
print("16-bit rows", flush=True)

# another stream than the tensors' own, ordered by torch's rules; and two streams at once, each call with a workspace of its own
streams = [torch.cuda.Stream() for _ in range(2)]
others = [case(10 + i, length=3000, seqs=2) for i in range(2)]
plains = [plain(p, b, x, 3000) for p, b, x, _ in others]
torch.cuda.synchronize()
got = [None, None]
for rep in range(5):
    for i, st in enumerate(streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got[i] = paged.attend(others[i][0], others[i][1], others[i][2])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for i in range(2):
        near(got[i], plains[i], 1e-4)
print("two streams at once", flush=True)

# captured: a decode step of append + attend, and a fork + select, replayed with changing inputs and the program's own eager work between
length = 2000
pool, batch, q, kv = case(3, length=length, seqs=2)
lens, fresh = batch.lens, torch.zeros((2, 2, 2, 64), device="cuda")
step = lambda: (paged.append(pool, batch, fresh[0], fresh[1]), paged.attend(pool, batch, q, window=1500, sinks=3))[1]  # noqa: E731
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
torch.cuda.current_stream().wait_stream(side)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph2 = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph2):
    out2 = step()
for rep in range(6):
    fresh.copy_(torch.randn_like(fresh) * (1 + rep))
    q.copy_(torch.randn_like(q))
    lens.copy_(ints([length - 3 * rep, length - 64 * rep]))
    graph.replay()
    once = out.clone()
    torch.cuda.synchronize()
    eager = step()
    graph2.replay()  # (the same step, another graph: its own workspace)
    assert torch.equal(once, eager) and torch.equal(out2, eager), rep
print("captured and replayed", flush=True)

refs = torch.ones(pool.n_pages, dtype=torch.int32, device="cuda")
parents = ints([1, 1])
logits, scores, done = torch.randn((2, 5000), device="cuda"), torch.zeros((1, 2), device="cuda"), torch.zeros((1, 2), dtype=torch.bool, device="cuda")
table = batch.table
table[0] = -1
refs[:] = 0
refs[table[1].long()] = 1
lens.copy_(ints([0, 1990]))
graph3 = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph3):
    t2, r2 = paged.fork(pool, table, lens, refs, parents)
    t3, r3, live = paged.compact(pool, t2, r2)
    best = paged.beam_select(logits, scores, done, eos=7)
for rep in range(4):
    logits.copy_(torch.randn_like(logits))
    done.copy_(torch.tensor([[rep % 2 == 1, False]]))
    graph3.replay()
    a = [x.clone() for x in (t2, r2, t3, r3, live, *best)]
    torch.cuda.synchronize()
    e2 = paged.fork(pool, table, lens, refs, parents)
    e3 = paged.compact(pool, *e2)
    # (compact moved the pages: the same tables again, and the same places)
    for x, y in zip(a, (*e2, *e3, *paged.beam_select(logits, scores, done, eos=7))):
        assert torch.equal(x, y), rep
assert (best[3] == ((done.gather(1, best[1].long())) | (best[2] == 7))).all()
pool.check()
print("bookkeeping captured", flush=True)

# what the wrappers refuse of tensors
for bad, words in ((lambda: paged.attend(pool, batch, q.cpu()), "GPU only"), (lambda: paged.attend(pool, batch, q.clone().requires_grad_()), "no backward"),
                   (lambda: paged.attend(pool, batch, q.transpose(1, 2).contiguous().transpose(1, 2)), "not contiguous"), (lambda: paged.attend(pool, batch, q.double()), "float64"),
                   (lambda: paged.append(pool, batch, fresh[0], paged.DeviceArray.__new__(paged.DeviceArray)), "")):
    try:
        bad()
    except (ValueError, AttributeError) as e:
        assert words in str(e), e
    else:
        raise AssertionError(words)
with torch.no_grad():
    paged.attend(pool, batch, q.clone().requires_grad_())
print("refusals", flush=True)

# strided rows: the heads of a packed projection, and every other row
wide = torch.randn((4, 12, 64), device="cuda")
rows = wide[::2]
lens.copy_(ints([0, 1990]))
paged.append(pool, batch, rows[:, 8:10], rows[:, 10:12])
one = paged.attend(pool, batch, rows[:, :8])
two = paged.attend(pool, batch, rows[:, :8].contiguous())
assert torch.equal(one, two)
print("strides", flush=True)
print("ALL OK")
