"""The paged 8-bit cache's operators and the beam search's selection, as they are measured.

A cache of several sequences lives in pages of 64 tokens. A page holds, for every kv head, 8-bit codes c in [-127, 127] of K and of V and one
scale s (a power of two) for each block of 16 tokens: the value is c * s. The operators:

  append    new K / V rows, quantised into the pages of their sequences: a block's scale is the least power of two with max|x| <= 127 s over
            the block's tokens; a block that already holds tokens keeps the larger of its scale and the new rows', its codes rounded to it
  attend    softmax attention of query rows (the last rows of their sequences) over the cached tokens j of their sequence with
            j <= p and (no window, or j > p - window, or j < sinks), p the row's own position; heads share kv heads in groups
  fork      rows of the page table are replaced by their parents' (beam reordering): whole pages are shared and counted, a page that is
            not full gets a copy of its own for every child but the first
  compact   live pages beyond the first n_live move into the holes among them, tables and counts follow
  select    for every group of W beams the W best of W x vocabulary continuations by score + log softmax(logits), ties to the lowest index

`own` = False computes the plain forms with elementary torch operations, True calls the library.
"""
import torch

own = False

PAGE = 64   # tokens a page holds
BLOCK = 16  # tokens that share a scale, for one kv head
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of 48 sequences being decoded together: a few KB of work, latency
        dict(name="append decode", op="append", dtype="fp32", seqs=48, kv_heads=8, head_dim=128, length=2051, spread=1990, rows=1, ragged=False),
        # prompts of six sequences arriving together, ragged, behind tokens that are cached already
        dict(name="append prompts", op="append", dtype="fp16", seqs=6, kv_heads=8, head_dim=128, length=5003, spread=777, rows=4099, ragged=True),
        # one short sequence, fp32 activations as the decode step has them: the smallest call
        dict(name="attend short", op="attend", dtype="fp32", seqs=1, q_heads=32, kv_heads=8, head_dim=128, length=333, spread=0, rows=1, ragged=False, window=0, sinks=0),
        # eight beams over contexts of a few thousand tokens
        dict(name="attend beams", op="attend", dtype="fp32", seqs=8, q_heads=32, kv_heads=8, head_dim=128, length=4093, spread=61, rows=1, ragged=False, window=0, sinks=0),
        # many sequences of very different lengths, eight heads to a kv head of 64
        dict(name="attend ragged d64", op="attend", dtype="fp16", seqs=64, q_heads=32, kv_heads=4, head_dim=64, length=8191, spread=8100, rows=1, ragged=False, window=0, sinks=0),
        # long contexts, groups of six heads: the most bytes
        dict(name="attend long", op="attend", dtype="bf16", seqs=24, q_heads=48, kv_heads=8, head_dim=128, length=16389, spread=2500, rows=1, ragged=False, window=0, sinks=0),
        # a window of 1024 tokens and four first tokens, a few draft tokens to check at once
        dict(name="attend window draft", op="attend", dtype="bf16", seqs=16, q_heads=32, kv_heads=8, head_dim=128, length=9001, spread=3001, rows=5, ragged=True, window=1024, sinks=4),
        # a prompt chunk behind a cached prefix
        dict(name="attend chunk", op="attend", dtype="bf16", seqs=1, q_heads=32, kv_heads=8, head_dim=128, length=4099, spread=0, rows=2049, ragged=False, window=0, sinks=0),
        # ragged chunks of several sequences under a window with first tokens
        dict(name="attend chunk window", op="attend", dtype="fp16", seqs=5, q_heads=32, kv_heads=4, head_dim=64, length=6007, spread=2222, rows=1021, ragged=True, window=2048, sinks=2),
        # eight beams of each of six sequences are reordered, all layers
        dict(name="fork beams", op="fork", groups=6, beams=8, survivors=5, kv_heads=8, head_dim=128, layers=16, length=1037, spread=700),
        # a pool whose sequences came and went
        dict(name="compact pool", op="compact", pages=900, live=520, moved=150, rows=20, kv_heads=8, head_dim=128, layers=8),
        # eight beams of each of sixteen sequences over a large vocabulary, some of them finished
        dict(name="select beams", op="select", dtype="fp32", groups=16, beams=8, vocab=128256, finished=9),
    ]


def _log(rng, a, b):
    return int(round(a * (b / a) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "chunk", "fork", "compact", "select", "select"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    heads, group, dim = rng.choice([(8, 4, 128), (4, 8, 64), (8, 6, 128), (8, 1, 64), (2, 7, 128), (3, 2, 96), (4, 4, 256), (1, 8, 96)])
    if op == "append":
        rows = rng.choice([1, 1, _log(rng, 2, 1500)])
        length = rows + _log(rng, 1, 6000)
        seqs = max(1, min(_log(rng, 1, 64), 12000 // rows))
        return dict(op="append", dtype=dtype, seqs=seqs, kv_heads=heads, head_dim=dim, length=length, spread=rng.randrange(0, length - rows + 1), rows=rows,
                    ragged=rng.random() < 0.5)
    if op in ("attend", "chunk"):
        rows = _log(rng, 40, 1200) if op == "chunk" else rng.choice([1, 1, 1, rng.randrange(2, 9)])
        length = rows + _log(rng, 1, 2500 if op == "chunk" else 12000)
        seqs = max(1, min(_log(rng, 1, 6 if op == "chunk" else 64), 150000 // length))
        seqs = max(1, min(seqs, 80000000000 // (4 * rows * length * heads * group * dim)))
        window = rng.choice([0, 0, _log(rng, 8, 4096)])
        return dict(op="attend", dtype=dtype, seqs=seqs, q_heads=heads * group, kv_heads=heads, head_dim=dim, length=length, spread=rng.randrange(0, length - rows + 1), rows=rows,
                    ragged=rng.random() < 0.5, window=window, sinks=rng.choice([0, 1, 2, 4, 17]) if window else 0)
    if op == "fork":
        beams = rng.randrange(2, 17)
        length = _log(rng, 20, 3000)
        return dict(op="fork", groups=rng.randrange(1, 5), beams=beams, survivors=rng.randrange(1, beams + 1), kv_heads=heads, head_dim=dim, layers=rng.randrange(1, 17),
                    length=length, spread=rng.randrange(0, length))
    if op == "compact":
        pages = _log(rng, 12, 800)
        live = rng.randrange(2, pages - 1)
        return dict(op="compact", pages=pages, live=live, moved=rng.randrange(0, min(live, pages - live, 300) + 1), rows=rng.randrange(1, min(16, live) + 1), kv_heads=heads, head_dim=dim,
                    layers=rng.randrange(1, 9))
    beams = rng.randrange(1, 17)
    groups = _log(rng, 1, 16)
    return dict(op="select", dtype=dtype, groups=groups, beams=beams, vocab=min(_log(rng, 300, 150000), 15000000 // (groups * beams)), finished=rng.randrange(0, groups * beams // 2 + 1))


def _lengths(c):
    """tokens of every sequence, its new rows included: from `length` down to `length - spread`"""
    n = c["seqs"]
    return [c["length"] - (i * c["spread"] // (n - 1) if n > 1 else 0) for i in range(n)]


def _rows(c):
    """new rows of every sequence"""
    return [max(1, c["rows"] - (i * 977) % c["rows"]) if c["ragged"] else c["rows"] for i in range(c["seqs"])]


def _visible(c):
    """(query, key) pairs, and keys that some row of their sequence sees"""
    pairs = keys = 0
    w, s = c["window"], c["sinks"]
    for n, r in zip(_lengths(c), _rows(c)):
        first = n - r
        for p in range(first, n):
            pairs += p + 1 if not w else min(p + 1, w) + min(s, max(0, p + 1 - w))
        keys += n if not w else n - max(0, first + 1 - w) + min(s, max(0, first + 1 - w))
    return pairs, keys


def work(case):
    c, op = case, case["op"]
    if op == "append":
        t, per = sum(_rows(c)), 2 * c["kv_heads"] * c["head_dim"]
        # rows in, codes and scales out, the blocks read back as the values that they stand for
        blocks = sum(-(-n // BLOCK) - (n - r) // BLOCK for n, r in zip(_lengths(c), _rows(c)))
        back = c["seqs"] * _back(c) * per * 4
        return {"bytes": t * per * (SIZE[c["dtype"]] + 1) + blocks * 2 * c["kv_heads"] * 4 + back, "flops": 4 * t * per}
    if op == "attend":
        pairs, keys = _visible(c)
        t, d = sum(_rows(c)), c["head_dim"]
        return {"bytes": keys * c["kv_heads"] * 2 * (d + 4 / BLOCK) + 2 * t * c["q_heads"] * d * SIZE[c["dtype"]], "flops": 4 * pairs * c["q_heads"] * d}
    page = 2 * PAGE * c["kv_heads"] * (c["head_dim"] + 4 / BLOCK) * c["layers"] if op != "select" else 0
    if op == "fork":
        parts = sum((c["beams"] - c["survivors"]) for g in range(c["groups"]) if _fork_lengths(c)[g] % PAGE)
        return {"bytes": 2 * parts * page + 4 * _fork_table(c), "flops": 0}
    if op == "compact":
        return {"bytes": 2 * c["moved"] * page + 8 * c["pages"], "flops": 0}
    n = c["groups"] * c["beams"]
    return {"bytes": n * c["vocab"] * SIZE[c["dtype"]] + n * 25, "flops": 4 * n * c["vocab"]}


def _fork_lengths(c):
    return [c["length"] - (g * c["spread"] // (c["groups"] - 1) if c["groups"] > 1 else 0) for g in range(c["groups"])]


def _fork_table(c):
    return 3 * c["beams"] * sum(-(-n // PAGE) for n in _fork_lengths(c))


def _back(c):
    """rows that a read of the touched blocks takes for each sequence"""
    return -(-(c["rows"] + BLOCK - 1) // BLOCK) * BLOCK


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------

def _codes(shape, g):
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    for part in out.view(-1).split(1 << 26):  # (the normal numbers of a large pool at once would take four times its memory)
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(36).round_().clamp_(-127, 127))
    return out


def _two(e):
    """2^e, exactly (e: integers of a normal number)"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pool(layers, pages, heads, dim, g):
    """pages of K and V as a prompt leaves them: codes of normal values, scales that vary from block to block"""
    return dict(k=_codes((layers, pages, heads, PAGE, dim), g), v=_codes((layers, pages, heads, 4, dim, 16), g),
                k_scale=_two(torch.randint(-6, -3, (layers, pages, heads, PAGE // BLOCK), device="cuda", generator=g)),
                v_scale=_two(torch.randint(-7, -4, (layers, pages, heads, PAGE // BLOCK), device="cuda", generator=g)))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    if c["op"] == "select":
        n, w = c["groups"], c["beams"]
        logits = torch.randn((n * w, c["vocab"]), device="cuda", generator=g).mul_(2.5).to(TYPES[c["dtype"]])
        done = torch.zeros(n * w, dtype=torch.uint8, device="cuda")
        done[torch.randperm(n * w, device="cuda", generator=g)[: c["finished"]]] = 1
        return dict(c=c, logits=logits, scores=-8 * torch.rand((n, w), device="cuda", generator=g), done=done.view(n, w), eos=2 % c["vocab"])
    if c["op"] == "fork":
        lens, w = _fork_lengths(c), c["beams"]
        most = -(-max(lens) // PAGE) + 1
        # beams of a group share the full pages of their prompt and own the last one
        used = sum(n // PAGE for n in lens) + sum(w for n in lens if n % PAGE)
        pages = used + c["groups"] * w + 3
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        at, rows = 0, []
        for n in lens:
            full = list(range(at, at + n // PAGE))
            at += len(full)
            for b in range(w):
                last = [at] if n % PAGE else []
                at += len(last)
                rows.append(full + last + [-1] * (most - len(full) - len(last)))
        idx = _ints(rows)
        table = torch.where(idx >= 0, order[idx.clamp(min=0).long()], idx)
        parents = []
        for k in range(c["groups"]):
            p = torch.randperm(w, device="cuda", generator=g)[: c["survivors"]]
            parents.append(torch.cat([p, p.repeat(w)[: w - c["survivors"]]]).sort().values + k * w)
        refs = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
        refs.index_add_(0, torch.where(table >= 0, table, pages).view(-1).long(), torch.ones(table.numel(), dtype=torch.int32, device="cuda"))
        return dict(c=c, table=table, lens=_ints([n for n in lens for b in range(w)]), refs=refs[:pages].contiguous(), parents=torch.cat(parents).to(torch.int32),
                    **_pool(c["layers"], pages, c["kv_heads"], c["head_dim"], g))
    if c["op"] == "compact":
        live, moved, pages = c["live"], c["moved"], c["pages"]
        low, high = torch.randperm(live, device="cuda", generator=g), torch.randperm(pages - live, device="cuda", generator=g) + live
        kept = torch.cat([low[moved:], high[:moved]])
        kept = kept[torch.randperm(live, device="cuda", generator=g)].to(torch.int32)
        most = -(-live // c["rows"])
        table = torch.full((c["rows"], most + 2), -1, dtype=torch.int32, device="cuda")
        flat = torch.full((c["rows"] * most,), -1, dtype=torch.int32, device="cuda")
        flat[:live] = kept
        table[:, :most] = flat.view(c["rows"], most)
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[kept.long()] = 1
        return dict(c=c, table=table, refs=refs, **_pool(c["layers"], pages, c["kv_heads"], c["head_dim"], g))
    lens, rows = _lengths(c), _rows(c)
    need = [-(-n // PAGE) for n in lens]
    most, pages = max(need), sum(need) + 2
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = torch.arange(most, device="cuda")
    has = at[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(has, order[torch.where(has, first[:, None] + at[None], 0)], -1).to(torch.int32)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    s = dict(c=c, table=table, lens=_ints(lens), starts=_ints(starts), total=starts[-1], **_pool(1, pages, c["kv_heads"], c["head_dim"], g))
    real = lambda heads: torch.randn((starts[-1], heads, c["head_dim"]), device="cuda", generator=g)  # noqa: E731
    if c["op"] == "append":
        # new rows somewhat larger than what the blocks hold, now and then a large one
        s["new_k"], s["new_v"] = (real(c["kv_heads"]).mul_(m).to(TYPES[c["dtype"]]) for m in (1.3, 0.7))
        s["from"] = _ints([(n - r) // BLOCK * BLOCK for n, r in zip(lens, rows)])
    else:
        s["q"] = real(c["q_heads"]).to(TYPES[c["dtype"]])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _PLAIN[state["c"]["op"]](state)


def _own(s):
    from calm_amd import paged

    c = s["c"]
    if c["op"] == "select":
        return paged.beam_select(s["logits"], s["scores"], s["done"], eos=s["eos"])
    if "pool" not in s:  # the handles that a program keeps beside its cache and its batch
        s["pool"] = paged.KvPool.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if "starts" in s:
            s["batch"] = paged.KvBatch(s["table"], s["lens"], s["starts"], rows=s["total"], max_rows=c["rows"], max_len=c["length"])
    if c["op"] == "append":
        paged.append(s["pool"], s["batch"], s["new_k"], s["new_v"])
        return paged.read(s["pool"], s["table"], s["lens"], s["from"], _back(c))
    if c["op"] == "attend":
        return paged.attend(s["pool"], s["batch"], s["q"], window=c["window"], sinks=c["sinks"])
    if c["op"] == "fork":
        return (*paged.fork(s["pool"], s["table"], s["lens"], s["refs"], s["parents"]), s["k"], s["v"], s["k_scale"], s["v_scale"])
    return (*paged.compact(s["pool"], s["table"], s["refs"]), s["k"], s["v"], s["k_scale"], s["v_scale"])


def _page_rows(s, table):
    """codes and scales of the pages of a table, token by token: (seqs, tokens, heads, dim) and (seqs, blocks, heads), for K and for V"""
    n, m = table.shape
    p = table.clamp(min=0).long()
    k, v = s["k"][0][p], s["v"][0][p]  # (n, m, heads, 64, dim), (n, m, heads, 4, dim, 16)
    heads, dim = k.shape[2], k.shape[4]
    k = k.permute(0, 1, 3, 2, 4).reshape(n, m * PAGE, heads, dim)
    # a V page keeps, for four tokens of each block and a dim, 16 bytes: (token / 4 % 4, dim, (block, token % 4))
    v = v.view(n, m, heads, 4, dim, 4, 4).permute(0, 1, 5, 3, 6, 2, 4).reshape(n, m * PAGE, heads, dim)
    ks, vs = (s[x][0][p].permute(0, 1, 3, 2).reshape(n, m * 4, heads) for x in ("k_scale", "v_scale"))
    return k, v, ks, vs


def _row_index(s, most):
    """(seqs, most): which row of the packed rows is the i-th new one of its sequence, and whether there is one"""
    first, n = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(most, device="cuda")
    has = i[None] < n[:, None]
    return torch.where(has, first[:, None] + i[None], 0), has, n


def _plain_append(s):
    c = s["c"]
    back = _back(c)
    lens, start = s["lens"].long(), s["from"].long()
    _, _, n = _row_index(s, 1)
    before = lens - n
    pos = start[:, None] + torch.arange(back, device="cuda")[None]  # (seqs, back): absolute positions from the first touched block on
    live = pos < lens[:, None]
    is_new = live & (pos >= before[:, None])
    is_old = pos < before[:, None]
    page = s["table"].gather(1, (pos // PAGE).clamp(max=s["table"].shape[1] - 1)).clamp(min=0).long()
    src = torch.where(is_new, s["starts"][:-1].long()[:, None] + pos - before[:, None], 0)
    heads, dim = c["kv_heads"], c["head_dim"]
    t = pos % PAGE
    b = t // BLOCK
    out = []
    for name, new in (("k", s["new_k"]), ("v", s["new_v"])):
        codes, scale = s[name][0], s[name + "_scale"][0]
        h = torch.arange(heads, device="cuda")
        if name == "k":
            at = (page[:, :, None], h[None, None], t[:, :, None])
            view = codes
        else:
            view = codes.view(-1, heads, 4, dim, 4, 4).permute(0, 1, 4, 2, 5, 3)  # (page, head, block, token / 4 % 4, token % 4, dim)
            at = (page[:, :, None], h[None, None], b[:, :, None], (t // 4 % 4)[:, :, None], (t % 4)[:, :, None])
        old = view[at].float()  # (seqs, back, heads, dim)
        x = torch.where(is_new[:, :, None, None], new[src].float(), 0)
        blocks = lambda y: y.view(y.shape[0], back // BLOCK, BLOCK, *y.shape[2:])  # noqa: E731
        m, e = torch.frexp(blocks(x.abs().amax(3)).amax(2))  # the largest of a block, m in [1/2, 1)
        e = torch.where(m > 0, torch.where(m * 128 <= 127, e - 7, e - 6), -126).clamp(min=-126)
        at_block = (page[:, ::BLOCK, None], h[None, None], b[:, ::BLOCK, None])
        was = torch.frexp(scale[at_block])[1] - 1
        e = torch.where(blocks(is_old)[:, :, 0, None], torch.maximum(e, was), e).repeat_interleave(BLOCK, 1)
        was = was.repeat_interleave(BLOCK, 1)
        fresh = torch.where(is_new[:, :, None, None], x * _two(-e)[..., None], old * _two((was - e).clamp(min=-126))[..., None]).round()
        one = _two(e)
        keep = live[:, :, None, None]
        # positions that are not live write to no page of a sequence: their rows are left out
        sel = live.view(-1)
        flat = [torch.broadcast_to(a, (*live.shape, heads)).reshape(-1, heads)[sel] for a in at]
        view[tuple(flat)] = fresh.view(-1, heads, dim)[sel].to(torch.int8)
        first = live[:, ::BLOCK].reshape(-1)
        flat = [torch.broadcast_to(a, (live.shape[0], back // BLOCK, heads)).reshape(-1, heads)[first] for a in at_block]
        scale[tuple(flat)] = one[:, ::BLOCK].reshape(-1, heads)[first]
        out.append(torch.where(keep, fresh * one[..., None], 0))
    return tuple(out)


def _plain_attend(s):
    c = s["c"]
    k, v, ks, vs = _page_rows(s, s["table"])
    n, length, heads, dim = k.shape
    k = k.float() * ks.repeat_interleave(BLOCK, 1)[..., None]
    v = v.float() * vs.repeat_interleave(BLOCK, 1)[..., None]
    idx, has, count = _row_index(s, c["rows"])
    most, group = c["rows"], c["q_heads"] // heads
    q = s["q"].float()[idx].view(n, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n * heads, group * most, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).reshape(n * heads, dim, length)).mul_(dim ** -0.5).view(n, heads, group, most, length)
    p = (s["lens"].long() - count)[:, None] + torch.arange(most, device="cuda")[None]
    j = torch.arange(length, device="cuda")
    seen = j[None, None] <= p[..., None]
    if c["window"]:
        seen = seen & ((j[None, None] > p[..., None] - c["window"]) | (j < c["sinks"])[None, None])
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(n * heads, group * most, length), v.permute(0, 2, 1, 3).reshape(n * heads, length, dim))
    out = (out / total.view(n * heads, group * most, 1)).view(n, heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, c["q_heads"], dim)
    return out[has].to(s["q"].dtype)


def _plain_fork(s):
    table, lens, refs, parents = s["table"], s["lens"].long(), s["refs"], s["parents"].long()
    rows, most = table.shape
    pages = refs.shape[0]
    dev = torch.arange(rows, device="cuda")
    took = table[parents].clone()
    n = lens[parents]
    # the first child of a parent keeps its last page; the others get one of their own where it is not full
    first = torch.full((rows,), rows, device="cuda").scatter_reduce_(0, parents, dev, "amin")[parents] == dev
    col = torch.arange(most, device="cuda")
    took = torch.where(~first[:, None] & (col[None] >= (n // PAGE)[:, None]), -1, took)
    count = lambda t: torch.zeros(pages + 1, dtype=torch.int32, device="cuda").index_add_(  # noqa: E731
        0, torch.where(t >= 0, t, pages).view(-1).long(), torch.ones(t.numel(), dtype=torch.int32, device="cuda"))[:pages]
    now = refs - count(table) + count(took)
    want = ~first & (n % PAGE > 0)
    free = torch.sort((now > 0).to(torch.int32), stable=True).indices
    fresh = free[torch.where(want, want.cumsum(0) - 1, 0)]
    at = (n // PAGE).clamp(max=most - 1)
    src = table[parents].gather(1, at[:, None])[:, 0].long()[want]
    dst = fresh[want]
    took[want, at[want]] = dst.to(torch.int32)
    now[dst] = 1
    for x in ("k", "v", "k_scale", "v_scale"):
        s[x][:, dst] = s[x][:, src]
    return took, now, s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.shape[0], device="cuda")
    src, dst = at[live & (at >= n)], at[~live & (at < n)]
    to = at.clone()
    to[src] = dst
    now = refs.clone()
    now[dst] = refs[src]
    now[src] = 0
    for x in ("k", "v", "k_scale", "v_scale"):
        s[x][:, dst] = s[x][:, src]
    return torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table), now, n.to(torch.int32).view(1), s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_select(s):
    x, (n, w) = s["logits"].double(), s["scores"].shape  # 64 bits: candidates of two beams that are nearly equal keep their order
    vocab, eos = x.shape[1], s["eos"]
    top = x.amax(1, keepdim=True)
    total = x - top - torch.exp(x - top).sum(1, keepdim=True).log() + s["scores"].double().view(-1, 1)
    done = (s["done"].view(-1, 1) != 0)
    total = torch.where(done, float("-inf"), total)
    total[:, eos] = torch.where(done[:, 0], s["scores"].double().view(-1), total[:, eos])
    best, at = torch.sort(total.view(n, w * vocab), dim=1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    parent, token = at // vocab, at % vocab
    ended = (s["done"].gather(1, parent) != 0) | (token == eos)
    return best.float(), parent.to(torch.int32), token.to(torch.int32), ended.to(torch.uint8)


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact, "select": _plain_select}


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attend":
        return _exact_attend(c, s)
    if c["op"] == "append":
        return _exact_append(c, s)
    if c["op"] == "select":
        logp = s["logits"].double().log_softmax(1).view(c["groups"], c["beams"], c["vocab"])
        total = logp + s["scores"].double()[..., None]
        for g, b in s["done"].nonzero().tolist():
            total[g, b] = -float("inf")
            total[g, b, s["eos"]] = s["scores"][g, b].double()
        return total.flatten(1).topk(c["beams"], dim=1).values, None, None, None
    return None  # pages are moved, not computed


def _token(s, name, page, t):
    """values of tokens `t` of pages `page` in 64 bits: (tokens, heads, dim)"""
    if name == "k":
        codes = s["k"][0, page, :, t].double()
    else:
        codes = s["v"][0, page, :, t % 16 // 4]  # (tokens, heads, dim, 16)
        codes = codes.gather(3, (t // 16 * 4 + t % 4)[:, None, None, None].expand(-1, codes.shape[1], codes.shape[2], 1))[..., 0].double()
    return codes * s[name + "_scale"][0, page, :, t // 16].double()[..., None]


def _exact_attend(c, s):
    out = torch.empty((s["total"], c["q_heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
    group, at = c["q_heads"] // c["kv_heads"], 0
    for i, (n, r) in enumerate(zip(_lengths(c), _rows(c))):
        j = torch.arange(n, device="cuda")
        page = s["table"][i].long()[j // PAGE]
        k, v = (_token(s, x, page, j % PAGE).repeat_interleave(group, 1).permute(1, 0, 2).contiguous() for x in ("k", "v"))
        for lo in range(0, r, 512):
            hi = min(r, lo + 512)
            q = s["q"][at + lo:at + hi].double().permute(1, 0, 2).contiguous()
            p = torch.arange(n - r + lo, n - r + hi, device="cuda")[:, None]
            far = (p - j[None] < c["window"]) | (j[None] < c["sinks"]) if c["window"] else torch.ones_like(p - j[None], dtype=torch.bool)
            w = torch.where((j[None] <= p) & far, torch.bmm(q, k.transpose(1, 2).contiguous()) / c["head_dim"] ** 0.5, -float("inf")).softmax(-1)
            out[at + lo:at + hi] = torch.bmm(w, v).permute(1, 0, 2)
        at += r
    return out


def _exact_append(c, s):
    back, got = _back(c), []
    for name in ("k", "v"):
        out = torch.zeros((c["seqs"], back, c["kv_heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
        at = 0
        for i, (n, r) in enumerate(zip(_lengths(c), _rows(c))):
            first = (n - r) // BLOCK * BLOCK
            keep = n - r - first
            x = torch.zeros((back, c["kv_heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
            x[keep:n - first] = s["new_" + name][at:at + r].double()
            e = torch.ceil(torch.log2(x.abs().amax(2).view(-1, BLOCK, c["kv_heads"]).amax(1) / 127).clamp(min=-126)).to(torch.int64)
            step = ((e + 1023) << 52).view(torch.float64)  # 2^e, exactly: (blocks, heads)
            if keep:
                j = torch.arange(first, n - r, device="cuda")
                page = s["table"][i].long()[j // PAGE]
                x[:keep] = _token(s, name, page, j % PAGE)
                step[0] = torch.maximum(step[0], s[name + "_scale"][0, page[0], :, first % PAGE // BLOCK].double())
            step = step.repeat_interleave(BLOCK, 0)[..., None]
            out[i] = torch.round(x / step) * step
            at += r
        got.append(out)
    return tuple(got)
