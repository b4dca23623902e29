"""Workloads of the operators that address rows and pages through an index: the embedding lookup and its gradient
over the tokens of one or several ranks, and the page operations of a cache (copy, fork, free and extend, compact).

Every case is a dict of plain values.  `run` computes the operator in elementary torch operations where `own` is
false, and through dfccl_amd's entry points where it is true."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SHUFFLE = 1000003  # a prime above every vocabulary here: multiplication by it permutes the ids
IDS = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # one decode step of a small server: eight sequences, one token each
        dict(name="lookup of 8 tokens", op="lookup", vocab=32000, first=0, rows=32000, tokens=8, width=4096, pad=0,
             table="bf16", out="bf16", ids="i64", scale=64.0),
        # a training batch that reads a 32-bit master table into bfloat16 activations
        dict(name="lookup of 16385 tokens", op="lookup", vocab=131072, first=0, rows=131072, tokens=16385, width=4096,
             pad=0, table="f32", out="bf16", ids="i64", scale=1.0),
        # four data-parallel ranks' short ragged batches, summed into one rank's piece of the vocabulary
        # (gradient accumulation over micro-batches, 32-bit gradients)
        dict(name="gradient of 4 ranks, a piece", op="grad", vocab=50000, first=0, rows=12500, ranks=4, tokens=1001,
             width=1000, pad=0, grad="f16", table="f32", ids="i32", scale=0.25, padding=0.1, accumulate=True),
        # the whole table's gradient after one long batch
        dict(name="gradient of 16384 tokens", op="grad", vocab=131072, first=0, rows=131072, ranks=1, tokens=16384,
             width=4096, pad=0, grad="bf16", table="bf16", ids="i64", scale=64.0, padding=0.0, accumulate=False),
        # one prompt's three pages, 24 layers of keys and values, handed to another rank's cache
        dict(name="copy of 3 pages", op="copy", pools=48, pages=64, page_tokens=16, row=512, type="bf16", pairs=3),
        # a long prompt's pages, 32 layers of keys and values
        dict(name="copy of 300 pages", op="copy", pools=64, pages=512, page_tokens=16, row=1024, type="bf16",
             pairs=300),
        # one prompt answered four times
        dict(name="fork of 1 prompt into 4", op="fork", pools=48, pages=512, page_tokens=16, row=512, type="bf16",
             seqs=32, per_seq=128, prompts=1, forks=4, longest=1100),
        # a batch of prompts, sixteen samples each
        dict(name="fork of 32 prompts into 512", op="fork", pools=8, pages=8192, page_tokens=16, row=512, type="bf16",
             seqs=600, per_seq=256, prompts=32, forks=16, longest=3000),
        # between two decode steps of a small server: two sequences end, one is admitted, the others grow by a token
        dict(name="turn of 16 sequences", op="turn", pools=2, pages=2048, page_tokens=16, row=128, type="bf16",
             seqs=17, per_seq=128, running=16, ended=2, admitted=1, longest=1500),
        # the same for a large one, with admissions of whole prompts
        dict(name="turn of 2000 sequences", op="turn", pools=2, pages=262144, page_tokens=16, row=64, type="bf16",
             seqs=2400, per_seq=512, running=2000, ended=300, admitted=300, longest=3000),
        # a small cache before it is handed on, 8-bit values
        dict(name="compaction of 256 pages", op="compact", pools=16, pages=256, page_tokens=32, row=256, type="i8",
             seqs=24, per_seq=64, running=20, ended=10, longest=300),
        # a large one of which half has been freed
        dict(name="compaction of 4096 pages", op="compact", pools=16, pages=4096, page_tokens=16, row=512, type="bf16",
             seqs=128, per_seq=128, running=64, ended=32, longest=1500),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("lookup", "grad", "grad", "copy", "fork", "turn", "compact"))
    if op in ("lookup", "grad"):
        vocab = _spread(rng, 1000, 131072)
        pieces = rng.choice((1, 1, 2, 4, 7))
        rows = -(-vocab // pieces)
        first = rows * rng.randrange(pieces)
        rows = max(1, min(rows, vocab - first))
        width = min(rng.choice((_spread(rng, 64, 4096), 8 * _spread(rng, 8, 512))), (1 << 28) // rows)
        pad = rng.choice((0, 0, 0, 1, 8, 24))
        out = rng.choice(("bf16", "f16", "f32"))
        case = dict(op=op, vocab=vocab, first=first, rows=rows, width=width, pad=pad, ids=rng.choice(("i32", "i64")),
                    scale=rng.choice((1.0, 0.125, math.sqrt(width))))
        if op == "lookup":
            return dict(case, tokens=_spread(rng, 1 if pieces == 1 else 32, 16384), table=rng.choice((out, "f32")), out=out)
        ranks = rng.choice((1, 1, 2, 3, 8))
        accumulate, padding = rng.random() < 0.4, rng.choice((0.0, 0.1, 0.5))
        fewest = 1 if pieces == 1 and padding == 0 else 64
        return dict(case, ranks=ranks, tokens=_spread(rng, fewest, 16384 // ranks), grad=out,
                    table="f32" if accumulate else rng.choice((out, "f32")), padding=padding, accumulate=accumulate)
    page_tokens = rng.choice((1, 8, 16, 32, 64))
    row = rng.choice((64, 576, 1024, rng.randrange(33, 700)))
    kind = rng.choice(("bf16", "f16", "f32", "i8"))
    pools = _spread(rng, 1, 130)
    if op == "turn":
        running = _spread(rng, 2, 2000)
        per_seq = _spread(rng, 4, 512)
        longest = max(2, int(0.8 * per_seq * page_tokens))
        return dict(op=op, pools=2, pages=running * per_seq + per_seq * 8, page_tokens=page_tokens, row=1,
                    type=kind, seqs=running + 40, per_seq=per_seq, running=running, ended=rng.randrange(1, running),
                    admitted=rng.randrange(0, 8), longest=longest)
    most = max(48, min(8192, 250_000_000 // (pools * page_tokens * row)))  # pages, so that pools stay near 0.5 GB
    if op == "copy":
        pages = _spread(rng, 24, most)
        return dict(op=op, pools=pools, pages=pages, page_tokens=page_tokens, row=row, type=kind,
                    pairs=_spread(rng, 1, max(1, pages // 2)))
    if op == "fork":
        forks, prompts = rng.randrange(1, 9), _spread(rng, 1, max(1, most // 40))
        per_seq = max(2, (most - prompts * forks) // prompts)
        per_seq = _spread(rng, 2, min(256, per_seq))
        return dict(op=op, pools=pools, pages=prompts * (per_seq + forks) + 5, page_tokens=page_tokens, row=row, type=kind,
                    seqs=prompts * (1 + forks) + 3, per_seq=per_seq, prompts=prompts, forks=forks,
                    longest=per_seq * page_tokens)
    running = _spread(rng, 2, 64)
    per_seq = max(1, min(128, most // running))
    return dict(op=op, pools=pools, pages=running * per_seq + 3, page_tokens=page_tokens, row=row, type=kind,
                seqs=running + 5, per_seq=per_seq, running=running, ended=rng.randrange(1, running + 1),
                longest=per_seq * page_tokens)


# ---- inputs ---------------------------------------------------------------------------------------------------

class State:
    """What a user's program holds: tensors, and for the pages the handle of the cache."""


def _ids(case, tokens, g):
    """Token ids as text has them: the r-th most frequent one with a probability of about 1 / r, the frequent ones
    anywhere in the vocabulary."""
    u = torch.rand(tokens, device=DEVICE, generator=g, dtype=torch.float64)
    r = (torch.exp(u * math.log(case["vocab"] + 1)) - 1).long().clamp_(0, case["vocab"] - 1)
    return r * SHUFFLE % case["vocab"]


def _normal(shape, dtype, g):
    if dtype == torch.int8:
        return torch.randint(-128, 128, shape, device=DEVICE, generator=g, dtype=dtype)
    return torch.randn(shape, device=DEVICE, generator=g, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16
                       ).to(dtype)


def _rows(count, case, dtype, g):
    """count rows of the case's width, `pad` elements apart where it says so."""
    return _normal((count, case["width"] + case["pad"]), dtype, g)[:, :case["width"]]


def _prepare_rows(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = State()
    s.case = case
    if case["op"] == "lookup":
        s.table = _rows(case["rows"], case, TYPES[case["table"]], g)
        s.ids = _ids(case, case["tokens"], g).to(IDS[case["ids"]])
        s.out = torch.empty((case["tokens"], case["width"]), device=DEVICE, dtype=TYPES[case["out"]])
        return s
    # ranks' batches are ragged: each one a little shorter than the one before
    counts = [max(1, case["tokens"] - r * (case["tokens"] // 16)) for r in range(case["ranks"])]
    s.padding_id = case["vocab"] - 1
    s.grads = [_rows(n, case, TYPES[case["grad"]], g) for n in counts]
    s.ids = []
    for n in counts:
        ids = _ids(case, n, g)
        ids[n - int(n * case["padding"]):] = s.padding_id
        s.ids.append(ids.to(IDS[case["ids"]]))
    s.table_grad = _rows(case["rows"], case, TYPES[case["table"]], g)
    return s


def _fill(case, rs, sequences, lengths, refcounts, tables, shared=0):
    """Gives the sequences their pages, out of a shuffled order; the first `shared` of them share the first one's
    whole pages."""
    order, at, pt = rs.permutation(case["pages"]), 0, case["page_tokens"]
    for k, q in enumerate(sequences):
        n = -(-int(lengths[q]) // pt)
        same = 0
        if 0 < k < shared:
            same = min(int(lengths[q]) // pt, int(lengths[sequences[0]]) // pt)
            tables[q, :same] = tables[sequences[0], :same]
        tables[q, same:n] = order[at:at + n - same]
        at += n - same
        np.add.at(refcounts, tables[q, :n], 1)


def _prepare_pages(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    s = State()
    s.case = case
    op, pt = case["op"], case["page_tokens"]
    s.pools = _normal((case["pools"], case["pages"], pt * case["row"]), TYPES[case["type"]], g)
    seqs, per_seq = case.get("seqs", 1), case.get("per_seq", 1)
    refcounts = np.zeros(case["pages"], np.int32)
    tables = np.full((seqs, per_seq), -1, np.int32)
    lengths = np.zeros(seqs, np.int32)
    lists = {}
    if op == "copy":
        s.source = _normal(s.pools.shape, TYPES[case["type"]], g)
        lists = dict(src=rs.permutation(case["pages"])[:case["pairs"]], dst=rs.permutation(case["pages"])[:case["pairs"]])
    else:
        slots = rs.permutation(seqs)
        used = slots[:case["prompts"] if op == "fork" else case["running"]]
        longest = min(case["longest"], per_seq * pt)
        lengths[used] = rs.randint(max(1, longest // 4), longest + 1, len(used))
        _fill(case, rs, used, lengths, refcounts, tables, shared=0 if op == "fork" else len(used) // 4)
        if op == "fork":
            lists = dict(parents=np.repeat(used, case["forks"]),
                         children=slots[len(used):len(used) * (1 + case["forks"])])
        else:
            ended = used[rs.permutation(len(used))[:case["ended"]]]
            if op == "turn":
                staying = np.setdiff1d(used, ended)
                new = slots[len(used):len(used) + case["admitted"]]
                grown = np.minimum(lengths[staying] + 1, per_seq * pt)
                lists = dict(ended=ended, growing=np.concatenate([staying, new]),
                             lengths=np.concatenate([grown, rs.randint(1, longest + 1, len(new))]))
            else:
                for q in ended:
                    n = -(-int(lengths[q]) // pt)
                    np.add.at(refcounts, tables[q, :n], -1)
                    tables[q], lengths[q] = -1, 0
    # the cache's bookkeeping in one buffer, so that a pass can begin from the same state with one copy
    s.book = torch.from_numpy(np.concatenate([refcounts, tables.reshape(-1), lengths])).to(DEVICE)
    s.saved = s.book.clone()
    s.refcounts, s.tables, s.lengths = s.book.split([case["pages"], seqs * per_seq, seqs])
    s.tables = s.tables.view(seqs, per_seq)
    s.lists = {k: torch.from_numpy(v.astype(np.int32)).to(DEVICE) for k, v in lists.items()}
    if own:
        import dfccl_amd
        books = (s.refcounts, s.tables, s.lengths)
        s.cache = dfccl_amd.PageCache(list(s.pools.unbind(0)), pt, *books)
        s.other = dfccl_amd.PageCache(list(s.source.unbind(0)), pt, *books) if op == "copy" else None
    return s


def prepare(case, seed):
    return _prepare_rows(case, seed) if case["op"] in ("lookup", "grad") else _prepare_pages(case, seed)


# ---- the plain forms ------------------------------------------------------------------------------------------

def _plain_lookup(s):
    case = s.case
    r = s.ids.long() - case["first"]
    inside = (r >= 0) & (r < case["rows"])
    rows = s.table[torch.where(inside, r, 0)].float() * case["scale"]
    return torch.where(inside[:, None], rows, 0.0).to(s.out.dtype)


def _plain_grad(s):
    case = s.case
    ids = torch.cat(s.ids).long()
    r = ids - case["first"]
    counts = (r >= 0) & (r < case["rows"]) & (ids != s.padding_id)
    total = torch.zeros((case["rows"] + 1, case["width"]), device=DEVICE)
    total.index_add_(0, torch.where(counts, r, case["rows"]), torch.cat(s.grads).float())
    total = total[:case["rows"]] * case["scale"]
    s.table_grad.copy_(s.table_grad.float() + total if case["accumulate"] else total)
    return s.table_grad


def _plain_copy(s):
    s.pools[:, s.lists["dst"].long()] = s.source[:, s.lists["src"].long()]


def _pages_of(s, lengths):
    return (lengths + s.case["page_tokens"] - 1) // s.case["page_tokens"]


def _count(s, pages, used, by):
    """Adds `by` to the reference count of every used entry of `pages`."""
    more = torch.zeros(s.case["pages"] + 1, device=DEVICE, dtype=torch.int32)
    at = torch.where(used, pages, s.case["pages"]).reshape(-1).long()
    more.index_add_(0, at, torch.full_like(at, by, dtype=torch.int32))
    s.refcounts += more[:-1]


def _plain_fork(s):
    case, pt = s.case, s.case["page_tokens"]
    parents, children = s.lists["parents"].long(), s.lists["children"].long()
    lengths = s.lengths[parents]
    whole, need = lengths // pt, (lengths % pt != 0).int()
    free = torch.nonzero(s.refcounts == 0)[:, 0]
    taken = torch.cumsum(need, 0)
    served = taken <= free.numel()
    copies = torch.nonzero(served & (need != 0))[:, 0]
    new = free[taken[copies].long() - 1]
    rows = s.tables[parents]
    columns = torch.arange(case["per_seq"], device=DEVICE)
    used = (columns < whole[:, None]) & served[:, None]
    last = rows[copies, whole[copies].long()].long()
    s.pools[:, new] = s.pools[:, last]
    _count(s, rows, used, 1)
    s.refcounts[new] = 1
    child = torch.where(used, rows, -1)
    child[copies, whole[copies].long()] = new.int()
    s.tables[children] = child
    s.lengths[children] = torch.where(served, lengths, 0)


def _plain_free(s, sequences):
    used = torch.arange(s.case["per_seq"], device=DEVICE) < _pages_of(s, s.lengths[sequences])[:, None]
    _count(s, s.tables[sequences], used, -1)
    s.tables[sequences] = -1
    s.lengths[sequences] = 0


def _plain_extend(s, sequences, lengths):
    have, want = _pages_of(s, s.lengths[sequences]), _pages_of(s, lengths)
    free = torch.nonzero(s.refcounts == 0)[:, 0]
    taken = torch.cumsum(want - have, 0)
    served = taken <= free.numel()
    columns = torch.arange(s.case["per_seq"], device=DEVICE)
    new = (columns >= have[:, None]) & (columns < want[:, None]) & served[:, None]
    at = (taken - want)[:, None] + columns
    pages = free[torch.where(new, at, 0)].int()
    s.tables[sequences] = torch.where(new, pages, s.tables[sequences])
    s.refcounts[pages[new].long()] = 1
    s.lengths[sequences] = torch.where(served, lengths, s.lengths[sequences])


def _plain_compact(s):
    live = s.refcounts > 0
    below = torch.arange(s.case["pages"], device=DEVICE) < live.sum()
    holes, movers = torch.nonzero(~live & below)[:, 0], torch.nonzero(live & ~below)[:, 0]
    s.pools[:, holes] = s.pools[:, movers]
    moved = torch.arange(s.case["pages"], device=DEVICE, dtype=torch.int32)
    moved[movers] = holes.int()
    s.tables.copy_(torch.where(s.tables >= 0, moved[s.tables.long().clamp(min=0)], -1))
    s.refcounts[holes] = s.refcounts[movers]
    s.refcounts[movers] = 0


def run(s):
    case, op = s.case, s.case["op"]
    if op == "lookup":
        if not own:
            return _plain_lookup(s)
        import dfccl_amd
        dfccl_amd.embedding_lookup(s.table, s.ids, s.out, scale=case["scale"], first_row=case["first"])
        return s.out
    if op == "grad":
        if not own:
            return _plain_grad(s)
        import dfccl_amd
        dfccl_amd.embedding_grad(s.grads, s.ids, s.table_grad, scale=case["scale"], first_row=case["first"],
                                 padding_id=s.padding_id, accumulate=case["accumulate"])
        return s.table_grad
    if op == "copy":
        if own:
            s.cache.copy(s.lists["src"], s.lists["dst"], source=s.other)
        else:
            _plain_copy(s)
        return s.pools
    # the bookkeeping as it was before the pass (page contents only ever move into pages that were free)
    s.book.copy_(s.saved)
    if op == "fork":
        if own:
            s.cache.fork(s.lists["parents"], s.lists["children"])
        else:
            _plain_fork(s)
    elif op == "turn":
        if own:
            s.cache.free(s.lists["ended"])
            s.cache.extend(s.lists["growing"], s.lists["lengths"])
        else:
            _plain_free(s, s.lists["ended"].long())
            _plain_extend(s, s.lists["growing"].long(), s.lists["lengths"])
        return s.book
    elif own:
        s.cache.compact()
    else:
        _plain_compact(s)
    return s.pools, s.book


# ---- what a pass cannot do without ----------------------------------------------------------------------------

def _distinct(case, tokens):
    """Expected number of different rows of the piece among so many tokens."""
    r = torch.arange(case["vocab"])
    at = r * SHUFFLE % case["vocab"] - case["first"]
    r = r[(at >= 0) & (at < case["rows"])].double()
    p = (torch.log(r + 2) - torch.log(r + 1)) / math.log(case["vocab"] + 1)
    return float((1 - (1 - p) ** tokens).sum()), float(p.sum())


def work(case):
    op = case["op"]
    if op in ("lookup", "grad"):
        idsize, w = IDS[case["ids"]].itemsize, case["width"]
        tokens = case["tokens"] if op == "lookup" else sum(
            max(1, case["tokens"] - r * (case["tokens"] // 16)) for r in range(case["ranks"]))
        if op == "lookup":
            rows, _ = _distinct(case, tokens)
            return {"bytes": tokens * idsize + rows * w * TYPES[case["table"]].itemsize
                    + tokens * w * TYPES[case["out"]].itemsize, "flops": tokens * w}
        tokens *= 1 - case["padding"]
        rows, inside = _distinct(case, tokens)
        size = TYPES[case["table"]].itemsize
        table = 2 * rows * w * size if case["accumulate"] else case["rows"] * w * size
        return {"bytes": tokens * (idsize + inside * w * TYPES[case["grad"]].itemsize) + table,
                "flops": tokens * inside * w}
    page = case["pools"] * case["page_tokens"] * case["row"] * TYPES[case["type"]].itemsize
    mean = 0.625 * case.get("longest", 0) / case["page_tokens"]  # pages of a sequence, on average
    if op == "copy":
        return {"bytes": 2 * case["pairs"] * page + 8 * case["pairs"], "flops": 0}
    if op == "fork":
        n = case["prompts"] * case["forks"]
        partial = (case["page_tokens"] - 1) / case["page_tokens"]
        return {"bytes": n * (2 * partial * page + 16 * mean) + 4 * case["pages"], "flops": 0}
    if op == "turn":
        return {"bytes": 16 * mean * (case["ended"] + case["admitted"]) + 16 * case["running"] + 4 * case["pages"],
                "flops": 0}
    live = min(1.0, mean * (case["running"] - case["ended"]) / case["pages"])
    return {"bytes": 2 * live * (1 - live) * case["pages"] * page + 8 * case["pages"]
            + 8 * mean * (case["running"] - case["ended"]), "flops": 0}


# ---- the definitions in 64 bits, by themselves ----------------------------------------------------------------

def _exact_pages(case, s):
    """The bookkeeping on the host, one request after another; the contents follow the list of moves it leaves."""
    op, pt = case["op"], case["page_tokens"]
    refs, tables, lengths = (t.cpu().numpy().astype(np.int64) for t in (s.refcounts, s.tables, s.lengths))
    lists = {k: v.cpu().numpy() for k, v in s.lists.items()}
    moves = []
    if op == "fork":
        free = iter(np.flatnonzero(refs == 0).tolist())
        for p, c in zip(lists["parents"], lists["children"]):
            whole, rest = divmod(int(lengths[p]), pt)
            tables[c, :whole] = tables[p, :whole]
            refs[tables[p, :whole]] += 1
            if rest:
                moves.append((int(tables[p, whole]), next(free)))
                tables[c, whole] = moves[-1][1]
                refs[moves[-1][1]] = 1
            lengths[c] = lengths[p]
    elif op == "turn":
        for q in lists["ended"]:
            refs[tables[q, :-(-int(lengths[q]) // pt)]] -= 1
            tables[q], lengths[q] = -1, 0
        free = iter(np.flatnonzero(refs == 0).tolist())
        for q, n in zip(lists["growing"], lists["lengths"]):
            for k in range(-(-int(lengths[q]) // pt), -(-int(n) // pt)):
                tables[q, k] = next(free)
                refs[tables[q, k]] = 1
            lengths[q] = n
    else:
        alive = np.flatnonzero(refs > 0)
        live = len(alive)
        for src, dst in zip(alive[alive >= live], np.flatnonzero(refs[:live] == 0)):
            moves.append((int(src), int(dst)))
            tables[tables == src] = dst
            refs[dst], refs[src] = refs[src], 0
    return moves, torch.from_numpy(np.concatenate([refs, tables.reshape(-1), lengths]).astype(np.int32)).to(DEVICE)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        out = torch.zeros((case["tokens"], case["width"]), device=DEVICE, dtype=torch.float64)
        at = torch.nonzero((s.ids >= case["first"]) & (s.ids < case["first"] + case["rows"]))[:, 0]
        out[at] = s.table.double().index_select(0, s.ids[at].long() - case["first"]).mul_(case["scale"])
        return out
    if op == "grad":
        out = torch.zeros((case["rows"], case["width"]), device=DEVICE, dtype=torch.float64)
        for grad, ids in zip(s.grads, s.ids):
            at = torch.nonzero((ids >= case["first"]) & (ids < case["first"] + case["rows"]) & (ids != s.padding_id))[:, 0]
            rows = ids[at].long() - case["first"]
            out.index_put_((rows,), grad[at].double() * case["scale"], accumulate=True)
        return out + s.table_grad.double() if case["accumulate"] else out
    pools = s.pools if case["type"] == "i8" else s.pools.double()
    if op == "copy":
        for src, dst in zip(s.lists["src"].tolist(), s.lists["dst"].tolist()):
            pools[:, dst] = s.source[:, src].to(pools.dtype)
        return pools
    moves, book = _exact_pages(case, s)
    if op == "turn":
        return book
    for src, dst in moves:
        pools[:, dst] = pools[:, src].clone()
    return pools, book
