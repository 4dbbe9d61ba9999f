"""Step tables on the GPU against a plain host loop: whole numbers, so equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(seq_blocks, rows, ctx, query, new, bs, num_blocks, T):
    """The header's rules, one request and one token at a time. Returns the outputs and whether anything is reported."""
    num_rows, mb = seq_blocks.shape
    n, bad = len(query), False
    seq_blocks = seq_blocks.copy()
    r_of = rows if rows is not None else np.arange(n)
    table = np.full((n, mb), -1, np.int32)
    cu, lens, last = np.zeros(n + 1, np.int64), np.zeros(n, np.int32), np.zeros(n, np.int32)
    pos, slot = np.zeros(T, np.int32), np.full(T, -1, np.int64)
    used = 0
    ok, had, need, fresh = [], [], [], []
    for i in range(n):
        r, c, q = int(r_of[i]), int(ctx[i]), int(query[i])
        good = c >= 0 and q >= 0 and c + q < 2**31
        h = -(-c // bs) if good else 0
        m = -(-(c + q) // bs) - h if good else 0
        good = good and h + m <= mb
        cu[i + 1] = cu[i] + max(q, 0)
        good = good and r < num_rows and cu[i + 1] <= T
        if r >= 0 and not good:
            bad = True
        fresh.append(used)
        used += m if r >= 0 else 0
        ok.append(good and r >= 0), had.append(h), need.append(m)
    for i in range(n):
        fits = [k for k in range(n) if 0 <= r_of[k] < num_rows and ctx[k] >= 0 and query[k] >= 0
                and had[k] + need[k] <= mb]
        if ok[i] and sum(int(r_of[k]) == int(r_of[i]) for k in fits) > 1:
            ok[i], bad = False, True
    for i in range(n):
        last[i] = max(min(cu[i + 1], T) - 1, 0)
        if not ok[i]:
            continue
        r = int(r_of[i])
        lens[i] = ctx[i] + query[i]
        for c in range(had[i] + need[i]):
            if c < had[i]:
                b = seq_blocks[r, c]
            else:
                k = fresh[i] + c - had[i]
                b = new[k] if k < len(new) else -1
            if b < 0 or b >= num_blocks:
                b, bad = -1, True
            if c >= had[i]:
                seq_blocks[r, c] = b
            table[i, c] = b
        for t in range(query[i]):
            p = ctx[i] + t
            pos[cu[i] + t] = p
            if table[i, p // bs] >= 0:
                slot[cu[i] + t] = int(table[i, p // bs]) * bs + p % bs
    bad = bad or cu[n] > T
    return dict(block_tables=table, cu_seqlens=np.minimum(cu, T).astype(np.int32), seq_lens=lens, positions=pos,
                slot_mapping=slot, last_rows=last, seq_blocks=seq_blocks), bad


def run(ctx, seq_blocks, rows, c, q, new, bs, num_blocks, T, stream=None):
    import torch
    import zealot_b200 as zb
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    n, mb = len(q), seq_blocks.shape[1]
    junk = lambda *s, dtype=torch.int32: torch.full(s, 77, dtype=dtype, device="cuda")
    out = dict(block_tables=junk(n, mb), cu_seqlens=junk(n + 1), seq_lens=junk(n), positions=junk(T),
               slot_mapping=junk(T, dtype=torch.int64), last_rows=junk(n))
    tables = dev(seq_blocks)
    zb.CudaAttention(ctx).step_tables(tables, None if rows is None else dev(rows), dev(c), dev(q), dev(new), *out.values(),
                                      bs, num_blocks, stream=stream)
    return {**{k: t.cpu().numpy() for k, t in out.items()}, "seq_blocks": tables.cpu().numpy()}


def same(got, want):
    for k, w in want.items():
        assert np.array_equal(got[k], w), k


def make(rng, n, bs, mb, with_rows, longest_query):
    q = np.where(rng.random(n) < 0.5, 1, rng.integers(0, longest_query + 1, n)).astype(np.int32)
    c = rng.integers(0, max(1, mb * bs - longest_query + 1), n).astype(np.int32)
    c[rng.random(n) < 0.2] = 0
    q = np.minimum(q, mb * bs - c).astype(np.int32)
    num_rows = n + 5 if with_rows else n
    rows = rng.permutation(num_rows)[:n].astype(np.int32) if with_rows else None
    had = -(-c // bs)
    need = -(-(c + q) // bs) - had
    ids = rng.permutation(int(had.sum() + need.sum()) + 3).astype(np.int32)
    seq_blocks = np.full((num_rows, mb), -5, np.int32)  # what is behind a request's blocks is left as it was
    at = 0
    for i in range(n):
        seq_blocks[i if rows is None else rows[i], :had[i]] = ids[at:at + had[i]]
        at += had[i]
    return seq_blocks, rows, c, q, ids[at:at + need.sum()], len(ids)


@pytest.mark.parametrize("n,bs,mb,with_rows,longest,pad", [
    (1, 16, 1, False, 1, 0), (1, 16, 8, True, 128, 3), (7, 16, 5, True, 33, 0), (64, 16, 257, True, 1, 0),
    (33, 8, 64, False, 300, 17), (5, 1, 9, True, 4, 1), (3, 30, 131, True, 100, 0), (300, 64, 12, True, 200, 40),
    (1000, 16, 129, True, 40, 8), (257, 16, 128, True, 0, 5)])
def test_step_tables(ctx, n, bs, mb, with_rows, longest, pad):
    rng = np.random.default_rng(n * 1000 + mb)
    seq_blocks, rows, c, q, new, num_blocks = make(rng, n, bs, mb, with_rows, longest)
    T = int(q.sum()) + pad
    want, bad = plain(seq_blocks, rows, c, q, new, bs, num_blocks, T)
    assert not bad
    same(run(ctx, seq_blocks, rows, c, q, new, bs, num_blocks, T), want)
    ctx.check_status()


def test_step_tables_most_requests(ctx):
    """8192 requests, the most that a step takes, on another stream than the current one."""
    import torch
    rng = np.random.default_rng(8)
    seq_blocks, rows, c, q, new, num_blocks = make(rng, 8192, 16, 3, True, 2)
    T = int(q.sum())
    want, bad = plain_fast(seq_blocks, rows, c, q, new, 16, num_blocks, T)
    assert not bad
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(ctx, seq_blocks, rows, c, q, new, 16, num_blocks, T)
    same(got, want)
    ctx.check_status()


def plain_fast(seq_blocks, rows, c, q, new, bs, num_blocks, T):
    """plain() without its check for repeated rows, which is quadratic (the rows here are distinct)."""
    parts, used, at = [], 0, 0
    out = dict(block_tables=[], seq_lens=[], positions=[], slot_mapping=[])
    seq_blocks, bad, last = seq_blocks.copy(), False, []
    for i in range(len(q)):
        need = -(-(c[i] + q[i]) // bs) - -(-c[i] // bs)
        one, b = plain(seq_blocks[rows[i]][None], None, c[i:i + 1], q[i:i + 1], new[used:used + need], bs, num_blocks,
                       int(q[i]))
        used += need
        at += int(q[i])
        bad |= b
        last.append(max(at - 1, 0))
        seq_blocks[rows[i]] = one["seq_blocks"][0]
        for k in out:
            out[k].append(one[k])
        parts.append(at)
    out = {k: np.concatenate(v) for k, v in out.items()}
    return dict(out, cu_seqlens=np.array([0] + parts, np.int32), last_rows=np.array(last, np.int32),
                seq_blocks=seq_blocks), bad


BAD = {
    "empty slots": lambda a: a["rows"].__setitem__(slice(0, None, 3), -1),
    "row outside": lambda a: a["rows"].__setitem__(2, 999),
    "row twice": lambda a: a["rows"].__setitem__(4, a["rows"][1]),
    "row three times": lambda a: a["rows"].__setitem__(slice(2, 5), a["rows"][7]),
    "negative context": lambda a: a["c"].__setitem__(3, -4),
    "negative query": lambda a: a["q"].__setitem__(3, -4),
    "huge lengths": lambda a: (a["c"].__setitem__(3, 2**31 - 1), a["q"].__setitem__(3, 2**31 - 1)),
    "table too short": lambda a: a["c"].__setitem__(5, 16 * 40),
    "old id outside": lambda a: a["tables"].__setitem__((a["rows"][6], 0), 10**6),
    "new id outside": lambda a: a["new"].__setitem__(1, 10**6),
    "new id negative": lambda a: a["new"].__setitem__(1, -3),
    "too few new ids": lambda a: a.__setitem__("new", a["new"][:3]),
    "no new ids": lambda a: a.__setitem__("new", a["new"][:0]),
    "too few token rows": lambda a: a.__setitem__("T", a["T"] // 2),
    "no token rows": lambda a: a.__setitem__("T", 0),
}


@pytest.mark.parametrize("what", list(BAD))
def test_step_tables_bad_requests(ctx, what):
    """What cannot be served is reported and left out; the other requests keep their rows, blocks and slots."""
    import zealot_b200 as zb
    rng = np.random.default_rng(5)
    tables, rows, c, q, new, num_blocks = make(rng, 12, 16, 40, True, 60)
    c[6] = max(c[6], 1)
    a = dict(tables=tables, rows=rows, c=c, q=q, new=new, T=int(q.sum()) + 2)
    had = -(-c // 16)
    for i in range(12):  # the changed context needs its blocks too
        a["tables"][rows[i], :had[i]] = np.maximum(a["tables"][rows[i], :had[i]], 0)
    BAD[what](a)
    want, bad = plain(a["tables"], a["rows"], a["c"], a["q"], a["new"], 16, num_blocks, a["T"])
    assert bad == (what != "empty slots")
    same(run(ctx, a["tables"], a["rows"], a["c"], a["q"], a["new"], 16, num_blocks, a["T"]), want)
    if bad:
        with pytest.raises(zb.OobBlockError):
            ctx.check_status()
    ctx.check_status()


def test_step_tables_no_requests(ctx):
    got = run(ctx, np.zeros((0, 4), np.int32), None, [], [], [], 16, 8, 5)
    assert got["cu_seqlens"].tolist() == [0]
    assert got["positions"].tolist() == [0] * 5 and got["slot_mapping"].tolist() == [-1] * 5
    ctx.check_status()


def test_step_tables_overlaps_are_refused(ctx):
    """Outputs on inputs or on one another, the lengths in place above all: every CTA reads them while others write."""
    import torch
    import zealot_b200 as zb
    new = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device="cuda")
    names = ("seq_blocks rows context_lens query_lens new_blocks block_tables cu_seqlens seq_lens positions slot_mapping "
             "last_rows").split()
    shapes = dict(seq_blocks=(4, 4), block_tables=(3, 4), cu_seqlens=(4,), positions=(5,), slot_mapping=(5,))
    make = lambda: {n: new(*shapes.get(n, (3,)), dtype=torch.int64 if n == "slot_mapping" else torch.int32) for n in names}
    attn = zb.CudaAttention(ctx)

    def call(a):
        """A call that is taken; its requests all name row 0, which is reported."""
        attn.step_tables(*(a[n] for n in names), 16, 8)
        with pytest.raises(zb.OobBlockError):
            ctx.check_status()

    call(make())
    a = make()
    call(dict(a, context_lens=a["query_lens"], new_blocks=a["query_lens"]))  # inputs may be the same
    for one, other in (("seq_lens", "context_lens"), ("seq_lens", "query_lens"), ("last_rows", "rows"), ("seq_lens", "new_blocks"),
                       ("seq_lens", "last_rows"), ("last_rows", "query_lens")):
        with pytest.raises(zb.InvalidArgument, match="overlaps"):
            call(dict(a, **{one: a[other]}))
    with pytest.raises(zb.InvalidArgument, match="overlaps"):
        call(dict(a, cu_seqlens=a["positions"][:4]))
    with pytest.raises(zb.InvalidArgument, match="overlaps"):
        call(dict(a, context_lens=a["cu_seqlens"][1:]))
    with pytest.raises(zb.InvalidArgument, match="overlaps"):
        call(dict(a, rows=a["seq_blocks"].view(-1)[13:]))
    with pytest.raises(zb.InvalidArgument, match="overlaps"):
        call(dict(a, positions=a["slot_mapping"].view(torch.int32)[5:]))
    neighbours = new(7)  # side by side is no overlap
    call(dict(a, context_lens=neighbours[:3], cu_seqlens=neighbours[3:]))


@pytest.mark.parametrize("n,bs,mb,with_rows,longest,pad", [
    # more than 512 requests, tables of 16-byte columns (the step of every request's threads, and several steps)
    (700, 16, 132, True, 40, 8), (513, 16, 8, False, 20, 0), (600, 8, 1028, True, 5, 3),
    # rows of more than one stretch: past 2,048 columns of 4 bytes and past 8,192 of 16, few requests and many
    (3, 16, 2051, True, 70, 0), (2, 1, 6001, False, 300, 5), (3, 16, 8196, True, 200, 1), (2, 2, 20000, True, 50, 0),
    (520, 16, 4100, True, 3, 2)])
def test_step_tables_wide_and_many(ctx, n, bs, mb, with_rows, longest, pad):
    rng = np.random.default_rng(n * 1000 + mb)
    seq_blocks, rows, c, q, new, num_blocks = make(rng, n, bs, mb, with_rows, longest)
    T = int(q.sum()) + pad
    want, bad = plain(seq_blocks, rows, c, q, new, bs, num_blocks, T)
    assert not bad
    same(run(ctx, seq_blocks, rows, c, q, new, bs, num_blocks, T), want)
    ctx.check_status()
