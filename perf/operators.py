"""Cases for the operators of one serving step around the paged KV cache.

The operators, in the order in which a step uses them:

  tables   block tables, slot mapping, positions and row offsets of a step, built on the
           device from the requests' lengths (`CudaAttention.step_tables`)
  rope     RMS norm of every query and key head, rotation by position, and the write of
           keys and values into the paged pools (`CudaAttention.qk_norm_rope`)
  score    elementwise bounds of each block's keys (`CudaAttention.block_bounds`) and, from
           them, an upper bound of every block's attention scores for a query
           (`CudaAttention.block_scores`)
  select   the blocks that a query attends to: the first and last ones and the best of the
           others (`CudaAttention.select_blocks`)
  attend   attention of one token per sequence over its selected blocks
           (`CudaAttention.paged_forward_selected`)

With `own` false, `run` computes an operator from elementary torch operations; with `own`
true it makes the framework's calls. A case's lengths are spread evenly over its range, in
an order that the seed draws, so that the work of a case does not depend on the seed.
"""
import math

import torch

own = False

_attention = None


def _attn():
    """The framework's attention operators on one context, which a program creates once."""
    global _attention
    if _attention is None:
        import zealot_b200
        _attention = zealot_b200.CudaAttention(zealot_b200.GpuContext(torch.cuda.current_device()))
    return _attention


# ------------------------------------------------------------------------------- cases


def listed():
    return [
        # The metadata of a decode step: 64 sequences, contexts of 512 to 4096.
        dict(name="tables decode", op="tables", prefills=0, chunk=0, decodes=64, lo=512, hi=4096, bs=16, max_blocks=257,
             pad=0),
        # The metadata of a step of a large long-context batch: 32 prompt chunks of 2000 tokens next to
        # 992 decode rows, tables for 131072 tokens, the token rows padded to a fixed count.
        dict(name="tables mixed", op="tables", prefills=32, chunk=2000, decodes=992, lo=1, hi=120000, bs=16,
             max_blocks=8192, pad=544),
        # Five tokens of a small float32 model: rotation of the first half of each head, in neighbouring pairs.
        dict(name="rope f32 small", op="rope", tokens=5, heads=4, kv_heads=4, d=64, rot=32, inter=True, norm=True,
             packed=False, bs=16, f32=True, far=2048),
        # One decode step of 64 sequences of a layer with 32 query and 8 key heads; only the cache gets the keys.
        dict(name="rope decode", op="rope", tokens=64, heads=32, kv_heads=8, d=128, rot=128, inter=False, norm=True,
             packed=False, bs=16, f32=False, far=131072),
        # The prompt tokens of 16 sequences of 256 to 8192 tokens: the cache and the packed keys and values.
        dict(name="rope prefill", op="rope", tokens=53067, heads=32, kv_heads=8, d=128, rot=128, inter=False, norm=True,
             packed=True, bs=16, f32=False, far=8192),
        # One decode step: the newest block's bounds, then the scores of every block.
        dict(name="score decode", op="score", seqs=64, heads=32, kv_heads=8, d=128, lo=512, hi=4096, bs=16, f32=False,
             modulo=False, what="step"),
        # The scores of 8192 blocks for each of 8 long sequences, 8 query heads to a key head.
        dict(name="score long", op="score", seqs=8, heads=64, kv_heads=8, d=128, lo=131072, hi=131072, bs=16, f32=False,
             modulo=False, what="scores"),
        # The bounds of every block of 16 prompts, after their keys were written.
        dict(name="bounds prefill", op="score", seqs=16, heads=32, kv_heads=8, d=128, lo=256, hi=8192, bs=16, f32=False,
             modulo=False, what="bounds"),
        # 32 of some 100 blocks for a few sequences.
        dict(name="select small", op="select", seqs=4, kv_heads=8, lo=512, hi=2048, bs=16, top=32, first=1, last=2,
             max_blocks=128),
        # 256 of up to 8192 blocks for 64 sequences.
        dict(name="select long", op="select", seqs=64, kv_heads=8, lo=4096, hi=131072, bs=16, top=256, first=1, last=4,
             max_blocks=8192),
        # Two sequences in float32, 24 blocks each.
        dict(name="attend f32 small", op="attend", seqs=2, heads=12, kv_heads=4, d=64, lo=700, hi=2001, bs=16, top=24,
             f32=True, modulo=False),
        # 128 blocks (2048 tokens) for each of 64 sequences of 4096 to 32768 tokens.
        dict(name="attend decode", op="attend", seqs=64, heads=32, kv_heads=8, d=128, lo=4096, hi=32768, bs=16, top=128,
             f32=False, modulo=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((32, 8), (64, 8), (16, 16), (12, 4), (28, 4), (8, 1), (4, 4), (40, 8))


def draw(rng):
    op = rng.choice(("tables", "rope", "score", "select", "attend"))
    bs = rng.choice((8, 16, 16, 32, 64))
    heads, kv_heads = rng.choice(_HEADS)
    f32 = rng.random() < 0.3
    if op == "tables":
        prefills, decodes = rng.choice((0, 1, _log_int(rng, 1, 32))), _log_int(rng, 1, 992)
        chunk = _log_int(rng, 1, 2000) if prefills else 0
        max_blocks = _log_int(rng, max(4, -(-(chunk + 1) // bs) + 1), 8192 * 16 // bs if bs > 16 else 8192)
        top = max_blocks * bs - chunk - 1
        return dict(op=op, prefills=prefills, chunk=chunk, decodes=decodes, lo=rng.choice((0, 1, min(top, 300))),
                    hi=_log_int(rng, min(top, 300) or 1, max(top, 1)), bs=bs, max_blocks=max_blocks,
                    pad=rng.choice((0, 0, rng.randrange(1, 300))))
    if op == "rope":
        d = rng.choice((64, 80, 96, 128, 128, 256))
        row = (heads + 2 * kv_heads) * d * (2 if f32 else 1)
        most = 53067 * 48 * 128 // row
        rot = rng.choice((d, d, d // 2))
        return dict(op=op, tokens=_log_int(rng, 1, most), heads=heads, kv_heads=kv_heads, d=d, rot=rot,
                    inter=rng.random() < 0.3, norm=rng.random() < 0.7, packed=rng.random() < 0.5, bs=bs, f32=f32,
                    far=rng.choice((4096, 131072, 1000000)))
    d = rng.choice((64, 80, 96, 128, 128, 256))
    hi = _log_int(rng, 100, 131072)
    lo = rng.choice((0, 1, hi // 8, hi))
    if op == "score":
        what = rng.choice(("step", "scores", "bounds"))
        token = kv_heads * d * (4 if f32 else 2)  # bytes of one token's keys
        # the blocks' bounds for "scores", the keys themselves for "bounds" (and in the pool for "step")
        most = 138e6 if what == "bounds" else 268e6 * bs / 2
        most = min(most, 2e9)
        seqs = _log_int(rng, 1, max(1, min(256, int(most / (token * max(1, (lo + hi) // 2))))))
        return dict(op=op, seqs=seqs, heads=heads, kv_heads=kv_heads, d=d, lo=lo, hi=hi, bs=bs, f32=f32,
                    modulo=rng.random() < 0.2, what=what)
    if op == "select":
        n = -(-hi // bs)
        top = min(max(5, _log_int(rng, 5, 512)), max(5, n))
        most = 64 * 8 * 4096 // (kv_heads * max(1, n // 2))
        return dict(op=op, seqs=_log_int(rng, 1, max(1, min(256, most))), kv_heads=kv_heads, lo=lo, hi=hi, bs=bs, top=top,
                    first=rng.choice((0, 1, 2)), last=rng.choice((0, 1, 3)), max_blocks=n + rng.choice((0, 0, 7)))
    n = -(-hi // bs)
    top = max(1, min(n, _log_int(rng, 8, 256 * 16 // bs)))
    token = kv_heads * d * (8 if f32 else 4)  # bytes of one token's keys and values
    most = min(64 * 2048 * 4096 // (token * top * bs), int(8e9 / (token * max(1, (lo + hi) // 2))))
    return dict(op=op, seqs=_log_int(rng, 1, max(1, min(256, most))), heads=heads, kv_heads=kv_heads, d=d, lo=lo, hi=hi,
                bs=bs, top=top, f32=f32, modulo=rng.random() < 0.2)


# ------------------------------------------------------------------------------ inputs


def _spread(lo, hi, n):
    """n whole numbers spread evenly over [lo, hi]."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi] * n


def _blocks(tokens, bs):
    return -(-tokens // bs)


def _dtype(case):
    return torch.float32 if case["f32"] else torch.bfloat16


def _query_lens(case):
    """New tokens of each request: the prompt chunks, the last one cut short, then one token per decode row."""
    chunks = [case["chunk"]] * case["prefills"]
    if chunks:
        chunks[-1] = max(1, chunks[-1] // 3)
    return chunks + [1] * case["decodes"]


def _contexts(case):
    n = case["prefills"] + case["decodes"]
    return _spread(case["lo"], case["hi"], n)


def _lens(case, gen):
    """The case's sequence lengths on the device, in an order that the seed draws."""
    lens = torch.tensor(_spread(case["lo"], case["hi"], case["seqs"]), dtype=torch.int32)
    return lens[torch.randperm(len(lens), generator=gen)].cuda()


def _fill_tables(lens, width, bs, gen):
    """[n][width] tables of distinct blocks of a permuted pool, -1 after each sequence's last, and the pool's size.
    The pool's last block is nobody's."""
    need = (lens.long() + bs - 1) // bs
    ends = torch.cumsum(need, 0)
    num_blocks = int(ends[-1]) + 8
    perm = torch.randperm(num_blocks - 1, generator=gen).cuda()
    col = torch.arange(width, device="cuda")[None, :]
    at = (ends - need)[:, None] + col
    table = torch.where(col < need[:, None], perm[at.clamp(max=num_blocks - 2)], -1).to(torch.int32)
    return table.contiguous(), num_blocks, ends


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    return dict({"tables": _prepare_tables, "rope": _prepare_rope, "score": _prepare_score, "select": _prepare_select,
                 "attend": _prepare_attend}[case["op"]](case, gen, dev), case=case)


def _prepare_tables(case, gen, dev):
    bs, width = case["bs"], case["max_blocks"]
    query = torch.tensor(_query_lens(case), dtype=torch.int32).cuda()
    n = query.numel()
    ctx = torch.tensor(_contexts(case), dtype=torch.int32)
    ctx = ctx[torch.randperm(n, generator=gen)].cuda()
    num_rows = n + n // 4 + 1  # the engine keeps a table row for every request, the waiting ones too
    rows = torch.randperm(num_rows, generator=gen)[:n].to(torch.int32).cuda()
    old = torch.zeros(num_rows, dtype=torch.int32, device="cuda")
    old[rows.long()] = ctx
    need = _blocks(ctx.long() + query, bs) - _blocks(ctx.long(), bs)
    seq_blocks, _, ends = _fill_tables(old, width, bs, gen)
    num_new = int(need.sum())
    first = int(ends[-1]) + 8
    num_blocks = first + num_new
    new_blocks = (first + torch.randperm(max(1, num_new), generator=gen)).to(torch.int32).cuda()
    tokens = sum(_query_lens(case)) + case["pad"]

    def out(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    return dict(seq_blocks=seq_blocks, rows=rows, context_lens=ctx, query_lens=query, new_blocks=new_blocks,
                num_blocks=num_blocks, block_tables=out(n, width), cu_seqlens=out(n + 1), seq_lens=out(n),
                positions=out(tokens), slot_mapping=out(tokens, dtype=torch.int64), last_rows=out(n))


def _prepare_rope(case, gen, dev):
    t, h, hk, d, bs, kind = case["tokens"], case["heads"], case["kv_heads"], case["d"], case["bs"], _dtype(case)
    # One projection's output: the q, k and v of a token side by side.
    qkv = torch.randn((t, (h + 2 * hk) * d), generator=dev, device="cuda").to(kind)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((h * d, hk * d, hk * d), dim=1))
    num_blocks = _blocks(t, bs) + 8
    pool = (num_blocks, hk, bs, d)
    return dict(q=q, k=k, v=v,
                q_weight=(1 + 0.1 * torch.randn(d, generator=dev, device="cuda")).to(kind) if case["norm"] else None,
                k_weight=(1 + 0.1 * torch.randn(d, generator=dev, device="cuda")).to(kind) if case["norm"] else None,
                inv_freq=(500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).cuda(),
                positions=torch.randint(0, case["far"], (t,), generator=gen, dtype=torch.int32).cuda(),
                slot_mapping=torch.randperm(num_blocks * bs, generator=gen)[:t].cuda(),
                k_pool=torch.randn(pool, generator=dev, device="cuda").to(kind),
                v_pool=torch.randn(pool, generator=dev, device="cuda").to(kind),
                q_out=torch.zeros((t, h, d), dtype=kind, device="cuda"),
                k_out=torch.zeros((t, hk, d), dtype=kind, device="cuda") if case["packed"] else None,
                v_out=torch.zeros((t, hk, d), dtype=kind, device="cuda") if case["packed"] else None)


def _prepare_score(case, gen, dev):
    b, hk, d, bs, kind = case["seqs"], case["kv_heads"], case["d"], case["bs"], _dtype(case)
    lens = _lens(case, gen)
    width = max(1, _blocks(case["hi"], bs))
    table, num_blocks, _ = _fill_tables(lens, width, bs, gen)
    state = dict(lens=lens, table=table, q=torch.randn((b, case["heads"], d), generator=dev, device="cuda").to(kind),
                 scores=torch.zeros((b, hk, width), device="cuda"))
    if case["what"] == "scores":
        # the bounds of bs keys of N(0, 1): their extremes lie around -+sqrt(2 ln bs)
        ends = torch.randn((2, num_blocks, hk, d), generator=dev, device="cuda").mul_(0.4)
        mid = math.sqrt(2 * math.log(bs))
        state["bounds"] = torch.stack((ends[0] - mid, ends[1] + mid), dim=2).to(kind)
    else:
        state["k_pool"] = torch.randn((num_blocks, hk, bs, d), generator=dev, device="cuda").to(kind)
        state["bounds"] = torch.stack((state["k_pool"].amin(2), state["k_pool"].amax(2)), dim=2)
        # one new token per sequence, or a whole prompt
        state["begin"] = (lens - 1).clamp(min=0) if case["what"] == "step" else None
    return state


def _prepare_select(case, gen, dev):
    lens = _lens(case, gen)
    shape = (case["seqs"], case["kv_heads"], case["max_blocks"])
    # coarse enough for some equal scores
    scores = torch.randn(shape, generator=dev, device="cuda").mul_(2048).round_().div_(512)
    beyond = torch.arange(case["max_blocks"], device="cuda") >= _blocks(lens, case["bs"])[:, None, None]
    return dict(lens=lens, scores=scores.masked_fill_(beyond, -math.inf),
                selected=torch.zeros(shape[:2] + (case["top"],), dtype=torch.int32, device="cuda"))


def _prepare_attend(case, gen, dev):
    b, hk, d, bs, kind = case["seqs"], case["kv_heads"], case["d"], case["bs"], _dtype(case)
    lens = _lens(case, gen)
    width = max(1, _blocks(case["hi"], bs))
    table, num_blocks, _ = _fill_tables(lens, width, bs, gen)
    # a random choice of blocks for every sequence and key head, its first and last block among them
    need = _blocks(lens, bs)[:, None, None]
    col = torch.arange(width, device="cuda")
    chance = torch.rand((b, hk, width), generator=dev, device="cuda")
    chance = torch.where((col == 0) | (col == need - 1), 2.0, chance).masked_fill(col >= need, -1.0)
    top = min(case["top"], width)
    best, picked = chance.topk(top, dim=2)
    picked = torch.where(best < 0, width, picked).sort(dim=2).values
    selected = torch.where(picked == width, -1, picked).to(torch.int32)
    pool = (num_blocks, hk, bs, d)
    return dict(lens=lens, table=table, selected=selected.contiguous(),
                q=torch.randn((b, case["heads"], d), generator=dev, device="cuda").to(kind),
                k_pool=torch.empty(pool, dtype=kind, device="cuda").normal_(generator=dev),
                v_pool=torch.empty(pool, dtype=kind, device="cuda").normal_(generator=dev),
                o=torch.zeros((b, case["heads"], d), dtype=kind, device="cuda"))


# --------------------------------------------------------------------------- operators


def run(state):
    return {"tables": _tables, "rope": _rope, "score": _score, "select": _select, "attend": _attend}[state["case"]["op"]](state)


def _tables(s):
    case = s["case"]
    bs = case["bs"]
    if own:
        _attn().step_tables(s["seq_blocks"], s["rows"], s["context_lens"], s["query_lens"], s["new_blocks"],
                            s["block_tables"], s["cu_seqlens"], s["seq_lens"], s["positions"], s["slot_mapping"],
                            s["last_rows"], bs, s["num_blocks"])
        return {k: s[k] for k in ("block_tables", "cu_seqlens", "seq_lens", "positions", "slot_mapping", "last_rows",
                                  "seq_blocks")}
    rows, ctx, query = s["rows"].long(), s["context_lens"].long(), s["query_lens"].long()
    ends = torch.cumsum(query, 0)
    cu = torch.cat((torch.zeros_like(ends[:1]), ends))
    seq = ctx + query
    had, has = (ctx + bs - 1) // bs, (seq + bs - 1) // bs
    fresh = torch.cumsum(has - had, 0) - (has - had)
    col = torch.arange(case["max_blocks"], device="cuda")[None, :]
    kept = s["seq_blocks"][rows]
    at = (fresh[:, None] + col - had[:, None]).clamp(0, s["new_blocks"].numel() - 1)
    fresh_here = (col >= had[:, None]) & (col < has[:, None])
    kept = torch.where(fresh_here, s["new_blocks"][at], kept)
    s["seq_blocks"][rows] = kept
    table = torch.where(col < has[:, None], kept, -1)
    token = torch.arange(s["positions"].numel(), device="cuda")
    real = token < ends[-1]
    i = torch.searchsorted(ends, token, right=True).clamp(max=len(rows) - 1)
    pos = torch.where(real, token - cu[i] + ctx[i], 0)
    slot = torch.where(real, table[i, pos // bs].long() * bs + pos % bs, -1)
    return {"block_tables": table, "cu_seqlens": cu.int(), "seq_lens": seq.int(), "positions": pos.int(),
            "slot_mapping": slot, "last_rows": (cu[1:] - 1).clamp(min=0).int(), "seq_blocks": s["seq_blocks"]}


def _norm_rotate(x, weight, eps, cos, sin, inter):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()
    rot = 2 * cos.shape[-1]
    turn, rest = x[..., :rot], x[..., rot:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if inter else turn.chunk(2, dim=-1)
    both = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(both, dim=-1).flatten(-2) if inter else torch.cat(both, dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _rope(s):
    case = s["case"]
    if own:
        _attn().qk_norm_rope(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["q_out"], k_out=s["k_out"],
                             v_out=s["v_out"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                             interleaved=case["inter"], k_pool=s["k_pool"], v_pool=s["v_pool"],
                             slot_mapping=s["slot_mapping"])
        return {k: s[k] for k in ("q_out", "k_out", "v_out", "k_pool", "v_pool")}
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    kind = s["q"].dtype
    q = _norm_rotate(s["q"], s["q_weight"], 1e-6, cos, sin, case["inter"]).to(kind)
    k = _norm_rotate(s["k"], s["k_weight"], 1e-6, cos, sin, case["inter"]).to(kind)
    block, at = s["slot_mapping"] // case["bs"], s["slot_mapping"] % case["bs"]
    s["k_pool"][block, :, at] = k
    s["v_pool"][block, :, at] = s["v"]
    return {"q_out": q, "k_out": k if case["packed"] else None, "v_out": s["v"].contiguous() if case["packed"] else None,
            "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _by_group(q, hk, modulo):
    """[B][H][d] queries as [B][Hkv][H / Hkv][d]."""
    return q.unflatten(1, (-1, hk)).transpose(1, 2) if modulo else q.unflatten(1, (hk, -1))


def _score(s):
    case = s["case"]
    bs, hk, what = case["bs"], case["kv_heads"], case["what"]
    if own:
        if what != "scores":
            _attn().block_bounds(s["k_pool"], s["table"], s["lens"], s["bounds"], tok_begin=s["begin"])
        if what == "bounds":
            return s["bounds"]
        _attn().block_scores(s["q"], s["bounds"], s["table"], s["lens"], s["scores"], bs, gqa_map=int(case["modulo"]))
        return s["scores"] if what == "scores" else (s["bounds"], s["scores"])
    lens, table = s["lens"].long(), s["table"].long()
    col = torch.arange(table.shape[1], device="cuda")
    if what == "bounds":
        seq, j = torch.nonzero(col * bs < lens[:, None], as_tuple=True)
    if what == "step":
        seq = torch.arange(len(lens), device="cuda")
        j = ((lens - 1) // bs).clamp(min=0)
    if what != "scores":
        block = table[seq, j].clamp(min=0)  # a sequence without tokens has no block: the pool's last one stands in, unchanged
        keys = s["k_pool"][block]
        seen = (j[:, None] * bs + torch.arange(bs, device="cuda") < lens[seq, None])[:, None, :, None]
        low = keys.masked_fill(~seen, math.inf).amin(2)
        high = keys.masked_fill(~seen, -math.inf).amax(2)
        some = (lens[seq] > 0)[:, None, None, None]
        new = torch.where(some, torch.stack((low, high), dim=2), s["bounds"][block])
        s["bounds"][torch.where(lens[seq] > 0, block, s["bounds"].shape[0] - 1)] = torch.where(some, new, s["bounds"][-1])
        if what == "bounds":
            return s["bounds"]
    q = _by_group(s["q"], hk, case["modulo"]).float()
    ends = s["bounds"][table.clamp(min=0)].float()  # [B][blocks][Hkv][2][d]
    dot = torch.matmul(q.clamp(max=0), ends[:, :, :, 0].permute(0, 2, 3, 1))
    dot += torch.matmul(q.clamp(min=0), ends[:, :, :, 1].permute(0, 2, 3, 1))
    scores = dot.amax(2) / math.sqrt(case["d"])
    scores = scores.masked_fill(col * bs >= lens[:, None, None], -math.inf)
    return scores if what == "scores" else (s["bounds"], scores)


def _select(s):
    case = s["case"]
    if own:
        _attn().select_blocks(s["scores"], s["lens"], s["selected"], case["bs"], num_first=case["first"],
                              num_last=case["last"])
        return s["selected"]
    n = ((s["lens"] + case["bs"] - 1) // case["bs"])[:, None, None]
    col = torch.arange(case["max_blocks"], device="cuda")
    always = (col < case["first"]) | (col >= n - case["last"])
    score = s["scores"].masked_fill(always, math.inf)
    # blocks behind the last one sort behind every block, whatever its score
    order = torch.sort(score, dim=2, descending=True, stable=True).indices
    order = torch.gather(order, 2, torch.sort((order >= n).byte(), dim=2, stable=True).indices)[:, :, :case["top"]]
    picked = torch.where(order < n, order, case["max_blocks"]).sort(dim=2).values
    if picked.shape[2] < case["top"]:
        picked = torch.nn.functional.pad(picked, (0, case["top"] - picked.shape[2]), value=case["max_blocks"])
    return torch.where(picked == case["max_blocks"], -1, picked).int()


def _attend(s):
    case = s["case"]
    bs, hk = case["bs"], case["kv_heads"]
    if own:
        _attn().paged_forward_selected(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], s["selected"], s["o"],
                                       gqa_map=int(case["modulo"]))
        return s["o"]
    q = _by_group(s["q"], hk, case["modulo"]).float()
    picked = s["selected"].long()
    b, _, top = picked.shape
    block = torch.gather(s["table"].long()[:, None].expand(-1, hk, -1), 2, picked.clamp(min=0)).clamp(min=0)
    head = torch.arange(hk, device="cuda")[None, :, None]
    k = s["k_pool"][block, head].flatten(2, 3).float()
    v = s["v_pool"][block, head].flatten(2, 3).float()
    pos = picked[..., None] * bs + torch.arange(bs, device="cuda")
    seen = ((picked[..., None] >= 0) & (pos < s["lens"].long()[:, None, None, None])).flatten(2)[:, :, None]
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(case["d"])
    score = score.masked_fill(~seen, -math.inf)
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(most == -math.inf, 0.0, most)).masked_fill(~seen, 0.0)
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p, v.masked_fill(~seen.transpose(2, 3), 0.0)) / torch.where(total == 0, 1.0, total)
    o = o.transpose(1, 2) if case["modulo"] else o
    return o.reshape(b, case["heads"], case["d"]).to(s["q"].dtype)


# -------------------------------------------------------------------------------- work


def work(case):
    return {"tables": _work_tables, "rope": _work_rope, "score": _work_score, "select": _work_select,
            "attend": _work_attend}[case["op"]](case)


def _work_tables(case):
    query, n = _query_lens(case), case["prefills"] + case["decodes"]
    # Which request has which context the seed draws: a request's new blocks as on average.
    had = sum(_blocks(c, case["bs"]) for c in _contexts(case))
    new = sum(query) / case["bs"]
    tokens = sum(query) + case["pad"]
    # lengths and rows in, the blocks in; tables, offsets, lengths, last rows, new entries, positions and slots out
    moved = 12 * n + 4 * (had + new) + 4 * n * case["max_blocks"] + 12 * n + 4 * new + 12 * tokens
    return {"bytes": moved, "flops": 0}


def _work_rope(case):
    size = 4 if case["f32"] else 2
    t, d, h, hk = case["tokens"], case["d"], case["heads"], case["kv_heads"]
    copies = 2 if case["packed"] else 1
    moved = t * d * size * (h + 2 * hk + h + copies * 2 * hk) + 12 * t + 4 * case["rot"]
    return {"bytes": moved, "flops": t * (h + hk) * (4 * d * case["norm"] + 3 * case["rot"])}


def _work_score(case):
    size = 4 if case["f32"] else 2
    lens = _spread(case["lo"], case["hi"], case["seqs"])
    hk, d, bs = case["kv_heads"], case["d"], case["bs"]
    blocks = sum(_blocks(n, bs) for n in lens)
    token = hk * d * size
    moved = flops = 0
    if case["what"] != "scores":
        ends = [n if case["what"] == "bounds" else (n - 1) % bs + 1 if n else 0 for n in lens]
        moved += sum(ends) * token + 2 * token * sum(_blocks(n, bs) for n in ends) + 8 * len(lens)
        flops += 2 * sum(ends) * hk * d
    if case["what"] != "bounds":
        moved += len(lens) * case["heads"] * d * size + 2 * blocks * token + 4 * blocks
        moved += 4 * len(lens) * hk * max(1, _blocks(case["hi"], bs))
        flops += 4 * blocks * case["heads"] * d
    return {"bytes": moved, "flops": flops}


def _work_select(case):
    lens = _spread(case["lo"], case["hi"], case["seqs"])
    read = case["kv_heads"] * sum(_blocks(n, case["bs"]) for n in lens)
    return {"bytes": 4 * read + 4 * len(lens) * (1 + case["kv_heads"] * case["top"]), "flops": read}


def _work_attend(case):
    size = 4 if case["f32"] else 2
    lens = _spread(case["lo"], case["hi"], case["seqs"])
    hk, d, bs = case["kv_heads"], case["d"], case["bs"]
    top = min(case["top"], max(1, _blocks(case["hi"], bs)))
    # the last block, which may be part full, is always among the selected
    seen = sum(n if _blocks(n, bs) <= top else (top - 1) * bs + (n - 1) % bs + 1 for n in lens)
    picked = sum(min(top, _blocks(n, bs)) for n in lens)
    moved = 2 * seen * hk * d * size + 2 * len(lens) * case["heads"] * d * size + 4 * picked * (1 + hk)
    return {"bytes": moved, "flops": 4 * seen * case["heads"] * d}


# ------------------------------------------------------------------------------- exact


def exact(case, seed):
    """The definition in 64 bits, one sequence (or token range) at a time."""
    s = prepare(case, seed)
    return {"tables": _exact_tables, "rope": _exact_rope, "score": _exact_score, "select": _exact_select,
            "attend": _exact_attend}[case["op"]](case, s)


def _exact_tables(case, s):
    return None  # whole numbers only


def _exact_select(case, s):
    return None  # whole numbers only


def _exact_rope(case, s):
    rot, d, bs = case["rot"], case["d"], case["bs"]
    pair = torch.arange(rot // 2, device="cuda")
    first, second = (2 * pair, 2 * pair + 1) if case["inter"] else (pair, pair + rot // 2)
    out = {k: torch.empty(s[k].shape, dtype=torch.float64) if s[k] is not None else None for k in ("q_out", "k_out", "v_out")}
    for k in ("k_pool", "v_pool"):
        out[k] = s[k].double().transpose(1, 2).reshape(-1, case["kv_heads"], d)  # by slot
    for t in range(0, case["tokens"], 4096):
        part = slice(t, min(t + 4096, case["tokens"]))
        # a turn of the complex number first + i second
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"][part].double()[:, None, None] * s["inv_freq"])
        done = {}
        for name in ("q", "k"):
            x = s[name][part].double()
            if case["norm"]:
                x = x / (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * s[name + "_weight"].double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x = x.clone()
            x[..., first], x[..., second] = z.real, z.imag
            done[name] = x
        done["v"] = s["v"][part].double()
        for name, x in done.items():
            if out[name + "_out"] is not None:
                out[name + "_out"][part] = x.cpu()
            if name != "q":
                out[name + "_pool"][s["slot_mapping"][part]] = x
    for k in ("k_pool", "v_pool"):
        out[k] = out[k].reshape(-1, bs, case["kv_heads"], d).transpose(1, 2)
    return out


def _exact_score(case, s):
    bs, hk, what = case["bs"], case["kv_heads"], case["what"]
    lens, table = s["lens"].tolist(), s["table"].long()
    if what != "scores":
        low, high = s["bounds"][:, :, 0].double(), s["bounds"][:, :, 1].double()
        for b, n in enumerate(lens):
            # whole blocks at once, then the last one if it is part full
            begin = 0 if what == "bounds" else max(n - 1, 0) // bs
            full = table[b, begin:n // bs]
            low[full], high[full] = (f(s["k_pool"][full].double(), dim=2) for f in (torch.amin, torch.amax))
            if n % bs:
                last = table[b, n // bs]
                keys = s["k_pool"][last, :, :n % bs].double()
                low[last], high[last] = keys.amin(1), keys.amax(1)
        bounds = torch.stack((low, high), dim=2)
        if what == "bounds":
            return bounds
    else:
        bounds = s["bounds"].double()
    scores = torch.full(s["scores"].shape, -math.inf, dtype=torch.float64, device="cuda")
    group = case["heads"] // hk
    for b, n in enumerate(lens):
        ends = bounds[table[b, :_blocks(n, bs)]]  # [blocks][Hkv][2][d]
        for h in range(case["heads"] if n else 0):
            kv = h % hk if case["modulo"] else h // group
            q = s["q"][b, h].double()
            best = torch.where(q < 0, ends[:, kv, 0], ends[:, kv, 1])
            score = (best @ q) / math.sqrt(case["d"])
            scores[b, kv, :len(score)] = torch.maximum(scores[b, kv, :len(score)], score)
    return scores if what == "scores" else (bounds, scores)


def _exact_attend(case, s):
    bs, hk, d = case["bs"], case["kv_heads"], case["d"]
    group = case["heads"] // hk
    out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        for kv in range(hk):
            j = s["selected"][b, kv]
            j = j[j >= 0].long()
            if not n or not len(j):
                continue
            at = (j[:, None] * bs + torch.arange(bs, device="cuda")).flatten()
            block = s["table"][b, j].long()
            k = s["k_pool"][block, kv].reshape(-1, d)[at < n].double()
            v = s["v_pool"][block, kv].reshape(-1, d)[at < n].double()
            heads = slice(kv, None, hk) if case["modulo"] else slice(kv * group, (kv + 1) * group)
            out[b, heads] = torch.softmax(s["q"][b, heads].double() @ k.T / math.sqrt(d), dim=1) @ v
    return out
