"""The serving-step operators in a row, as a decode loop uses them: tables from lengths,
norm + rotation + cache write, block bounds, scores, selection and attention over the
selected blocks, eagerly and as one replayed CUDA graph."""
import numpy as np
import pytest

import test_gpu_block_select as blocks
import test_gpu_rope as rope
import test_gpu_selected_decode as selected
import test_gpu_step_tables as tables

pytestmark = pytest.mark.gpu

H, HKV, D, BS, MB, NB, TOP, B = 8, 2, 64, 16, 12, 80, 5, 3


class Loop:
    """Three sequences in the rows of a persistent table, with everything on the device."""

    def __init__(self, ctx, seed):
        import torch
        import zealot_b200 as zb
        self.ctx, self.attn, self.rng = ctx, zb.CudaAttention(ctx), np.random.default_rng(seed)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
        self.seq_blocks = torch.full((6, MB), -1, dtype=torch.int32, device="cuda")
        self.rows = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
        self.ctx_lens, self.q_lens, self.new = i32(B), i32(B), torch.full((16,), -1, dtype=torch.int32, device="cuda")
        self.k_pool, self.v_pool, self.bounds = bf(NB, HKV, BS, D), bf(NB, HKV, BS, D), bf(NB, HKV, 2, D)
        self.freq = torch.from_numpy(rope.freqs(D)).cuda()
        self.weights = [bf(D).add_(1.0), bf(D).add_(0.5)]
        self.free = list(self.rng.permutation(NB))
        self.out = dict(block_tables=i32(B, MB), cu_seqlens=i32(B + 1), seq_lens=i32(B), last_rows=i32(B))
        self.scores = torch.zeros((B, HKV, MB), device="cuda")
        self.sel, self.q_out, self.o = i32(B, HKV, TOP), bf(B, H, D), bf(B, H, D)
        self.decode_qkv = bf(B, (H + 2 * HKV) * D)
        self.decode_pos, self.decode_slots = i32(B), torch.zeros(B, dtype=torch.int64, device="cuda")

    def set_step(self, context, query):
        """Uploads a step's lengths and the ids of the blocks that it opens."""
        import torch
        need = sum(-(-(c + q) // BS) - -(-c // BS) for c, q in zip(context, query))
        new = np.full(16, -1, np.int32)
        new[:need] = [self.free.pop() for _ in range(need)]
        self.new.copy_(torch.from_numpy(new))
        self.ctx_lens.copy_(torch.tensor(context, dtype=torch.int32))
        self.q_lens.copy_(torch.tensor(query, dtype=torch.int32))
        return new

    def write(self, qkv, pos, slots, q_out):
        t = qkv.shape[0]
        q, k, v = (x.reshape(t, -1, D) for x in qkv.split((H * D, HKV * D, HKV * D), dim=1))
        self.attn.step_tables(self.seq_blocks, self.rows, self.ctx_lens, self.q_lens, self.new, self.out["block_tables"],
                              self.out["cu_seqlens"], self.out["seq_lens"], pos, slots, self.out["last_rows"], BS, NB)
        self.attn.qk_norm_rope(q, k, v, pos, self.freq, q_out=q_out, q_weight=self.weights[0], k_weight=self.weights[1],
                               k_pool=self.k_pool, v_pool=self.v_pool, slot_mapping=slots)
        self.attn.block_bounds(self.k_pool, self.out["block_tables"], self.out["seq_lens"], self.bounds,
                               tok_begin=self.ctx_lens)

    def decode(self):
        self.write(self.decode_qkv, self.decode_pos, self.decode_slots, self.q_out)
        t, n = self.out["block_tables"], self.out["seq_lens"]
        self.attn.block_scores(self.q_out, self.bounds, t, n, self.scores, BS)
        self.attn.select_blocks(self.scores, n, self.sel, BS, num_first=1, num_last=1)
        self.attn.paged_forward_selected(self.q_out, self.k_pool, self.v_pool, t, n, self.sel, self.o)


@pytest.mark.parametrize("graph", [False, True])
def test_decode_loop(ctx, graph):
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    loop = Loop(ctx, 5)
    keys = [np.zeros((0, HKV, D)) for _ in range(B)]  # what each sequence's cache should hold, in 64 bits
    vals = [np.zeros((0, HKV, D)) for _ in range(B)]
    lens = [0, 0, 0]

    def expect(qkv, query):
        """Appends a step's keys and values from the formula; returns the queries."""
        x = qkv.float().cpu().numpy().reshape(len(qkv), -1, D)
        pos = np.concatenate([np.arange(c, c + n) for c, n in zip(lens, query)])
        w = [t.float().cpu().numpy() for t in loop.weights]
        q, _ = rope.formula(x[:, :H], w[0], 1e-6, pos, rope.freqs(D), False)
        k, _ = rope.formula(x[:, H:H + HKV], w[1], 1e-6, pos, rope.freqs(D), False)
        at = 0
        for b in range(B):
            keys[b] = np.concatenate([keys[b], k[at:at + query[b]]])
            vals[b] = np.concatenate([vals[b], x[at:at + query[b], H + HKV:]])
            at += query[b]
            lens[b] += query[b]
        return q

    # prompts of 100, 1 and 47 tokens, with two padding rows
    query = [100, 1, 47]
    qkv = torch.randn((150, (H + 2 * HKV) * D), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.zeros(150, dtype=torch.int32, device="cuda")
    slots = torch.zeros(150, dtype=torch.int64, device="cuda")
    loop.set_step(lens, query)
    loop.write(qkv, pos, slots, torch.empty((150, H, D), dtype=torch.bfloat16, device="cuda"))
    expect(qkv[:148], query)
    ctx.check_status()

    run = loop.decode
    if graph:
        # capture on lengths of no tokens, so that the warm-up leaves the state as it is
        loop.q_lens.zero_(), loop.ctx_lens.zero_()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            loop.decode()
        torch.cuda.current_stream().wait_stream(stream)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            loop.decode()
        run = captured.replay
    for step in range(20):
        qkv = torch.randn((B, (H + 2 * HKV) * D), generator=g, device="cuda").to(torch.bfloat16)
        loop.decode_qkv.copy_(qkv)
        loop.set_step(lens, [1, 1, 1])
        run()
        q = expect(qkv, [1, 1, 1])
        ctx.check_status()
        t = loop.out["block_tables"].cpu().numpy()
        assert loop.out["seq_lens"].tolist() == lens
        assert loop.decode_pos.tolist() == [n - 1 for n in lens]
        # queries and cache: within their rounding to bf16 (and fp32 work, far below it)
        assert np.allclose(loop.q_out.double().cpu().numpy(), q, rtol=2.0 ** -8, atol=1e-4)
        kp, vp = loop.k_pool.double().cpu().numpy(), loop.v_pool.double().cpu().numpy()
        for b in range(B):
            rows = t[b, np.arange(lens[b]) // BS], np.arange(lens[b]) % BS
            assert np.allclose(kp[rows[0], :, rows[1]], keys[b], rtol=2.0 ** -8, atol=1e-4)
            assert np.array_equal(vp[rows[0], :, rows[1]], vals[b])
        # each later stage against what it was given
        bounds = blocks.plain_bounds(loop.k_pool, t, lens, None, loop.bounds, BS)
        for b in range(B):
            ids = t[b, :-(-lens[b] // BS)]
            assert np.array_equal(loop.bounds.float().cpu().numpy()[ids], bounds[ids])
        want, tol = blocks.plain_scores(loop.q_out, loop.bounds, t, lens, HKV, BS, D ** -0.5, False)
        got = loop.scores.double().cpu().numpy()
        assert np.array_equal(np.isinf(got), np.isinf(want)) and np.all(np.abs(got - want)[np.isfinite(want)]
                                                                      <= tol[np.isfinite(want)])
        sel = loop.sel.cpu().numpy()
        assert np.array_equal(sel, blocks.plain_select(loop.scores.cpu().numpy(), lens, BS, TOP, 1, 1))
        want, tol = selected.plain(loop.q_out.double().cpu().numpy(), kp, vp, t, lens, sel, D ** -0.5, False, True)
        assert np.all(np.abs(loop.o.double().cpu().numpy() - want) <= tol)
    if graph:
        del captured


@pytest.mark.parametrize("first_ahead", [False, True])
def test_decode_that_reads_ahead_behind_step_tables(first_ahead):
    """Step tables, a decode on other tables, then a decode of the new tables that reads them ahead of the kernel
    before it: they were written before that kernel's place in the stream, so it finds the new ones."""
    import torch
    import zealot_b200 as zb
    from zealot_b200.context import CTX_INPUTS_AHEAD
    n, width, nb, bs = 1024, 64, 4096, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    k_pool, v_pool, q = rand(nb, 1, bs, 128), rand(nb, 1, bs, 128), rand(n, 4, 128)
    seq_blocks = torch.randint(0, nb, (n, width), generator=g, device="cuda", dtype=torch.int32)
    other, other_lens = torch.randint(0, nb, (4, width), generator=g, device="cuda", dtype=torch.int32), i32(4) + 40
    tables, cu, lens, last, ones = i32(n, width), i32(n + 1), i32(n), i32(n), i32(n) + 1
    pos, slots, o, o4, want = i32(n), i32(n).long(), torch.empty_like(q), rand(4, 4, 128), torch.empty_like(q)
    new = torch.randint(0, nb, (n,), generator=g, device="cuda", dtype=torch.int32)
    with zb.GpuContext(0) as own:
        attn = zb.CudaAttention(own)
        decode = lambda q, t, l, out: attn.paged_forward(q, k_pool, v_pool, t, l, out, len(l), 4, 1, 128, bs, width, num_blocks=nb)
        decode(q, tables, lens, want)  # (the first call sets the workspace up)
        for step in range(30):
            context = torch.randint(1, 400, (n,), generator=g, device="cuda", dtype=torch.int32)
            context[::3] = 0
            tables.zero_(), lens.fill_(1 + step % 2 * 200)
            torch.cuda.synchronize()
            attn.step_tables(seq_blocks, None, context, ones, new, tables, cu, lens, pos, slots, last, bs, nb)
            own.set_flags(CTX_INPUTS_AHEAD if first_ahead else 0)
            decode(q[:4], other, other_lens, o4)
            own.set_flags(CTX_INPUTS_AHEAD)
            decode(q, tables, lens, o)
            own.check_status()
            own.set_flags(0)
            decode(q, tables, lens, want)
            torch.cuda.synchronize()
            assert torch.equal(lens, context + 1) and torch.equal(o, want)
        own.check_status()


def test_several_tokens_of_a_sequence(ctx):
    """Three new tokens of each of two sequences, which end in one block and in two: bounds once for each sequence, then
    a row for each token. A shorter row's bounds cover the later tokens too and still bound its own."""
    import torch
    import zealot_b200 as zb
    g = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    before, after = [130, 94], [133, 97]
    k_pool, v_pool, q = rand(NB, HKV, BS, D), rand(NB, HKV, BS, D), rand(6, H, D)
    table = torch.randperm(NB, generator=g, device="cuda")[:2 * MB].reshape(2, MB).to(torch.int32)
    attn = zb.CudaAttention(ctx)
    bounds = torch.zeros((NB, HKV, 2, D), dtype=torch.bfloat16, device="cuda")
    attn.block_bounds(k_pool, table, dev(before), bounds)
    attn.block_bounds(k_pool, table, dev(after), bounds, tok_begin=dev(before))
    t = table.cpu().numpy()
    want = blocks.plain_bounds(k_pool, t, after, None, torch.zeros_like(bounds), BS)
    for b in range(2):
        ids = t[b, :-(-after[b] // BS)]
        assert np.array_equal(bounds.float().cpu().numpy()[ids], want[ids])
    lens = [131, 132, 133, 95, 96, 97]
    rows = table.repeat_interleave(3, 0)
    scores, sel = torch.zeros((6, HKV, MB), device="cuda"), torch.zeros((6, HKV, TOP), dtype=torch.int32, device="cuda")
    o = torch.empty_like(q)
    attn.block_scores(q, bounds, rows, dev(lens), scores, BS)
    attn.select_blocks(scores, dev(lens), sel, BS)
    attn.paged_forward_selected(q, k_pool, v_pool, rows, dev(lens), sel, o)
    ctx.check_status()
    t, qh, kh, got = rows.cpu().numpy(), q.double().cpu().numpy(), k_pool.double().cpu().numpy(), scores.double().cpu().numpy()
    _, tol = blocks.plain_scores(q, bounds, t, lens, HKV, BS, D ** -0.5, False)
    for b, n in enumerate(lens):
        for j in range(-(-n // BS)):
            for h in range(H):
                kv = h // (H // HKV)
                s = kh[t[b, j], kv, :min(BS, n - j * BS)] @ qh[b, h] * D ** -0.5
                assert s.max() <= got[b, kv, j] + tol[b, kv, j]
    picked = sel.cpu().numpy()
    assert np.array_equal(picked, blocks.plain_select(scores.cpu().numpy(), lens, BS, TOP, 1, 1))
    want, tol = selected.plain(qh, kh, v_pool.double().cpu().numpy(), t, lens, picked, D ** -0.5, False, True)
    assert np.all(np.abs(o.double().cpu().numpy() - want) <= tol)


def test_other_shapes_of_the_same_size_are_refused(ctx):
    """As many elements in another shape would be read as if they had the documented one."""
    import torch
    import zealot_b200 as zb
    attn = zb.CudaAttention(ctx)
    f32 = lambda *s: torch.zeros(s, device="cuda")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    q, pool, bounds, table, lens, sel, scores = f32(3, 8, 64), f32(5, 2, 16, 64), f32(5, 2, 2, 64), i32(3, 4), i32(3), i32(3, 2, 4), f32(3, 2, 4)
    attn.paged_forward_selected(q, pool, pool, table, lens, sel, torch.empty_like(q))
    attn.block_scores(q, bounds, table, lens, scores, 16)
    attn.select_blocks(scores, lens, sel, 16)
    for bad in (q.view(6, 8, 32), q.view(1, 8, 192), q.view(2, 12, 64)):
        with pytest.raises(zb.InvalidArgument):
            attn.paged_forward_selected(bad, pool, pool, table, lens, sel, torch.empty_like(q))
        with pytest.raises(zb.InvalidArgument):
            attn.block_scores(bad, bounds, table, lens, scores, 16)
    for bad in (sel.view(2, 3, 4), sel.view(1, 6, 4)):
        with pytest.raises(zb.InvalidArgument):
            attn.paged_forward_selected(q, pool, pool, table, lens, bad, torch.empty_like(q))
        with pytest.raises(zb.InvalidArgument):
            attn.select_blocks(scores, lens, bad, 16)
    with pytest.raises(zb.InvalidArgument):
        attn.paged_forward_selected(q, pool, pool.view(5, 16, 2, 64), table, lens, sel, torch.empty_like(q))
    x, slots = f32(3, 2, 64), torch.zeros(3, dtype=torch.int64, device="cuda") - 1
    attn.qk_norm_rope(q, x, x, None, None, k_pool=pool, v_pool=pool.clone(), slot_mapping=slots)
    with pytest.raises(zb.InvalidArgument):
        attn.qk_norm_rope(q, x, x, None, None, k_pool=pool, v_pool=pool.clone().view(5, 16, 2, 64), slot_mapping=slots)
    ctx.check_status()
