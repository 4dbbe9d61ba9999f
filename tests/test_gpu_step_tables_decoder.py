"""Decoder steps whose batch StepTables built on the device against the same steps laid out on
the host by StepBatch.build: equal bytes in logits and pools, over a prompt step and decode steps
in which requests come and go."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_decoder_steps_from_device_tables(ctx):
    import torch
    import zealot_b200 as zb
    from zealot_b200.decoder import Decoder, DecoderConfig, StepBatch, StepTables, random_weights
    cfg = DecoderConfig(num_layers=2, hidden=512, num_heads=4, num_kv_heads=2, head_dim=128, intermediate=1024, vocab=1000)
    dec = Decoder(ctx, cfg, random_weights(cfg, 3))
    rng = np.random.default_rng(1)
    nb, bs, mb = 64, 16, 6
    bm = zb.BlockManager(nb, bs)
    steps = StepTables(ctx, num_rows=5, max_blocks_per_seq=mb, max_seqs=5, max_tokens=200, block_size=bs, num_blocks=nb)
    pools, pools_host = dec.new_pools(nb, bs), dec.new_pools(nb, bs)
    seqs = {}  # row -> (length, block ids)

    def step(new, old):
        """new: {row: prompt length}, old: rows that decode one token."""
        rows = [*new, *old]
        context = [0] * len(new) + [seqs[r][0] for r in old]
        query = [*new.values()] + [1] * len(old)
        for r in new:
            seqs[r] = (0, [])
        ids = []
        for r, c, q in zip(rows, context, query):
            ids += [bm.allocate().block_id for _ in range(steps.blocks_needed(c, q))]
            seqs[r] = (c + q, seqs[r][1] + ids[len(ids) - steps.blocks_needed(c, q):])
        toks = [rng.integers(0, cfg.vocab, q) for q in query]
        table = np.full((len(old), mb), -1, np.int32)
        for i, r in enumerate(old):
            table[i, :len(seqs[r][1])] = seqs[r][1]
        host = StepBatch.build(toks[:len(new)], [int(t[0]) for t in toks[len(new):]], table, [seqs[r][0] for r in old],
                               [seqs[r][1] for r in new], bs)
        dev = steps.build(torch.from_numpy(np.concatenate(toks)).cuda(), rows, context, query, ids, len(new))
        a = dec.step(dev, *pools, bs)
        b = dec.step(host, *pools_host, bs)
        ctx.check_status()
        assert torch.equal(a, b)
        for x, y in zip([*pools[0], *pools[1]], [*pools_host[0], *pools_host[1]]):
            assert torch.equal(x, y)

    step({3: 40, 0: 1, 2: 17}, [])
    for _ in range(10):
        step({}, [0, 3, 2])
    step({4: 33, 1: 16}, [2, 0])        # row 3 waits, two prompts arrive
    del seqs[0]                         # a finished sequence's row is taken over
    step({0: 20}, [3, 1, 4, 2])
    for _ in range(8):
        step({}, [0, 1, 2, 3, 4])


def test_step_tables_build_refusals(ctx):
    import torch
    import zealot_b200 as zb
    from zealot_b200.decoder import StepTables
    steps = StepTables(ctx, 4, 4, 2, 10, 16, 32)
    toks = lambda n: torch.zeros(n, dtype=torch.int64, device="cuda")
    with pytest.raises(zb.InvalidArgument):
        steps.build(toks(3), [0], [1], [3], [0], 1)          # a prompt chunk that does not start at 0
    with pytest.raises(zb.InvalidArgument):
        steps.build(toks(2), [0], [1], [2], [], 0)           # a decode row of two tokens
    with pytest.raises(zb.InvalidArgument):
        steps.build(toks(1), [0], [0], [3], [0], 1)          # tokens missing
    with pytest.raises(zb.InvalidArgument):
        steps.build(toks(3), [0, 1, 2], [1, 1, 1], [1, 1, 1], [], 0)  # three requests
    with pytest.raises(zb.InvalidArgument):
        steps.build(toks(11), [0], [0], [11], [0], 1)        # eleven tokens


def test_step_tables_build_on_a_raw_stream(ctx, monkeypatch):
    """A raw handle is a stream of the context's device, whatever the current one is: the upload is held back for that
    device's stream. The batch is that of the current stream."""
    import torch
    from zealot_b200.decoder import StepTables
    seen, real = [], torch.cuda.ExternalStream

    def stream(handle, device=None, **rest):
        seen.append(device)
        return real(handle, device=device, **rest)

    monkeypatch.setattr(torch.cuda, "ExternalStream", stream)
    toks = torch.zeros(22, dtype=torch.int64, device="cuda")
    batches = []
    for raw in (False, True):
        steps = StepTables(ctx, 4, 4, 3, 30, 16, 32)
        own = torch.cuda.Stream()
        own.wait_stream(torch.cuda.current_stream())
        b = steps.build(toks, [2, 0, 3], [0, 0, 17], [20, 1, 1], [5, 6, 7], 2, stream=own.cuda_stream if raw else None)
        torch.cuda.synchronize()
        batches.append([getattr(b, n).clone() for n in ("slot_mapping", "cu_prefill", "block_tables", "seq_lens", "last_rows")])
    assert seen == [toks.device]
    assert all(torch.equal(x, y) for x, y in zip(*batches))
    import zealot_b200 as zb
    with pytest.raises(zb.OobBlockError):  # row 3 has no blocks yet for its 17 tokens
        ctx.check_status()


def test_step_tables_build_refuses_lengths_and_counts_that_are_none(ctx):
    import torch
    import zealot_b200 as zb
    from zealot_b200.decoder import StepTables
    steps = StepTables(ctx, 4, 4, 3, 30, 16, 32)
    toks = lambda n: torch.zeros(n, dtype=torch.int64, device="cuda")
    for tokens, query, num_prefill in ((4, [5], 2),        # more chunks than requests: a decode row of minus one
                                       (4, [2, 1], -1),    # counted from the end
                                       (2, [3, -1], 2),    # the sum fits, one length is none
                                       (0, [-1], 1)):
        with pytest.raises(zb.InvalidArgument):
            steps.build(toks(tokens), list(range(len(query))), [0] * len(query), query, [0], num_prefill)
    b = steps.build(toks(0), [0], [0], [0], [], 1)         # an empty prompt is one
    assert b.prefill_tokens == 0 and b.seq_lens.numel() == 0 and b.last_rows.tolist() == [0]
    ctx.check_status()
