"""Block bounds, block scores and block selection on the GPU.

Bounds and selections are exact. A score is a sum of 2 d products, each exact in fp32 for
bf16 inputs and rounded once (u = 2^-24) for fp32 ones; sums of 2 d terms in any order, with
adds that may drop up to a whole step (2 u), and the scale's product are off by at most
(4 d + 4) u of the terms' absolute sum."""
import numpy as np
import pytest

from helpers import decode_case

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


SHAPES = [  # lens, H, Hkv, d, bs
    ([1], 32, 8, 128, 16), ([40, 16, 0, 17, 1000], 32, 8, 128, 16), ([300, 1, 2000], 64, 8, 128, 16),
    ([129, 5], 16, 16, 64, 8), ([500, 31, 32, 33], 8, 1, 128, 32), ([77, 130], 12, 4, 80, 16),
    ([90, 300], 6, 2, 96, 64), ([50, 9], 3, 3, 33, 5), ([1000], 20, 2, 128, 16), ([200, 64], 28, 4, 256, 16),
    ([70], 6, 1, 8, 1), ([3000] * 3, 40, 8, 128, 16), ([64, 65], 24, 2, 72, 16)]


def keys(rng, lens, H, Hkv, d, bs, bf16, max_blocks=None):
    import torch
    dt = torch.bfloat16 if bf16 else torch.float32
    nb = int(sum(-(-n // bs) for n in lens)) + 3
    q, kp, _, table, lens = decode_case(rng, len(lens), lens, H, Hkv, d, bs, nb, max_blocks)
    return dev(q, dt), dev(kp, dt), dev(table), dev(lens), nb


def plain_bounds(kp, table, lens, begin, bounds, bs):
    """One block at a time, on the values as float32 (the minimum of bf16 values is one of them)."""
    kp, out = kp.float().cpu().numpy(), bounds.float().cpu().numpy().copy()
    for b, n in enumerate(lens):
        for j in range(max(begin[b], 0) // bs if begin is not None else 0, -(-int(n) // bs)):
            if j >= table.shape[1] or not 0 <= table[b, j] < kp.shape[0]:
                continue
            x = kp[table[b, j], :, :min(bs, int(n) - j * bs)]
            out[table[b, j], :, 0], out[table[b, j], :, 1] = x.min(1), x.max(1)
    return out


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("lens,H,Hkv,d,bs", SHAPES)
def test_bounds(ctx, lens, H, Hkv, d, bs, bf16):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(d + bs)
    _, kp, table, tl, nb = keys(rng, lens, H, Hkv, d, bs, bf16)
    for begin in (None, [max(n - 1, 0) for n in lens], [n // 2 for n in lens], [n for n in lens], [-3 for n in lens]):
        bounds = torch.full((nb, Hkv, 2, d), 7.0, dtype=kp.dtype, device="cuda")
        want = plain_bounds(kp, table.cpu().numpy(), lens, begin, bounds, bs)
        zb.CudaAttention(ctx).block_bounds(kp, table, tl, bounds,
                                           tok_begin=None if begin is None else dev(np.array(begin, np.int32)))
        ctx.check_status()
        assert np.array_equal(bounds.float().cpu().numpy(), want), begin


@pytest.mark.parametrize("bf16", [True, False])
def test_bounds_special(ctx, bf16):
    """NaN keys, infinities, -0, a table entry that is not there, an id outside the pool and a length past the table."""
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(3)
    _, kp, table, tl, nb = keys(rng, [64, 64, 64, 64], 4, 2, 64, 16, bf16)
    t = table.cpu().numpy()
    kp[t[0, 1], 0, 3, 5] = float("nan")
    kp[t[0, 2], 1, 0, 9] = float("-inf")
    kp[t[0, 2], 1, 1, 9] = float("inf")
    t[1, 2] = -1
    t[2, 0] = nb
    table.copy_(torch.from_numpy(t))
    lens = [64, 64, 64, 900]
    bounds = torch.full((nb, 2, 2, 64), 7.0, dtype=kp.dtype, device="cuda")
    want = plain_bounds(kp, t, lens, None, bounds, 16)
    zb.CudaAttention(ctx).block_bounds(kp, table, dev(np.array(lens, np.int32)), bounds)
    with pytest.raises(zb.OobBlockError):
        ctx.check_status()
    got = bounds.float().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got).sum() == 2
    assert got[t[0, 2], 1, 0, 9] == -np.inf and got[t[0, 2], 1, 1, 9] == np.inf


def plain_scores(q, bounds, table, lens, Hkv, bs, scale, modulo):
    """64 bits: (scores, their tolerance)."""
    q, bounds = q.double().cpu().numpy(), bounds.double().cpu().numpy()
    B, H, d = q.shape
    out = np.full((B, Hkv, table.shape[1]), -np.inf)
    tol = np.zeros_like(out)
    for b in range(B):
        n = min(-(-int(lens[b]) // bs), table.shape[1]) if lens[b] > 0 else 0
        ids = table[b, :n]
        ok = (ids >= 0) & (ids < bounds.shape[0])
        for h in range(H):
            kv = h % Hkv if modulo else h // (H // Hkv)
            e = bounds[np.where(ok, ids, 0), kv]
            terms = np.maximum(q[b, h], 0) * e[:, 1] + np.minimum(q[b, h], 0) * e[:, 0]
            s = np.where(ok, terms.sum(1) * scale, -np.inf)
            out[b, kv, :n] = np.maximum(out[b, kv, :n], s)
            tol[b, kv, :n] = np.maximum(tol[b, kv, :n], (4 * d + 4) * 2.0 ** -24 * np.abs(terms).sum(1) * scale)
    return out, tol


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("modulo", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,d,bs", SHAPES)
def test_scores(ctx, lens, H, Hkv, d, bs, modulo, bf16):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(d * 3 + bs)
    q, kp, table, tl, nb = keys(rng, lens, H, Hkv, d, bs, bf16, max_blocks=-(-max(lens) // bs) + (3 if modulo else 0))
    bounds = torch.zeros((nb, Hkv, 2, d), dtype=kp.dtype, device="cuda")
    attn = zb.CudaAttention(ctx)
    attn.block_bounds(kp, table, tl, bounds)
    scores = torch.full((len(lens), Hkv, table.shape[1]), 5.0, device="cuda")
    scale = 0.0 if modulo else 0.3
    attn.block_scores(q, bounds, table, tl, scores, bs, scale=scale, gqa_map=int(modulo))
    ctx.check_status()
    want, tol = plain_scores(q, bounds, table.cpu().numpy(), lens, Hkv, bs, scale or d ** -0.5, modulo)
    got = scores.double().cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    assert np.all(np.abs(got - want)[~inf] <= tol[~inf])
    # no attention score of a block is above its bound
    qh, kh = q.double().cpu().numpy(), kp.double().cpu().numpy()
    t = table.cpu().numpy()
    for b, n in enumerate(lens):
        for j in range(-(-n // bs)):
            for h in range(H):
                kv = h % Hkv if modulo else h // (H // Hkv)
                s = kh[t[b, j], kv, :min(bs, n - j * bs)] @ qh[b, h] * (scale or d ** -0.5)
                assert s.max() <= got[b, kv, j] + tol[b, kv, j]
            if j > 40:
                break


@pytest.mark.parametrize("bf16", [True, False])
def test_scores_special(ctx, bf16):
    """A NaN bound gives a NaN score; blocks that are not there, outside the pool or past the table -inf."""
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(4)
    q, kp, table, tl, nb = keys(rng, [64, 64, 64, 64, 0], 8, 2, 128, 16, bf16)
    bounds = torch.randn((nb, 2, 2, 128), device="cuda").to(kp.dtype)
    t = table.cpu().numpy()
    bounds[t[0, 1], 0, :, 5] = float("nan")
    t[1, 2] = -1
    t[2, 0] = nb + 5
    table.copy_(torch.from_numpy(t))
    lens = np.array([64, 64, 64, 70, -9], np.int32)
    scores = torch.full((5, 2, 4), 5.0, device="cuda")
    zb.CudaAttention(ctx).block_scores(q, bounds, table, dev(lens), scores, 16)
    with pytest.raises(zb.OobBlockError):
        ctx.check_status()
    got = scores.double().cpu().numpy()
    assert np.isnan(got[0, 0, 1]) and np.isnan(got).sum() == 1
    assert np.all(got[1, :, 2] == -np.inf) and np.all(got[2, :, 0] == -np.inf) and np.all(got[4] == -np.inf)
    assert np.isinf(got).sum() == 2 + 2 + 8
    bounds[t[0, 1], 0] = 0
    want, tol = plain_scores(q, bounds, t, lens, 2, 16, 128 ** -0.5, False)
    ok = np.isfinite(got)
    assert np.all(np.abs(got - want)[ok] <= tol[ok])


def plain_select(scores, lens, bs, top, first, last):
    B, Hkv, mb = scores.shape
    out = np.full((B, Hkv, top), -1, np.int32)
    key = np.where(np.isnan(scores), np.inf, scores)  # NaN above every score, inf included
    for b in range(B):
        n = min(-(-int(lens[b]) // bs), mb) if lens[b] > 0 else 0
        for h in range(Hkv):
            if n <= top:
                out[b, h, :n] = np.arange(n)
                continue
            mid = np.arange(first, n - last)
            order = sorted(mid, key=lambda j: (not np.isnan(scores[b, h, j]), -key[b, h, j], j))
            pick = list(range(first)) + order[:top - first - last] + list(range(n - last, n))
            out[b, h] = np.sort(pick)
    return out


@pytest.mark.parametrize("kind", ["normal", "ties", "equal", "special"])
@pytest.mark.parametrize("lens,Hkv,bs,top,first,last,mb", [
    ([1000, 17, 0, 16, 530], 8, 16, 32, 1, 2, 70), ([5], 1, 16, 1, 0, 0, 1), ([500], 1, 16, 1, 0, 1, 32),
    ([500], 2, 16, 1, 1, 0, 40), ([4000, 3999], 2, 8, 300, 0, 0, 500), ([700, 90], 3, 1, 64, 5, 7, 701),
    ([131072], 2, 16, 256, 1, 4, 8192), ([900] * 70, 4, 16, 20, 2, 2, 57), ([600], 1, 16, 6, 3, 3, 38),
    ([20000], 1, 1, 5000, 1, 1, 20000), ([65536, 70000], 1, 1, 777, 1, 1, 70001), ([33 * 16], 1, 16, 32, 0, 1, 33)])
def test_select(ctx, lens, Hkv, bs, top, first, last, mb, kind):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(len(lens) + top)
    scores = rng.standard_normal((len(lens), Hkv, mb)).astype(np.float32)
    if kind == "ties":
        scores = np.round(scores * 2) / 2
    elif kind == "equal":
        scores[:] = 0.0
        scores[..., ::2] = -0.0
    elif kind == "special":
        scores[..., ::3] = -np.inf
        scores[..., 1::50] = np.nan
        scores[..., 7::60] = np.inf
        scores[..., 5::40] = np.float32(-3.4028235e38)
    selected = torch.full((len(lens), Hkv, top), 9, dtype=torch.int32, device="cuda")
    zb.CudaAttention(ctx).select_blocks(dev(scores), dev(np.array(lens, np.int32)), selected, bs, num_first=first,
                                        num_last=last)
    ctx.check_status()
    assert np.array_equal(selected.cpu().numpy(), plain_select(scores, lens, bs, top, first, last))


def test_select_length_past_table(ctx):
    import torch
    import zealot_b200 as zb
    scores = torch.randn((2, 1, 10), device="cuda")
    selected = torch.empty((2, 1, 4), dtype=torch.int32, device="cuda")
    zb.CudaAttention(ctx).select_blocks(scores, dev(np.array([161, -7], np.int32)), selected, 16)
    with pytest.raises(zb.OobBlockError):
        ctx.check_status()
    assert np.array_equal(selected.cpu().numpy(), plain_select(scores.cpu().numpy(), [160, 0], 16, 4, 1, 1))


@pytest.mark.parametrize("kind", ["normal", "ties", "equal", "special"])
@pytest.mark.parametrize("rows,top,first,last,mb", [
    (40, 64, 1, 2, 1025), (40, 200, 0, 0, 2048), (5, 1, 0, 0, 1600), (400, 50, 2, 3, 2049), (330, 256, 1, 4, 8192),
    (320, 700, 0, 1, 5000), (7, 256, 1, 1, 2049), (6, 100, 1, 0, 4099), (9, 300, 2, 2, 8193), (8, 256, 1, 4, 16384),
    (4, 900, 0, 0, 12001), (5, 64, 1, 1, 16385), (3, 64, 1, 1, 24577)])
def test_select_wide_tables(ctx, rows, top, first, last, mb, kind):
    """Each range of widths that has a kernel of its own, with few rows and with more than the GPU takes at once; rows of
    every length, some of them with nothing to choose from."""
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(mb + rows)
    lens = rng.integers(0, mb + 1, rows) * 8 - rng.integers(0, 8, rows)
    lens[0], lens[-1] = mb * 8, min(top + 1, mb) * 8
    scores = rng.standard_normal((rows, 1, mb)).astype(np.float32)
    if kind == "ties":
        scores = np.round(scores * 4) / 4
    elif kind == "equal":
        scores[:] = 1.5
    elif kind == "special":
        scores[..., ::3] = -np.inf
        scores[..., 1::500] = np.nan
        scores[..., 7::600] = np.inf
        scores[..., 5::40] = np.float32(-3.4028235e38)
        scores[..., 6::40] = np.float32(1e-45)
    want = np.full((rows, 1, top), -1, np.int32)
    for b in range(rows):
        n = max(0, -(-int(lens[b]) // 8))
        if n <= top:
            want[b, 0, :n] = np.arange(n)
            continue
        mid = np.arange(first, n - last)
        s = scores[b, 0, mid]
        nan = np.isnan(s)
        order = mid[np.lexsort((mid, -np.where(nan, 0, s), ~nan))]
        want[b, 0] = np.sort(np.concatenate([np.arange(first), order[:top - first - last], np.arange(n - last, n)]))
    selected = torch.full((rows, 1, top), 9, dtype=torch.int32, device="cuda")
    zb.CudaAttention(ctx).select_blocks(dev(scores), dev(lens.astype(np.int32)), selected, 8, num_first=first, num_last=last)
    ctx.check_status()
    assert np.array_equal(selected.cpu().numpy(), want)


@pytest.mark.parametrize("lens,H,Hkv,d,bs", [([90, 300, 0], 9, 1, 256, 16), ([500, 31], 24, 2, 160, 8), ([77], 40, 4, 256, 64),
                                             ([200, 64], 34, 2, 136, 16)])
@pytest.mark.parametrize("bf16", [True, False])
def test_scores_of_many_heads_of_more_than_128(ctx, lens, H, Hkv, d, bs, bf16):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(d * 5 + bs)
    q, kp, table, tl, nb = keys(rng, lens, H, Hkv, d, bs, bf16, max_blocks=-(-max(lens) // bs) + 2)
    bounds = torch.zeros((nb, Hkv, 2, d), dtype=kp.dtype, device="cuda")
    attn = zb.CudaAttention(ctx)
    attn.block_bounds(kp, table, tl, bounds)
    scores = torch.full((len(lens), Hkv, table.shape[1]), 5.0, device="cuda")
    attn.block_scores(q, bounds, table, tl, scores, bs)
    ctx.check_status()
    want, tol = plain_scores(q, bounds, table.cpu().numpy(), lens, Hkv, bs, d ** -0.5, False)
    got = scores.double().cpu().numpy()
    there = np.isfinite(want)
    assert np.array_equal(got[~there], want[~there])
    assert np.all(np.abs(got[there] - want[there]) <= tol[there])
