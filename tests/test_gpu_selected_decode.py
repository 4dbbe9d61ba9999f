"""Decode over selected blocks on the GPU against the formula in 64 bits.

Tolerance, u = 2^-24. A score is off by at most (2 d + 4) u of its terms' absolute sum times
the scale (adds may drop a whole step), and its exponential by 8 u more and by the error of the
argument, which is rounded at the size of |s - m| log2(e): with e the largest such error of a row,
every weight is off by a factor within 1 +- 2 e, the result by 2 e sum(p |v|) twice (numerator and
denominator), and the sums over n tokens by (n + 8) u more. For bf16 the weights enter the
product as two bf16 parts (2^-17 of each is lost) and the result is rounded: 2^-8 of its value."""
import numpy as np
import pytest

from helpers import decode_case

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def plain(q, kp, vp, table, lens, selected, scale, modulo, bf16):
    """64 bits: (out, tolerance). Rows without tokens are zero."""
    B, H, d = q.shape
    nb, Hkv, bs, _ = kp.shape
    out, tol = np.zeros((B, H, d)), np.zeros((B, H, d))
    for b in range(B):
        for h in range(H):
            kv = h % Hkv if modulo else h // (H // Hkv)
            rows = []
            for j in selected[b, kv]:
                if j < 0:
                    break
                if j >= table.shape[1] or not 0 <= table[b, j] < nb:
                    continue
                rows += [(table[b, j], t) for t in range(bs) if j * bs + t < lens[b]]
            if not rows:
                continue
            ids, ts = np.array(rows).T
            k, v = kp[ids, kv, ts], vp[ids, kv, ts]
            s = k @ q[b, h] * scale
            m = s.max()
            p = np.exp(s - m)
            p /= p.sum()
            e = (2 * d + 4) * U * (np.abs(k) @ np.abs(q[b, h])).max() * scale + 8 * U + 4 * U * np.abs(s - m).max()
            e += 4 * U * np.abs(s).max() + (2.0 ** -17 if bf16 else 0)
            out[b, h] = p @ v
            tol[b, h] = (4 * e + (len(rows) + 8) * U) * (p @ np.abs(v)) + (2.0 ** -8 * np.abs(out[b, h]) if bf16 else 0)
    return out, tol


def lists(rng, lens, Hkv, bs, top, shuffle=False):
    """Distinct blocks of each sequence, a last one that may be part full among them."""
    out = np.full((len(lens), Hkv, top), -1, np.int32)
    for b, n in enumerate(lens):
        blocks = -(-n // bs)
        for h in range(Hkv):
            pick = rng.permutation(blocks)[:top]
            if blocks > top:
                pick[0] = blocks - 1 if blocks - 1 not in pick else pick[0]
            out[b, h, :len(pick)] = pick if shuffle else np.sort(pick)
    return out


def check(ctx, q, kp, vp, table, lens, selected, bf16, scale=0.0, modulo=False, reported=False):
    import torch
    import zealot_b200 as zb
    dt = torch.bfloat16 if bf16 else torch.float32
    tq, tk, tv = dev(q, dt), dev(kp, dt), dev(vp, dt)
    o = torch.full(q.shape, 9.0, dtype=dt, device="cuda")
    zb.CudaAttention(ctx).paged_forward_selected(tq, tk, tv, dev(table), dev(np.asarray(lens, np.int32)), dev(selected),
                                                 o, scale=scale, gqa_map=int(modulo))
    if reported:
        with pytest.raises(zb.OobBlockError):
            ctx.check_status()
    ctx.check_status()
    x = [t.double().cpu().numpy() for t in (tq, tk, tv)]
    want, tol = plain(*x, table, lens, selected, scale or q.shape[2] ** -0.5, modulo, bf16)
    got = o.double().cpu().numpy()
    err = np.abs(got - want)
    assert np.all(err <= tol), f"off by {np.nanmax(err / np.maximum(tol, 1e-300)):.2f} of the tolerance"
    return got


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("lens,H,Hkv,d,bs,top,modulo", [
    ([1], 32, 8, 128, 16, 1, False), ([1000, 17, 0, 16, 530], 32, 8, 128, 16, 20, False), ([4000], 64, 8, 128, 16, 128, False),
    ([700] * 40, 32, 8, 128, 16, 7, True), ([300, 77], 16, 16, 64, 16, 9, False), ([2000, 100, 65], 8, 1, 128, 32, 30, False),
    ([500, 33], 12, 4, 80, 16, 11, False), ([500, 33], 12, 4, 96, 8, 40, True), ([90, 300], 28, 4, 256, 64, 3, False),
    ([50, 9], 6, 3, 33, 5, 6, False), ([400], 20, 1, 128, 16, 25, False), ([100, 64], 40, 8, 128, 1, 70, False),
    ([100, 64], 9, 3, 64, 30, 4, False), ([40], 6, 2, 8, 16, 3, True), ([9000], 2, 2, 128, 16, 500, False),
    ([600, 20], 24, 2, 64, 16, 30, False), ([333], 4, 4, 112, 16, 12, False)])
def test_selected(ctx, lens, H, Hkv, d, bs, top, modulo, bf16):
    rng = np.random.default_rng(H * 100 + d + top)
    nb = int(sum(-(-n // bs) for n in lens)) + 3
    q, kp, vp, table, lens = decode_case(rng, len(lens), lens, H, Hkv, d, bs, nb)
    check(ctx, q, kp, vp, table, lens, lists(rng, lens, Hkv, bs, top), bf16, modulo=modulo)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("B", [15, 16, 33, 34, 71, 72, 75, 149])
def test_selected_lists_about_the_clusters_that_run_at_once(ctx, B, d, bf16):
    """Lists of 1,024 tokens, so that all cluster sizes are open to the choice."""
    rng = np.random.default_rng(B + d)
    q, kp, vp, _, _ = decode_case(rng, B, [1] * B, 2, 1, d, 64, 150)
    table = rng.integers(0, 150, (B, 16), dtype=np.int32)  # sequences that share blocks
    lens = np.array([1024 - i % 3 * 500 for i in range(B)], np.int32)
    check(ctx, q, kp, vp, table, lens, np.tile(np.arange(16, dtype=np.int32), (B, 1, 1)), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 8), (72, 5)])
def test_selected_odd_lists(ctx, d, bs, bf16):
    """Any order, an index twice, an empty list, a list ended early, blocks past the length."""
    rng = np.random.default_rng(d)
    lens = [400, 390, 64, 7, 300]
    q, kp, vp, table, lens = decode_case(rng, 5, lens, 8, 2, d, bs, 400, max_blocks=90)
    sel = lists(rng, lens, 2, bs, 30, shuffle=True)
    sel[0, 0, 3] = sel[0, 0, 5]
    sel[1, 0, 0] = -1            # nothing
    sel[1, 1, 7] = -7            # the rest is not read
    sel[1, 1, 9] = 10**9
    table[2, 80:] = 1
    sel[2, :, :3] = [80, 81, 0]  # blocks past the length, with a table entry
    sel[2, :, 3] = -1
    sel[3, 0, :] = 70            # only blocks past the length: zeros
    table[4, 2] = -1             # a block that is not there
    sel[4, :, :2] = [2, 0]
    got = check(ctx, q, kp, vp, table, lens, sel, bf16)
    assert np.all(got[1, :4] == 0) and np.all(got[3, :4] == 0)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,B", [(64, 40), (128, 3)])
def test_selected_long_lists(ctx, d, B, bf16):
    """Lists of more blocks than a CTA resolves at a time (512), ending in its first part, in its second
    and not at all; many lists (one CTA each) and few (eight CTAs each)."""
    rng = np.random.default_rng(B)
    top = 700 if B > 8 else 4800
    lens = [top + 60] * B
    q, kp, vp, table, lens = decode_case(rng, B, lens, 8, 4, d, 1, B * (top + 60))
    sel = lists(rng, lens, 4, 1, top)
    sel[0, :, 511] = -1
    sel[1, :, 512] = -1
    sel[1, 0, 600] = -2
    sel[2, 1, 600] = -1
    check(ctx, q, kp, vp, table, lens, sel, bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_selected_bad_ids(ctx, bf16):
    rng = np.random.default_rng(9)
    q, kp, vp, table, lens = decode_case(rng, 3, [200, 200, 200], 8, 2, 128, 16, 60)
    sel = lists(rng, lens, 2, 16, 6)
    table[0, sel[0, 0, 2]] = 60
    table[2, sel[2, 1, 0]] = 2**31 - 1
    check(ctx, q, kp, vp, table, lens, sel, bf16, reported=True)
    sel[1, 0, 1] = 13
    sel[1, 1, 1] = 2**31 - 1
    check(ctx, q, kp, vp, table, lens, sel, bf16, reported=True)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 8), (72, 5)])
def test_selected_masked_places_hold_anything(ctx, d, bs, bf16):
    """NaN and infinities in tokens past the length, in unselected blocks and in the rest of the pool."""
    import torch
    rng = np.random.default_rng(d + 1)
    lens = [37, 200, 1]
    q, kp, vp, table, lens = decode_case(rng, 3, lens, 8, 2, d, bs, 80)
    sel = lists(rng, lens, 2, bs, 5)
    for pool, bad in ((kp, np.nan), (vp, np.inf)):
        keep = np.zeros(pool.shape[:3], bool)
        for b in range(3):
            for h in range(2):
                for j in sel[b, h][sel[b, h] >= 0]:
                    keep[table[b, j], h, :max(0, min(bs, lens[b] - j * bs))] = True
        pool[~keep] = bad
    want_k, want_v = np.where(np.isfinite(kp), kp, 0), np.where(np.isfinite(vp), vp, 0)
    import zealot_b200 as zb
    dt = torch.bfloat16 if bf16 else torch.float32
    outs = []
    for a, b in ((kp, vp), (want_k, want_v)):
        o = torch.empty(q.shape, dtype=dt, device="cuda")
        zb.CudaAttention(ctx).paged_forward_selected(dev(q, dt), dev(a.astype(np.float32), dt), dev(b.astype(np.float32), dt),
                                                     dev(table), dev(lens), dev(sel), o)
        outs.append(o)
    assert torch.isfinite(outs[0]).all() and torch.equal(*outs)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("size", [30.0, 3000.0])
def test_selected_large_scores(ctx, bf16, size):
    """Scores far from zero, rising along the list: the running maximum moves in every tile."""
    rng = np.random.default_rng(2)
    q, kp, vp, table, lens = decode_case(rng, 2, [900, 700], 8, 2, 128, 16, 110)
    for b in range(2):
        for j in range(-(-lens[b] // 16)):
            kp[table[b, j]] *= size * j / 60
    check(ctx, q, kp, vp, table, lens, lists(rng, lens, 2, 16, 40), bf16)
    check(ctx, -q, kp, vp, table, lens, lists(rng, lens, 2, 16, 40), bf16, scale=1e-3)


@pytest.mark.parametrize("bf16", [True, False])
def test_selected_repeats_bit_for_bit(ctx, bf16):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(1)
    q, kp, vp, table, lens = decode_case(rng, 2, [5000, 3000], 32, 8, 128, 16, 510)
    sel = dev(lists(rng, lens, 8, 16, 200))
    dt = torch.bfloat16 if bf16 else torch.float32
    args = dev(q, dt), dev(kp, dt), dev(vp, dt), dev(table), dev(lens), sel
    outs = [torch.empty(q.shape, dtype=dt, device="cuda") for _ in range(5)]
    streams = [torch.cuda.Stream() for _ in range(5)]
    torch.cuda.synchronize()
    for o, s in zip(outs, streams):  # at the same time, on one context
        zb.CudaAttention(ctx).paged_forward_selected(*args, o, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs)


def test_selected_is_paged_decode_when_all_blocks_are_listed(ctx):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(6)
    q, kp, vp, table, lens = decode_case(rng, 3, [1000, 31, 512], 32, 8, 128, 16, 100)
    bf = torch.bfloat16
    args = dev(q, bf), dev(kp, bf), dev(vp, bf), dev(table), dev(lens)
    sel = np.full((3, 8, table.shape[1]), -1, np.int32)
    for b, n in enumerate(lens):
        sel[b, :, :-(-n // 16)] = np.arange(-(-n // 16))
    a, b = (torch.empty(q.shape, dtype=bf, device="cuda") for _ in range(2))
    attn = zb.CudaAttention(ctx)
    attn.paged_forward(*args, a, 3, 32, 8, 128, 16, table.shape[1])
    attn.paged_forward_selected(*args, dev(sel), b)
    # paged_forward rounds its weights to bf16 (2^-9 of each, over sums of |v| of about 1)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -6
    empty = torch.empty((3, 8, 0), dtype=torch.int32, device="cuda")
    attn.paged_forward_selected(*args, empty, b)
    assert torch.all(b == 0)
    ctx.check_status()


def test_closed_context_is_refused(ctx):
    import torch
    import zealot_b200 as zb
    other = zb.GpuContext(0)
    attn = zb.CudaAttention(other)
    scores = torch.zeros((1, 1, 4), device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    selected = torch.full((1, 1, 2), 5, dtype=torch.int32, device="cuda")
    attn.select_blocks(scores, lens, selected, 16)
    other.check_status()
    assert selected.tolist() == [[[-1, -1]]]
    other.close()
    with pytest.raises(zb.InvalidArgument, match="null context"):
        attn.select_blocks(scores, lens, selected, 16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("lens,d,bs,top", [([1], 128, 16, 1), ([60, 17], 128, 16, 4), ([60, 17], 64, 16, 4), ([60, 17], 256, 16, 4),
                                           ([60, 17], 72, 5, 12), ([60, 17], 33, 16, 4), ([5000], 128, 16, 300), ([40] * 90, 128, 8, 5)])
def test_selected_infinite_values(ctx, lens, d, bs, top, bf16):
    """Infinite and NaN values in places that count: infinity of the value's sign where all of them agree, NaN where they
    do not, whatever the token's weight (the scores here leave each token 2^-40 of its row or more), and the other
    elements as if nothing were there. In every kernel."""
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(len(lens) + d)
    H, Hkv = 8, 2
    nb = sum(-(-n // bs) for n in lens) + 3
    q, kp, vp, table, lens = decode_case(rng, len(lens), lens, H, Hkv, d, bs, nb)
    sel = lists(rng, lens, Hkv, bs, top)
    places = {}  # (sequence, kv head, element) -> values
    for b in range(len(lens)):
        for h in range(Hkv):
            tokens = [j * bs + t for j in sel[b, h] if j >= 0 for t in range(bs) if j * bs + t < lens[b]]
            for t, e, x in zip(rng.permutation(tokens * 8)[:8], (0, 1, 2, 3, 3, 4, 4, d - 1),
                               (np.inf, -np.inf, np.inf, np.inf, np.inf, np.inf, -np.inf, np.nan)):
                old = vp[table[b, t // bs], h, t % bs, e]
                vp[table[b, t // bs], h, t % bs, e] = x if np.isfinite(old) else old + x  # one token twice: both
                places.setdefault((b, h, e), []).append(x)
    dt = torch.bfloat16 if bf16 else torch.float32
    tq, tk, tv = dev(q, dt), dev(kp, dt), dev(vp, dt)
    o = torch.empty(q.shape, dtype=dt, device="cuda")
    zb.CudaAttention(ctx).paged_forward_selected(tq, tk, tv, dev(table), dev(lens), dev(sel), o)
    ctx.check_status()
    got = o.double().cpu().numpy()
    finite = torch.where(torch.isfinite(tv), tv, torch.zeros_like(tv))
    want, tol = plain(*(t.double().cpu().numpy() for t in (tq, tk, finite)), table, lens, sel, d ** -0.5, False, bf16)
    for (b, h, e), x in places.items():
        heads = slice(h * H // Hkv, (h + 1) * H // Hkv)
        assert np.array_equal(got[b, heads, e], np.full(H // Hkv, sum(x)), equal_nan=True), (b, h, e, x)
        got[b, heads, e] = want[b, heads, e] = 0
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 8), (256, 16), (72, 5), (33, 16), (8, 16)])
def test_selected_nan_reaches_the_output(ctx, d, bs, bf16):
    """A NaN in a query head: that head's row. Lists whose keys are all NaN, short or longer than one chunk of keys, and
    one NaN key among others: the kv head's rows. The rest as the formula has it."""
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(d)
    q, kp, vp, table, lens = decode_case(rng, 4, [60, 7, 400, 300], 8, 2, d, bs, 400)
    sel = lists(rng, lens, 2, bs, 400 // bs)
    dt = torch.bfloat16 if bf16 else torch.float32
    clean = [dev(x, dt).double().cpu().numpy() for x in (q, kp, vp)]
    want, tol = plain(*clean, table, lens, sel, d ** -0.5, False, bf16)
    q[0, 5, 0] = np.nan
    want[0, 5] = np.nan
    for b, h in ((1, 0), (2, 1)):
        for j in sel[b, h][sel[b, h] >= 0]:
            kp[table[b, j], h, :, d - 1] = np.nan
        want[b, 4 * h:4 * h + 4] = np.nan
    j = sel[3, 0, 2]
    kp[table[3, j], 0, 1, 0] = np.nan
    want[3, :4] = np.nan
    o = torch.full(q.shape, 9.0, dtype=dt, device="cuda")
    zb.CudaAttention(ctx).paged_forward_selected(dev(q, dt), dev(kp, dt), dev(vp, dt), dev(table), dev(lens), dev(sel), o)
    ctx.check_status()
    got = o.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.all(np.abs(got - want)[ok] <= tol[ok])
