"""Offsets past 32 bits: the operators around the paged cache on pools of more than 2^31 elements, of
which only the last blocks are used. The same call on a small pool that holds just those blocks gives
the same bytes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _pools(num_blocks, used, Hkv, bs, d, dtype, seed):
    """(large, small): a pool whose last `used` blocks are those of the small one."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    small = torch.randn((used, Hkv, bs, d), generator=g, device="cuda").to(dtype)
    large = torch.empty((num_blocks, Hkv, bs, d), dtype=dtype, device="cuda")
    large[num_blocks - used:] = small
    return large, small


@pytest.mark.parametrize("dtype,num_blocks,Hkv,bs,d", [("bfloat16", 140000, 8, 16, 128), ("float32", 70000, 8, 16, 256),
                                                       ("bfloat16", 1200000, 2, 16, 72)])
def test_pool_offsets_past_32_bits(ctx, dtype, num_blocks, Hkv, bs, d):
    import torch
    import zealot_b200 as zb
    dtype = getattr(torch, dtype)
    assert num_blocks * Hkv * bs * d > 2**31
    attn, used, H, lens = zb.CudaAttention(ctx), 40, 2 * Hkv, [300, 17, 320]
    rng = np.random.default_rng(d)
    table = np.full((3, 20), -1, np.int32)
    perm = rng.permutation(used).astype(np.int32)
    table[0, :19], table[1, :2], table[2, :19] = perm[:19], perm[19:21], perm[21:40]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    tl = dev(np.array(lens, np.int32).clip(max=304))
    (k, ks), (v, vs) = _pools(num_blocks, used, Hkv, bs, d, dtype, 1), _pools(num_blocks, used, Hkv, bs, d, dtype, 2)
    far = num_blocks - used
    far_table = np.where(table >= 0, table + far, -1).astype(np.int32)
    q = torch.randn((3, H, d), device="cuda").to(dtype)
    x = torch.randn((3, H + 2 * Hkv, d), device="cuda").to(dtype)
    pos = tl - 1
    freq = dev(10000.0 ** (-np.arange(0, d // 2, 2) / (d // 2)))
    results = []
    for kp, vp, t, n in ((k, v, far_table, num_blocks), (ks, vs, table, used)):
        last = t[np.arange(3), [18, 1, 18]].astype(np.int64)
        slots = dev(last * bs + np.array([299 % 16, 0, 303 % 16]))
        attn.qk_norm_rope(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], pos, freq, k_pool=kp, v_pool=vp, slot_mapping=slots)
        bounds = torch.empty((n, Hkv, 2, d), dtype=dtype, device="cuda")
        attn.block_bounds(kp, dev(t), tl, bounds)
        scores = torch.empty((3, Hkv, 20), device="cuda")
        attn.block_scores(q, bounds, dev(t), tl, scores, bs)
        sel = torch.empty((3, Hkv, 6), dtype=torch.int32, device="cuda")
        attn.select_blocks(scores, tl, sel, bs)
        o = torch.empty_like(q)
        attn.paged_forward_selected(q, kp, vp, dev(t), tl, sel, o)
        ctx.check_status()
        results.append((kp[n - used:].clone(), vp[n - used:].clone(), bounds[n - used:][:, :, :, :].clone(), scores, sel, o))
        del bounds
    for name, a, b in zip(("k", "v", "bounds", "scores", "selected", "out"), *results):
        if name == "bounds":  # only blocks of the tables are written
            a, b = a[perm], b[perm]
        assert torch.equal(a, b), name
    assert torch.isfinite(results[0][5]).all()


def test_bounds_offsets_past_32_bits(ctx):
    """Bounds of more than 2^31 elements (blocks of one token)."""
    import torch
    import zealot_b200 as zb
    num_blocks, used, Hkv, d = 1100000, 64, 8, 128
    assert num_blocks * Hkv * 2 * d > 2**31
    attn = zb.CudaAttention(ctx)
    k, ks = _pools(num_blocks, used, Hkv, 1, d, torch.bfloat16, 3)
    q = torch.randn((1, 16, d), device="cuda").to(torch.bfloat16)
    table = torch.randperm(used).to(torch.int32).cuda()[None]
    lens = torch.tensor([used], dtype=torch.int32, device="cuda")
    results = []
    for kp, t, n in ((k, table + (num_blocks - used), num_blocks), (ks, table, used)):
        bounds = torch.empty((n, Hkv, 2, d), dtype=torch.bfloat16, device="cuda")
        attn.block_bounds(kp, t, lens, bounds)
        scores = torch.empty((1, Hkv, used), device="cuda")
        attn.block_scores(q, bounds, t, lens, scores, 1)
        ctx.check_status()
        results.append((bounds[n - used:].clone(), scores))
        del bounds
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
