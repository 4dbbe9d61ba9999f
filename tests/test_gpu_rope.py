"""Norm, rotation and cache write on the GPU against the formula in 64 bits.

Tolerance. With u = 2^-24 (half a step of fp32): a sum of squares adds up to max(8, d/32)
products in a lane and five sums over lanes, so it is off by at most (d/32 + 13) u, mean and
eps add 2 u, and the root halves that; root, its correction and two products add 4 u; cos and
sin are off by at most 5 u (the reduced angle, below pi, is rounded to fp32: pi u, and the
functions' own 2 u); the two products and their sum add 3 u. So each result is within
C u (|a| + |b|), C = d/64 + 20, of the pair (a, b) that it is turned from, and rounding to
bf16 adds half a step, 2^-8 of the value."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def formula(x, w, eps, pos, freq, inter):
    """x [T][heads][d] in 64 bits -> (result, the scale of its rounding errors)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w.astype(np.float64)
    y, scale = x.copy(), np.abs(x)
    half = len(freq)
    ia, ib = (np.arange(half) * 2, np.arange(half) * 2 + 1) if inter else (np.arange(half), np.arange(half) + half)
    ang = (pos.astype(np.float64)[:, None] * freq)[:, None]
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
    scale[..., ia] = scale[..., ib] = np.abs(a) + np.abs(b)
    return y, scale


def near(got, want, bf16, d):
    y, scale = want
    tol = (d / 64 + 20) * U * scale + (2.0 ** -8 * np.abs(y) if bf16 else 0)
    err = np.abs(got.double().cpu().numpy() - y)
    assert np.all(err <= tol), f"off by {np.max(err / np.maximum(tol, 1e-300)):.2f} of the tolerance"


def make(T, H, Hkv, d, bf16, seed=0, extra=0):
    """A projection's rows [q | k | v | extra], and views of its parts."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if bf16 else torch.float32
    row = torch.randn((T, (H + 2 * Hkv) * d + extra), generator=g, device="cuda").to(dt)
    q, k, v = (row[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2)]
    return row, q, k, v, w


def freqs(rot, base=10000.0):
    return base ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1))


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,H,Hkv,d,rot,inter,norm,far", [
    (1, 32, 8, 128, 128, False, True, 131072), (64, 32, 8, 128, 128, False, True, 4096),
    (37, 16, 16, 64, 64, False, False, 1000000), (5, 4, 4, 8, 8, False, True, 32), (19, 12, 4, 96, 48, False, True, 9999),
    (33, 28, 4, 128, 64, True, True, 131072), (9, 8, 1, 256, 256, False, True, 4096), (9, 8, 1, 256, 256, True, True, 70000),
    (13, 6, 2, 80, 80, False, True, 4096), (13, 6, 2, 80, 40, True, False, 4096), (11, 3, 1, 72, 16, False, True, 100),
    (7, 3, 3, 33, 10, False, True, 100), (7, 3, 3, 33, 32, True, True, 100), (3, 2, 1, 1, 0, False, True, 10),
    (300, 40, 8, 128, 128, False, True, 2**31 - 1), (1000, 5, 1, 64, 0, False, True, 10), (2, 1, 1, 120, 8, False, True, 50),
    # enough tokens for several to a CTA: rows that fill their lanes and rows that do not, heads that share the groups
    # evenly and heads that do not, a last CTA with fewer tokens
    (2503, 8, 1, 96, 96, False, True, 4096), (1777, 12, 4, 64, 64, False, True, 9999), (1301, 3, 1, 256, 256, True, True, 500),
    (3001, 8, 2, 80, 40, True, True, 4096), (2049, 28, 4, 128, 64, False, False, 70000), (1999, 40, 8, 72, 24, False, True, 100),
    (1500, 1, 1, 8, 8, False, True, 100), (4001, 16, 16, 48, 0, False, True, 10), (1400, 70, 2, 128, 128, False, True, 1000)])
def test_norm_rotate_and_cache(ctx, T, H, Hkv, d, rot, inter, norm, far, bf16):
    import torch
    import zealot_b200 as zb
    rng = np.random.default_rng(T * 7 + d)
    _, q, k, v, w = make(T, H, Hkv, d, bf16, seed=d)
    wq, wk = w if norm else (None, None)
    pos = rng.integers(0, far, T).astype(np.int32)
    pos[0] = far - 1
    freq = freqs(rot)
    bs, nb = 16, T // 16 + 4
    slots = rng.permutation(nb * bs)[:T].astype(np.int64)
    slots[1::5] = -1
    pools = [torch.randn((nb, Hkv, bs, d), device="cuda").to(q.dtype) for _ in range(2)]
    before = [p.clone() for p in pools]
    out = [torch.full((T, n, d), 9.0, dtype=q.dtype, device="cuda") for n in (H, Hkv, Hkv)]
    dev = lambda a: torch.from_numpy(a).cuda()
    zb.CudaAttention(ctx).qk_norm_rope(q, k, v, dev(pos), dev(freq) if rot else None, *out, q_weight=wq, k_weight=wk,
                                       eps=1e-5, interleaved=inter, k_pool=pools[0], v_pool=pools[1],
                                       slot_mapping=dev(slots))
    ctx.check_status()
    host = lambda t: None if t is None else t.float().cpu().numpy()
    near(out[0], formula(host(q), host(wq), 1e-5, pos, freq, inter), bf16, d)
    near(out[1], formula(host(k), host(wk), 1e-5, pos, freq, inter), bf16, d)
    assert torch.equal(out[2], v)
    for pool, old, new in zip(pools, before, out[1:]):  # the same bytes at the slots, and nothing else
        for t in np.nonzero(slots >= 0)[0]:
            old[slots[t] // bs, :, slots[t] % bs] = new[t]
        assert torch.equal(pool, old)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("extra", [0, 8, 1])
def test_strides(ctx, bf16, extra):
    """Rows with something behind them; one element more puts every other row off 16 bytes."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(21, 8, 2, 64, bf16, extra=extra)
    pos = torch.arange(21, dtype=torch.int32, device="cuda")
    freq = torch.from_numpy(freqs(64)).cuda()
    out = [torch.empty((21, n, 64), dtype=q.dtype, device="cuda") for n in (8, 2, 2)]
    packed = [torch.empty_like(o) for o in out]
    attn = zb.CudaAttention(ctx)
    attn.qk_norm_rope(q, k, v, pos, freq, *out, q_weight=w[0], k_weight=w[1])
    attn.qk_norm_rope(q.contiguous(), k.contiguous(), v.contiguous(), pos, freq, *packed, q_weight=w[0], k_weight=w[1])
    # Other alignments may take another kernel. Both results are within C u (|a| + |b|) plus half a
    # bf16 step of the formula's y, so they differ by at most twice that: with normed rows of 64,
    # |a| + |b| <= 2 * 8 * 1.8 (weights below 1.8), and a whole step of bf16 is 2^-7 of the larger.
    for x, y in zip(out, packed):
        x, y = x.double().cpu().numpy(), y.double().cpu().numpy()
        step = 2.0 ** -7 * np.maximum(np.abs(x), np.abs(y)) if bf16 else 0
        assert np.all(np.abs(x - y) <= step + 2 * (64 / 64 + 20) * U * 2 * 8 * 1.8)
    assert w[0].max() < 1.8 and w[1].max() < 1.8
    near(out[0], formula(q.float().cpu().numpy(), w[0].float().cpu().numpy(), 1e-6, pos.cpu().numpy(), freqs(64), False),
         bf16, 64)
    assert torch.equal(out[2], v)


@pytest.mark.parametrize("d,rot,inter", [(128, 128, False), (64, 32, True), (80, 80, False), (33, 32, False)])
def test_in_place(ctx, d, rot, inter):
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(50, 8, 2, d, True)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = torch.arange(50, dtype=torch.int32, device="cuda") * 31
    freq = torch.from_numpy(freqs(rot)).cuda()
    out = [torch.empty_like(t) for t in (q, k, v)]
    attn = zb.CudaAttention(ctx)
    attn.qk_norm_rope(q, k, v, pos, freq, *out, q_weight=w[0], k_weight=w[1], interleaved=inter)
    attn.qk_norm_rope(q, k, v, pos, freq, q, k, v, q_weight=w[0], k_weight=w[1], interleaved=inter)
    for a, b in zip(out, (q, k, v)):
        assert torch.equal(a, b)


def test_parts_and_bad_slots(ctx):
    """Only the queries; only the pools; a slot outside the pool is reported and the others written."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(4, 8, 2, 64, True)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    freq = torch.from_numpy(freqs(64)).cuda()
    attn = zb.CudaAttention(ctx)
    full = [torch.empty((4, n, 64), dtype=q.dtype, device="cuda") for n in (8, 2, 2)]
    attn.qk_norm_rope(q, k, v, pos, freq, *full, q_weight=w[0], k_weight=w[1])
    only = torch.empty_like(full[0])
    attn.qk_norm_rope(q, k, v, pos, freq, q_out=only, q_weight=w[0], k_weight=w[1])
    assert torch.equal(only, full[0])
    ctx.check_status()
    pools = [torch.zeros((2, 2, 16, 64), dtype=q.dtype, device="cuda") for _ in range(2)]
    slots = torch.tensor([3, 32, 2**40, 31], dtype=torch.int64, device="cuda")
    attn.qk_norm_rope(q, k, v, pos, freq, q_weight=w[0], k_weight=w[1], k_pool=pools[0], v_pool=pools[1],
                      slot_mapping=slots)
    with pytest.raises(zb.OobBlockError):
        ctx.check_status()
    for pool, new in zip(pools, full[1:]):
        want = torch.zeros_like(pool)
        want[0, :, 3], want[1, :, 15] = new[0], new[3]
        assert torch.equal(pool, want)


def test_special_values(ctx):
    """Zero rows stay zero (eps keeps them finite); NaN and infinity stay in their own head."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(3, 4, 2, 64, True)
    q, k = q.clone(), k.clone()
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    k[2, 0, 7] = float("inf")
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    out = [torch.empty((3, n, 64), dtype=q.dtype, device="cuda") for n in (4, 2)]
    zb.CudaAttention(ctx).qk_norm_rope(q, k, v, pos, torch.from_numpy(freqs(64)).cuda(), *out, q_weight=w[0],
                                       k_weight=w[1])
    assert torch.all(out[0][0, 1] == 0)
    assert torch.isnan(out[0][1, 2]).all()
    clean = torch.isfinite(out[0]).all(-1)
    clean[1, 2] = True
    assert clean.all()
    assert torch.isfinite(out[1]).all(-1).sum() == 5


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,d", [(3, 128), (3000, 128), (3, 33)])
def test_squares_past_the_range(ctx, T, d, bf16):
    """A row whose squares add up to infinity is divided by it, in every kernel: 0, NaN where it is infinite itself.
    Without eps a row of zeros is 0 / 0."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(T, 2, 1, d, bf16)
    q, k = q.clone(), k.clone()
    q[0, 0, 5] = 1e30
    q[1, 1, 7] = -float("inf")
    k[2, 0] = 0
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    zb.CudaAttention(ctx).qk_norm_rope(q, k, v, None, None, q_out=qo, k_out=ko, q_weight=w[0], k_weight=w[1], eps=0.0)
    ctx.check_status()
    assert torch.all(qo[0, 0] == 0)
    assert torch.isnan(qo[1, 1, 7]) and torch.all(qo[1, 1, :7] == 0) and torch.all(qo[1, 1, 8:] == 0)
    assert torch.all(torch.isnan(ko[2]))
    assert torch.all(torch.isfinite(ko[:2])) and torch.all(torch.isfinite(qo[0])) and torch.all(torch.isfinite(qo[2:]))


def test_refusals(ctx):
    import torch
    import zealot_b200 as zb
    row, q, k, v, w = make(4, 8, 2, 64, True)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    freq = torch.from_numpy(freqs(64)).cuda()
    o = torch.empty((4, 8, 64), dtype=q.dtype, device="cuda")
    attn = zb.CudaAttention(ctx)
    pool = torch.zeros((2, 2, 16, 64), dtype=q.dtype, device="cuda")
    for bad in (dict(q_out=o[:, :4].contiguous()), dict(q_out=o.float()), dict(q_weight=w[0][:32].contiguous(), q_out=o),
                dict(q_out=o, k_pool=pool), dict(q_out=o, k_pool=pool, v_pool=pool, slot_mapping=pos), dict()):
        with pytest.raises(zb.InvalidArgument):
            attn.qk_norm_rope(q, k, v, pos, freq, **bad)
    for args in ((q.transpose(1, 2), k, v, pos, freq), (q, k, v, pos.long(), freq), (q, k, v, pos, freq.float()),
                 (q, k, v, pos[:3], freq), (q, k[..., :32], v, pos, freq), (q.float(), k, v, pos, freq),
                 (q, k, v, pos, torch.zeros(33, dtype=torch.float64, device="cuda"))):
        with pytest.raises(zb.InvalidArgument):
            attn.qk_norm_rope(*args, q_out=o)


def c_call(ctx, **args):
    """zl_qk_norm_rope by its C signature; what is not named is NULL or 0. Tensors give their addresses."""
    order = ("q k v q_stride k_stride v_stride q_weight k_weight eps positions inv_freq rotary_dim interleaved q_out k_out "
             "v_out k_pool v_pool slot_mapping block_size num_blocks num_tokens num_heads num_kv_heads head_dim dtype stream").split()
    assert not set(args) - set(order)
    value = lambda x: x.data_ptr() if hasattr(x, "data_ptr") else x
    return ctx.lib.zl_qk_norm_rope(ctx.handle, *(value(args.get(n, 0.0 if n == "eps" else 0)) for n in order))


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,d", [(3, 64), (2000, 64), (3, 33)])
def test_values_alone_need_no_positions(ctx, T, d, bf16):
    """A model's rotary size with only values to move, in each kernel: no angle is needed, so no position is read."""
    import torch
    _, _, _, v, _ = make(T, 2, 3, d, bf16)
    out = torch.empty((T, 3, d), dtype=v.dtype, device="cuda")
    assert c_call(ctx, v=v, v_stride=v.stride(0), rotary_dim=d // 2 * 2, v_out=out, num_tokens=T, num_heads=2, num_kv_heads=3,
                  head_dim=d, q_stride=2 * d, dtype=int(bf16), stream=torch.cuda.current_stream().cuda_stream) == 0
    ctx.check_status()
    assert torch.equal(out, v)


@pytest.mark.parametrize("T,d", [(5, 64), (1500, 64), (5, 33)])
def test_keys_or_values_alone(ctx, T, d):
    """Without queries, from Python and with any query stride in the C call; values alone; None with something asked of it."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(T, 8, 2, d, True)
    rot = d // 2 * 2
    pos, freq = torch.arange(T, dtype=torch.int32, device="cuda"), torch.from_numpy(freqs(rot)).cuda()
    attn = zb.CudaAttention(ctx)
    full = [torch.empty((T, n, d), dtype=q.dtype, device="cuda") for n in (8, 2, 2)]
    attn.qk_norm_rope(q, k, v, pos, freq, *full, q_weight=w[0], k_weight=w[1])
    out = [torch.empty_like(full[1]) for _ in range(3)]
    attn.qk_norm_rope(None, k, None, pos, freq, k_out=out[0], k_weight=w[1])
    attn.qk_norm_rope(None, None, v, None, None, v_out=out[1])
    assert c_call(ctx, k=k, q_stride=1, k_stride=k.stride(0), k_weight=w[1], eps=1e-6, positions=pos, inv_freq=freq, rotary_dim=rot,
                  k_out=out[2], num_tokens=T, num_heads=8, num_kv_heads=2, head_dim=d, dtype=1,
                  stream=torch.cuda.current_stream().cuda_stream) == 0
    ctx.check_status()
    # another query stride may take another kernel: within both of their tolerances
    near(out[0], formula(k.float().cpu().numpy(), w[1].float().cpu().numpy(), 1e-6, pos.cpu().numpy(), freqs(rot), False), True, d)
    near(out[2], formula(k.float().cpu().numpy(), w[1].float().cpu().numpy(), 1e-6, pos.cpu().numpy(), freqs(rot), False), True, d)
    assert torch.equal(out[1], v)
    for args, asked in (((None, k, v), "q_out"), ((q, None, v), "k_out"), ((q, k, None), "v_out")):
        with pytest.raises(zb.InvalidArgument):
            attn.qk_norm_rope(*args, pos, freq, **{asked: full["qkv".index(asked[0])]})
    with pytest.raises(zb.InvalidArgument):
        attn.qk_norm_rope(None, None, None, pos, freq, q_out=full[0])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,d", [(3, 64), (2000, 128), (2000, 72), (3, 33), (1500, 20)])
def test_values_keep_their_bits(ctx, T, d, bf16):
    """Every kind of number in the values, NaNs of any sign and payload among them: the same bits in the packed rows and
    in the pools, as reshape_and_cache leaves them."""
    import torch
    import zealot_b200 as zb
    g = torch.Generator(device="cuda").manual_seed(d)
    bits, kind = (torch.int16, torch.bfloat16) if bf16 else (torch.int32, torch.float32)
    size = torch.iinfo(bits)
    v = torch.randint(size.min, size.max + 1, (T, 3, d), generator=g, device="cuda", dtype=torch.int64).to(bits)
    v.view(-1)[:6] = torch.tensor([-1, size.min, size.max, 0, 0x7F81 << (0 if bf16 else 16), -2], dtype=torch.int64).to(bits).cuda()
    v = v.view(kind)
    assert torch.isnan(v).any()
    k = torch.randn((T, 3, d), generator=g, device="cuda").to(kind)
    nb = T // 16 + 2
    slots = torch.randperm(nb * 16, generator=g, device="cuda")[:T]
    pools = [torch.zeros((nb, 3, 16, d), dtype=kind, device="cuda") for _ in range(4)]
    out = torch.empty_like(v)
    pos, freq = torch.arange(T, dtype=torch.int32, device="cuda"), torch.from_numpy(freqs(d // 4 * 2)).cuda()
    attn = zb.CudaAttention(ctx)
    attn.qk_norm_rope(k, k, v, pos, freq, v_out=out, k_weight=k[0, 0].contiguous(), k_pool=pools[0], v_pool=pools[1], slot_mapping=slots)
    attn.reshape_and_cache(k, v, pools[2], pools[3], slots, 3, d, 16, nb)
    ctx.check_status()
    assert torch.equal(out.view(bits), v.view(bits)) and torch.equal(pools[1].view(bits), pools[3].view(bits))


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,d,rot,inter", [(1500, 128, 128, False), (9700, 64, 32, True), (2500, 80, 80, False), (1500, 33, 32, False)])
def test_in_place_many_tokens(ctx, T, d, rot, inter, bf16):
    """Rows that are copied ahead while others are stored over their inputs; NaN values among them."""
    import torch
    import zealot_b200 as zb
    _, q, k, v, w = make(T, 8, 2, d, bf16)
    q, k, v = q.contiguous(), k.contiguous(), v.clone()
    v[::7, 1, 3] = float("nan")
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 31
    freq = torch.from_numpy(freqs(rot)).cuda()
    out = [torch.empty_like(t) for t in (q, k, v)]
    attn = zb.CudaAttention(ctx)
    attn.qk_norm_rope(q, k, v, pos, freq, *out, q_weight=w[0], k_weight=w[1], interleaved=inter)
    attn.qk_norm_rope(q, k, v, pos, freq, q, k, v, q_weight=w[0], k_weight=w[1], interleaved=inter)
    ctx.check_status()
    bits = torch.int16 if bf16 else torch.int32
    for a, b in zip(out, (q, k, v)):
        assert torch.equal(a.view(bits), b.view(bits))
