"""Refusals of the serving-step operators, without a GPU: the C entry points check
their arguments before they touch a device, the Python methods before they call."""
import ctypes

import numpy as np
import pytest

INVALID, UNSUPPORTED = 1, 6
P = 4096  # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    from zealot_b200 import _capi
    return _capi.load()


def _refused(lib, name, base, code, text, **change):
    args = dict(base, **change)
    assert getattr(lib, name)(*args.values()) == code
    assert text in lib.zl_last_error().decode(), lib.zl_last_error()


TABLES = dict(ctx=None, seq_blocks=8 * P, num_rows=4, rows=P, context_lens=P, query_lens=P, new_blocks=P, num_new=1,
              block_tables=P, cu_seqlens=P, seq_lens=P, positions=P, slot_mapping=P, last_rows=P, num_seqs=2,
              num_tokens=3, max_blocks=8, block_size=16, num_blocks=64, stream=None)


@pytest.mark.parametrize("code,text,change", [
    (INVALID, "null context", {}),
    (INVALID, "bad sizes", dict(num_seqs=-1)), (INVALID, "bad sizes", dict(num_rows=-1)),
    (INVALID, "bad sizes", dict(num_new=-1)), (INVALID, "bad sizes", dict(num_tokens=-1)),
    (INVALID, "bad sizes", dict(max_blocks=-1)), (INVALID, "bad sizes", dict(block_size=0)),
    (INVALID, "bad sizes", dict(num_blocks=-1)), (INVALID, "2^31-1", dict(num_tokens=2**31)), (INVALID, "2^31-1", dict(num_tokens=2**31 - 1)),
    (INVALID, "2^31-1", dict(max_blocks=2**30 + 1)), (INVALID, "overlaps", dict(seq_blocks=P)),
    (INVALID, "overlaps", dict(seq_blocks=P + 2 * 8 * 4 - 4)), (INVALID, "overlaps", dict(seq_blocks=P - 4 * 8 * 4 + 4)),
    (INVALID, "2^31-1", dict(num_blocks=2**31)),
    (UNSUPPORTED, "at most", dict(num_seqs=8193, num_rows=9000)), (UNSUPPORTED, "at most", dict(num_rows=2**18 + 1)),
    (INVALID, "without `rows`", dict(rows=None, num_rows=1)),
    *[(INVALID, "null pointer", {k: None}) for k in ("seq_blocks", "context_lens", "query_lens", "new_blocks",
                                                     "block_tables", "cu_seqlens", "seq_lens", "positions",
                                                     "slot_mapping", "last_rows")]])
def test_step_tables_refusals(lib, code, text, change):
    _refused(lib, "zl_step_tables", TABLES, code, text, **change)


ROPE = dict(ctx=None, q=P, k=2 * P, v=3 * P, q_stride=512, k_stride=128, v_stride=128, q_weight=None, k_weight=None,
            eps=1e-6, positions=P, inv_freq=P, rotary_dim=64, interleaved=0, q_out=4 * P, k_out=5 * P, v_out=None,
            k_pool=None, v_pool=None, slots=None, block_size=0, num_blocks=0, num_tokens=3, H=8, Hkv=2, d=64, dtype=1,
            stream=None)


@pytest.mark.parametrize("code,text,change", [
    (INVALID, "null context", {}),
    (INVALID, "dtype", dict(dtype=7)), (INVALID, "bad sizes", dict(num_tokens=-1)), (INVALID, "bad sizes", dict(H=0)),
    (INVALID, "bad sizes", dict(Hkv=0)), (INVALID, "bad sizes", dict(d=0)),
    (UNSUPPORTED, "head_dim", dict(d=257, q_stride=8 * 257, k_stride=2 * 257)),
    (INVALID, "rotary_dim", dict(rotary_dim=63)), (INVALID, "rotary_dim", dict(rotary_dim=66)),
    (INVALID, "rotary_dim", dict(rotary_dim=-2)),
    (INVALID, "both pools", dict(k_pool=P)), (INVALID, "both pools", dict(v_pool=P)),
    (INVALID, "both pools", dict(k_pool=P, v_pool=P, block_size=16)),
    (INVALID, "both pools", dict(k_pool=P, v_pool=P, slots=P, block_size=0)),
    (INVALID, "both pools", dict(k_pool=P, v_pool=P, slots=P, block_size=16, num_blocks=-1)),
    (INVALID, "null pointer", dict(q=None)), (INVALID, "null pointer", dict(k=None)),
    (INVALID, "null pointer", dict(v=None, v_out=P)), (INVALID, "null pointer", dict(positions=None)),
    (INVALID, "null pointer", dict(inv_freq=None)), (INVALID, "null pointer", dict(q_out=None, k_out=None)),
    (INVALID, "stride", dict(q_stride=511)), (INVALID, "stride", dict(k_stride=127)),
    (INVALID, "stride", dict(v_out=P, v_stride=64)),
    (INVALID, "in place", dict(q_out=P, q_stride=768)), (INVALID, "in place", dict(k_out=2 * P, k_stride=768))])
def test_qk_norm_rope_refusals(lib, code, text, change):
    _refused(lib, "zl_qk_norm_rope", ROPE, code, text, **change)


BOUNDS = dict(ctx=None, k_pool=P, tables=P, tok_begin=None, seq_lens=P, bounds=P, B=2, Hkv=2, d=64, bs=16,
              max_blocks=8, num_blocks=64, dtype=1, stream=None)
SCORES = dict(ctx=None, q=P, bounds=P, tables=P, seq_lens=P, scores=P, B=2, H=8, Hkv=2, d=64, bs=16, max_blocks=8,
              num_blocks=64, scale=0.0, gqa_map=0, dtype=1, stream=None)


@pytest.mark.parametrize("name,base", [("zl_block_bounds", BOUNDS), ("zl_block_scores", SCORES)])
@pytest.mark.parametrize("text,change", [
    ("null context", {}), ("dtype", dict(dtype=2)), ("head shape", dict(Hkv=0)), ("head shape", dict(d=0)),
    ("bad sizes", dict(B=-1)), ("bad sizes", dict(bs=0)), ("bad sizes", dict(max_blocks=-1)),
    ("bad sizes", dict(max_blocks=2**30 + 1)),
    ("bad sizes", dict(num_blocks=-1)), ("null pointer", dict(tables=None)), ("null pointer", dict(seq_lens=None)),
    ("null pointer", dict(bounds=None))])
def test_block_bounds_and_scores_refusals(lib, name, base, text, change):
    _refused(lib, name, base, INVALID, text, **change)


def test_block_scores_refusals(lib):
    _refused(lib, "zl_block_scores", SCORES, INVALID, "head shape", H=7)
    for k in ("q", "scores"):
        _refused(lib, "zl_block_scores", SCORES, INVALID, "null pointer", **{k: None})
    _refused(lib, "zl_block_bounds", BOUNDS, INVALID, "null pointer", k_pool=None)


SELECT = dict(ctx=None, scores=P, seq_lens=P, selected=P, B=2, Hkv=2, bs=16, max_blocks=8, max_selected=4, num_first=1,
              num_last=1, stream=None)


@pytest.mark.parametrize("text,change", [
    ("null context", {}), ("bad sizes", dict(B=-1)), ("bad sizes", dict(Hkv=0)), ("bad sizes", dict(bs=0)),
    ("bad sizes", dict(max_blocks=-1)), ("bad sizes", dict(max_selected=-1)), ("first", dict(num_first=-1)),
    ("bad sizes", dict(max_blocks=2**30 + 1)), ("bad sizes", dict(max_selected=2**30 + 1)),
    ("first", dict(num_last=-1)), ("first", dict(num_first=3, num_last=2)), ("too large", dict(B=2**30, Hkv=2)),
    ("null pointer", dict(scores=None)), ("null pointer", dict(seq_lens=None)), ("null pointer", dict(selected=None))])
def test_select_blocks_refusals(lib, text, change):
    _refused(lib, "zl_select_blocks", SELECT, INVALID, text, **change)


SELECTED = dict(ctx=None, q=P, k_pool=P, v_pool=P, tables=P, seq_lens=P, selected=P, out=P, B=2, H=8, Hkv=2, d=64,
                bs=16, max_blocks=8, num_blocks=64, max_selected=4, scale=0.0, gqa_map=0, dtype=1, stream=None)


@pytest.mark.parametrize("code,text,change", [
    (INVALID, "null context", {}), (INVALID, "dtype", dict(dtype=-1)), (INVALID, "multiple", dict(H=7)),
    (INVALID, "head shape", dict(d=0)), (UNSUPPORTED, "head_dim", dict(d=512)), (INVALID, "bad sizes", dict(B=-1)),
    (INVALID, "bad sizes", dict(bs=0)), (INVALID, "bad sizes", dict(max_blocks=-1)),
    (INVALID, "bad sizes", dict(num_blocks=-1)), (INVALID, "bad sizes", dict(max_selected=-1)),
    (INVALID, "bad sizes", dict(max_selected=2**30 + 1)),
    (INVALID, "too large", dict(B=2**28, H=8)),
    *[(INVALID, "null pointer", {k: None}) for k in ("q", "k_pool", "v_pool", "tables", "seq_lens", "selected", "out")]])
def test_paged_decode_selected_refusals(lib, code, text, change):
    _refused(lib, "zl_paged_decode_selected", SELECTED, code, text, **change)


@pytest.mark.parametrize("name,base,change", [
    ("zl_qk_norm_rope", ROPE, dict(num_tokens=0, q=None, k=None)), ("zl_block_bounds", BOUNDS, dict(B=0)),
    ("zl_block_scores", SCORES, dict(B=0)), ("zl_block_scores", SCORES, dict(max_blocks=0)),
    ("zl_select_blocks", SELECT, dict(B=0)), ("zl_select_blocks", SELECT, dict(max_selected=0, num_first=0, num_last=0)),
    ("zl_paged_decode_selected", SELECTED, dict(B=0))])
def test_nothing_to_do_needs_no_device(lib, name, base, change):
    assert getattr(lib, name)(*dict(base, **change).values()) == 0


class _Context:
    """Stands in for a GpuContext: the Python checks come before any call on it."""
    device = 0
    lib = None
    address = 0


@pytest.fixture()
def attn():
    import zealot_b200 as zb
    return zb.CudaAttention(_Context())


def test_python_checks_refuse_other_devices(attn):
    """Tensors on the CPU (any device but the context's) never reach the library."""
    import torch
    import zealot_b200 as zb
    i = torch.zeros(4, dtype=torch.int32)
    i2 = torch.zeros((4, 4), dtype=torch.int32)
    f = torch.zeros((4, 4, 8))
    pool = torch.zeros((4, 4, 16, 8))
    with pytest.raises(zb.InvalidArgument, match="cuda:0"):
        attn.step_tables(i2, None, i, i, i, i2, torch.zeros(5, dtype=torch.int32), i, i, i.long(), i, 16, 4)
    with pytest.raises(zb.InvalidArgument, match="device"):
        attn.qk_norm_rope(f, f, f, i, torch.zeros(4, dtype=torch.float64), f)
    with pytest.raises(zb.InvalidArgument, match="cuda:0"):
        attn.block_bounds(pool, i2, i, pool[:, :, :2].contiguous())
    with pytest.raises(zb.InvalidArgument, match="cuda:0"):
        attn.block_scores(f, pool[:, :, :2].contiguous(), i2, i, f, 16)
    with pytest.raises(zb.InvalidArgument, match="cuda:0"):
        attn.select_blocks(f, i, i2[None], 16)
    with pytest.raises(zb.InvalidArgument, match="cuda:0"):
        attn.paged_forward_selected(f, pool, pool, i2, i, i2[None], f)


def test_qk_norm_rope_takes_keys_alone(lib):
    """No queries: their stride says nothing. (With a context the call would launch: "null context" is its last check.)"""
    for change in (dict(q_stride=0), dict(q_stride=1), dict(q_stride=768), dict(q_stride=512)):
        _refused(lib, "zl_qk_norm_rope", ROPE, INVALID, "null context", q=None, q_out=None, **change)
    _refused(lib, "zl_qk_norm_rope", ROPE, INVALID, "null context", q=None, q_out=None, k=None, k_out=None, v_out=P,
             positions=None, q_stride=0, k_stride=0)
