"""CudaAttention: the attention operators of the hot path.

Mirrors src/attention/cuda.rs:20-210 of the reference (paged_forward,
forward_gpu) plus the KV scatter that replaced KVCache::store_kv's copies, and,
without a counterpart there, a step's metadata from lengths (step_tables), the
norm and rotation of queries and keys with the cache write (qk_norm_rope) and
decode over selected blocks (block_bounds, block_scores, select_blocks,
paged_forward_selected).
Arguments keep the reference's names and meaning; tensors are torch device
tensors, checked here and handed to the C ABI by address.
"""
from __future__ import annotations

from .context import GpuContext, GQA_GROUPED, dtype_code, ptr
from .errors import check, InvalidArgument

try:
    from . import calls  # native, built by build.py beside the library
except ImportError as _error:  # not built for this Python: the operators that go through it say so, the others work
    class _NoCalls:
        def __init__(self, why: str):
            self._why = why

        def __getattr__(self, name):
            raise ImportError(f"this call needs zealot_b200's call path for this Python ({self._why}): build it with "
                              "`python zealot_b200/build.py`")

    calls = _NoCalls(str(_error))


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise InvalidArgument(msg)


class CudaAttention:
    def __init__(self, ctx: GpuContext):
        self.ctx = ctx
        self.lib = ctx.lib

    def _addresses(self, *triples):
        """(tensor or None, dtype, elements or shape), flat: the addresses of tensors that are contiguous, of
        that dtype and size and on the context's device. Small calls are bound by such checks, so one native
        pass does them (calls.c)."""
        got = calls.addresses(self.ctx.device, *triples)
        if type(got) is not tuple:
            t, dtype, n = triples[3 * got:3 * got + 3]
            what = f"{n} elements" if isinstance(n, int) else f"shape {n}"
            raise InvalidArgument(f"need a contiguous {dtype} tensor of {what} on cuda:{self.ctx.device}, got "
                                  f"{t.dtype} {tuple(t.shape)} on {t.device}, strides {t.stride()}")
        return got

    # ----------------------------------------------------------- step tables
    def step_tables(self, seq_blocks, rows, context_lens, query_lens, new_blocks, block_tables, cu_seqlens,
                    seq_lens, positions, slot_mapping, last_rows, block_size: int, num_blocks: int,
                    stream=None) -> None:
        """One step's metadata from the requests' lengths. Request i adds query_lens[i] tokens to
        context_lens[i] cached ones; its blocks are row rows[i] (None: row i) of the persistent
        seq_blocks [num_rows][max_blocks], which gets the new ones from new_blocks, in request order.
        Writes block_tables [n][max_blocks], cu_seqlens [n+1], seq_lens [n], last_rows [n], and for each
        token row positions [T] and slot_mapping [T] (int64; all others int32)."""
        import torch
        i32, n, T, new = torch.int32, query_lens.numel(), slot_mapping.numel(), new_blocks.numel()
        _need(seq_blocks.dim() == 2, "seq_blocks is [num_rows][max_blocks]")
        num_rows, width = seq_blocks.shape
        old, row, c, q, fresh, tables, cu, lens, pos, slots, last = self._addresses(
            seq_blocks, i32, num_rows * width, rows, i32, n, context_lens, i32, n, query_lens, i32, n, new_blocks, i32, new,
            block_tables, i32, n * width, cu_seqlens, i32, n + 1, seq_lens, i32, n, positions, i32, T,
            slot_mapping, torch.int64, T, last_rows, i32, n)
        check(calls.step_tables(self.ctx.address, old, num_rows, row, c, q, fresh, new, tables, cu, lens, pos,
                                slots, last, n, T, width, block_size, num_blocks, self.ctx.stream(stream)))

    # ------------------------------------- query / key norm, rotation, scatter
    def qk_norm_rope(self, q, k, v, positions, inv_freq, q_out=None, k_out=None, v_out=None, q_weight=None,
                     k_weight=None, eps: float = 1e-6, interleaved: bool = False, k_pool=None, v_pool=None,
                     slot_mapping=None, stream=None) -> None:
        """RMS norm of each head of q [T][H][d] and k [T][Hkv][d] (a weight [d] or None), rotation of the
        first 2 * inv_freq.numel() elements of each head by positions[t] * inv_freq (float64; None: no
        rotation), and the stores: q_out, k_out, v_out packed, and the pools [num_blocks][Hkv][bs][d] at
        slot_mapping. q, k and v may be views of one projection's rows (any stride from token to token), and
        None where nothing of them is asked for."""
        import torch
        x = q if q is not None else k if k is not None else v
        _need(x is not None, "one of q, k and v")
        dtype = x.dtype
        T, heads, d = x.shape
        Hkv = k.shape[1] if k is not None else v.shape[1] if v is not None else heads
        H = heads if q is not None else Hkv
        rows = calls.head_rows(self.ctx.device, dtype, T, d, q, H, k, Hkv, v, Hkv)
        if type(rows) is not tuple:
            raise InvalidArgument("q [T][H][d], k and v [T][Hkv][d]: one dtype, on the context's device, the heads of a "
                                  f"token packed; {'qkv'[rows]} is not")
        qa, qs, ka, ks, va, vs = rows
        rot = bs = num_blocks = pool = 0
        if inv_freq is not None:
            _need(positions is not None, "inv_freq needs positions")
            rot = 2 * inv_freq.numel()
        if k_pool is not None or v_pool is not None:
            _need(k_pool is not None and v_pool is not None and slot_mapping is not None,
                  "both pools and a slot_mapping, or none")
            num_blocks, pool_heads, bs, pool_d = k_pool.shape
            _need(pool_heads == Hkv and pool_d == d, "pools are [num_blocks][Hkv][bs][d]")
            pool = (num_blocks, Hkv, bs, d)
        nk = T * Hkv * d
        qo, ko, vo, qw, kw, pos, freq, kp, vp, slots = self._addresses(
            q_out, dtype, T * H * d, k_out, dtype, nk, v_out, dtype, nk, q_weight, dtype, d, k_weight, dtype, d,
            positions, torch.int32, T, inv_freq, torch.float64, rot // 2, k_pool, dtype, pool, v_pool, dtype, pool,
            slot_mapping, torch.int64, T)
        check(calls.qk_norm_rope(self.ctx.address, qa, ka, va, qs, ks, vs, qw, kw, eps, pos, freq, rot,
                                 int(interleaved), qo, ko, vo, kp, vp, slots, bs, num_blocks, T, H, Hkv, d,
                                 dtype_code(dtype), self.ctx.stream(stream)))

    # ------------------------------------------------------------ KV scatter
    def reshape_and_cache(self, k, v, k_pool, v_pool, slot_mapping, num_kv_heads: int,
                          head_dim: int, block_size: int, num_blocks: int, stream=None) -> None:
        """k, v [T][Hkv][d] -> pools [num_blocks][Hkv][bs][d] at slot_mapping[T] (int64)."""
        import torch
        _need(k.dtype == v.dtype == k_pool.dtype == v_pool.dtype, "dtype mismatch")
        _need(slot_mapping.dtype == torch.int64, "slot_mapping must be int64")
        for t in (k, v, k_pool, v_pool, slot_mapping):
            _need(t.is_contiguous() and t.is_cuda, "tensors must be contiguous CUDA tensors")
        T = slot_mapping.numel()
        _need(k.numel() == T * num_kv_heads * head_dim and v.numel() == k.numel(), "k/v shape")
        _need(k_pool.numel() >= num_blocks * block_size * num_kv_heads * head_dim, "pool too small")
        check(self.lib.zl_reshape_and_cache(self.ctx.handle, ptr(k), ptr(v), ptr(k_pool), ptr(v_pool),
                                            ptr(slot_mapping), T, num_kv_heads, head_dim, block_size,
                                            num_blocks, dtype_code(k.dtype), self.ctx.stream(stream)))

    # ----------------------------------------------------------- paged decode
    def paged_forward(self, q, k_pool, v_pool, block_tables, seq_lens, o, num_seqs: int,
                      num_heads: int, num_kv_heads: int, head_dim: int, block_size: int,
                      max_blocks_per_seq: int, num_blocks: int | None = None, scale: float = 0.0,
                      gqa_map: int = GQA_GROUPED, num_splits: int = 0, stream=None) -> None:
        """CudaAttention::paged_forward (cuda.rs:126-210): q/o [B][H][d], block_tables
        [B][max_blocks] int32 (negative = end), seq_lens [B] int32."""
        import torch
        _need(q.dtype == k_pool.dtype == v_pool.dtype == o.dtype, "dtype mismatch")
        _need(block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32, "int32 tables")
        for t in (q, k_pool, v_pool, block_tables, seq_lens, o):
            _need(t.is_contiguous() and t.is_cuda, "tensors must be contiguous CUDA tensors")
        _need(q.numel() == num_seqs * num_heads * head_dim and o.numel() == q.numel(), "q/o shape")
        _need(block_tables.numel() >= num_seqs * max_blocks_per_seq, "block_tables shape")
        per_block = block_size * num_kv_heads * head_dim
        if num_blocks is None:
            num_blocks = k_pool.numel() // per_block
        _need(k_pool.numel() >= num_blocks * per_block, "pool smaller than num_blocks")
        check(self.lib.zl_paged_decode(self.ctx.handle, ptr(q), ptr(k_pool), ptr(v_pool),
                                       ptr(block_tables), ptr(seq_lens), ptr(o), num_seqs, num_heads,
                                       num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                                       num_blocks, scale, gqa_map, num_splits, dtype_code(q.dtype),
                                       self.ctx.stream(stream)))

    def paged_forward_partial(self, q, k_pool, v_pool, block_tables, tok_begin, tok_end, m, l, o,
                              num_seqs: int, num_heads: int, num_kv_heads: int, head_dim: int,
                              block_size: int, max_blocks_per_seq: int, num_blocks: int | None = None,
                              scale: float = 0.0, gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """Unnormalised (m, l, o) over tokens [tok_begin, tok_end) of each sequence."""
        import torch
        _need(m.dtype == l.dtype == o.dtype == torch.float32, "partials are float32")
        per_block = block_size * num_kv_heads * head_dim
        if num_blocks is None:
            num_blocks = k_pool.numel() // per_block
        check(self.lib.zl_paged_decode_partial(
            self.ctx.handle, ptr(q), ptr(k_pool), ptr(v_pool), ptr(block_tables), ptr(tok_begin),
            ptr(tok_end), ptr(m), ptr(l), ptr(o), num_seqs, num_heads, num_kv_heads, head_dim,
            block_size, max_blocks_per_seq, num_blocks, scale, gqa_map, dtype_code(q.dtype),
            self.ctx.stream(stream)))

    def merge_partials(self, m, l, o, out, stream=None) -> None:
        """m, l [P][rows], o [P][rows][d] float32 -> out [rows][d]."""
        P = m.shape[0]
        rows = m[0].numel()
        d = o.shape[-1]
        check(self.lib.zl_merge_partials(self.ctx.handle, ptr(m), ptr(l), ptr(o), P, rows, d,
                                         ptr(out), dtype_code(out.dtype), self.ctx.stream(stream)))

    # ------------------------------------------- decode over selected blocks
    def block_bounds(self, k_pool, block_tables, seq_lens, bounds, tok_begin=None, stream=None) -> None:
        """Elementwise minimum and maximum of the keys of each block from that of token tok_begin[b] (None: 0)
        to that of the last of seq_lens[b]: k_pool [num_blocks][Hkv][bs][d] -> bounds [num_blocks][Hkv][2][d].
        A sequence is listed once, with its largest length: rows that bound the same block must agree on how
        many of its tokens there are."""
        import torch
        _need(k_pool.dim() == 4 and block_tables.dim() == 2, "k_pool [num_blocks][Hkv][bs][d], block_tables [B][max]")
        num_blocks, Hkv, bs, d = k_pool.shape
        B, width = block_tables.shape
        i32, dtype, row = torch.int32, k_pool.dtype, num_blocks * Hkv * d
        k, table, begin, lens, out = self._addresses(
            k_pool, dtype, row * bs, block_tables, i32, B * width, tok_begin, i32, B, seq_lens, i32, B, bounds, dtype, row * 2)
        check(calls.block_bounds(self.ctx.address, k, table, begin, lens, out, B, Hkv, d, bs, width, num_blocks,
                                 dtype_code(dtype), self.ctx.stream(stream)))

    def block_scores(self, q, bounds, block_tables, seq_lens, scores, block_size: int, scale: float = 0.0,
                     gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """Upper bound of every block's attention scores for q [B][H][d] (the largest over a kv head's
        query heads): scores [B][Hkv][max_blocks] float32, -inf where a sequence has no block."""
        import torch
        _need(q.dim() == 3 and bounds.dim() == 4 and block_tables.dim() == 2,
              "q [B][H][d], bounds [num_blocks][Hkv][2][d], block_tables [B][max]")
        num_blocks, Hkv, two, d = bounds.shape
        B, width = block_tables.shape
        H, i32, dtype = q.shape[1], torch.int32, q.dtype
        _need(two == 2, "bounds is [num_blocks][Hkv][2][d]")
        x, ends, table, lens, out = self._addresses(
            q, dtype, (B, H, d), bounds, dtype, num_blocks * Hkv * 2 * d, block_tables, i32, B * width, seq_lens, i32, B,
            scores, torch.float32, B * Hkv * width)
        check(calls.block_scores(self.ctx.address, x, ends, table, lens, out, B, H, Hkv, d, block_size, width,
                                 num_blocks, scale, gqa_map, dtype_code(dtype), self.ctx.stream(stream)))

    def select_blocks(self, scores, seq_lens, selected, block_size: int, num_first: int = 1, num_last: int = 1,
                      stream=None) -> None:
        """Of each sequence's blocks the first num_first, the last num_last and the best others by
        scores [B][Hkv][max_blocks]: selected [B][Hkv][max_selected] int32, ascending, -1 after the last."""
        import torch
        _need(scores.dim() == 3 and selected.dim() == 3, "scores [B][Hkv][max_blocks], selected [B][Hkv][max_selected]")
        B, Hkv, width = scores.shape
        top = selected.shape[2]
        sc, lens, out = self._addresses(scores, torch.float32, B * Hkv * width, seq_lens, torch.int32, B,
                                        selected, torch.int32, (B, Hkv, top))
        check(calls.select_blocks(self.ctx.address, sc, lens, out, B, Hkv, block_size, width, top, num_first,
                                  num_last, self.ctx.stream(stream)))

    def paged_forward_selected(self, q, k_pool, v_pool, block_tables, seq_lens, selected, o, scale: float = 0.0,
                               gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """paged_forward over the blocks that selected [B][Hkv][max_selected] lists (indices into a
        sequence's table row; a negative one ends the list): q/o [B][H][d]."""
        import torch
        _need(q.dim() == 3 and k_pool.dim() == 4 and block_tables.dim() == 2 and selected.dim() == 3,
              "q [B][H][d], pools [num_blocks][Hkv][bs][d], block_tables [B][max], selected [B][Hkv][max_selected]")
        num_blocks, Hkv, bs, d = k_pool.shape
        B, width = block_tables.shape
        H, top, i32, dtype = q.shape[1], selected.shape[2], torch.int32, q.dtype
        pool = (num_blocks, Hkv, bs, d)
        x, k, v, table, lens, picked, out = self._addresses(
            q, dtype, (B, H, d), k_pool, dtype, pool, v_pool, dtype, pool, block_tables, i32, B * width, seq_lens, i32, B,
            selected, i32, (B, Hkv, top), o, dtype, B * H * d)
        check(calls.paged_decode_selected(self.ctx.address, x, k, v, table, lens, picked, out, B, H, Hkv, d, bs,
                                          width, num_blocks, top, scale, gqa_map, dtype_code(dtype),
                                          self.ctx.stream(stream)))

    # ---------------------------------------------------------------- prefill
    def forward_gpu(self, q, k, v, cu_seqlens, o, num_heads: int, num_kv_heads: int,
                    head_dim: int, max_seq_len: int, causal: bool = True, scale: float = 0.0,
                    gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """Varlen form of CudaAttention::forward_gpu (cuda.rs:56-110): q/o [T][H][d],
        k/v [T][Hkv][d], cu_seqlens [n+1] int32."""
        import torch
        _need(q.dtype == k.dtype == v.dtype == o.dtype, "dtype mismatch")
        _need(cu_seqlens.dtype == torch.int32, "cu_seqlens must be int32")
        for t in (q, k, v, cu_seqlens, o):
            _need(t.is_contiguous() and t.is_cuda, "tensors must be contiguous CUDA tensors")
        n = cu_seqlens.numel() - 1
        T = q.shape[0]
        _need(q.numel() == T * num_heads * head_dim and k.numel() == T * num_kv_heads * head_dim
              and v.numel() == k.numel() and o.numel() == q.numel(), "q/k/v/o shapes")
        check(self.lib.zl_prefill_varlen(self.ctx.handle, ptr(q), ptr(k), ptr(v), ptr(cu_seqlens), n,
                                         max_seq_len, T, ptr(o), num_heads, num_kv_heads, head_dim, scale,
                                         int(causal), gqa_map, dtype_code(q.dtype),
                                         self.ctx.stream(stream)))
