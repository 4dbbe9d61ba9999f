"""CudaAttention: the attention operators of the hot path.

Mirrors src/attention/cuda.rs:20-210 of the reference (paged_forward,
forward_gpu) plus the KV scatter that replaced KVCache::store_kv's copies.
Arguments keep the reference's names and meaning; tensors are torch device
tensors, checked here and handed to the C ABI by address.
"""
from __future__ import annotations

from .context import GpuContext, GQA_GROUPED, dtype_code, ptr
from .errors import check, InvalidArgument


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise InvalidArgument(msg)


class CudaAttention:
    def __init__(self, ctx: GpuContext):
        self.ctx = ctx
        self.lib = ctx.lib

    def _check(self, dtype, *tensors) -> None:
        """Each tensor is a contiguous one of `dtype` on the context's device."""
        device = self.ctx.device
        for t in tensors:
            if t.dtype != dtype or t.get_device() != device or not t.is_contiguous():
                raise InvalidArgument(f"need a contiguous {dtype} tensor on cuda:{device}, got {t.dtype} on "
                                      f"{t.device}, strides {tuple(t.stride())}")

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
        n, T = query_lens.numel(), slot_mapping.numel()
        self._check(torch.int32, seq_blocks, context_lens, query_lens, new_blocks, block_tables, cu_seqlens,
                    seq_lens, positions, last_rows)
        self._check(torch.int64, slot_mapping)
        _need(seq_blocks.dim() == 2, "seq_blocks is [num_rows][max_blocks]")
        num_rows, max_blocks = seq_blocks.shape
        if rows is not None:
            self._check(torch.int32, rows)
            _need(rows.numel() == n, "one table row per request")
        _need(context_lens.numel() == n and seq_lens.numel() == n and last_rows.numel() == n
              and cu_seqlens.numel() == n + 1 and block_tables.numel() == n * max_blocks
              and positions.numel() == T, "step_tables shapes")
        check(self.lib.zl_step_tables(
            self.ctx.handle, seq_blocks.data_ptr(), num_rows, ptr(rows), context_lens.data_ptr(),
            query_lens.data_ptr(), new_blocks.data_ptr(), new_blocks.numel(), block_tables.data_ptr(),
            cu_seqlens.data_ptr(), seq_lens.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
            last_rows.data_ptr(), n, T, max_blocks, block_size, num_blocks, self.ctx.stream(stream)))

    # ------------------------------------- query / key norm, rotation, scatter
    def qk_norm_rope(self, q, k, v, positions, inv_freq, q_out=None, k_out=None, v_out=None, q_weight=None,
                     k_weight=None, eps: float = 1e-6, interleaved: bool = False, k_pool=None, v_pool=None,
                     slot_mapping=None, stream=None) -> None:
        """RMS norm of each head of q [T][H][d] and k [T][Hkv][d] (a weight [d] or None), rotation of the
        first 2 * inv_freq.numel() elements of each head by positions[t] * inv_freq (float64), and the
        stores: q_out, k_out, v_out packed, and the pools [num_blocks][Hkv][bs][d] at slot_mapping.
        q, k and v may be views of one projection's rows (any stride from token to token)."""
        import torch
        T, Hkv, d = k.shape
        device, dtype = self.ctx.device, q.dtype
        _need(q.dim() == 3 and q.shape[0] == T and q.shape[2] == d and v.shape == k.shape, "q/k/v shapes")
        H = q.shape[1]
        for t, heads in ((q, H), (k, Hkv), (v, Hkv)):
            _need(t.dtype == dtype and t.get_device() == device, "q, k and v: one dtype, on the context's device")
            _need(t.stride(2) == 1 and (t.stride(1) == d or heads == 1), "the heads of a token are packed")
        for t, heads in ((q_out, H), (k_out, Hkv), (v_out, Hkv)):
            if t is not None:
                self._check(dtype, t)
                _need(t.shape == (T, heads, d), "output shape")
        for w in (q_weight, k_weight):
            if w is not None:
                self._check(dtype, w)
                _need(w.numel() == d, "a norm weight has head_dim elements")
        rot = 0
        if inv_freq is not None:
            self._check(torch.float64, inv_freq)
            self._check(torch.int32, positions)
            _need(positions.numel() == T, "one position per token")
            rot = 2 * inv_freq.numel()
        bs = num_blocks = 0
        if k_pool is not None or v_pool is not None:
            _need(k_pool is not None and v_pool is not None and slot_mapping is not None,
                  "both pools and a slot_mapping, or none")
            self._check(dtype, k_pool, v_pool)
            self._check(torch.int64, slot_mapping)
            _need(k_pool.dim() == 4 and k_pool.shape == v_pool.shape and k_pool.shape[1] == Hkv
                  and k_pool.shape[3] == d and slot_mapping.numel() == T, "pools [num_blocks][Hkv][bs][d], slots [T]")
            num_blocks, bs = k_pool.shape[0], k_pool.shape[2]
        check(self.lib.zl_qk_norm_rope(
            self.ctx.handle, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0),
            ptr(q_weight), ptr(k_weight), eps, ptr(positions), ptr(inv_freq), rot, int(interleaved), ptr(q_out),
            ptr(k_out), ptr(v_out), ptr(k_pool), ptr(v_pool), ptr(slot_mapping), bs, num_blocks, T, H, Hkv, d,
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
    def _paged(self, block_tables, seq_lens):
        """(B, max_blocks) of a table [B][max_blocks] and its lengths [B], both int32."""
        import torch
        self._check(torch.int32, block_tables, seq_lens)
        _need(block_tables.dim() == 2 and seq_lens.numel() == block_tables.shape[0],
              "block_tables [B][max_blocks], seq_lens [B]")
        return block_tables.shape

    def block_bounds(self, k_pool, block_tables, seq_lens, bounds, tok_begin=None, stream=None) -> None:
        """Elementwise minimum and maximum of the keys of each block that holds a token in
        [tok_begin[b], seq_lens[b]): k_pool [num_blocks][Hkv][bs][d] -> bounds [num_blocks][Hkv][2][d]."""
        import torch
        B, max_blocks = self._paged(block_tables, seq_lens)
        self._check(k_pool.dtype, k_pool, bounds)
        if tok_begin is not None:
            self._check(torch.int32, tok_begin)
            _need(tok_begin.numel() == B, "one tok_begin per sequence")
        _need(k_pool.dim() == 4, "k_pool is [num_blocks][Hkv][bs][d]")
        num_blocks, Hkv, bs, d = k_pool.shape
        _need(bounds.shape == (num_blocks, Hkv, 2, d), "bounds is [num_blocks][Hkv][2][d]")
        check(self.lib.zl_block_bounds(
            self.ctx.handle, k_pool.data_ptr(), block_tables.data_ptr(), ptr(tok_begin), seq_lens.data_ptr(),
            bounds.data_ptr(), B, Hkv, d, bs, max_blocks, num_blocks, dtype_code(k_pool.dtype),
            self.ctx.stream(stream)))

    def block_scores(self, q, bounds, block_tables, seq_lens, scores, block_size: int, scale: float = 0.0,
                     gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """Upper bound of every block's attention scores for q [B][H][d] (the largest over a kv head's
        query heads): scores [B][Hkv][max_blocks] float32, -inf where a sequence has no block."""
        import torch
        B, max_blocks = self._paged(block_tables, seq_lens)
        self._check(q.dtype, q, bounds)
        self._check(torch.float32, scores)
        _need(q.dim() == 3 and q.shape[0] == B and bounds.dim() == 4, "q [B][H][d], bounds [num_blocks][Hkv][2][d]")
        num_blocks, Hkv, two, d = bounds.shape
        _need(two == 2 and q.shape[2] == d and scores.shape == (B, Hkv, max_blocks), "block_scores shapes")
        check(self.lib.zl_block_scores(
            self.ctx.handle, q.data_ptr(), bounds.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
            scores.data_ptr(), B, q.shape[1], Hkv, d, block_size, max_blocks, num_blocks, scale, gqa_map,
            dtype_code(q.dtype), self.ctx.stream(stream)))

    def select_blocks(self, scores, seq_lens, selected, block_size: int, num_first: int = 1, num_last: int = 1,
                      stream=None) -> None:
        """Of each sequence's blocks the first num_first, the last num_last and the best others by
        scores [B][Hkv][max_blocks]: selected [B][Hkv][max_selected] int32, ascending, -1 after the last."""
        import torch
        self._check(torch.float32, scores)
        self._check(torch.int32, seq_lens, selected)
        _need(scores.dim() == 3 and selected.dim() == 3 and selected.shape[:2] == scores.shape[:2]
              and seq_lens.numel() == scores.shape[0], "select_blocks shapes")
        B, Hkv, max_blocks = scores.shape
        check(self.lib.zl_select_blocks(
            self.ctx.handle, scores.data_ptr(), seq_lens.data_ptr(), selected.data_ptr(), B, Hkv, block_size,
            max_blocks, selected.shape[2], num_first, num_last, self.ctx.stream(stream)))

    def paged_forward_selected(self, q, k_pool, v_pool, block_tables, seq_lens, selected, o, scale: float = 0.0,
                               gqa_map: int = GQA_GROUPED, stream=None) -> None:
        """paged_forward over the blocks that selected [B][Hkv][max_selected] lists (indices into a
        sequence's table row; a negative one ends the list): q/o [B][H][d]."""
        import torch
        B, max_blocks = self._paged(block_tables, seq_lens)
        self._check(q.dtype, q, k_pool, v_pool, o)
        self._check(torch.int32, selected)
        _need(k_pool.dim() == 4 and k_pool.shape == v_pool.shape, "pools are [num_blocks][Hkv][bs][d]")
        num_blocks, Hkv, bs, d = k_pool.shape
        _need(q.dim() == 3 and q.shape[0] == B and q.shape[2] == d and o.shape == q.shape, "q/o shape")
        _need(selected.dim() == 3 and selected.shape[:2] == (B, Hkv), "selected is [B][Hkv][max_selected]")
        check(self.lib.zl_paged_decode_selected(
            self.ctx.handle, q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(),
            seq_lens.data_ptr(), selected.data_ptr(), o.data_ptr(), B, q.shape[1], Hkv, d, bs, max_blocks,
            num_blocks, selected.shape[2], scale, gqa_map, dtype_code(q.dtype), self.ctx.stream(stream)))

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
