// block_select.cu -- which blocks of a long paged context a query attends to:
// bounds of each block's keys, an upper bound of each block's scores from them,
// and the choice of the best blocks.
//
// Bounds: lo_i = min and hi_i = max over a block's cached keys of element i.
// For every key k of the block and every query q,
//   q . k = sum_i q_i k_i <= sum_i max(q_i, 0) hi_i + min(q_i, 0) lo_i,
// so the score of a block, scale * the largest right side over the query heads
// of the kv head's group, is never below the largest attention score in it.
// A block's bounds are two rows where its keys are block_size: scoring reads
// 2 / block_size of the keys (1/16 of keys and values at 16).
//
// NaN goes through: a key that is NaN makes its bound, its block's score and,
// once that block is selected (NaN ranks above every score), the output NaN,
// as attention over all blocks would be.
#include "zl_internal.h"
#include "zl_pages.h"

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
// min and max that return NaN when an operand is NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct PagedArgs {
  const int32_t* tables;
  const int32_t* seq_lens;
  int B, H, Hkv, d, bs, max_blocks;
  int64_t num_blocks;
  int modulo;
  int* status;
};

// Length of sequence b, cut to its table (a longer one is reported).
__device__ __forceinline__ int64_t seq_len(const PagedArgs& g, int b) {
  int64_t len = max(g.seq_lens[b], 0);
  const int64_t most = (int64_t)g.max_blocks * g.bs;
  if (len > most) {
    atomicOr(g.status, ZL_DEV_OOB);
    len = most;
  }
  return len;
}

// Block j of sequence b: its id, or -1 (none, or outside the pool and reported).
__device__ __forceinline__ int64_t block_id(const PagedArgs& g, int b, int64_t j) {
  const int32_t id = g.tables[(int64_t)b * g.max_blocks + j];
  if (id >= g.num_blocks) {
    atomicOr(g.status, ZL_DEV_OOB);
    return -1;
  }
  return id < 0 ? -1 : id;
}

// ------------------------------------------------------------------- bounds

// One warp per (sequence, kv head) and every gridDim.x-th block, one element
// per lane and pass. Any head_dim and alignment.
template <typename T>
__global__ void __launch_bounds__(256)
bounds_elem_kernel(PagedArgs g, const T* __restrict__ k_pool, const int32_t* __restrict__ tok_begin,
                   T* __restrict__ bounds) {
  const int lane = threadIdx.x & 31;
  for (int64_t u = blockIdx.y; u < (int64_t)g.B * g.Hkv; u += gridDim.y) {
    const int b = (int)(u / g.Hkv), h = (int)(u - (int64_t)b * g.Hkv);
    const int64_t len = seq_len(g, b), n = zl::blocks_of(len, g.bs);
    const int64_t first = tok_begin ? max(tok_begin[b], 0) / g.bs : 0;
    for (int64_t j = first + blockIdx.x * 8 + (threadIdx.x >> 5); j < n; j += (int64_t)gridDim.x * 8) {
      const int64_t id = block_id(g, b, j);
      if (id < 0) continue;
      const T* rows = k_pool + zl::pool_row(id, g.num_blocks, g.Hkv, h, g.bs, 0) * g.d;
      const int toks = (int)min((int64_t)g.bs, len - j * g.bs);
      T* out = bounds + (id * g.Hkv + h) * 2 * g.d;
      for (int e = lane; e < g.d; e += 32) {
        float lo = to_f(rows[e]), hi = lo;
        for (int t = 1; t < toks; t++) {
          const float x = to_f(rows[(int64_t)t * g.d + e]);
          lo = min_nan(lo, x);
          hi = max_nan(hi, x);
        }
        put(out + e, lo);
        put(out + g.d + e, hi);
      }
    }
  }
}

// ------------------------------------------------------------------- scores

// One warp per (sequence, kv head, block), one element per lane and pass.
template <typename T>
__global__ void __launch_bounds__(256)
scores_elem_kernel(PagedArgs g, const T* __restrict__ q, const T* __restrict__ bounds, float scale,
                   float* __restrict__ scores) {
  const int lane = threadIdx.x & 31;
  const int group = g.H / g.Hkv;
  for (int64_t u = blockIdx.y; u < (int64_t)g.B * g.Hkv; u += gridDim.y) {
    const int b = (int)(u / g.Hkv), h = (int)(u - (int64_t)b * g.Hkv);
    const int64_t n = zl::blocks_of(seq_len(g, b), g.bs);
    for (int64_t j = blockIdx.x * 8 + (threadIdx.x >> 5); j < g.max_blocks; j += (int64_t)gridDim.x * 8) {
      float best = -INFINITY;
      const int64_t id = j < n ? block_id(g, b, j) : -1;
      if (id >= 0) {
        const T* lo = bounds + (id * g.Hkv + h) * 2 * g.d;
        for (int i = 0; i < group; i++) {
          const int head = g.modulo ? i * g.Hkv + h : h * group + i;
          const T* x = q + ((int64_t)b * g.H + head) * g.d;
          float s = 0.f;
          for (int e = lane; e < g.d; e += 32) {
            const float f = to_f(x[e]);
            s = fmaf(max_nan(f, 0.f), to_f(lo[g.d + e]), fmaf(min_nan(f, 0.f), to_f(lo[e]), s));
          }
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          best = max_nan(best, s * scale);
        }
      }
      if (lane == 0) scores[u * g.max_blocks + j] = best;
    }
  }
}

// ---------------------------------------------------------------- selection

// The `top` blocks of one (sequence, kv head), ascending: the first `nf`, the
// last `nl` and the best of those between, equal scores by the lower index.
// With m = top - (nf + nl) still to choose from the middle, the threshold is
// the largest key that at least m middle keys reach; it is found bit by bit by
// counting, which needs no atomics and costs the same for every distribution
// of the scores.
constexpr int kSelThreads = 256;

__device__ __forceinline__ int block_count(int c, int* red) {  // sum over the CTA, to every thread
  c = __reduce_add_sync(0xffffffffu, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = c;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < kSelThreads / 32; w++) s += red[w];
  return s;
}

__global__ void __launch_bounds__(kSelThreads)
select_kernel(const float* __restrict__ scores, const int32_t* __restrict__ seq_lens, int Hkv, int max_blocks, int bs,
              int top, int num_first, int num_last, int32_t* __restrict__ selected, int* status) {
  __shared__ int red[kSelThreads / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const float* sc = scores + row * max_blocks;
  int32_t* out = selected + row * top;
  const int64_t want = zl::blocks_of(seq_lens[row / Hkv], bs);
  if (want > max_blocks && tid == 0) atomicOr(status, ZL_DEV_OOB);
  const int n = (int)min(want, (int64_t)max_blocks);
  if (n <= top) {
    for (int j = tid; j < top; j += kSelThreads) out[j] = j < n ? j : -1;
    return;
  }
  // n > top >= num_first + num_last: the three parts do not meet
  const int lo = num_first, hi = n - num_last, m = top - num_first - num_last;
  for (int j = tid; j < num_first; j += kSelThreads) out[j] = j;
  for (int j = tid; j < num_last; j += kSelThreads) out[top - num_last + j] = hi + j;
  if (m == 0) return;
  auto key = [&](int j) { return zl::score_key(__float_as_uint(sc[j])); };
  uint32_t limit = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t cand = limit | 1u << bit;
    int c = 0;
    for (int j = lo + tid; j < hi; j += kSelThreads) c += key(j) >= cand;
    if (block_count(c, red) >= m) limit = cand;
  }
  int above = 0;
  for (int j = lo + tid; j < hi; j += kSelThreads) above += key(j) > limit;
  int ties = m - block_count(above, red);  // of the keys equal to the limit, the first so many
  // write in index order: each pass handles one index per thread
  int at = num_first;
  for (int base = lo; base < hi; base += kSelThreads) {
    const int j = base + tid;
    const uint32_t kj = j < hi ? key(j) : 0;
    const int eq = j < hi && kj == limit;
    // equal keys before this one in the pass
    const unsigned eqs = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = __popc(eqs);
    __syncthreads();
    int before = __popc(eqs & ((1u << (tid & 31)) - 1)), all = 0;
    for (int w = 0; w < kSelThreads / 32; w++) {
      before += w < (tid >> 5) ? red[w] : 0;
      all += red[w];
    }
    const int take = j < hi && (kj > limit || (eq && before < ties));
    ties -= min(ties, all);
    const unsigned takes = __ballot_sync(0xffffffffu, take);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = __popc(takes);
    __syncthreads();
    int place = __popc(takes & ((1u << (tid & 31)) - 1)), total = 0;
    for (int w = 0; w < kSelThreads / 32; w++) {
      place += w < (tid >> 5) ? red[w] : 0;
      total += red[w];
    }
    if (take) out[at + place] = j;
    at += total;
  }
}

zl_status check_paged(const char* who, int B, int H, int Hkv, int d, int bs, int max_blocks, int64_t num_blocks,
                      zl_dtype dtype) {
  using namespace zl;
  if (!dtype_ok(dtype)) return set_error(ZL_ERR_INVALID_ARG, "%s: bad dtype %d", who, (int)dtype);
  if (H <= 0 || Hkv <= 0 || d <= 0 || H % Hkv)
    return set_error(ZL_ERR_INVALID_ARG, "%s: bad head shape H=%d Hkv=%d d=%d", who, H, Hkv, d);
  if (B < 0 || bs <= 0 || max_blocks < 0 || num_blocks < 0)
    return set_error(ZL_ERR_INVALID_ARG, "%s: bad sizes B=%d bs=%d max_blocks=%d blocks=%lld", who, B, bs, max_blocks,
                     (long long)num_blocks);
  return ZL_OK;
}

// CTAs of 8 warps for `units` (sequence, kv head) pairs with up to `blocks` blocks each.
dim3 grid_of(int64_t units, int64_t blocks) {
  const int64_t y = units < 65535 ? units : 65535, x = (blocks + 7) / 8;
  return dim3((unsigned)(x < 1 ? 1 : x > 4096 ? 4096 : x), (unsigned)y);
}

}  // namespace

using namespace zl;

extern "C" {

zl_status zl_block_bounds(zl_ctx* ctx, const void* k_pool, const int32_t* block_tables, const int32_t* tok_begin,
                          const int32_t* seq_lens, void* bounds, int num_seqs, int num_kv_heads, int head_dim,
                          int block_size, int max_blocks_per_seq, int64_t num_blocks, zl_dtype dtype,
                          zl_stream stream) {
  zl_status s = check_paged("block_bounds", num_seqs, num_kv_heads, num_kv_heads, head_dim, block_size,
                            max_blocks_per_seq, num_blocks, dtype);
  if (s != ZL_OK) return s;
  if (num_seqs == 0 || max_blocks_per_seq == 0) return ZL_OK;
  if (!k_pool || !block_tables || !seq_lens || !bounds)
    return set_error(ZL_ERR_INVALID_ARG, "block_bounds: null pointer");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  PagedArgs g{block_tables, seq_lens, num_seqs, num_kv_heads, num_kv_heads, head_dim, block_size,
              max_blocks_per_seq, num_blocks, 0, ctx->d_status};
  const dim3 grid = grid_of((int64_t)num_seqs * num_kv_heads, max_blocks_per_seq);
  if (dtype == ZL_F32)
    bounds_elem_kernel<float><<<grid, 256, 0, S(stream)>>>(g, (const float*)k_pool, tok_begin, (float*)bounds);
  else
    bounds_elem_kernel<__nv_bfloat16><<<grid, 256, 0, S(stream)>>>(g, (const __nv_bfloat16*)k_pool, tok_begin,
                                                                   (__nv_bfloat16*)bounds);
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

zl_status zl_block_scores(zl_ctx* ctx, const void* q, const void* bounds, const int32_t* block_tables,
                          const int32_t* seq_lens, float* scores, int num_seqs, int num_heads, int num_kv_heads,
                          int head_dim, int block_size, int max_blocks_per_seq, int64_t num_blocks, float scale,
                          zl_gqa_map gqa_map, zl_dtype dtype, zl_stream stream) {
  zl_status s = check_paged("block_scores", num_seqs, num_heads, num_kv_heads, head_dim, block_size,
                            max_blocks_per_seq, num_blocks, dtype);
  if (s != ZL_OK) return s;
  if (num_seqs == 0 || max_blocks_per_seq == 0) return ZL_OK;
  if (!q || !bounds || !block_tables || !seq_lens || !scores)
    return set_error(ZL_ERR_INVALID_ARG, "block_scores: null pointer");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  PagedArgs g{block_tables, seq_lens, num_seqs, num_heads, num_kv_heads, head_dim, block_size,
              max_blocks_per_seq, num_blocks, gqa_map == ZL_GQA_MODULO, ctx->d_status};
  const dim3 grid = grid_of((int64_t)num_seqs * num_kv_heads, max_blocks_per_seq);
  const float sc = resolve_scale(scale, head_dim);
  if (dtype == ZL_F32)
    scores_elem_kernel<float><<<grid, 256, 0, S(stream)>>>(g, (const float*)q, (const float*)bounds, sc, scores);
  else
    scores_elem_kernel<__nv_bfloat16><<<grid, 256, 0, S(stream)>>>(g, (const __nv_bfloat16*)q,
                                                                   (const __nv_bfloat16*)bounds, sc, scores);
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

zl_status zl_select_blocks(zl_ctx* ctx, const float* scores, const int32_t* seq_lens, int32_t* selected, int num_seqs,
                           int num_kv_heads, int block_size, int max_blocks_per_seq, int max_selected, int num_first,
                           int num_last, zl_stream stream) {
  if (num_seqs < 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq < 0 || max_selected < 0)
    return set_error(ZL_ERR_INVALID_ARG, "select_blocks: bad sizes B=%d Hkv=%d bs=%d max_blocks=%d max_selected=%d",
                     num_seqs, num_kv_heads, block_size, max_blocks_per_seq, max_selected);
  if (num_first < 0 || num_last < 0 || (int64_t)num_first + num_last > max_selected)
    return set_error(ZL_ERR_INVALID_ARG, "select_blocks: %d first and %d last blocks of %d selected", num_first,
                     num_last, max_selected);
  if (num_seqs == 0 || max_selected == 0) return ZL_OK;
  const int64_t rows = (int64_t)num_seqs * num_kv_heads;
  if (rows > INT32_MAX) return set_error(ZL_ERR_INVALID_ARG, "select_blocks: B*Hkv too large");
  if ((!scores && max_blocks_per_seq) || !seq_lens || !selected)
    return set_error(ZL_ERR_INVALID_ARG, "select_blocks: null pointer");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  select_kernel<<<(unsigned)rows, kSelThreads, 0, S(stream)>>>(scores, seq_lens, num_kv_heads, max_blocks_per_seq,
                                                               block_size, max_selected, num_first, num_last, selected,
                                                               ctx->d_status);
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

}  // extern "C"
