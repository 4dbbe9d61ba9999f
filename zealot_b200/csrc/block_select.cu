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
#include "zl_ptx.cuh"

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
  zl::ptx::griddep_enter();
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

// Elementwise min and max of four 32-bit words of T, NaN where an operand is.
template <typename T> __device__ __forceinline__ uint32_t word_min(uint32_t a, uint32_t b);
template <typename T> __device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t word_min<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(min_nan(__uint_as_float(a), __uint_as_float(b)));
}
template <> __device__ __forceinline__ uint32_t word_max<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
}
template <> __device__ __forceinline__ uint32_t word_min<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t word_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ void merge(uint4& lo, uint4& hi, const uint4& a, const uint4& b) {
  lo.x = word_min<T>(lo.x, a.x);
  lo.y = word_min<T>(lo.y, a.y);
  lo.z = word_min<T>(lo.z, a.z);
  lo.w = word_min<T>(lo.w, a.w);
  hi.x = word_max<T>(hi.x, b.x);
  hi.y = word_max<T>(hi.y, b.y);
  hi.z = word_max<T>(hi.z, b.z);
  hi.w = word_max<T>(hi.w, b.w);
}

// Rows of 16-byte chunks, up to 32 CH of them: one warp per block and kv head, LPR lanes
// to a row (a power of two), CH chunks to a lane, ROWS = 32 / LPR * DEPTH rows at a time,
// all of whose loads are in flight at once. A warp keeps to one head; the warps of the
// heads of one block, whose keys lie side by side, are neighbours. HBM-bound: 16 prompts of
// 256 to 8,192 tokens, 8 heads of 128 bf16, 27.3 us for 156 MB (5.7 TB/s); 64 of 2,048 to 4,096
// 72 us (6.2 TB/s). The work per block had to shrink for that: with a division and a search for
// each block 34 us, and 37 with copies ahead through shared memory on top.
template <typename T, int LPR, int CH>
__global__ void __launch_bounds__(256, 4)
bounds_vec_kernel(PagedArgs g, const T* __restrict__ k_pool, const int32_t* __restrict__ tok_begin,
                  T* __restrict__ bounds) {
  zl::ptx::griddep_enter();
  constexpr int RPL = 32 / LPR, DEPTH = CH == 1 ? 8 : 4, ROWS = RPL * DEPTH, VEC = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, sub = lane / LPR, ch = lane % LPR;
  const int chunks = g.d / VEC, warps = gridDim.x * 8, step = warps / g.Hkv;  // blocks at a time
  const int gw = blockIdx.x * 8 + (threadIdx.x >> 5), j0 = gw / g.Hkv, h = gw - j0 * g.Hkv;
  if (j0 >= step) return;
  const bool mine[2] = {ch < chunks, ch + LPR < chunks};
  const int64_t block = (int64_t)g.Hkv * g.bs * chunks, head = (int64_t)h * g.bs * chunks;  // in 16-byte chunks
  const uint4* pool = reinterpret_cast<const uint4*>(k_pool) + head + ch;
  uint4* out0 = reinterpret_cast<uint4*>(bounds) + (int64_t)h * 2 * chunks + ch;
  for (int b = blockIdx.y; b < g.B; b += gridDim.y) {
    const int64_t len = seq_len(g, b);
    const int n = (int)zl::blocks_of(len, g.bs);
    const int64_t first = (tok_begin ? max(tok_begin[b], 0) / g.bs : 0) + (int64_t)j0;
    if (first >= n) continue;
    int j = (int)first;
    int64_t id = block_id(g, b, j), next;
    for (; j < n; j += step, id = next) {
      next = j + step < n ? block_id(g, b, j + step) : -1;
      if (id < 0) continue;
      const uint4* rows = pool + id * block;
      const int toks = (int)min((int64_t)g.bs, len - (int64_t)j * g.bs);
      uint4 lo[CH], hi[CH];
      for (int t = 0; t < toks; t += ROWS) {
        uint4 v[DEPTH][CH];
        if (t + ROWS <= toks) {
          const uint4* p = rows + (int64_t)(t + sub) * chunks;
#pragma unroll
          for (int k = 0; k < DEPTH; k++, p += RPL * chunks)
#pragma unroll
            for (int c = 0; c < CH; c++) v[k][c] = mine[c] ? __ldg(p + c * LPR) : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
          for (int k = 0; k < DEPTH; k++) {
            const int r = min(t + k * RPL + sub, toks - 1);  // a row twice changes nothing
#pragma unroll
            for (int c = 0; c < CH; c++)
              v[k][c] = mine[c] ? __ldg(rows + (int64_t)r * chunks + c * LPR) : make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
          if (t == 0) lo[c] = hi[c] = v[0][c];
          else merge<T>(lo[c], hi[c], v[0][c], v[0][c]);
#pragma unroll
          for (int k = 1; k < DEPTH; k++) merge<T>(lo[c], hi[c], v[k][c], v[k][c]);
        }
      }
      uint4* out = out0 + id * g.Hkv * 2 * chunks;
#pragma unroll
      for (int c = 0; c < CH; c++) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) {
          uint4 a, z;
          a.x = __shfl_xor_sync(0xffffffffu, lo[c].x, o);
          a.y = __shfl_xor_sync(0xffffffffu, lo[c].y, o);
          a.z = __shfl_xor_sync(0xffffffffu, lo[c].z, o);
          a.w = __shfl_xor_sync(0xffffffffu, lo[c].w, o);
          z.x = __shfl_xor_sync(0xffffffffu, hi[c].x, o);
          z.y = __shfl_xor_sync(0xffffffffu, hi[c].y, o);
          z.z = __shfl_xor_sync(0xffffffffu, hi[c].z, o);
          z.w = __shfl_xor_sync(0xffffffffu, hi[c].w, o);
          merge<T>(lo[c], hi[c], a, z);
        }
        if (mine[c] && sub == 0) {
          out[c * LPR] = lo[c];
          out[chunks + c * LPR] = hi[c];
        }
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
  zl::ptx::griddep_enter();
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

// Bounds rows that 16-byte loads can read.
//
// bf16: a warp scores 16 blocks with matrix instructions: the blocks are M = 16, the
// (at most 8) query heads N, and the 2 d products of a block's two rows with min(q, 0)
// and max(q, 0) the sum. A lane's 16 bytes of its two blocks' rows are its operands for
// two steps of K = 16, q loaded in the same order; products of bf16 are exact in fp32.
// Each warp keeps a ring of ST tiles (16 blocks' bounds) in shared memory, filled by
// asynchronous copies, and the block ids of one tile more. Chunk ch of row r lies at
// ch ^ swz(r), so that the two rows that a quarter warp reads do not meet in a bank.
// HBM-bound: 8 sequences of 131,072 tokens, 64 query and 8 key heads, 45.8 us for 271 MB (5.9
// TB/s). Loads straight into registers took 74 us, the ring 60, 32-bit row numbers and whole
// rounds of CTAs 45. CTAs of one warp start and end on their own: 64 sequences of 2,048 to 4,096
// tokens 11.6 us against 13.4 with four warps to a CTA, of 512 to 4,096 9.8.
constexpr int kScoreWarps = 1, kScoreCtas = 12;
template <int DT, int ST>
__global__ void __launch_bounds__(kScoreWarps * 32)
scores_mma_kernel(PagedArgs g, int parts, const __nv_bfloat16* __restrict__ q,
                  const __nv_bfloat16* __restrict__ bounds, float scale, float* __restrict__ scores) {
  zl::ptx::griddep_enter();
  constexpr int KC = DT / 32, ROW = DT * 4;  // a row: lo and hi side by side, DT elements each
  constexpr int CPR = DT / 4;                // its 16-byte chunks
  extern __shared__ __align__(128) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const int group = g.H / g.Hkv;
  // the heads of the same blocks, whose bounds lie side by side, run at the same time
  const int h = (int)(blockIdx.x % g.Hkv), part = (int)(blockIdx.x / g.Hkv % parts), b = (int)(blockIdx.x / g.Hkv / parts);
  const int64_t u = (int64_t)b * g.Hkv + h;
  const uint32_t mine = zl::ptx::smem_u32(ring) + warp * ST * 16 * ROW;
  const int32_t* table = g.tables + (int64_t)b * g.max_blocks;
  auto swz = [](int r) { return (r & 1) << 2 | (r >> 1 & 3); };
  const int nb = (int)zl::blocks_of(seq_len(g, b), g.bs), tiles = (g.max_blocks + 15) / 16, some = (nb + 15) / 16;
  const int t0 = part * kScoreWarps + warp, step = parts * kScoreWarps;
  auto load_ids = [&](int tile) {  // lane i < 16: the id of the tile's block i
    const int j = tile * 16 + lane;
    return lane < 16 && j < nb ? table[j] : -1;
  };
  // copy `it` of a lane: chunk ch of the tile's row r; a row of 64 chunks takes two copies
  const int z0 = lane % CPR / (CPR / 2), e0 = (lane % CPR - z0 * (CPR / 2)) * 8;
  const bool used = e0 < g.d;
  const uint8_t* mine_src = reinterpret_cast<const uint8_t*>(bounds + (used ? z0 * g.d + e0 : 0));
  const int64_t row_bytes = 4 * g.d;
  auto fetch = [&](int tile, int slot, int32_t id) {  // which of the 16 blocks there are
    uint32_t there = 0;
    if (tile < some) {
      if (id >= g.num_blocks) {
        atomicOr(g.status, ZL_DEV_OOB);
        id = -1;
      }
      there = __ballot_sync(0xffffffffu, id >= 0);
      const int row = id < 0 ? -1 : id * g.Hkv + h;
#pragma unroll
      for (int it = 0; it < 16 * CPR / 32; it++) {
        const int r = (it * 32 + lane) / CPR, ch = (it * 32 + lane) % CPR;
        const int from = __shfl_sync(0xffffffffu, row, r);
        const bool use = from >= 0 && used;
        const uint8_t* src = mine_src + (use ? from : 0) * row_bytes + (CPR == 64 && it % 2 && used ? 2 * g.d : 0);
        zl::ptx::copy16(mine + (slot * 16 + r) * ROW + (ch ^ swz(r)) * 16, src, use);
      }
    }
    zl::ptx::copies_commit();
    return there;
  };
  int32_t id = load_ids(t0);
  uint32_t seen[ST];
#pragma unroll
  for (int i = 0; i < ST - 1; i++) {
    const int32_t next = load_ids(t0 + (i + 1) * step);
    seen[i] = fetch(t0 + i * step, i, id);
    id = next;
  }
  uint4 x[KC];
#pragma unroll
  for (int k = 0; k < KC; k++) {
    x[k] = make_uint4(0, 0, 0, 0);
    if (n < group && k * 32 + c * 8 < g.d) {
      const int head = g.modulo ? n * g.Hkv + h : h * group + n;
      x[k] = __ldg(reinterpret_cast<const uint4*>(q + ((int64_t)b * g.H + head) * g.d + k * 32 + c * 8));
    }
  }
  float* out = scores + u * g.max_blocks;
  for (int tile = t0; tile < some;) {
#pragma unroll
    for (int slot = 0; slot < ST; slot++, tile += step) {
      if (tile >= some) break;
      const int32_t next = load_ids(tile + ST * step);
      seen[(slot + ST - 1) % ST] = fetch(tile + (ST - 1) * step, (slot + ST - 1) % ST, id);
      id = next;
      zl::ptx::copies_wait<ST - 1>();
      __syncwarp();
      const uint32_t rows = mine + (slot * 16 + n) * ROW;
      float s[2][4];
#pragma unroll
      for (int z = 0; z < 2; z++) {
        s[z][0] = s[z][1] = s[z][2] = s[z][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
          auto side = [&](uint32_t a) { return z ? word_max<__nv_bfloat16>(a, 0u) : word_min<__nv_bfloat16>(a, 0u); };
          const uint32_t at = rows + ((z * (CPR / 2) + k * 4 + c) ^ swz(n)) * 16;  // swz(n + 8) is the same
          const uint4 v = zl::ptx::lds16(at), w = zl::ptx::lds16(at + 8 * ROW);
          zl::ptx::mma_bf16_16816(s[z], v.x, w.x, v.y, w.y, side(x[k].x), side(x[k].y));
          zl::ptx::mma_bf16_16816(s[z], v.z, w.z, v.w, w.w, side(x[k].z), side(x[k].w));
        }
      }
      // rows n and n + 8, heads 2 c and 2 c + 1
#pragma unroll
      for (int r = 0; r < 2; r++) {
        float best = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; i++)
          if (2 * c + i < group) best = max_nan(best, (s[0][2 * r + i] + s[1][2 * r + i]) * scale);
        best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, 1));
        best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, 2));
        const int j = tile * 16 + n + 8 * r;
        if (c == r && j < g.max_blocks) out[j] = seen[slot] >> (n + 8 * r) & 1 ? best : -INFINITY;
      }
      __syncwarp();  // the next fetch takes this slot
    }
  }
  zl::ptx::copies_wait<0>();
  // after the sequence's last tile
  for (int tile = some + t0; tile < tiles; tile += step)
    if (lane < 16 && tile * 16 + lane < g.max_blocks) out[tile * 16 + lane] = -INFINITY;
}

// fp32 (and bf16 with more than 8 query heads to a kv head): eight lanes share a
// block's rows, a warp scores four blocks at a time on the CUDA cores; q's two sides
// are in shared memory, 8 heads at a time. 8 sequences of 65,536 to 131,072 tokens, 32
// fp32 query heads: 91 us for 402 MB (4.4 TB/s), bound by the latency of each tile's
// loads and products; three CTAs of more registers to an SM took 115.
// bf16, 8 sequences of 131,072 tokens, 8 key heads of 128: 9 query heads to each 321 us, 16 531
// (8, on the matrix instructions, 46): bound by the products, one head at a time.
template <typename T, int NV>
__global__ void __launch_bounds__(256) scores_vec_kernel(PagedArgs g, int parts, const T* __restrict__ q,
                                                         const T* __restrict__ bounds, float scale,
                                                         float* __restrict__ scores) {
  zl::ptx::griddep_enter();
  constexpr int VEC = 16 / sizeof(T), DT = NV * 8 * VEC;
  __shared__ __align__(16) float sides[2][8][DT];
  const int lane = threadIdx.x & 31, tg = lane >> 3, li = lane & 7;
  const int group = g.H / g.Hkv;
  // the heads of the same blocks, whose bounds lie side by side, run at the same time
  const int h = (int)(blockIdx.x % g.Hkv), part = (int)(blockIdx.x / g.Hkv % parts), b = (int)(blockIdx.x / g.Hkv / parts);
  const int64_t u = (int64_t)b * g.Hkv + h;
  const int nb = (int)zl::blocks_of(seq_len(g, b), g.bs), tiles = (g.max_blocks + 3) / 4;
  float* out = scores + u * g.max_blocks;
  for (int h0 = 0; h0 < group; h0 += 8) {
    const int heads = min(8, group - h0);
    if (h0) __syncthreads();
    for (int i = threadIdx.x; i < heads * DT; i += 256) {
      const int k = i / DT, e = i - k * DT;
      const int head = g.modulo ? (h0 + k) * g.Hkv + h : h * group + h0 + k;
      const float f = e < g.d ? to_f(q[((int64_t)b * g.H + head) * g.d + e]) : 0.f;
      sides[0][k][e] = min_nan(f, 0.f);
      sides[1][k][e] = max_nan(f, 0.f);
    }
    __syncthreads();
    const int32_t* table = g.tables + (int64_t)b * g.max_blocks;
    const T* mine = bounds + (int64_t)h * 2 * g.d + li * VEC;
    const int64_t block = (int64_t)g.Hkv * 2 * g.d;
    int j = (part * 8 + (threadIdx.x >> 5)) * 4 + tg;
    int32_t id = j < nb ? table[j] : -1, next;
    for (int tile = part * 8 + (threadIdx.x >> 5); tile < tiles; tile += parts * 8, j += parts * 32, id = next) {
      next = j + parts * 32 < nb ? table[j + parts * 32] : -1;
      if (id >= g.num_blocks) {
        atomicOr(g.status, ZL_DEV_OOB);
        id = -1;
      }
      uint4 v[2][NV];
#pragma unroll
      for (int z = 0; z < 2; z++)
#pragma unroll
        for (int k = 0; k < NV; k++) {
          v[z][k] = make_uint4(0, 0, 0, 0);
          if (id >= 0 && (k * 8 + li) * VEC < g.d)
            v[z][k] = __ldg(reinterpret_cast<const uint4*>(mine + id * block + z * g.d + k * 8 * VEC));
        }
      float best = -INFINITY;
      for (int i = 0; i < heads; i++) {
        float s = 0.f;
#pragma unroll
        for (int z = 0; z < 2; z++)
#pragma unroll
          for (int k = 0; k < NV; k++) {
            const T* e = reinterpret_cast<const T*>(&v[z][k]);
            const float* f = &sides[z][i][(k * 8 + li) * VEC];
#pragma unroll
            for (int y = 0; y < VEC; y++) s = fmaf(f[y], to_f(e[y]), s);
          }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        best = max_nan(best, s * scale);
      }
      if (li == 0 && j < g.max_blocks) {
        if (id < 0) best = -INFINITY;
        out[j] = h0 ? max_nan(out[j], best) : best;
      }
    }
  }
}

// ---------------------------------------------------------------- selection

// The `top` blocks of one (sequence, kv head), ascending: the first `first`, the
// last `last` and the best of those between, equal scores by the lower index.
// With m = top - (first + last) still to choose from the middle, the threshold is
// the largest key that at least m middle keys reach. A key's place in the output is
// the number of keys above the threshold before it and of equal ones, of which the
// first few count: no key's place depends on the order of the threads.
//
// Reads 4 bytes a block, so bound by its own steps: the instructions for each key, and
// the barriers between digits. 256 of up to 8,192 blocks in 512 rows 14.7 us, in 8 rows
// 6.2 us; 32 of some 100 in 32 rows 2.8 us. On the way there 512 rows took 18.5 with every
// lane finding its own keys' places (now one lane walks the chosen bits of 32 keys) and the
// keys past a row's end taken along.
struct SelectArgs {
  const float* scores;
  const int32_t* seq_lens;
  int32_t* selected;
  int Hkv, max_blocks, bs, top, first, last;
  int* status;
};

// The parts of a row that need no search; returns whether that was all. [lo, hi): the
// middle blocks, of which m are to be chosen.
template <int THREADS>
__device__ __forceinline__ bool select_ends(const SelectArgs& g, int64_t row, int& lo, int& hi, int& m) {
  const int tid = threadIdx.x;
  int32_t* out = g.selected + row * g.top;
  const int64_t want = zl::blocks_of(g.seq_lens[row / g.Hkv], g.bs);
  if (want > g.max_blocks && tid == 0) atomicOr(g.status, ZL_DEV_OOB);
  const int n = (int)min(want, (int64_t)g.max_blocks);
  lo = g.first;
  hi = n - g.last;
  m = g.top - g.first - g.last;
  if (n <= g.top) {
    for (int j = tid; j < g.top; j += THREADS) out[j] = j < n ? j : -1;
    return true;
  }
  // n > top >= first + last: the three parts do not meet
  for (int j = tid; j < g.first; j += THREADS) out[j] = j;
  for (int j = tid; j < g.last; j += THREADS) out[g.top - g.last + j] = hi + j;
  return m == 0;
}

// The threshold among keys in registers, BITS bits at a time (the last digit has what is
// left): a histogram in shared memory for each digit over the keys that share the digits
// before it. Keys past the first `used` of each thread are 0, as are those that do not count:
// below every score's, so that they change no digit that is found. m becomes the number of
// keys at the threshold that are to be chosen, `whole` whether that is all of them.
template <int THREADS, int R, int BITS>
__device__ __forceinline__ uint32_t limit_by_digits(const uint32_t (&key)[R], int used, int& m, bool& whole) {
  constexpr int BINS = 1 << BITS, PER = BINS > THREADS ? BINS / THREADS : 1, W = THREADS / 32;
  __shared__ int hist[BINS];
  __shared__ int sums[W];
  __shared__ int found[3];  // the digit, how many keys of its bin are still to be chosen, how many it has
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t limit = 0, mask = 0;
#pragma unroll
  for (int left = 32; left > 0; left -= BITS) {
    const int width = left < BITS ? left : BITS, shift = left - width;
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (k * THREADS + tid < BINS) hist[k * THREADS + tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; i++) {
      if (i >= used) break;
      const bool in = key[i] != 0 && ((key[i] ^ limit) & mask) == 0;
      const int bin = key[i] >> shift & ((1 << width) - 1);
      if (in) atomicAdd(&hist[bin], 1);
    }
    __syncthreads();
    // sums from the top bin down: this thread has bins [top - PER + 1, top], or none
    const int top = BINS - 1 - tid * PER;
    int own = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) own += top >= 0 ? hist[top - k] : 0;
    int incl = own;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    const int s = lane < W ? sums[lane] : 0;
    int above = incl - own + __reduce_add_sync(0xffffffffu, lane < warp ? s : 0);
#pragma unroll
    for (int k = 0; k < PER; k++) {  // one bin holds the m-th key from the top
      const int c = top >= 0 ? hist[top - k] : 0;
      if (above < m && m <= above + c) {
        found[0] = top - k;
        found[1] = m - above;
        found[2] = c;
      }
      above += c;
    }
    __syncthreads();
    limit |= (uint32_t)found[0] << shift;
    m = found[1];
    mask |= ((1u << width) - 1) << shift;
  }
  whole = m == found[2];
  return limit;
}

// Tables of up to THREADS R blocks: each thread keeps R keys, key i of thread t being
// block i * THREADS + t.
template <int THREADS, int R, int BITS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 4 : 1) select_reg_kernel(SelectArgs g) {
  zl::ptx::griddep_enter();
  constexpr int W = THREADS / 32;
  __shared__ uint32_t before[R * W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const float* sc = g.scores + row * g.max_blocks;
  int32_t* out = g.selected + row * g.top;
  uint32_t key[R];
#pragma unroll
  for (int i = 0; i < R; i++) {  // loaded before the length is known
    const int j = i * THREADS + tid;
    key[i] = j < g.max_blocks ? __float_as_uint(__ldg(sc + j)) : 0;
  }
  int lo, hi, m;
  if (select_ends<THREADS>(g, row, lo, hi, m)) return;
  const int used = R < 8 ? R : (hi + THREADS - 1) / THREADS;  // keys of a thread that can be in the middle
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int j = i * THREADS + tid;
    if (i < used) key[i] = j >= lo && j < hi ? zl::score_key(key[i]) : 0;  // 0 is no score's key (-inf has 0x007fffff)
  }
  bool whole;
  const uint32_t limit = limit_by_digits<THREADS, R, BITS>(key, used, m, whole);
  // each warp's keys above the limit and, where only some of those at it are chosen, those at
  // it: bit l of lane i's words for key i of lane l
  const uint32_t over = whole ? limit - 1 : limit;
  uint32_t gts = 0, eqs = 0;
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (i >= used) break;
    const uint32_t gt = __ballot_sync(0xffffffffu, key[i] > over);
    const uint32_t eq = whole ? 0 : __ballot_sync(0xffffffffu, key[i] == limit);
    if (lane == i) {
      gts = gt;
      eqs = eq;
    }
  }
  if (lane < R) before[lane * W + warp] = __popc(gts) | __popc(eqs) << 16;  // counts, in index order
  __syncthreads();
  if (warp == 0) {  // exclusive sums of both halves; no total passes 31 * 1024
    constexpr int PER = (R * W + 31) / 32;
    uint32_t mine[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int at = lane * PER + k;
      mine[k] = at < R * W ? before[at] : 0;
      sum += mine[k];
    }
    uint32_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    uint32_t at = incl - sum;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      if (lane * PER + k < R * W) before[lane * PER + k] = at;
      at += mine[k];
    }
  }
  __syncthreads();
  const int ties = whole ? 0 : m;
  const uint32_t b = lane < R ? before[lane * W + warp] : 0;
  int at = lo + (int)(b & 0xffff) + min((int)(b >> 16), ties);
  const int take = min(max(ties - (int)(b >> 16), 0), __popc(eqs));  // of the equal keys, the first so many
  while (__popc(eqs) > take) eqs &= ~(0x80000000u >> __clz(eqs));
  if constexpr (R >= 8) {  // lane i writes its words' keys: few are chosen of many
    for (uint32_t out_keys = gts | eqs; out_keys; out_keys &= out_keys - 1)
      out[at++] = lane * THREADS + warp * 32 + __ffs(out_keys) - 1;
  } else {
#pragma unroll
    for (int i = 0; i < R; i++) {
      const uint32_t chosen = __shfl_sync(0xffffffffu, gts | eqs, i);
      const int from = __shfl_sync(0xffffffffu, at, i);
      if (chosen >> lane & 1) out[from + __popc(chosen & ((1u << lane) - 1))] = i * THREADS + tid;
    }
  }
}

// Longer tables: the keys are read again, from L2, in every pass.
constexpr int kSelThreads = 1024;

__device__ __forceinline__ int block_count(int c, int* red) {  // sum over the CTA, to every thread
  c = __reduce_add_sync(0xffffffffu, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = c;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, red[threadIdx.x & 31]);
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(SelectArgs g) {
  zl::ptx::griddep_enter();
  __shared__ int red[kSelThreads / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* sc = g.scores + row * g.max_blocks;
  int32_t* out = g.selected + row * g.top;
  int lo, hi, m;
  if (select_ends<kSelThreads>(g, row, lo, hi, m)) return;
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
  // write in index order, one index per thread and pass
  int at = lo;
  for (int64_t base = lo; base < hi; base += kSelThreads) {
    const int64_t j = base + tid;
    const uint32_t kj = j < hi ? key((int)j) : 0;
    const unsigned gts = __ballot_sync(0xffffffffu, kj > limit), eqs = __ballot_sync(0xffffffffu, kj == limit);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(gts) | __popc(eqs) << 16;
    __syncthreads();
    const int mine = red[lane];
    const int all = __reduce_add_sync(0xffffffffu, mine), pre = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
    const int gt = (pre & 0xffff) + __popc(gts & ((1u << lane) - 1)), eq = (pre >> 16) + __popc(eqs & ((1u << lane) - 1));
    if (kj > limit || (j < hi && kj == limit && eq < ties)) out[at + gt + min(eq, ties)] = (int)j;
    const int used = min(ties, all >> 16);
    at += (all & 0xffff) + used;
    ties -= used;
  }
}

zl_status check_paged(const char* who, int B, int H, int Hkv, int d, int bs, int max_blocks, int64_t num_blocks,
                      zl_dtype dtype) {
  using namespace zl;
  if (!dtype_ok(dtype)) return set_error(ZL_ERR_INVALID_ARG, "%s: bad dtype %d", who, (int)dtype);
  if (H <= 0 || Hkv <= 0 || d <= 0 || H % Hkv)
    return set_error(ZL_ERR_INVALID_ARG, "%s: bad head shape H=%d Hkv=%d d=%d", who, H, Hkv, d);
  if (B < 0 || bs <= 0 || max_blocks < 0 || max_blocks > 1 << 30 || num_blocks < 0)
    return set_error(ZL_ERR_INVALID_ARG, "%s: bad sizes B=%d bs=%d max_blocks=%d blocks=%lld", who, B, bs, max_blocks,
                     (long long)num_blocks);
  return ZL_OK;
}

// CTAs of 8 warps for `units` (sequence, kv head) pairs with up to `blocks` blocks each.
dim3 grid_of(int64_t units, int64_t blocks) {
  const int64_t y = units < 65535 ? units : 65535, x = (blocks + 7) / 8;
  return dim3((unsigned)(x < 1 ? 1 : x > 4096 ? 4096 : x), (unsigned)y);
}

constexpr int kBoundsWaves = 16;
template <typename T>
void launch_bounds_vec(const PagedArgs& g, const void* k_pool, const int32_t* tok_begin, void* bounds, int num_sms,
                       cudaStream_t st) {
  const int chunks = g.d * (int)sizeof(T) / 16;
  // CTAs for each sequence: some kBoundsWaves to an SM in all for whole prompts of any lengths. With
  // tok_begin, which is a step's few tokens or a chunk of a prompt (the lengths, on the device, say
  // which), some 4 to an SM, or one where there are many sequences, which are seldom chunks. One and
  // 4 to an SM: 16 sequences of a new token 1.9 and 4.4 us, 64 2.0 and 4.7, 128 2.4 and 4.6; chunks
  // of 512 tokens of 16 sequences 5.8 and 4.0, of 37 8.2 and 5.7, of 64 12.8 and 11.2, of 128 28 and
  // 31; of 8,192 tokens of 16 68 and 54, of 64 229 and 217 (184 with kBoundsWaves). So few sequences
  // of one token pay 2.5 us, and long chunks of many up to a fifth.
  int64_t x = ((int64_t)g.max_blocks * g.Hkv + 7) / 8;
  const int an_sm = !tok_begin ? kBoundsWaves : g.B >= num_sms / 4 ? 1 : 4;
  const int64_t few = (an_sm * (int64_t)num_sms + g.B - 1) / g.B, least = (g.Hkv + 7) / 8;
  x = x > few ? few : x;
  x = x < least ? least : x;
  const dim3 grid((unsigned)x, (unsigned)(g.B < 65535 ? g.B : 65535));
  const T* k = (const T*)k_pool;
  T* o = (T*)bounds;
  if (chunks <= 8) zl::launch_ahead(bounds_vec_kernel<T, 8, 1>, grid, 256, 0, st, g, k, tok_begin, o);
  else if (chunks <= 16) zl::launch_ahead(bounds_vec_kernel<T, 16, 1>, grid, 256, 0, st, g, k, tok_begin, o);
  else if (chunks <= 32) zl::launch_ahead(bounds_vec_kernel<T, 32, 1>, grid, 256, 0, st, g, k, tok_begin, o);
  else zl::launch_ahead(bounds_vec_kernel<T, 32, 2>, grid, 256, 0, st, g, k, tok_begin, o);
}

// CTAs for each of `rows` rows of `tiles` tiles, `warps` tiles at a time: not more than
// `ctas` in all where that leaves one for each row, each warp then taking several tiles of
// long rows with one load of q.
int scores_parts(int64_t rows, int64_t tiles, int warps, int64_t ctas) {
  int64_t x = ctas / rows;
  if (x > (tiles + warps - 1) / warps) x = (tiles + warps - 1) / warps;
  return (int)(x < 1 ? 1 : x);
}

template <int DT, int ST>
zl_status launch_scores_mma(const PagedArgs& g, int parts, unsigned grid, const __nv_bfloat16* q,
                            const __nv_bfloat16* bounds, float scale, float* scores, cudaStream_t st) {
  using namespace zl;
  constexpr int smem = kScoreWarps * ST * 16 * DT * 4;
  ZL_CUDA_TRY(cudaFuncSetAttribute(scores_mma_kernel<DT, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  zl::launch_ahead(scores_mma_kernel<DT, ST>, grid, kScoreWarps * 32, smem, st, g, parts, q, bounds, scale, scores);
  return ZL_OK;
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
  const cudaStream_t st = S(stream);
  if (head_dim * dtype_size(dtype) % 16 == 0 && head_dim <= 256 && aligned16(k_pool) && aligned16(bounds)) {
    if (dtype == ZL_F32) launch_bounds_vec<float>(g, k_pool, tok_begin, bounds, ctx->num_sms, st);
    else launch_bounds_vec<__nv_bfloat16>(g, k_pool, tok_begin, bounds, ctx->num_sms, st);
  } else {
    const dim3 grid = grid_of((int64_t)num_seqs * num_kv_heads, max_blocks_per_seq);
    if (dtype == ZL_F32)
      zl::launch_ahead(bounds_elem_kernel<float>, grid, 256, 0, st, g, (const float*)k_pool, tok_begin, (float*)bounds);
    else
      zl::launch_ahead(bounds_elem_kernel<__nv_bfloat16>, grid, 256, 0, st, g, (const __nv_bfloat16*)k_pool, tok_begin,
                                                              (__nv_bfloat16*)bounds);
  }
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
  const float sc = resolve_scale(scale, head_dim);
  const cudaStream_t st = S(stream);
  const int64_t rows = (int64_t)num_seqs * num_kv_heads;
  const int p16 = scores_parts(rows, (max_blocks_per_seq + 15) / 16, kScoreWarps, kScoreCtas * ctx->num_sms),
            p4 = scores_parts(rows, (max_blocks_per_seq + 3) / 4, 8, 4 * ctx->num_sms);
  const bool vec = head_dim * dtype_size(dtype) % 16 == 0 && head_dim <= 256 && aligned16(q) && aligned16(bounds) &&
                   rows * p4 <= INT32_MAX && rows * p16 <= INT32_MAX &&
                   (double)num_blocks * num_kv_heads <= INT32_MAX;
  const unsigned n16 = (unsigned)(rows * p16), n4 = (unsigned)(rows * p4);
  const auto *qb = (const __nv_bfloat16*)q, *bb = (const __nv_bfloat16*)bounds;
  const auto *qf = (const float*)q, *bf = (const float*)bounds;
  if (vec && dtype == ZL_BF16 && num_heads / num_kv_heads <= 8) {
    s = head_dim <= 64    ? launch_scores_mma<64, 4>(g, p16, n16, qb, bb, sc, scores, st)
        : head_dim <= 128 ? launch_scores_mma<128, 2>(g, p16, n16, qb, bb, sc, scores, st)
                          : launch_scores_mma<256, 2>(g, p16, n16, qb, bb, sc, scores, st);
    if (s != ZL_OK) return s;
  } else if (vec && dtype == ZL_BF16) {
    if (head_dim <= 128) zl::launch_ahead(scores_vec_kernel<__nv_bfloat16, 2>, n4, 256, 0, st, g, p4, qb, bb, sc, scores);
    else zl::launch_ahead(scores_vec_kernel<__nv_bfloat16, 4>, n4, 256, 0, st, g, p4, qb, bb, sc, scores);
  } else if (vec) {
    if (head_dim <= 64) zl::launch_ahead(scores_vec_kernel<float, 2>, n4, 256, 0, st, g, p4, qf, bf, sc, scores);
    else if (head_dim <= 128) zl::launch_ahead(scores_vec_kernel<float, 4>, n4, 256, 0, st, g, p4, qf, bf, sc, scores);
    else zl::launch_ahead(scores_vec_kernel<float, 8>, n4, 256, 0, st, g, p4, qf, bf, sc, scores);
  } else {
    const dim3 grid = grid_of(rows, max_blocks_per_seq);
    if (dtype == ZL_F32) zl::launch_ahead(scores_elem_kernel<float>, grid, 256, 0, st, g, qf, bf, sc, scores);
    else zl::launch_ahead(scores_elem_kernel<__nv_bfloat16>, grid, 256, 0, st, g, qb, bb, sc, scores);
  }
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

zl_status zl_select_blocks(zl_ctx* ctx, const float* scores, const int32_t* seq_lens, int32_t* selected, int num_seqs,
                           int num_kv_heads, int block_size, int max_blocks_per_seq, int max_selected, int num_first,
                           int num_last, zl_stream stream) {
  if (num_seqs < 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq < 0 ||
      max_blocks_per_seq > 1 << 30 || max_selected < 0 || max_selected > 1 << 30)
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
  const SelectArgs g{scores, seq_lens, selected, num_kv_heads, max_blocks_per_seq, block_size, max_selected,
                     num_first, num_last, ctx->d_status};
  const unsigned n = (unsigned)rows;
  const cudaStream_t st = S(stream);
  // Threads by the table's width, a few keys to each: with 256 threads and 32 keys instead of
  // 1,024 and 8, 8 rows of 8,192 blocks take 10.1 us, not 6.2. Digits of 8 bits need 256 bins to
  // clear and sum, of 11 bits one pass less: 1,600 rows of 650 blocks 9.5 and 25.8 us, 512 rows of
  // 8,192 15.1 and 14.7. More rows than CTAs of 1,024 threads at once take half the threads (512
  // rows of 8,192 14.7 us, not 20.6; 20.5 with 256). One key to a thread for narrow tables: 32 rows
  // of some 100 blocks 2.8 us, 3.3 with 4.
  const bool many = rows > 2 * ctx->num_sms;
  if (max_blocks_per_seq <= 128) zl::launch_ahead(select_reg_kernel<128, 1, 8>, n, 128, 0, st, g);
  else if (max_blocks_per_seq <= 512) zl::launch_ahead(select_reg_kernel<128, 4, 8>, n, 128, 0, st, g);
  else if (max_blocks_per_seq <= 1024) zl::launch_ahead(select_reg_kernel<256, 4, 8>, n, 256, 0, st, g);
  else if (max_blocks_per_seq <= 2048) zl::launch_ahead(select_reg_kernel<512, 4, 8>, n, 512, 0, st, g);
  else if (max_blocks_per_seq <= 8192 && many) zl::launch_ahead(select_reg_kernel<512, 16, 11>, n, 512, 0, st, g);
  else if (max_blocks_per_seq <= 8192) zl::launch_ahead(select_reg_kernel<1024, 8, 11>, n, 1024, 0, st, g);
  else if (max_blocks_per_seq <= 16384) zl::launch_ahead(select_reg_kernel<1024, 16, 11>, n, 1024, 0, st, g);
  else if (max_blocks_per_seq <= 24576) zl::launch_ahead(select_reg_kernel<1024, 24, 11>, n, 1024, 0, st, g);
  else zl::launch_ahead(select_kernel, n, kSelThreads, 0, st, g);
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

}  // extern "C"
