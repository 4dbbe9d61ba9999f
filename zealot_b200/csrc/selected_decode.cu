// selected_decode.cu -- attention of one token per sequence over the blocks
// that a list gives for each (sequence, kv head).
//
// HBM-bound: the keys and values of the listed blocks are read once for the
// whole group of query heads, and 4 d operations per token and head are little
// beside that. The list of one (sequence, kv head) is split over the CTAs of a
// cluster, each CTA's part over its warps; every warp keeps a running maximum,
// sum and output, which are joined in shared memory and then through the
// cluster's distributed shared memory, in a fixed order. So a call takes no
// workspace and no counter, and a launch for few sequences still fills the GPU.
//
// Every warp keeps a ring of small tiles of keys and values in shared memory,
// filled by asynchronous 16-byte copies: any block size and order, and rows that
// do not count are zeros.
//
// bf16 (selected_mma_kernel), tiles of 16 tokens: S = q K^T has the (at most 8) query
// heads as the upper half of M = 16 and 8 tokens as N: a lane's 16 bytes of a key
// row are its B operands for two steps of K = 16 once q is loaded in the same
// order. O^T = V^T P^T has 16 elements of a value row as M and the heads as N: a
// lane reads 16 bytes of each of four token rows and pairs two tokens' elements
// with a byte permute. S's accumulators are P^T's operands as they stand. P enters
// as two bf16 parts that are both positive: the weights then keep 16 bits, for one more
// instruction per tile in a kernel that waits for memory, and an infinite value gives infinity,
// as it does with one weight (a second part of 0 or below would make it NaN), down to weights
// of 2^-110 of the largest, where the second part leaves bf16's range.
//
// fp32 (selected_f32_kernel), tiles of 8 tokens: eight lanes share a token's row,
// on the CUDA cores with packed pairs.
//
// Measured on one B200 (GPU time, replayed back to back), 32 query and 8 key heads of
// 128: 64 sequences, 128 blocks of 16 tokens each, bf16, 88 us for 535 MB (6.07 TB/s, 93 %
// of the copy rate); one sequence 8.9 us, of which 6 are the chain list -> table -> first
// keys and the join. Loads straight into registers took 174-188 us, the ring 92, the shorter
// join 88. fp32, 64 blocks each: 94 us (5.7 TB/s).
#include <cooperative_groups.h>

#include "zl_internal.h"
#include "zl_pages.h"
#include "zl_ptx.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;
constexpr int kEntries = 512;  // list entries of a CTA that are resolved at a time

struct SelArgs {
  const void *q, *k_pool, *v_pool;
  const int32_t *tables, *seq_lens, *selected;
  void* out;
  int H, Hkv, d, bs, max_blocks, max_selected;
  int64_t num_blocks;
  float scale2;  // scale * log2(e)
  int modulo, group, subs, per_sub;
  int* status;
};

// A listed block: the pool row of its first token and how many of its tokens count.
struct Entry {
  int32_t row, tokens;
};

// Where a CTA works: its (sequence, kv head), its query heads, its part of the list.
struct Job {
  int b, kvh, head0, heads;
  int e0, e1;
  const int32_t* list;
  __device__ int head(const SelArgs& g, int i) const {
    return g.modulo ? (head0 + i) * g.Hkv + kvh : kvh * g.group + head0 + i;
  }
};

// The part is one of `cluster` equal ones of max_selected entries: a list that
// ends early leaves its last CTAs idle, and none has to read the list first.
__device__ __forceinline__ Job find_job(const SelArgs& g, int cluster, int rank) {
  Job w;
  int u = blockIdx.x / cluster;
  const int sub = u % g.subs;
  u /= g.subs;
  w.b = u / g.Hkv;
  w.kvh = u - w.b * g.Hkv;
  w.head0 = sub * g.per_sub;
  w.heads = min(g.per_sub, g.group - w.head0);
  w.list = g.selected + (int64_t)u * g.max_selected;
  const int n = g.max_selected, step = (16 + g.bs - 1) / g.bs;  // whole tiles of 16 tokens
  int per = (n + cluster - 1) / cluster;
  per = (per + step - 1) / step * step;
  w.e0 = min(n, rank * per);
  w.e1 = min(n, w.e0 + per);
  return w;
}

// Resolves list entries [e, e + count) into shared memory and returns how many
// of them come before the list's first negative entry (`end`, kept over calls).
__device__ __forceinline__ int resolve(const SelArgs& g, const Job& w, int e, int count, Entry* sh, int* end) {
  const int32_t* table = g.tables + (int64_t)w.b * g.max_blocks;
  if (threadIdx.x == 0 && e == w.e0) *end = g.max_selected;
  __syncthreads();
  int neg = g.max_selected;
  const int64_t len = g.seq_lens[w.b];
  if (e == w.e0)  // entries of the CTAs before this one
    for (int i = threadIdx.x; i < e; i += kThreads)
      if (w.list[i] < 0) neg = min(neg, i);
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int j = w.list[e + i];
    Entry t{0, 0};
    if (j < 0) {
      neg = min(neg, e + i);
    } else if (j < g.max_blocks) {
      const int64_t left = len - (int64_t)j * g.bs, id = table[j];
      const int64_t row = zl::pool_row(id, g.num_blocks, g.Hkv, w.kvh, g.bs, 0);
      if (left > 0) {
        t.row = (int32_t)(row >= 0 ? row : id >= 0 ? -2 : -1);
        t.tokens = row >= 0 ? (int32_t)min(left, (int64_t)g.bs) : 0;
      }
    } else {
      t.row = -2;
    }
    sh[i] = t;
  }
  if (neg < g.max_selected) atomicMin(end, neg);
  __syncthreads();
  const int used = max(0, min(count, *end - e));
  for (int i = threadIdx.x; i < used; i += kThreads)  // outside the table row or the pool
    if (sh[i].row == -2) atomicOr(g.status, ZL_DEV_OOB);
  return used;
}

// Joins the warps' (m, l, o) and then the cluster's, and writes the heads' outputs.
// o: [kWarps][HEADS][DT] unnormalised, in units of 2^m; rows of DT elements, d used. A
// part that saw nothing has l = 0 and is left out, its m being -inf.
template <typename T, int HEADS, int DT>
__device__ __forceinline__ void finish(const SelArgs& g, const Job& w, int cluster, int rank, float* o,
                                       float (*m)[HEADS], float (*l)[HEADS]) {
  __shared__ float mc[HEADS], lc[HEADS];
  __shared__ float factor[kWarps][HEADS];
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < HEADS) {
    float M = -INFINITY, L = 0.f;
    for (int i = 0; i < kWarps; i++) M = fmaxf(M, m[i][tid]);
    for (int i = 0; i < kWarps; i++) {
      const float f = l[i][tid] != 0.f ? exp2f(m[i][tid] - M) : 0.f;
      factor[i][tid] = f;
      L = fmaf(l[i][tid], f, L);
    }
    mc[tid] = M;
    lc[tid] = L;
  }
  __syncthreads();
  for (int i = tid; i < w.heads * DT; i += kThreads) {
    const int h = i / DT;
    float acc = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; k++) {
      const float f = factor[k][h];
      if (f != 0.f) acc = fmaf(o[k * HEADS * DT + i], f, acc);
    }
    o[i] = acc;
  }
  cg::cluster_group cl = cg::this_cluster();
  if (cluster > 1) cl.sync();
  else __syncthreads();
  T* out = (T*)g.out;
  for (int i = rank * kThreads + tid; i < w.heads * DT; i += cluster * kThreads) {
    const int h = i / DT, e = i - h * DT;
    if (e >= g.d) continue;
    float y = o[i], L = lc[h];
    if (cluster > 1) {
      // all remote loads at once: one trip over the cluster's network for most threads
      float mr[kMaxCluster], lr[kMaxCluster], yr[kMaxCluster], M = -INFINITY;
#pragma unroll
      for (int r = 0; r < kMaxCluster; r++) {
        mr[r] = -INFINITY;
        lr[r] = yr[r] = 0.f;
        if (r < cluster) {
          mr[r] = *cl.map_shared_rank(&mc[h], r);
          lr[r] = *cl.map_shared_rank(&lc[h], r);
          yr[r] = *cl.map_shared_rank(o + i, r);
        }
      }
#pragma unroll
      for (int r = 0; r < kMaxCluster; r++) M = fmaxf(M, mr[r]);
      y = L = 0.f;
#pragma unroll
      for (int r = 0; r < kMaxCluster; r++) {
        const float f = lr[r] != 0.f ? exp2f(mr[r] - M) : 0.f;
        L = fmaf(lr[r], f, L);
        if (f != 0.f) y = fmaf(yr[r], f, y);
      }
    }
    y = L != 0.f ? y / L : 0.f;
    T* at = out + ((int64_t)w.b * g.H + w.head(g, h)) * g.d + e;
    if constexpr (sizeof(T) == 2) *at = __float2bfloat16_rn(y);
    else *at = y;
  }
  if (cluster > 1) cl.sync();  // a CTA's shared memory stays until all have read it
}

// Starts the copies of one tile, TOK tokens' key rows and then their value rows of ROWB
// bytes each (what is behind the real row_bytes is zeros, as are the rows of tokens that do
// not count), as one group; an empty group where there is no such tile. Returns which tokens
// count. With SWIZZLE a row's 16-byte chunks lie at chunk ^ (row & 7).
template <int ROWB, int TOK, bool SWIZZLE>
__device__ __forceinline__ uint32_t fetch_tile(const SelArgs& g, const Entry* entries, int tile, int toks, uint32_t dst,
                                               int row_bytes) {
  constexpr int CPR = ROWB / 16;
  const int lane = threadIdx.x & 31;
  uint32_t there = 0;
  if (tile * TOK < toks) {
    int row = -1;
    const int tok = tile * TOK + lane;
    if (lane < TOK && tok < toks) {
      const int i = tok / g.bs, t = tok - i * g.bs;
      const Entry en = entries[i];
      if (t < en.tokens) row = en.row + t;
    }
    there = __ballot_sync(0xffffffffu, row >= 0);
#pragma unroll
    for (int it = 0; it < TOK * CPR / 32; it++) {
      const int r = (it * 32 + lane) / CPR, ch = (it * 32 + lane) % CPR;
      const int from = __shfl_sync(0xffffffffu, row, r);
      const bool use = from >= 0 && ch * 16 < row_bytes;
      const int64_t at = use ? (int64_t)from * row_bytes + ch * 16 : 0;
      const uint32_t to = dst + r * ROWB + ((SWIZZLE ? ch ^ (r & 7) : ch) * 16);
      zl::ptx::copy16(to, (const uint8_t*)g.k_pool + at, use);
      zl::ptx::copy16(to + TOK * ROWB, (const uint8_t*)g.v_pool + at, use);
    }
  }
  zl::ptx::copies_commit();
  return there;
}

// Shared memory of either kernel: each warp's ring of ST tiles, which the warps' outputs
// take over at the end.
constexpr size_t ring_bytes(int rowb, int tok, int st) { return (size_t)kWarps * st * tok * rowb * 2; }

// The bits of the largest float below p > 0; of 0 where p is 0.
__device__ __forceinline__ uint32_t below(float p) { return max(__float_as_int(p), 1) - 1; }

// head_dim up to DT, a multiple of 8. Column n of the score tile i in {0, 1} is token 2 (n / 2) + i for even n and
// 8 + i + (2 (n / 2) + 4) % 8 for odd n: the two rows that a quarter warp reads of the
// keys then differ in bit 2 of the row, the four that it reads of the values in bits 1
// and 2, and neither has a bank conflict.
template <int DT, int ST>
__global__ void __launch_bounds__(kThreads) selected_mma_kernel(SelArgs g, int cluster) {
  zl::ptx::griddep_enter();
  constexpr int KC = DT / 32, VH = DT / 64, ROW = DT * 2;
  constexpr uint32_t TILE = 16 * ROW;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ Entry entries[kEntries];
  __shared__ float m_sh[kWarps][8], l_sh[kWarps][8];
  __shared__ int list_end;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % cluster;
  const Job w = find_job(g, cluster, rank);
  const uint32_t mine = zl::ptx::smem_u32(ring) + warp * ST * 2 * TILE;

  uint4 q[KC];
#pragma unroll
  for (int k = 0; k < KC; k++) {
    const int e = k * 32 + c * 8;
    q[k] = make_uint4(0, 0, 0, 0);
    if (n < w.heads && e < g.d)
      q[k] = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)g.q + ((int64_t)w.b * g.H + w.head(g, n)) * g.d + e);
  }
  float o[VH][4][4];
#pragma unroll
  for (int a = 0; a < VH; a++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int x = 0; x < 4; x++) o[a][j][x] = 0.f;
  float m = -INFINITY, l = 0.f;
  // this lane's key rows (column n of either tile) and value rows (columns 2 c, 2 c + 1)
  const int krow = n & 1 ? 8 + ((2 * (n >> 1) + 4) & 7) : 2 * (n >> 1);
  const int vrow[2] = {2 * c, 8 + ((2 * c + 4) & 7)};

  for (int e = w.e0; e < w.e1; e += kEntries) {
    if (e > w.e0) __syncthreads();
    const int toks = resolve(g, w, e, min(kEntries, w.e1 - e), entries, &list_end) * g.bs;
    const int tiles = (toks + 15) / 16;
    uint32_t seen[ST];  // which of a tile's 16 tokens there are, by ring slot
    auto fetch = [&](int tile, int slot) {
      return fetch_tile<ROW, 16, true>(g, entries, tile, toks, mine + slot * 2 * TILE, g.d * 2);
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) seen[i] = fetch(warp + i * kWarps, i);
    for (int tile = warp; tile < tiles;) {
#pragma unroll
      for (int slot = 0; slot < ST; slot++, tile += kWarps) {
        if (tile >= tiles) break;
        seen[(slot + ST - 1) % ST] = fetch(tile + (ST - 1) * kWarps, (slot + ST - 1) % ST);
        zl::ptx::copies_wait<ST - 1>();
        __syncwarp();
        const uint32_t ks = mine + slot * 2 * TILE, vs = ks + TILE;
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float s2[4] = {0.f, 0.f, 0.f, 0.f};  // a second chain of products: half the latency
          s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
          const int r = krow + i;
#pragma unroll
          for (int k = 0; k < KC; k++) {
            const uint4 x = zl::ptx::lds16(ks + r * ROW + (((k * 4 + c) ^ (r & 7)) * 16));
            zl::ptx::mma_bf16_16816(s[i], q[k].x, 0, q[k].y, 0, x.x, x.y);
            zl::ptx::mma_bf16_16816(s2, q[k].z, 0, q[k].w, 0, x.z, x.w);
          }
          s[i][0] += s2[0];
          s[i][1] += s2[1];
        }
        // row n of S: head n over this lane's tokens vrow[x] + i
        float best = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            s[i][x] = seen[slot] >> (vrow[x] + i) & 1 ? s[i][x] * g.scale2 : -INFINITY;
            best = fmaxf(best, s[i][x]);
          }
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        if (__any_sync(0xffffffffu, best > m)) {
          const float to = fmaxf(m, best);
          const float a = m == -INFINITY ? 0.f : zl::ptx::ex2(m - to);
          m = to;
          l *= a;
          const float a0 = __shfl_sync(0xffffffffu, a, 8 * c), a1 = __shfl_sync(0xffffffffu, a, 8 * c + 4);
#pragma unroll
          for (int h = 0; h < VH; h++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              o[h][j][0] *= a0;
              o[h][j][1] *= a1;
              o[h][j][2] *= a0;
              o[h][j][3] *= a1;
            }
        }
        const float base = m == -INFINITY ? 0.f : m;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float p0 = zl::ptx::ex2(s[i][0] - base), p1 = zl::ptx::ex2(s[i][1] - base);
          l += p0 + p1;
          // hi: what lies below p, cut to 8 bits; so lo = p - hi > 0 wherever p > 0
          const uint32_t h0 = below(p0) & 0xffff0000u, h1 = below(p1) & 0xffff0000u;
          hi[i] = __byte_perm(h0, h1, 0x7632);
          lo[i] = zl::ptx::pack_bf16x2(p0 - __uint_as_float(h0), p1 - __uint_as_float(h1));
        }
        // O^T: rows n and n + 8 of tile (a, j) are elements 64 a + 8 n + j and + 4
#pragma unroll
        for (int a = 0; a < VH; a++) {
          uint32_t r[4][4];
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
              const int t = vrow[x] + i;
              const uint4 y = zl::ptx::lds16(vs + t * ROW + (((a * 8 + n) ^ (t & 7)) * 16));
              r[2 * i + x][0] = y.x;
              r[2 * i + x][1] = y.y;
              r[2 * i + x][2] = y.z;
              r[2 * i + x][3] = y.w;
            }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
            const uint32_t a0 = __byte_perm(r[0][j / 2], r[1][j / 2], sel), a1 = __byte_perm(r[0][2 + j / 2], r[1][2 + j / 2], sel);
            const uint32_t a2 = __byte_perm(r[2][j / 2], r[3][j / 2], sel), a3 = __byte_perm(r[2][2 + j / 2], r[3][2 + j / 2], sel);
            zl::ptx::mma_bf16_16816(o[a][j], a0, a1, a2, a3, hi[0], hi[1]);
            zl::ptx::mma_bf16_16816(o[a][j], a0, a1, a2, a3, lo[0], lo[1]);
          }
        }
        __syncwarp();  // the next fetch takes this slot
      }
    }
    zl::ptx::copies_wait<0>();
  }
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (c == 0) {
    m_sh[warp][n] = m;
    l_sh[warp][n] = l;
  }
  __syncthreads();  // every warp is done with its ring
  float* o_sh = reinterpret_cast<float*>(ring);
  float* ow = o_sh + warp * 8 * DT;
#pragma unroll
  for (int a = 0; a < VH; a++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int x = 0; x < 4; x++) ow[(2 * c + (x & 1)) * DT + a * 64 + n * 8 + j + 4 * (x >> 1)] = o[a][j][x];
  finish<__nv_bfloat16, 8, DT>(g, w, cluster, rank, o_sh, m_sh, l_sh);
}

// fp32, head_dim up to 32 NV, a multiple of 4; HEADS query heads at a time.
template <int NV, int HEADS, int ST>
__global__ void __launch_bounds__(kThreads) selected_f32_kernel(SelArgs g, int cluster) {
  zl::ptx::griddep_enter();
  constexpr int DT = NV * 32, ROW = DT * 4;
  constexpr uint32_t TILE = 8 * ROW;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ Entry entries[kEntries];
  __shared__ __align__(16) float q_sh[HEADS * DT];
  __shared__ float m_sh[kWarps][HEADS], l_sh[kWarps][HEADS];
  __shared__ int list_end;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tg = lane >> 3, li = lane & 7;
  const int rank = blockIdx.x % cluster;
  const Job w = find_job(g, cluster, rank);
  const uint32_t mine = zl::ptx::smem_u32(ring) + warp * ST * 2 * TILE;
  for (int i = threadIdx.x; i < HEADS * DT; i += kThreads) {
    const int h = i / DT, e = i - h * DT;
    q_sh[i] = h < w.heads && e < g.d ? ((const float*)g.q)[((int64_t)w.b * g.H + w.head(g, h)) * g.d + e] * g.scale2 : 0.f;
  }
  namespace px = zl::ptx;
  uint64_t o[HEADS][NV][2];  // packed pairs: half the instructions of single ones
  float m[HEADS], l[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++) o[h][v][0] = o[h][v][1] = 0;
  }
  const uint32_t qs = px::smem_u32(q_sh) + li * 16;
  for (int e = w.e0; e < w.e1; e += kEntries) {
    if (e > w.e0) __syncthreads();
    const int toks = resolve(g, w, e, min(kEntries, w.e1 - e), entries, &list_end) * g.bs;
    const int tiles = (toks + 7) / 8;
    uint32_t seen[ST];
    auto fetch = [&](int tile, int slot) {
      return fetch_tile<ROW, 8, false>(g, entries, tile, toks, mine + slot * 2 * TILE, g.d * 4);
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) seen[i] = fetch(warp + i * kWarps, i);
    auto work = [&](int slot, uint32_t there) {
      // this lane's elements of rows tg and 4 + tg
      const uint32_t ks = mine + slot * 2 * TILE + tg * ROW + li * 16, vs = ks + TILE;
      uint64_t s2[HEADS][2];
#pragma unroll
      for (int h = 0; h < HEADS; h++) s2[h][0] = s2[h][1] = 0;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const ulonglong2 k0 = px::lds_f2x2(ks + v * 128), k1 = px::lds_f2x2(ks + 4 * ROW + v * 128);
#pragma unroll
        for (int h = 0; h < HEADS; h++) {
          const ulonglong2 x = px::lds_f2x2(qs + (h * DT + v * 32) * 4);
          s2[h][0] = px::f2_fma(x.x, k0.x, px::f2_fma(x.y, k0.y, s2[h][0]));
          s2[h][1] = px::f2_fma(x.x, k1.x, px::f2_fma(x.y, k1.y, s2[h][1]));
        }
      }
      uint64_t a[HEADS], p[HEADS][2];
#pragma unroll
      for (int h = 0; h < HEADS; h++) {
        float s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const float2 both = px::f2_unpack(s2[h][u]);
          s[u] = both.x + both.y;
          s[u] += __shfl_xor_sync(0xffffffffu, s[u], 1);
          s[u] += __shfl_xor_sync(0xffffffffu, s[u], 2);
          s[u] += __shfl_xor_sync(0xffffffffu, s[u], 4);
          if (!(there >> (4 * u + tg) & 1)) s[u] = -INFINITY;
        }
        const float to = fmaxf(m[h], fmaxf(s[0], s[1])), base = to == -INFINITY ? 0.f : to;
        const float f = m[h] == -INFINITY ? 0.f : px::ex2(m[h] - base), p0 = px::ex2(s[0] - base), p1 = px::ex2(s[1] - base);
        m[h] = to;
        l[h] = fmaf(l[h], f, p0 + p1);
        a[h] = px::f2_pack(f, f);
        p[h][0] = px::f2_pack(p0, p0);
        p[h][1] = px::f2_pack(p1, p1);
      }
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const ulonglong2 v0 = px::lds_f2x2(vs + v * 128), v1 = px::lds_f2x2(vs + 4 * ROW + v * 128);
#pragma unroll
        for (int h = 0; h < HEADS; h++) {
          o[h][v][0] = px::f2_fma(o[h][v][0], a[h], px::f2_fma(p[h][0], v0.x, px::f2_mul(p[h][1], v1.x)));
          o[h][v][1] = px::f2_fma(o[h][v][1], a[h], px::f2_fma(p[h][0], v0.y, px::f2_mul(p[h][1], v1.y)));
        }
      }
    };
    if constexpr (HEADS * NV >= 32) {
      // one copy of this long body: unrolled by the ring it does not stay in the instruction cache
      // (48 x 8 lists of 40 blocks, 5 heads each, 84.7 us; so 72.5)
      for (int tile = warp, slot = 0; tile < tiles; tile += kWarps, slot = slot + 1 == ST ? 0 : slot + 1) {
        seen[ST - 1] = fetch(tile + (ST - 1) * kWarps, slot == 0 ? ST - 1 : slot - 1);
        zl::ptx::copies_wait<ST - 1>();
        __syncwarp();
        work(slot, seen[0]);
        __syncwarp();  // the next fetch takes this slot
#pragma unroll
        for (int i = 0; i < ST - 1; i++) seen[i] = seen[i + 1];
      }
    } else {
      for (int tile = warp; tile < tiles;) {
#pragma unroll
        for (int slot = 0; slot < ST; slot++, tile += kWarps) {
          if (tile >= tiles) break;
          seen[(slot + ST - 1) % ST] = fetch(tile + (ST - 1) * kWarps, (slot + ST - 1) % ST);
          zl::ptx::copies_wait<ST - 1>();
          __syncwarp();
          work(slot, seen[slot]);
          __syncwarp();
        }
      }
    }
    zl::ptx::copies_wait<0>();
  }
  __syncthreads();  // every warp is done with its ring
  float* o_sh = reinterpret_cast<float*>(ring);
  // join the warp's four token groups
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    float M = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 8));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
    const float a = l[h] == 0.f ? 0.f : exp2f(m[h] - M);
    float L = l[h] * a;
    L += __shfl_xor_sync(0xffffffffu, L, 8);
    L += __shfl_xor_sync(0xffffffffu, L, 16);
    if (lane == 0) {
      m_sh[warp][h] = M;
      l_sh[warp][h] = L;
    }
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const float2 lo = px::f2_unpack(o[h][v][0]), hi = px::f2_unpack(o[h][v][1]);
      float x[4] = {lo.x * a, lo.y * a, hi.x * a, hi.y * a};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] += __shfl_xor_sync(0xffffffffu, x[i], 8);
        x[i] += __shfl_xor_sync(0xffffffffu, x[i], 16);
      }
      if (tg == 0)
        *reinterpret_cast<float4*>(&o_sh[(warp * HEADS + h) * DT + v * 32 + li * 4]) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  finish<float, HEADS, DT>(g, w, cluster, rank, o_sh, m_sh, l_sh);
}

zl_status launch(zl_ctx* ctx, void (*kernel)(SelArgs, int), size_t smem, const SelArgs& g, int64_t jobs, int cluster,
                 cudaStream_t st) {
  using namespace zl;
  if (smem > 48 * 1024)
    ZL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(jobs * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_ahead
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ZL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, g, cluster));
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

}  // namespace

namespace zl {

// A cluster's CTAs share a GPC, and the GPCs' SMs are no multiple of its size: with one CTA to
// an SM 148 clusters of one, 74 of two, 33 of four, 15 of eight run at once. A size that cannot
// be asked for is taken not to run.
void find_cluster_room(zl_ctx* ctx) {
  for (int two = 0; two < 2; two++) {
    ctx->cluster_room[two][0] = ctx->num_sms << two;
    void (*const kernel)(SelArgs, int) = two ? selected_mma_kernel<128, 3> : selected_mma_kernel<256, 3>;
    const size_t smem = ring_bytes(two ? 256 : 512, 16, 3);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    for (int log = 1; log < 4; log++) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1 << log;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(1 << log);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
      ctx->cluster_room[two][log] = e == cudaSuccess ? clusters << log : 0;
    }
    if (e != cudaSuccess) cudaGetLastError();  // answered: no later call reports it
  }
}

zl_status launch_decode_selected_fast(zl_ctx* ctx, const void* q, const void* k_pool, const void* v_pool,
                                      const int32_t* block_tables, const int32_t* seq_lens,
                                      const int32_t* selected, void* out, int B, int H, int Hkv, int d, int bs,
                                      int max_blocks, int64_t num_blocks, int max_selected, float scale,
                                      zl_gqa_map map, zl_dtype dtype, cudaStream_t st) {
  // 16-byte loads of rows, and row numbers in 32 bits
  const int vec = dtype == ZL_F32 ? 4 : 8;
  if (d % vec || !aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) ||
      (double)num_blocks * Hkv * bs > INT32_MAX || (int64_t)kEntries * bs > 1 << 30)
    return ZL_ERR_UNSUPPORTED;
  const int group = H / Hkv;
  // query heads that share a read of the keys and values (fp32, 5 heads to a key head, 148 lists of
  // 11 blocks: 80 us with up to 8 at a time, 91 with 4 and two reads). More heads than that are two
  // reads or more: bf16, 64 x 8 lists of 128 blocks, 8 heads to a key head 89 us, 9 132, 16 136; fp32
  // heads of 256, 32 blocks each, 4 heads 126, 8 heads 219.
  const int most = dtype == ZL_BF16 || d <= 128 ? 8 : 4;
  const int subs = (group + most - 1) / most, per_sub = (group + subs - 1) / subs;
  SelArgs g{q, k_pool, v_pool, block_tables, seq_lens, selected, out, H, Hkv, d, bs, max_blocks, max_selected,
            num_blocks, scale * 1.4426950408889634f, map == ZL_GQA_MODULO, group, subs, per_sub, ctx->d_status};
  const int64_t jobs = (int64_t)B * Hkv * subs;
  // CTAs per list: as many as one wave of the GPU has room for, while each warp has a tile or
  // two of its own. A CTA costs some 5 us beside its tokens: one sequence (8 lists of 128 blocks)
  // 28.5 / 17.8 / 11.8 / 8.9 us with 1 / 2 / 4 / 8 CTAs to a list, 64 sequences 88 / 103 / 119
  // with 1 / 2 / 4; sizes that are no power of two and 16 gave nothing. One cluster more than
  // run at once costs a second round: 34 lists 19.4 us with 8 CTAs to a list, 14.2 with 4; heads
  // of 256, 16 lists 23.6 and 18.1.
  const int64_t tokens = (int64_t)max_selected * bs;
  const int* room = ctx->cluster_room[d <= 128];  // two CTAs to an SM, or one
  int log_cluster = 0;
  while (2 << log_cluster <= kMaxCluster && jobs << (log_cluster + 1) <= room[log_cluster + 1] &&
         tokens >= 128 << log_cluster)
    log_cluster++;
  const int cluster = 1 << log_cluster;
  if (jobs * cluster > INT32_MAX) return ZL_ERR_UNSUPPORTED;
  // Heads of 65 to 128 elements: two CTAs of three ring slots or three of two to an SM, the
  // same bytes on their way but other rounds. A round that fills the SMs costs its bytes, the
  // last one at least a CTA's own latency, which is that of 1.25 CTAs to an SM (measured with
  // 1 MB lists: 2 x 148 CTAs 48 us, 148 or fewer 30 us). At 384 lists the two give 86 and 76 us,
  // at 512 89 and 98 us.
  auto rounds = [&](int64_t ctas) {
    const int64_t rest = jobs * cluster % ctas, least = ctx->num_sms * 5 / 4;
    return jobs * cluster - rest + (rest == 0 ? 0 : rest > least ? rest : least);
  };
  const bool three = rounds(3 * ctx->num_sms) < rounds(2 * ctx->num_sms);
  auto run = [&](void (*kernel)(SelArgs, int), size_t smem) { return launch(ctx, kernel, smem, g, jobs, cluster, st); };
  if (dtype == ZL_BF16) {
    if (d <= 64) return run(selected_mma_kernel<64, 4>, ring_bytes(128, 16, 4));
    if (d <= 128)
      return three ? run(selected_mma_kernel<128, 2>, ring_bytes(256, 16, 2))
                   : run(selected_mma_kernel<128, 3>, ring_bytes(256, 16, 3));
    return run(selected_mma_kernel<256, 3>, ring_bytes(512, 16, 3));
  }
  // elements / 32, heads at a time, ring slots
  if (d <= 64)
    return per_sub <= 2   ? run(selected_f32_kernel<2, 2, 4>, ring_bytes(256, 8, 4))
           : per_sub <= 4 ? run(selected_f32_kernel<2, 4, 4>, ring_bytes(256, 8, 4))
                          : run(selected_f32_kernel<2, 8, 4>, ring_bytes(256, 8, 4));
  if (d <= 128 && per_sub <= 4)
    return three ? run(per_sub <= 2 ? selected_f32_kernel<4, 2, 2> : selected_f32_kernel<4, 4, 2>, ring_bytes(512, 8, 2))
                 : run(per_sub <= 2 ? selected_f32_kernel<4, 2, 3> : selected_f32_kernel<4, 4, 3>, ring_bytes(512, 8, 3));
  if (d <= 128) return run(selected_f32_kernel<4, 8, 3>, ring_bytes(512, 8, 3));  // its registers allow two to an SM
  return run(per_sub <= 2 ? selected_f32_kernel<8, 2, 3> : selected_f32_kernel<8, 4, 3>, ring_bytes(1024, 8, 3));
}

}  // namespace zl
