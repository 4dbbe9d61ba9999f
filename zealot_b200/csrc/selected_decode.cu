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
// bf16 (selected_mma_kernel): a warp takes 32 tokens at a time straight from
// global memory into the registers that its matrix instructions read. S = q K^T
// has the (at most 8) query heads as the upper half of M = 16 and 8 tokens as
// N: a lane's 16 bytes of a key row are its B operands for two steps of K = 16
// once q is loaded in the same order, so keys need no shared memory. O^T = V^T P^T
// has 16 elements of a value row as M and the heads as N: a lane loads 16 bytes
// of each of four token rows and pairs two tokens' elements with a byte
// permute. S's accumulators are P^T's operands as they stand. P enters as two
// bf16 parts, p - bf16(p) being the second: the weights then keep 16 bits, for
// one more instruction per tile in a kernel that waits for memory.
//
// fp32 (selected_f32_kernel): eight lanes share a token's row, a warp four
// tokens at a time, on the CUDA cores.
#include <cooperative_groups.h>

#include "zl_internal.h"
#include "zl_pages.h"
#include "zl_ptx.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
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

__device__ __forceinline__ Job find_job(const SelArgs& g, int cluster, int rank) {
  __shared__ int first_neg;
  Job w;
  int u = blockIdx.x / cluster;
  const int sub = u % g.subs;
  u /= g.subs;
  w.b = u / g.Hkv;
  w.kvh = u - w.b * g.Hkv;
  w.head0 = sub * g.per_sub;
  w.heads = min(g.per_sub, g.group - w.head0);
  w.list = g.selected + (int64_t)u * g.max_selected;
  if (threadIdx.x == 0) first_neg = g.max_selected;
  __syncthreads();
  int neg = g.max_selected;
  for (int i = threadIdx.x; i < g.max_selected; i += kThreads)
    if (w.list[i] < 0) {
      neg = i;
      break;
    }
  if (neg < g.max_selected) atomicMin(&first_neg, neg);
  __syncthreads();
  const int n = first_neg, step = (32 + g.bs - 1) / g.bs;  // whole tiles of 32 tokens
  int per = (n + cluster - 1) / cluster;
  per = (per + step - 1) / step * step;
  w.e0 = min(n, rank * per);
  w.e1 = min(n, w.e0 + per);
  return w;
}

// Resolves list entries [e, e + count) into shared memory.
__device__ __forceinline__ void resolve(const SelArgs& g, const Job& w, int e, int count, Entry* sh) {
  const int32_t* table = g.tables + (int64_t)w.b * g.max_blocks;
  const int64_t len = g.seq_lens[w.b];
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int j = w.list[e + i];
    Entry t{0, 0};
    if (j >= g.max_blocks) {
      atomicOr(g.status, ZL_DEV_OOB);
    } else {
      const int64_t left = len - (int64_t)j * g.bs;
      const int32_t id = table[j];
      if (left > 0 && id >= g.num_blocks) atomicOr(g.status, ZL_DEV_OOB);
      const int64_t row = zl::pool_row(id, g.num_blocks, g.Hkv, w.kvh, g.bs, 0);
      if (row >= 0 && left > 0) {
        t.row = (int32_t)row;
        t.tokens = (int32_t)min(left, (int64_t)g.bs);
      }
    }
    sh[i] = t;
  }
}

// Joins the warps' (m, l, o) and then the cluster's, and writes the heads' outputs.
// o: [kWarps][HEADS][DT] unnormalised, in units of 2^m; rows of DT elements, d used.
template <typename T, int HEADS, int DT>
__device__ __forceinline__ void finish(const SelArgs& g, const Job& w, int cluster, int rank, float* o,
                                       float (*m)[HEADS], float (*l)[HEADS]) {
  __shared__ float mc[HEADS], lc[HEADS];
  __syncthreads();
  if (threadIdx.x < HEADS) {
    const int h = threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int i = 0; i < kWarps; i++) M = fmaxf(M, m[i][h]);
    for (int i = 0; i < kWarps; i++)
      if (m[i][h] != -INFINITY || l[i][h] != 0.f) L += l[i][h] * exp2f(m[i][h] - M);
    mc[h] = M;
    lc[h] = L;
  }
  for (int i = threadIdx.x; i < HEADS * DT; i += kThreads) {
    const int h = i / DT;
    float M = -INFINITY, acc = 0.f;
    for (int k = 0; k < kWarps; k++) M = fmaxf(M, m[k][h]);
    for (int k = 0; k < kWarps; k++)
      if (l[k][h] != 0.f) acc += o[k * HEADS * DT + i] * exp2f(m[k][h] - M);
    o[i] = acc;
  }
  T* out = (T*)g.out;
  cg::cluster_group cl = cg::this_cluster();
  if (cluster > 1) cl.sync();
  else __syncthreads();
  for (int i = rank * kThreads + threadIdx.x; i < w.heads * DT; i += cluster * kThreads) {
    const int h = i / DT, e = i - h * DT;
    if (e >= g.d) continue;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int r = 0; r < cluster; r++) M = fmaxf(M, *cl.map_shared_rank(&mc[h], r));
    for (int r = 0; r < cluster; r++) {
      const float lr = *cl.map_shared_rank(&lc[h], r);
      if (lr == 0.f) continue;  // nothing seen there
      const float a = exp2f(*cl.map_shared_rank(&mc[h], r) - M);
      L += lr * a;
      acc += *cl.map_shared_rank(o + i, r) * a;
    }
    const float y = L != 0.f ? acc / L : 0.f;
    T* at = out + ((int64_t)w.b * g.H + w.head(g, h)) * g.d + e;
    if constexpr (sizeof(T) == 2) *at = __float2bfloat16_rn(y);
    else *at = y;
  }
  if (cluster > 1) cl.sync();  // a CTA's shared memory stays until all have read it
}

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// head_dim up to DT, a multiple of 8; NT: 8-token tiles a warp takes at a time.
template <int DT, int NT>
__global__ void __launch_bounds__(kThreads, 2) selected_mma_kernel(SelArgs g, int cluster) {
  constexpr int KC = DT / 32, VH = DT / 64, TOK = NT * 8;
  __shared__ Entry entries[kEntries];
  __shared__ __align__(16) float o_sh[kWarps * 8 * DT];
  __shared__ float m_sh[kWarps][8], l_sh[kWarps][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % cluster;
  const Job w = find_job(g, cluster, rank);
  const __nv_bfloat16* kp = (const __nv_bfloat16*)g.k_pool;
  const __nv_bfloat16* vp = (const __nv_bfloat16*)g.v_pool;

  uint4 q[KC];
#pragma unroll
  for (int k = 0; k < KC; k++) {
    const int e = k * 32 + c * 8;
    q[k] = make_uint4(0, 0, 0, 0);
    if (n < w.heads && e < g.d)
      q[k] = load16((const __nv_bfloat16*)g.q + ((int64_t)w.b * g.H + w.head(g, n)) * g.d + e);
  }
  float o[VH][4][4];
#pragma unroll
  for (int a = 0; a < VH; a++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int x = 0; x < 4; x++) o[a][j][x] = 0.f;
  float m = -INFINITY, l = 0.f;

  for (int e = w.e0; e < w.e1; e += kEntries) {
    const int count = min(kEntries, w.e1 - e);
    if (e > w.e0) __syncthreads();
    resolve(g, w, e, count, entries);
    __syncthreads();
    const int toks = count * g.bs;
    for (int t0 = warp * TOK; t0 < toks; t0 += kWarps * TOK) {
      // lane i resolves token t0 + i (the first TOK lanes)
      int row = -1;
      if (lane < TOK && t0 + lane < toks) {
        const int i = (t0 + lane) / g.bs, t = t0 + lane - i * g.bs;
        const Entry en = entries[i];
        if (t < en.tokens) row = en.row + t;
      }
      uint4 kr[NT][KC], vr[NT][2][VH];
      bool see[NT][2];
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const int r = __shfl_sync(0xffffffffu, row, 8 * i + n);
#pragma unroll
        for (int k = 0; k < KC; k++) {
          kr[i][k] = make_uint4(0, 0, 0, 0);
          if (r >= 0 && k * 32 + c * 8 < g.d) kr[i][k] = load16(kp + (int64_t)r * g.d + k * 32 + c * 8);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const int r = __shfl_sync(0xffffffffu, row, 8 * i + 2 * c + s);
          see[i][s] = r >= 0;
#pragma unroll
          for (int a = 0; a < VH; a++) {
            vr[i][s][a] = make_uint4(0, 0, 0, 0);
            if (r >= 0 && a * 64 + n * 8 < g.d) vr[i][s][a] = load16(vp + (int64_t)r * g.d + a * 64 + n * 8);
          }
        }
      float s[NT][4];
#pragma unroll
      for (int i = 0; i < NT; i++) {
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KC; k++) {
          zl::ptx::mma_bf16_16816(s[i], q[k].x, 0, q[k].y, 0, kr[i][k].x, kr[i][k].y);
          zl::ptx::mma_bf16_16816(s[i], q[k].z, 0, q[k].w, 0, kr[i][k].z, kr[i][k].w);
        }
      }
      // row n of S: head n over this lane's tokens 8 i + 2 c and + 1
      float best = -INFINITY;
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          s[i][x] = see[i][x] ? s[i][x] * g.scale2 : -INFINITY;
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
      uint32_t hi[NT], lo[NT];
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const float p0 = zl::ptx::ex2(s[i][0] - base), p1 = zl::ptx::ex2(s[i][1] - base);
        l += p0 + p1;
        hi[i] = zl::ptx::pack_bf16x2(p0, p1);
        const __nv_bfloat162 hb = *reinterpret_cast<const __nv_bfloat162*>(&hi[i]);
        lo[i] = zl::ptx::pack_bf16x2(p0 - __low2float(hb), p1 - __high2float(hb));
      }
      // O^T: rows n and n + 8 of tile (a, j) are elements 64 a + 8 n + j and + 4
#pragma unroll
      for (int i = 0; i < NT; i += 2)
#pragma unroll
        for (int a = 0; a < VH; a++) {
          const uint32_t* r[4] = {&vr[i][0][a].x, &vr[i][1][a].x, &vr[i + 1][0][a].x, &vr[i + 1][1][a].x};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
            const uint32_t a0 = __byte_perm(r[0][j / 2], r[1][j / 2], sel), a1 = __byte_perm(r[0][2 + j / 2], r[1][2 + j / 2], sel);
            const uint32_t a2 = __byte_perm(r[2][j / 2], r[3][j / 2], sel), a3 = __byte_perm(r[2][2 + j / 2], r[3][2 + j / 2], sel);
            zl::ptx::mma_bf16_16816(o[a][j], a0, a1, a2, a3, hi[i], hi[i + 1]);
            zl::ptx::mma_bf16_16816(o[a][j], a0, a1, a2, a3, lo[i], lo[i + 1]);
          }
        }
    }
  }
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (c == 0) {
    m_sh[warp][n] = m;
    l_sh[warp][n] = l;
  }
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
template <int NV, int HEADS>
__global__ void __launch_bounds__(kThreads, 2) selected_f32_kernel(SelArgs g, int cluster) {
  constexpr int DT = NV * 32;
  __shared__ Entry entries[kEntries];
  __shared__ __align__(16) float o_sh[kWarps * HEADS * DT];
  __shared__ __align__(16) float q_sh[HEADS * DT];
  __shared__ float m_sh[kWarps][HEADS], l_sh[kWarps][HEADS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tg = lane >> 3, li = lane & 7;
  const int rank = blockIdx.x % cluster;
  const Job w = find_job(g, cluster, rank);
  const float* kp = (const float*)g.k_pool;
  const float* vp = (const float*)g.v_pool;
  for (int i = threadIdx.x; i < HEADS * DT; i += kThreads) {
    const int h = i / DT, e = i - h * DT;
    q_sh[i] = h < w.heads && e < g.d ? ((const float*)g.q)[((int64_t)w.b * g.H + w.head(g, h)) * g.d + e] * g.scale2 : 0.f;
  }
  float4 o[HEADS][NV];
  float m[HEADS], l[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++) o[h][v] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int e = w.e0; e < w.e1; e += kEntries) {
    const int count = min(kEntries, w.e1 - e);
    if (e > w.e0) __syncthreads();
    resolve(g, w, e, count, entries);
    __syncthreads();
    const int toks = count * g.bs;
    for (int t0 = warp * 4; t0 < toks; t0 += kWarps * 4) {
      int row = -1;
      if (t0 + tg < toks) {
        const int i = (t0 + tg) / g.bs, t = t0 + tg - i * g.bs;
        const Entry en = entries[i];
        if (t < en.tokens) row = en.row + t;
      }
      float4 kr[NV], vr[NV];
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int x = v * 32 + li * 4;
        kr[v] = vr[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row >= 0 && x < g.d) {
          kr[v] = __ldg(reinterpret_cast<const float4*>(kp + (int64_t)row * g.d + x));
          vr[v] = __ldg(reinterpret_cast<const float4*>(vp + (int64_t)row * g.d + x));
        }
      }
#pragma unroll
      for (int h = 0; h < HEADS; h++) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const float4 qv = *reinterpret_cast<const float4*>(&q_sh[h * DT + v * 32 + li * 4]);
          s = fmaf(qv.x, kr[v].x, fmaf(qv.y, kr[v].y, fmaf(qv.z, kr[v].z, fmaf(qv.w, kr[v].w, s))));
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        if (row < 0) s = -INFINITY;
        const float to = fmaxf(m[h], s), base = to == -INFINITY ? 0.f : to;
        const float a = m[h] == -INFINITY ? 0.f : exp2f(m[h] - base), p = exp2f(s - base);
        m[h] = to;
        l[h] = fmaf(l[h], a, p);
#pragma unroll
        for (int v = 0; v < NV; v++) {
          o[h][v].x = fmaf(o[h][v].x, a, p * vr[v].x);
          o[h][v].y = fmaf(o[h][v].y, a, p * vr[v].y);
          o[h][v].z = fmaf(o[h][v].z, a, p * vr[v].z);
          o[h][v].w = fmaf(o[h][v].w, a, p * vr[v].w);
        }
      }
    }
  }
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
      float x[4] = {o[h][v].x * a, o[h][v].y * a, o[h][v].z * a, o[h][v].w * a};
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

zl_status launch(zl_ctx* ctx, void (*kernel)(SelArgs, int), const SelArgs& g, int64_t jobs, int cluster,
                 cudaStream_t st) {
  using namespace zl;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(jobs * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ZL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, g, cluster));
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}

}  // namespace

namespace zl {

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
  // query heads that share a read of the keys and values
  const int most = dtype == ZL_BF16 ? 8 : d <= 128 ? 4 : 2;
  const int subs = (group + most - 1) / most, per_sub = (group + subs - 1) / subs;
  SelArgs g{q, k_pool, v_pool, block_tables, seq_lens, selected, out, H, Hkv, d, bs, max_blocks, max_selected,
            num_blocks, scale * 1.4426950408889634f, map == ZL_GQA_MODULO, group, subs, per_sub, ctx->d_status};
  const int64_t jobs = (int64_t)B * Hkv * subs;
  // CTAs per list
  const int64_t tokens = (int64_t)max_selected * bs;
  int cluster = 1;
  while (cluster < 8 && jobs * cluster < 4 * ctx->num_sms && tokens / (2 * cluster) >= 128) cluster *= 2;
  if (jobs * cluster > INT32_MAX) return ZL_ERR_UNSUPPORTED;
  void (*kernel)(SelArgs, int);
  if (dtype == ZL_BF16)
    kernel = d <= 64 ? selected_mma_kernel<64, 4> : d <= 128 ? selected_mma_kernel<128, 4> : selected_mma_kernel<256, 2>;
  else
    kernel = d <= 64 ? selected_f32_kernel<2, 4> : d <= 128 ? selected_f32_kernel<4, 4> : selected_f32_kernel<8, 2>;
  return launch(ctx, kernel, g, jobs, cluster, st);
}

}  // namespace zl
