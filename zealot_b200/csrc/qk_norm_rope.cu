// qk_norm_rope.cu -- RMS norm of every query and key head, rotation by the
// token's position and the write of keys and values into the paged pools, in
// one pass over a projection's output.
//
// For a head x of a token at position p, with weight w and frequencies f:
//   y = x / sqrt(mean(x^2) + eps) * w              (without w: y = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = p f_i
// for the pairs i < rotary_dim / 2, which are elements (i, i + rotary_dim / 2)
// or, interleaved, (2i, 2i + 1). Elements from rotary_dim on are not turned.
// Keys go to the slot of kv_cache.rs:245-247 (reshape_and_cache.cu) and, where
// asked for, into packed rows for zl_prefill_varlen; values are copied.
//
// Everything is kept in fp32 and rounded once, at the store. The angle is
// p f_i in 64 bits, and its whole turns are taken off in 64 bits too: at p = 10^6
// the product in fp32 would be off by 0.06 radians.
//
// Measured on one B200 (GPU time, replayed back to back), 32 query and 8 key
// heads of 128, bf16: 64 tokens into the cache 3.1 us, bound by latency; 53,067
// tokens into the cache and packed rows 253-257 us, 1.52 GB at 5.9-6.0 TB/s
// (92 % of the copy rate), bound by HBM with the SMs' issue slots half used.
#include "zl_internal.h"
#include "zl_pages.h"
#include "zl_ptx.cuh"

namespace {

constexpr int kMaxDim = 256;

struct RopeArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const void *q_weight, *k_weight;
  float eps;
  const int32_t* positions;
  const double* inv_freq;
  int rot, interleaved;
  void *q_out, *k_out, *v_out, *k_pool, *v_pool;
  const int64_t* slots;
  int bs;
  int64_t num_blocks, tokens;
  int H, Hkv, d;
  float inv_d;
  int* status;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// cos and sin of position * frequency: the angle in turns, with 1 / (2 pi) in two parts, less
// its whole turns.
__device__ __forceinline__ float2 turn(int32_t pos, double freq) {
  const double a = (double)pos * freq, t = a * 0.15915494309189535;
  const double rest = fma(a, -9.839338337591243e-18, fma(a, 0.15915494309189535, -t));  // what the product lost
  float s, c;
  sincospif((float)(2. * ((t - rint(t)) + rest)), &s, &c);
  return make_float2(c, s);
}

// Row of the pools that token t's kv head h is written to, -1 for none.
__device__ __forceinline__ int64_t cache_row(const RopeArgs& g, int64_t t, int h) {
  if (!g.slots) return -1;
  const int64_t slot = g.slots[t];
  if (slot < 0) return -1;
  const int64_t blk = slot / g.bs;
  if (blk >= g.num_blocks) {
    atomicOr(g.status, ZL_DEV_OOB);
    return -1;
  }
  return zl::pool_row(blk, g.num_blocks, g.Hkv, h, g.bs, (int)(slot - blk * g.bs));
}

// Any head_dim up to 256, any alignment: one warp per (token, head), the row in
// the warp's shared memory so that a pair's elements meet.
template <typename T>
__global__ void __launch_bounds__(256) rope_elem_kernel(RopeArgs g) {
  zl::ptx::griddep_enter();
  __shared__ float rows[8][kMaxDim];
  const int lane = threadIdx.x & 31;
  float* x = rows[threadIdx.x >> 5];
  const int heads = g.H + 2 * g.Hkv;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < g.tokens * heads; u += warps) {
    const int64_t t = u / heads;
    const int h = (int)(u - t * heads);
    const bool isq = h < g.H, isk = !isq && h < g.H + g.Hkv;
    const int hh = isq ? h : isk ? h - g.H : h - g.H - g.Hkv;
    const T* src = (const T*)(isq ? g.q : isk ? g.k : g.v);
    T* out = (T*)(isq ? g.q_out : isk ? g.k_out : g.v_out);
    T* pool = (T*)(isq ? nullptr : isk ? g.k_pool : g.v_pool);
    if (!out && !pool) continue;
    src += t * (isq ? g.q_stride : isk ? g.k_stride : g.v_stride) + (int64_t)hh * g.d;
    float ss = 0.f;
    __syncwarp();
    for (int e = lane; e < g.d; e += 32) {
      const float f = to_f(src[e]);
      x[e] = f;
      ss = fmaf(f, f, ss);
    }
    const T* w = (const T*)(isq ? g.q_weight : isk ? g.k_weight : nullptr);
    if (w) {
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = 1.f / sqrtf(ss / g.d + g.eps);
      for (int e = lane; e < g.d; e += 32) x[e] = x[e] * inv * to_f(w[e]);
    }
    __syncwarp();
    if (isq || isk) {
      for (int i = lane; i < g.rot / 2; i += 32) {
        const float2 cs = turn(g.positions[t], g.inv_freq[i]);
        const int ia = g.interleaved ? 2 * i : i, ib = g.interleaved ? 2 * i + 1 : i + g.rot / 2;
        const float a = x[ia], b = x[ib];
        x[ia] = a * cs.x - b * cs.y;
        x[ib] = b * cs.x + a * cs.y;
      }
    }
    __syncwarp();
    if (out) {
      out += (t * (isq ? g.H : g.Hkv) + hh) * (int64_t)g.d;
      for (int e = lane; e < g.d; e += 32) put(out + e, x[e]);
    }
    if (pool) {
      const int64_t row = cache_row(g, t, hh);
      if (row >= 0)
        for (int e = lane; e < g.d; e += 32) put(pool + row * g.d + e, x[e]);
    }
  }
}

// E elements: 16 bytes, or 8 for four of bf16.
template <int E>
struct Run {
  float x[E];
};
__device__ __forceinline__ Run<4> load_run(const float* p, Run<4>) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  return {{v.x, v.y, v.z, v.w}};
}
__device__ __forceinline__ Run<4> load_run(const __nv_bfloat16* p, Run<4>) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  return {{a.x, a.y, b.x, b.y}};
}
__device__ __forceinline__ Run<8> load_run(const __nv_bfloat16* p, Run<8>) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  Run<8> r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __bfloat1622float2(h[i]);
    r.x[2 * i] = f.x;
    r.x[2 * i + 1] = f.y;
  }
  return r;
}
__device__ __forceinline__ void store_run(float* p, const Run<4>& q) {
  *reinterpret_cast<float4*>(p) = make_float4(q.x[0], q.x[1], q.x[2], q.x[3]);
}
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const Run<4>& q) {
  *reinterpret_cast<uint2*>(p) = make_uint2(zl::ptx::pack_bf16x2(q.x[0], q.x[1]), zl::ptx::pack_bf16x2(q.x[2], q.x[3]));
}
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const Run<8>& q) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(zl::ptx::pack_bf16x2(q.x[0], q.x[1]), zl::ptx::pack_bf16x2(q.x[2], q.x[3]),
                 zl::ptx::pack_bf16x2(q.x[4], q.x[5]), zl::ptx::pack_bf16x2(q.x[6], q.x[7]));
}

// Rotates a lane's two runs by the angles of its E pairs. Two pairs' angles are 16 bytes, and
// those of neighbouring lanes lie side by side: `lanes` such pieces, then the next two pairs'.
template <int E>
__device__ __forceinline__ void rotate(Run<E>& a, Run<E>& b, const float4* cs, int lanes, bool interleaved) {
#pragma unroll
  for (int x = 0; x < E; x += 2) {
    const float4 t = cs[x / 2 * lanes];
    if (interleaved) {  // 2 x, 2 x + 1 and 2 x + 2, 2 x + 3 of the 2 E elements in a row
      Run<E>& q = x < E / 2 ? a : b;
      const int i = 2 * (x % (E / 2));
      const float y0 = q.x[i], z0 = q.x[i + 1], y1 = q.x[i + 2], z1 = q.x[i + 3];
      q.x[i] = y0 * t.x - z0 * t.y;
      q.x[i + 1] = z0 * t.x + y0 * t.y;
      q.x[i + 2] = y1 * t.z - z1 * t.w;
      q.x[i + 3] = z1 * t.z + y1 * t.w;
    } else {
      const float y0 = a.x[x], z0 = b.x[x], y1 = a.x[x + 1], z1 = b.x[x + 1];
      a.x[x] = y0 * t.x - z0 * t.y;
      b.x[x] = z0 * t.x + y0 * t.y;
      a.x[x + 1] = y1 * t.z - z1 * t.w;
      b.x[x + 1] = z1 * t.z + y1 * t.w;
    }
  }
}

// Rows that loads of E elements can read, head_dim and rotary_dim multiples of 2 E. LG lanes
// (a power of two, at least d / (2 E)) share a row; a lane has two runs of E of its elements,
// the pairs E u .. E u + E - 1, whose elements lie in the two halves of the rotated part (or,
// interleaved, side by side), so that a rotation needs no exchange between lanes. A CTA takes
// `per` tokens; their angles, once for all heads, and their cache rows go to shared memory.
// A lane group keeps to one head (of q, then k, then v) over its tokens, then takes the next.
// HeadRows is that head: where its rows come from and go to.
template <typename T>
struct HeadRows {
  const T* src;  // the head's row of the CTA's first token
  T *out, *pool;
  const T* w;
  int64_t stride, out_stride;
  bool use, turn;
  __device__ __forceinline__ HeadRows(const RopeArgs& g, int h, int64_t t0, bool mine, bool turned) {
    const bool isq = h < g.H, isk = !isq && h < g.H + g.Hkv;
    const int hh = isq ? h : isk ? h - g.H : h - g.H - g.Hkv;
    out = (T*)(isq ? g.q_out : isk ? g.k_out : g.v_out);
    pool = (T*)(isq ? nullptr : isk ? g.k_pool : g.v_pool);
    w = (const T*)(isq ? g.q_weight : isk ? g.k_weight : nullptr);
    use = mine && h < g.H + 2 * g.Hkv && (out || pool);
    turn = turned && (isq || isk);
    stride = isq ? g.q_stride : isk ? g.k_stride : g.v_stride;
    out_stride = (int64_t)(isq ? g.H : g.Hkv) * g.d;
    src = (const T*)(isq ? g.q : isk ? g.k : g.v);
    if (use) src += t0 * stride + (int64_t)hh * g.d;
    if (out) out += t0 * out_stride + (int64_t)hh * g.d;
    if (pool) pool += (int64_t)hh * g.bs * g.d;
  }
};

template <int LG, int E>
struct Lane {  // a lane's place in its row
  int u, e0, e1;
  bool mine, turned;
  __device__ __forceinline__ explicit Lane(const RopeArgs& g) {
    u = threadIdx.x % LG;
    mine = u * 2 * E < g.d;
    turned = u * 2 * E < g.rot;
    const bool halves = turned && !g.interleaved;
    e0 = halves ? E * u : 2 * E * u;
    e1 = halves ? g.rot / 2 + E * u : 2 * E * u + E;
  }
};

// Norms and rotates one row and stores it: token c of the CTA, whose angles are cs and
// whose pool rows start at element `at` (-1: none).
template <typename T, int LG, int E>
__device__ __forceinline__ void finish_row(const RopeArgs& g, const Lane<LG, E>& ln, const HeadRows<T>& r, int c,
                                           Run<E> a, Run<E> b, const float2* cs, int64_t at) {
  float ss = 0.f, s2 = 0.f;
#pragma unroll
  for (int x = 0; x < E; x++) {
    ss = fmaf(a.x[x], a.x[x], ss);
    s2 = fmaf(b.x[x], b.x[x], s2);
  }
  ss += s2;
#pragma unroll
  for (int o = LG / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (!r.use) return;
  if (r.w) {
    const Run<E> wa = load_run(r.w + ln.e0, Run<E>{}), wb = load_run(r.w + ln.e1, Run<E>{});
    const float y = ss * g.inv_d + g.eps, q = rsqrtf(y);
    const float inv = q * fmaf(-0.5f * y * q, q, 1.5f);  // a Newton step: right to fp32's last place or so
#pragma unroll
    for (int x = 0; x < E; x++) {
      a.x[x] = a.x[x] * inv * wa.x[x];
      b.x[x] = b.x[x] * inv * wb.x[x];
    }
  }
  if (r.turn) rotate(a, b, reinterpret_cast<const float4*>(cs) + ln.u, g.rot / (2 * E), g.interleaved);
  if (r.out) {
    T* to = r.out + c * r.out_stride;
    store_run(to + ln.e0, a);
    store_run(to + ln.e1, b);
  }
  if (r.pool && at >= 0) {
    store_run(r.pool + at + ln.e0, a);
    store_run(r.pool + at + ln.e1, b);
  }
}

// The CTA's angles, in rotate()'s order, and, in elements, the pool rows of its tokens' kv head 0.
template <int E>
__device__ __forceinline__ void token_tables(const RopeArgs& g, int64_t t0, int tokens, float2* cs, int64_t* cache) {
  const int half = g.rot / 2;
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int t = i / half, p = i - t * half, u = p / E, x = p % E;  // pair x of lane u
    cs[t * half + (x / 2 * (half / E) + u) * 2 + x % 2] = turn(g.positions[t0 + t], g.inv_freq[p]);
  }
  if (threadIdx.x < tokens) {
    const int64_t row = cache_row(g, t0 + threadIdx.x, 0);
    cache[threadIdx.x] = row < 0 ? -1 : row * g.d;
  }
}

// Few tokens: one to a CTA, and its heads over gridDim.y of them.
template <typename T, int LG, int E>
__global__ void __launch_bounds__(256) rope_token_kernel(RopeArgs g) {
  zl::ptx::griddep_enter();
  __shared__ __align__(16) float2 cs[kMaxDim / 2];
  __shared__ int64_t cache[1];
  const Lane<LG, E> ln(g);
  const int64_t t0 = blockIdx.x;
  bool tables = false;
  // every group of a CTA goes through the loop equally often (the barrier inside)
  for (int h0 = blockIdx.y * (256 / LG); h0 < g.H + 2 * g.Hkv; h0 += gridDim.y * (256 / LG)) {
    const HeadRows<T> r(g, h0 + threadIdx.x / LG, t0, ln.mine, ln.turned);
    Run<E> a{}, b{};
    if (r.use) {
      a = load_run(r.src + ln.e0, a);
      b = load_run(r.src + ln.e1, b);
    }
    if (!tables) {  // while the row is on its way
      token_tables<E>(g, t0, 1, cs, cache);
      __syncthreads();
      tables = true;
    }
    finish_row(g, ln, r, 0, a, b, cs, cache[0]);
  }
}

// Many tokens: HBM-bound. Every thread copies its own two runs of the rows that it will need
// kAhead - 1 steps from now into its own slots of shared memory, in the background: bytes on
// their way without registers, and without a barrier, since each thread waits for its own.
// 53,067 tokens as above: loads into registers 649 us (462 with two tokens at a time: too few
// bytes on their way), these copies in runs of 8 bytes 268-284, of 16 bytes 273, and with the
// angles in an order without bank conflicts 254-260.
// The groups are shared out as `hpb` heads by `slices` parts of the tokens.
constexpr int kTokens = 16, kAhead = 4, kFew = 2;
// CTAs to an SM, by registers (80 or 64 a thread): bf16 254 us with 3 and 260 with 4, fp32 (20,000
// tokens of the same heads) 193 and 190.
template <typename T> constexpr int kResident = sizeof(T) == 2 ? 3 : 4;
template <typename T, int LG, int E>
__global__ void __launch_bounds__(256, kResident<T>) rope_tokens_kernel(RopeArgs g, int per, int hpb, int slices) {
  zl::ptx::griddep_enter();
  constexpr int RUN = E * sizeof(T);
  extern __shared__ __align__(16) uint8_t dyn[];  // [kAhead][2][256] runs, then the angles
  __shared__ int64_t cache[kTokens];
  float2* cs = reinterpret_cast<float2*>(dyn + kAhead * 256 * 2 * RUN);
  const Lane<LG, E> ln(g);
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int tokens = (int)min((int64_t)per, g.tokens - t0), half = g.rot / 2, group = threadIdx.x / LG;
  const int slice = group / hpb, heads = slice < slices ? g.H + 2 * g.Hkv : 0;  // a group that is left over: none
  const uint32_t slots = zl::ptx::smem_u32(dyn) + threadIdx.x * RUN;
  int h2 = group - slice * hpb, c2 = slice;  // head and token of the next copy
  if (c2 >= tokens) h2 = heads;
  HeadRows<T> ahead(g, h2, t0, ln.mine, ln.turned), r = ahead;
  int h = h2, c = c2;
  auto fetch = [&](int slot) {
    if (h2 < heads) {
      if (ahead.use) {
        const uint32_t to = slots + slot * 256 * 2 * RUN;
        const T* src = ahead.src + c2 * ahead.stride;
        zl::ptx::copy_async<RUN>(to, src + ln.e0);
        zl::ptx::copy_async<RUN>(to + 256 * RUN, src + ln.e1);
      }
      if ((c2 += slices) >= tokens) {
        c2 = slice;
        h2 += hpb;
        ahead = HeadRows<T>(g, h2, t0, ln.mine, ln.turned);
      }
    }
    zl::ptx::copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kAhead - 1; i++) fetch(i);
  token_tables<E>(g, t0, tokens, cs, cache);
  __syncthreads();
  // a warp's groups take their last steps together: the sum over lanes needs them all
  int s = 0;
  while (__any_sync(0xffffffffu, h < heads)) {
    fetch((s + kAhead - 1) % kAhead);
    zl::ptx::copies_wait<kAhead - 1>();
    const T* slot = reinterpret_cast<const T*>(dyn + (s % kAhead * 2 * 256 + threadIdx.x) * RUN);
    r.use = r.use && h < heads;
    Run<E> a{}, b{};  // zeros in the lanes behind the row's end: they take part in its sum
    if (r.use) {
      a = load_run(slot, a);
      b = load_run(slot + 256 * E, b);
    }
    finish_row(g, ln, r, c, a, b, cs + c * half, r.use ? cache[c] : -1);
    if (h < heads && (c += slices) >= tokens) {
      c = slice;
      h += hpb;
      r = HeadRows<T>(g, h, t0, ln.mine, ln.turned);
    }
    s++;
  }
  zl::ptx::copies_wait<0>();
}

template <typename T, int LG, int E>
zl_status launch_rope_vec(const RopeArgs& g, int num_sms, cudaStream_t st) {
  using namespace zl;
  constexpr int NG = 256 / LG;
  const int heads = g.H + 2 * g.Hkv, blocks = (heads + NG - 1) / NG;
  // CTAs that the GPU has room for at once, and tokens to a CTA that fill whole rounds of them
  const int64_t room = kResident<T> * (int64_t)num_sms, rounds = (g.tokens + room * kTokens - 1) / (room * kTokens);
  const int64_t per = (g.tokens + room * rounds - 1) / (room * rounds);
  if (per < kFew) {  // one token to a CTA: 1,024 tokens 13.2 us this way, 10.9 two to a CTA; 64 tokens 3.1
    launch_ahead(rope_token_kernel<T, LG, E>, dim3((unsigned)g.tokens, blocks < 65535 ? blocks : 65535), 256, 0, st, g);
    return ZL_OK;
  }
  const int hpb = (heads + blocks - 1) / blocks, slices = NG / hpb < per ? NG / hpb : (int)per;
  const size_t smem = (size_t)kAhead * 256 * 2 * E * sizeof(T) + per * (g.rot / 2) * sizeof(float2);
  const auto kernel = rope_tokens_kernel<T, LG, E>;
  ZL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  launch_ahead(kernel, (unsigned)((g.tokens + per - 1) / per), 256, smem, st, g, (int)per, hpb, slices);
  return ZL_OK;
}

template <typename T, int E>
zl_status launch_rope_vec(const RopeArgs& g, int num_sms, cudaStream_t st) {
  const int lanes = g.d / (2 * E);
  return lanes <= 4    ? launch_rope_vec<T, 4, E>(g, num_sms, st)
         : lanes <= 8  ? launch_rope_vec<T, 8, E>(g, num_sms, st)
         : lanes <= 16 ? launch_rope_vec<T, 16, E>(g, num_sms, st)
                       : launch_rope_vec<T, 32, E>(g, num_sms, st);
}

}  // namespace

extern "C" zl_status zl_qk_norm_rope(zl_ctx* ctx, const void* q, const void* k, const void* v, int64_t q_stride,
                                     int64_t k_stride, int64_t v_stride, const void* q_weight, const void* k_weight,
                                     float eps, const int32_t* positions, const double* inv_freq, int rotary_dim,
                                     int interleaved, void* q_out, void* k_out, void* v_out, void* k_pool,
                                     void* v_pool, const int64_t* slot_mapping, int block_size, int64_t num_blocks,
                                     int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim,
                                     zl_dtype dtype, zl_stream stream) {
  using namespace zl;
  if (!dtype_ok(dtype)) return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: bad dtype %d", (int)dtype);
  if (num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0)
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: bad sizes T=%lld H=%d Hkv=%d d=%d", (long long)num_tokens,
                     num_heads, num_kv_heads, head_dim);
  if (head_dim > kMaxDim) return set_error(ZL_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d > %d", head_dim, kMaxDim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: rotary_dim %d of head_dim %d", rotary_dim, head_dim);
  if (!k_pool != !v_pool || (k_pool && (!slot_mapping || block_size <= 0 || num_blocks < 0)))
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: both pools with slots, block_size and num_blocks, or neither");
  if (num_tokens == 0) return ZL_OK;
  const bool need_k = k_out || k_pool, need_v = v_out || v_pool;
  if ((!q_out && !need_k && !need_v) || (q_out && !q) || (need_k && !k) || (need_v && !v) ||
      (rotary_dim && (q_out || need_k) && (!positions || !inv_freq)))
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: null pointer");
  const int64_t nq = (int64_t)num_heads * head_dim, nk = (int64_t)num_kv_heads * head_dim;
  if (num_tokens > 1 && ((q_out && q_stride < nq) || (need_k && k_stride < nk) || (need_v && v_stride < nk)))
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: a token stride is below its row");
  if ((q_out == q && q_stride != nq && num_tokens > 1) || (k_out && k_out == k && k_stride != nk && num_tokens > 1) ||
      (v_out && v_out == v && v_stride != nk && num_tokens > 1))
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: in place only on packed rows");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  RopeArgs g{q, k, v, q_stride, k_stride, v_stride, q_weight, k_weight, eps, positions, inv_freq, rotary_dim,
             interleaved, q_out, k_out, v_out, k_pool, v_pool, k_pool ? slot_mapping : nullptr, block_size,
             num_blocks, num_tokens, num_heads, num_kv_heads, head_dim, 1.f / head_dim, ctx->d_status};
  // rows of runs of `n` elements
  auto runs = [&](int n) {
    const size_t bytes = n * dtype_size(dtype);
    for (const void* p : {q, k, v, q_weight, k_weight, (const void*)q_out, (const void*)k_out, (const void*)v_out,
                          (const void*)k_pool, (const void*)v_pool})
      if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    return head_dim % (2 * n) == 0 && rotary_dim % (2 * n) == 0 &&
           (num_tokens == 1 || (q_stride % n == 0 && k_stride % n == 0 && v_stride % n == 0));
  };
  const bool vec = num_tokens <= INT32_MAX && num_heads + 2 * (int64_t)num_kv_heads <= 1 << 20 && runs(4);
  const cudaStream_t st = S(stream);
  if (vec) {
    const zl_status s = dtype == ZL_F32 ? launch_rope_vec<float, 4>(g, ctx->num_sms, st)
                        : runs(8)       ? launch_rope_vec<__nv_bfloat16, 8>(g, ctx->num_sms, st)
                                        : launch_rope_vec<__nv_bfloat16, 4>(g, ctx->num_sms, st);
    if (s != ZL_OK) return s;
  } else {
    const int64_t units = num_tokens * (num_heads + 2 * (int64_t)num_kv_heads);
    int64_t blocks = (units + 7) / 8;
    if (blocks > (int64_t)ctx->num_sms * 32) blocks = (int64_t)ctx->num_sms * 32;
    if (dtype == ZL_F32) launch_ahead(rope_elem_kernel<float>, (unsigned)blocks, 256, 0, st, g);
    else launch_ahead(rope_elem_kernel<__nv_bfloat16>, (unsigned)blocks, 256, 0, st, g);
  }
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}
