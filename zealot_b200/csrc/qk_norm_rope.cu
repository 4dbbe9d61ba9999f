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
// heads of 128, bf16: 64 tokens into the cache 3.0 us, bound by latency; 53,067
// tokens into the cache and packed rows 251 us, 1.52 GB at 6.07 TB/s (93 % of
// the copy rate), bound by HBM.
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
// With `copied` x is an element as it was loaded, which keeps its bits: a rounding would make
// every NaN the same one.
__device__ __forceinline__ void put(float* p, float x, bool) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x, bool copied) {
  *p = copied ? __ushort_as_bfloat16((unsigned short)(__float_as_uint(x) >> 16)) : __float2bfloat16_rn(x);
}

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
      for (int e = lane; e < g.d; e += 32) put(out + e, x[e], !isq && !isk);
    }
    if (pool) {
      const int64_t row = cache_row(g, t, hh);
      if (row >= 0)
        for (int e = lane; e < g.d; e += 32) put(pool + row * g.d + e, x[e], !isk);
    }
  }
}

// E elements as packed fp32 pairs (one instruction for two): 16 bytes of a row, or 8 for four
// of bf16.
namespace px = zl::ptx;
template <int E>
struct Run {
  uint64_t p[E / 2];
};
__device__ __forceinline__ uint64_t pair_of(uint32_t w) {  // two bf16
  return px::f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ Run<4> load_run(const float* p, Run<4>) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  return {{v.x, v.y}};
}
__device__ __forceinline__ Run<4> load_run(const __nv_bfloat16* p, Run<4>) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return {{pair_of(v.x), pair_of(v.y)}};
}
__device__ __forceinline__ Run<8> load_run(const __nv_bfloat16* p, Run<8>) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  return {{pair_of(v.x), pair_of(v.y), pair_of(v.z), pair_of(v.w)}};
}
__device__ __forceinline__ uint32_t bf16_pair(uint64_t p) {
  const float2 f = px::f2_unpack(p);
  return px::pack_bf16x2(f.x, f.y);
}
__device__ __forceinline__ void store_run(float* p, const Run<4>& q) {
  *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(q.p[0], q.p[1]);
}
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const Run<4>& q) {
  *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair(q.p[0]), bf16_pair(q.p[1]));
}
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const Run<8>& q) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(q.p[0]), bf16_pair(q.p[1]), bf16_pair(q.p[2]), bf16_pair(q.p[3]));
}

// The bits of bf16 elements as they were loaded.
__device__ __forceinline__ uint32_t bits_of(uint64_t p) {
  const float2 f = px::f2_unpack(p);
  return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
}
__device__ __forceinline__ uint2 bits_of(const Run<4>& q) { return make_uint2(bits_of(q.p[0]), bits_of(q.p[1])); }
__device__ __forceinline__ uint4 bits_of(const Run<8>& q) {
  return make_uint4(bits_of(q.p[0]), bits_of(q.p[1]), bits_of(q.p[2]), bits_of(q.p[3]));
}

// Rotates a lane's two runs by the angles of its E pairs: 16 bytes (c0, c1, s0, s1) for two of
// them, `lanes` such pieces of neighbouring lanes side by side, then the next two pairs'.
template <int E>
__device__ __forceinline__ void rotate(Run<E>& a, Run<E>& b, const ulonglong2* cs, int lanes, bool interleaved) {
  constexpr uint64_t kSigns = 0x8000000080000000ull;
#pragma unroll
  for (int x = 0; x < E / 2; x++) {
    const ulonglong2 t = cs[x * lanes];
    if (interleaved) {  // the two pairs are two whole p's of a run
      uint64_t(&q)[E / 2] = x < E / 4 ? a.p : b.p;
      const int i = 2 * (x % (E / 4));
      const float2 c = px::f2_unpack(t.x), s = px::f2_unpack(t.y), u = px::f2_unpack(q[i]), v = px::f2_unpack(q[i + 1]);
      q[i] = px::f2_pack(u.x * c.x - u.y * s.x, u.y * c.x + u.x * s.x);
      q[i + 1] = px::f2_pack(v.x * c.y - v.y * s.y, v.y * c.y + v.x * s.y);
    } else {
      const uint64_t y = a.p[x], z = b.p[x];
      a.p[x] = px::f2_fma(z, t.y ^ kSigns, px::f2_mul(y, t.x));
      b.p[x] = px::f2_fma(y, t.y, px::f2_mul(z, t.x));
    }
  }
}

// Rows that loads of E elements can read, head_dim and rotary_dim multiples of 2 E. LG lanes
// (a power of two, at least d / (2 E)) share a row; a lane has two runs of E of its elements,
// one in either half of the rotated part: E pairs (or, interleaved, E / 2 whole pairs in each
// run), so that a rotation needs no exchange between lanes. A CTA takes
// `per` tokens; their angles, once for all heads, and their cache rows go to shared memory.
// A lane group keeps to one head (of q, then k, then v) over its tokens, then takes the next.
// HeadRows is that head: where its rows come from and go to.
template <typename T>
struct HeadRows {
  const T* src;  // this lane's first run in the head's row of the CTA's first token; so in out and pool
  T *out, *pool;
  int64_t stride, out_stride;
  bool use, turn, norm, isk;
  template <typename L>
  __device__ __forceinline__ HeadRows(const RopeArgs& g, const L& ln, int h, int64_t t0) {
    const bool isq = h < g.H;
    isk = !isq && h < g.H + g.Hkv;
    const int hh = isq ? h : isk ? h - g.H : h - g.H - g.Hkv;
    out = (T*)(isq ? g.q_out : isk ? g.k_out : g.v_out);
    pool = (T*)(isq ? nullptr : isk ? g.k_pool : g.v_pool);
    norm = isq ? g.q_weight != nullptr : isk && g.k_weight;
    use = ln.mine && h < g.H + 2 * g.Hkv && (out || pool);
    turn = ln.turned && (isq || isk);
    stride = isq ? g.q_stride : isk ? g.k_stride : g.v_stride;
    out_stride = (int64_t)(isq ? g.H : g.Hkv) * g.d;
    src = (const T*)(isq ? g.q : isk ? g.k : g.v);
    if (use) src += t0 * stride + (int64_t)hh * g.d + ln.e0;
    if (out) out += t0 * out_stride + (int64_t)hh * g.d + ln.e0;
    if (pool) pool += (int64_t)hh * g.bs * g.d + ln.e0;
  }
};

template <int LG, int E>
struct Lane {  // a lane's place in its row
  int u, e0, gap;  // its first run's place and how far behind it the second lies
  bool mine, turned;
  __device__ __forceinline__ explicit Lane(const RopeArgs& g, int lane = threadIdx.x % LG) {
    u = lane;
    mine = u * 2 * E < g.d;
    turned = u * 2 * E < g.rot;
    // the two halves of the rotated part, or of the rest: neighbouring lanes' runs lie side by side
    const int from = turned ? 0 : g.rot, len = turned ? g.rot : g.d - g.rot, v = u - from / (2 * E);
    e0 = from + E * v;
    gap = len / 2;
  }
};

// What a CTA's rows share: the weights of q and k in fp32, each lane's in the order of its two
// runs, 16 bytes of neighbouring lanes side by side; its tokens' angles in rotate()'s order; and,
// in elements, the pool rows of its tokens' kv head 0 (-1: none).
template <int LG, int E>
struct Shared {
  float4 weights[2][E / 2][LG];
  ulonglong2* cs;
  int64_t* cache;
};
template <typename T, int LG, int E>
__device__ __forceinline__ void fill_shared(const RopeArgs& g, int64_t t0, int tokens, Shared<LG, E>& sh) {
  const int half = g.rot / 2;
  float* cs = reinterpret_cast<float*>(sh.cs);
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int t = i / half, p = i - t * half;
    // pair x of lane u: its E pairs' elements are in both runs; interleaved, E / 2 pairs in either run
    int u = p / E, x = p % E;
    if (g.interleaved) {
      const int second = p >= half / 2, q = second ? p - half / 2 : p;
      u = q / (E / 2);
      x = q % (E / 2) + (second ? E / 2 : 0);
    }
    const float2 y = turn(g.positions[t0 + t], g.inv_freq[p]);
    float* to = cs + 2 * t * half + (x / 2 * (half / E) + u) * 4 + x % 2;
    to[0] = y.x;
    to[2] = y.y;
  }
  for (int i = threadIdx.x; i < 2 * (E / 2) * LG; i += 256) {
    const int which = i / (E / 2 * LG), j = i / LG % (E / 2);
    const T* w = (const T*)(which ? g.k_weight : g.q_weight);
    const Lane<LG, E> ln(g, i % LG);
    if (w && ln.mine) {
      w += ln.e0 + (j < E / 4 ? 0 : ln.gap - E) + 4 * j;
      sh.weights[which][j][ln.u] = make_float4(to_f(w[0]), to_f(w[1]), to_f(w[2]), to_f(w[3]));
    }
  }
  if (threadIdx.x < tokens) {
    const int64_t row = cache_row(g, t0 + threadIdx.x, 0);
    sh.cache[threadIdx.x] = row < 0 ? -1 : row * g.d;
  }
}

// Norms and rotates one row and stores it to `out` (unless r.out is null) and to the pool row at
// element `at` (unless -1); cs: its token's angles. Returns whether the row is of values with a NaN,
// which the rounding has made another one: copy_row then puts its bits right.
template <typename T, int LG, int E>
__device__ __forceinline__ bool finish_row(const RopeArgs& g, const Lane<LG, E>& ln, const HeadRows<T>& r, Run<E> a,
                                           Run<E> b, const Shared<LG, E>& sh, const ulonglong2* cs, T* out, int64_t at) {
  uint64_t sa = 0, sb = 0;
#pragma unroll
  for (int x = 0; x < E / 2; x++) {
    sa = px::f2_fma(a.p[x], a.p[x], sa);
    sb = px::f2_fma(b.p[x], b.p[x], sb);
  }
  const float2 both = px::f2_unpack(px::f2_add(sa, sb));
  float ss = both.x + both.y;
#pragma unroll
  for (int o = LG / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (!r.use) return false;
  if (r.norm) {
    const float y = ss * g.inv_d + g.eps, q = rsqrtf(y);
    const float step = q * fmaf(-0.5f * y * q, q, 1.5f);  // a Newton step: right to fp32's last place or so
    const float inv = step == step ? step : q;             // a sum past fp32's range, or 0 without eps: 1 / sqrt as it is
    const uint64_t inv2 = px::f2_pack(inv, inv);
    const ulonglong2* w = reinterpret_cast<const ulonglong2*>(&sh.weights[r.isk][0][ln.u]);
#pragma unroll
    for (int j = 0; j < E / 4; j++) {
      const ulonglong2 wa = w[j * LG], wb = w[(E / 4 + j) * LG];
      a.p[2 * j] = px::f2_mul(px::f2_mul(a.p[2 * j], inv2), wa.x);
      a.p[2 * j + 1] = px::f2_mul(px::f2_mul(a.p[2 * j + 1], inv2), wa.y);
      b.p[2 * j] = px::f2_mul(px::f2_mul(b.p[2 * j], inv2), wb.x);
      b.p[2 * j + 1] = px::f2_mul(px::f2_mul(b.p[2 * j + 1], inv2), wb.y);
    }
  }
  if (r.turn) rotate(a, b, cs + ln.u, g.rot / (2 * E), g.interleaved);
  if (r.out) {
    store_run(out, a);
    store_run(out + ln.gap, b);
  }
  if (r.pool && at >= 0) {
    store_run(r.pool + at, a);
    store_run(r.pool + at + ln.gap, b);
  }
  return ss != ss && !r.norm && !r.turn;
}

// Stores a row's two runs with their bits as they are, where finish_row stores them.
template <typename Bits, typename T, int LG, int E>
__device__ __forceinline__ void copy_row(const Lane<LG, E>& ln, const HeadRows<T>& r, Bits a, Bits b, T* out, int64_t at) {
  static_assert(sizeof(Bits) == E * sizeof(T), "a run");
  if (r.out) {
    *reinterpret_cast<Bits*>(out) = a;
    *reinterpret_cast<Bits*>(out + ln.gap) = b;
  }
  if (r.pool && at >= 0) {
    *reinterpret_cast<Bits*>(r.pool + at) = a;
    *reinterpret_cast<Bits*>(r.pool + at + ln.gap) = b;
  }
}

// Few tokens: one to a CTA, and its heads over gridDim.y of them.
template <typename T, int LG, int E>
__global__ void __launch_bounds__(256) rope_token_kernel(RopeArgs g) {
  zl::ptx::griddep_enter();
  __shared__ Shared<LG, E> sh;
  __shared__ ulonglong2 cs[kMaxDim / 4];
  __shared__ int64_t cache[1];
  const Lane<LG, E> ln(g);
  const int64_t t0 = blockIdx.x;
  bool tables = false;
  // every group of a CTA goes through the loop equally often (the barrier inside)
  for (int h0 = blockIdx.y * (256 / LG); h0 < g.H + 2 * g.Hkv; h0 += gridDim.y * (256 / LG)) {
    const HeadRows<T> r(g, ln, h0 + threadIdx.x / LG, t0);
    Run<E> a{}, b{};
    if (r.use) {
      a = load_run(r.src, a);
      b = load_run(r.src + ln.gap, b);
    }
    if (!tables) {  // while the row is on its way
      if (threadIdx.x == 0) {
        sh.cs = cs;
        sh.cache = cache;
      }
      __syncthreads();
      fill_shared<T, LG, E>(g, t0, 1, sh);
      __syncthreads();
      tables = true;
    }
    const bool lost = finish_row(g, ln, r, a, b, sh, cs, r.out, cache[0]);
    if constexpr (sizeof(T) == 2) {
      if (lost) copy_row(ln, r, bits_of(a), bits_of(b), r.out, cache[0]);
    }
  }
}

// Many tokens: HBM-bound. Every thread copies its own two runs of the rows that it will need
// kAhead - 1 steps from now into its own slots of shared memory, in the background: bytes on
// their way without registers, and without a barrier, since each thread waits for its own.
// 53,067 tokens as above: loads into registers 649 us (462 with two tokens at a time: too few
// bytes on their way), these copies in runs of 8 bytes 268-284, of 16 bytes 273, with the
// angles in an order without bank conflicts 254-260, on packed pairs 251. Run for a second the
// board's power limit holds it at 268-272.
// The groups are shared out as `hpb` heads by `slices` parts of the tokens.
constexpr int kTokens = 16, kAhead = 4, kFew = 2;
constexpr int kResident = 4;  // CTAs to an SM: 64 registers a thread; with 3 of 80, 252 us and, at 4,096 tokens, 25.6, not 24.1
template <typename T, int LG, int E>
__global__ void __launch_bounds__(256, kResident) rope_tokens_kernel(RopeArgs g, int per, int hpb, int slices) {
  zl::ptx::griddep_enter();
  constexpr int RUN = E * sizeof(T), SLOT = 256 * 2 * RUN;
  extern __shared__ __align__(16) uint8_t dyn[];  // [kAhead][2][256] runs, then the angles
  __shared__ Shared<LG, E> sh;
  __shared__ int64_t cache[kTokens];
  ulonglong2* cs = reinterpret_cast<ulonglong2*>(dyn + kAhead * SLOT);
  if (threadIdx.x == 0) {
    sh.cs = cs;
    sh.cache = cache;
  }
  const Lane<LG, E> ln(g);
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int tokens = (int)min((int64_t)per, g.tokens - t0), group = threadIdx.x / LG;
  const int slice = group / hpb, heads = slice < slices ? g.H + 2 * g.Hkv : 0;  // a group that is left over: none
  const uint32_t mine = zl::ptx::smem_u32(dyn) + threadIdx.x * RUN;
  int h2 = group - slice * hpb, c2 = slice;  // head and token of the next copy
  if (c2 >= tokens) h2 = heads;
  HeadRows<T> ahead(g, ln, h2, t0), r = ahead;
  int h = h2, c = c2;
  const T* src = ahead.src + c2 * ahead.stride;
  T* out = r.out + c * r.out_stride;
  uint32_t to = mine, from = threadIdx.x * RUN;  // slots of the next copy and of the next step
  auto fetch = [&]() {
    if (h2 < heads) {
      if (ahead.use) {
        zl::ptx::copy_async<RUN>(to, src);
        zl::ptx::copy_async<RUN>(to + 256 * RUN, src + ln.gap);
      }
      src += slices * ahead.stride;
      if ((c2 += slices) >= tokens) {
        c2 = slice;
        h2 += hpb;
        ahead = HeadRows<T>(g, ln, h2, t0);
        src = ahead.src + c2 * ahead.stride;
      }
    }
    to = to == mine + (kAhead - 1) * SLOT ? mine : to + SLOT;
    zl::ptx::copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kAhead - 1; i++) fetch();
  __syncthreads();
  fill_shared<T, LG, E>(g, t0, tokens, sh);
  __syncthreads();
  // a warp's groups take their last steps together: the sum over lanes needs them all
  while (__any_sync(0xffffffffu, h < heads)) {
    fetch();
    zl::ptx::copies_wait<kAhead - 1>();
    r.use = r.use && h < heads;
    Run<E> a{}, b{};  // zeros in the lanes behind the row's end: they take part in its sum
    if (r.use) {
      a = load_run(reinterpret_cast<const T*>(dyn + from), a);
      b = load_run(reinterpret_cast<const T*>(dyn + from + 256 * RUN), b);
    }
    const int64_t at = r.use && r.pool ? cache[c] : -1;
    const bool lost = finish_row(g, ln, r, a, b, sh, cs + c * (g.rot / 4), out, at);
    if constexpr (sizeof(T) == 2) {
      using Bits = decltype(bits_of(a));
      if (lost)
        copy_row(ln, r, *reinterpret_cast<const Bits*>(dyn + from), *reinterpret_cast<const Bits*>(dyn + from + 256 * RUN), out, at);
    }
    from = from == threadIdx.x * RUN + (kAhead - 1) * SLOT ? threadIdx.x * RUN : from + SLOT;
    out += slices * r.out_stride;
    if (h < heads && (c += slices) >= tokens) {
      c = slice;
      h += hpb;
      r = HeadRows<T>(g, ln, h, t0);
      out = r.out + c * r.out_stride;
    }
  }
  zl::ptx::copies_wait<0>();
}

template <typename T, int LG, int E>
zl_status launch_rope_vec(const RopeArgs& g, int num_sms, cudaStream_t st) {
  using namespace zl;
  constexpr int NG = 256 / LG;
  const int heads = g.H + 2 * g.Hkv, blocks = (heads + NG - 1) / NG;
  // CTAs that the GPU has room for at once, and tokens to a CTA that fill whole rounds of them
  const int64_t room = kResident * (int64_t)num_sms, rounds = (g.tokens + room * kTokens - 1) / (room * kTokens);
  const int64_t per = (g.tokens + room * rounds - 1) / (room * rounds);
  if (per < kFew) {  // one token to a CTA: 1,024 tokens 13.2 us this way, 10.9 two to a CTA; 64 tokens 3.1
    launch_ahead(rope_token_kernel<T, LG, E>, dim3((unsigned)g.tokens, blocks < 65535 ? blocks : 65535), 256, 0, st, g);
    return ZL_OK;
  }
  const int hpb = (heads + blocks - 1) / blocks, slices = NG / hpb < per ? NG / hpb : (int)per;
  const size_t smem = (size_t)kAhead * 256 * 2 * E * sizeof(T) + per * (g.rot / 2) * sizeof(float2);
  // the limit is one of the function on the device, for all threads' calls: always the same, the largest
  constexpr int most = kAhead * 256 * 2 * E * (int)sizeof(T) + kTokens * (kMaxDim / 2) * (int)sizeof(float2);
  const auto kernel = rope_tokens_kernel<T, LG, E>;
  ZL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
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
  if ((q_out && q_out == q && q_stride != nq && num_tokens > 1) || (k_out && k_out == k && k_stride != nk && num_tokens > 1) ||
      (v_out && v_out == v && v_stride != nk && num_tokens > 1))
    return set_error(ZL_ERR_INVALID_ARG, "qk_norm_rope: in place only on packed rows");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  if (!q_out && !need_k) rotary_dim = 0;  // values alone: there are no angles, and positions may be missing
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
