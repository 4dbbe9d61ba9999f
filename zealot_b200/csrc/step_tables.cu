// step_tables.cu -- the metadata of one serving step, built on the device from
// the requests' lengths.
//
// The reference builds it on the host, one sequence at a time
// (src/cuda_runner.rs:446, src/kv_cache.rs:107-161); zl_decode_graph advances
// one token of a fixed set of rows. Here request i adds q_i tokens to c_i
// cached ones. With had = ceil(c/bs) and has = ceil((c+q)/bs) it opens
// has - had new blocks, taken from the list of new block ids in request order:
// two exclusive sums, of q_i (the packed token rows) and of has - had (where a
// request's new ids start), give everything else by indexing.
//
// One launch and no communication between CTAs: every CTA takes both sums over
// all requests itself (a few numbers per thread, from L2), then its share of
// the table entries and of the token rows. No CTA reads what another writes:
// entries below `had` are only read, entries from `had` on are taken from the
// list of new ids.
//
// Measured on one B200 (GPU time, replayed back to back): 64 decode rows with
// tables of 257 blocks 3.6 us, bound by latency (two dependent reads, the sums,
// one more read). 1,024 requests with tables of 8,192 blocks and 65,536 token
// rows 14.8 us: 49.7 MB, 3.4 TB/s, of which 3.9 us are the launch and every CTA's
// own sums. The rest is bound by instructions, not by HBM: 63 % of the issue slots
// are taken, by one CTA of 1,024 threads to an SM, and 12 % of the DRAM's rate. On
// the way there: 4-byte entries 88 us, 16-byte ones 25, 32-bit divisions 20, all of
// a stretch's loads before its first store and larger CTAs 17. Stretches shared out
// by warps instead of CTAs: 15.3; eight loads ahead: 15.5.
#include "zl_internal.h"
#include "zl_pages.h"
#include "zl_ptx.cuh"

namespace {

constexpr int kMaxSeqs = 8192;      // requests of one step: 16 bytes of shared memory each
constexpr int kMaxRows = 1 << 18;   // rows of the persistent table: 2 bits of shared memory each
constexpr int kMostShared = 4 * (4 * kMaxSeqs + 1) + 2 * kMaxRows / 8;

struct StepArgs {
  int32_t* seq_blocks;
  const int32_t* rows;
  const int32_t* context_lens;
  const int32_t* query_lens;
  const int32_t* new_blocks;
  int32_t* block_tables;
  int32_t* cu_seqlens;
  int32_t* seq_lens;
  int32_t* positions;
  int64_t* slot_mapping;
  int32_t* last_rows;
  int64_t num_new, num_tokens, num_blocks;
  int num_rows, num_seqs, max_blocks, bs;
  int* status;
};

// Exclusive sums of a[0..n) and b[0..n) in place, total of a returned in a[n].
template <int kThreads>
__device__ void scan2(int32_t* a, int32_t* b, int n) {
  __shared__ int32_t wa[kThreads / 32], wb[kThreads / 32];
  const int per = (n + kThreads - 1) / kThreads, lo = min(n, (int)threadIdx.x * per), hi = min(n, lo + per);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t sa = 0, sb = 0;
  for (int i = lo; i < hi; i++) {
    sa = zl::sat_add(sa, a[i]);
    sb = zl::sat_add(sb, b[i]);
  }
  int32_t ia = sa, ib = sb;  // inclusive over the warp
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia = zl::sat_add(ia, ua);
      ib = zl::sat_add(ib, ub);
    }
  }
  if (lane == 31) {
    wa[warp] = ia;
    wb[warp] = ib;
  }
  int32_t ea = __shfl_up_sync(0xffffffffu, ia, 1), eb = __shfl_up_sync(0xffffffffu, ib, 1);
  if (lane == 0) ea = eb = 0;
  __syncthreads();
  for (int w = 0; w < warp; w++) {
    ea = zl::sat_add(ea, wa[w]);
    eb = zl::sat_add(eb, wb[w]);
  }
  for (int i = lo; i < hi; i++) {
    const int32_t va = a[i], vb = b[i];
    a[i] = ea;
    b[i] = eb;
    ea = zl::sat_add(ea, va);
    eb = zl::sat_add(eb, vb);
  }
  if (threadIdx.x == kThreads - 1) a[n] = ea;
}

// N table entries, as one load or store.
template <int N>
struct Ids {
  int32_t x[N];
};
template <int N>
__device__ __forceinline__ Ids<N> load_ids(const int32_t* p) {
  Ids<N> r;
  if constexpr (N == 4) {
    const int4 v = *reinterpret_cast<const int4*>(p);
    r.x[0] = v.x;
    r.x[1] = v.y;
    r.x[2] = v.z;
    r.x[3] = v.w;
  } else {
    r.x[0] = *p;
  }
  return r;
}

// Columns [c, c + N) of request i's table row from its old ones `id`: r is its row of
// seq_blocks, `had` and `has` its blocks before and after, `fresh` the place of its first new id.
template <int N>
__device__ __forceinline__ bool table_columns(const StepArgs& g, int i, int c, int r, int had, int has, int fresh,
                                              Ids<N> id) {
  bool bad = false;
  if (c >= has) {
#pragma unroll
    for (int k = 0; k < N; k++) id.x[k] = -1;
  } else if (c + N > had) {  // past the old blocks: new ones, then nothing
#pragma unroll
    for (int k = 0; k < N; k++) {
      if (c + k < had) continue;
      const int64_t at = (int64_t)fresh + c + k - had;
      id.x[k] = c + k < has && at < g.num_new ? g.new_blocks[at] : -1;
      if ((uint32_t)id.x[k] >= (uint32_t)g.num_blocks) id.x[k] = -1;
      if (c + k < has) g.seq_blocks[(int64_t)r * g.max_blocks + c + k] = id.x[k];
    }
  }
  // ids that are no block's become -1: seldom any but those past the end
  bool other = false;
#pragma unroll
  for (int k = 0; k < N; k++) other |= (uint32_t)id.x[k] >= (uint32_t)g.num_blocks;
  if (other && c < has) {
#pragma unroll
    for (int k = 0; k < N; k++)
      if ((uint32_t)id.x[k] >= (uint32_t)g.num_blocks) {
        id.x[k] = -1;
        bad |= c + k < has;
      }
  }
  int32_t* to = g.block_tables + (int64_t)i * g.max_blocks + c;
  if constexpr (N == 4) *reinterpret_cast<int4*>(to) = make_int4(id.x[0], id.x[1], id.x[2], id.x[3]);
  else *to = id.x[0];
  return bad;
}

// A CTA takes units: kThreads / lanes stretches of table rows at a time, `lanes` threads (a
// power of two) to a stretch of lanes * N * kDepth columns, then stretches of kThreads token rows.
constexpr int kDepth = 4;
template <int N, int kThreads>
__global__ void __launch_bounds__(kThreads) step_tables_kernel(StepArgs g, int log_lanes) {
  zl::ptx::griddep_enter();
  extern __shared__ int32_t sh[];
  const int n = g.num_seqs;
  int32_t* cu = sh;                                             // [n + 1] first token row
  int32_t* fresh = cu + n + 1;                                  // [n] first new id
  int32_t* row = fresh + n;                                     // [n] row of seq_blocks, -1: nothing to serve
  int32_t* ctx = row + n;                                       // [n] context length
  uint32_t* once = reinterpret_cast<uint32_t*>(ctx + n);        // rows seen
  const int words = g.rows ? (g.num_rows + 31) / 32 : 0;
  uint32_t* twice = once + words;                               // rows seen again
  bool bad = false;

  for (int w = threadIdx.x; w < 2 * words; w += kThreads) once[w] = 0;
  if (words) __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = g.rows ? g.rows[i] : i;
    const int32_t c = g.context_lens[i];
    const zl::StepRequest q = zl::step_request(c, g.query_lens[i], g.bs, g.max_blocks);
    const bool ok = r >= 0 && r < g.num_rows && q.ok;
    cu[i] = q.tokens;
    fresh[i] = r < 0 ? 0 : q.need;
    row[i] = ok ? r : -1;
    ctx[i] = c;
    bad |= r >= 0 && !ok;
    if (g.rows && ok) {
      const uint32_t bit = 1u << (r & 31);
      if (atomicOr(once + (r >> 5), bit) & bit) atomicOr(twice + (r >> 5), bit);
    }
  }
  __syncthreads();
  scan2<kThreads>(cu, fresh, n);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = row[i];
    // every request of a row that is listed twice, or whose tokens do not fit
    if (r >= 0 && ((g.rows && (twice[r >> 5] >> (r & 31) & 1)) || cu[i + 1] > g.num_tokens)) {
      row[i] = -1;
      bad = true;
    }
  }
  __syncthreads();

  const int32_t cap = (int32_t)(g.num_tokens < 0x7fffffff ? g.num_tokens : 0x7fffffff);
  for (int i = blockIdx.x * kThreads + threadIdx.x; i <= n; i += gridDim.x * kThreads) {
    g.cu_seqlens[i] = min(cu[i], cap);
    if (i < n) {
      g.seq_lens[i] = row[i] < 0 ? 0 : ctx[i] + cu[i + 1] - cu[i];
      g.last_rows[i] = max(min(cu[i + 1], cap) - 1, 0);
    }
  }
  const int lanes = 1 << log_lanes, width = lanes * N * kDepth, stretches = (g.max_blocks + width - 1) / width;
  const int at_once = kThreads >> log_lanes;
  // fewer than 2^32: at most 2^13 requests of 2^18 stretches (a table row of at most 2^30 columns, and all
  // threads to a stretch of such), and fewer than 2^22 stretches of tokens
  const uint32_t pieces = (uint32_t)n * stretches, tables = (pieces + at_once - 1) / at_once;
  const uint32_t units = tables + (uint32_t)((g.num_tokens + kThreads - 1) / kThreads);
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    if (u < tables) {
      const uint32_t piece = u * at_once + (threadIdx.x >> log_lanes);
      if (piece >= pieces) continue;
      const int i = (int)(piece / stretches), c0 = (int)(piece - (uint32_t)i * stretches) * width;
      const int r = row[i];
      int had = 0, has = 0;
      if (r >= 0) {
        had = zl::blocks_of32(ctx[i], g.bs);
        has = zl::blocks_of32(ctx[i] + cu[i + 1] - cu[i], g.bs);
      }
      const int c = c0 + (threadIdx.x & (lanes - 1)) * N, step = lanes * N;
      Ids<N> old[kDepth];  // all loads before the first store
#pragma unroll
      for (int k = 0; k < kDepth; k++)
        if (c + k * step < min(had, g.max_blocks)) old[k] = load_ids<N>(g.seq_blocks + (int64_t)r * g.max_blocks + c + k * step);
#pragma unroll
      for (int k = 0; k < kDepth; k++)
        if (c + k * step < g.max_blocks) bad |= table_columns<N>(g, i, c + k * step, r, had, has, fresh[i], old[k]);
      continue;
    }
    const int64_t t = (int64_t)(u - tables) * kThreads + threadIdx.x;
    if (t >= g.num_tokens) continue;
    int32_t pos = 0;
    int64_t slot = -1;
    if (t < cu[n]) {
      int lo = 0, hi = n;  // the last request that starts at or before t: cu[lo] <= t < cu[lo + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int r = row[lo];
      if (r >= 0) {
        pos = ctx[lo] + (int32_t)(t - cu[lo]);
        const int had = zl::blocks_of32(ctx[lo], g.bs), c = pos / g.bs;
        const int64_t k = (int64_t)fresh[lo] + c - had;
        const int32_t id = c < had ? g.seq_blocks[(int64_t)r * g.max_blocks + c] : k < g.num_new ? g.new_blocks[k] : -1;
        if (id >= 0 && id < g.num_blocks) slot = (int64_t)id * g.bs + pos % g.bs;
        else bad = true;
      }
    }
    g.positions[t] = pos;
    g.slot_mapping[t] = slot;
  }
  if (threadIdx.x == 0 && cu[n] > g.num_tokens) bad = true;
  if (bad) atomicOr(g.status, ZL_DEV_OOB);
}

}  // namespace

extern "C" zl_status zl_step_tables(zl_ctx* ctx, int32_t* seq_blocks, int num_rows, const int32_t* rows,
                                    const int32_t* context_lens, const int32_t* query_lens,
                                    const int32_t* new_blocks, int64_t num_new, int32_t* block_tables,
                                    int32_t* cu_seqlens, int32_t* seq_lens, int32_t* positions,
                                    int64_t* slot_mapping, int32_t* last_rows, int num_seqs, int64_t num_tokens,
                                    int max_blocks_per_seq, int block_size, int64_t num_blocks, zl_stream stream) {
  using namespace zl;
  if (num_seqs < 0 || num_rows < 0 || num_new < 0 || num_tokens < 0 || max_blocks_per_seq < 0 || block_size <= 0 ||
      num_blocks < 0)
    return set_error(ZL_ERR_INVALID_ARG,
                     "step_tables: bad sizes n=%d rows=%d new=%lld T=%lld max_blocks=%d bs=%d blocks=%lld", num_seqs,
                     num_rows, (long long)num_new, (long long)num_tokens, max_blocks_per_seq, block_size,
                     (long long)num_blocks);
  // (2^31 - 1 token rows is what a saturated sum reads as)
  if (num_tokens >= INT32_MAX || num_blocks > INT32_MAX || max_blocks_per_seq > 1 << 30)
    return set_error(ZL_ERR_INVALID_ARG, "step_tables: 2^31-1 token rows, more blocks, or more than 2^30 to a row");
  if (num_seqs > kMaxSeqs || (rows && num_rows > kMaxRows))
    return set_error(ZL_ERR_UNSUPPORTED, "step_tables: at most %d requests (have %d) and %d table rows (have %d)",
                     kMaxSeqs, num_seqs, kMaxRows, num_rows);
  if (!rows && num_rows < num_seqs)
    return set_error(ZL_ERR_INVALID_ARG, "step_tables: %d table rows for %d requests without `rows`", num_rows, num_seqs);
  if (!cu_seqlens || (num_seqs && (!context_lens || !query_lens || !seq_lens || !last_rows)) ||
      (num_seqs && max_blocks_per_seq && (!block_tables || (num_rows && !seq_blocks))) || (num_new && !new_blocks) ||
      (num_tokens && (!positions || !slot_mapping)))
    return set_error(ZL_ERR_INVALID_ARG, "step_tables: null pointer");
  const size_t row_bytes = (size_t)max_blocks_per_seq * 4;
  const auto lo = reinterpret_cast<uintptr_t>(seq_blocks), to = reinterpret_cast<uintptr_t>(block_tables);
  if (row_bytes && num_seqs && num_rows && lo < to + num_seqs * row_bytes && to < lo + num_rows * row_bytes)
    return set_error(ZL_ERR_INVALID_ARG, "step_tables: block_tables overlaps seq_blocks");
  DeviceScope dev(ctx);
  if (dev.status != ZL_OK) return dev.status;
  // Every CTA reads all requests, at no known time beside another's writes: what is written (the
  // first seven) overlaps nothing.
  const struct {
    const void* p;
    size_t bytes;
  } parts[] = {{seq_blocks, num_rows * row_bytes}, {block_tables, num_seqs * row_bytes}, {cu_seqlens, 4 * (size_t)num_seqs + 4},
               {seq_lens, 4 * (size_t)num_seqs}, {last_rows, 4 * (size_t)num_seqs}, {positions, 4 * (size_t)num_tokens},
               {slot_mapping, 8 * (size_t)num_tokens}, {rows, rows ? 4 * (size_t)num_seqs : 0},
               {context_lens, 4 * (size_t)num_seqs}, {query_lens, 4 * (size_t)num_seqs}, {new_blocks, 4 * (size_t)num_new}};
  for (int i = 0; i < 7; i++)
    for (int j = i + 1; j < 11; j++) {
      const auto a = reinterpret_cast<uintptr_t>(parts[i].p), b = reinterpret_cast<uintptr_t>(parts[j].p);
      if (parts[i].bytes && parts[j].bytes && a < b + parts[j].bytes && b < a + parts[i].bytes)
        return set_error(ZL_ERR_INVALID_ARG, "step_tables: an output overlaps another argument");
    }
  StepArgs g{seq_blocks, rows, context_lens, query_lens, new_blocks, block_tables, cu_seqlens, seq_lens, positions,
             slot_mapping, last_rows, num_new, num_tokens, num_blocks, num_rows, num_seqs, max_blocks_per_seq,
             block_size, ctx->d_status};
  const size_t smem = sizeof(int32_t) * (4 * (size_t)num_seqs + 1) + (rows ? 8 * (size_t)((num_rows + 31) / 32) : 0);
  const bool vec = max_blocks_per_seq % 4 == 0 && aligned16(seq_blocks) && aligned16(block_tables);
  // Two CTAs of 512 threads to an SM, or one of 1,024 that takes the sums over many requests once:
  // 64 rows of 257 blocks 3.6 and 4.3 us, 256 rows 5.5 and 4.6, 1,024 rows 7.6 and 5.9, 4,000 rows
  // 23.8 and 11.9.
  const bool many = num_seqs > 512;
  const int kThreads = many ? 1024 : 512;
  const auto kernel = many ? (vec ? step_tables_kernel<4, 1024> : step_tables_kernel<1, 1024>)
                           : (vec ? step_tables_kernel<4, 512> : step_tables_kernel<1, 512>);
  if (smem > 32 * 1024)  // with the static part it may pass 48 KB
    // one limit of the function on the device, for all threads' calls: always the same, the largest
    ZL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
  // Threads to a table row: one step of each while all rows then fit the GPU at once, the shortest
  // way for a small step, kDepth steps otherwise. One and kDepth steps: 64 rows of 256 blocks 3.7 and
  // 4.3 us, of 1,024 3.8 and 4.1; 1,024 rows of 8,192 17.5 and 14.8. Between them either: 256 rows
  // of 256 blocks 4.0 and 4.7, of 257 5.2 and 3.9, 512 rows of 1,024 5.3 and 4.4.
  const int wide = vec ? 4 : 1;
  const int64_t most = (many ? 1 : 2) * ctx->num_sms;
  int log_lanes = 3;
  while (1 << log_lanes < kThreads && (int64_t)wide << log_lanes < max_blocks_per_seq) log_lanes++;
  while (log_lanes > 3 && ((int64_t)num_seqs << log_lanes) > most * kThreads &&
         ((int64_t)wide * kDepth << (log_lanes - 1)) >= max_blocks_per_seq)
    log_lanes--;
  const int64_t width = (int64_t)wide * kDepth << log_lanes, lanes = 1 << log_lanes;
  const int64_t pieces = num_seqs * ((max_blocks_per_seq + width - 1) / width);
  int64_t blocks = (pieces * lanes + kThreads - 1) / kThreads + (num_tokens + kThreads - 1) / kThreads;
  blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
  launch_ahead(kernel, (unsigned)blocks, kThreads, smem, S(stream), g, log_lanes);
  ZL_LAUNCH_CHECK(ctx);
  return ZL_OK;
}
