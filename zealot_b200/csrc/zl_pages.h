// zl_pages.h -- index arithmetic of the paged cache shared by the kernels of
// the serving-step operators and checked on the host (tests/test_pages_cpu.py
// compiles it with a plain C++ compiler). No CUDA header is needed.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define ZL_HD __host__ __device__ __forceinline__
#else
#define ZL_HD inline
#endif

namespace zl {

// Blocks that `tokens` cached tokens take.
ZL_HD int64_t blocks_of(int64_t tokens, int bs) { return tokens <= 0 ? 0 : (tokens + bs - 1) / bs; }
// The same for a length in [0, 2^31 - 1]: a division in 32 bits.
ZL_HD int32_t blocks_of32(uint32_t tokens, int bs) { return (int32_t)((tokens + (uint32_t)bs - 1) / (uint32_t)bs); }

// Row (of head_dim elements) of token `t` of block `id` and kv head `kvh` in a
// pool [num_blocks][hkv][bs][d]; -1 when the id is outside the pool.
ZL_HD int64_t pool_row(int64_t id, int64_t num_blocks, int hkv, int kvh, int bs, int t) {
  if (id < 0 || id >= num_blocks) return -1;
  return (id * hkv + kvh) * bs + t;
}

// What one request adds to a step, from its lengths alone.
struct StepRequest {
  int32_t tokens;  // rows that it takes in the step's packed token order
  int32_t had;     // blocks that its context fills
  int32_t need;    // new blocks that its tokens open
  bool ok;         // false: the lengths are no lengths, or do not fit its table
};
ZL_HD StepRequest step_request(int64_t context, int64_t query, int bs, int64_t max_blocks) {
  StepRequest r;
  r.ok = context >= 0 && query >= 0 && context + query <= INT32_MAX;
  r.tokens = query > 0 ? (int32_t)query : 0;
  r.had = r.need = 0;
  if (r.ok) {
    const int32_t has = blocks_of32((uint32_t)(context + query), bs);
    r.had = blocks_of32((uint32_t)context, bs);
    r.need = has - r.had;
    r.ok = has <= max_blocks;
  }
  return r;
}

// Sum of two counts in [0, 2^31 - 1] that stays there: a total beyond is cut
// to 2^31 - 1, and sums in any order agree (the scans over requests use it).
ZL_HD int32_t sat_add(int32_t a, int32_t b) {
  const uint32_t s = (uint32_t)a + (uint32_t)b;
  return s > 0x7fffffffu ? 0x7fffffff : (int32_t)s;
}

// Order of scores as unsigned keys: larger scores have larger keys, -0 equals
// +0, and NaN is above everything.
ZL_HD uint32_t score_key(uint32_t bits) {
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (bits == 0x80000000u) bits = 0;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

}  // namespace zl
