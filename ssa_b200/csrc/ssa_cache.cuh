// ssa_cache.cuh -- the 8-bit block cache's device parameter block and the
// code paths its kernels share (ssa_cache.cu, ssa_cache_attn.cu).
#pragma once

#include "ssa_common.cuh"
#include "ssa_internal.h"

namespace ssa {

// Tokens of sequence b's current step (q rows / appended tokens that count).
__device__ __forceinline__ int cache_step_tokens(const CacheDev& c, int b, int& start, int& len) {
  start = __ldg(c.start + b);
  len = __ldg(c.lens + b);
  const int64_t cap = (int64_t)c.max_blocks * c.bs;
  if (start < 0 || len < 0) { start = 0; len = 0; }
  if (len > cap) len = (int)cap;
  const int fresh = len - start;
  return fresh < 0 ? 0 : fresh < c.n ? fresh : c.n;
}

// Page of a sequence's logical block, or -1: blocks outside the table and
// page numbers outside the pool are left out instead of being dereferenced.
__device__ __forceinline__ int cache_page(const CacheDev& c, int b, int blk) {
  if (blk < 0 || blk >= c.max_blocks) return -1;
  const int page = __ldg(c.table + (int64_t)b * c.max_blocks + blk);
  return (unsigned)page < (unsigned)c.num_pages ? page : -1;
}

// The code bytes of one key row that lane t (0..3) of a quad holds, as words
// of four channels: with D = 64 a + r, word w of the first 4a covers channels
// (w / 4) * 64 + 16 t + 4 (w % 4) .. + 3 (one 16-byte load for each 64
// channels), the last two (r = 32) channels 64 a + 8 t + 4 (w - 4a) .. + 3.
// The four lanes of a quad read whole 32-byte sectors, and the other operand
// of the product only has to list its channels in the same order.
template <int D>
__device__ __forceinline__ int cache_word_channel(int w, int t) {
  constexpr int kFull = D / 64 * 4;
  return w < kFull ? (w >> 2) * 64 + t * 16 + (w & 3) * 4 : D / 64 * 64 + t * 8 + (w - kFull) * 4;
}

template <int D>
__device__ __forceinline__ void cache_load_row(const int8_t* row, int t, uint32_t (&w)[D / 16]) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + i * 64 + t * 16));
    w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
  }
  if constexpr (D % 64 != 0) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + D / 64 * 64 + t * 8));
    w[D / 16 - 2] = u.x; w[D / 16 - 1] = u.y;
  }
}

}  // namespace ssa
