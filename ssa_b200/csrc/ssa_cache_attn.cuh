// ssa_cache_attn.cuh -- what the cache attention's kernels share: the counting
// and cutting of the work, row and page conventions, code conversion.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include "ssa_cache.cuh"

namespace ssa {

constexpr int kGroup = 64;       // keys a block takes at a time
constexpr float kEmpty = -1e30f; // offset of a row that has seen no key
constexpr float kHead = 13.f;    // weights run up to 2^13, and 2^15 before the offset moves
constexpr float kSlack = 2.f;
// A page of V that is all zeros has a share in the weights' sum only. Its step
// counts as one, and its scores move the offset only so that its weights stay
// below 2^(13 + 48): at a step of one they would hide pages whose values are
// small (a score 12 octaves up beside an amax of 1e-4 cost 8 % of the output).
// 48 octaves keep the bits of every page with an amax above 2^-57, and the
// weights' sum right for those below 2^60.
constexpr float kZeroHead = 48.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes (biased by 128) in bytes SEL picks -> two fp16: 0x6400 | u is 1024 + u.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, SEL);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Weights: those of a page of zeros may lie beyond fp16's range and become its
// largest number (infinity times a code of 0 would be NaN).
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t v;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Rows of a tile for the kernel that takes many (ssa_cache_prompt.cu). It is
// taken from 64 rows a kv head where rows x keys, by the table's width, come
// to 3 * 2^22, or from 256 rows and 2^23. Measured (us; two kv heads, d 128 / 64):
//   rows  sequences x keys   32-row tiles   128-row tiles
//     64     8 x 8192          30 / 23         29 / 24      2^23
//     64    32 x 8192          63 / 46         58 / 47
//     96     8 x 8192          37 / 28         30 / 25      3 * 2^22
//    128     1 x 16384         27 / 21         28 / 22
//    128     8 x 8192          40 / 31         31 / 25      2^24
//    128    32 x 8192         107 / 77         63 / 50
//    256     1 x 2048          20 / 16         21 / 18
//    256     1 x 16384         36 / 28         33 / 26      2^23
//    512     1 x 2048          24 / 19         22 / 19
//    512    32 x 8192         401 / 279       160 / 124
//   2048     1 x 2048          38 / 30         29 / 25      2^23
//   2048    32 x 8192        1531 / 1064      520 / 407
// Those tables are as wide as the sequences are long; the host knows no lengths,
// so a wider one may bring the 128-row tiles to shorter sequences. Measured at
// the same lengths (us, d 128, table of the length against 64 times it):
//     64    32 x 512  22.5 -> 19.2     64    8 x 1024  15.8 -> 16.6
//     64    32 x 1024 28.2 -> 24.5     64    1 x 2048  12.7 -> 16.4
//    128     8 x 1024 21.9 -> 17.3     64   64 x 128   20.5 -> 24.1
//    256     8 x 512  22.4 -> 18.7    512    2 x 512   15.9 -> 16.6
constexpr int kPromptRows = 128, kPromptMin = 64;
constexpr int64_t prompt_work(int64_t rows) { return rows >= 256 ? 1 << 23 : 3 << 22; }
// Groups of 64 keys that are worth a thread block and its share of the join.
constexpr int least_groups(int rows) { return rows == kPromptRows ? 4 : 1; }

// Blocks that share an SM (registers for 16 and 32 rows, the rings for 8).
constexpr int blocks_per_sm(int d, int rows) { return rows >= 32 ? 2 : rows == 16 || d >= 96 ? 3 : 4; }

// Four elements as they lie in memory: widened where they are used, so that
// a load does not wait where it is issued.
template <bool F32>
struct Raw4 {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const void* row, int i) {
    if constexpr (F32) u = *reinterpret_cast<const uint4*>(static_cast<const float*>(row) + i);
    else {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + i);
      u.x = v.x;
      u.y = v.y;
    }
  }
  __device__ __forceinline__ float4 f() const {
    if constexpr (F32) return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
    else
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
  }
};

// Units and work of the call. Without a list a unit is (sequence, kv head,
// tile of query rows) and its work the sequence's groups of 64 keys; with one
// it is (sequence, token, kv head, tile of heads) and its work the list's.
struct Plan {
  int rows, tiles_max, list_groups;
};

__device__ __forceinline__ int seq_work(const CacheDev& c, const Plan& pl, int b, int rows, int* tiles, int* groups) {
  if (c.blocks) {
    *tiles = c.n * pl.tiles_max;
    *groups = pl.list_groups;
  } else {
    int start, len;
    const int fresh = cache_step_tokens(c, b, start, len);
    *tiles = (fresh * c.rep + rows - 1) / rows;
    *groups = (len + kGroup - 1) / kGroup;
  }
  return *tiles * c.n_kv * *groups;
}

// Equal ranges of the work: block i of `nblk` takes [begin(i), begin(i + 1)),
// one group more in the first `more`. With little work the first blocks get
// `least` groups each, so that no range between two of a unit's is empty.
struct Ranges {
  int nblk, each, more;
  __device__ __forceinline__ Ranges(int total, int grid, int least) {
    nblk = min(grid, (int)((unsigned)total / (unsigned)least));
    if (nblk == 0 && total) nblk = 1;
    each = nblk ? (int)((unsigned)total / (unsigned)nblk) : 0;
    more = total - each * nblk;
  }
  __device__ __forceinline__ int begin(int i) const { return i * each + (i < more ? i : more); }
  __device__ __forceinline__ int of(int x) const {  // the block whose range holds group x
    const int first = more * (each + 1);
    return x < first ? (int)((unsigned)x / (unsigned)(each + 1)) : more + (int)((unsigned)(x - first) / (unsigned)each);
  }
};

// This thread block's range, and the sequence it begins in: up to as many
// sequences as threads take one scan of their work. Block 0 leaves the work
// before each sequence, and all of it, in `prefix`.
struct RangeSmem {
  int sum[32], scan[32], b, base;
};
struct BlockRange {
  int lo, hi, b, base;
  template <class Work>
  __device__ __forceinline__ BlockRange(int B, int32_t* prefix, int least, RangeSmem& s, const Work& work) {
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, threads = blockDim.x, nw = threads >> 5;
    const int mine0 = tid < B ? work(tid) : 0;
    int sum = mine0;
    for (int i = tid + threads; i < B; i += threads) sum += work(i);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) s.sum[w] = sum;
    __syncthreads();
    const int total = __reduce_add_sync(0xffffffffu, lane < nw ? s.sum[lane] : 0);
    const Ranges rg(total, gridDim.x, least);
    lo = rg.begin(min((int)blockIdx.x, rg.nblk));
    hi = (int)blockIdx.x < rg.nblk ? rg.begin(blockIdx.x + 1) : lo;
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += threads) {
      const int mine = b0 == 0 ? mine0 : b0 + tid < B ? work(b0 + tid) : 0;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      if (b0) __syncthreads();
      if (lane == 31) s.scan[w] = upto;
      __syncthreads();
      const int x = lane < nw ? s.scan[lane] : 0;
      const int from = before + upto - mine + __reduce_add_sync(0xffffffffu, lane < w ? x : 0);
      if (lo >= from && lo < from + mine) { s.b = b0 + tid; s.base = from; }
      if (prefix && blockIdx.x == 0 && b0 + tid < B) prefix[b0 + tid] = from;
      before += __reduce_add_sync(0xffffffffu, x);
    }
    if (prefix && blockIdx.x == 0 && tid == 0) prefix[B] = total;
    __syncthreads();
    b = s.b;
    base = s.base;
  }
};

struct Unit {
  int b, kv, tile, start, len, fresh, row0, nrows;  // row0: its first query row, of nrows valid ones
  const int32_t* list;
};

template <int ROWS>
__device__ __forceinline__ Unit unit_of(const CacheDev& c, const Plan& pl, int b, int u, int tiles) {
  Unit x;
  x.b = b;
  x.fresh = cache_step_tokens(c, b, x.start, x.len);
  x.kv = u / tiles;
  x.tile = u - x.kv * tiles;
  x.list = nullptr;
  if (c.blocks) {
    const int tok = x.tile / pl.tiles_max, ht = x.tile - tok * pl.tiles_max;
    x.row0 = tok * c.rep + ht * ROWS;
    x.nrows = tok < x.fresh ? min(ROWS, c.rep - ht * ROWS) : 0;
    x.list = c.blocks + (((int64_t)b * c.n + tok) * c.n_kv + x.kv) * c.top;
  } else {
    x.row0 = x.tile * ROWS;
    x.nrows = min(ROWS, x.fresh * c.rep - x.row0);
  }
  return x;
}

// A unit's final rows (or zeros): row r of the tile is token (row0 + r) / rep
// and the group's head (row0 + r) % rep.
template <bool F32>
__device__ __forceinline__ void store_out(const CacheDev& c, const Unit& x, int r, int ch, float4 o) {
  const int row = x.row0 + r, tok = row / c.rep, h = x.kv * c.rep + row - tok * c.rep;
  const int64_t at = x.b * c.o_sb + h * c.o_sh + tok * c.o_sn + ch;
  if constexpr (F32) *reinterpret_cast<float4*>(static_cast<float*>(c.out) + at) = o;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(c.out) + at) =
        make_uint2(f32_to_bf16_bits(o.x) | (uint32_t)f32_to_bf16_bits(o.y) << 16,
                   f32_to_bf16_bits(o.z) | (uint32_t)f32_to_bf16_bits(o.w) << 16);
}
__device__ __forceinline__ void store_lse(const CacheDev& c, const Unit& x, int r, float m, float l) {
  const int row = x.row0 + r, tok = row / c.rep, h = x.kv * c.rep + row - tok * c.rep;
  c.lse[((int64_t)x.b * c.H + h) * c.n + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

cudaError_t launch_cache_prompt(const CacheDev& c, const Plan& pl, cudaStream_t st);

}  // namespace ssa
