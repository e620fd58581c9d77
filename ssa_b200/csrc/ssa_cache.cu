// ssa_cache.cu -- the 8-bit block cache's bookkeeping: pages handed out from
// request lengths, keys and values quantised into pages, and blocks selected
// for each query token by an upper bound of q.k.
//
// A page holds bs tokens of one sequence: int8 codes of keys and values, one
// amax for each (page, kv head, K / V), and -- once the page is complete --
// the least and greatest key code of every channel. A code c stands for
// c * amax / 127, c = rint(127 x / amax) with ties to even, always of the
// token as it came: the open page's tokens stay in `tail` in the model's
// type, and a page whose amax grows is quantised again from there.
#include <math.h>

#include "ssa_cache.cuh"

namespace ssa {

namespace {

// Inclusive scan of v over the block; total in the last return. `part` holds
// one int for each warp.
__device__ __forceinline__ int block_scan(int v, int* part, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) part[w] = v;
  __syncthreads();
  const int x = lane < nw ? part[lane] : 0;
  total = __reduce_add_sync(0xffffffffu, x);
  return v + __reduce_add_sync(0xffffffffu, lane < w ? x : 0);
}

// ---------------------------------------------------------------- reserve
constexpr int kReserveThreads = 1024;
constexpr int kReserveCluster = 8;

// A sequence's pages are taken from the top of the free stack in sequence
// order, so the stack position of every page follows from a prefix sum of the
// needs. A sequence whose pages no longer fit gets none, nor does a later one
// that needs any: those served are a prefix, and the last served sum is what
// the stack loses.
//
// One thread block for one step of up to 1024 sequences; a cluster of eight,
// each with every eighth sequence's table row, where prompts open many pages:
// writing the rows is a chain of load latencies (1024 prompts of up to 128
// pages: 36 us in one block, 6.3 in the cluster; 64 sequences' step 6.3 us,
// which is a launch with its way from Python).
__global__ void __launch_bounds__(kReserveThreads) k_cache_reserve(const ReserveDev r) {
  __shared__ int part[32];
  __shared__ int s_at[kReserveThreads], s_held[kReserveThreads], s_need[kReserveThreads];
  __shared__ int s_given, s_refused;
  const int rank = blockIdx.x, ranks = gridDim.x, threads = blockDim.x;
  const int lane = threadIdx.x & 31;
  grid_wait();
  const int failed = r.state[1];
  const int count = max(0, min(r.state[0], r.num_pages));
  if (threadIdx.x == 0) s_given = s_refused = 0;
  // With several blocks the lengths are written after all of them have read
  // theirs (lens_out may be lens): in a second pass, by the first block.
  for (int pass = 0; pass < (ranks > 1 ? 2 : 1); ++pass) {
    const bool rows = pass == 0, lengths = ranks == 1 || pass == 1;
    if (pass) {
      asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
      if (rank) return;
    }
    int64_t before = 0;
    for (int b0 = 0; b0 < r.B; b0 += threads) {
      const int b = b0 + threadIdx.x;
      int len = 0, more = 0;
      if (b < r.B) {
        len = max(r.lens[b], 0);
        more = max(r.new_lens[b], 0);
      }
      const int64_t after = (int64_t)len + more;
      const int held = (int)(((int64_t)len + r.bs - 1) / r.bs);
      const int64_t want = (after + r.bs - 1) / r.bs;
      const bool wide = want > r.max_blocks;
      const int need = wide ? 0 : (int)(want - held);
      // 1024 needs of 2^21 pages each would pass 32 bits: wider tables add them up in two halves
      int64_t upto, total;
      if (r.max_blocks < (1 << 21)) {
        int sum;
        upto = block_scan(need, part, sum);
        total = sum;
      } else {
        int high, low;
        upto = (int64_t)block_scan(need >> 16, part, high) << 16;
        upto += block_scan(need & 0xffff, part, low);
        total = ((int64_t)high << 16) + low;
      }
      const bool ok = !wide && (need == 0 || before + upto <= count);
      if (lengths) {
        if (b < r.B) {
          r.start_out[b] = len;
          r.lens_out[b] = ok ? (int)after : len;
        }
        const int given = __reduce_max_sync(0xffffffffu, ok && need ? (int)(before + upto) : 0);
        const int refused = __popc(__ballot_sync(0xffffffffu, b < r.B && !ok));
        if (lane == 0 && given) atomicMax(&s_given, given);
        if (lane == 0 && refused) atomicAdd(&s_refused, refused);
      }
      if (rows) {
        s_at[threadIdx.x] = count - 1 - (int)(before + upto - need);
        s_held[threadIdx.x] = held;
        s_need[threadIdx.x] = ok ? need : 0;
        __syncthreads();
        const int many = min(threads, r.B - b0);
        for (int i = (threadIdx.x >> 5) * ranks + rank; i < many; i += (threads >> 5) * ranks) {
          const int m = s_need[i], at = s_at[i];
          int32_t* row = r.table + (int64_t)(b0 + i) * r.max_blocks + s_held[i];
          for (int j = lane; j < m; j += 128) {
            int pg[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pg[e] = j + 32 * e < m ? r.free_pages[at - j - 32 * e] : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j + 32 * e < m) row[j + 32 * e] = pg[e];
          }
        }
      }
      before += total;
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    r.state_out[0] = count - s_given;
    r.state_out[1] = failed + s_refused;
  }
}

// ---------------------------------------------------------------- append
// An amax below this counts as zero: 127 / amax and the logarithm of the
// step stay far inside the fp32 range.
constexpr float kTinyAmax = 0x1p-80f;

// rint(127 x / amax), ties to even, as in exact arithmetic. inv = 127 / amax is
// within 2^-24 of its value and the multiply-adds round once, so x inv is
// within 1e-5 of the quotient; only within that of a half h can the rounding
// be in doubt. Ties are common (a bf16 amax that is a power of two makes every
// eighth code one), so they are decided in fp32 too: by the sign of
// 127 x - h amax, both scaled by 2^-8 -- the product in two parts, the
// multiply-add with one rounding; next to a half the difference has few bits
// left and is exact.
constexpr float kRound = 12582912.f;  // 1.5 2^23: x + kRound is rounded to a whole number, its low byte the code
constexpr float kNearHalf = 0.49998f;

// kRound + the code, where x inv = r + f.
__device__ __forceinline__ float quantize_near_half(float x, float r, float f, float amax) {
  if (!(fabsf(f) > kNearHalf)) return r + kRound;
  const float h = r + copysignf(0.5f, f);
  const float p = x * (127.f / 256.f), p2 = fmaf(x, 127.f / 256.f, -p);
  const float d = fmaf(-h * (1.f / 256.f), amax, p) + p2;
  return (d > 0.f ? h + 0.5f : d < 0.f ? h - 0.5f : h) + kRound;
}

// Four codes of x as bytes; r: the codes as floats, in pairs. inv = 0: all zero.
__device__ __forceinline__ uint32_t quantize4(const float4& x, float inv, float amax, unsigned long long (&r)[2]) {
  const unsigned long long i2 = f2_pack(inv, inv), up = f2_pack(kRound, kRound), down = f2_pack(-kRound, -kRound);
  const unsigned long long neg = 0x8000000080000000ull;
  const unsigned long long x0 = f2_pack(x.x, x.y), x1 = f2_pack(x.z, x.w);
  unsigned long long b0 = f2_fma(x0, i2, up), b1 = f2_fma(x1, i2, up);
  r[0] = f2_add(b0, down);
  r[1] = f2_add(b1, down);
  float fx, fy, fz, fw;
  f2_unpack(f2_fma(x0, i2, r[0] ^ neg), fx, fy);
  f2_unpack(f2_fma(x1, i2, r[1] ^ neg), fz, fw);
  if (fmaxf(fmaxf(fabsf(fx), fabsf(fy)), fmaxf(fabsf(fz), fabsf(fw))) > kNearHalf) {
    float rx, ry, rz, rw;
    f2_unpack(r[0], rx, ry);
    f2_unpack(r[1], rz, rw);
    b0 = f2_pack(quantize_near_half(x.x, rx, fx, amax), quantize_near_half(x.y, ry, fy, amax));
    b1 = f2_pack(quantize_near_half(x.z, rz, fz, amax), quantize_near_half(x.w, rw, fw, amax));
    r[0] = f2_add(b0, down);
    r[1] = f2_add(b1, down);
  }
  float bx, by, bz, bw;
  f2_unpack(b0, bx, by);
  f2_unpack(b1, bz, bw);
  const uint32_t lo = __byte_perm(__float_as_uint(bx), __float_as_uint(by), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(bz), __float_as_uint(bw), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// What the codes stand for.
__device__ __forceinline__ float4 scaled(const unsigned long long (&r)[2], float step) {
  const unsigned long long s2 = f2_pack(step, step);
  float4 v;
  f2_unpack(f2_mul(r[0], s2), v.x, v.y);
  f2_unpack(f2_mul(r[1], s2), v.z, v.w);
  return v;
}

// Four consecutive elements as they lie in memory, and packed minima and
// maxima of them (NaN stays).
template <int DT>
struct Vec4;
template <>
struct Vec4<kDtF32> {
  float4 v;
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const void* p) { v = *static_cast<const float4*>(p); }
  __device__ __forceinline__ void store(void* p) const { *static_cast<float4*>(p) = v; }
  __device__ __forceinline__ float4 f() const { return v; }
  static __device__ __forceinline__ float mn(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
  static __device__ __forceinline__ float mx(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
  __device__ __forceinline__ void min_with(const Vec4& o) { v = make_float4(mn(v.x, o.v.x), mn(v.y, o.v.y), mn(v.z, o.v.z), mn(v.w, o.v.w)); }
  __device__ __forceinline__ void max_with(const Vec4& o) { v = make_float4(mx(v.x, o.v.x), mx(v.y, o.v.y), mx(v.z, o.v.z), mx(v.w, o.v.w)); }
  __device__ __forceinline__ void from(const float4& x) { v = x; }
};
template <>
struct Vec4<kDtBF16> {
  uint2 v;
  __device__ __forceinline__ void zero() { v = make_uint2(0u, 0u); }
  __device__ __forceinline__ void load(const void* p) { v = *static_cast<const uint2*>(p); }
  __device__ __forceinline__ void store(void* p) const { *static_cast<uint2*>(p) = v; }
  __device__ __forceinline__ float4 f() const {
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                       __uint_as_float(v.y & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t mn(uint32_t a, uint32_t b) { uint32_t r; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  static __device__ __forceinline__ uint32_t mx(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  __device__ __forceinline__ void min_with(const Vec4& o) { v = make_uint2(mn(v.x, o.v.x), mn(v.y, o.v.y)); }
  __device__ __forceinline__ void max_with(const Vec4& o) { v = make_uint2(mx(v.x, o.v.x), mx(v.y, o.v.y)); }
  __device__ __forceinline__ void from(const float4& x) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.x) : "f"(x.y), "f"(x.x));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.y) : "f"(x.w), "f"(x.z));
  }
};

// |x| as an integer orders like |x|, with infinities and NaN above.
__device__ __forceinline__ uint32_t abs_top(const float4& x) {
  return max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
             max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
}

// Threads of a block: at most 8 vectors of four elements each, and a whole
// number of token rows, so that a thread stays on its four channels.
template <int D, int BS>
constexpr int kAppendThreads = BS * D / 16 < (D == 96 ? 192 : 256) ? BS * D / 16 : (D == 96 ? 192 : 256);

// One block of a sequence, one kv head, K or V: read the block's tokens (old
// ones from the tail, new ones from the step's input), their least and
// greatest values -- which give the amax and, rounding being monotone, the
// bounds -- then the codes. The tokens stay in registers as they came.
//
// Bound by HBM and, nearly as much, by the arithmetic of the codes (a multiply
// and two additions each, packed in pairs): 16 prompts of up to 8192 tokens, 8
// heads of 128 channels, read 388 MB and write 582 MB in 209 to 216 us, 4.5 TB/s
// of a copy's 6.55 at 57 % of the issue slots. More than half of it is writes,
// and writes alone (a fill of 563 MB) run at 3.85 TB/s. Without the values, as
// the models call it, it reads 388 MB and writes 194 in 165 us. Resident thread blocks that send
// for the next block's rows while they write this one were slower (235 us).
template <int DT, int D, int BS>
__device__ __forceinline__ void append_block(const CacheDev& c, int b, int kv, int s, int blk, int start, int len,
                                             float4* red) {
  using V = Vec4<DT>;
  constexpr int kT = kAppendThreads<D, BS>;
  constexpr int kVec = D / 4, kRg = kT / kVec, kPasses = BS / kRg;
  constexpr int kSize = DT == kDtF32 ? 4 : 2;
  const int tid = threadIdx.x, cv = tid % kVec, r0 = tid / kVec;
  const int p0 = blk * BS;
  // a block of padding, or of a sequence without new tokens, is only cleared in the values
  const int page = p0 < len && start < len ? cache_page(c, b, blk) : -1;
  // rows of the block: [0, old) from the tail, [old, end) from the input, the rest absent
  const int old = page < 0 ? 0 : max(0, min(BS, start - p0)), end = page < 0 ? 0 : min(BS, len - p0);
  char* values = static_cast<char*>(s ? c.v_values : c.k_values);
  if (values) values += (b * c.o_sb + kv * c.o_sh + (int64_t)(p0 - start) * c.o_sn + cv * 4) * kSize;
  if (end == 0) {
    if (values) {
      V o;
      o.zero();
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int row = p * kRg + r0;
        if (p0 + row >= start && p0 + row - start < c.n) o.store(values + row * c.o_sn * kSize);
      }
    }
    return;
  }
  const int64_t sn = s ? c.v_sn : c.k_sn;
  const char* in = static_cast<const char*>(s ? c.v : c.k) +
                   ((s ? b * c.v_sb + kv * c.v_sh : b * c.k_sb + kv * c.k_sh) + (int64_t)(p0 - start) * sn + cv * 4) * kSize;
  char* tail = static_cast<char*>(c.tail) + (((((int64_t)b * c.n_kv + kv) * 2 + s) * BS) * D + cv * 4) * kSize;
  const bool whole = old == 0 && end == BS;  // a complete block of new tokens: no row to leave out
  V x[kPasses];
  if (whole) {
    const char* row = in + r0 * sn * kSize;
    const int64_t stride = kRg * sn * kSize;
#pragma unroll
    for (int p = 0; p < kPasses; ++p, row += stride) x[p].load(row);
  } else {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kRg + r0;
      x[p].zero();
      if (row >= old && row < end) x[p].load(in + row * sn * kSize);
      if (row < old) x[p].load(tail + (int64_t)row * D * kSize);
    }
  }
  // Absent rows are zero: the amax does not see them, and bounds are of whole blocks.
  V lo = x[0], hi = x[0];
#pragma unroll
  for (int p = 1; p < kPasses; ++p) {
    lo.min_with(x[p]);
    hi.max_with(x[p]);
  }
  uint32_t top = max(abs_top(lo.f()), abs_top(hi.f()));
  top = __reduce_max_sync(0xffffffffu, top);
  uint32_t* rt = reinterpret_cast<uint32_t*>(red);
  if ((tid & 31) == 0) rt[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kT / 32; ++i) top = max(top, rt[i]);
  float amax = __uint_as_float(top);
  if (amax < kTinyAmax) amax = 0.f;
  const bool finite = amax > 0.f && amax < INFINITY;
  const float inv = finite ? __fdiv_rn(127.f, amax) : 0.f;
  const float step = __fdiv_rn(amax, 127.f);
  if (tid == 0) c.amax[((int64_t)page * c.n_kv + kv) * 2 + s] = amax;
  if (!finite) {  // no codes: zeros, which stand for 0 or for NaN
#pragma unroll
    for (int p = 0; p < kPasses; ++p) x[p].zero();
    lo.zero();
    hi.zero();
    // 0 * step is the value of every code: 0, or NaN of an amax that is infinite or NaN
  }
  int8_t* codes = (s ? c.v_codes : c.k_codes) + ((int64_t)page * c.n_kv + kv) * BS * D + cv * 4;
  const bool open = p0 + BS > len;
  if (whole) {
    if (values) {
      values += r0 * c.o_sn * kSize;
      const int64_t stride = kRg * c.o_sn * kSize;
#pragma unroll
      for (int p = 0; p < kPasses; ++p, values += stride) {
        unsigned long long r[2];
        *reinterpret_cast<uint32_t*>(codes + (p * kRg + r0) * D) = quantize4(x[p].f(), inv, amax, r);
        V o;
        o.from(scaled(r, step));
        o.store(values);
      }
    } else {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        unsigned long long r[2];
        *reinterpret_cast<uint32_t*>(codes + (p * kRg + r0) * D) = quantize4(x[p].f(), inv, amax, r);
      }
    }
  } else {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kRg + r0;
      const bool have = row < end;
      unsigned long long r[2];
      const uint32_t q = quantize4(x[p].f(), inv, amax, r);
      if (have) *reinterpret_cast<uint32_t*>(codes + row * D) = q;
      if (values && p0 + row >= start && p0 + row - start < c.n) {
        V o;
        o.zero();
        if (have) o.from(scaled(r, step));
        o.store(values + row * c.o_sn * kSize);
      }
    }
  }
  if (open) {  // the open block's new tokens, as they came (zeroed above where there are no codes: read again)
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kRg + r0;
      if (row >= old && row < end) {
        if (!finite) x[p].load(in + row * sn * kSize);
        x[p].store(tail + (int64_t)row * D * kSize);
      }
    }
  }
  __syncthreads();  // red is free again
  if (!open && s == 0) {
    V* rl = reinterpret_cast<V*>(red);
    rl[tid] = lo;
    rl[kT + tid] = hi;
    __syncthreads();
    if (tid < kVec) {
      for (int i = 1; i < kRg; ++i) {
        lo.min_with(rl[i * kVec + tid]);
        hi.max_with(rl[kT + i * kVec + tid]);
      }
      unsigned long long r[2];
      uint32_t* bd = reinterpret_cast<uint32_t*>(c.bounds + ((int64_t)page * c.n_kv + kv) * 2 * D) + tid;
      bd[0] = quantize4(lo.f(), inv, amax, r);
      bd[D / 4] = quantize4(hi.f(), inv, amax, r);
    }
    __syncthreads();
  }
}

// Block j of the touched ones, K or V of one kv head. The first block reads
// the tail and the last one may write it, so one thread block does both, in
// that order. Heads run fastest: thread blocks that run together then read
// whole rows of (B, N, heads, d) tensors (1023 fp32 tokens of two sequences,
// 8 heads of 64: 5.7 us; with the blocks of a head fastest 6.7).
template <int DT, int D, int BS>
__global__ void __launch_bounds__(kAppendThreads<D, BS>, DT == kDtF32 ? 2 : 4) k_cache_append(const CacheDev c, const int nt) {
  __shared__ float4 red[(DT == kDtF32 ? 2 : 1) * kAppendThreads<D, BS>];
  unsigned i = blockIdx.x;
  const int kv = (int)(i % (unsigned)c.n_kv);
  i /= (unsigned)c.n_kv;
  const int s = (int)(i & 1);
  i >>= 1;
  const int j = (int)(i % (unsigned)nt), b = (int)(i / (unsigned)nt);
  grid_wait();
  int start, len;
  const int fresh = cache_step_tokens(c, b, start, len);
  len = start + fresh;
  const int first = start / BS, last = fresh ? (len - 1) / BS : first - 1;
  const bool pad = (s ? c.v_values : c.k_values) != nullptr;
  if (j > 0 && first + j == last) return;
  if (first + j <= last || pad) append_block<DT, D, BS>(c, b, kv, s, first + j, start, len, red);
  if (j == 0 && last > first) append_block<DT, D, BS>(c, b, kv, s, last, start, len, red);
}

template <int DT, int D, int BS>
cudaError_t run_append(const CacheDev& c, cudaStream_t st) {
  const int nt = (c.n + BS - 2) / BS + 1;
  const int64_t grid = (int64_t)c.B * c.n_kv * 2 * nt;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  CacheLaunch l((unsigned)grid, kAppendThreads<D, BS>, 0, st);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, k_cache_append<DT, D, BS>, c, nt);
  note_launch();
  return e;
}

template <int DT, int D>
cudaError_t run_append_bs(const CacheDev& c, cudaStream_t st) {
  return c.bs == 16 ? run_append<DT, D, 16>(c, st) : c.bs == 32 ? run_append<DT, D, 32>(c, st) : run_append<DT, D, 64>(c, st);
}

template <int DT>
cudaError_t run_append_d(const CacheDev& c, cudaStream_t st) {
  return c.d == 32 ? run_append_bs<DT, 32>(c, st) : c.d == 64 ? run_append_bs<DT, 64>(c, st)
         : c.d == 96 ? run_append_bs<DT, 96>(c, st) : run_append_bs<DT, 128>(c, st);
}

// ---------------------------------------------------------------- select
constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr int kSelStages = 3;  // 16 blocks' bounds each, for every warp

// Shared memory of k_cache_select: rings, what comes with a stage, the query
// operand, keys.
template <int D>
struct SelSmem {
  static constexpr int kTile = 16 * kPitch<D>, kRing = kSelStages * 2 * kTile;
  static constexpr int kMeta = kSelWarps * kRing;                  // [kSelWarps][kSelStages]: [16] amax, [16] page
  static constexpr int kQ = kMeta + kSelWarps * kSelStages * 128;  // [tiles of 8 heads][2][D / 16][32] words of q-, q+
  static size_t bytes(const CacheDev& c) {
    return kQ + (size_t)((c.rep + 7) / 8) * 2 * (D / 16) * 32 * 4 + (size_t)c.max_blocks * 8;
  }
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Ordered like the double, above 0 and below ~0 - 1. A NaN (of a block that
// stands for NaN) comes before every number, whatever its bits.
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);  // -0 -> 0
  return v != v ? ~0ull - 2 : (u >> 63) ? ~u : u | (1ull << 63);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// The first block of the cluster's copy of a shared variable.
template <typename T>
__device__ __forceinline__ uint32_t at_rank0(const T* p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
  return a;
}

// One cluster of thread blocks per (sequence, token, kv head). The bound of a
// block is sum_c max(q lo_c, q hi_c) = q- . lo + q+ . hi (q-, q+ the negative
// and positive parts): a product of 8-bit rows of length 2 d, exact in the
// tensor cores' 32-bit sums; times amax it is exact in 64 bits, so the order
// of two blocks never depends on how the sum was formed. The cluster's blocks
// score equal parts into the first one's shared memory, which then narrows
// the range of keys in which the last listed one lies, 256 bins at a time.
//
// Bound by latency: one token's 8 heads over 8192 keys take 5.6 us, a launch.
// 32 sequences of up to 32768 keys (blocks of 32, 52 MB of bounds) take 19.4 us
// with one block of 256 threads a head, 2.7 TB/s: the query's two rounds of
// loads, the ring's start and the narrowing together are as long as the
// reading, and ragged lengths leave SMs idle at the end. Straight from global
// memory to registers it was 31 us, as two kernels 34.
template <int DT, int D>
__global__ void __launch_bounds__(kSelThreads, 2) k_cache_select(const CacheDev c) {
  using Sm = SelSmem<D>;
  extern __shared__ __align__(128) unsigned char sm[];
  const int nht = (c.rep + 7) / 8;  // tiles of 8 heads
  uint32_t* qf = reinterpret_cast<uint32_t*>(sm + Sm::kQ);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(qf + nht * 2 * (D / 16) * 32);
  __shared__ uint32_t red[32];
  __shared__ int hist[256];
  __shared__ int part[32];
  __shared__ unsigned long long s_lo[64], s_hi[64];  // for each warp of the cluster: range of the keys not forced
  __shared__ int s_forced[64], s_bin, s_above, s_cnt, s_n;
  __shared__ int s_idx[kSelThreads];
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, t = lane & 3;
  const unsigned unit = blockIdx.x / ranks;
  unsigned u = unit;
  const int kv = (int)(u % (unsigned)c.n_kv);
  u /= (unsigned)c.n_kv;
  const int tok = (int)(u % (unsigned)c.n), b = (int)(u / (unsigned)c.n);
  int32_t* out = c.blocks_out + (int64_t)unit * c.top;
  grid_wait();
  int start, len;
  const int fresh = cache_step_tokens(c, b, start, len);
  const int here = tok < fresh ? (start + tok) / c.bs + 1 : 0;       // blocks that stand for election
  const bool few = here <= c.top;

  if (few) {
    if (rank) return;
    for (int i = tid; i < here; i += kSelThreads) keys[i] = cache_page(c, b, i) < 0 ? 0ull : ~0ull;
    __syncthreads();
  } else {
    if (ranks > 1) cluster_arrive();  // waited for before the first block's memory is written
    if (tid == 0) s_n = 0;

    // q's amax: its first elements ahead of the bounds in the memory's queue
    const int64_t q0 = b * c.q_sb + (int64_t)kv * c.rep * c.q_sh + (int64_t)tok * c.q_sn;
    Vec4<DT> qv;
    qv.zero();
    if (tid < c.rep * (D / 4)) qv.load(row_ptr<DT>(c.q, q0 + (int64_t)(tid / (D / 4)) * c.q_sh + tid % (D / 4) * 4));

    // Tile i (blocks 16 i .. 16 i + 15) is warp i mod nw's. Lanes 0-15 hold the
    // pages of its next tile, lanes 16-31 those of the one after; the table's
    // entries of the two behind them are on their way.
    const int nw = (int)ranks * kSelWarps, tiles = (here + 15) / 16;
    const uint32_t ring_a = smem_addr(sm) + w * Sm::kRing;
    unsigned char* meta = sm + Sm::kMeta + w * kSelStages * 128 + (lane & 15) * 4;
    const auto look_up = [&](int tile) {
      const int e = (tile + (lane >> 4) * nw) * 16 + (lane & 15);
      return e < here ? cache_entry(c, b, e) : -1;
    };
    const int first = (int)rank * kSelWarps + w;
    int pages = look_up(first), entries = look_up(first + 2 * nw);
    pages = cache_checked(c, pages);
    // 16 rows of 2 D / 16 chunks, a row's chunks side by side: copy i of a lane
    // is chunk (32 i + lane) mod (D / 8) of row (32 i + lane) / (D / 8)
    const int8_t* kv_bounds = c.bounds + (int64_t)kv * 2 * D;
    const unsigned page_bytes = (unsigned)c.n_kv * 2 * D;
    int sent = 0, sent_stage = 0;
    const auto issue = [&]() {
      if (first + sent * nw < tiles) {
        const int half = (sent & 1) * 16;
        const uint32_t to = ring_a + sent_stage * 2 * Sm::kTile;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int id = i * 32 + lane, row = id / (D / 8), ch = id % (D / 8);
          const unsigned pg = (unsigned)max(__shfl_sync(0xffffffffu, pages, half + row), 0);
          copy16(to + (ch >= D / 16) * Sm::kTile + tile_at<D>(row, ch % (D / 16)), kv_bounds + (uint64_t)pg * page_bytes + ch * 16);
        }
        const int pg = __shfl_sync(0xffffffffu, pages, half + (lane & 15));
        if (lane < 16) {
          copy4(smem_addr(meta + sent_stage * 128), c.amax + ((int64_t)max(pg, 0) * c.n_kv + kv) * 2);
          *reinterpret_cast<int*>(meta + sent_stage * 128 + 64) = pg;
        }
        ++sent;
        sent_stage = sent_stage == kSelStages - 1 ? 0 : sent_stage + 1;
        if (!(sent & 1)) {
          pages = cache_checked(c, entries);
          entries = look_up(first + (sent + 2) * nw);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kSelStages - 1; ++i) issue();

    // q in 8 bits, one amax for the group's heads
    uint32_t top = abs_top(qv.f());
    for (int i = tid + kSelThreads; i < c.rep * (D / 4); i += kSelThreads) {
      qv.load(row_ptr<DT>(c.q, q0 + (int64_t)(i / (D / 4)) * c.q_sh + i % (D / 4) * 4));
      top = max(top, abs_top(qv.f()));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[w] = top;
    __syncthreads();
    for (int i = 0; i < kSelWarps; ++i) top = max(top, red[i]);
    const float amax = __uint_as_float(top);
    const float inv = amax >= kTinyAmax && amax < INFINITY ? __fdiv_rn(127.f, amax) : 0.f;
    for (int i = tid; i < nht * (D / 16) * 32; i += kSelThreads) {
      const int ln = i & 31, wd = i / 32 % (D / 16), ht = i / 32 / (D / 16);
      const int head = ht * 8 + (ln >> 2);
      uint32_t neg = 0, pos = 0;
      if (head < c.rep && inv > 0.f) {
        unsigned long long r[2];
        qv.load(row_ptr<DT>(c.q, q0 + (int64_t)head * c.q_sh + wd * 16 + (ln & 3) * 4));
        const uint32_t v = quantize4(qv.f(), inv, amax, r);
        const uint32_t sign = (v >> 7 & 0x01010101u) * 255u;
        neg = v & sign;
        pos = v & ~sign;
      }
      qf[((ht * 2 + 0) * (D / 16) + wd) * 32 + ln] = neg;
      qf[((ht * 2 + 1) * (D / 16) + wd) * 32 + ln] = pos;
    }
    __syncthreads();
    if (ranks > 1) cluster_wait();

    const uint32_t keys0 = at_rank0(keys);
    unsigned long long my_lo = ~0ull, my_hi = 0;
    int my_forced = 0;
    uint32_t q1[2][D / 16];  // the query operand of up to 8 heads stays in registers
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < D / 16; ++k) q1[h][k] = qf[(h * (D / 16) + k) * 32 + lane];
    int done = 0, stage = 0;
    while (true) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kSelStages - 2) : "memory");
      __syncwarp();  // the oldest stage is there for the whole warp, and the one before it free
      issue();
      if (done == sent) break;
      const uint32_t at = ring_a + stage * 2 * Sm::kTile;
      uint32_t x[2][D / 32][4];  // lo, hi: the A operand of every 32 channels
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        ldmatrix4(x[0][k], at + tile_at<D>(lane & 15, 2 * k + (lane >> 4)));
        ldmatrix4(x[1][k], at + Sm::kTile + tile_at<D>(lane & 15, 2 * k + (lane >> 4)));
      }
      int best0 = INT32_MIN, best1 = INT32_MIN;
      const auto heads = [&](int ht, const uint32_t (&q)[2][D / 16]) {
        int acc[2][4] = {};
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            mma_s8(acc[h], x[h][k][0], x[h][k][1], x[h][k][2], x[h][k][3], q[h][2 * k], q[h][2 * k + 1]);
        const int head = ht * 8 + 2 * t;
        if (head < c.rep) { best0 = max(best0, acc[0][0] + acc[1][0]); best1 = max(best1, acc[0][2] + acc[1][2]); }
        if (head + 1 < c.rep) { best0 = max(best0, acc[0][1] + acc[1][1]); best1 = max(best1, acc[0][3] + acc[1][3]); }
      };
      heads(0, q1);
      for (int ht = 1; ht < nht; ++ht) {
        uint32_t q[2][D / 16];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) q[h][k] = qf[((ht * 2 + h) * (D / 16) + k) * 32 + lane];
        heads(ht, q);
      }
      best0 = max(best0, __shfl_xor_sync(0xffffffffu, best0, 1));
      best1 = max(best1, __shfl_xor_sync(0xffffffffu, best1, 1));
      best0 = max(best0, __shfl_xor_sync(0xffffffffu, best0, 2));
      best1 = max(best1, __shfl_xor_sync(0xffffffffu, best1, 2));
      // lane l < 16 takes block e0 + l, whose row is the quad g = l % 8's
      const int v0 = __shfl_sync(0xffffffffu, best0, (lane & 7) * 4), v1 = __shfl_sync(0xffffffffu, best1, (lane & 7) * 4);
      const int blk = (first + done * nw) * 16 + lane;
      if (lane < 16 && blk < here) {
        unsigned long long k = 0;
        if (*reinterpret_cast<const int*>(meta + stage * 128 + 64) >= 0) {
          if (blk < c.sink || blk >= here - c.local) {
            k = ~0ull;
            ++my_forced;
          } else {
            k = order_key((double)(lane < 8 ? v0 : v1) * (double)*reinterpret_cast<const float*>(meta + stage * 128));
            my_lo = min(my_lo, k);
            my_hi = max(my_hi, k);
          }
        }
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(keys0 + blk * 8), "l"(k) : "memory");
      }
      ++done;
      stage = stage == kSelStages - 1 ? 0 : stage + 1;
    }
    __syncwarp();
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      my_lo = min(my_lo, __shfl_xor_sync(0xffffffffu, my_lo, o));
      my_hi = max(my_hi, __shfl_xor_sync(0xffffffffu, my_hi, o));
    }
    my_forced = __reduce_add_sync(0xffffffffu, my_forced);
    if (lane == 0) {
      const int slot = (int)rank * kSelWarps + w;
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_rank0(&s_lo[slot])), "l"(my_lo) : "memory");
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_rank0(&s_hi[slot])), "l"(my_hi) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at_rank0(&s_forced[slot])), "r"(my_forced) : "memory");
    }
    __syncwarp();
    if (ranks > 1) {
      cluster_arrive();
      cluster_wait();
      if (rank) return;
    } else {
      __syncthreads();
    }
  }

  // Keys from `above` up are listed, and those of ~0 (forced, or chosen below).
  unsigned long long above = ~0ull;
  unsigned long long tie = 0;  // a key of which only the first `rem` blocks are listed
  int rem = 0;
  if (!few) {
    unsigned long long lo = ~0ull, hi = 0;
    rem = c.top;
    for (int i = 0; i < (int)ranks * kSelWarps; ++i) {
      lo = min(lo, s_lo[i]);
      hi = max(hi, s_hi[i]);
      rem -= s_forced[i];
    }
    while (rem > 0 && lo <= hi) {  // lo > hi: nothing but forced blocks
      const int bits = hi == lo ? 0 : 64 - __clzll((long long)(hi - lo));
      const int sh = max(0, bits - 8);
      hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < here; i += kSelThreads) {
        const unsigned long long k = keys[i];
        if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> sh)], 1);
      }
      __syncthreads();
      if (w == 0) {
        // lane l holds bins 255 - 8 l .. 248 - 8 l, so an inclusive scan counts from the top
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += hist[255 - lane * 8 - e];
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        int over = upto - sum;
        const bool last = lane == 31 && upto < rem;  // fewer keys than places: down to the lowest bin
        if ((over < rem && upto >= rem) || last) {
          for (int e = 0; e < 8; ++e) {
            const int bin = 255 - lane * 8 - e, n = hist[bin];
            if (over + n >= rem || (last && e == 7)) {
              s_bin = bin;
              s_above = over;
              s_cnt = n;
              break;
            }
            over += n;
          }
        }
      }
      __syncthreads();
      const unsigned long long from = lo + ((unsigned long long)s_bin << sh);
      // a bin's end may lie beyond hi, and for infinite scores beyond 64 bits
      const unsigned long long width = 1ull << sh, upto = hi - from < width ? hi : from + (width - 1);
      const int cnt = s_cnt;
      rem -= s_above;
      if (cnt <= rem) {  // the whole bin
        above = from;
        rem = 0;
        break;
      }
      above = upto + 1;  // no key is ~0 - 1 or above but forced ones: no overflow
      if (cnt <= kSelThreads) {
        // rank the bin's keys against each other; a key of equal value ranks by its block
        for (int i = tid; i < here; i += kSelThreads)
          if (keys[i] >= from && keys[i] <= upto) s_idx[atomicAdd(&s_n, 1)] = i;
        __syncthreads();
        unsigned long long k = 0;
        int place = 0, i = 0;
        if (tid < cnt) {
          i = s_idx[tid];
          k = keys[i];
          for (int j = 0; j < cnt; ++j) {
            const int o = s_idx[j];
            place += keys[o] > k || (keys[o] == k && o < i);
          }
        }
        __syncthreads();
        if (tid < cnt) keys[i] = place < rem ? ~0ull : 0ull;
        __syncthreads();
        rem = 0;
        break;
      }
      if (sh == 0) {  // more equal keys than places
        tie = from;
        break;
      }
      lo = from;
      hi = upto;
    }
  } else {
    above = 1;
  }

  // Ascending block order: each thread a run of blocks, one scan of the counts.
  const int run = (here + kSelThreads - 1) / kSelThreads;
  const int i0 = min(here, tid * run), i1 = min(here, i0 + run);
  int ties_before = 0, total;
  if (tie) {
    int n = 0;
    for (int i = i0; i < i1; ++i) n += keys[i] == tie;
    ties_before = block_scan(n, part, total) - n;
  }
  int n = 0, seen = ties_before;
  for (int i = i0; i < i1; ++i) {
    const unsigned long long k = keys[i];
    n += k >= above || (tie && k == tie && seen++ < rem);
  }
  int at = block_scan(n, part, total) - n;
  seen = ties_before;
  for (int i = i0; i < i1; ++i) {
    const unsigned long long k = keys[i];
    if (k >= above || (tie && k == tie && seen++ < rem)) {
      if (at < c.top) out[at] = i;
      ++at;
    }
  }
  for (int i = total + tid; i < c.top; i += kSelThreads) out[i] = -1;
}

// Blocks of a cluster: one where the units alone give every SM one, else as
// many as give two, with a round of the warps (128 blocks of tokens) for each.
int select_ranks(const CacheDev& c) {
  const int64_t units = (int64_t)c.B * c.n * c.n_kv;
  int ranks = 1;
  while (ranks < 8 && units * ranks < 148 && c.max_blocks > ranks * kSelWarps * 16) ranks *= 2;
  return ranks;
}

template <int DT, int D>
cudaError_t run_select(const CacheDev& c, cudaStream_t st) {
  const int ranks = select_ranks(c);
  const int64_t grid = (int64_t)c.B * c.n * c.n_kv * ranks;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const size_t smem = SelSmem<D>::bytes(c);
  cudaError_t e = allow_smem<k_cache_select<DT, D>>(kSelSmemMax);
  if (e != cudaSuccess) return e;
  CacheLaunch l((unsigned)grid, kSelThreads, smem, st, ranks);
  e = cudaLaunchKernelEx(&l.cfg, k_cache_select<DT, D>, c);
  note_launch();
  return e;
}

template <int DT>
cudaError_t run_select_d(const CacheDev& c, cudaStream_t st) {
  return c.d == 32 ? run_select<DT, 32>(c, st) : c.d == 64 ? run_select<DT, 64>(c, st)
         : c.d == 96 ? run_select<DT, 96>(c, st) : run_select<DT, 128>(c, st);
}

}  // namespace

cudaError_t launch_cache_reserve(const ReserveDev& r, cudaStream_t st) {
  const bool many = r.B > 64;
  CacheLaunch l(many ? kReserveCluster : 1, many ? kReserveThreads : 256, 0, st, many ? kReserveCluster : 1);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, k_cache_reserve, r);
  note_launch();
  return e;
}

cudaError_t launch_cache_append(const CacheDev& c, cudaStream_t st) {
  return c.dtype == kDtF32 ? run_append_d<kDtF32>(c, st) : run_append_d<kDtBF16>(c, st);
}

size_t cache_select_smem(const CacheDev& c) {
  return c.d == 32 ? SelSmem<32>::bytes(c) : c.d == 64 ? SelSmem<64>::bytes(c)
         : c.d == 96 ? SelSmem<96>::bytes(c) : SelSmem<128>::bytes(c);
}

cudaError_t launch_cache_select(const CacheDev& c, cudaStream_t st) {
  return c.dtype == kDtF32 ? run_select_d<kDtF32>(c, st) : run_select_d<kDtBF16>(c, st);
}

}  // namespace ssa
