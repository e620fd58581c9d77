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

// ---------------------------------------------------------------- reserve
constexpr int kReserveThreads = 1024;

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
  int before = 0, all = 0;
  for (int i = 0; i < nw; ++i) {
    const int x = part[i];
    if (i < w) before += x;
    all += x;
  }
  total = all;
  return v + before;
}

// A sequence's pages are taken from the top of the free stack in sequence
// order, so the stack position of every page follows from a prefix sum of the
// needs. A sequence whose pages no longer fit gets none, nor does a later one
// that needs any.
__global__ void __launch_bounds__(kReserveThreads) k_cache_reserve(const ReserveDev r) {
  __shared__ int part[32];
  __shared__ int s_at[kReserveThreads], s_held[kReserveThreads], s_need[kReserveThreads];
  int count = r.state[0];
  const int failed = r.state[1];
  if (count > r.num_pages) count = r.num_pages;
  if (count < 0) count = 0;
  int64_t before = 0;
  int given_all = 0, rejected = 0;
  for (int b0 = 0; b0 < r.B; b0 += kReserveThreads) {
    const int b = b0 + threadIdx.x;
    int len = 0, more = 0;
    if (b < r.B) {
      len = max(r.lens[b], 0);
      more = max(r.new_lens[b], 0);
    }
    const int64_t after = (int64_t)len + more;
    const int held = (len + r.bs - 1) / r.bs;
    const int64_t want = (after + r.bs - 1) / r.bs;
    const bool wide = want > r.max_blocks;
    const int need = wide ? 0 : (int)(want - held);
    int total;
    const int upto = block_scan(need, part, total);
    const bool ok = !wide && (need == 0 || before + upto <= count);
    const int given = ok ? need : 0;
    s_at[threadIdx.x] = count - 1 - (int)(before + upto - need);
    s_held[threadIdx.x] = held;
    s_need[threadIdx.x] = given;
    if (b < r.B) {
      r.start_out[b] = len;
      r.lens_out[b] = ok ? (int)after : len;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < kReserveThreads && b0 + i < r.B; i += kReserveThreads / 32) {
      const int m = s_need[i], at = s_at[i];
      int32_t* row = r.table + (int64_t)(b0 + i) * r.max_blocks + s_held[i];
      for (int j = lane; j < m; j += 32) row[j] = r.free_pages[at - j];
    }
    int sum;
    block_scan(given, part, sum);
    given_all += sum;
    block_scan(b < r.B && !ok, part, sum);
    rejected += sum;
    before += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    r.state_out[0] = count - given_all;
    r.state_out[1] = failed + rejected;
  }
}

// ---------------------------------------------------------------- append
// An amax below this counts as zero: 127 / amax and the logarithm of the
// step stay far inside the fp32 range.
constexpr float kTinyAmax = 0x1p-80f;

// rint(127 x / amax), ties to even, as in exact arithmetic. inv = 127 / amax
// and the product are each within 2^-24 of their values, so t is within 2e-5
// of the quotient; only where that could decide the rounding is the quotient
// formed in 64 bits (127 x is exact there, and a quotient that is not a tie
// is further than 2^-53 from one).
constexpr float kRound = 12582912.f;  // 1.5 2^23: t + kRound is rounded to a whole number, its low byte the code

__device__ __noinline__ float quantize_exact(float x, float amax) {
  return kRound + (float)rint((double)x * 127.0 / (double)amax);
}

// Four codes of x as bytes; r: the codes as floats. inv = 0: all zero.
__device__ __forceinline__ uint32_t quantize4(const float4& x, float inv, float amax, float4& r) {
  const float4 t = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  float4 b = make_float4(t.x + kRound, t.y + kRound, t.z + kRound, t.w + kRound);
  r = make_float4(b.x - kRound, b.y - kRound, b.z - kRound, b.w - kRound);
  const float far = fmaxf(fmaxf(fabsf(t.x - r.x), fabsf(t.y - r.y)), fmaxf(fabsf(t.z - r.z), fabsf(t.w - r.w)));
  if (far > 0.4999f) {
    b = make_float4(quantize_exact(x.x, amax), quantize_exact(x.y, amax), quantize_exact(x.z, amax), quantize_exact(x.w, amax));
    r = make_float4(b.x - kRound, b.y - kRound, b.z - kRound, b.w - kRound);
  }
  const uint32_t lo = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(b.z), __float_as_uint(b.w), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
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
  __device__ __forceinline__ void load_nc(const void* p) { v = __ldg(static_cast<const float4*>(p)); }
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
  __device__ __forceinline__ void load_nc(const void* p) { v = __ldg(static_cast<const uint2*>(p)); }
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
template <int DT, int D, int BS>
__device__ __forceinline__ void append_block(const CacheDev& c, int b, int kv, int s, int blk, int start, int len,
                                             float4* red) {
  using V = Vec4<DT>;
  constexpr int kT = kAppendThreads<D, BS>;
  constexpr int kVec = D / 4, kRg = kT / kVec, kPasses = BS / kRg;
  constexpr int kSize = DT == kDtF32 ? 4 : 2;
  const int tid = threadIdx.x, cv = tid % kVec, r0 = tid / kVec;
  const int p0 = blk * BS;
  const int page = p0 < len ? cache_page(c, b, blk) : -1;  // a block of padding is only cleared in the values
  // rows of the block: [0, old) from the tail, [old, end) from the input, the rest absent
  const int old = page < 0 ? 0 : max(0, min(BS, start - p0)), end = page < 0 ? 0 : min(BS, len - p0);
  const int64_t sn = s ? c.v_sn : c.k_sn;
  const char* in = static_cast<const char*>(s ? c.v : c.k) +
                   ((s ? b * c.v_sb + kv * c.v_sh : b * c.k_sb + kv * c.k_sh) + (int64_t)(p0 - start) * sn + cv * 4) * kSize;
  char* tail = static_cast<char*>(c.tail) + (((((int64_t)b * c.n_kv + kv) * 2 + s) * BS) * D + cv * 4) * kSize;
  V x[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = p * kRg + r0;
    x[p].zero();
    if (row >= old && row < end) x[p].load_nc(in + row * sn * kSize);
  }
  if (old) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kRg + r0;
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
  if (tid == 0 && page >= 0) c.amax[((int64_t)page * c.n_kv + kv) * 2 + s] = amax;
  if (!finite) {  // no codes: zeros, which stand for 0 or for NaN
#pragma unroll
    for (int p = 0; p < kPasses; ++p) x[p].zero();
    lo.zero();
    hi.zero();
    // 0 * step is the value of every code: 0, or NaN of an amax that is infinite or NaN
  }
  int8_t* codes = (s ? c.v_codes : c.k_codes) + ((int64_t)page * c.n_kv + kv) * BS * D + cv * 4;
  char* values = static_cast<char*>(s ? c.v_values : c.k_values);
  const bool open = p0 + BS > len;
  if (values) values += (b * c.o_sb + kv * c.o_sh + (int64_t)(p0 - start) * c.o_sn + cv * 4) * kSize;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = p * kRg + r0;
    const bool have = row < end;
    float4 r;
    const uint32_t q = quantize4(x[p].f(), inv, amax, r);
    if (have) *reinterpret_cast<uint32_t*>(codes + row * D) = q;
    if (values && p0 + row >= start && p0 + row - start < c.n) {
      V o;
      o.zero();
      if (have) o.from(make_float4(r.x * step, r.y * step, r.z * step, r.w * step));
      o.store(values + row * c.o_sn * kSize);
    }
  }
  if (open) {  // the open block's new tokens, as they came (zeroed above where there are no codes: read again)
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kRg + r0;
      if (row >= old && row < end) {
        if (!finite) x[p].load_nc(in + row * sn * kSize);
        x[p].store(tail + (int64_t)row * D * kSize);
      }
    }
  }
  __syncthreads();  // red is free again
  if (!open && s == 0 && page >= 0) {
    V* rl = reinterpret_cast<V*>(red);
    rl[tid] = lo;
    rl[kT + tid] = hi;
    __syncthreads();
    if (tid < kVec) {
      for (int i = 1; i < kRg; ++i) {
        lo.min_with(rl[i * kVec + tid]);
        hi.max_with(rl[kT + i * kVec + tid]);
      }
      float4 r;
      uint32_t* bd = reinterpret_cast<uint32_t*>(c.bounds + ((int64_t)page * c.n_kv + kv) * 2 * D) + tid;
      bd[0] = quantize4(lo.f(), inv, amax, r);
      bd[D / 4] = quantize4(hi.f(), inv, amax, r);
    }
    __syncthreads();
  }
}

// Block j of the touched ones, K or V of one kv head. The first block reads
// the tail and the last one may write it, so one thread block does both, in
// that order.
template <int DT, int D, int BS>
__global__ void __launch_bounds__(kAppendThreads<D, BS>) k_cache_append(const CacheDev c, const int nt) {
  __shared__ float4 red[(DT == kDtF32 ? 2 : 1) * kAppendThreads<D, BS>];
  int64_t i = blockIdx.x;
  const int j = (int)(i % nt);
  i /= nt;
  const int s = (int)(i & 1);
  i >>= 1;
  const int kv = (int)(i % c.n_kv), b = (int)(i / c.n_kv);
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
  k_cache_append<DT, D, BS><<<(unsigned)grid, kAppendThreads<D, BS>, 0, st>>>(c, nt);
  note_launch();
  return cudaGetLastError();
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
constexpr int kSelThreads = 256;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Ordered like the double, 0 below every number.
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);  // -0 -> 0
  return (u >> 63) ? ~u : u | (1ull << 63);
}

// One thread block per (sequence, token, kv head). The bound of a block is
// sum_c max(q lo_c, q hi_c) = q- . lo + q+ . hi (q-, q+ the negative and
// positive parts): a product of 8-bit rows of length 2 d, exact in the
// tensor cores' 32-bit sums; times amax it is exact in 64 bits, so the
// order of two blocks never depends on how the sum was formed.
template <int DT, int D>
__global__ void __launch_bounds__(kSelThreads) k_cache_select(const CacheDev c) {
  extern __shared__ __align__(16) unsigned char sm[];
  const int nht = (c.rep + 7) / 8;                                   // tiles of 8 heads
  uint32_t* qf = reinterpret_cast<uint32_t*>(sm);                    // [nht][2][D / 16][32]: words of q-, q+
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(qf + nht * 2 * (D / 16) * 32);
  __shared__ uint32_t red[32];
  __shared__ int hist[256];
  __shared__ int part[32];
  __shared__ int s_bin, s_rem, s_full;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  int64_t u = blockIdx.x;
  const int kv = (int)(u % c.n_kv);
  u /= c.n_kv;
  const int tok = (int)(u % c.n), b = (int)(u / c.n);
  int32_t* out = c.blocks_out + (int64_t)blockIdx.x * c.top;
  int start, len;
  const int fresh = cache_step_tokens(c, b, start, len);
  const int here = tok < fresh ? (start + tok) / c.bs + 1 : 0;       // blocks that stand for election

  if (here > c.top) {
    // q in 8 bits, one amax for the group's heads
    const int64_t q0 = b * c.q_sb + (int64_t)kv * c.rep * c.q_sh + (int64_t)tok * c.q_sn;
    uint32_t top = 0;
    for (int i = tid; i < c.rep * (D / 4); i += kSelThreads) {
      const float4 x = load4<DT>(row_ptr<DT>(c.q, q0 + (int64_t)(i / (D / 4)) * c.q_sh), i % (D / 4) * 4);
      top = max(top, abs_top(x));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[w] = top;
    __syncthreads();
    for (int i = 0; i < kSelThreads / 32; ++i) top = max(top, red[i]);
    const float amax = __uint_as_float(top);
    const float inv = amax >= kTinyAmax && amax < INFINITY ? __fdiv_rn(127.f, amax) : 0.f;
    for (int i = tid; i < nht * (D / 16) * 32; i += kSelThreads) {
      const int ln = i & 31, wd = i / 32 % (D / 16), ht = i / 32 / (D / 16);
      const int head = ht * 8 + (ln >> 2);
      uint32_t neg = 0, pos = 0;
      if (head < c.rep && inv > 0.f) {
        const float4 x = load4<DT>(row_ptr<DT>(c.q, q0 + (int64_t)head * c.q_sh), cache_word_channel<D>(wd, ln & 3));
        float4 r;
        const uint32_t v = quantize4(x, inv, amax, r), sign = (v >> 7 & 0x01010101u) * 255u;
        neg = v & sign;
        pos = v & ~sign;
      }
      qf[((ht * 2 + 0) * (D / 16) + wd) * 32 + ln] = neg;
      qf[((ht * 2 + 1) * (D / 16) + wd) * 32 + ln] = pos;
    }
    __syncthreads();

    // 16 blocks a warp
    for (int u16 = w; u16 * 16 < here; u16 += kSelThreads / 32) {
      const int e0 = u16 * 16 + g, e1 = e0 + 8;
      const int pg0 = e0 < here ? cache_page(c, b, e0) : -1, pg1 = e1 < here ? cache_page(c, b, e1) : -1;
      uint32_t lo0[D / 16], hi0[D / 16], lo1[D / 16], hi1[D / 16];
      const int8_t* r0 = c.bounds + ((int64_t)max(pg0, 0) * c.n_kv + kv) * 2 * D;
      const int8_t* r1 = c.bounds + ((int64_t)max(pg1, 0) * c.n_kv + kv) * 2 * D;
      cache_load_row<D>(r0, t, lo0);
      cache_load_row<D>(r1, t, lo1);
      cache_load_row<D>(r0 + D, t, hi0);
      cache_load_row<D>(r1 + D, t, hi1);
      const float am0 = __ldg(c.amax + ((int64_t)max(pg0, 0) * c.n_kv + kv) * 2);
      const float am1 = __ldg(c.amax + ((int64_t)max(pg1, 0) * c.n_kv + kv) * 2);
      int best0 = INT32_MIN, best1 = INT32_MIN;
      for (int ht = 0; ht < nht; ++ht) {
        int acc[4] = {0, 0, 0, 0};
        const uint32_t* fn = qf + (ht * 2) * (D / 16) * 32 + lane;
        const uint32_t* fp = fn + (D / 16) * 32;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          mma_s8(acc, lo0[2 * k], lo1[2 * k], lo0[2 * k + 1], lo1[2 * k + 1], fn[2 * k * 32], fn[(2 * k + 1) * 32]);
          mma_s8(acc, hi0[2 * k], hi1[2 * k], hi0[2 * k + 1], hi1[2 * k + 1], fp[2 * k * 32], fp[(2 * k + 1) * 32]);
        }
        const int h = ht * 8 + 2 * t;
        if (h < c.rep) { best0 = max(best0, acc[0]); best1 = max(best1, acc[2]); }
        if (h + 1 < c.rep) { best0 = max(best0, acc[1]); best1 = max(best1, acc[3]); }
      }
      best0 = max(best0, __shfl_xor_sync(0xffffffffu, best0, 1));
      best1 = max(best1, __shfl_xor_sync(0xffffffffu, best1, 1));
      best0 = max(best0, __shfl_xor_sync(0xffffffffu, best0, 2));
      best1 = max(best1, __shfl_xor_sync(0xffffffffu, best1, 2));
      if (t == 0) {
        if (e0 < here)
          keys[e0] = pg0 < 0 ? 0ull : e0 < c.sink || e0 >= here - c.local ? ~0ull : order_key((double)best0 * (double)am0);
        if (e1 < here)
          keys[e1] = pg1 < 0 ? 0ull : e1 < c.sink || e1 >= here - c.local ? ~0ull : order_key((double)best1 * (double)am1);
      }
    }
    __syncthreads();
  } else {
    for (int i = tid; i < here; i += kSelThreads) keys[i] = cache_page(c, b, i) < 0 ? 0ull : ~0ull;
    __syncthreads();
  }

  // The top-th largest key, eight bits at a time from the highest.
  unsigned long long prefix = 0, mask = 0;
  int rem = c.top;
  for (int shift = 56; shift >= 0 && here > c.top; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < here; i += kSelThreads) {
      const unsigned long long k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(int)(k >> shift) & 255], 1);
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
      int above = upto - sum;
      if (above < rem && upto >= rem) {
        for (int e = 0; e < 8; ++e) {
          const int bin = 255 - lane * 8 - e, n = hist[bin];
          if (above + n >= rem) {
            s_bin = bin;
            s_rem = rem - above;
            s_full = n == rem - above;
            break;
          }
          above += n;
        }
      }
    }
    __syncthreads();
    prefix |= (unsigned long long)s_bin << shift;
    mask |= 255ull << shift;
    rem = s_rem;
    if (s_full) break;
  }
  if (here <= c.top) { prefix = 0; mask = ~0ull; rem = 0; }  // every block with a page

  // Ascending block order; among equal keys the lowest blocks.
  int written = 0, ties = 0;
  for (int i0 = 0; i0 < here; i0 += kSelThreads) {
    const int i = i0 + tid;
    const unsigned long long k = i < here ? keys[i] : 0ull;
    const bool eq = i < here && k != 0 && (k & mask) == prefix && here > c.top;
    int n_eq, n_take;
    const int rank = block_scan(eq, part, n_eq) - eq + ties;
    const bool take = i < here && k != 0 && ((k & mask) > prefix || (eq && rank < rem));
    const int at = block_scan(take, part, n_take) - take + written;
    if (take && at < c.top) out[at] = i;
    ties += n_eq;
    written += n_take;
  }
  for (int i = written + tid; i < c.top; i += kSelThreads) out[i] = -1;
}

template <int DT, int D>
cudaError_t run_select(const CacheDev& c, cudaStream_t st) {
  const int64_t grid = (int64_t)c.B * c.n * c.n_kv;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const size_t smem = cache_select_smem(c);
  cudaError_t e = cudaFuncSetAttribute(k_cache_select<DT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  k_cache_select<DT, D><<<(unsigned)grid, kSelThreads, smem, st>>>(c);
  note_launch();
  return cudaGetLastError();
}

template <int DT>
cudaError_t run_select_d(const CacheDev& c, cudaStream_t st) {
  return c.d == 32 ? run_select<DT, 32>(c, st) : c.d == 64 ? run_select<DT, 64>(c, st)
         : c.d == 96 ? run_select<DT, 96>(c, st) : run_select<DT, 128>(c, st);
}

}  // namespace

cudaError_t launch_cache_reserve(const ReserveDev& r, cudaStream_t st) {
  k_cache_reserve<<<1, kReserveThreads, 0, st>>>(r);
  note_launch();
  return cudaGetLastError();
}

cudaError_t launch_cache_append(const CacheDev& c, cudaStream_t st) {
  return c.dtype == kDtF32 ? run_append_d<kDtF32>(c, st) : run_append_d<kDtBF16>(c, st);
}

size_t cache_select_smem(const CacheDev& c) {
  return (size_t)((c.rep + 7) / 8) * 2 * (c.d / 16) * 32 * 4 + (size_t)c.max_blocks * 8;
}

cudaError_t launch_cache_select(const CacheDev& c, cudaStream_t st) {
  return c.dtype == kDtF32 ? run_select_d<kDtF32>(c, st) : run_select_d<kDtBF16>(c, st);
}

}  // namespace ssa
