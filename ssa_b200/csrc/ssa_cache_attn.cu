// ssa_cache_attn.cu -- attention of a few query tokens over the 8-bit block
// cache, over every block of a sequence or the blocks a list names.
//
// s = scale q . k, k = code * amax_k / 127; out = sum 2^(s' - m) v / sum
// 2^(s' - m) with s' = s log2(e) and a running offset m, one pass over the
// codes. A group's query rows (its heads times its tokens) are the 8-wide
// side of the tensor products and 16 keys or channels the 16-wide one:
//   S^T (keys x rows)     = K . Q^T    (K codes as fp16, exact)
//   O^T (channels x rows) = V^T . P^T  (V codes as fp16, exact)
// so eight rows fill an instruction; q and the weights P are fp16 -- q scaled
// by a power of two for each row (a bf16 q is then exact), P below 2^15 -- or,
// for fp32 tensors, fp16 pairs (high part and remainder, 22 bits). fp16 is what
// the products take beside codes that are exact in it: a weight is then off by
// 2^-12 of itself where a bf16 output is by 2^-9, and the weights' sum takes
// them before that rounding. Sums are fp32. The step of V, which differs from page to page, goes into the
// exponent: P = 2^(s' + log2(step) - m), and the weights' sum takes P / step.
// mma.sync rather than tcgen05: with 8 to 32 rows the operation is bound by
// reading the codes, and a 128-row tile would be mostly padding.
//
// Measured: 32 sequences of up to 8192 keys, 32 heads over 8, d 128 (408 MB):
// 74 to 80 us, 5.1 to 5.5 TB/s of a copy's 6.55. The same of 64 listed blocks
// for 16 sequences (135 MB): 33 to 34 us, 4.0 TB/s -- as long as a launch's start,
// the first look-ups and the join weigh at that size. One fp32 sequence of 333
// keys: 8 us, two launches. Four drafts of 32 heads over one (8 x 8192 keys,
// d 64, four tiles of 32 rows): 23 us, bound by latency and the exponentials.
//
// Work is counted in groups of 64 keys over all (sequence, row tile, kv head)
// units and cut into one equal range for each thread block, so ragged batches
// balance; a unit that spans several blocks leaves its partial sums in the
// workspace and k_cache_combine joins them in range order.
#include "ssa_cache_attn.cuh"

namespace ssa {

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// High part and remainder of a pair; of a pair of weights.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_f16(a - f.x, b - f.y);
}
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_weights(a, b);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_weights(a - f.x, b - f.y);
}

// Shared memory of a block: for each warp a ring of staged tiles (keys and
// values of 16 keys a stage), used for the warp's partial output afterwards;
// what comes with each stage; the query operand.
constexpr int kStages = 4;
template <int D, int NT, bool F32>
struct Smem {
  static constexpr int kTile = 16 * kPitch<D>;
  static constexpr int kRing = kStages * 2 * kTile, kOut = 8 * NT * (D + 4) * 4;
  static constexpr int kWarp = kRing > kOut ? kRing : kOut;
  static constexpr int kMeta = kWarps * kWarp;                           // [kWarps][kStages] {amax k, v, first key, -}
  static constexpr int kMl = kMeta + kWarps * kStages * 16;              // [kWarps][8 NT] {offset, sum}
  static constexpr int kScale = kMl + kWarps * 8 * NT * 8;               // [8 NT] score factor of a row
  static constexpr int kQ = kScale + 8 * NT * 4;                         // [F32 ? 2 : 1][NT][D / 16][32] uint2
  static constexpr int kBytes = kQ + (F32 ? 2 : 1) * NT * (D / 16) * 32 * 8;
};
// Tiles of 8 rows leave registers for one more block an SM: the join's, which
// set up while the last ranges run.
template <int D, int NT, bool F32>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(D, 8 * NT) + (NT == 1)) k_cache_attn(const CacheDev c, const Plan pl) {
  using Sm = Smem<D, NT, F32>;
  constexpr int ROWS = 8 * NT, W16 = D / 16, PC = F32 ? 2 : 1, OP = D + 4;
  constexpr int kDt = F32 ? kDtF32 : kDtBF16;
  extern __shared__ __align__(128) unsigned char sm[];
  uint2* qf = reinterpret_cast<uint2*>(sm + Sm::kQ);
  float* sml = reinterpret_cast<float*>(sm + Sm::kMl);
  float* srow = reinterpret_cast<float*>(sm + Sm::kScale);
  __shared__ RangeSmem rs;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  const int bs_shift = c.bs == 16 ? 4 : c.bs == 32 ? 5 : 6;
  grid_wait();  // k_cache_combine may take its place behind it
  const BlockRange br(c.B, c.prefix, least_groups(ROWS), rs, [&](int i) {
    int tiles, groups;
    return seq_work(c, pl, i, ROWS, &tiles, &groups);
  });
  const int lo = br.lo, hi = br.hi;
  if (lo >= hi) return;

  int b = br.b, base = br.base;
  for (int at = lo; at < hi;) {
    int tiles, groups;
    const int mine = seq_work(c, pl, b, ROWS, &tiles, &groups);
    if (at >= base + mine) { base += mine; ++b; continue; }
    const int u = (int)((unsigned)(at - base) / (unsigned)groups);
    const int ubeg = base + u * groups, uend = ubeg + groups;
    const int g0 = at - ubeg, g1 = min(hi, uend) - ubeg;
    at = ubeg + g1;
    const Unit x = unit_of<ROWS>(c, pl, b, u, tiles);

    // keys a row of the tile sees: at least lim_min, at most lim_max
    const int lim_max = x.nrows <= 0 ? 0 : c.causal ? x.start + (x.row0 + x.nrows - 1) / c.rep + 1 : x.len;
    const int lim_min = c.causal ? x.start + x.row0 / c.rep + 1 : x.len;

    // Warp i < NT fetches the i-th 8 query rows, ahead of the codes in the memory's queue.
    Raw4<F32> qv[W16];
    if (w < NT && w * 8 + g < x.nrows) {
      const int row = x.row0 + w * 8 + g, tok = row / c.rep, h = x.kv * c.rep + row - tok * c.rep;
      const void* qr = row_ptr<kDt>(c.q, x.b * c.q_sb + h * c.q_sh + tok * c.q_sn);
#pragma unroll
      for (int i = 0; i < W16; ++i) qv[i].load(qr, i * 16 + t * 4);
    } else {
#pragma unroll
      for (int i = 0; i < W16; ++i) qv[i].zero();
    }

    // The warp's 16 keys of each group, in order, through its ring. Lane l
    // holds the page of group s0 + l, and of group s0 + 32 + l (loaded ahead).
    unsigned char* ring = sm + w * Sm::kWarp;
    const uint32_t ring_a = smem_addr(ring), meta_a = smem_addr(sm + Sm::kMeta + w * kStages * 16);
    int page, kb, off, entry_n, kb_n, off_n;
    const auto look_up = [&](int s0, int& entry, int& first, int& o) {
      entry = -1;
      if (s0 + lane < g1) {
        const int64_t key = (int64_t)(s0 + lane) * kGroup + w * 16;
        const int e = (int)(key >> bs_shift);
        o = (int)key & (c.bs - 1);
        const int blk = !x.list ? e : e < c.top ? x.list[e] : -1;
        if (blk >= 0 && blk < c.max_blocks) {
          first = blk * c.bs + o;
          if (first < lim_max) entry = cache_entry(c, x.b, blk);
        }
      }
    };
    int s0 = g0;
    look_up(s0, page, kb, off);
    look_up(s0 + 32, entry_n, kb_n, off_n);
    page = cache_checked(c, page);
    uint32_t todo = __ballot_sync(0xffffffffu, page >= 0);
    int issued = 0, used = 0;
    const auto issue = [&]() {
      while (!todo && s0 + 32 < g1) {
        s0 += 32;
        page = cache_checked(c, entry_n); kb = kb_n; off = off_n;
        look_up(s0 + 32, entry_n, kb_n, off_n);
        todo = __ballot_sync(0xffffffffu, page >= 0);
      }
      if (todo) {
        const int j = __ffs(todo) - 1, st = issued & (kStages - 1);
        todo &= todo - 1;
        const int64_t head = (int64_t)__shfl_sync(0xffffffffu, page, j) * c.n_kv + x.kv;
        const int64_t row = head * c.bs + __shfl_sync(0xffffffffu, off, j);
        const int first = __shfl_sync(0xffffffffu, kb, j);
        const int8_t* ks = c.k_codes + row * D + lane * 16;
        const int8_t* vs = c.v_codes + row * D + lane * 16;
        const uint32_t at = ring_a + st * 2 * Sm::kTile;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const int id = i * 32 + lane, to = tile_at<D>(id / W16, id % W16);
          copy16(at + to, ks + i * 512);
          copy16(at + Sm::kTile + to, vs + i * 512);
        }
        if (lane == 0) {
          copy8(meta_a + st * 16, c.amax + head * 2);
          *reinterpret_cast<int*>(sm + Sm::kMeta + (w * kStages + st) * 16 + 8) = first;
        }
        ++issued;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();

    // Q as the products' 8-wide operand: rows scaled into fp16's range by a power of two
    if (w < NT) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < W16; ++i) {
        const float4 v = qv[i].f();
        top = max(top, max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                           max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e brings the row's largest element into [2^9, 2^10); e in [-118, 100]
      int e = 9 - ((int)(top >> 23) - 127);
      e = top >= 0x7f800000u ? 0 : min(e, 100);
      const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < W16; ++i) {
        const float4 v = qv[i].f();
        uint2 hi2, lo2;
        split_f16(v.x * up, v.y * up, hi2.x, lo2.x);
        split_f16(v.z * up, v.w * up, hi2.y, lo2.y);
        qf[(w * W16 + i) * 32 + lane] = hi2;
        if constexpr (F32) qf[((NT + w) * W16 + i) * 32 + lane] = lo2;
      }
      if (t == 0) srow[w * 8 + g] = c.scale * 1.4426950408889634f * down;
    }
    __syncthreads();
    float sfac[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int rr = nt * 8 + 2 * t + k;
        sfac[nt][k] = srow[rr];
        lim[nt][k] = INT32_MAX;  // rows behind the last one: computed, never stored
        if (rr < x.nrows) lim[nt][k] = c.causal ? x.start + (x.row0 + rr) / c.rep + 1 : x.len;
      }

    float acc[W16][NT][4], mref[NT][2], lsum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mref[nt][0] = mref[nt][1] = kEmpty;
      lsum[nt][0] = lsum[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < W16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][nt][k] = 0.f;
    }

    // row and half of the 8x8 tile whose row address this lane gives
    const int mrow = lane & 15, mchunk = lane >> 4;
    while (true) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();  // the oldest stage is there for the whole warp, and the one before it free
      issue();
      if (used == issued) break;
      const int st = used & (kStages - 1);
      ++used;
      const uint32_t ka_at = ring_a + st * 2 * Sm::kTile, va_at = ka_at + Sm::kTile;
      const float4 meta = *reinterpret_cast<const float4*>(sm + Sm::kMeta + (w * kStages + st) * 16);
      const float ka = meta.x * (1.f / 127.f), va = meta.y * (1.f / 127.f);
      const int kbj = __float_as_int(meta.z);

      float s[NT][4], s2[NT][4];  // two chains
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[nt][k] = s2[nt][k] = 0.f;
#pragma unroll
      for (int i = 0; i < W16; i += 2) {
        uint32_t x4[4];  // rows 0-7 and 8-15 of chunk i, then of chunk i + 1: channels 4 t .. 4 t + 3
        ldmatrix4(x4, ka_at + tile_at<D>(mrow, i + mchunk));
#pragma unroll
        for (int k = 0; k < 4; ++k) x4[k] ^= 0x80808080u;
        const uint32_t a[4] = {codes_f16<0x4140>(x4[0]), codes_f16<0x4140>(x4[1]), codes_f16<0x4342>(x4[0]), codes_f16<0x4342>(x4[1])};
        const uint32_t e[4] = {codes_f16<0x4140>(x4[2]), codes_f16<0x4140>(x4[3]), codes_f16<0x4342>(x4[2]), codes_f16<0x4342>(x4[3])};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int pc = 0; pc < PC; ++pc) {
            const uint2 b0 = qf[((pc * NT + nt) * W16 + i) * 32 + lane], b1 = qf[((pc * NT + nt) * W16 + i + 1) * 32 + lane];
            mma_f16(s[nt], a, b0.x, b0.y);
            mma_f16(s2[nt], e, b1.x, b1.y);
          }
      }

      // weights 2^(s' + log2(step_v) - m + 13)
      const bool plain = va > 0.f && va < INFINITY;
      const float vs = plain ? va : 1.f, head = plain ? kHead : kHead + kZeroHead;
      const float lv = F32 ? log2f(vs) : __log2f(vs), iv = 1.f / vs;
      const bool edge = kbj + 16 > lim_min;
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v = fmaf(s[nt][k] + s2[nt][k], ka * sfac[nt][k & 1], lv);
          if (edge && kbj + g + 8 * (k >> 1) >= lim[nt][k & 1]) v = -INFINITY;
          s[nt][k] = v;
          move |= v > mref[nt][k & 1] + (head + kSlack);
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float m = fmaxf(s[nt][k], s[nt][k + 2]);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            m = fmaxf(mref[nt][k], m - head);
            const float f = ex2(mref[nt][k] - m);
            mref[nt][k] = m;
            lsum[nt][k] *= f;
#pragma unroll
            for (int i = 0; i < W16; ++i) {
              acc[i][nt][k] *= f;
              acc[i][nt][k + 2] *= f;
            }
          }
      }
      uint32_t pf[PC][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = ex2(s[nt][k] - mref[nt][k & 1]);
        lsum[nt][0] = fmaf(p[0] + p[2], iv, lsum[nt][0]);
        lsum[nt][1] = fmaf(p[1] + p[3], iv, lsum[nt][1]);
        if constexpr (F32) {
          uint32_t h0, l0, h1, l1;
          split_weights(p[0], p[1], h0, l0);
          split_weights(p[2], p[3], h1, l1);
          pf[0][nt][0] = transpose8x8(h0);
          pf[0][nt][1] = transpose8x8(h1);
          pf[PC - 1][nt][0] = transpose8x8(l0);
          pf[PC - 1][nt][1] = transpose8x8(l1);
        } else {
          pf[0][nt][0] = transpose8x8(pack_weights(p[0], p[1]));
          pf[0][nt][1] = transpose8x8(pack_weights(p[2], p[3]));
        }
      }

      // transposed as pairs of codes: a lane has channels 2 g, 2 g + 1 of keys 2 t, 2 t + 1
#pragma unroll
      for (int i = 0; i < W16; i += 2) {
        uint32_t x4[4];  // keys 0-7 and 8-15 of chunk i, then of chunk i + 1
        ldmatrix4_trans(x4, va_at + tile_at<D>(mrow, i + mchunk));
#pragma unroll
        for (int k = 0; k < 4; ++k) x4[k] ^= 0x80808080u;
        const uint32_t a[4] = {codes_f16<0x4240>(x4[0]), codes_f16<0x4341>(x4[0]), codes_f16<0x4240>(x4[1]), codes_f16<0x4341>(x4[1])};
        const uint32_t e[4] = {codes_f16<0x4240>(x4[2]), codes_f16<0x4341>(x4[2]), codes_f16<0x4240>(x4[3]), codes_f16<0x4341>(x4[3])};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int pc = 0; pc < PC; ++pc) {
            mma_f16(acc[i][nt], a, pf[pc][nt][0], pf[pc][nt][1]);
            mma_f16(acc[i + 1][nt], e, pf[pc][nt][0], pf[pc][nt][1]);
          }
      }
      if (!(va < INFINITY)) {  // V stands for NaN where a key is seen; the weights' sum is K's alone
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (kbj < lim[nt][k])
#pragma unroll
              for (int i = 0; i < W16; ++i) acc[i][nt][k] = acc[i][nt][k + 2] = NAN;
      }
    }
    __syncwarp();

    // Join the four warps.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = lsum[nt][k];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int r = nt * 8 + 2 * t + k;
        if (g == 0) {
          sml[(w * ROWS + r) * 2] = mref[nt][k];
          sml[(w * ROWS + r) * 2 + 1] = l;
        }
        float* row = reinterpret_cast<float*>(ring) + r * OP + 2 * g;
#pragma unroll
        for (int i = 0; i < W16; ++i)
          *reinterpret_cast<float2*>(row + 16 * i) = make_float2(acc[i][nt][k], acc[i][nt][k + 2]);
      }
    __syncthreads();
    const bool full = g0 == 0 && g1 == groups;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (g0 == 0);
    for (int i = tid; i < ROWS * (D / 4); i += kThreads) {
      const int r = i / (D / 4), ch = i % (D / 4) * 4;
      if (r >= x.nrows) break;
      float m = kEmpty;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) m = fmaxf(m, sml[(k * ROWS + r) * 2]);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = ex2(sml[(k * ROWS + r) * 2] - m);
        l = fmaf(f, sml[(k * ROWS + r) * 2 + 1], l);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm + k * Sm::kWarp) + r * OP + ch);
        o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
      }
      if (full) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store_out<F32>(c, x, r, ch, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        if (ch == 0 && c.lse) store_lse(c, x, r, m, l);
      } else {
        *reinterpret_cast<float4*>(c.part_o + (slot * ROWS + r) * D + ch) = o;
        if (ch == 0) *reinterpret_cast<float2*>(c.part_ml + (slot * ROWS + r) * 2) = make_float2(m, l);
      }
    }
    __syncthreads();
  }
}

// Joins the partial sums of a query row that several blocks worked on, and
// writes zeros to rows without work. PARTS warps share a row's sums, each in
// range order and then one after the other: one where there are many rows,
// four where few rows have many sums (one sequence of 16384 tokens, two kv
// heads: 74 sums a row). The kernel is launched while the other still runs
// and waits for it behind its set-up.
template <int D, int NT, bool F32, int PARTS>
__global__ void __launch_bounds__(kThreads) k_cache_combine(const CacheDev c, const Plan pl, const int ngrid,
                                                            const int rows_used, const int nrows) {
  constexpr int ROWS = 8 * NT, E = D / 32;
  constexpr int kDt = F32 ? kDtF32 : kDtBF16;
  __shared__ float s_ml[PARTS][2], s_o[PARTS][D];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int part = PARTS == 1 ? 0 : w;
  const unsigned id = PARTS == 1 ? blockIdx.x * kWarps + w : blockIdx.x;
  // k_cache_attn lets this kernel come up only after its own wait, so lengths
  // may be read before this one's. Every warp waits: this kernel's end then
  // implies the other's.
  if (id >= (unsigned)nrows) {
    grid_wait();
    return;
  }
  const int per = pl.tiles_max * (c.blocks ? c.n : 1);  // row tiles a (sequence, kv head) can have
  const unsigned unit = id / (unsigned)rows_used, units_b = (unsigned)per * c.n_kv;
  const int r = (int)(id - unit * rows_used);
  const int b = (int)(unit / units_b), u = (int)(unit % units_b);
  const int kv = (int)((unsigned)u / (unsigned)per), tile = u - kv * per;
  int tiles, groups;
  const int mine = seq_work(c, pl, b, ROWS, &tiles, &groups);
  const Unit x = unit_of<ROWS>(c, pl, b, u, per);
  const int row = x.row0 + r, tok = row / c.rep, h = kv * c.rep + row - tok * c.rep;
  const int64_t at = x.b * c.o_sb + h * c.o_sh + tok * c.o_sn;
  int total = mine * c.B, base = mine * b;
  if (!c.blocks && c.B <= 128) {
    // what the other kernel has found out too, while it still runs
    total = base = 0;
    for (int i = lane; i < c.B; i += 32) {
      int a, e;
      const int v = seq_work(c, pl, i, ROWS, &a, &e);
      total += v;
      base += i < b ? v : 0;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    base = __reduce_add_sync(0xffffffffu, base);
  }
  grid_wait();
  if (r >= (c.blocks ? c.rep - tile % pl.tiles_max * ROWS : c.n * c.rep - x.row0)) return;
  float m = kEmpty, l = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  if (tile < tiles && mine > 0 && r < x.nrows) {
    if (!c.blocks && c.B > 128) {
      total = c.prefix[c.B];
      base = c.prefix[b];
    }
    const int ubeg = base + (kv * tiles + tile) * groups;
    const Ranges rg(total, ngrid, least_groups(ROWS));
    const int c0 = rg.of(ubeg), c1 = rg.of(ubeg + groups - 1);
    if (c0 == c1) return;  // that block stored the row
    // sums part, part + PARTS, ... of the row's
    const int cnt = (c1 - c0 + PARTS - part) / PARTS;
    const auto slot = [&](int i) {
      const int k = c0 + part + i * PARTS;
      return ((int64_t)k * 2 + (k == c0)) * ROWS + r;
    };
    // sums come in batches of loads; the first is under way while the weights are found
    constexpr int kBatch = PARTS > 1 ? 16 : 8;
    float batch[kBatch][E];
    const auto load = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < cnt) {
          const float* p = c.part_o + slot(j0 + j) * D + lane;
#pragma unroll
          for (int i = 0; i < E; ++i) batch[j][i] = p[32 * i];
        }
    };
    load(0);
    float2 ml = make_float2(kEmpty, 0.f);
    if (lane < cnt) ml = *reinterpret_cast<const float2*>(c.part_ml + slot(lane) * 2);
    m = ml.x;
    for (int k = 32 + lane; k < cnt; k += 32) m = fmaxf(m, c.part_ml[slot(k) * 2]);
#pragma unroll
    for (int q = 16; q; q >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, q));
    for (int k0 = 0; k0 < cnt; k0 += 32) {
      if (k0) {
        ml = make_float2(kEmpty, 0.f);
        if (k0 + lane < cnt) ml = *reinterpret_cast<const float2*>(c.part_ml + slot(k0 + lane) * 2);
      }
      const float f = ex2(ml.x - m);
      l = fmaf(f, ml.y, l);
      for (int j0 = 0; j0 < 32 && k0 + j0 < cnt; j0 += kBatch) {
        if (k0 + j0) load(k0 + j0);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const float fj = __shfl_sync(0xffffffffu, f, j0 + j);
          if (k0 + j0 + j < cnt)
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = fmaf(fj, batch[j][i], o[i]);
        }
      }
    }
#pragma unroll
    for (int q = 16; q; q >>= 1) l += __shfl_xor_sync(0xffffffffu, l, q);
    if constexpr (PARTS > 1) {  // the whole block has one row: everyone is here
      if (lane == 0) {
        s_ml[part][0] = m;
        s_ml[part][1] = l;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) s_o[part][lane + 32 * i] = o[i];
      __syncthreads();
      if (part) return;
#pragma unroll
      for (int k = 1; k < PARTS; ++k) m = fmaxf(m, s_ml[k][0]);
      l = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        const float f = ex2(s_ml[k][0] - m);
        l = fmaf(f, s_ml[k][1], l);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf(f, s_o[k][lane + 32 * i], o[i]);
      }
    }
  }
  if (part) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) store1<kDt>(row_ptr_mut<kDt>(c.out, at), lane + 32 * i, o[i] * inv);
  if (lane == 0 && c.lse) store_lse(c, x, r, m, l);
}

// Rows of a tile: 8, 16 or 32 (the rows a group has, as far as they go), or
// 128 on the 5th-generation tensor cores.
int tile_rows(const CacheDev& c) {
  const int64_t rows = c.blocks ? c.rep : (int64_t)c.n * c.rep;
  if (rows >= kPromptMin && !c.blocks && c.dtype == kDtBF16 &&
      rows * c.B * c.n_kv * c.max_blocks * c.bs >= prompt_work(rows))
    return kPromptRows;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}

Plan plan_of(const CacheDev& c) {
  Plan p;
  p.rows = tile_rows(c);
  p.tiles_max = (int)(((c.blocks ? c.rep : (int64_t)c.n * c.rep) + p.rows - 1) / p.rows);
  p.list_groups = c.blocks ? (int)(((int64_t)c.top * c.bs + kGroup - 1) / kGroup) : 0;
  return p;
}

int64_t units_of(const CacheDev& c, const Plan& p) {
  return (int64_t)c.B * c.n_kv * p.tiles_max * (c.blocks ? c.n : 1);
}

template <int D, int NT, bool F32>
cudaError_t run_combine(const CacheDev& c, const Plan& pl, cudaStream_t st) {
  constexpr int ROWS = 8 * NT;
  const int64_t units = units_of(c, pl);
  if (units > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const int rows_used = (int)((c.blocks ? c.rep : (int64_t)c.n * c.rep) < ROWS ? (c.blocks ? c.rep : c.n * c.rep) : ROWS);
  const int64_t nrows = units * rows_used;
  if (nrows > 0x7fffffff - kWarps) return cudaErrorInvalidConfiguration;
  // a block a row where a unit may be in many ranges and the rows leave the SMs room
  const bool wide = c.grid > 16 * units && nrows <= 148 * 16;
  CacheLaunch join((unsigned)(wide ? nrows : (nrows + kWarps - 1) / kWarps), kThreads, 0, st);
  const cudaError_t e = wide ? cudaLaunchKernelEx(&join.cfg, k_cache_combine<D, NT, F32, kWarps>, c, pl, c.grid, rows_used, (int)nrows)
                             : cudaLaunchKernelEx(&join.cfg, k_cache_combine<D, NT, F32, 1>, c, pl, c.grid, rows_used, (int)nrows);
  note_launch();
  return e;
}

template <int D, int NT, bool F32>
cudaError_t run_attn(const CacheDev& c, const Plan& pl, cudaStream_t st) {
  constexpr size_t smem = Smem<D, NT, F32>::kBytes;
  cudaError_t e = allow_smem<k_cache_attn<D, NT, F32>>(smem);
  if (e != cudaSuccess) return e;
  CacheLaunch main(c.grid, kThreads, smem, st);
  e = cudaLaunchKernelEx(&main.cfg, k_cache_attn<D, NT, F32>, c, pl);
  note_launch();
  return e != cudaSuccess ? e : run_combine<D, NT, F32>(c, pl, st);
}

template <int D, bool F32>
cudaError_t run_attn_rows(const CacheDev& c, cudaStream_t st) {
  const Plan pl = plan_of(c);
  if constexpr (!F32)
    if (pl.rows == kPromptRows) return launch_cache_prompt(c, pl, st);
  return pl.rows == 8 ? run_attn<D, 1, F32>(c, pl, st) : pl.rows == 16 ? run_attn<D, 2, F32>(c, pl, st)
                                                                       : run_attn<D, 4, F32>(c, pl, st);
}

template <bool F32>
cudaError_t run_attn_d(const CacheDev& c, cudaStream_t st) {
  return c.d == 32 ? run_attn_rows<32, F32>(c, st) : c.d == 64 ? run_attn_rows<64, F32>(c, st)
         : c.d == 96 ? run_attn_rows<96, F32>(c, st) : run_attn_rows<128, F32>(c, st);
}

}  // namespace

size_t cache_attn_workspace_layout(CacheDev* c, void* ws) {
  const Plan p = plan_of(*c);
  const int64_t groups = p.list_groups ? p.list_groups : ((int64_t)c->max_blocks * c->bs + kGroup - 1) / kGroup;
  const int64_t most = units_of(*c, p) * groups;  // no use for more blocks than groups
  if (most > 0x7fffffff) return 0;                // the kernels count groups in 32 bits
  const int64_t full = 148 * blocks_per_sm(c->d, p.rows);
  c->grid = (int)(most < full ? most : full);
  const size_t o_pre = ((size_t)(c->B + 1) * 4 + 255) / 256 * 256;
  const size_t o_ml = o_pre + ((size_t)c->grid * 2 * p.rows * 2 * 4 + 255) / 256 * 256;
  char* base = static_cast<char*>(ws);
  c->prefix = reinterpret_cast<int32_t*>(base);
  c->part_ml = reinterpret_cast<float*>(base + o_pre);
  c->part_o = reinterpret_cast<float*>(base + o_ml);
  return o_ml + (size_t)c->grid * 2 * p.rows * c->d * 4;
}

cudaError_t launch_cache_attn(const CacheDev& c, cudaStream_t st) {
  return c.dtype == kDtF32 ? run_attn_d<true>(c, st) : run_attn_d<false>(c, st);
}

}  // namespace ssa
