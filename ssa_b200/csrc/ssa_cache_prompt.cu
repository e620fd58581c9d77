// ssa_cache_prompt.cu -- attention over the 8-bit block cache for many query
// rows (a prompt's chunk, drafts of a multi-query model), on the
// 5th-generation tensor cores.
//
// The mathematics is k_cache_attn's (ssa_cache_attn.cu), whose tiles of 8 to
// 32 rows read and convert the codes again for every tile. Here 128 rows share
// that:
//   warps 4-7 load the codes of 64 keys a block of steps ahead, convert them
//             to fp16 and store K and V as swizzled 128-byte rows (two stages);
//   warp 8    issues S = Q K^T (128 x 64 x d, fp32 in TMEM) for the next keys,
//             then O += P V (128 x d x 64) with P in TMEM and V key-major, as
//             it lies;
//   warps 0-3 own a row a thread: read S, mask, move the row's offset when a
//             score outgrows it, and write P = 2^(s - m) as fp16 to TMEM.
// Where it takes over from k_cache_attn, ssa_cache_attn.cuh has measured.
//
// Two sequences' 256 tokens behind up to 7936, 32 heads over 8, d 128: 82 to 84
// us with the join, 475 TFLOP/s of 1679, the tensor pipe 29 % busy; the codes come
// from L2 at a tenth of its rate. What bounds it is the converting warps: by
// the clock, 64 keys take them about 3200 cycles, of which they wait 700, while
// the rows compute for 1650 and the products are issued in 700. Two blocks
// share an SM, so one's products run under the other's conversion. Rows that
// run further ahead only take issue slots from the converting warps (P in two
// buffers: 5 % slower; a barrier of their own for the steps: 30 %); half of Q
// in TMEM, which spares the products shared memory: 5 % slower.
#include "ssa_cache_attn.cuh"
#include "ssa_tcgen05.cuh"

namespace ssa {

using namespace tc;

int read_cache_error(int clear) { return tc_read_error(clear); }

namespace {

constexpr int kSoftWarps = 4, kConvWarps = 4, kThreads = (kSoftWarps + kConvWarps + 1) * 32;
constexpr int kConvThreads = kConvWarps * 32;
// Registers: the launch's 96 a thread (9 warps, two blocks an SM) are dealt out
// as 72 to the 128 converting threads and 120 to the 128 with a row:
// 128 * 72 + 128 * 120 + 32 * 96 = 288 * 96.
constexpr uint32_t kTmemCols = 256, kColP = 64, kColO = 128;  // S at 0

// Element (row, channel) of a tile's partial sums: four channels of all rows
// side by side, as a row a thread writes them.
template <int D>
__device__ __forceinline__ int part_at(int row, int ch) { return ((ch >> 2) * kPromptRows + row) * 4 + (ch & 3); }

template <int D>
struct PromptSmem {
  static constexpr int kAtoms = (D + 63) / 64;                         // 64 channels: rows of 128 bytes
  static constexpr int kQ = 0;                                         // [kAtoms][128 rows][128 bytes]
  static constexpr int kTile = kAtoms * 64 * 128;                      // [kAtoms][64 keys][128 bytes]
  static constexpr int kKV = kAtoms * kPromptRows * 128;               // [2 stages][K, V] tiles
  // [2 stages][4] {step_k, log2 step_v, 1 / step_v (negative where V stands for NaN), octaves kept from moving the offset}
  static constexpr int kMeta = kKV + 4 * kTile;
  static constexpr int kBars = kMeta + 2 * 4 * 16;
  static constexpr int kBytes = kBars + 128 + 1024;                    // the base is rounded up to 1024
};

// fp16 A and B, fp32 sums, M x N; B key-major or (transposed) channel-major.
constexpr uint32_t idesc_f16(int m, int n, bool b_transposed) {
  return (1u << 4) | (b_transposed ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// V's operand: the product's N (channels) runs along the 128-byte rows, its K
// (keys) down them: 64-channel atoms `atom` bytes apart, groups of 8 keys 1024.
__device__ __forceinline__ uint64_t desc_channels_inner(uint32_t saddr, uint32_t atom) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(atom >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}

// Bounded wait of a warp: one look, then polls that may sleep in the hardware,
// `limit` in all (mbar_wait's, which reports the one that runs out).
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort, int code, uint32_t limit) {
  uint32_t there;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(there)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  const bool ok = there || mbar_wait(bar, parity, abort, code, limit - 1);
  return __all_sync(0xffffffffu, ok);
}

// D (+)= A B with A in TMEM.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The units of a thread block's range, one after the other (every warp walks
// them for itself).
struct Segments {
  int at, hi, b, base;
  __device__ __forceinline__ Segments(const BlockRange& r) : at(r.lo), hi(r.hi), b(r.b), base(r.base) {}
  __device__ __forceinline__ bool next(const CacheDev& c, const Plan& pl, Unit& x, int& g0, int& g1, int& groups) {
    while (at < hi) {
      int tiles;
      const int mine = seq_work(c, pl, b, kPromptRows, &tiles, &groups);
      if (at >= base + mine) { base += mine; ++b; continue; }
      const int u = (int)((unsigned)(at - base) / (unsigned)groups), ubeg = base + u * groups, uend = ubeg + groups;
      g0 = at - ubeg;
      g1 = min(hi, uend) - ubeg;
      at = ubeg + g1;
      x = unit_of<kPromptRows>(c, pl, b, u, tiles);
      return true;
    }
    return false;
  }
};

// Keys a row of the tile sees: at most `lim_max`; groups of 64 a segment has to visit.
__device__ __forceinline__ int lim_max_of(const CacheDev& c, const Unit& x) {
  return c.causal ? x.start + (x.row0 + x.nrows - 1) / c.rep + 1 : x.len;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2) k_cache_prompt(const CacheDev c, const Plan pl) {
  using Sm = PromptSmem<D>;
  extern __shared__ __align__(16) unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  float4* meta = reinterpret_cast<float4*>(sm + Sm::kMeta);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sm::kBars);
  uint64_t *kfull = bars, *vfull = bars + 2, *kempty = bars + 4, *vempty = bars + 6, *sfull = bars + 8, *sempty = bars + 9,
           *pfull = bars + 10, *odone = bars + 11, *qfull = bars + 12, *mma_done = bars + 13;
  __shared__ RangeSmem rs;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  volatile int* abort_flag = &abort_flag_s;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  grid_wait();
  const BlockRange br(c.B, c.prefix, least_groups(kPromptRows), rs, [&](int i) {
    int tiles, groups;
    return seq_work(c, pl, i, kPromptRows, &tiles, &groups);
  });
  if (br.lo >= br.hi) return;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull + i, kConvWarps);
      mbar_init(vfull + i, kConvWarps);
      mbar_init(kempty + i, 1 + kSoftWarps);
      mbar_init(vempty + i, 1);
    }
    mbar_init(sfull, 1);
    mbar_init(sempty, kSoftWarps);
    mbar_init(pfull, kSoftWarps);
    mbar_init(odone, 1);
    mbar_init(qfull, kSoftWarps);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (w == kSoftWarps + kConvWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  Segments seg(br);
  Unit x;
  int g0, g1, groups;
  int it = 0;  // blocks of 64 keys so far, the same count in every role

  if (w >= kSoftWarps && w < kSoftWarps + kConvWarps) {
    // ------------------------------------------------------------ codes to fp16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int ct = tid - kSoftWarps * 32;
    const int bs_shift = c.bs == 16 ? 4 : c.bs == 32 ? 5 : 6;
    constexpr int kLoads = D / 32;  // 16-byte pieces of a tile's codes a thread has
    bool ok = true;
    while (ok && seg.next(c, pl, x, g0, g1, groups)) {
      const int lim_max = lim_max_of(c, x);
      const int ge = min(g1, (lim_max + 63) / 64);
      // lane l: the table's entry for keys 16 (l % 4) .. of a block
      const auto entry = [&](int gr) {
        const int key = gr * 64 + (lane & 3) * 16;
        return gr < ge && key < lim_max ? cache_entry(c, x.b, key >> bs_shift) : -1;
      };
      // where those keys lie, in units of 16 rows of codes
      const auto place = [&](int gr, int pages) {
        return (uint32_t)(((int64_t)max(pages, 0) * c.n_kv + x.kv) * (c.bs / 16)) + (uint32_t)((gr * 4 + (lane & 3)) & (c.bs / 16 - 1));
      };
      // Piece i of a thread: 16 codes of a row, the id-th of the tile. Eight lanes
      // store 16 bytes at a time: with 128 channels they take four pieces of two
      // rows, whose swizzled chunks are the even and the odd ones of 128 bytes.
      const auto piece_of = [&](int i, int& row, int& part) {
        const int id = i * kConvThreads + ct;
        row = D == 128 ? (id >> 4) * 2 + (id >> 2 & 1) : id / (D / 16);
        part = D == 128 ? (id & 3) + (id >> 3 & 1) * 4 : id % (D / 16);
      };
      const auto load = [&](const int8_t* codes, uint32_t at, uint4 (&r)[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          int row, part;
          piece_of(i, row, part);
          const uint32_t rows = __shfl_sync(0xffffffffu, at, row >> 4);
          r[i] = *reinterpret_cast<const uint4*>(codes + ((uint64_t)rows * (16 * D) + (unsigned)((row & 15) * D + part * 16)));
        }
      };
      const auto store = [&](unsigned char* tile, const uint4 (&r)[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          int row, part;
          piece_of(i, row, part);
          // chunks 2 part, 2 part + 1 of the row (96 channels: the last two pieces' second one first, for the banks)
          const int first = D == 96 ? part >> 2 : 0, c0 = (part & 3) * 2;
          const uint32_t w4[4] = {(first ? r[i].z : r[i].x) ^ 0x80808080u, (first ? r[i].w : r[i].y) ^ 0x80808080u,
                                  (first ? r[i].x : r[i].z) ^ 0x80808080u, (first ? r[i].y : r[i].w) ^ 0x80808080u};
          unsigned char* at = tile + (part >> 2) * (64 * 128) + row * 128;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<uint4*>(at + (((c0 + (first ^ e)) ^ (row & 7)) << 4)) =
                make_uint4(codes_f16<0x4140>(w4[2 * e]), codes_f16<0x4342>(w4[2 * e]), codes_f16<0x4140>(w4[2 * e + 1]),
                           codes_f16<0x4342>(w4[2 * e + 1]));
        }
      };
      int pages = cache_checked(c, entry(g0)), ahead = entry(g0 + 1);
      uint32_t at = place(g0, pages);
      uint4 kr[kLoads], vr[kLoads];
      float2 am = make_float2(0.f, 0.f);
      float4 mt = make_float4(0.f, -INFINITY, 0.f, 0.f);
      const auto steps = [&]() {
        if (w == kSoftWarps && lane < 4) {
          const float va = am.y * (1.f / 127.f);
          const bool plain = va > 0.f && va < INFINITY;
          const float vs = plain ? va : 1.f;
          // keys without a page: scores of minus infinity; a page of K that stands for NaN: scores of NaN;
          // 1 / step to two units of the last place is enough for a sum of weights
          mt = pages >= 0 ? make_float4(am.x * (1.f / 127.f), __log2f(vs), va < INFINITY ? __fdividef(1.f, vs) : -1.f,
                                        plain ? 0.f : kZeroHead)
                          : make_float4(0.f, -INFINITY, 0.f, 0.f);
        }
      };
      const auto load_amax = [&](int pg) {
        return w == kSoftWarps && lane < 4 && pg >= 0
                   ? *(reinterpret_cast<const float2*>(c.amax) + (int64_t)pg * c.n_kv + x.kv) : make_float2(0.f, 0.f);
      };
      if (g0 < ge) {
        load(c.k_codes, at, kr);
        am = load_amax(pages);
        load(c.v_codes, at, vr);
        steps();
      }
      for (int gr = g0; gr < ge; ++gr, ++it) {
        const int st = it & 1;
        unsigned char* tile = sm + Sm::kKV + st * 2 * Sm::kTile;
        if (!(ok = wait_for(kempty + st, ((it >> 1) & 1) ^ 1, abort_flag, 31, c.wait_limit))) break;
        if (w == kSoftWarps && lane < 4) meta[st * 4 + lane] = mt;
        store(tile, kr);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(kfull + st);
        pages = cache_checked(c, ahead);
        ahead = entry(gr + 2);
        at = place(gr + 1, pages);
        if (gr + 1 < ge) {
          load(c.k_codes, at, kr);
          am = load_amax(pages);
        }
        if (!(ok = wait_for(vempty + st, ((it >> 1) & 1) ^ 1, abort_flag, 41, c.wait_limit))) break;
        store(tile + Sm::kTile, vr);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(vfull + st);
        if (gr + 1 < ge) {
          load(c.v_codes, at, vr);
          steps();
        }
      }
    }
  } else if (w == kSoftWarps + kConvWarps) {
    // ------------------------------------------------------------ products
    // The warp stays together and one thread of it issues: addresses and
    // descriptors are then in uniform registers, where the products want them.
    const bool lead = elect_one();
    const auto same = [](auto v) { return __shfl_sync(0xffffffffu, v, 0); };
    const uint32_t tm = same(tmem);
    const uint64_t q_desc = same(umma_desc(smem_u32(sm + Sm::kQ)));
    const uint64_t k_desc = same(umma_desc(smem_u32(sm + Sm::kKV)));
    const uint64_t v_desc = same(desc_channels_inner(smem_u32(sm + Sm::kKV + Sm::kTile), 64 * 128));
    constexpr uint32_t kStage = 2 * Sm::kTile / 16;
    constexpr uint32_t kDescS = idesc_f16(kPromptRows, 64, false), kDescO = idesc_f16(kPromptRows, D, true);
    bool ok = true;
    int segs = 0;
    const auto scores = [&](int i) {
      const int st = i & 1;
      if (!wait_for(kfull + st, (i >> 1) & 1, abort_flag, 32, c.wait_limit)) return false;
      if (i && !wait_for(sempty, (i - 1) & 1, abort_flag, 33, c.wait_limit)) return false;
      tc_fence_after();
      const uint64_t kd = k_desc + (uint32_t)st * kStage;
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16(tm, q_desc + ((kk >> 2) * (kPromptRows * 128) + (kk & 3) * 32) / 16,
                    kd + ((kk >> 2) * (64 * 128) + (kk & 3) * 32) / 16, kDescS, kk > 0);
        umma_commit(sfull);
        umma_commit(kempty + st);
      }
      __syncwarp();
      return true;
    };
    while (ok && seg.next(c, pl, x, g0, g1, groups)) {
      const int nb = same(min(g1, (lim_max_of(c, x) + 63) / 64) - g0);
      if (nb <= 0) continue;
      ok = wait_for(qfull, segs++ & 1, abort_flag, 34, c.wait_limit) && scores(it);
      for (int j = 0; ok && j < nb; ++j, ++it) {
        const int st = it & 1;
        if (j + 1 < nb && !(ok = scores(it + 1))) break;
        ok = wait_for(vfull + st, (it >> 1) & 1, abort_flag, 35, c.wait_limit) &&
             wait_for(pfull, it & 1, abort_flag, 36, c.wait_limit);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = v_desc + (uint32_t)st * kStage;
        if (lead) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts(tm + kColO, tm + kColP + kk * 8, vd + kk * (16 * 128 / 16), kDescO, (j | kk) > 0);
          umma_commit(vempty + st);
          umma_commit(odone);
        }
        __syncwarp();
      }
    }
    // Products still in flight (also after a wait that ran out) end before TMEM is freed.
    if (lead) {
      umma_commit(mma_done);
      mbar_drain(mma_done, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
    const int r = tid;
    const uint32_t trow = tmem + ((uint32_t)(w * 32) << 16);
    bool ok = true;
    while (ok && seg.next(c, pl, x, g0, g1, groups)) {
      const bool have = r < x.nrows;
      const int nb = min(g1, (lim_max_of(c, x) + 63) / 64) - g0;
      const int lim_min = c.causal ? x.start + x.row0 / c.rep + 1 : x.len;
      const int row = x.row0 + (have ? r : 0), tok = row / c.rep, hd = x.kv * c.rep + row - tok * c.rep;
      const int lim = !have ? INT32_MAX : c.causal ? x.start + tok + 1 : x.len;
      // this thread's row in q and out (rows behind the last one: the first, never stored)
      const int64_t q_at = x.b * c.q_sb + hd * c.q_sh + tok * c.q_sn, o_at = x.b * c.o_sb + hd * c.o_sh + tok * c.o_sn;
      // A row behind the last one computes the first row's scores over all keys,
      // stale ones too: its offset is out of reach, so that it moves nothing.
      float m = have ? kEmpty : -kEmpty, l = 0.f;
      bool bad = false;  // the row sees a page of V that stands for NaN: its output is NaN, the weights' sum is K's alone
      if (nb > 0) {
        // Q: rows into their swizzled places as they come, 8 bytes a lane, then
        // each thread turns its own into fp16 where it lies, scaled by a power of
        // two; the scale's sign goes with it.
        const char* q0 = static_cast<const char*>(c.q) + lane * 8;
        const uint32_t qs = smem_u32(sm + Sm::kQ) + (lane >> 4) * (kPromptRows * 128) + (lane & 1) * 8;
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
          const int64_t at = __shfl_sync(0xffffffffu, q_at, i);
          const int rr = w * 32 + i;
          if (lane < D / 4) copy8(qs + rr * 128 + ((((lane >> 1) & 7) ^ (rr & 7)) << 4), q0 + at * 2);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        unsigned char* mine = sm + Sm::kQ + r * 128;
        const auto piece = [&](int i) {
          return reinterpret_cast<uint4*>(mine + (i >> 3) * (kPromptRows * 128) + (((i & 7) ^ (r & 7)) << 4));
        };
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint4 u = *piece(i);
          top = max(top, max(max(max((u.x << 16) & 0x7fffffffu, u.x & 0x7fff0000u), max((u.y << 16) & 0x7fffffffu, u.y & 0x7fff0000u)),
                             max(max((u.z << 16) & 0x7fffffffu, u.z & 0x7fff0000u), max((u.w << 16) & 0x7fffffffu, u.w & 0x7fff0000u))));
        }
        int e = 9 - ((int)(top >> 23) - 127);
        e = top >= 0x7f800000u ? 0 : min(e, 100);
        const float up0 = __uint_as_float((uint32_t)(e + 127) << 23), up = c.scale < 0.f ? -up0 : up0;
        const float sfac = fabsf(c.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - e) << 23);
        const auto half2 = [&](uint32_t u) { return pack_f16(__uint_as_float(u << 16) * up, __uint_as_float(u & 0xffff0000u) * up); };
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 u = *piece(i);
          *piece(i) = make_uint4(half2(u.x), half2(u.y), half2(u.z), half2(u.w));
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);

        for (int j = 0; j < nb; ++j, ++it) {
          const int st = it & 1, key0 = (g0 + j) * 64;
          if (!(ok = wait_for(kfull + st, (it >> 1) & 1, abort_flag, 37, c.wait_limit))) break;  // the steps
          float4 mt[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) mt[k] = meta[st * 4 + k];
          __syncwarp();
          if (lane == 0) mbar_arrive(kempty + st);  // seen: the stage's next phase may come
          if (fminf(fminf(mt[0].z, mt[1].z), fminf(mt[2].z, mt[3].z)) < 0.f) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (mt[k].z < 0.f && key0 + 16 * k < lim) bad = true;
          }
          if (!(ok = wait_for(sfull, it & 1, abort_flag, 38, c.wait_limit))) break;
          tc_fence_after();
          float s[64];
          tmem_ld32(trow, s);
          tmem_ld32(trow + 32, s + 32);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty);

          // scores less the row's offset, in one step; a row without one yet has them whole
          const float m0 = m == kEmpty ? 0.f : m;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float f = mt[k].x * sfac, a = mt[k].y - m0;
            const unsigned long long f2 = f2_pack(f, f), a2 = f2_pack(a, a);
#pragma unroll
            for (int i = 0; i < 16; i += 2)
              f2_unpack(f2_fma(f2_pack(s[k * 16 + i], s[k * 16 + i + 1]), f2, a2), s[k * 16 + i], s[k * 16 + i + 1]);
          }
          if (key0 + 64 > lim_min) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (key0 + i >= lim) s[i] = -INFINITY;
          }
          float mx4[4] = {s[0], s[16], s[32], s[48]};
#pragma unroll
          for (int i = 1; i < 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(mx4[k], s[k * 16 + i]);
#pragma unroll
          for (int k = 0; k < 4; ++k) mx4[k] -= mt[k].w;
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          const bool move = mx > (m == kEmpty ? kEmpty : kHead + kSlack);
          float f = 1.f;
          if (__any_sync(0xffffffffu, move)) {
            const float by = move ? mx - kHead : 0.f;
            if (move) {
              f = m == kEmpty ? 0.f : ex2(-by);
              m = m0 + by;
              l *= f;
            }
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] -= by;
          }
          // weights, fp16; the sum before the rounding
          uint32_t p[32];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            unsigned long long sum2 = 0ull;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float a = ex2(s[k * 16 + i]), e2 = ex2(s[k * 16 + i + 1]);
              sum2 = f2_add(sum2, f2_pack(a, e2));
              p[k * 8 + i / 2] = pack_weights(a, e2);
            }
            float sum0, sum1;
            f2_unpack(sum2, sum0, sum1);
            l = fmaf(sum0 + sum1, fabsf(mt[k].z), l);
          }
          if (j > 0) {
            // the product before has read P and added to O
            if (!(ok = wait_for(odone, (it - 1) & 1, abort_flag, 39, c.wait_limit))) break;
            tc_fence_after();
            if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
              for (int ch = 0; ch < D; ch += 32) {
                float o[32];
                uint32_t u[32];
                tmem_ld32(trow + kColO + ch, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(o[i] * f);
                tmem_st32(trow + kColO + ch, u);
              }
            }
          }
          tmem_st32(trow + kColP, p);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pfull);
        }
        if (ok) {
          ok = wait_for(odone, (it - 1) & 1, abort_flag, 40, c.wait_limit);
          tc_fence_after();
        }
      }
      if (!ok) break;
      const bool full = g0 == 0 && g1 == groups;
      const int64_t slot = ((int64_t)blockIdx.x * 2 + (g0 == 0)) * kPromptRows;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int ch = 0; ch < D; ch += 32) {
        float o[32];
        if (nb > 0) {
          tmem_ld32(trow + kColO + ch, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (!have) continue;
        if (bad)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = NAN;
        if (full) {
          uint16_t* to = static_cast<uint16_t*>(c.out) + o_at + ch;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint2*>(to + i) =
                make_uint2(f32_to_bf16_bits(o[i] * inv) | (uint32_t)f32_to_bf16_bits(o[i + 1] * inv) << 16,
                           f32_to_bf16_bits(o[i + 2] * inv) | (uint32_t)f32_to_bf16_bits(o[i + 3] * inv) << 16);
        } else {
          float* to = c.part_o + slot * D + part_at<D>(r, ch);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(to + i * kPromptRows) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      tc_fence_before();
      if (have) {
        if (!full) *reinterpret_cast<float2*>(c.part_ml + (slot + r) * 2) = make_float2(m, l);
        else if (c.lse) store_lse(c, x, r, m, l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (w == kSoftWarps + kConvWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

// Joins the partial sums of 16 rows of a unit that several blocks worked on, in
// range order, and writes zeros to rows without work: 16 threads have the rows
// side by side, as they lie, each of eight such groups every eighth four
// channels. PARTS groups of 128 threads share the sums where few units have
// many. One set-up serves 16 rows: with k_cache_combine's warp a row the call
// above took 89 us. Batches of two sums leave registers for twice the blocks
// that batches of four do (81 against 85 us).
constexpr int kJoinRows = 16, kJoinThreads = 128;

template <int D, int PARTS>
__global__ void __launch_bounds__(kJoinThreads * PARTS) k_cache_join(const CacheDev c, const Plan pl, const int ngrid) {
  constexpr int E = D / 32, kBatch = 2, kBlocks = kPromptRows / kJoinRows;
  __shared__ __align__(16) float s_o[PARTS][kJoinRows][D + 4];
  __shared__ float2 s_ml[PARTS][kJoinRows];
  const int t = threadIdx.x % kJoinThreads, part = threadIdx.x / kJoinThreads, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int jr = t % kJoinRows, cg = t / kJoinRows;
  const unsigned unit = blockIdx.x / kBlocks, units_b = (unsigned)pl.tiles_max * c.n_kv;
  const int r0 = (int)(blockIdx.x % kBlocks) * kJoinRows;
  const int b = (int)(unit / units_b), u = (int)(unit % units_b);
  // Lengths may be read before the wait: the other kernel lets this one come up
  // only after its own.
  int tiles, groups;
  const int mine = seq_work(c, pl, b, kPromptRows, &tiles, &groups);
  const Unit x = unit_of<kPromptRows>(c, pl, b, u, pl.tiles_max);
  int total = 0, base = 0;
  if (c.B <= 128) {
    for (int i = lane; i < c.B; i += 32) {
      int a, e;
      const int v = seq_work(c, pl, i, kPromptRows, &a, &e);
      total += v;
      base += i < b ? v : 0;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    base = __reduce_add_sync(0xffffffffu, base);
  }
  grid_wait();
  const int rows = min(kPromptRows, c.n * c.rep - x.row0) - r0;  // of this block, in the padded step
  if (rows <= 0) return;
  int c0 = 0, c1 = 0;
  const bool work = x.tile < tiles && mine > 0;
  if (work) {
    if (c.B > 128) {
      total = c.prefix[c.B];
      base = c.prefix[b];
    }
    const int ubeg = base + (x.kv * tiles + x.tile) * groups;
    const Ranges rg(total, ngrid, least_groups(kPromptRows));
    c0 = rg.of(ubeg);
    c1 = rg.of(ubeg + groups - 1);
  }
  const auto joined = [&](int row) { return work && row < x.nrows; };
  if (work && c0 == c1 && r0 + min(rows, kJoinRows) <= x.nrows) return;  // that block stored the rows

  const int r = r0 + jr;
  float m = kEmpty, l = 0.f;
  float4 o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (joined(r) && c0 != c1) {
    const int cnt = (c1 - c0 + PARTS - part) / PARTS;  // sums part, part + PARTS, ...
    const auto slot = [&](int i) {
      const int k = c0 + part + i * PARTS;
      return ((int64_t)k * 2 + (k == c0)) * kPromptRows;
    };
    for (int i = 0; i < cnt; ++i) m = fmaxf(m, c.part_ml[(slot(i) + r) * 2]);
    for (int i0 = 0; i0 < cnt; i0 += kBatch) {
      float4 v[kBatch][E];
      float2 ml[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (i0 + i < cnt) {
          const int64_t s = slot(i0 + i);
          ml[i] = *reinterpret_cast<const float2*>(c.part_ml + (s + r) * 2);
#pragma unroll
          for (int e = 0; e < E; ++e) v[i][e] = *reinterpret_cast<const float4*>(c.part_o + s * D + part_at<D>(r, (cg + 8 * e) * 4));
        }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (i0 + i < cnt) {
          const float f = ex2(ml[i].x - m);
          l = fmaf(f, ml[i].y, l);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            o[e].x = fmaf(f, v[i][e].x, o[e].x);
            o[e].y = fmaf(f, v[i][e].y, o[e].y);
            o[e].z = fmaf(f, v[i][e].z, o[e].z);
            o[e].w = fmaf(f, v[i][e].w, o[e].w);
          }
        }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) *reinterpret_cast<float4*>(&s_o[part][jr][(cg + 8 * e) * 4]) = o[e];
  if (cg == 0) s_ml[part][jr] = make_float2(m, l);
  __syncthreads();

  for (int j = w; j < min(rows, kJoinRows); j += kJoinThreads * PARTS / 32) {
    if (joined(r0 + j) && c0 == c1) continue;
    float mj = kEmpty, lj = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) mj = fmaxf(mj, s_ml[k][j].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      const float f = PARTS == 1 ? 1.f : ex2(s_ml[k][j].x - mj);
      lj = fmaf(f, s_ml[k][j].y, lj);
      if (lane < D / 4) {
        const float4 a = *reinterpret_cast<const float4*>(&s_o[k][j][lane * 4]);
        v = make_float4(fmaf(f, a.x, v.x), fmaf(f, a.y, v.y), fmaf(f, a.z, v.z), fmaf(f, a.w, v.w));
      }
    }
    const float inv = lj == 0.f ? 0.f : 1.f / lj;
    if (lane < D / 4) store_out<false>(c, x, r0 + j, lane * 4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    if (lane == 0 && c.lse) store_lse(c, x, r0 + j, mj, lj);
  }
}

template <int D>
cudaError_t run_prompt(const CacheDev& c, const Plan& pl, cudaStream_t st) {
  constexpr size_t smem = PromptSmem<D>::kBytes;
  cudaError_t e = allow_smem<k_cache_prompt<D>>(smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)c.B * c.n_kv * pl.tiles_max, joins = units * (kPromptRows / kJoinRows);
  if (joins > 0x7fffffff) return cudaErrorInvalidConfiguration;
  CacheLaunch l((unsigned)c.grid, kThreads, smem, st);
  e = cudaLaunchKernelEx(&l.cfg, k_cache_prompt<D>, c, pl);
  note_launch();
  if (e != cudaSuccess) return e;
  const bool wide = c.grid > 16 * units;  // a unit may have more sums than a batch or two
  CacheLaunch j((unsigned)joins, kJoinThreads * (wide ? 4 : 1), 0, st);
  e = wide ? cudaLaunchKernelEx(&j.cfg, k_cache_join<D, 4>, c, pl, c.grid) : cudaLaunchKernelEx(&j.cfg, k_cache_join<D, 1>, c, pl, c.grid);
  note_launch();
  return e;
}

}  // namespace

cudaError_t launch_cache_prompt(const CacheDev& c, const Plan& pl, cudaStream_t st) {
  return c.d == 32 ? run_prompt<32>(c, pl, st) : c.d == 64 ? run_prompt<64>(c, pl, st)
         : c.d == 96 ? run_prompt<96>(c, pl, st) : run_prompt<128>(c, pl, st);
}

}  // namespace ssa
