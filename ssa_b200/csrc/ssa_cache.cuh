// ssa_cache.cuh -- the 8-bit block cache's device parameter block and the
// code paths its kernels share (ssa_cache.cu, ssa_cache_attn.cu).
#pragma once

#include <atomic>

#include "ssa_common.cuh"
#include "ssa_internal.h"

namespace ssa {

// Every kernel here is launched while the one before it in the stream may
// still run, and waits for its end -- with it everything that one waited for
// -- before it reads anything; then it lets the next one come up. Loads are
// plain ones: a read-only load might be moved above the wait.
// Two kernels read before their wait: k_cache_combine and k_cache_join take
// start and lens while the attention they join still runs. That is sound only
// because they are launched directly behind it and it lets them come up after
// its own wait, so launch_dependents has to stay behind the wait.
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launch attributes of these kernels: programmatic dependency on the launch
// before, and a cluster size.
struct CacheLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  CacheLaunch(unsigned grid, unsigned threads, size_t smem, cudaStream_t st, unsigned cluster = 1) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
  }
};

__device__ __forceinline__ unsigned long long f2_add(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Lets kernel K use `bytes` of dynamic shared memory, once on each device (the
// call takes a third of a launch's time).
template <auto K>
inline cudaError_t allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Tokens of sequence b's current step (q rows / appended tokens that count).
__device__ __forceinline__ int cache_step_tokens(const CacheDev& c, int b, int& start, int& len) {
  start = c.start[b];
  len = c.lens[b];
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
  const int page = c.table[(int64_t)b * c.max_blocks + blk];
  return (unsigned)page < (unsigned)c.num_pages ? page : -1;
}

// The same in two steps, for a look-up ahead: the table's entry, and the
// check, made only where the entry is used (it waits for the load).
__device__ __forceinline__ int cache_entry(const CacheDev& c, int b, int blk) {
  return blk >= 0 && blk < c.max_blocks ? c.table[(int64_t)b * c.max_blocks + blk] : -1;
}
__device__ __forceinline__ int cache_checked(const CacheDev& c, int entry) {
  return (unsigned)entry < (unsigned)c.num_pages ? entry : -1;
}

// A staged tile: 16 key rows of D code bytes, as 16-byte chunks exchanged
// within 128 bytes so that the eight rows of an 8x8 tile lie in eight banks
// of 16 bytes (rows of 96 bytes are spaced as rows of 128).
template <int D>
constexpr int kPitch = D == 96 ? 128 : D;
template <int D>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  constexpr int kRows = 128 / kPitch<D>;  // rows in 128 bytes
  return row * kPitch<D> + ((chunk ^ (row / kRows & (kPitch<D> / 16 - 1))) << 4);
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

}  // namespace ssa
