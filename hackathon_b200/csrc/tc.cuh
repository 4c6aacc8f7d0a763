// tcgen05 (5th-generation tensor core) building blocks of the prompt-side
// kernels (fp8_gemm.cu, scan_tc.cu): shared-memory descriptors, the MMA and its
// commit, TMEM loads and stores, TMA tile loads and their host-side maps.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "mbarrier.cuh"

namespace b2e {
namespace tc {

// Tile load; (x, y) = (inner, row) coordinates, x * element size a multiple of 16.
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Descriptor of a K-major operand: rows of 128 bytes, 128-byte swizzle, 8-row
// atoms 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}

// One lane of a converged warp. MMAs and commits are issued under it in code that
// the whole warp runs, which leaves their descriptors in uniform registers: under
// a test of the lane instead, each MMA of a chain took 100 to 200 cycles to issue
// against the 32 to 128 it runs.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Descriptors `bytes` further on (the address is the low field, in 16 bytes).
__device__ __forceinline__ uint64_t desc_at(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One whole warp each.
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}

#define B2E_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define B2E_R16(r, i) B2E_R4(r, i), B2E_R4(r, i + 4), B2E_R4(r, i + 8), B2E_R4(r, i + 12)
#define B2E_I4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
#define B2E_I16(r, i) B2E_I4(r, i), B2E_I4(r, i + 4), B2E_I4(r, i + 8), B2E_I4(r, i + 12)

// N consecutive 32-bit columns of this thread's TMEM lane; tmem_wait_ld() before
// the values are used.
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : B2E_R16(r, 0)
      : "r"(t));
}
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : B2E_R16(r, 0), B2E_R16(r, 16)
      : "r"(t));
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::B2E_I4(r, 0), B2E_I4(r, 4), "r"(t)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::B2E_I16(
          r, 0),
      "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Register values that an asynchronous TMEM load filled: keeps their uses below
// the wait.
template <int N>
__device__ __forceinline__ void landed(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// ---- host
// Lets a kernel take `bytes` of shared memory, once a device (`done`: a bit each of
// the first 64).
template <class F>
inline void allow_smem(F* kernel, size_t bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  B2E_CUDA(cudaGetDevice(&dev));
  const unsigned long long bit = 1ULL << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return;
  B2E_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  if (dev < 64) done.fetch_or(bit, std::memory_order_acq_rel);
}

// A [rows, inner] tensor of elements of `size` bytes, row stride ld
// elements (a multiple of 16 bytes), read in tiles of box_inner x box_rows with
// the 128-byte swizzle; elements outside read as zero.
void make_map(CUtensorMap* m, CUtensorMapDataType type, int size, const void* base, uint64_t inner, uint64_t rows,
              uint64_t ld, uint32_t box_inner, uint32_t box_rows);

}  // namespace tc
}  // namespace b2e
