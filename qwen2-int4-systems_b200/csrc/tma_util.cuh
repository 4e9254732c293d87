// TMA tensor maps (host) and mbarrier / bulk-tensor PTX wrappers (device).
//
// Rules this code keeps (sm_100a):
//   * every tiled TMA load starts at an inner coordinate that is a multiple of
//     16 bytes, and the inner box is at most the 128-byte swizzle span;
//   * no cluster-broadcast form of a copy is used anywhere - each CTA loads
//     its own tiles into its own shared memory;
//   * every wait on an mbarrier is bounded; on time-out the kernel records an
//     error code in a device flag and carries on without the data.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/qi4_b200.h"

namespace qi4 {

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// 2-D uint8 / 16-bit tensor map over a row-major [rows][inner] array with a
// [box_rows][box_inner] box. Encodings are cached per (device, address,
// shape, box) and copied out; returns false on failure (error recorded).
bool tensor_map_2d(CUtensorMap* out, const void* base, CUtensorMapDataType dtype, uint64_t inner, uint64_t rows,
                   uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle);
// A row-major byte matrix [rows][row_bytes] (row_bytes a multiple of 128) as a
// 3-D map (128-byte box, row, box index) with 128-byte swizzle: one copy of
// [box_rows rows x boxes_per_copy boxes] lands box-major in shared memory
// (box b of row r at (b * box_rows + r) * 128), the layout of as many 2-D
// [box_rows x 128 B] copies, in one request.
bool tensor_map_row_boxes(CUtensorMap* out, const void* base, uint64_t row_bytes, uint64_t rows, uint32_t box_rows,
                          uint32_t boxes_per_copy);

// The pages of a paged cache (16-bit elements) as a 4-D map (dims, slots of a
// page, KV heads, pages) at the descriptor's strides, with a box of 64 dims x
// box_rows slots and 128-byte swizzle. Encoded anew for every call.
bool tensor_map_pages(CUtensorMap* out, const void* base, const qi4_paged_kv& kv, uint32_t box_rows);

// A [rows][heads][dims] 16-bit array (dims contiguous, strides in elements) as
// a 3-D map (dims, heads, rows) with a box of 64 dims x box_heads x box_rows
// and 128-byte swizzle. Encoded anew for every call.
bool tensor_map_rows3(CUtensorMap* out, const void* base, bool f16, int64_t dims, int64_t heads, int64_t rows,
                      int64_t head_stride, int64_t row_stride, uint32_t box_heads, uint32_t box_rows);

// Device-side error flags (one word per translation unit), read and cleared on
// host. A word may hold reports of a call's inputs (QI4_DEVICE_*) beside this
// bit, which alone says that a wait ran out.
constexpr int kErrWaitTimeout = 1;

// ---------------------------------------------------------------------------
// Device side
// ---------------------------------------------------------------------------

// Time limit for mbarrier waits (global timer, ns): far above any legitimate
// wait, short enough that a lost arrival ends the kernel instead of hanging it.
constexpr uint64_t kWaitLimitNs = 2000000000ull;

__device__ __forceinline__ uint64_t global_timer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Explicit 8- and 16-byte shared-memory accesses on 32-bit shared addresses.
__device__ __forceinline__ void sts128(uint32_t saddr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(saddr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t saddr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(saddr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t saddr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(saddr)
               : "memory");
  return v;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}

// Makes barrier initialisation visible to the async (TMA / tensor core) proxy.
__device__ __forceinline__ void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait: returns false (and sets *err) if the phase did not complete
// within limit_ns.
__device__ __forceinline__ bool mbar_wait_for(uint64_t* bar, uint32_t parity, int* err, uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = global_timer_ns();
  for (;;) {
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    // A wait that already timed out somewhere means the pipeline is broken:
    // give up instead of queueing further time-outs. (Checked here, not
    // before the first spin, so that an ordinary short wait never pays a
    // global-memory round trip.) The word's other bits report inputs and say
    // nothing about the pipeline: a wait that gave up for one of them would
    // let its data be read before it is there.
    if (*reinterpret_cast<volatile int*>(err) & kErrWaitTimeout) return false;
    if (global_timer_ns() - start > limit_ns) break;
  }
  atomicOr(err, kErrWaitTimeout);
  return false;
}

__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* err) {
  return mbar_wait_for(bar, parity, err, kWaitLimitNs);
}

// 2-D tiled bulk tensor load global -> this CTA's shared memory, completing
// `bytes` on `bar`. x is the inner coordinate (elements), y the row.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}

// 2-D tiled bulk tensor store shared -> global (elements outside the tensor
// are not written); completion tracked with the bulk-group mechanism.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_addr(src))
               : "memory");
}
__device__ __forceinline__ void tma_store_commit_and_wait() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Untiled bulk copy global -> this CTA's shared memory (both addresses 16-byte
// aligned, bytes a multiple of 16), completing on `bar`, with an L2
// evict-first policy (data read once per pass, e.g. streamed weights).
__device__ __forceinline__ uint64_t l2_evict_first_policy() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void bulk_load_1d(void* dst, const void* src, uint32_t bytes, uint64_t* bar,
                                             uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::
          "r"(smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}

// Barrier among the first `threads` threads of the CTA (warp-aligned), id > 0.
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// GPU-scope acquire load / release add on a global counter.
__device__ __forceinline__ int ld_acquire_gpu(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void red_release_gpu_add(int* p, int v) {
  asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// Loads that bypass L1 (data written by other SMs during the same kernel).
__device__ __forceinline__ uint4 ld_cg_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_cg_f32(const float* p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

}  // namespace qi4
