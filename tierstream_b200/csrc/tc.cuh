// What the tcgen05 kernels share: barriers with bounded waits, TMA loads, the tensor core's instructions and their
// descriptors, and the tensor maps.
#pragma once

#include <cuda.h>

#include <atomic>
#include <cstring>

#include "ops.hpp"

namespace tsb {
namespace ops {
namespace {

constexpr int kBM = 128, kBK = 64;  // a CTA's rows, and a slice of k
constexpr int kABytes = kBM * kBK * 2, kRingBytes = 192 << 10;
constexpr int kMaxStages = 12;
constexpr int kEpiWarps = 8, kThreads = 128 + 32 * kEpiWarps;
constexpr int kStoreBytes = 4096;  // a warp's two store buffers
constexpr int kSmemBytes = 1024 + kRingBytes + kEpiWarps * kStoreBytes + 256;
constexpr unsigned long long kWaitNs = 2000000000ull;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// false: the wait ran out, here or elsewhere in the CTA. A try sleeps in hardware for up to 20 us; the clock is read
// between runs of tries.
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t parity, volatile uint32_t* dead) {
  unsigned long long t0 = 0;
  for (;;) {
    for (int i = 0; i < 256; ++i)
      if (bar_try(b, parity)) return true;
    if (*dead) return false;
    const unsigned long long t = now_ns();
    if (!t0) t0 = t;
    if (t - t0 > kWaitNs) {
      *dead = 1;
      return false;
    }
  }
}
// CG = 2: `bar` may be the peer's
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t b) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// One lane of a whole warp, always the same. The loading and the issuing warp run their loops as whole warps, so that
// addresses and descriptors stay in uniform registers (a loop of one thread spent about 500 clocks a k slice).
__device__ __forceinline__ bool elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Shared memory descriptors, 128-byte swizzle. K-major: 8-row groups 1024 bytes apart. MN-major: a stage holds 64-wide
// chunks of [64 k rows][128 bytes], 8 KiB apart, 8-row groups of k 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, bool mn) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(mn ? 8192 >> 4 : 1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}
// the barrier at this offset, in both CTAs of a pair
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(uint16_t(3))
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  T v[2] = {from_f<T>(a), from_f<T>(b)};
  uint32_t r;
  memcpy(&r, v, 4);
  return r;
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
  static const Encode e = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult r{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  return e;
}

// [slots][rows][cols], boxes of box_rows rows of 128 (an output: 64) swizzled bytes
bool make_map(CUtensorMap* m, int dtype, const void* p, uint64_t cols, uint64_t rows, uint64_t ld, uint64_t slots,
              uint64_t slot_bytes, uint32_t box_rows, bool out = false) {
  const uint32_t size = dtype == TSB_F32 ? 4 : 2;
  const cuuint64_t dims[3] = {cols, rows, slots}, strides[2] = {ld * size, slots > 1 ? slot_bytes : ld * size};
  const cuuint32_t box[3] = {(out ? 64 : 128) / size, box_rows, 1}, one[3] = {1, 1, 1};
  return encoder()(m,
                   dtype == TSB_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                   : dtype == TSB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                   3, const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   out ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The kernel's shared memory, allowed once per kernel and device.
int allow_smem(const void* kernel, std::atomic<uint64_t>& devices) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return int(e);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (devices.load(std::memory_order_acquire) & bit) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_release);
  return int(e);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

}  // namespace
}  // namespace ops
}  // namespace tsb
