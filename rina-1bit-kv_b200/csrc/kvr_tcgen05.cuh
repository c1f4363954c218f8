// tcgen05, TMA and mbarrier helpers of the kernels that feed the tensor cores from
// shared memory, and the encoding of their tensor maps.
#pragma once

#include <cuda.h>

#include "kvr_common.cuh"

namespace kvr {

// ---------------------------------------------------------------- tcgen05 ----

// Shared-memory matrix descriptors with 128-byte swizzle, as a low word to
// which an address step >> 4 can be added (addresses stay below 2^18) and a
// constant high word.
// K-major operands: 8-row atoms of 1 KB, 1 KB apart.
constexpr uint32_t kTcDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc_desc_k(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint64_t tc_desc(uint32_t lo) { return ((uint64_t)kTcDescHi << 32) | lo; }
// D (+)= A B^T, both operands in shared memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// One lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool tc_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
// A value that is the same in all lanes, in a form the compiler knows to be:
// MMA descriptors live in uniform registers, and moving each one there from
// per-lane registers made an MMA cost 95 to 160 cycles to issue instead of 64.
__device__ __forceinline__ uint32_t tc_uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tc_ld32(uint32_t taddr, float *f) {
  uint32_t *r = reinterpret_cast<uint32_t *>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, float *f) {
  uint32_t *r = reinterpret_cast<uint32_t *>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// ---------------------------------------------------------------- waiting ----

__device__ __forceinline__ void tc_bar_init(uint64_t *bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ bool tc_wait(uint64_t *bar, unsigned phase, volatile int *abort_s) {
#pragma unroll 1
  for (uint32_t it = 0; !mbar_try_wait(bar, phase); ++it)
    if (it >= kSpinLimit || *abort_s) return false;
  return true;
}
// All lanes go on, or none does.
__device__ __forceinline__ bool tc_wait_warp(uint64_t *bar, unsigned phase, volatile int *abort_s) {
  return __all_sync(~0u, tc_wait(bar, phase, abort_s));
}
// The issuing warps' wait: returns in any case, and a wait that gives up only raises the abort flag.  No lane
// takes another path by its own outcome, so the lanes cannot part (some in a shuffle that the others have left):
// they go on issuing, within the CTA's own memory, and leave together at the piece's end, by a vote on the flag.
// (A vote at each wait instead made a chunk of 512 at 32256 4 % slower.)
__device__ __forceinline__ void tc_wait_on(uint64_t *bar, unsigned phase, volatile int *abort_s, unsigned *err) {
#pragma unroll 1
  for (uint32_t it = 0; !mbar_try_wait(bar, phase) && !*abort_s; ++it)
    if (it >= kSpinLimit) {
      atomicOr(err, 1u);
      *abort_s = 1;
    }
}
__device__ __forceinline__ void tc_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ------------------------------------------------------------------- host ----

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// The driver's calls need a context in the calling thread; a thread that has made no runtime call with a device yet
// (its memory came from a cache) has none.
inline void bind_context() {
  static thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != bound && cudaSetDevice(dev) == cudaSuccess) bound = dev;
}

// A tensor of 16-bit values with dims[0] = 64 channels (one swizzle row);
// strides (bytes) and boxes of the other dimensions follow.
inline bool make_map(CUtensorMap *m, int dtype, const void *base, int rank, const cuuint64_t *dims,
                     const cuuint64_t *strides, const cuuint32_t *box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  return encode_tiled()(m, dtype == KVR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace kvr
