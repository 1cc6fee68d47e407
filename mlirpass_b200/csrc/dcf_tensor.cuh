// dcf_tensor.cuh — what the kernels that feed the tensor cores share: PTX
// wrappers for pairs of CTAs and TMEM, the tensor-map encoder, and the launch.
#pragma once

#include <cuda.h>

#include <mutex>

#include "dcf_kernels.cuh"

namespace dcf {

// Products are made by pairs of CTAs (clusters of two): one instruction
// multiplies what both have loaded, into the TMEM of both.
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on this barrier of both CTAs once the products issued before are done.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// Into this CTA's memory; the bytes are reported to a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Arrives on the first CTA's barrier, from either.  A barrier operation that names no scope orders within its own
// CTA only, so these, and the waits for them, name the cluster.  Tensor memory is ordered by the tcgen05 fences
// around them and needs no more.  What shared memory holds (PUBLISH) is released here and acquired by pair_acquire,
// for which a thread waits: warps that have nothing else to do take that on themselves.  (48 x 16384 x 4095 with
// a weight that threads read: 51 us where each of them releases and the thread that issues products acquires, 34 us
// so; the gradient of 8192 x 4096 x 4096, where TMEM alone is handed over: 402 and 275 us.)
template <bool PUBLISH> __device__ __forceinline__ void arrive_first(uint64_t* bar) {
  const uint32_t at = smem_addr(bar);
  if constexpr (PUBLISH)
    asm volatile(
        "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, 0;\n"
        " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n}\n" ::"r"(at)
        : "memory");
  else
    asm volatile(
        "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, 0;\n"
        " mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [r];\n}\n" ::"r"(at)
        : "memory");
}

// Bounded wait for phase `parity` of a barrier at which both CTAs arrive, like mbar_wait_bounded.
__device__ __forceinline__ bool pair_wait(uint64_t* bar, unsigned parity) {
  const uint32_t at = smem_addr(bar);
  for (long spins = 0; spins <= kWaitLimit; spins++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(at), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

// Until the loads issued before have arrived; `r` is named so that no use of it moves ahead.
template <int N> __device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < N; j++) asm volatile("" : "+r"(r[j]));
}
// Two f32 values to an instruction, each rounded as by itself.  (A packed sum
// after a packed product would be fused with it, whatever rounding is written.)
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// 384 threads start with 168 registers each; the first four warps keep 40 and
// the eight that add up get 232: 128 * 40 + 256 * 232 = 384 * 168.
__device__ __forceinline__ void shrink_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 40;"); }
__device__ __forceinline__ void grow_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 232;"); }

// Bounded wait for phase `parity` of `bar`, like mbar_wait_bounded, but the
// thread sleeps for up to a microsecond at a time: warps that look again at
// once take issue slots from those that have something to do.
constexpr int kParkLimit = 1 << 20;
__device__ __forceinline__ bool mbar_wait_parked(uint64_t* bar, unsigned parity) {
  const uint32_t at = smem_addr(bar);
  for (int turns = 0; turns < kParkLimit; turns++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(at), "r"(parity), "r"(1000)
        : "memory");
    if (ok) return true;
  }
  return false;
}

// The same for barriers at which both CTAs arrive; pair_acquire sees what was published.
__device__ __forceinline__ bool pair_wait_parked(uint64_t* bar, unsigned parity) {
  const uint32_t at = smem_addr(bar);
  for (int turns = 0; turns < kParkLimit; turns++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(at), "r"(parity), "r"(1000)
        : "memory");
    if (ok) return true;
  }
  return false;
}

__device__ __forceinline__ bool pair_acquire(uint64_t* bar, unsigned parity) {
  const uint32_t at = smem_addr(bar);
  for (int turns = 0; turns < kParkLimit; turns++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(at), "r"(parity), "r"(1000)
        : "memory");
    if (ok) return true;
  }
  return false;
}

// Whether phase `parity` of `bar` is over.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, unsigned parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// The same for a barrier at which both CTAs arrive.
__device__ __forceinline__ bool pair_test(uint64_t* bar, unsigned parity) {
  const uint32_t at = smem_addr(bar);
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(at), "r"(parity)
      : "memory");
  return ok != 0;
}

// A place in a ring of S stages and the parity of its turn.  Stepped, not
// divided out: the one thread that issues products would spend as long on
// that as four products take.
template <int S> struct Ring {
  int s = 0;
  unsigned turn = 0;
  __device__ __forceinline__ void next() {
    if (++s == S) {
      s = 0;
      turn ^= 1;
    }
  }
  // The place n <= S steps before this one.
  __device__ __forceinline__ Ring back(int n) const {
    Ring r = *this;
    r.s -= n;
    if (r.s < 0) {
      r.s += S;
      r.turn ^= 1;
    }
    return r;
  }
};

// ---------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encoder() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiled)p;
    cudaGetLastError();
  });
  return fn;
}

// Launches as a programmatic dependent (unless DCF_PDL=0): the kernel's start overlaps
// the end of the one before it, whose results it reads only after griddepcontrol.wait.
template <class... P, class... A>
int launch(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  cudaLaunchAttribute a[2];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  a[1].id = cudaLaunchAttributeClusterDimension;
  a[1].val.clusterDim.x = (unsigned)cluster;
  a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
  c.attrs = a;
  c.numAttrs = cluster > 1 ? 2 : 1;
  note_launch();
  return cudaLaunchKernelEx(&c, kernel, args...) == cudaSuccess ? DCF_OK : DCF_ECUDA;
}

}  // namespace dcf
