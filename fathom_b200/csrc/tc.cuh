// Blackwell building blocks for the attention kernels: mbarriers with bounded waits, TMA tile loads, and the
// fifth-generation tensor cores (tcgen05) with their accumulators in tensor memory.
#pragma once
#include "common.cuh"

namespace fathom {
namespace tc {

constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// ---- mbarriers -----------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t mb, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(mb), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t mb) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(mb) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t mb, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(mb), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t mb, uint32_t parity) {
  uint32_t done;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }\n"
               : "=r"(done)
               : "r"(mb), "r"(parity)
               : "memory");
  return done != 0;
}
// Waits until the phase with this parity completes.  False once *gave_up (shared by the CTA) is set: by this wait
// after WAIT_LIMIT_NS, or by another thread's.  Every role then leaves its loop, so the CTA always ends.
__device__ __forceinline__ bool mbar_wait(uint32_t mb, uint32_t parity, volatile int* gave_up) {
  if (mbar_try(mb, parity)) return true;
  const unsigned long long t0 = now_ns();
  while (!mbar_try(mb, parity)) {
    if (*gave_up) return false;
    if (now_ns() - t0 > WAIT_LIMIT_NS) {
      *gave_up = 1;
      return false;
    }
  }
  return true;
}

// One lane of a converged warp, the same one every time.  Code that issues tensor-core work runs in the whole warp and
// only the instructions themselves in this lane: their operands then stay in uniform registers (moved there one by
// one, they cost more issue time than the products take).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }\n" : "=r"(r));
  return r != 0;
}
// A value that is the same in the whole warp, as the compiler can see.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// ---- proxies -------------------------------------------------------------------------------------
// Orders this thread's shared-memory writes before later reads by the tensor cores and TMA.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory"); }

// Programmatic dependent launch: lets the next kernel of the stream start, and waits for the one before to finish.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void wait_dependency() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// Barrier `id` among `n` threads: waiting, not waiting, and waiting with an OR of a predicate.
__device__ __forceinline__ void named_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int n) {
  asm volatile("bar.arrive %0, %1;\n" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ bool named_or(int id, int n, bool v) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, %2, %3, p; selp.u32 %0, 1, 0, q; }\n"
               : "=r"(r)
               : "r"((uint32_t)v), "r"(id), "r"(n)
               : "memory");
  return r != 0;
}

// ---- TMA -----------------------------------------------------------------------------------------
// A tile of a 3-D tensor map into this CTA's shared memory; x (innermost coordinate, in bytes) is a multiple of 16.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t mb) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(mb)
      : "memory");
}

// ---- tensor memory and matrix instructions ----------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t cols) {   // one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_dst), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {        // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// This thread's loads from tensor memory are complete.  Names their N registers: an asm statement that returns a register
// after the wait is what keeps the uses of its value from being moved before it.
template <int N> __device__ __forceinline__ void wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Shared-memory operand in the 128-byte swizzle, rows (K-major) or K slices (MN-major) of 128 bytes in groups of
// 8 that follow each other at 1024 bytes; `lead` is the distance of the next 128 bytes of a longer MN extent.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead = 16) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         1ull << 46 | 2ull << 61;
}
// fp32 accumulators, M = 128; a_mn / b_mn: the operand is MN-major.  Types: kind::f16 f16 x f16, kind::f8f6f4
// e4m3 x e4m3 (both coded 0) or, a_e5m2, e5m2 x e4m3.
constexpr uint32_t instr(uint32_t N, bool a_mn, bool b_mn, bool a_e5m2 = false) {
  return 1u << 4 | (a_e5m2 ? 1u << 7 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (N >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }\n" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
               : "memory");
}
// A from tensor memory.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }\n" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
               : "memory");
}
// The mbarrier is arrived on once every matrix instruction that this thread issued before has completed.
__device__ __forceinline__ void mma_commit(uint32_t mb) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(mb) : "memory");
}

// 32 lanes x N columns of fp32: thread = lane of its warp's quarter.  Complete after wait_ld / wait_st.
template <int N> struct Tmem;
#define FATHOM_TMEM_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define FATHOM_TMEM_W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
template <> struct Tmem<4> {
  static __device__ __forceinline__ void ld(uint32_t a, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n" : FATHOM_TMEM_R4(r, 0) : "r"(a));
  }
  static __device__ __forceinline__ void st(uint32_t a, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), FATHOM_TMEM_W4(r, 0) : "memory");
  }
};
template <> struct Tmem<8> {
  static __device__ __forceinline__ void ld(uint32_t a, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : FATHOM_TMEM_R4(r, 0), FATHOM_TMEM_R4(r, 4)
                 : "r"(a));
  }
  static __device__ __forceinline__ void st(uint32_t a, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(a),
                 FATHOM_TMEM_W4(r, 0), FATHOM_TMEM_W4(r, 4)
                 : "memory");
  }
};
template <> struct Tmem<16> {
  static __device__ __forceinline__ void ld(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        : FATHOM_TMEM_R4(r, 0), FATHOM_TMEM_R4(r, 4), FATHOM_TMEM_R4(r, 8), FATHOM_TMEM_R4(r, 12)
        : "r"(a));
  }
  static __device__ __forceinline__ void st(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};\n" ::"r"(a),
        FATHOM_TMEM_W4(r, 0), FATHOM_TMEM_W4(r, 4), FATHOM_TMEM_W4(r, 8), FATHOM_TMEM_W4(r, 12)
        : "memory");
  }
};
template <> struct Tmem<32> {
  static __device__ __forceinline__ void ld(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : FATHOM_TMEM_R4(r, 0), FATHOM_TMEM_R4(r, 4), FATHOM_TMEM_R4(r, 8), FATHOM_TMEM_R4(r, 12), FATHOM_TMEM_R4(r, 16),
          FATHOM_TMEM_R4(r, 20), FATHOM_TMEM_R4(r, 24), FATHOM_TMEM_R4(r, 28)
        : "r"(a));
  }
  static __device__ __forceinline__ void st(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(a),
        FATHOM_TMEM_W4(r, 0), FATHOM_TMEM_W4(r, 4), FATHOM_TMEM_W4(r, 8), FATHOM_TMEM_W4(r, 12), FATHOM_TMEM_W4(r, 16),
        FATHOM_TMEM_W4(r, 20), FATHOM_TMEM_W4(r, 24), FATHOM_TMEM_W4(r, 28)
        : "memory");
  }
};
#undef FATHOM_TMEM_R4
#undef FATHOM_TMEM_W4

}  // namespace tc
}  // namespace fathom
