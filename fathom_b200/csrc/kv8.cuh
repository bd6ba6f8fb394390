// 8-bit key/value cache: layout and conversions shared by its kernels (kv8.cu, kv8_attn.cu).
//
//   rows    [BH][cap][2][128] uint8   e4m3 codes of a token's key (0) and value (1): one 256-byte row per token
//   scales  [BH][cap/64][2]   fp32    a power of two per 64-token block, for its keys and for its values
//   value = code * scale
//
// K and V of a token are adjacent because every reader wants both: a picked row is one 256-byte read (host
// link included), and a 128-byte half is one 128-byte-swizzle row of a tensor-core operand.  The scales
// are powers of two, so a block whose scale grows while tokens are appended re-rounds only codes that
// become e4m3 subnormals, a dequantised value is exact in bf16, and a scale folded into a score is exact.
#pragma once
#include "common.cuh"
#include "tc.cuh"

#include <cuda_fp8.h>

namespace fathom {

constexpr int KV8_ROW = 2 * D;          // bytes of one token's key and value codes
constexpr int64_t KV8_MAX_CAP = 1 << 30;      // tokens: positions and tile ends fit 32 bits
constexpr int KV8_EMIN = -120, KV8_EMAX = 120;   // 2^e and 2^-e are normal fp32 numbers

// Smallest e in [KV8_EMIN, KV8_EMAX] with amax <= 448 * 2^e, from the bits of amax (finite, >= 0): 448 is
// 1.75 * 2^8, so the exponent of amax less 8, one more when its mantissa is above 1.75.
__device__ __forceinline__ int kv8_exponent(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < KV8_EMIN ? KV8_EMIN : (e > KV8_EMAX ? KV8_EMAX : e);
}

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e in [-126, 127]

// Two values already divided by their scale (|y| <= 448 or not finite) to two codes, to nearest even.  The
// hardware conversion saturates infinities, so they are turned into NaN first.
__device__ __forceinline__ uint32_t kv8_encode2(float y0, float y1) {
  if (fabsf(y0) == INFINITY) y0 = __uint_as_float(0x7FFFFFFFu);
  if (fabsf(y1) == INFINITY) y1 = __uint_as_float(0x7FFFFFFFu);
  return __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
}

// Two codes to fp32 (exact).
__device__ __forceinline__ float2 kv8_decode2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Launches a kernel that may start while the one before it in the stream still ends: every thread
// calls tc::wait_dependency() before it touches memory or returns (so a kernel that has ended says that those before it have).  No
// pointer is __restrict__: a load of memory declared constant could be moved before the wait.
template <typename K, typename... A>
int launch_after(K kernel, dim3 grid, int threads, int smem, cudaStream_t st, const char* what, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace fathom
