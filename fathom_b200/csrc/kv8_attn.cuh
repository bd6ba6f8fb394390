// What the attention kernels over the 8-bit cache share: their arguments, the softmax's units, conversions.
#pragma once
#include "kv8.cuh"

#include <cuda.h>

#include <atomic>

namespace fathom {
namespace kv8 {

constexpr float QSCALE = (float)(1.4426950408889634 / 11.313708498984761);   // log2(e) / sqrt(128): base-2 scores
// (A weight's exponent s + (log2 vs - m + HEAD) is exact to a rounding of s for scores up to 2^24, where whole numbers are
// multiples of their spacing; beyond it a weight may be off by the spacing's power of two.)
constexpr int PART = D + 4;      // floats of a partial result: 128 dims, reference, denominator, padding

// Attention over a whole cache: T queries for each of Hkv * G heads of B sequences.  Strides in elements.
struct Args {
  const void* q;
  int64_t qb, qh, qt;
  void* out;
  int64_t ob, oh, ot;
  const uint8_t* rows;
  const float* scales;
  int64_t cap, end;
  const int64_t* end_dev;         // per sequence, or NULL
  int B, Hkv, G;
  int64_t T;
  float* part;                    // workspace: partial results
  unsigned long long* timeouts;   // counts waits that gave up
  // Set by plan_shares (kv8_line.cuh) where the lengths are known to the host: tiles per CTA, and the distance of two
  // items in the line.  share = 0: the device cuts the line, into shares of at least `least` tiles.
  int share, stride, least;
  int64_t tiles_bh;               // tiles of one row bh, where the host knows them; else 0
  int ctas;                       // of the prompt kernel
  float inv_g, inv_hkv;           // 1 / G, 1 / Hkv for div_small
};

// x / d for 0 <= x < 2^20 from 1 / d: x + 0.5 is half a step of 1 / d away from the next whole number, which the three
// roundings cannot cross.  (Code that runs once is paid for by its instructions' way to the SM: a division has ~25.)
__device__ __forceinline__ int div_small(int x, float inv_d) { return __float2int_rd(((float)x + 0.5f) * inv_d); }

// Tokens of sequence b that exist.
__device__ __forceinline__ int seq_end(const Args& a, int b) {
  int64_t e = a.end_dev ? a.end_dev[b] : a.end;
  e = e > a.cap ? a.cap : e;
  return e > 0 ? (int)e : 0;
}

__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(float x, __half* p) { *p = __float2half_rn(x); }

// 2^x by the special-function unit (2 ulp; results below 2^-126 are 0).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float redux_max(float x) {      // over the warp; NaN if none is a number
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(y) : "f"(x));
  return y;
}

// Lets `kernel` use `smem` bytes of dynamic shared memory on the current device; done: one bit per device that has been told.
template <typename K> int allow_smem(K kernel, int smem, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return FATHOM_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return FATHOM_OK;
}

int sm_count();

// kv8_token.cu: up to TOKEN_ROWS query rows (G * T) per KV head.
constexpr int TOKEN_ROWS = 32;
size_t token_workspace(int64_t BH, int64_t R);
int token_attend(const CUtensorMap& map, Args a, int dtype, cudaStream_t st);
// kv8_prompt.cu: any number of query rows, 256 at a time.
size_t prompt_workspace();
int prompt_attend(const CUtensorMap& map, Args a, int dtype, cudaStream_t st);

}  // namespace kv8
}  // namespace fathom
