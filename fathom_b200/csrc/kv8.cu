// Writing and reading back the 8-bit key/value cache (layout in kv8.cuh).
#include "kv8.cuh"

namespace fathom {
namespace {

constexpr int WT = 128;                       // write threads per (row, block, K or V)
constexpr int EPT = 16;                       // elements per access: 8 threads per 128-element row
constexpr int TPR = D / EPT;                  // threads per row
constexpr int RPP = WT / TPR;                 // rows per pass
constexpr int PASSES = BLK / RPP;             // 4

// 16 consecutive elements as fp32.
__device__ __forceinline__ void load16(const float* p, float (&x)[EPT]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(p + 4 * i);
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}
template <typename T, typename T2> __device__ __forceinline__ void load16_half(const T* p, float (&x)[EPT]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 v = *reinterpret_cast<const uint4*>(p + 8 * i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T2 t = *reinterpret_cast<const T2*>(&w[j]);
      x[8 * i + 2 * j] = (float)t.x;
      x[8 * i + 2 * j + 1] = (float)t.y;
    }
  }
}
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float (&x)[EPT]) {
  load16_half<__nv_bfloat16, __nv_bfloat162>(p, x);
}
__device__ __forceinline__ void load16(const __half* p, float (&x)[EPT]) { load16_half<__half, __half2>(p, x); }

struct WriteArgs {
  const void *K, *V;
  int64_t sb, sh, st;        // strides of K and of V, in elements
  int64_t T, cap, start;
  const int64_t* start_dev;  // per sequence, or NULL
  int Hkv;
  uint8_t* rows;
  float* scales;
};

// One CTA per (block of the written span, row bh, K or V).  Thread = 16 elements of 4 rows, kept in
// registers between the absmax and the conversion, so every input is read once.
template <typename T>
__global__ void __launch_bounds__(WT) kv8_write_kernel(WriteArgs a) {
  __shared__ uint32_t s_max[WT / 32];
  const int64_t bh = blockIdx.y;
  const int b = (int)(bh / a.Hkv), h = (int)(bh % a.Hkv), which = blockIdx.z;
  const int64_t start = a.start_dev ? a.start_dev[b] : a.start;
  if (start < 0 || start >= a.cap) return;
  const int64_t blk = start / BLK + blockIdx.x, tok0 = blk * BLK;
  const int64_t end = start + a.T < a.cap ? start + a.T : a.cap;
  if (tok0 >= end) return;
  const T* src = reinterpret_cast<const T*>(which ? a.V : a.K) + b * a.sb + h * a.sh;
  const int r0 = threadIdx.x / TPR, c0 = threadIdx.x % TPR * EPT;
  float x[PASSES][EPT];
  uint32_t top = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int64_t tok = tok0 + p * RPP + r0;
    if (tok >= start && tok < end) {
      load16(src + (tok - start) * a.st + c0, x[p]);
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) x[p][i] = 0.0f;
    }
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint32_t u = __float_as_uint(x[p][i]) & 0x7FFFFFFFu;   // |x|; the order of the bits is that of the values
      top = max(top, u < 0x7F800000u ? u : 0u);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
  float* scale = a.scales + (bh * (a.cap / BLK) + blk) * 2 + which;
  const int lead = start > tok0 ? (int)(start - tok0) : 0;    // tokens of the block written before
  const float old = lead ? *scale : 0.0f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WT / 32; ++w) top = max(top, s_max[w]);
  const float s = fmaxf(pow2i(kv8_exponent(top)), old);
  const float inv = __uint_as_float(0x7F000000u - __float_as_uint(s));   // 2^-e of s = 2^e
  uint8_t* dst = a.rows + (bh * a.cap + tok0) * KV8_ROW + which * D + c0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + r0;
    if (tok0 + r < start || tok0 + r >= end) continue;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = kv8_encode2(x[p][4 * i] * inv, x[p][4 * i + 1] * inv) |
             kv8_encode2(x[p][4 * i + 2] * inv, x[p][4 * i + 3] * inv) << 16;
    *reinterpret_cast<uint4*>(dst + (int64_t)r * KV8_ROW) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lead && s > old) {                                      // the block's scale grew: round its older codes to it
    const float f = old * inv;
    for (int r = r0; r < lead; r += RPP) {
      uint4* p = reinterpret_cast<uint4*>(dst + (int64_t)r * KV8_ROW);
      const uint4 v = *p;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = kv8_decode2(w[i]), hi = kv8_decode2(w[i] >> 16);
        w[i] = kv8_encode2(lo.x * f, lo.y * f) | kv8_encode2(hi.x * f, hi.y * f) << 16;
      }
      *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

__device__ __forceinline__ void store16(float* p, const float (&x)[EPT]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4*>(p + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&x)[EPT]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void store16(__half* p, const float (&x)[EPT]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 t = __floats2half2_rn(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

constexpr int RT = 256;                       // read threads: 16 tokens per pass
constexpr int RTOK = RT / (2 * TPR);
constexpr int RPASS = 4;

// Thread = 16 codes of 4 tokens; a token's 16 threads cover its key and value halves.
template <typename T>
__global__ void __launch_bounds__(RT) kv8_read_kernel(const uint8_t* __restrict__ rows, const float* __restrict__ scales,
                                                      int64_t cap, int64_t start, int64_t n, T* __restrict__ K,
                                                      T* __restrict__ V) {
  const int64_t bh = blockIdx.y;
  const int c = threadIdx.x % (2 * TPR), which = c / TPR, c0 = c % TPR * EPT;
  const int64_t t0 = (int64_t)blockIdx.x * (RTOK * RPASS) + threadIdx.x / (2 * TPR);
  uint4 v[RPASS];
  float s[RPASS];
#pragma unroll
  for (int p = 0; p < RPASS; ++p) {
    const int64_t t = t0 + p * RTOK;
    if (t < n) {
      v[p] = *reinterpret_cast<const uint4*>(rows + (bh * cap + start + t) * KV8_ROW + c * EPT);
      s[p] = scales[(bh * (cap / BLK) + (start + t) / BLK) * 2 + which];
    }
  }
  T* out = which ? V : K;
#pragma unroll
  for (int p = 0; p < RPASS; ++p) {
    const int64_t t = t0 + p * RTOK;
    if (t >= n) return;
    const uint32_t w[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
    float x[EPT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 lo = kv8_decode2(w[i]), hi = kv8_decode2(w[i] >> 16);
      x[4 * i] = lo.x * s[p], x[4 * i + 1] = lo.y * s[p], x[4 * i + 2] = hi.x * s[p], x[4 * i + 3] = hi.y * s[p];
    }
    store16(out + (bh * n + t) * D + c0, x);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace fathom

using namespace fathom;

extern "C" int fathom_kv8_write(const void* K, const void* V, int dtype, int64_t B, int64_t Hkv, int64_t T,
                                int64_t stride_b, int64_t stride_h, int64_t stride_t, int64_t start,
                                const int64_t* start_dev, int64_t cap, uint8_t* rows, float* scales, void* stream) {
  FATHOM_REQUIRE(K && V && rows && scales, FATHOM_ERR_NULL, "kv8_write: NULL pointer");
  FATHOM_REQUIRE(dtype >= FATHOM_DTYPE_F32 && dtype <= FATHOM_DTYPE_F16, FATHOM_ERR_UNSUPPORTED,
                 "kv8_write: dtype must be fp32, bf16 or fp16");
  FATHOM_REQUIRE(B >= 1 && Hkv >= 1 && B <= 65535 && Hkv <= 65535 && B * Hkv <= 65535 && T >= 0 && cap >= BLK &&
                     cap % BLK == 0 && cap <= KV8_MAX_CAP, FATHOM_ERR_SHAPE,
                 "kv8_write: need B*Hkv in 1..65535, T >= 0 and cap a multiple of 64 up to 2^30");
  FATHOM_REQUIRE(start_dev || (start >= 0 && T <= cap && start <= cap - T), FATHOM_ERR_SHAPE,
                 "kv8_write: tokens [%lld, %lld + %lld) exceed the cache's %lld", (long long)start, (long long)start,
                 (long long)T, (long long)cap);
  const int64_t per16 = dtype == FATHOM_DTYPE_F32 ? 4 : 8;
  FATHOM_REQUIRE(aligned16(K) && aligned16(V) && aligned16(rows) && stride_b % per16 == 0 && stride_h % per16 == 0 &&
                     stride_t % per16 == 0, FATHOM_ERR_SHAPE,
                 "kv8_write: K, V (with their strides) and the rows must be 16-byte aligned");
  if (T == 0) return FATHOM_OK;
  const int64_t span = T < cap ? T : cap;    // a device start may leave fewer
  const int64_t nb = start_dev ? cdiv(span + BLK - 1, BLK) : (start + T - 1) / BLK - start / BLK + 1;
  const WriteArgs a{K, V, stride_b, stride_h, stride_t, T, cap, start, start_dev, (int)Hkv, rows, scales};
  const dim3 grid((unsigned)nb, (unsigned)(B * Hkv), 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FATHOM_DTYPE_F32) kv8_write_kernel<float><<<grid, WT, 0, st>>>(a);
  else if (dtype == FATHOM_DTYPE_BF16) kv8_write_kernel<__nv_bfloat16><<<grid, WT, 0, st>>>(a);
  else kv8_write_kernel<__half><<<grid, WT, 0, st>>>(a);
  return check_launch("kv8_write");
}

extern "C" int fathom_kv8_read(const uint8_t* rows, const float* scales, int64_t BH, int64_t cap, int64_t start, int64_t n,
                               int dtype, void* K, void* V, void* stream) {
  FATHOM_REQUIRE(rows && scales && K && V, FATHOM_ERR_NULL, "kv8_read: NULL pointer");
  FATHOM_REQUIRE(dtype >= FATHOM_DTYPE_F32 && dtype <= FATHOM_DTYPE_F16, FATHOM_ERR_UNSUPPORTED,
                 "kv8_read: dtype must be fp32, bf16 or fp16");
  FATHOM_REQUIRE(BH >= 1 && BH <= 65535 && cap >= BLK && cap % BLK == 0 && cap <= KV8_MAX_CAP && start >= 0 && n >= 0 &&
                     n <= cap && start <= cap - n, FATHOM_ERR_SHAPE,
                 "kv8_read: tokens [%lld, %lld + %lld) of a cache of %lld, BH = %lld", (long long)start, (long long)start,
                 (long long)n, (long long)cap, (long long)BH);
  FATHOM_REQUIRE(aligned16(rows) && aligned16(K) && aligned16(V), FATHOM_ERR_SHAPE,
                 "kv8_read: rows, K and V must be 16-byte aligned");
  if (n == 0) return FATHOM_OK;
  const dim3 grid((unsigned)cdiv(n, RTOK * RPASS), (unsigned)BH);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FATHOM_DTYPE_F32)
    kv8_read_kernel<<<grid, RT, 0, st>>>(rows, scales, cap, start, n, (float*)K, (float*)V);
  else if (dtype == FATHOM_DTYPE_BF16)
    kv8_read_kernel<<<grid, RT, 0, st>>>(rows, scales, cap, start, n, (__nv_bfloat16*)K, (__nv_bfloat16*)V);
  else
    kv8_read_kernel<<<grid, RT, 0, st>>>(rows, scales, cap, start, n, (__half*)K, (__half*)V);
  return check_launch("kv8_read");
}
