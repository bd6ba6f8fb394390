// Writing and reading back the 8-bit key/value cache (layout in kv8.cuh).
#include "kv8.cuh"

#include <type_traits>

namespace fathom {
namespace {

constexpr int WT = 128;                       // write threads per (row, block, K or V)
constexpr int EPT = 16;                       // elements per access: 8 threads per 128-element row
constexpr int TPR = D / EPT;                  // threads per row
constexpr int RPP = WT / TPR;                 // rows per pass
constexpr int PASSES = BLK / RPP;             // 4

// 16 consecutive elements as they were loaded.
template <typename T> struct Raw {
  uint4 v[EPT * sizeof(T) / 16];
};
template <typename T> __device__ __forceinline__ float2 pair(const Raw<T>& r, int i) {   // elements 2i, 2i + 1
  if constexpr (sizeof(T) == 4) {
    const float2* p = reinterpret_cast<const float2*>(&r.v[i / 2]);
    return p[i & 1];
  } else {
    const uint4& q = r.v[i / 4];
    const uint32_t w = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else
      return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Bits of the largest |x| as fp32, 16-bit elements two at a time: the order of the bits is that of the values, with
// infinity and NaN above all numbers.
template <typename T> __device__ __forceinline__ uint32_t largest(const Raw<T>* r, int n) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 4) {
    for (int k = 0; k < n; ++k)
#pragma unroll
      for (int i = 0; i < EPT / 4; ++i) {
        const uint4 v = r[k].v[i];
        top = __vimax3_u32(top, __vimax3_u32(v.x & 0x7FFFFFFFu, v.y & 0x7FFFFFFFu, v.z & 0x7FFFFFFFu), v.w & 0x7FFFFFFFu);
      }
    return top;
  } else {
    for (int k = 0; k < n; ++k)
#pragma unroll
      for (int i = 0; i < EPT / 8; ++i) {
        const uint4 v = r[k].v[i];
        top = __vimax3_u16x2(top, v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu);
        top = __vimax3_u16x2(top, v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu);
      }
    top = max(top & 0xFFFFu, top >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return top << 16;
    else return top >= 0x7C00u ? 0x7F800000u : __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  }
}

struct WriteArgs {
  const void *K, *V;
  int64_t sb, sh, st;        // strides of K and of V, in elements
  int64_t T, cap, start;
  const int64_t* start_dev;  // per sequence, or NULL
  int Hkv;
  uint8_t* rows;
  float* scales;
};

// One CTA per (block of the written span, row bh, K or V).  Thread = 16 elements of 4 rows, kept as they are in
// registers between the absmax and the conversion, so every input is read once.
//
// Bound by HBM: a bf16 element is 2 bytes read, 1 written.  The conversion is kept to ~3 instructions an element
// (packed maximum, no test for infinities unless the block has one): at ~8 its issue showed, 200 us for 128k tokens of
// 8 KV heads in bf16.  Measured: 117-128 us, 6.3-6.9 TB/s, the copy rate (token-major input 138).  One token:
// 1.7-1.9 us in a graph, launch and latency.
template <typename T>
__global__ void __launch_bounds__(WT) kv8_write_kernel(WriteArgs a) {
  __shared__ uint32_t s_max[WT / 32];
  tc::launch_dependents();
  tc::wait_dependency();
  const int64_t bh = blockIdx.y;
  const int b = (int)bh / a.Hkv, h = (int)bh % a.Hkv, which = blockIdx.z;
  const int64_t start = a.start_dev ? a.start_dev[b] : a.start;
  if (start < 0 || start >= a.cap) return;
  const int64_t blk = start / BLK + blockIdx.x, tok0 = blk * BLK;
  const int64_t end = start + a.T < a.cap ? start + a.T : a.cap;
  if (tok0 >= end) return;
  // rows of the block that are written: [lead, stop); those before were written earlier
  const int lead = start > tok0 ? (int)(start - tok0) : 0, stop = end - tok0 < BLK ? (int)(end - tok0) : BLK;
  const T* src = reinterpret_cast<const T*>(which ? a.V : a.K) + b * a.sb + h * a.sh + (tok0 - start) * a.st;
  const int r0 = threadIdx.x / TPR, c0 = threadIdx.x % TPR * EPT;
  float* scale = a.scales + (bh * (a.cap / BLK) + blk) * 2 + which;
  const float old = lead ? *scale : 0.0f;
  Raw<T> x[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + r0;
#pragma unroll
    for (int i = 0; i < (int)(EPT * sizeof(T) / 16); ++i)
      x[p].v[i] = r >= lead && r < stop ? reinterpret_cast<const uint4*>(src + r * a.st + c0)[i] : make_uint4(0, 0, 0, 0);
  }
  uint32_t top = largest(x, PASSES);
  const bool odd = __syncthreads_or(top >= 0x7F800000u);      // an infinity or NaN somewhere in the block
  if (odd) {
    top = 0;
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int i = 0; i < EPT / 2; ++i) {
        const float2 y = pair(x[p], i);
        const uint32_t u = __float_as_uint(y.x) & 0x7FFFFFFFu, v = __float_as_uint(y.y) & 0x7FFFFFFFu;
        top = max(top, max(u < 0x7F800000u ? u : 0u, v < 0x7F800000u ? v : 0u));
      }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WT / 32; ++w) top = max(top, s_max[w]);
  const float s = fmaxf(pow2i(kv8_exponent(top)), old);
  const float inv = __uint_as_float(0x7F000000u - __float_as_uint(s));   // 2^-e of s = 2^e
  const float2 inv2 = make_float2(inv, inv);
  uint8_t* dst = a.rows + (bh * a.cap + tok0) * KV8_ROW + which * D + c0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + r0;
    if (r < lead || r >= stop) continue;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      const float2 y = __fmul2_rn(pair(x[p], i), inv2);
      const uint32_t c = odd ? kv8_encode2(y.x, y.y) : __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
      w[i / 2] = i & 1 ? w[i / 2] | c << 16 : c;
    }
    *reinterpret_cast<uint4*>(dst + r * KV8_ROW) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lead && s > old) {                                      // the block's scale grew: round its older codes to it
    const float f = old * inv;
    for (int r = r0; r < lead; r += RPP) {
      uint4* p = reinterpret_cast<uint4*>(dst + r * KV8_ROW);
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

// Values of 16 bytes of output: 4 codes to fp32, 8 codes to 16 bits.
__device__ __forceinline__ uint4 values16(uint32_t w, float s, float) {
  const float2 lo = kv8_decode2(w), hi = kv8_decode2(w >> 16);
  return make_uint4(__float_as_uint(lo.x * s), __float_as_uint(lo.y * s), __float_as_uint(hi.x * s),
                    __float_as_uint(hi.y * s));
}
template <typename T> __device__ __forceinline__ uint32_t two_values(uint32_t c, float s) {
  const float2 x = kv8_decode2(c);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(x.x * s, x.y * s);
    return *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const __half2 y = __floats2half2_rn(x.x * s, x.y * s);
    return *reinterpret_cast<const uint32_t*>(&y);
  }
}
template <typename T> __device__ __forceinline__ uint4 values16(uint2 w, float s, T) {
  return make_uint4(two_values<T>(w.x, s), two_values<T>(w.x >> 16, s), two_values<T>(w.y, s), two_values<T>(w.y >> 16, s));
}

constexpr int RT = 256;                       // read threads
constexpr int RPASS = 4;

// Thread = 16 bytes of output at a time, so that every store of a warp is one contiguous stretch (with 16 codes a thread
// the fp32 stores were 64 bytes apart: 69% of the copy rate).  Bound by HBM: a code read, 2 or 4 bytes written.
// Measured, 128k tokens of 8 KV heads: to bf16 122 us, 6.6 TB/s; to fp32 207 us, 6.5 TB/s; the copy rate.
template <typename T>
__global__ void __launch_bounds__(RT) kv8_read_kernel(const uint8_t* rows, const float* scales, int64_t cap, int64_t start,
                                                      int64_t n, T* K, T* V) {
  using Codes = std::conditional_t<sizeof(T) == 4, uint32_t, uint2>;
  constexpr int E = sizeof(Codes), PER = KV8_ROW / E;        // codes of a thread; threads per token
  constexpr int TOK = RT / PER;                              // tokens per pass
  tc::launch_dependents();
  tc::wait_dependency();
  const int64_t bh = blockIdx.y;
  const int c = threadIdx.x % PER, which = c / (PER / 2);
  const int64_t t0 = (int64_t)blockIdx.x * (TOK * RPASS) + threadIdx.x / PER;
  Codes v[RPASS];
  float s[RPASS];
#pragma unroll
  for (int p = 0; p < RPASS; ++p) {
    const int64_t t = t0 + p * TOK;
    if (t < n) {
      v[p] = *reinterpret_cast<const Codes*>(rows + (bh * cap + start + t) * KV8_ROW + c * E);
      s[p] = scales[(bh * (cap / BLK) + (start + t) / BLK) * 2 + which];
    }
  }
  T* out = (which ? V : K) + c % (PER / 2) * E;
#pragma unroll
  for (int p = 0; p < RPASS; ++p) {
    const int64_t t = t0 + p * TOK;
    if (t >= n) return;
    *reinterpret_cast<uint4*>(out + (bh * n + t) * D) = values16(v[p], s[p], T());
  }
}

template <typename T>
int launch_read(const uint8_t* rows, const float* scales, int64_t BH, int64_t cap, int64_t start, int64_t n, void* K, void* V,
                cudaStream_t st) {
  constexpr int tokens = RT / (KV8_ROW / (sizeof(T) == 4 ? 4 : 8)) * RPASS;
  const dim3 grid((unsigned)cdiv(n, tokens), (unsigned)BH);
  return launch_after(kv8_read_kernel<T>, grid, RT, 0, st, "kv8_read", rows, scales, cap, start, n,
                      reinterpret_cast<T*>(K), reinterpret_cast<T*>(V));
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
  return launch_after(dtype == FATHOM_DTYPE_F32    ? kv8_write_kernel<float>
                      : dtype == FATHOM_DTYPE_BF16 ? kv8_write_kernel<__nv_bfloat16>
                                                   : kv8_write_kernel<__half>,
                      grid, WT, 0, st, "kv8_write", a);
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FATHOM_DTYPE_F32) return launch_read<float>(rows, scales, BH, cap, start, n, K, V, st);
  if (dtype == FATHOM_DTYPE_BF16) return launch_read<__nv_bfloat16>(rows, scales, BH, cap, start, n, K, V, st);
  return launch_read<__half>(rows, scales, BH, cap, start, n, K, V, st);
}
