// Attention over every row of the 8-bit key/value cache (layout in kv8.cuh): the entry point, and what its kernels share.
#include "kv8_attn.cuh"

namespace fathom {
namespace kv8 {

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = v > 0 ? v : 148;
  }
  return cached[dev];
}

namespace {

__device__ unsigned long long g_timeouts = 0;    // waits of the attention kernels that gave up

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The current device's counter (its address is looked up once per device).
unsigned long long* timeout_counter() {
  static std::atomic<unsigned long long*> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  unsigned long long* p = dev < 64 ? cached[dev].load(std::memory_order_relaxed) : nullptr;
  if (!p) {
    if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_timeouts) != cudaSuccess) return nullptr;
    if (dev < 64) cached[dev].store(p, std::memory_order_relaxed);
  }
  return p;
}

// The rows as a 3-D tensor of bytes [BH][cap][256], read in 128-byte wide tiles of 128 tokens (the key or the
// value half of each) in the 128-byte swizzle; tokens past cap read as 0.
int rows_map(const Args& a, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e =
        cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess || found != cudaDriverEntryPointSuccess || !fn)
      return set_error(FATHOM_ERR_CUDA, "kv8_attend: the driver has no cuTensorMapEncodeTiled");
    encode = reinterpret_cast<Encode>(fn);
  }
  const cuuint64_t dims[3] = {(cuuint64_t)KV8_ROW, (cuuint64_t)a.cap, (cuuint64_t)a.B * a.Hkv};
  const cuuint64_t strides[2] = {(cuuint64_t)KV8_ROW, (cuuint64_t)a.cap * KV8_ROW};
  const cuuint32_t box[3] = {(cuuint32_t)D, 128, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(a.rows), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FATHOM_ERR_CUDA, "kv8_attend: tensor map: error %d", (int)r);
  return FATHOM_OK;
}

}  // namespace

// Adds the waits that gave up to *count, and zeroes them on request.
int wait_timeouts(unsigned long long* count, int reset) {
  unsigned long long v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(v));
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(g_timeouts, &zero, sizeof(zero));
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "wait_timeouts: %s", cudaGetErrorString(e));
  *count += v;
  return FATHOM_OK;
}

}  // namespace kv8
}  // namespace fathom

using namespace fathom;
using namespace fathom::kv8;

extern "C" size_t fathom_kv8_attend_workspace_bytes(int64_t B, int64_t Hkv, int G, int64_t T) {
  if (B <= 0 || Hkv <= 0 || G <= 0 || T <= 0) return 0;
  return G * T <= TOKEN_ROWS ? token_workspace(B * Hkv, G * T) : prompt_workspace();
}

extern "C" int fathom_kv8_attend(const void* q, int dtype, int64_t B, int64_t Hkv, int G, int64_t T, int64_t q_stride_b,
                                 int64_t q_stride_h, int64_t q_stride_t, const uint8_t* rows, const float* scales,
                                 int64_t cap, int64_t end, const int64_t* end_dev, void* out, int64_t o_stride_b,
                                 int64_t o_stride_h, int64_t o_stride_t, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  FATHOM_REQUIRE(q && rows && scales && out && workspace, FATHOM_ERR_NULL, "kv8_attend: NULL pointer");
  FATHOM_REQUIRE(dtype == FATHOM_DTYPE_BF16 || dtype == FATHOM_DTYPE_F16, FATHOM_ERR_UNSUPPORTED,
                 "kv8_attend: queries must be bf16 or fp16");
  FATHOM_REQUIRE(B >= 1 && Hkv >= 1 && B <= 65535 && Hkv <= 65535 && B * Hkv <= 65535 && G >= 1 && G <= 65535 && T >= 1 &&
                     T <= INT32_MAX / G && B * Hkv * G * T <= INT32_MAX / 4 && cap >= BLK && cap % BLK == 0 &&
                     cap <= KV8_MAX_CAP, FATHOM_ERR_SHAPE, "kv8_attend: bad shape");
  FATHOM_REQUIRE(end_dev || (end >= 0 && end <= cap), FATHOM_ERR_SHAPE, "kv8_attend: end %lld is outside the cache's %lld",
                 (long long)end, (long long)cap);
  FATHOM_REQUIRE((reinterpret_cast<uintptr_t>(scales) & 7) == 0, FATHOM_ERR_SHAPE,
                 "kv8_attend: the scales must be 8-byte aligned");
  FATHOM_REQUIRE(aligned16(rows) && aligned16(q) && aligned16(out) && (q_stride_b | q_stride_h | q_stride_t) % 8 == 0 &&
                     (o_stride_b | o_stride_h | o_stride_t) % 8 == 0, FATHOM_ERR_SHAPE,
                 "kv8_attend: rows, q and out (with their strides) must be 16-byte aligned");
  FATHOM_REQUIRE(workspace_bytes >= fathom_kv8_attend_workspace_bytes(B, Hkv, G, T) &&
                     (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, FATHOM_ERR_WORKSPACE,
                 "kv8_attend: workspace needs %zu bytes, 16-byte aligned",
                 fathom_kv8_attend_workspace_bytes(B, Hkv, G, T));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned long long* timeouts = timeout_counter();
  if (!timeouts) return set_error(FATHOM_ERR_CUDA, "kv8_attend: no address of the wait counter");
  const Args a{q, q_stride_b, q_stride_h, q_stride_t, out, o_stride_b, o_stride_h, o_stride_t, rows, scales, cap, end,
               end_dev, (int)B, (int)Hkv, G, T, reinterpret_cast<float*>(workspace), timeouts, 0, 0, 1, 0, 0,
               1.0f / (float)G, 1.0f / (float)Hkv};
  CUtensorMap map;
  const int r = rows_map(a, &map);
  if (r != FATHOM_OK) return r;
  return G * T <= TOKEN_ROWS ? token_attend(map, a, dtype, st) : prompt_attend(map, a, dtype, st);
}
