// Attention over the 8-bit key/value cache (layout in kv8.cuh): over listed rows, and over every row.
#include "kv8.cuh"
#include "kv8_attn.cuh"

#include <cooperative_groups.h>

#include <atomic>

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

namespace cg = cooperative_groups;

constexpr int AW = 8;            // warps per CTA
constexpr int PG = 4;            // rows per warp instruction: lane groups of 8, a lane holds 16 dims
constexpr int DPL = 16;
constexpr int DU = 4;            // rows per lane group per step
struct RowsArgs {
  const int64_t* idx;        // [BH*G][k], or NULL: rows 0 .. end
  int64_t k;
  const uint8_t* rows;
  const float* scales;
  int64_t cap, end;
  const int64_t* end_dev;    // per sequence, or NULL
  int Hkv, G;
  int64_t T, qb, qh, qt, ob, oh, ot;   // query strides in elements
};

// One lane's share of its group's online softmax (base 2).
struct State {
  float m = -INFINITY, l = 0.0f;
  float a[DPL];
  __device__ __forceinline__ State() {
#pragma unroll
    for (int e = 0; e < DPL; ++e) a[e] = 0.0f;
  }
  __device__ __forceinline__ void merge(float mo, float lo, const float (&ao)[DPL]) {
    const float M = fmaxf(m, mo);
    const float e1 = m == -INFINITY ? 0.0f : exp2f(m - M);
    const float e2 = mo == -INFINITY ? 0.0f : exp2f(mo - M);
    l = l * e1 + lo * e2;
#pragma unroll
    for (int e = 0; e < DPL; ++e) a[e] = a[e] * e1 + ao[e] * e2;
    m = M;
  }
};

template <typename T, int CS>
__global__ void __launch_bounds__(AW * 32) kv8_rows_kernel(const T* __restrict__ q, RowsArgs a, T* __restrict__ out) {
  __shared__ float s_m[AW * CS], s_l[AW * CS];
  __shared__ __align__(16) float s_acc[AW * CS][D];
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane >> 3, sl = lane & 7;
  const unsigned crank = CS == 1 ? 0u : cluster.block_rank();
  int64_t row = blockIdx.x / CS;                 // ((b * Hkv + h) * G + g) * T + t
  const int64_t t = row % a.T, bhg = row / a.T, bh = bhg / a.G, b = bh / a.Hkv;
  const int64_t hq = bhg % ((int64_t)a.Hkv * a.G);
  int64_t end = a.end_dev ? a.end_dev[b] : a.end;
  if (end > a.cap) end = a.cap;
  if (!a.idx) end -= a.T - 1 - t;
  const int64_t k = a.idx ? a.k : (end > 0 ? end : 0);
  float qf[DPL];
  const T* qp = q + b * a.qb + hq * a.qh + t * a.qt + sl * DPL;
#pragma unroll
  for (int e = 0; e < DPL; ++e) qf[e] = to_f32(qp[e]) * QSCALE;
  const int64_t PW = (k + AW * CS - 1) / (AW * CS);
  const int64_t p0 = ((int64_t)crank * AW + warp) * PW, p1 = p0 + PW < k ? p0 + PW : k;
  const uint8_t* base = a.rows + bh * a.cap * KV8_ROW + sl * DPL;
  const float2* sc = reinterpret_cast<const float2*>(a.scales) + bh * (a.cap / BLK);
  State st;
  for (int64_t c0 = p0; c0 < p1; c0 += 32) {
    int32_t mine = -1;                           // this lane's row of the chunk
    float2 ms = make_float2(0.0f, 0.0f);
    if (c0 + lane < p1) {
      const int64_t r = a.idx ? a.idx[bhg * a.k + c0 + lane] : c0 + lane;
      if (r >= 0 && r < end) {
        mine = (int32_t)r;
        ms = sc[r / BLK];
      }
    }
    for (int s0 = 0; s0 < 32 && c0 + s0 < p1; s0 += PG * DU) {
      uint4 kw[DU], vw[DU];
      float s[DU], vs[DU];
#pragma unroll
      for (int u = 0; u < DU; ++u) {
        const int src = s0 + u * PG + grp;
        const int32_t r = __shfl_sync(0xffffffffu, mine, src);
        s[u] = __shfl_sync(0xffffffffu, ms.x, src);
        vs[u] = __shfl_sync(0xffffffffu, ms.y, src);
        kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
        if (r >= 0) {
          kw[u] = *reinterpret_cast<const uint4*>(base + (int64_t)r * KV8_ROW);
          vw[u] = *reinterpret_cast<const uint4*>(base + (int64_t)r * KV8_ROW + D);
        } else {
          s[u] = -INFINITY;
        }
      }
      float mx = st.m;
#pragma unroll
      for (int u = 0; u < DU; ++u) {
        const uint32_t w[4] = {kw[u].x, kw[u].y, kw[u].z, kw[u].w};
        float d = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 lo = kv8_decode2(w[i]), hi = kv8_decode2(w[i] >> 16);
          d = fmaf(qf[4 * i], lo.x, d);
          d = fmaf(qf[4 * i + 1], lo.y, d);
          d = fmaf(qf[4 * i + 2], hi.x, d);
          d = fmaf(qf[4 * i + 3], hi.y, d);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        // a NaN score counts as +inf: the differences below become NaN, and so does the row
        if (s[u] != -INFINITY) s[u] = d * s[u] == d * s[u] ? d * s[u] : INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      if (mx == -INFINITY) continue;
      const float corr = st.m == -INFINITY ? 0.0f : exp2f(st.m - mx);
      st.m = mx;
      st.l *= corr;
#pragma unroll
      for (int e = 0; e < DPL; ++e) st.a[e] *= corr;
#pragma unroll
      for (int u = 0; u < DU; ++u) {
        const float p = exp2f(s[u] - mx);
        st.l += p;
        const float pv = p * vs[u];
        const uint32_t w[4] = {vw[u].x, vw[u].y, vw[u].z, vw[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 lo = kv8_decode2(w[i]), hi = kv8_decode2(w[i] >> 16);
          st.a[4 * i] = fmaf(pv, lo.x, st.a[4 * i]);
          st.a[4 * i + 1] = fmaf(pv, lo.y, st.a[4 * i + 1]);
          st.a[4 * i + 2] = fmaf(pv, hi.x, st.a[4 * i + 2]);
          st.a[4 * i + 3] = fmaf(pv, hi.y, st.a[4 * i + 3]);
        }
      }
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    float ao[DPL];
    const float mo = __shfl_xor_sync(0xffffffffu, st.m, o), lo = __shfl_xor_sync(0xffffffffu, st.l, o);
#pragma unroll
    for (int e = 0; e < DPL; ++e) ao[e] = __shfl_xor_sync(0xffffffffu, st.a[e], o);
    st.merge(mo, lo, ao);
  }
  float *dm = s_m, *dl = s_l, *da = &s_acc[0][0];
  if constexpr (CS > 1) {
    dm = cluster.map_shared_rank(s_m, 0);
    dl = cluster.map_shared_rank(s_l, 0);
    da = cluster.map_shared_rank(&s_acc[0][0], 0);
  }
  const int gw = (int)crank * AW + warp;
  if (lane == 0) dm[gw] = st.m, dl[gw] = st.l;
  if (lane < 8) {
    float4* dst = reinterpret_cast<float4*>(da + gw * D + sl * DPL);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      dst[e] = make_float4(st.a[4 * e], st.a[4 * e + 1], st.a[4 * e + 2], st.a[4 * e + 3]);
  }
  if constexpr (CS == 1) __syncthreads();
  else cluster.sync();
  if (crank != 0 || threadIdx.x >= D) return;
  float M = -INFINITY, L = 0.0f, O = 0.0f;
  for (int w = 0; w < AW * CS; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < AW * CS; ++w) {
    const float e = s_m[w] == -INFINITY ? 0.0f : exp2f(s_m[w] - M);
    L = fmaf(s_l[w], e, L);
    O = fmaf(s_acc[w][threadIdx.x], e, O);
  }
  from_f32(L == 0.0f ? 0.0f : O / L, out + b * a.ob + hq * a.oh + t * a.ot + threadIdx.x);
}

template <typename T, int CS>
int launch_rows_cs(const void* q, const RowsArgs& a, int64_t rows, void* out, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * CS));
  cfg.blockDim = dim3(AW * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_rows_kernel<T, CS>, (const T*)q, a, (T*)out);
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "kv8_attend: launch: %s", cudaGetErrorString(e));
  return check_launch("kv8_attend");
}

template <typename T>
int launch_rows(const void* q, const RowsArgs& a, int64_t rows, void* out, cudaStream_t st) {
  const int64_t sms = sm_count();
  if (rows >= 2 * sms) return launch_rows_cs<T, 1>(q, a, rows, out, st);
  return launch_rows_cs<T, 4>(q, a, rows, out, st);
}

int dispatch_rows(int dtype, const void* q, const RowsArgs& a, int64_t rows, void* out, cudaStream_t st) {
  if (dtype == FATHOM_DTYPE_F32) return launch_rows<float>(q, a, rows, out, st);
  if (dtype == FATHOM_DTYPE_BF16) return launch_rows<__nv_bfloat16>(q, a, rows, out, st);
  return launch_rows<__half>(q, a, rows, out, st);
}

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
  FATHOM_REQUIRE(aligned16(rows) && aligned16(q) && aligned16(out) && (q_stride_b | q_stride_h | q_stride_t) % 8 == 0 &&
                     (o_stride_b | o_stride_h | o_stride_t) % 8 == 0, FATHOM_ERR_SHAPE,
                 "kv8_attend: rows, q and out (with their strides) must be 16-byte aligned");
  FATHOM_REQUIRE(workspace_bytes >= fathom_kv8_attend_workspace_bytes(B, Hkv, G, T), FATHOM_ERR_WORKSPACE,
                 "kv8_attend: workspace too small");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned long long* timeouts = timeout_counter();
  if (!timeouts) return set_error(FATHOM_ERR_CUDA, "kv8_attend: no address of the wait counter");
  const Args a{q, q_stride_b, q_stride_h, q_stride_t, out, o_stride_b, o_stride_h, o_stride_t, rows, scales, cap, end,
               end_dev, (int)B, (int)Hkv, G, T, reinterpret_cast<float*>(workspace), timeouts, 0, 0};
  CUtensorMap map;
  const int r = rows_map(a, &map);
  if (r != FATHOM_OK) return r;
  return G * T <= TOKEN_ROWS ? token_attend(map, a, dtype, st) : prompt_attend(map, a, dtype, st);
}

extern "C" size_t fathom_kv8_attend_picks_workspace_bytes(int64_t B, int64_t Hkv, int G, int64_t k) {
  if (B <= 0 || Hkv <= 0 || G <= 0 || k <= 0) return 0;
  return 256;
}

extern "C" int fathom_kv8_attend_picks(const void* q, int dtype, int64_t B, int64_t Hkv, int G, const int64_t* idx,
                                       int64_t k, const uint8_t* rows, const float* scales, int64_t cap, int64_t end,
                                       const int64_t* end_dev, void* out, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  FATHOM_REQUIRE(q && idx && rows && scales && out && workspace, FATHOM_ERR_NULL, "kv8_attend_picks: NULL pointer");
  FATHOM_REQUIRE(dtype >= FATHOM_DTYPE_F32 && dtype <= FATHOM_DTYPE_F16, FATHOM_ERR_UNSUPPORTED,
                 "kv8_attend_picks: queries must be fp32, bf16 or fp16");
  FATHOM_REQUIRE(B >= 1 && Hkv >= 1 && B <= 65535 && Hkv <= 65535 && B * Hkv <= 65535 && G >= 1 && G <= 65535 &&
                     B * Hkv * G <= INT32_MAX / 8 && k >= 1 && k <= INT32_MAX && cap >= BLK && cap % BLK == 0 &&
                     cap <= KV8_MAX_CAP, FATHOM_ERR_SHAPE, "kv8_attend_picks: bad shape");
  FATHOM_REQUIRE(end_dev || (end >= 0 && end <= cap), FATHOM_ERR_SHAPE,
                 "kv8_attend_picks: end %lld is outside the cache's %lld", (long long)end, (long long)cap);
  FATHOM_REQUIRE(aligned16(rows) && aligned16(q) && aligned16(out), FATHOM_ERR_SHAPE,
                 "kv8_attend_picks: rows, q and out must be 16-byte aligned");
  FATHOM_REQUIRE(workspace_bytes >= fathom_kv8_attend_picks_workspace_bytes(B, Hkv, G, k), FATHOM_ERR_WORKSPACE,
                 "kv8_attend_picks: workspace too small");
  const RowsArgs a{idx, k, rows, scales, cap, end, end_dev, (int)Hkv, G, 1, (int64_t)Hkv * G * D, D, D,
                   (int64_t)Hkv * G * D, D, D};
  return dispatch_rows(dtype, q, a, B * Hkv * G, out, reinterpret_cast<cudaStream_t>(stream));
}
