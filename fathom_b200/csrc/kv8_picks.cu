// Attention over listed rows of the 8-bit cache (layout in kv8.cuh), one list per query head.
//
// The floor is the rows' bytes, 256 at random addresses per pick, and for one sequence latency.  A warp takes 16 picks at
// a time; their rows come into shared memory by 16-byte asynchronous copies while it works on the 16 before: 64 KB on
// their way per SM.  With one query row per list a product has nothing to share, but
// dequantising and multiplying on the fp32 pipes took ~290 instructions per 4 picks; as fragments of 16-bit matrix
// instructions (an e4m3 is exact in f16) it is ~190 per 16:
//
//   scores   [16 picks x 8] = K [16 x 128] q^T          columns: q as a sum of three f16 terms (33 bits)
//   output^T [128 dims x 8] += V^T [128 x 16 picks] p   columns: the weights as two f16 terms (22 bits)
//
// The order of dims within a score, and of picks within a sum, is free, so a lane's fragments are 16-byte pieces of rows as
// they lie: K piece j and j + 4 of picks g and g + 8, V piece g of picks 2j, 2j + 1, 2j + 8, 2j + 9 (lane = 4 g + j).
// Softmax state per warp, in fp32 as in kv8_token.cu: references of s + log2(value scale) for the output and of s for
// the denominator.  The warps of a (batch, query head) lie in one CTA or a cluster; their states are joined in warp
// order in the first CTA's shared memory.
//
// Measured over 128k: 2116 picks for each of 224 heads 34 us, 3.6 TB/s of rows (58 us on the fp32 pipes); with the rows
// in L2 it takes 29: the warps' own steps are the bound, and 16 warps per SM with 2 stages are better than 12 with 3.
// 580 picks for 32 heads: 8.0 us with its launch.
#include "dedupe.cuh"
#include "kv8_attn.cuh"

#include <cooperative_groups.h>

#include <stddef.h>

namespace fathom {
namespace kv8 {
namespace {

namespace cg = cooperative_groups;

constexpr int CHUNK = 16;                // picks per step of a warp
constexpr int STAGES = 2;                // chunks in shared memory: being used, and on its way
constexpr int WARPS_PER_SM = 16;         // 16 x 2 x 4.3 KB of shared memory, 16 x 32 threads of 128 registers
constexpr int MAX_CS = 8, MAX_PW = 4;    // CTAs of a cluster, warps of a CTA
constexpr float SLACK = 6.0f;            // a chunk may exceed the reference by 2^6
constexpr float HEAD = 8.0f;             // weights at the reference are 2^8: f16 from 2^-24 to 2^15

struct PicksArgs {
  const int64_t* idx;        // [BH*G][k]
  const int32_t* slot;       // [BH*G][k] row of `rows` that holds the pick, -1: none; NULL: the pick itself
  int64_t k;
  const uint8_t* rows;       // [BH][row_cap][256]
  int64_t row_cap;
  const float* scales;
  int64_t cap, end;
  const int64_t* end_dev;
  int Hkv, G;
};

struct alignas(128) Stage {              // halves of rows 128-byte aligned: pieces are permuted by XOR on addresses
  uint8_t row[CHUNK][KV8_ROW];           // 16-byte pieces permuted within each half (piece_of)
  float2 scale[CHUNK];
  int valid[CHUNK];
};

// Piece c (0..7) of a row's key or value half lies at c ^ permuted(row), so that the 8 lanes of a shared-memory phase meet
// 8 different bank groups: keys are read as rows 2p, 2p + 1 x 4 pieces, values as 4 even or odd rows x 2 pieces.
__device__ __forceinline__ int permuted(int row) { return ((row >> 1 & 3) ^ (row & 1) << 1) << 1; }

// dst: shared-memory addresses; zeros where there is no row.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_of(uint32_t codes) {       // two codes in the low 16 bits
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xFFFFu), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// 16 consecutive elements of q, 16-byte aligned.
__device__ __forceinline__ void load16(const void* p, int dtype, int64_t i, float* x) {
  if (dtype == FATHOM_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<float4*>(x + 4 * e) = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint4 v = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i)[e];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 f = dtype == FATHOM_DTYPE_BF16
                           ? make_float2(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xFFFF0000u))
                           : __half22float2(*reinterpret_cast<const __half2*>(&w[u]));
      x[8 * e + 2 * u] = f.x, x[8 * e + 2 * u + 1] = f.y;
    }
  }
}

__global__ void __launch_bounds__(MAX_PW * 32, WARPS_PER_SM / MAX_PW)
    picks_kernel(const void* __restrict__ q, int dtype, const PicksArgs a,
                                                                   void* __restrict__ out) {
  const int PW = blockDim.x >> 5, NW = PW * (int)gridDim.y;      // one cluster of gridDim.y CTAs per (batch, query head)
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int MAX_NW = MAX_PW * MAX_CS;
  __shared__ float s_m[MAX_NW], s_lm[MAX_NW], s_l[MAX_NW];       // the cluster's first CTA: every warp's state
  float(*const s_acc)[D] = reinterpret_cast<float(*)[D]>(smem_raw + PW * STAGES * sizeof(Stage));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  Stage* const st = reinterpret_cast<Stage*>(smem_raw) + warp * STAGES;
  const unsigned crank = blockIdx.y;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                            // waited for before the first store into another CTA
  const int64_t bhg = blockIdx.x;
  const int bh = (int)bhg / a.G, gw = (int)crank * PW + warp;
  int64_t end = a.end_dev ? a.end_dev[bh / a.Hkv] : a.end;
  if (end > a.cap) end = a.cap;
  const float2* sc = reinterpret_cast<const float2*>(a.scales) + (int64_t)bh * (a.cap / BLK);
  const int k = (int)a.k, chunks = (k + CHUNK - 1) / CHUNK;
  const int n = chunks > gw ? (chunks - gw + NW - 1) / NW : 0;   // this warp's chunks: gw, gw + NW, ..

  // lanes 0..15: the next chunk's picks and the rows that hold them (-1: none)
  int next = lane < CHUNK ? gw * CHUNK + lane : k;
  auto pick = [&](int& tok, int& row) {
    tok = row = -1;
    if (next < k) {
      const int64_t t = a.idx[bhg * k + next];
      if (t >= 0 && t < end) tok = (int)t, row = a.slot ? a.slot[bhg * k + next] : tok;
      next += NW * CHUNK;
    }
  };
  // copies of a chunk into stage s: a lane has piece lane & 15 of rows 2 u + (lane >> 4)
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(st);
  const uint32_t lane_at = (lane >> 4) * KV8_ROW + (lane & 8) * 16 + ((lane & 7) ^ permuted(lane >> 4)) * 16;
  const uint8_t* const from = a.rows + (int64_t)bh * a.row_cap * KV8_ROW + (lane & 15) * 16;
  auto bring = [&](int s, int tok, int row) {
    const uint32_t at = ring + s * (uint32_t)sizeof(Stage);
    if (lane < CHUNK) {
      st[s].valid[lane] = row;
      if (row >= 0) copy8(at + (uint32_t)offsetof(Stage, scale) + lane * 8, sc + tok / BLK);
    }
#pragma unroll
    for (int u = 0; u < CHUNK / 2; ++u) {
      const int r = __shfl_sync(0xffffffffu, row, 2 * u + (lane >> 4));
      copy16((at + lane_at + u * 2 * KV8_ROW) ^ ((u & 3) << 5), from + (int64_t)max(r, 0) * KV8_ROW, r >= 0);
    }
  };
  auto commit = []() { asm volatile("cp.async.commit_group;\n" ::: "memory"); };
  int tok, row;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    pick(tok, row);
    if (i < n) bring(i, tok, row);
    commit();
  }
  pick(tok, row);

  // q: this lane's dims, 16 j .. and 64 + 16 j .., of term g (0, 1, 2; zeros for the others)
  uint32_t qf[16];
  float rs;
  {
    float x[32];
    load16(q, dtype, bhg * D + 16 * j, x);
    load16(q, dtype, bhg * D + 64 + 16 * j, x + 16);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    const int e = kv8_exponent(top);
    const float inv = top < 0x7F800000u ? pow2i(-e) : __uint_as_float(0x7FFFFFFFu);   // a row with inf or NaN is NaN
    rs = pow2i(e) * QSCALE;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 y = make_float2(x[2 * i] * inv, x[2 * i + 1] * inv);
      __half2 h[3];
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        h[t] = __floats2half2_rn(y.x, y.y);
        const float2 f = __half22float2(h[t]);
        y = make_float2(y.x - f.x, y.y - f.y);         // what the terms so far leave
      }
      qf[i] = g == 0 ? bits(h[0]) : g == 1 ? bits(h[1]) : g == 2 ? bits(h[2]) : 0u;
    }
  }

  // this lane's pieces within a stage: of keys g and g + 8 (permuted alike), of values 2 j + (e & 1) + 4 (e & 2)
  const int key_at = g * KV8_ROW + (j ^ permuted(g)) * 16;
  int value_at[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) value_at[e] = (2 * j + e) * KV8_ROW + D + (g ^ permuted(2 * j + e)) * 16;
  float acc[8][4];                                     // dims 16 g + 2 t and + 1; columns 2 j, 2 j + 1
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
  float m = -INFINITY, lm = -1e30f, l = 0.0f;          // m is the warp's; l is of picks g and g + 8 of its chunks
  int here = 0;                                        // stage of chunk i
  for (int i = 0; i < n; ++i) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                      // chunk i is there; chunk i - 1 has been read
    if (i + STAGES - 1 < n) bring(here == 0 ? STAGES - 1 : here - 1, tok, row);
    commit();
    pick(tok, row);
    const Stage& s = st[here];
    const uint8_t* const bytes = &s.row[0][0];
    here = here + 1 == STAGES ? 0 : here + 1;
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, c2[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // two chains of products
    const uint4 k0 = *reinterpret_cast<const uint4*>(bytes + key_at),
                k1 = *reinterpret_cast<const uint4*>(bytes + (key_at ^ 64));
    const uint4 k8 = *reinterpret_cast<const uint4*>(bytes + 8 * KV8_ROW + key_at),
                k9 = *reinterpret_cast<const uint4*>(bytes + 8 * KV8_ROW + (key_at ^ 64));
    uint32_t x[4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint4 y = *reinterpret_cast<const uint4*>(bytes + (e >> 1) * 8 * KV8_ROW + value_at[e & 1]);
      x[e][0] = y.x, x[e][1] = y.y, x[e][2] = y.z, x[e][3] = y.w;
    }
    {
      const uint32_t lo[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
      const uint32_t hi[8] = {k8.x, k8.y, k8.z, k8.w, k9.x, k9.y, k9.z, k9.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mma(c, half2_of(lo[w]), half2_of(hi[w]), half2_of(lo[w] >> 16), half2_of(hi[w] >> 16), qf[2 * w], qf[2 * w + 1]);
        mma(c2, half2_of(lo[w + 4]), half2_of(hi[w + 4]), half2_of(lo[w + 4] >> 16), half2_of(hi[w + 4] >> 16), qf[8 + 2 * w],
            qf[9 + 2 * w]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] += c2[e];
    // scores of picks g and g + 8: the sum of their columns, 2 of them in each lane of a quad
    float v[2] = {c[0] + c[1], c[2] + c[3]}, lv[2], w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[e] += __shfl_xor_sync(0xffffffffu, v[e], 1);
      v[e] += __shfl_xor_sync(0xffffffffu, v[e], 2);
      const int r = g + 8 * e;
      const bool there = s.valid[r] >= 0;
      const float2 ks = there ? s.scale[r] : make_float2(0.0f, 1.0f);
      v[e] = there ? v[e] * (ks.x * rs) : -INFINITY;
      lv[e] = (float)((int)(__float_as_uint(ks.y) >> 23) - 127);
    }
    float top = fmaxf(v[0] + lv[0], v[1] + lv[1]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top > m + SLACK) {                             // the same in every lane; also the first time: m = -inf
      const float f = m == -INFINITY ? 0.0f : ex2(m - top);
      m = top;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] *= f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w[e] = m == -INFINITY && !(v[e] != v[e]) ? 0.0f : ex2(v[e] + (lv[e] - m + HEAD));
      const float d = v[e] - lm, p = ex2(-fabsf(d));
      l = d > 0.0f ? fmaf(l, p, 1.0f) : l + p;
      lm = fmaxf(lm, v[e]);
    }
    // weights of picks 2 j, 2 j + 1 and 2 j + 8, 2 j + 9 as term g
    uint32_t b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = __shfl_sync(0xffffffffu, w[e], 8 * j), y = __shfl_sync(0xffffffffu, w[e], 8 * j + 4);
      const __half2 hi = __floats2half2_rn(x, y);
      const float2 f = __half22float2(hi);
      b[e] = g == 0 ? bits(hi) : g == 1 ? bits(__floats2half2_rn(x - f.x, y - f.y)) : 0u;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // bytes 4 u + 2 h and + 1 of two picks side by side
        const uint32_t s01 = __byte_perm(x[0][u], x[1][u], h ? 0x7362 : 0x5140);
        const uint32_t s89 = __byte_perm(x[2][u], x[3][u], h ? 0x7362 : 0x5140);
        mma(acc[2 * u + h], half2_of(s01), half2_of(s01 >> 16), half2_of(s89), half2_of(s89 >> 16), b[0], b[1]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  // the warp's state: picks are spread over g
  float ref = lm;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
  l *= ex2(lm - ref);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  cluster.barrier_wait();
  float *dm = cluster.map_shared_rank(s_m, 0), *dlm = cluster.map_shared_rank(s_lm, 0);
  float *dl = cluster.map_shared_rank(s_l, 0), *da = cluster.map_shared_rank(&s_acc[0][0], 0);
  if (lane == 0) dm[gw] = m, dlm[gw] = ref, dl[gw] = l;
  if (j == 0) {                                        // columns 0 and 1: the two terms' sums
    float4* dst = reinterpret_cast<float4*>(da + gw * D + 16 * g);
#pragma unroll
    for (int t = 0; t < 8; t += 2)
      dst[t / 2] = make_float4(acc[t][0] + acc[t][1], acc[t][2] + acc[t][3], acc[t + 1][0] + acc[t + 1][1],
                               acc[t + 1][2] + acc[t + 1][3]);
  }
  cluster.sync();
  if (crank != 0) return;
  // lane = warp state: its factor, then every thread a dim or more
  float M = lane < NW ? s_lm[lane] : -1e30f;
  M = warp_max(M);
  const float L = warp_sum(lane < NW ? s_l[lane] * ex2(s_lm[lane] - M) : 0.0f);
  const float mine = lane < NW && s_m[lane] != -INFINITY ? exp2f(s_m[lane] - HEAD - M) : 0.0f;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float O = 0.0f;
#pragma unroll 8
    for (int v = 0; v < NW; ++v) {
      const float f = __shfl_sync(0xffffffffu, mine, v);
      if (f != 0.0f) O = fmaf(s_acc[v][d], f, O);
    }
    const float o = O * inv;
    const int64_t at = bhg * D + d;
    if (dtype == FATHOM_DTYPE_F32) from_f32(o, reinterpret_cast<float*>(out) + at);
    else if (dtype == FATHOM_DTYPE_BF16) from_f32(o, reinterpret_cast<__nv_bfloat16*>(out) + at);
    else from_f32(o, reinterpret_cast<__half*>(out) + at);
  }
}

int launch_picks(const void* q, int dtype, const PicksArgs& a, int64_t heads, int pw, int cs, void* out, cudaStream_t st) {
  const int smem = pw * STAGES * (int)sizeof(Stage) + pw * cs * D * (int)sizeof(float);
  constexpr int most = MAX_PW * STAGES * (int)sizeof(Stage) + MAX_PW * MAX_CS * D * (int)sizeof(float);
  static std::atomic<uint64_t> told{0};
  const int r = allow_smem(picks_kernel, most, told, "kv8_attend_picks");
  if (r != FATHOM_OK) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)heads, (unsigned)cs);
  cfg.blockDim = dim3((unsigned)pw * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)cs;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, picks_kernel, q, dtype, a, out);
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "kv8_attend_picks: launch: %s", cudaGetErrorString(e));
  return check_launch("kv8_attend_picks");
}

// Rows in host memory: each distinct row of a KV head once over the host link into the workspace, in ascending order.
// 16 lanes x 16 bytes per row, 4 rows in flight per lane.
constexpr int GT = 256, GROWS = GT / 16 * 4;
__global__ void __launch_bounds__(GT) gather_kernel(const int32_t* __restrict__ ucount, const int64_t* __restrict__ uniq,
                                                    int64_t M, const uint4* __restrict__ rows, int64_t cap,
                                                    uint4* __restrict__ stage) {
  constexpr int LPR = KV8_ROW / 16, RPP = GT / LPR, PASSES = GROWS / RPP;
  const int64_t bh = blockIdx.y, U = ucount[bh], r0 = (int64_t)blockIdx.x * GROWS;
  if (r0 >= U) return;
  const int c = threadIdx.x % LPR;
  uint4 v[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int64_t r = r0 + p * RPP + threadIdx.x / LPR;
    if (r < U) v[p] = rows[(bh * cap + uniq[bh * M + r]) * LPR + c];
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int64_t r = r0 + p * RPP + threadIdx.x / LPR;
    if (r < U) stage[(bh * M + r) * LPR + c] = v[p];
  }
}

struct StageWs {
  int32_t* slot;       // [BH][M] pick -> row of the stage (-1: none)
  int64_t* uniq;       // [BH][M] distinct picks, ascending
  int32_t* ucount;     // [BH]
  uint8_t* rows;       // [BH][M][256]
};
size_t stage_bytes(int64_t BH, int64_t M) {
  return align256(BH * M * sizeof(int32_t)) + align256(BH * M * sizeof(int64_t)) + align256(BH * sizeof(int32_t)) +
         (size_t)(BH * M) * KV8_ROW;
}
StageWs carve(void* base, int64_t BH, int64_t M) {
  char* p = static_cast<char*>(base);
  StageWs w;
  w.slot = reinterpret_cast<int32_t*>(p);
  p += align256(BH * M * sizeof(int32_t));
  w.uniq = reinterpret_cast<int64_t*>(p);
  p += align256(BH * M * sizeof(int64_t));
  w.ucount = reinterpret_cast<int32_t*>(p);
  p += align256(BH * sizeof(int32_t));
  w.rows = reinterpret_cast<uint8_t*>(p);
  return w;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace kv8
}  // namespace fathom

using namespace fathom;
using namespace fathom::kv8;

extern "C" size_t fathom_kv8_attend_picks_workspace_bytes(int64_t B, int64_t Hkv, int G, int64_t k, int host_rows) {
  if (B <= 0 || Hkv <= 0 || G <= 0 || k <= 0) return 0;
  return host_rows && G * k <= MAX_M ? stage_bytes(B * Hkv, G * k) : 256;
}

extern "C" int fathom_kv8_attend_picks(const void* q, int dtype, int64_t B, int64_t Hkv, int G, const int64_t* idx,
                                       int64_t k, const uint8_t* rows, int host_rows, const float* scales, int64_t cap,
                                       int64_t end, const int64_t* end_dev, void* out, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  FATHOM_REQUIRE(q && idx && rows && scales && out && workspace, FATHOM_ERR_NULL, "kv8_attend_picks: NULL pointer");
  FATHOM_REQUIRE(dtype >= FATHOM_DTYPE_F32 && dtype <= FATHOM_DTYPE_F16, FATHOM_ERR_UNSUPPORTED,
                 "kv8_attend_picks: queries must be fp32, bf16 or fp16");
  FATHOM_REQUIRE(B >= 1 && Hkv >= 1 && B <= 65535 && Hkv <= 65535 && B * Hkv <= 65535 && G >= 1 && G <= 65535 &&
                     B * Hkv * G <= INT32_MAX / 8 && k >= 1 && k <= 1 << 30 && cap >= BLK && cap % BLK == 0 &&
                     cap <= KV8_MAX_CAP, FATHOM_ERR_SHAPE, "kv8_attend_picks: bad shape");
  FATHOM_REQUIRE(end_dev || (end >= 0 && end <= cap), FATHOM_ERR_SHAPE,
                 "kv8_attend_picks: end %lld is outside the cache's %lld", (long long)end, (long long)cap);
  FATHOM_REQUIRE(aligned16(rows) && aligned16(q) && aligned16(out) && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
                 FATHOM_ERR_SHAPE, "kv8_attend_picks: rows, q and out must be 16-byte aligned, scales 8-byte");
  FATHOM_REQUIRE(workspace_bytes >= fathom_kv8_attend_picks_workspace_bytes(B, Hkv, G, k, host_rows) &&
                     (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, FATHOM_ERR_WORKSPACE,
                 "kv8_attend_picks: workspace needs %zu bytes, 256-byte aligned",
                 fathom_kv8_attend_picks_workspace_bytes(B, Hkv, G, k, host_rows));
  PicksArgs a{idx, nullptr, k, rows, cap, scales, cap, end, end_dev, (int)Hkv, G};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t BH = B * Hkv, M = G * k;
  if (host_rows && M <= MAX_M) {             // longer lists read their rows in place, over the link, once per pick
    const StageWs w = carve(workspace, BH, M);
    int r = launch_dedupe(idx, BH, M, 0, cap, cap, w.slot, w.uniq, w.ucount, st);
    if (r != FATHOM_OK) return r;
    gather_kernel<<<dim3((unsigned)cdiv(M, GROWS), (unsigned)BH), GT, 0, st>>>(
        w.ucount, w.uniq, M, reinterpret_cast<const uint4*>(rows), cap, reinterpret_cast<uint4*>(w.rows));
    r = check_launch("kv8_attend_picks (dedupe, gather)");
    if (r != FATHOM_OK) return r;
    a.slot = w.slot, a.rows = w.rows, a.row_cap = M;
  }
  // as many warps per head as the GPU holds at once, 32 at most, and no more than there are chunks; in CTAs of 2 (in
  // whose number a wave is filled best) or of 4
  const int64_t heads = B * Hkv * G, chunks = cdiv(k, CHUNK);
  int64_t warps = (int64_t)WARPS_PER_SM * sm_count() / heads;
  if (warps > chunks) warps = chunks;
  const int pw = warps > 2 * MAX_CS ? 4 : warps > 1 ? 2 : 1;
  const int64_t cs = warps / pw < 1 ? 1 : warps / pw > MAX_CS ? MAX_CS : warps / pw;
  return launch_picks(q, dtype, a, heads, pw, (int)cs, out, st);
}
