// Attention over listed rows of the 8-bit cache (layout in kv8.cuh), one list per query head.
//
// The floor is the rows' bytes, 256 at random addresses per pick, and for one sequence latency.  A warp takes 32 picks at
// a time; their rows come into shared memory by 16-byte asynchronous copies while it works on the 32 before.  With one
// query row per list a product has nothing to share, but the matrix instructions take e4m3 as it lies in memory, so
// nothing is dequantised:
//
//   scores   [32 picks x 8] = K [32 x 128] q^T          columns: q as a sum of six e4m3 terms, 16^-n apart (24 bits)
//   output^T [128 dims x 8] += V^T [128 x 32 picks] p   columns: the weights as six such terms
//
// (m16n8k32 keeps 24 bits of a sum; measured with single large and small products.)  The order of dims within a score,
// and of picks within a sum, is free, so a lane's fragments are 16-byte pieces of rows as they lie: lane 4 g + j has key
// pieces j and j + 4 of picks g, g + 8, g + 16, g + 24, and value piece g of picks 4 j .. 4 j + 3 and 16 + 4 j .., whose
// bytes it transposes 4 x 4.  Softmax, lane = pick, in fp32 as in kv8_token.cu: references of s + log2(value scale)
// for the output and of s for the denominator.  The warps of a (batch, query head) lie in one CTA or a cluster; their
// states are joined in warp order in the first CTA's shared memory.
//
// Measured over 128k: 2116 picks for each of 224 heads 24.4-25.7 us, 4.7 TB/s of rows (34 with 16-bit matrix instructions on
// rows turned to f16, 58 on the fp32 pipes; 32.5 while a step waited for its entry of the list); with the rows in L2 24,
// so the bound is a warp's chain of steps at 8 warps per SM (issue 47% busy), not HBM.  ~5 us of it begin and join; the rest is
// 32 picks per 340 cycles and SM, 6 TB/s.  12 warps per SM, or 3 stages, are
// slower (29 us), so are TMA gathers of 4 rows (28; for the keys alone 28.5), bulk copies of one (34) and rows loaded into
// registers (29).  580 picks for 32 heads: 4.9-5.1 us in a graph.
#include "dedupe.cuh"
#include "kv8_attn.cuh"

#include <cooperative_groups.h>

#include <stddef.h>

namespace fathom {
namespace kv8 {
namespace {

namespace cg = cooperative_groups;

constexpr int CHUNK = 32;                // picks per step of a warp
constexpr int STAGES = 2;                // chunks in shared memory: being used, and on its way
constexpr int WARPS_PER_SM = 8;          // what the SM holds with ~180 registers per thread
constexpr int MAX_CS = 8, MAX_PW = 4;    // CTAs of a cluster, warps of a CTA
constexpr int TERMS = 6;                 // e4m3 terms of q and of the weights, 4 bits each
constexpr float SLACK = 6.0f;            // a chunk may exceed the reference by 2^6
constexpr float HEAD = 2.0f;             // weights at the reference are 4: 2^(HEAD + SLACK) = 256 <= 448

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
  uint8_t row[CHUNK][KV8_ROW];           // 16-byte pieces permuted within each half
  float2 scale[CHUNK];
  int valid[CHUNK];
};
struct alignas(128) Warp {
  Stage stage[STAGES];
  uint32_t weight[8][CHUNK / 4];         // term n of the chunk's weights; rows TERMS .. stay 0
};

// Piece c (0..7) of a row's key or value half lies at c ^ permuted(row), so that the 8 lanes of a shared-memory phase meet
// 8 different bank groups: keys are read as rows 2p, 2p + 1 x 4 pieces, values as rows i, i + 4, i + 8, i + 12 x 2.
__device__ __forceinline__ int permuted(int row) { return ((row >> 2 & 3) ^ (row & 1) << 1) << 1; }

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
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes b of four words side by side: x[b] = (w0.b, w1.b, w2.b, w3.b).
__device__ __forceinline__ void transpose4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&x)[4]) {
  const uint32_t t0 = __byte_perm(w0, w1, 0x5140), t1 = __byte_perm(w0, w1, 0x7362);
  const uint32_t t2 = __byte_perm(w2, w3, 0x5140), t3 = __byte_perm(w2, w3, 0x7362);
  x[0] = __byte_perm(t0, t2, 0x5410), x[1] = __byte_perm(t0, t2, 0x7632);
  x[2] = __byte_perm(t1, t3, 0x5410), x[3] = __byte_perm(t1, t3, 0x7632);
}
// Two values to two codes; what they leave, times 16.
__device__ __forceinline__ uint32_t next_term(float2& y) {
  const uint32_t code = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
  const float2 d = kv8_decode2(code);
  y = make_float2(fmaf(d.x, -16.0f, 16.0f * y.x), fmaf(d.y, -16.0f, 16.0f * y.y));
  return code;
}

// 4 consecutive elements of q, as they are and as fp32.  (A branch around the load would wait for it.)
__device__ __forceinline__ uint4 load4(const void* p, bool f32) {
  uint4 v = make_uint4(0, 0, 0, 0);
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %5, 0; @p ld.global.v4.u32 {%0, %1, %2, %3}, [%4]; @!p ld.global.v2.u32 {%0, %1}, [%4]; }\n"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"((uint32_t)f32)
      : "memory");
  return v;
}
// An entry of a list, if `there`.
__device__ __forceinline__ void load_entry(int64_t& x, const int64_t* p, bool there) {
  asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; @p ld.global.b64 %0, [%1]; }\n"
               : "+l"(x)
               : "l"(p), "r"((uint32_t)there)
               : "memory");
}
__device__ __forceinline__ void load_entry(int& x, const int32_t* p, bool there) {
  asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; @p ld.global.b32 %0, [%1]; }\n"
               : "+r"(x)
               : "l"(p), "r"((uint32_t)there)
               : "memory");
}
__device__ __forceinline__ void unpack4(uint4 v, int dtype, float (&x)[4]) {
  if (dtype == FATHOM_DTYPE_F32) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    return;
  }
  const uint32_t w[2] = {v.x, v.y};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const float2 f = dtype == FATHOM_DTYPE_BF16
                         ? make_float2(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xFFFF0000u))
                         : __half22float2(*reinterpret_cast<const __half2*>(&w[u]));
    x[2 * u] = f.x, x[2 * u + 1] = f.y;
  }
}

__global__ void __launch_bounds__(MAX_PW * 32, WARPS_PER_SM / MAX_PW)
    picks_kernel(const void* q, int dtype, const PicksArgs a, void* out) {
  const int PW = blockDim.x >> 5, NW = PW * (int)gridDim.y;      // one cluster of gridDim.y CTAs per (batch, query head)
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int MAX_NW = MAX_PW * MAX_CS;
  __shared__ float s_m[MAX_NW], s_lm[MAX_NW], s_l[MAX_NW];       // the cluster's first CTA: every warp's state
  __shared__ __align__(16) uint32_t s_q[8][D / 4];               // term n of q; rows TERMS .. are 0
  __shared__ float s_rs;
  float(*const s_acc)[D] = reinterpret_cast<float(*)[D]>(smem_raw + PW * sizeof(Warp));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  Warp& mine = reinterpret_cast<Warp*>(smem_raw)[warp];
  Stage* const st = mine.stage;
  const unsigned crank = blockIdx.y;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                            // waited for before the first store into another CTA
  tc::wait_dependency();                               // (nothing is let start early: clusters of the next call in the gaps
                                                       // of this one's leave it no room for whole ones, 39 us for 26)
  const int64_t bhg = blockIdx.x;
  const int bh = (int)bhg / a.G, gw = (int)crank * PW + warp;
  const uint4 qv = load4(reinterpret_cast<const char*>(q) + (bhg * D + 4 * lane) * (dtype == FATHOM_DTYPE_F32 ? 4 : 2),
                         dtype == FATHOM_DTYPE_F32);
  int64_t end = a.end_dev ? a.end_dev[bh / a.Hkv] : a.end;
  if (end > a.cap) end = a.cap;
  const float2* sc = reinterpret_cast<const float2*>(a.scales) + (int64_t)bh * (a.cap / BLK);
  const int k = (int)a.k, chunks = (k + CHUNK - 1) / CHUNK;
  const int n = chunks > gw ? (chunks - gw + NW - 1) / NW : 0;   // this warp's chunks: gw, gw + NW, ..

  // lane: the next chunk's pick and the row that holds it (-1: none)
  int next = gw * CHUNK + lane;
  // listed() only loads; what it loads is looked at one step later, in pick(): a step never waits for the list.
  int64_t listed_tok = -1;
  int listed_row = -1;
  auto listed = [&]() {
    listed_tok = -1;
    const bool more = next < k;
    load_entry(listed_tok, a.idx + bhg * k + next, more);
    load_entry(listed_row, a.slot ? a.slot + bhg * k + next : nullptr, more && a.slot);
    next += more ? NW * CHUNK : 0;
  };
  auto pick = [&](int& tok, int& row) {
    const bool there = listed_tok >= 0 && listed_tok < end;
    tok = there ? (int)listed_tok : -1;
    row = there && a.slot ? listed_row : tok;
  };
  // copies of a chunk into stage s: a lane has piece lane & 15 of rows 2 u + (lane >> 4)
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(st);
  const uint32_t lane_at = (lane >> 4) * KV8_ROW + (lane & 8) * 16 + ((lane & 7) ^ permuted(lane >> 4)) * 16;
  const uint8_t* const from = a.rows + (int64_t)bh * a.row_cap * KV8_ROW + (lane & 15) * 16;
  auto bring = [&](int s, int tok, int row) {
    const uint32_t at = ring + s * (uint32_t)sizeof(Stage);
    st[s].valid[lane] = row;
    if (row >= 0) copy8(at + (uint32_t)offsetof(Stage, scale) + lane * 8, sc + tok / BLK);
#pragma unroll
    for (int u = 0; u < CHUNK / 2; ++u) {
      const int r = __shfl_sync(0xffffffffu, row, 2 * u + (lane >> 4));
      copy16((at + lane_at + u * 2 * KV8_ROW) ^ ((u >> 1 & 3) << 5), from + (int64_t)max(r, 0) * KV8_ROW, r >= 0);
    }
  };
  auto commit = []() { asm volatile("cp.async.commit_group;\n" ::: "memory"); };
  listed();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    int tok, row;
    pick(tok, row);
    listed();
    if (i < n) bring(i, tok, row);
    commit();
  }
  if (lane < 2 * 8) mine.weight[TERMS + lane / 8][lane % 8] = 0;

  // q as terms: one warp, a lane 4 dims; then term g of this lane's dims, 16 j .. and 64 + 16 j ..
  if (warp == 0) {
    float x[4];
    unpack4(qv, dtype, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    const int e = kv8_exponent(top);
    const float inv = top < 0x7F800000u ? pow2i(-e) : __uint_as_float(0x7FFFFFFFu);   // a row with inf or NaN is NaN
    float2 y0 = make_float2(x[0] * inv, x[1] * inv), y1 = make_float2(x[2] * inv, x[3] * inv);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      uint32_t code = 0;
      if (t < TERMS) {
        code = next_term(y0);
        code |= next_term(y1) << 16;
      }
      s_q[t][lane] = code;
    }
    if (lane == 0) s_rs = pow2i(e) * QSCALE;
  }
  __syncthreads();
  const float rs = s_rs;
  uint32_t qf[8];
  *reinterpret_cast<uint4*>(qf) = *reinterpret_cast<const uint4*>(&s_q[g][4 * j]);
  *reinterpret_cast<uint4*>(qf + 4) = *reinterpret_cast<const uint4*>(&s_q[g][16 + 4 * j]);
  const float f0 = exp2f((float)(-8 * j)), f1 = f0 * 0.0625f;          // columns 2 j and 2 j + 1 are terms: 16^-(2 j), ..

  // this lane's pieces within a stage, of keys g (+ 8, 16, 24: the piece permuted alike for + 16) and of values 4 j + e
  const int key_at = g * KV8_ROW + (j ^ permuted(g)) * 16, key8_at = (g + 8) * KV8_ROW + (j ^ permuted(g + 8)) * 16;
  int value_at[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) value_at[e] = (4 * j + e) * KV8_ROW + D + (g ^ permuted(4 * j + e)) * 16;
  float acc[8][4];                                     // dims 16 g + 2 t and + 1; terms 2 j, 2 j + 1
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
  float m = -INFINITY, lm = -1e30f, l = 0.0f;          // m is the warp's; lm, l: of this lane's picks
  int here = 0;                                        // stage of chunk i
  for (int i = 0; i < n; ++i) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                      // chunk i is there; chunk i - 1 has been read
    int tok, row;
    pick(tok, row);
    listed();
    if (i + STAGES - 1 < n) bring(here == 0 ? STAGES - 1 : here - 1, tok, row);
    commit();
    const Stage& s = st[here];
    const uint8_t* const bytes = &s.row[0][0];
    here = here + 1 == STAGES ? 0 : here + 1;
    float c[2][4];                                     // picks g, g + 8; g + 16, g + 24
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* const at = bytes + h * 16 * KV8_ROW;
      uint32_t lo[8], hi[8];
      *reinterpret_cast<uint4*>(lo) = *reinterpret_cast<const uint4*>(at + key_at);
      *reinterpret_cast<uint4*>(lo + 4) = *reinterpret_cast<const uint4*>(at + (key_at ^ 64));
      *reinterpret_cast<uint4*>(hi) = *reinterpret_cast<const uint4*>(at + key8_at);
      *reinterpret_cast<uint4*>(hi + 4) = *reinterpret_cast<const uint4*>(at + (key8_at ^ 64));
#pragma unroll
      for (int e = 0; e < 4; ++e) c[h][e] = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; w += 2) mma(c[h], lo[w], hi[w], lo[w + 1], hi[w + 1], qf[w], qf[w + 1]);
    }
    // scores: the sums over a quad's columns, of pick g + 8 j in lane (g, j)
    float v;
    {
      const float s0 = fmaf(c[0][1], f1, c[0][0] * f0), s1 = fmaf(c[0][3], f1, c[0][2] * f0);
      const float s2 = fmaf(c[1][1], f1, c[1][0] * f0), s3 = fmaf(c[1][3], f1, c[1][2] * f0);
      const bool odd = j & 1, high = j & 2;
      const float x = (odd ? s1 : s0) + __shfl_xor_sync(0xffffffffu, odd ? s0 : s1, 1);
      const float y = (odd ? s3 : s2) + __shfl_xor_sync(0xffffffffu, odd ? s2 : s3, 1);
      v = (high ? y : x) + __shfl_xor_sync(0xffffffffu, high ? x : y, 2);
    }
    const int mypick = g + 8 * j;
    const bool there = s.valid[mypick] >= 0;
    const float2 ks = there ? s.scale[mypick] : make_float2(0.0f, 1.0f);
    v = there ? v * (ks.x * rs) : -INFINITY;
    const float lv = (float)((int)(__float_as_uint(ks.y) >> 23) - 127);
    const float top = redux_max(v + lv);
    if (top > m + SLACK) {                             // the same in every lane; also the first time: m = -inf
      const float f = m == -INFINITY ? 0.0f : ex2(m - top);
      m = top;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] *= f;
    }
    // this pick's weight as terms, and its part of the denominator
    {
      float2 y = make_float2(m == -INFINITY && !(v != v) ? 0.0f : ex2(v + (lv - m + HEAD)), 0.0f);
      uint8_t* const at = reinterpret_cast<uint8_t*>(mine.weight) + mypick;
#pragma unroll
      for (int t = 0; t < TERMS; ++t) at[t * CHUNK] = (uint8_t)next_term(y);
      const float d = v - lm, p = ex2(-fabsf(d));
      l = d > 0.0f ? fmaf(l, p, 1.0f) : l + p;
      lm = fmaxf(lm, v);
    }
    uint32_t x[8][4];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<uint4*>(x[e]) = *reinterpret_cast<const uint4*>(bytes + (e >> 2) * 16 * KV8_ROW + value_at[e & 3]);
    __syncwarp();
    const uint32_t b0 = mine.weight[g][j], b1 = mine.weight[g][4 + j];
#pragma unroll
    for (int u = 0; u < 4; ++u) {                      // bytes 4 u .. of the lane's 16 dims
      uint32_t lo[4], hi[4];
      transpose4(x[0][u], x[1][u], x[2][u], x[3][u], lo);
      transpose4(x[4][u], x[5][u], x[6][u], x[7][u], hi);
      mma(acc[2 * u], lo[0], lo[1], hi[0], hi[1], b0, b1);
      mma(acc[2 * u + 1], lo[2], lo[3], hi[2], hi[3], b0, b1);
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  // the warp's state: picks are spread over its lanes, the terms of an output over the columns of a quad
  const float ref = redux_max(lm);
  l = warp_sum(l * ex2(lm - ref));
#pragma unroll
  for (int t = 0; t < 8; ++t) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float o = fmaf(acc[t][e + 1], f1, acc[t][e] * f0);
      o += __shfl_xor_sync(0xffffffffu, o, 1);
      acc[t][e] = o + __shfl_xor_sync(0xffffffffu, o, 2);
    }
  }
  cluster.barrier_wait();
  float *dm = cluster.map_shared_rank(s_m, 0), *dlm = cluster.map_shared_rank(s_lm, 0);
  float *dl = cluster.map_shared_rank(s_l, 0), *da = cluster.map_shared_rank(&s_acc[0][0], 0);
  if (lane == 0) dm[gw] = m, dlm[gw] = ref, dl[gw] = l;
  if (j == 0) {
    float4* dst = reinterpret_cast<float4*>(da + gw * D + 16 * g);
#pragma unroll
    for (int t = 0; t < 8; t += 2) dst[t / 2] = make_float4(acc[t][0], acc[t][2], acc[t + 1][0], acc[t + 1][2]);
  }
  cluster.sync();
  if (crank != 0) return;
  // lane = warp state: its factor, then every thread a dim or more
  float M = lane < NW ? s_lm[lane] : -1e30f;
  M = warp_max(M);
  const float L = warp_sum(lane < NW ? s_l[lane] * ex2(s_lm[lane] - M) : 0.0f);
  const float factor = lane < NW && s_m[lane] != -INFINITY ? exp2f(s_m[lane] - HEAD - M) : 0.0f;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float O = 0.0f;
#pragma unroll 8
    for (int v = 0; v < NW; ++v) {
      const float f = __shfl_sync(0xffffffffu, factor, v);
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
  const int smem = pw * (int)sizeof(Warp) + pw * cs * D * (int)sizeof(float);
  constexpr int most = MAX_PW * (int)sizeof(Warp) + MAX_PW * MAX_CS * D * (int)sizeof(float);
  static std::atomic<uint64_t> told{0};
  const int r = allow_smem(picks_kernel, most, told, "kv8_attend_picks");
  if (r != FATHOM_OK) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)heads, (unsigned)cs);
  cfg.blockDim = dim3((unsigned)pw * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)cs;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;     // may start while the kernel before it ends
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
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
  // as many warps per head as the GPU holds at once, 32 at most, and no more than there are chunks
  const int64_t heads = B * Hkv * G, chunks = cdiv(k, CHUNK), fit = (int64_t)WARPS_PER_SM * sm_count() / heads;
  int64_t warps = fit < chunks ? fit : chunks;
  warps = warps < 1 ? 1 : warps > MAX_PW * MAX_CS ? MAX_PW * MAX_CS : warps;
  const int pw = warps > 2 * MAX_CS ? 4 : warps > MAX_CS ? 2 : 1;
  const int64_t cs = cdiv(warps, pw) * pw <= fit ? cdiv(warps, pw) : warps / pw;
  return launch_picks(q, dtype, a, heads, pw, (int)(cs < 1 ? 1 : cs), out, st);
}
