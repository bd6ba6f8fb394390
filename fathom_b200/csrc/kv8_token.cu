// Attention of a few query rows per KV head over the whole 8-bit cache (layout in kv8.cuh): single tokens and drafts.
//
// Bound by the cache's bytes: 256 per token and KV head.  CUDA cores cannot keep up with them (each byte meets
// every query head of its group), so the e4m3 codes go to the tensor cores as they lie in memory:
//
//   S^T [128 tokens x rows]  = K [128 tokens x 128] q^T         K-major tile, straight from TMA
//   O^T [128 dims x rows]   += V^T [128 dims x 128 tokens] P^T   the value tile read MN-major, straight from TMA
//
// The other operand of an e4m3 product has to be e4m3 too.  A row of q is split into terms q = s (t1 + t2 / 16 +
// t3 / 256), each the rounding of what the ones before left (4 significant bits a term: 2 terms hold a
// bf16 exactly, 3 an fp16), and so is a row of the weights; the terms are further columns of the product,
// which the tensor cores have to spare: with M = 128 tokens a tile of 32 KB takes them ~250 cycles, its
// bytes ~1400.  A score is then the sum of its term columns times the block's key scale; weights carry the
// block's value scale (a power of two) in their exponent, so nothing is ever rescaled.
//
// Softmax, thread = token: with m the running reference of a row's (score + log2 of the value scale), a weight is
// 2^(s + log2 vs - m); m moves only when a tile exceeds it by 2^6 (then O^T in tensor memory is rescaled), which
// leaves e4m3's range room on both sides.  The denominator is kept per thread in fp32 with a reference of its
// own, because the value scale must not enter it.
//
// Work: the 128-token tiles of all rows bh in a line, cut into equal contiguous shares, one per CTA, whatever
// the lengths; a row's parts in different CTAs are joined by a second kernel in a fixed order.
#include "kv8.cuh"
#include "kv8_attn.cuh"
#include "tc.cuh"

namespace fathom {
namespace kv8 {
namespace {

constexpr int TILE = 128;                        // tokens per tile
constexpr int TERMS = 3;                         // e4m3 terms of a weight
constexpr int SOFT = 128;                        // softmax threads (warps 0-3); warp 4 loads, warp 5 multiplies
constexpr int THREADS = SOFT + 64;
constexpr int STAGE_BYTES = 2 * TILE * D;        // key tile, value tile
constexpr float SLACK = 6.0f;                    // a tile may exceed the reference by 2^6
constexpr float HEAD = 2.0f;                     // weights at the reference are 4: 2^(HEAD + SLACK) = 256 <= 448

constexpr int up16(int n) { return (n + 15) / 16 * 16; }

template <int NR, int QT> struct Shape {
  static constexpr int NQ = up16(NR * QT), NP = up16(NR * TERMS);
  static constexpr int COLS = 2 * NQ + NP;
  static constexpr int TMEM = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr int STAGES = NR <= 16 ? 6 : 5;
  // byte offsets in dynamic shared memory (1024-byte aligned operands first)
  static constexpr int Q = STAGES * STAGE_BYTES, P = Q + NQ * D, END = P + 2 * NP * TILE;
  static constexpr int SMEM = END + 1024;        // room to align
};

// This CTA's place in the line of tiles.
struct Share {
  int64_t first, count;      // tiles
  int64_t share;             // tiles per CTA
  int bh;                    // row of the first tile
  int64_t tile;              // its tile within the row
};

__device__ __forceinline__ int64_t tiles_of(const Args& a, int b) { return (seq_end(a, b) + TILE - 1) / TILE; }

// One warp: tiles of all rows, and the row (b, all its heads) that holds tile `at` of the line (b = B past the end).
__device__ int64_t locate(const Args& a, int64_t at, int* b_out, int64_t* before_out) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0, before = 0;
  int found = a.B;
  if (!a.end_dev) {
    const int64_t per = tiles_of(a, 0) * a.Hkv;
    total = per * a.B;
    if (per > 0 && at < total) {
      found = (int)(at / per);
      before = (int64_t)found * per;
    }
  } else {
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int64_t mine = b0 + lane < a.B ? tiles_of(a, b0 + lane) * a.Hkv : 0;
      int64_t x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, total + x > at && total + x - mine <= at);
      if (hit) {
        const int l = __ffs(hit) - 1;
        found = b0 + l;
        before = total + __shfl_sync(0xffffffffu, x - mine, l);
      }
      total += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  *b_out = found;
  *before_out = before;
  return total;
}

template <typename T> __device__ __forceinline__ void load4(const T* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (float)e[i];
}

template <typename T, int NR, int QT>
__global__ void __launch_bounds__(THREADS, 1) token_kernel(const __grid_constant__ CUtensorMap map, const Args a) {
  using S = Shape<NR, QT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = tc::smem_u32(smem);
  __shared__ __align__(8) uint64_t bars[2 * S::STAGES + 10];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gave_up;
  __shared__ Share s_share;
  __shared__ float s_rs[NR];                     // scale of a row's scores: 2^e log2(e) / sqrt(128)
  __shared__ float s_red[4][NR], s_redl[4][NR];
  const uint32_t bar0 = tc::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (S::STAGES + s); };
  const uint32_t B = bar0 + 16 * S::STAGES;
  auto s_full = [&](int i) { return B + 8 * i; };
  auto s_free = [&](int i) { return B + 16 + 8 * i; };
  auto p_full = [&](int i) { return B + 32 + 8 * i; };
  auto p_free = [&](int i) { return B + 48 + 8 * i; };
  const uint32_t q_full = B + 64, drain = B + 72;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < S::STAGES; ++s) tc::mbar_init(full(s), 1), tc::mbar_init(empty(s), 1);
    for (int i = 0; i < 2; ++i)
      tc::mbar_init(s_full(i), 1), tc::mbar_init(s_free(i), 4), tc::mbar_init(p_full(i), 4), tc::mbar_init(p_free(i), 1);
    tc::mbar_init(q_full, 4);
    tc::mbar_init(drain, 1);
    tc::fence_mbar_init();
    s_gave_up = 0;
  }
  if (warp == 0) {
    int b;
    int64_t before;
    const int64_t total = locate(a, 0, &b, &before);
    const int64_t share = (total + gridDim.x - 1) / gridDim.x, first = share * blockIdx.x;
    locate(a, first, &b, &before);
    if (lane == 0) {
      Share w{first, total - first < share ? total - first : share, share, 0, 0};
      if (w.count > 0) {
        const int64_t nt = tiles_of(a, b);
        w.bh = b * a.Hkv + (int)((first - before) / nt);
        w.tile = (first - before) % nt;
      }
      s_share = w;
    }
  }
  if (warp == 5) tc::tmem_alloc(tc::smem_u32(&s_tmem), S::TMEM);
  // operand columns that no row writes stay 0
  for (int i = tid; i < (S::END - S::Q) / 16; i += THREADS)
    reinterpret_cast<uint4*>(smem + S::Q)[i] = make_uint4(0, 0, 0, 0);
  tc::fence_async_smem();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tm = s_tmem;
  const Share w = s_share;
  volatile int* gave_up = &s_gave_up;
  const uint32_t tm_o = tm + 2 * S::NQ;          // S^T of even and odd tiles, then O^T

  if (warp == 4) {
    // ---- loads: the share's tiles in order, as stages come free
    if (lane == 0) {
      int bh = w.bh;
      int64_t t = w.tile, nt = w.count > 0 ? tiles_of(a, bh / a.Hkv) : 0, i = 0;
      for (; i < w.count; ++i) {
        while (t >= nt) {
          ++bh;
          t = 0;
          nt = tiles_of(a, bh / a.Hkv);
        }
        const int s = (int)(i % S::STAGES);
        if (!tc::mbar_wait(empty(s), ((i / S::STAGES) & 1) ^ 1, gave_up)) break;
        tc::mbar_expect_tx(full(s), STAGE_BYTES);
        tc::tma_load_3d(sbase + s * STAGE_BYTES, &map, 0, (int)(t * TILE), bh, full(s));
        tc::tma_load_3d(sbase + s * STAGE_BYTES + TILE * D, &map, D, (int)(t * TILE), bh, full(s));
        ++t;
      }
      if (*gave_up) {          // copies in flight land before the CTA ends (bounded: the flag is up, so by time alone)
        for (int64_t j = i > S::STAGES ? i - S::STAGES : 0; j < i; ++j) {
          const unsigned long long t0 = tc::now_ns();
          while (!tc::mbar_try(full((int)(j % S::STAGES)), (j / S::STAGES) & 1) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
        }
      }
    }
  } else if (warp == 5) {
    // ---- products: S^T of tile i, then O^T of tile i - 1, whose weights were made meanwhile
    if (lane == 0) {
      constexpr uint32_t id_s = tc::instr(S::NQ, false, false), id_o = tc::instr(S::NP, true, false);
      const uint64_t dq = tc::operand(sbase + S::Q);
      int64_t t = w.tile, nt = w.count > 0 ? tiles_of(a, w.bh / a.Hkv) : 0;
      int bh = w.bh;
      int64_t seg = 0;                            // rows begun: each fills q once
      bool ok = true, fresh_prev = true;          // fresh: a row's first tile, O^T starts at 0
      auto scores = [&](int64_t i) {
        const int s = (int)(i % S::STAGES), k = (int)(i & 1);
        if (!tc::mbar_wait(full(s), (i / S::STAGES) & 1, gave_up)) return false;
        if (!tc::mbar_wait(s_free(k), ((i >> 1) & 1) ^ 1, gave_up)) return false;
        tc::fence_after();
        const uint64_t dk = tc::operand(sbase + s * STAGE_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)       // 32 dims a step: 32 bytes along the swizzled rows
          tc::mma_fp8(tm + k * S::NQ, dk + kk * 2, dq + kk * 2, id_s, kk > 0);
        tc::mma_commit(s_full(k));
        return true;
      };
      auto values = [&](int64_t i, bool accumulate) {
        const int s = (int)(i % S::STAGES), k = (int)(i & 1);
        if (!tc::mbar_wait(p_full(k), (i >> 1) & 1, gave_up)) return false;
        tc::fence_after();
        const uint64_t dv = tc::operand(sbase + s * STAGE_BYTES + TILE * D), dp = tc::operand(sbase + S::P + k * S::NP * TILE);
#pragma unroll
        for (int kk = 0; kk < TILE / 32; ++kk)    // 32 tokens a step: 4 groups of 8 value rows
          tc::mma_fp8(tm_o, dv + kk * (32 * D / 16), dp + kk * 2, id_o, kk > 0 || accumulate);
        tc::mma_commit(empty(s));
        tc::mma_commit(p_free(k));
        return true;
      };
      for (int64_t i = 0; i <= w.count && ok; ++i) {
        bool next = i < w.count, fresh = i == 0;
        while (next && t >= nt) {
          ++bh;
          t = 0;
          nt = tiles_of(a, bh / a.Hkv);
          fresh = true;
        }
        // a row's q takes the place of the last one's, which needs that row's last product done
        if (next && !fresh) ok = scores(i);
        if (ok && i > 0) ok = values(i - 1, !fresh_prev);
        if (ok && next && fresh) ok = tc::mbar_wait(q_full, seg++ & 1, gave_up) && scores(i);
        fresh_prev = fresh;
        ++t;
      }
      if (*gave_up) {
        tc::mma_commit(drain);
        const unsigned long long t0 = tc::now_ns();
        while (!tc::mbar_try(drain, 0) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
      }
    }
  } else {
    // ---- softmax: thread = token of the tile; lane of tensor memory = token of S^T, dim of O^T
    const int R = a.G * (int)a.T;
    const uint32_t my = (uint32_t)(warp * 32) << 16;
    int bh = w.bh;
    int64_t t = w.tile, i = 0;
    bool ok = true, bad = false;                  // ok: this thread's waits; bad: some thread's gave up (uniform)
    while (i < w.count) {
      const int b = bh / a.Hkv, h = bh % a.Hkv;
      const int64_t end = seq_end(a, b), nt = (end + TILE - 1) / TILE;
      if (t >= nt) {
        ++bh;
        t = 0;
        continue;
      }
      // this row's queries as terms: a warp takes every fourth, a lane 4 dims.  The products of the row before are
      // complete (its O^T was read below), so its q may go.
      for (int r = warp; r < R; r += 4) {
        const int g = r / (int)a.T, tt = r % (int)a.T;
        float x[4];
        load4(reinterpret_cast<const T*>(a.q) + b * a.qb + ((int64_t)h * a.G + g) * a.qh + tt * a.qt + lane * 4, x);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
        top = __reduce_max_sync(0xffffffffu, top);
        const int e2 = kv8_exponent(top);
        const float inv = pow2i(-e2);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= inv;
#pragma unroll
        for (int term = 0; term < QT; ++term) {
          const uint32_t code = kv8_encode2(x[0], x[1]) | kv8_encode2(x[2], x[3]) << 16;
          const int n = term * NR + r;
          *reinterpret_cast<uint32_t*>(smem + S::Q + n * D + (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4) = code;
          const float2 lo = kv8_decode2(code), hi = kv8_decode2(code >> 16);
          x[0] = (x[0] - lo.x) * 16.0f, x[1] = (x[1] - lo.y) * 16.0f;
          x[2] = (x[2] - hi.x) * 16.0f, x[3] = (x[3] - hi.y) * 16.0f;
        }
        if (lane == 0) s_rs[r] = pow2i(e2) * QSCALE;
      }
      tc::fence_async_smem();
      tc::named_sync(1, SOFT);
      if (lane == 0) tc::mbar_arrive(q_full);
      float m[NR], lm[NR], l[NR];                 // the row's reference, this thread's denominator and its reference
#pragma unroll
      for (int r = 0; r < NR; ++r) m[r] = -INFINITY, lm[r] = -1e30f, l[r] = 0.0f;
      const int64_t t0 = t;
      const float2* sc = reinterpret_cast<const float2*>(a.scales) + (int64_t)bh * (a.cap / BLK);
      for (; t < nt && i < w.count && !bad; ++t, ++i) {
        const int k = (int)(i & 1);
        const int64_t tok = t * TILE + tid;
        const float2 ks = tok < end ? sc[tok / BLK] : make_float2(0.0f, 1.0f);
        const float lv = (float)((int)(__float_as_uint(ks.y) >> 23) - 127);      // log2 of the value scale
        ok = ok && tc::mbar_wait(s_full(k), (i >> 1) & 1, gave_up);
        __syncwarp();
        tc::fence_after();
        float s[NR];
        {
          uint32_t c[QT][NR];
#pragma unroll
          for (int term = 0; term < QT; ++term) tc::Tmem<NR>::ld(tm + k * S::NQ + my + term * NR, c[term]);
          tc::wait_ld();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(s_free(k));
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float v = __uint_as_float(c[QT - 1][r]);
#pragma unroll
            for (int term = QT - 2; term >= 0; --term) v = fmaf(v, 0.0625f, __uint_as_float(c[term][r]));
            s[r] = r < R ? v * (ks.x * s_rs[r < R ? r : 0]) : -INFINITY;
          }
        }
        // keys that a row does not see: past the end, or in the last T - 1 after its own
        bool void_row = tok >= end;
        if (t * TILE + TILE > end - (a.T - 1)) {
          const int64_t room = end - tok - (a.T - 1);      // seen by query tt while room + tt > 0
          int tt = 0;
          bool nan_v = false;
          uint4* vrow = reinterpret_cast<uint4*>(smem + (i % S::STAGES) * STAGE_BYTES + TILE * D + tid * D);
          if (a.T > 1 && !void_row) {
            // the mask differs between rows here, and 0 * NaN would reach rows that do not see the key: a value row
            // with a NaN leaves the product, and the rows that see it become NaN by their denominators
            tc::mbar_wait(full((int)(i % S::STAGES)), (i / S::STAGES) & 1, gave_up);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              const uint4 v = vrow[c];
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) nan_v = nan_v || __vcmpeq4(x[e] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
            }
          }
          if (void_row || nan_v) {
            tc::mbar_wait(full((int)(i % S::STAGES)), (i / S::STAGES) & 1, gave_up);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) vrow[c] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            if (room + tt <= 0) s[r] = -INFINITY;
            else if (nan_v && r < R) l[r] = __uint_as_float(0x7FFFFFFFu);
            tt = tt + 1 == a.T ? 0 : tt + 1;
          }
        }
        bool above = false;
#pragma unroll
        for (int r = 0; r < NR; ++r) above = above || s[r] + lv > m[r] + SLACK;
        if (tc::named_or(1, SOFT, above || !ok)) {
          bad = tc::named_or(1, SOFT, !ok);
          // some row outgrew its reference: the tile's largest becomes every row's
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float mx = warp_max(s[r] + lv);
            if (lane == 0) s_red[warp][r] = mx;
          }
          tc::named_sync(1, SOFT);
          float f[NR];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float mx = fmaxf(fmaxf(s_red[0][r], s_red[1][r]), fmaxf(s_red[2][r], s_red[3][r]));
            mx = fmaxf(mx, m[r]);
            f[r] = m[r] == -INFINITY ? 0.0f : exp2f(m[r] - mx);
            m[r] = mx;
          }
          tc::named_sync(1, SOFT);
          if (t > t0) {
            ok = ok && tc::mbar_wait(p_free((int)((i - 1) & 1)), ((i - 1) >> 1) & 1, gave_up);   // O^T of the tiles before
            __syncwarp();
            tc::fence_after();
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
              uint32_t o[NR];
              tc::Tmem<NR>::ld(tm_o + my + term * NR, o);
              tc::wait_ld();
#pragma unroll
              for (int r = 0; r < NR; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * f[r]);
              tc::Tmem<NR>::st(tm_o + my + term * NR, o);
            }
            tc::wait_st();
          }
        }
        // weights as terms into the operand buffer, once the product of two tiles before has read it
        ok = ok && tc::mbar_wait(p_free(k), ((i >> 1) & 1) ^ 1, gave_up);
        uint8_t* pb = smem + S::P + k * S::NP * TILE;
#pragma unroll
        for (int r = 0; r < NR; r += 2) {
          float x[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float sv = s[r + e], mv = m[r + e];
            x[e] = mv == -INFINITY && !(sv != sv) ? 0.0f : ex2(sv + lv - mv + HEAD);
            const float d = sv - lm[r + e], p = ex2(-fabsf(d));
            l[r + e] = d > 0.0f ? fmaf(l[r + e], p, 1.0f) : l[r + e] + p;
            lm[r + e] = fmaxf(lm[r + e], sv);
          }
          if (r >= R) continue;
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            const uint32_t code = kv8_encode2(x[0], x[1]);
            const int n = term * NR + r;
            pb[n * TILE + (((tid >> 4) ^ (n & 7)) << 4) + (tid & 15)] = (uint8_t)code;
            pb[(n + 1) * TILE + (((tid >> 4) ^ ((n + 1) & 7)) << 4) + (tid & 15)] = (uint8_t)(code >> 8);
            const float2 c = kv8_decode2(code);
            x[0] = (x[0] - c.x) * 16.0f, x[1] = (x[1] - c.y) * 16.0f;
          }
        }
        tc::fence_async_smem();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(k));
      }
      // the row's part (or whole): denominators over the threads, O^T out of tensor memory
      if (t > t0) ok = ok && tc::mbar_wait(p_free((int)((i - 1) & 1)), ((i - 1) >> 1) & 1, gave_up);
      __syncwarp();
      tc::fence_after();
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float mx = warp_max(lm[r]);
        const float sum = warp_sum(l[r] * ex2(lm[r] - mx));
        if (lane == 0) s_red[warp][r] = mx, s_redl[warp][r] = sum;
      }
      bad = tc::named_or(1, SOFT, !ok);
      const bool whole = t0 == 0 && (t == nt || bad);
      uint32_t o[TERMS][NR];
#pragma unroll
      for (int term = 0; term < TERMS; ++term) tc::Tmem<NR>::ld(tm_o + my + term * NR, o[term]);
      tc::wait_ld();
      tc::fence_before();
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r >= R) continue;
        float mx = s_red[0][r], sum = 0.0f;
#pragma unroll
        for (int v = 1; v < 4; ++v) mx = fmaxf(mx, s_red[v][r]);
#pragma unroll
        for (int v = 0; v < 4; ++v) sum += s_redl[v][r] * ex2(s_red[v][r] - mx);
        float x = __uint_as_float(o[TERMS - 1][r]);
#pragma unroll
        for (int term = TERMS - 2; term >= 0; --term) x = fmaf(x, 0.0625f, __uint_as_float(o[term][r]));
        // O^T is relative to m - HEAD: bring it to the denominator's reference
        x = m[r] == -INFINITY ? 0.0f : x * exp2f(m[r] - HEAD - mx);
        if (bad) x = __uint_as_float(0x7FFFFFFFu);
        const int g = r / (int)a.T, tt = r % (int)a.T;
        if (whole) {
          T* op = reinterpret_cast<T*>(a.out) + b * a.ob + ((int64_t)h * a.G + g) * a.oh + tt * a.ot;
          from_f32(bad ? x : sum == 0.0f ? 0.0f : x / sum, op + tid);
        } else {
          float* part = a.part + (((int64_t)blockIdx.x + bh) * R + r) * PART;
          part[tid] = x;
          if (tid == 0) part[D] = mx, part[D + 1] = sum;
        }
      }
      tc::named_sync(1, SOFT);                    // s_red and s_rs are read
      if (bad) {                                  // nothing more is computed: NaN for every row of the share
        i += nt - t;
        t = nt;
      }
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 5) tc::tmem_free(tm, S::TMEM);
  if (tid == 0 && s_gave_up) atomicAdd(a.timeouts, 1ull);
}

// Joins a row's parts: CTA = (bh, query row), thread = dim.  Rows of one part were written whole.
template <typename T>
__global__ void __launch_bounds__(D) token_join_kernel(const Args a, int ctas) {
  __shared__ int64_t s_before, s_total;
  const int R = a.G * (int)a.T;
  const int64_t bh = blockIdx.x / R;
  const int r = (int)(blockIdx.x % R), b = (int)(bh / a.Hkv), h = (int)(bh % a.Hkv);
  const int64_t nt = tiles_of(a, b);
  if (threadIdx.x < 32) {
    // tiles of the sequences before b, and of all
    int64_t before = 0, total = 0;
    if (!a.end_dev) {
      before = nt * a.Hkv * b, total = nt * a.Hkv * a.B;
    } else {
      for (int j = threadIdx.x; j < a.B; j += 32) {
        const int64_t x = tiles_of(a, j) * a.Hkv;
        total += x;
        if (j < b) before += x;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
      }
    }
    if (threadIdx.x == 0) s_before = before, s_total = total;
  }
  __syncthreads();
  const int64_t share = (s_total + ctas - 1) / ctas, first = s_before + h * nt;
  const int g = r / (int)a.T, tt = r % (int)a.T;
  T* op = reinterpret_cast<T*>(a.out) + b * a.ob + ((int64_t)h * a.G + g) * a.oh + tt * a.ot + threadIdx.x;
  if (nt == 0) {
    from_f32(0.0f, op);
    return;
  }
  const int64_t c0 = first / share, c1 = (first + nt - 1) / share;
  if (c0 == c1) return;
  float M = -INFINITY, L = 0.0f, O = 0.0f;
  for (int64_t c = c0; c <= c1; ++c) M = fmaxf(M, a.part[((c + bh) * R + r) * PART + D]);
  for (int64_t c = c0; c <= c1; ++c) {
    const float* p = a.part + ((c + bh) * R + r) * PART;
    const float e = exp2f(p[D] - M);
    L = fmaf(p[D + 1], e, L);
    O = fmaf(p[threadIdx.x], e, O);
  }
  from_f32(L == 0.0f ? 0.0f : O / L, op);
}

template <typename T, int NR, int QT>
int launch(const CUtensorMap& map, const Args& a, int ctas, cudaStream_t st) {
  using S = Shape<NR, QT>;
  static_assert(S::SMEM <= 227 * 1024 - 2048, "shared memory");
  const cudaError_t e =
      cudaFuncSetAttribute(token_kernel<T, NR, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return set_error(FATHOM_ERR_CUDA, "kv8_attend: %s", cudaGetErrorString(e));
  token_kernel<T, NR, QT><<<ctas, THREADS, S::SMEM, st>>>(map, a);
  token_join_kernel<T><<<(unsigned)((int64_t)a.B * a.Hkv * a.G * a.T), D, 0, st>>>(a, ctas);
  return check_launch("kv8_attend");
}

template <typename T, int QT>
int launch_rows(const CUtensorMap& map, const Args& a, int ctas, cudaStream_t st) {
  const int64_t R = a.G * a.T;
  if (R <= 4) return launch<T, 4, QT>(map, a, ctas, st);
  if (R <= 8) return launch<T, 8, QT>(map, a, ctas, st);
  if (R <= 16) return launch<T, 16, QT>(map, a, ctas, st);
  return launch<T, 32, QT>(map, a, ctas, st);
}

}  // namespace

// One CTA per SM, but no more than there can be tiles.
int token_ctas(const Args& a) {
  const int64_t most = (int64_t)a.B * a.Hkv * cdiv(a.end_dev ? a.cap : a.end, TILE);
  const int64_t sms = sm_count();
  return (int)(most < 1 ? 1 : most < sms ? most : sms);
}

size_t token_workspace(int64_t BH, int64_t R) { return (size_t)((sm_count() + BH) * R * PART * sizeof(float)); }

int token_attend(const CUtensorMap& map, const Args& a, int dtype, cudaStream_t st) {
  const int ctas = token_ctas(a);
  return dtype == FATHOM_DTYPE_BF16 ? launch_rows<__nv_bfloat16, 2>(map, a, ctas, st)
                                    : launch_rows<__half, 3>(map, a, ctas, st);
}

}  // namespace kv8
}  // namespace fathom
