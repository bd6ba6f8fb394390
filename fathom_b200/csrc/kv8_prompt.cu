// Attention of many query rows per KV head over the 8-bit cache (layout in kv8.cuh): prompt chunks, long drafts.
//
// Bound by the tensor cores, and as closely by the special-function units: a 128-token tile against 256 query
// rows is 2 x 2 products of 128 x 128 x 128, ~2048 cycles, and 32768 exponentials at 16 a cycle.  Rows are
// the (token, head) pairs of one KV head, token-major, so G heads share every tile.  Per CTA:
//
//   S_i [128 rows x 128 tokens] = (q1 + q2 [+ q3]) K^T   8-bit products: q as a sum of an e4m3 term (4 bits) and e5m2
//                                                        ones, whose 3 bits each hold what a rounding leaves of 8 and
//                                                        of 11, and whose range goes on where e4m3's ends: a bf16
//                                                        exactly or to 2^-21 of its row's largest, an fp16 to 2^-25.
//                                                        The key tile comes straight from TMA; 2 terms at twice the
//                                                        rate cost one 16-bit product, and no key is converted
//   O_i [128 rows x 128 dims]  += P_i V                  f16 x f16: an e4m3 value is exact in f16; weights in
//                                                        tensor memory over the scores they came from
//
// for the two halves i of the rows, in turn: while 8 warps take the softmax of one half's scores, the tensor cores work for
// the other.  4 more warps turn value tiles into f16.  The key scale multiplies the score and the value scale 2^ev, a
// constant of each 64-token block, enters the weight's exponent, so a row sees its own range whatever other blocks
// hold.  Softmax, two threads per row, one for each block of a tile: m, the reference of s + ev, follows the row's
// maximum only when that exceeds it by 2^12 (then O is rescaled; at 2^7 that cost 3%); weights are 2^(s + ev - m + 3), at
// most 2^15 in f16 (the product's other operand is f16, and the outputs have 8 or 11 bits), rounded to 11 bits down to 2^-17 of the reference and to steps of 2^-27 of it below; sums in fp32.  The
// denominator has a reference of its own, without the value scales: each block's sum of weights enters it once.  Parts
// and outputs are weighted means, whatever the values' range is.  (One thread per row, 8 softmax warps instead
// of 16: 1.34 ms against 0.95 for the chunk below, the steps of a tile waiting for each other; exponentials partly by
// polynomial: slower, the warps' issue is as near its limit as the special-function units.)
//
// Measured, 2048 queries at 32k, 8 KV heads, G = 4, bf16: single calls 1.04-1.07 ms = 1.06-1.09 PFLOP/s, 0.65 of the
// measured 16-bit product rate; back to back 1.04-1.13 ms under the power cap, 0.71-0.77 of the sustained rate.
//
// Work: the tiles of all (bh, 256 rows) items in a line, cut into equal contiguous shares, one per CTA; an item cut
// by a share's end leaves parts in the workspace, which a second kernel joins in a fixed order.
#include "kv8_line.cuh"

namespace fathom {
namespace kv8 {
namespace {

constexpr int HALF = ROWS / 2;               // query rows that share an accumulator
constexpr int KSTAGES = 3, VSTAGES = 2;
constexpr int KBYTES = TILE * D, VBYTES = 2 * TILE * D;
constexpr int SOFT = 256;                    // softmax threads of a half: two per row, one for each 64-token block of a tile
constexpr int THREADS = 2 * SOFT + 256;      // warps 0-7, 8-15: softmax; 16-19: values; 20: products; 21: key loads
constexpr float SLACK = 12.0f;               // a row may exceed its reference by 2^12
constexpr float HEAD = 3.0f;                 // weights at the reference are 2^3
// registers per thread of the softmax, value and other warps: together no more than the 768 * 80 of the launch
constexpr int REG_LAUNCH = 80, REG_SOFT = 88, REG_VALUE = 64, REG_OTHER = 64;
static_assert(4 * REG_SOFT + REG_VALUE + REG_OTHER <= 6 * REG_LAUNCH, "register split");
constexpr int PIECE = 4;                     // tiles (~1.7 us each) that beginning and ending a piece takes
constexpr int LEAST = 4;                     // so shares are no shorter
constexpr int WHOLE = 6;                     // tiles that take no longer than their halves and the second kernel
constexpr float FAR = 60.0f;                 // below 2^-60 of the reference no weight of a block is above f16's least

template <int QT> struct Shape {
  static constexpr int Q = 0, K = 2 * QT * HALF * D, V = K + KSTAGES * KBYTES, END = V + VSTAGES * VBYTES;
  static constexpr int SMEM = END + 1024;
};

// log2 of a power of two, as a number (no conversion instruction: those share the special-function units).
__device__ __forceinline__ float log2_of(float scale) {
  return __uint_as_float(0x4B000000u | __float_as_uint(scale) >> 23) - (8388608.0f + 127.0f);
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int N> __device__ __forceinline__ void reg_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

// What a CTA's share left to join, after the parts (two slots per CTA): see prompt_join_kernel.
__device__ __forceinline__ int4* cuts_of(const Args& a) {
  return reinterpret_cast<int4*>(a.part + 2 * (int64_t)a.ctas * ROWS * PART);
}

template <typename T, int QT>
__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(const __grid_constant__ CUtensorMap map,
                                                           const __grid_constant__ Args a) {
  using S = Shape<QT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = tc::smem_u32(smem);
  __shared__ __align__(8) uint64_t bars[2 * KSTAGES + 2 * VSTAGES + 7];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gave_up;
  __shared__ __align__(4) uint8_t s_nan[VSTAGES][TILE];   // tokens whose value holds a NaN (tiles whose mask differs by row)
  __shared__ float s_rs[2][HALF];                  // scale of a row's scores: 2^e log2(e) / sqrt(128)
  __shared__ float2 s_pair[2 * SOFT];              // by thread: what a row's two threads (tid, tid ^ HALF) tell each other
  const uint32_t bar = tc::smem_u32(bars);
  auto k_full = [&](uint32_t i) { return bar + 8 * (i % KSTAGES); };
  auto k_free = [&](uint32_t i) { return bar + 8 * (KSTAGES + i % KSTAGES); };
  const uint32_t bar2 = bar + 16 * KSTAGES;
  auto v_full = [&](uint32_t i) { return bar2 + 8 * (i % VSTAGES); };
  auto v_free = [&](uint32_t i) { return bar2 + 8 * (VSTAGES + i % VSTAGES); };
  const uint32_t bar3 = bar2 + 16 * VSTAGES;
  auto s_full = [&](int h) { return bar3 + 8 * h; };
  auto p_full = [&](int h) { return bar3 + 16 + 8 * h; };
  auto q_full = [&](int h) { return bar3 + 32 + 8 * h; };
  const uint32_t drain = bar3 + 48;
  const int tid = threadIdx.x, lane = tid & 31, warp = (int)tc::uniform(tid >> 5), group = warp >> 2;
  volatile int* gave_up = &s_gave_up;

  if (tid == 0) {
    for (int i = 0; i < KSTAGES; ++i) tc::mbar_init(k_full(i), 1), tc::mbar_init(k_free(i), 1);
    for (int i = 0; i < VSTAGES; ++i) tc::mbar_init(v_full(i), 4), tc::mbar_init(v_free(i), 1);
    for (int h = 0; h < 2; ++h)
      tc::mbar_init(s_full(h), 1), tc::mbar_init(p_full(h), SOFT / 32), tc::mbar_init(q_full(h), SOFT / 32);
    tc::mbar_init(drain, 1);
    tc::fence_mbar_init();
    s_gave_up = 0;
  }
  if (warp == 20) tc::tmem_alloc(tc::smem_u32(&s_tmem), 512);
  tc::wait_dependency();
  int count, share;
  const Place place = my_share(a, &count, &share);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  tc::launch_dependents();
  const uint32_t tm = s_tmem;                      // S_0, S_1, O_0, O_1: 128 columns each
  Walk<> w(a, place, count);

  if (group < 4) {
    // ---- softmax of half h2: two threads per row, thread `ch` for the tile's 64-token block ch and dims 64 ch ..
    reg_more<REG_SOFT>();
    const int h2 = group >> 1, ch = group & 1, r = tid & (HALF - 1);
    const int pair_bar = 1 + h2 * 4 + (warp & 3);  // the two warps of 32 rows
    const uint32_t my = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tm_s = tm + h2 * 128 + 64 * ch + my, tm_o = tm + 256 + h2 * 128 + 64 * ch + my;
    uint32_t phase = 0, vt = 0;                    // completions of s_full seen; tiles seen
    bool ok = true;
    int4 cut = make_int4(-1, 0, 0, 0);             // the item that this share begins and another ends
    while (w.next()) {
      if (w.j0 == 0 && w.j1 < w.n) cut = make_int4(w.item - 1, w.n, w.j1, share);
      if (w.halves() <= h2) {                      // no row in this half
        vt += w.j1 - w.j0;
        continue;
      }
      const int total = rows_of(a), row = w.it * ROWS + h2 * HALF + r;
      // no row in this warp: it only keeps the barriers going (uniform as the compiler sees it, or the loop below loses 4%)
      const bool idle = w.it * ROWS + h2 * HALF + (warp & 3) * 32 >= total;
      const bool real = row < total;
      const int rr = real ? row : total - 1, tt = rr / a.G, hq = (w.bh % a.Hkv) * a.G + rr - tt * a.G;
      const int limit = w.end - (int)a.T + 1 + tt;               // keys that the row sees
      // the half's queries as 8-bit terms of their own scales: 16 lanes per row, a lane 8 dims; a warp takes rows
      // 2 (warp mod 8) and the next of every 16, 8 at a time.  What a term leaves of 11 bits is exact in f16.
      const int first = w.it * ROWS + h2 * HALF, rows = min(HALF, total - first), piece = lane & 15;
      const T* const qb = reinterpret_cast<const T*>(a.q) + w.b * a.qb + (int64_t)(w.bh % a.Hkv) * a.G * a.qh + 8 * piece;
      const int tk0 = first / a.G, head0 = first - tk0 * a.G;
      const float per_head = 1.0f / (float)a.G;
#pragma unroll 1                                   // run once a piece: small code over fast code
      for (int r0 = 2 * (warp & 7) + (lane >> 4); r0 - (lane >> 4) < rows; r0 += 64) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = head0 + min(r0 + 16 * i, rows - 1), tk = (int)(((float)x + 0.5f) * per_head);   // x / G, x < 128 + G
          v[i] = *reinterpret_cast<const uint4*>(qb + (int64_t)(x - tk * a.G) * a.qh + (tk0 + tk) * a.qt);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rl = r0 + 16 * i;
          const T* e = reinterpret_cast<const T*>(&v[i]);
          float2 x[4];
          float most = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[k] = make_float2(to_f32(e[2 * k]), to_f32(e[2 * k + 1]));
            most = max3(most, fabsf(x[k].x), fabsf(x[k].y));
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          const int e2 = kv8_exponent(__float_as_uint(most));
          const float inv = most < INFINITY ? pow2i(-e2) : __uint_as_float(0x7FFFFFFFu);   // a row with an infinity is NaN
          if (rl >= rows) continue;
          if (piece == 0) s_rs[h2][rl] = pow2i(e2) * QSCALE;
          __half2 y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = __floats2half2_rn(x[k].x * inv, x[k].y * inv);
          uint8_t* const at = smem + S::Q + h2 * QT * HALF * D + rl * D + (((piece >> 1) ^ (rl & 7)) << 4) + (piece & 1) * 8;
#pragma unroll
          for (int term = 0; term < QT; ++term) {
            uint32_t code[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_fp8_interpretation_t type = term == 0 ? __NV_E4M3 : __NV_E5M2;
              code[k] = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&y[k]), __NV_SATFINITE, type);
              const __half2_raw d = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)code[k], type);
              y[k] = __hsub2(y[k], *reinterpret_cast<const __half2*>(&d));
            }
            *reinterpret_cast<uint2*>(at + term * HALF * D) = make_uint2(code[0] | code[1] << 16, code[2] | code[3] << 16);
          }
        }
      }
      __syncwarp();
      tc::fence_async_smem();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full(h2));
      tc::named_sync(9 + h2, SOFT);                // the scales are there
      const float rs = s_rs[h2][r];
      // keys that every row of the CTA sees need no mask
      const int all_see = seen(a, w.end, w.it * ROWS);
      const float2* sc = reinterpret_cast<const float2*>(a.scales) + (int64_t)w.bh * (a.cap / BLK);
      if (idle) {                                  // weights of rows that no one reads may be anything
        for (int j = w.j0; j <= w.j1; ++j) {
          ok = ok && tc::mbar_wait(s_full(h2), phase & 1, gave_up);
          ++phase;
          __syncwarp();
          if (j < w.j1 && lane == 0) tc::mbar_arrive(p_full(h2));
        }
        vt += w.j1 - w.j0;
        continue;
      }
      // m is the same in both threads of a row; l is this thread's share of the denominator, lm its reference
      float m = -INFINITY, lm = -1e30f, l = 0.0f;
      for (int j = w.j0; j < w.j1; ++j, ++vt) {
        const int blk = j * (TILE / BLK) + ch;
        const float2 s2 = blk < a.cap / BLK ? sc[blk] : make_float2(0.0f, 0.0f);
        // above 0, so that a masked score stays -inf; void blocks may hold anything, NaN too
        const float cs = fmaxf(s2.x * rs, 1e-37f);
        ok = ok && tc::mbar_wait(s_full(h2), phase & 1, gave_up);
        ++phase;
        __syncwarp();
        tc::fence_after();
        const float es = log2_of(s2.y);
        int see = BLK;                             // tokens of the block that this row sees
        const bool masked = (j + 1) * TILE > all_see;
        if (masked) {
          see = min(max(limit - blk * BLK, 0), BLK);
          // (this late the barrier is at this tile's phase or the one before, which its parity tells apart, also where this half
          // had no rows in the pieces before: S follows every earlier tile's products)
          ok = ok && tc::mbar_wait(v_full(vt), (vt / VSTAGES) & 1, gave_up);
          for (int i = 0; i < BLK; i += 4)
            if (const uint32_t f = *reinterpret_cast<const uint32_t*>(&s_nan[vt % VSTAGES][ch * BLK + i]))
              if (i + (__ffs(f) - 1) / 8 < see) l = __uint_as_float(0x7FFFFFFFu);
          __syncwarp();
        }
        uint32_t x[32];
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          tc::Tmem<32>::ld(tm_s + 32 * u, x);
          tc::wait_ld<32>(x);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * u + i >= see) x[i] = 0xFF800000u;                  // -inf
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            t0 = max3(t0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
            t1 = max3(t1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
          }
        }
        const float smax = fmaxf(t0, t1) * cs, top = smax + es;
        if (tc::named_or(pair_bar, 64, top > m + SLACK)) {        // also the first time: m = -inf
          s_pair[tid].x = top;
          tc::named_sync(pair_bar, 64);
          const float both = fmaxf(top, s_pair[tid ^ HALF].x);
          tc::named_sync(pair_bar, 64);
          const bool up = both > m + SLACK;
          const float f = !up ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - both);
          if (up) m = both;
          __syncwarp();
          if (j > w.j0) {                          // O of the tiles before is complete: their products precede this S
#pragma unroll 1
            for (int i = 0; i < 64; i += 16) {
              uint32_t o[16];
              tc::Tmem<16>::ld(tm_o + i, o);
              tc::wait_ld<16>(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tc::Tmem<16>::st(tm_o + i, o);
            }
          }
        }
        // A block that is far below the reference weighs nothing in f16 but may still count in the denominator: its sum is
        // taken from its own largest.
        const bool far = top < m - FAR;
        const float off = smax == -INFINITY ? 0.0f : far ? HEAD - smax : HEAD - m + es;
        const float2 cc = make_float2(cs, cs), oo = make_float2(off, off);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        // weights over the scores they came from: columns 32 u .. 32 u + 15 of the block's 64
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int u = v ^ 1;                     // the second 32 are still in registers
          if (v == 1) {
            tc::Tmem<32>::ld(tm_s + 32 * u, x);
            tc::wait_ld<32>(x);
            if (masked) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * u + i >= see) x[i] = 0xFF800000u;
            }
          }
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 e2 = __ffma2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), cc, oo);
            const float2 w2 = make_float2(ex2(e2.x), ex2(e2.y));
            sum[i & 1] = __fadd2_rn(sum[i & 1], w2);
            p[i] = pack_h2(w2.x, w2.y);
          }
          if (__any_sync(0xffffffffu, far)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = far ? 0u : p[i];
          }
          tc::Tmem<16>::st(tm_s + 32 * u, p);
        }
        {
          // this block's sum is relative to -off, without the value scale
          const float part = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), ref = smax == -INFINITY ? -1e30f : -off;
          const float d = ref - lm, f = ex2(-fabsf(d));
          l = d > 0.0f ? fmaf(l, f, part) : fmaf(part, f, l);
          lm = fmaxf(lm, ref);
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(h2));
      }
      ok = ok && tc::mbar_wait(s_full(h2), phase & 1, gave_up);      // the piece's last product
      ++phase;
      __syncwarp();
      s_pair[tid] = make_float2(l, lm);
      tc::named_sync(pair_bar, 64);
      const float2 other = s_pair[tid ^ HALF];
      const float ref = fmaxf(lm, other.y);
      l = ch == 0 ? fmaf(l, ex2(lm - ref), other.x * ex2(other.y - ref)) : fmaf(other.x, ex2(other.y - ref), l * ex2(lm - ref));
      tc::fence_after();
      const bool whole = w.j0 == 0 && w.j1 == w.n;
      // O is relative to m - HEAD; the difference of the references is a block's value exponent at most
      const float f = !ok ? __uint_as_float(0x7FFFFFFFu) : l == 0.0f ? 0.0f : ex2(m - HEAD - ref) / l;
      T* op = reinterpret_cast<T*>(a.out) + w.b * a.ob + hq * a.oh + tt * a.ot + 64 * ch;
      float* part = a.part + ((2 * (int64_t)blockIdx.x + (w.j0 == 0 ? 1 : 0)) * ROWS + h2 * HALF + r) * PART;
#pragma unroll 1
      for (int i = 0; i < 64; i += 16) {
        uint32_t o[16];
        __syncwarp();
        tc::Tmem<16>::ld(tm_o + i, o);
        tc::wait_ld<16>(o);
        if (!real) continue;
        if (whole) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            T y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) from_f32(l == 0.0f ? 0.0f : __uint_as_float(o[8 * c + e]) * f, &y[e]);
            *reinterpret_cast<uint4*>(op + i + 8 * c) = *reinterpret_cast<const uint4*>(y);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<float4*>(part + 64 * ch + i + 4 * c) =
                make_float4(__uint_as_float(o[4 * c]) * f, __uint_as_float(o[4 * c + 1]) * f,
                            __uint_as_float(o[4 * c + 2]) * f, __uint_as_float(o[4 * c + 3]) * f);
        }
      }
      if (real && !whole && ch == 0) part[D] = ref, part[D + 1] = l;
      __syncwarp();
      tc::fence_before();
    }
    if (tid == 0 && (!a.share || a.share != a.stride)) cuts_of(a)[blockIdx.x] = cut;
  } else if (group == 4) {
    // ---- values: e4m3 rows from memory to f16, MN-major tiles of two 64-dim halves.  Thread = 16 dims of 8 tokens.
    reg_less<REG_VALUE>();
    const int t = tid - 2 * SOFT, u = t & 7, row0 = t >> 3;
    uint32_t i = 0;
    bool ok = true;
    while (ok && w.next()) {
      const uint8_t* base = a.rows + (int64_t)w.bh * a.cap * KV8_ROW + D + u * 16;
      const int all_see = seen(a, w.end, w.it * ROWS);
      for (int j = w.j0; j < w.j1; ++j, ++i) {
        uint4 v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const int tok = j * TILE + p * 16 + row0;
          v[p] = tok < w.end ? *reinterpret_cast<const uint4*>(base + (int64_t)tok * KV8_ROW) : make_uint4(0, 0, 0, 0);
        }
        ok = ok && tc::mbar_wait(v_free(i), ((i / VSTAGES) & 1) ^ 1, gave_up);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* vb = smem + S::V + (i % VSTAGES) * VBYTES + (u >> 2) * (TILE * 128);
        const bool differs = (j + 1) * TILE > all_see;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const int tk = p * 16 + row0;
          uint32_t x[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
          if (differs) {
            // 0 * NaN would reach rows that do not see the token: its NaNs leave the product, and the rows that do
            // see it become NaN by their denominators
            bool nan = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t is = __vcmpeq4(x[e] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
              nan = nan || is;
              x[e] &= ~is;
            }
            const unsigned any = __ballot_sync(0xffffffffu, nan) >> (lane & 24) & 255u;
            if (u == 0) s_nan[i % VSTAGES][tk] = any != 0;
          }
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x[e >> 1] >> (16 * (e & 1))), __NV_E4M3);
            y[e] = *reinterpret_cast<const uint32_t*>(&h);
          }
          uint8_t* dst = vb + tk * 128;
          const int c = (u & 3) * 2;
          *reinterpret_cast<uint4*>(dst + ((c ^ (tk & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(dst + (((c + 1) ^ (tk & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(v_full(i));
      }
    }
  } else {
    reg_less<REG_OTHER>();
    if (warp == 21 && lane == 0) {
      // ---- key tiles
      uint32_t i = 0;
      bool ok = true;
      while (ok && w.next()) {
        for (int j = w.j0; j < w.j1; ++j, ++i) {
          ok = tc::mbar_wait(k_free(i), ((i / KSTAGES) & 1) ^ 1, gave_up);
          if (!ok) break;
          tc::mbar_expect_tx(k_full(i), KBYTES);
          tc::tma_load_3d(sbase + S::K + (i % KSTAGES) * KBYTES, &map, 0, j * TILE, w.bh, k_full(i));
        }
      }
      if (*gave_up) {
        for (uint32_t j = i > KSTAGES ? i - KSTAGES : 0; j < i; ++j) {   // copies in flight land first
          const unsigned long long t0 = tc::now_ns();
          while (!tc::mbar_try(k_full(j), (j / KSTAGES) & 1) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
        }
      }
    } else if (warp == 20) {
      // ---- products (the whole warp: elect_one)
      constexpr uint32_t id_s = tc::instr(TILE, false, false), id_t = tc::instr(TILE, false, false, true), id_o = tc::instr(D, false, true);
      const uint32_t tmu = tc::uniform(tm);
      uint32_t i = 0;                              // tiles done
      uint32_t pn[2] = {0, 0}, seg[2] = {0, 0};    // by half: weight tiles done, pieces begun
      uint32_t ks = 0, vs = 0;                     // stages of the next key tile, of the next value tile
      bool ok = true;
      // S_h of the next key tile, which is spent with the last half
      auto scores = [&](int h, bool spent) {
        const uint64_t dk = tc::operand(sbase + S::K + tc::uniform(ks) * KBYTES);
        if (tc::elect_one()) {
#pragma unroll
          for (int term = 0; term < QT; ++term) {
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
              tc::mma_fp8(tmu + h * 128, tc::operand(sbase + S::Q + (h * QT + term) * HALF * D) + kk * 2, dk + kk * 2,
                          term > 0 ? id_t : id_s, term > 0 || kk > 0);
          }
          if (spent) tc::mma_commit(bar + 8 * (KSTAGES + ks));
          tc::mma_commit(s_full(h));
        }
        __syncwarp();
        if (spent) ks = ks + 1 == KSTAGES ? 0 : ks + 1;
      };
      // O_h of the next value tile; the piece's last is announced as scores are
      auto values = [&](int h, bool spent, bool accumulate, bool last) {
        const uint64_t dv = tc::operand(sbase + S::V + tc::uniform(vs) * VBYTES, TILE * 128);
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)   // 16 tokens a step: 8 columns of weights, 2 groups of 8 value rows
            tc::mma_f16_ts(tmu + 256 + h * 128, tmu + h * 128 + kk / 2 * 32 + kk % 2 * 8, dv + kk * (16 * 128 / 16), id_o,
                           accumulate || kk > 0);
          if (spent) tc::mma_commit(bar2 + 8 * (VSTAGES + vs));
          if (last) tc::mma_commit(s_full(h));
        }
        __syncwarp();
        if (spent) vs = vs + 1 == VSTAGES ? 0 : vs + 1;
      };
      while (ok && w.next()) {
        const int n = w.j1 - w.j0;
        const bool two = w.halves() == 2;
        ok = tc::mbar_wait(q_full(0), seg[0]++ & 1, gave_up);
        if (two) ok = ok && tc::mbar_wait(q_full(1), seg[1]++ & 1, gave_up);
        ok = ok && tc::mbar_wait(k_full(i), (i / KSTAGES) & 1, gave_up);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after();
        scores(0, !two);
        if (two) scores(1, true);
        for (int j = 1; j <= n; ++j) {
          const uint32_t v = i + j - 1;
          const bool last = j == n;
          ok = last || tc::mbar_wait(k_full(i + j), ((i + j) / KSTAGES) & 1, gave_up);
          ok = ok && tc::mbar_wait(v_full(v), (v / VSTAGES) & 1, gave_up);
          ok = ok && tc::mbar_wait(p_full(0), pn[0]++ & 1, gave_up);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc::fence_after();
          values(0, !two, j > 1, last);
          if (!last) scores(0, !two);
          if (!two) continue;
          ok = tc::mbar_wait(p_full(1), pn[1]++ & 1, gave_up);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc::fence_after();
          values(1, true, j > 1, last);
          if (!last) scores(1, true);
        }
        i += n;
      }
      if (*gave_up && tc::elect_one()) {
        tc::mma_commit(drain);
        const unsigned long long t0 = tc::now_ns();
        while (!tc::mbar_try(drain, 0) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
      }
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 20) tc::tmem_free(tm, 512);
  if (tid == 0 && s_gave_up) atomicAdd(a.timeouts, 1ull);
}

// Joins the items that shares cut: block (c, ..) the one that share c begins and does not end.  Warp = row, lane = 4 dims.
constexpr int JOIN_WARPS = 8, JOIN_BLOCKS = 16;    // blocks per cut
template <typename T>
__global__ void __launch_bounds__(JOIN_WARPS * 32) prompt_join_kernel(const Args a, int ctas) {
  tc::launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = items_per_bh(a);
  tc::wait_dependency();                           // the parts are written; and nothing ends before they are
  const int4 cut = cuts_of(a)[blockIdx.x];         // item, its tiles, those in share c, tiles per share
  if (cut.x < 0) return;
  const int bh = cut.x / per, it = cut.x % per, b = bh / a.Hkv, total = rows_of(a);
  const int c0 = blockIdx.x, c1 = c0 + (cut.y - cut.z + cut.w - 1) / cut.w;
  for (int r = blockIdx.y * JOIN_WARPS + warp; r < ROWS; r += JOIN_BLOCKS * JOIN_WARPS) {
    const int row = it * ROWS + r;
    if (row >= total) return;
    // parts: share c0 holds the item's first tiles (its second slot), the others begin with it (first slot)
    auto part = [&](int c) { return a.part + ((2 * (int64_t)c + (c == c0 ? 1 : 0)) * ROWS + r) * PART; };
    // lane = part, 32 at a time: the denominator, then each part's share of it (parts are weighted means)
    float M = -INFINITY, L = 0.0f;
    for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, part(c)[D]);
    M = warp_max(M);
    for (int c = c0 + lane; c <= c1; c += 32) L = fmaf(part(c)[D + 1], ex2(part(c)[D] - M), L);
    L = warp_sum(L);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = c0; c <= c1; c += 32) {
      const int n = min(32, c1 - c + 1);
      const float e = lane < n ? part(c + lane)[D + 1] * ex2(part(c + lane)[D] - M) * inv : 0.0f;
#pragma unroll 8
      for (int v = 0; v < n; ++v) {
        const float4 o = *reinterpret_cast<const float4*>(part(c + v) + 4 * lane);
        const float ev = __shfl_sync(0xffffffffu, e, v);
        O.x = fmaf(o.x, ev, O.x), O.y = fmaf(o.y, ev, O.y), O.z = fmaf(o.z, ev, O.z), O.w = fmaf(o.w, ev, O.w);
      }
    }
    T y[4];
    from_f32(O.x, &y[0]), from_f32(O.y, &y[1]), from_f32(O.z, &y[2]), from_f32(O.w, &y[3]);
    const int tt = row / a.G, hq = (bh % a.Hkv) * a.G + row - tt * a.G;
    T* op = reinterpret_cast<T*>(a.out) + b * a.ob + hq * a.oh + tt * a.ot + 4 * lane;
    *reinterpret_cast<uint2*>(op) = *reinterpret_cast<const uint2*>(y);
  }
}

template <typename T, int QT> int launch(const CUtensorMap& map, const Args& a, int ctas, cudaStream_t st) {
  using S = Shape<QT>;
  static_assert(S::SMEM <= 226 * 1024, "shared memory");
  static std::atomic<uint64_t> told{0};
  const int r = allow_smem(prompt_kernel<T, QT>, S::SMEM, told, "kv8_attend");
  if (r != FATHOM_OK) return r;
  const int e = launch_after(prompt_kernel<T, QT>, dim3(ctas), THREADS, S::SMEM, st, "kv8_attend", map, a);
  if (e != FATHOM_OK || ctas == 1 || (a.share && a.share == a.stride)) return e;          // no item is cut
  return launch_after(prompt_join_kernel<T>, dim3(ctas - 1, JOIN_BLOCKS), JOIN_WARPS * 32, 0, st, "kv8_attend", a, ctas);
}

}  // namespace

size_t prompt_workspace() { return (size_t)sm_count() * (2 * ROWS * PART * sizeof(float) + sizeof(int4)); }

int prompt_attend(const CUtensorMap& map, Args a, int dtype, cudaStream_t st) {
  const int ctas = a.ctas = plan_shares(a, sm_count(), PIECE, WHOLE, LEAST);
  return dtype == FATHOM_DTYPE_BF16 ? launch<__nv_bfloat16, 2>(map, a, ctas, st) : launch<__half, 3>(map, a, ctas, st);
}

}  // namespace kv8
}  // namespace fathom
