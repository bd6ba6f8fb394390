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
// bf16 exactly, 3 an fp16, down to 2^-21 and 2^-25 of the row's largest), and a row of the weights into five: three hold
// the 11 bits of the largest, two more continue to steps of 2^-28 of the reference, because the tail of a long context weighs
// that little a token beside one dominant key and a tenth of everything together (with three terms it was lost from O
// and kept in the denominator; five cost a draft of 20 rows 6%, other calls 0 to 4%).  The terms are further columns
// of the product, which the tensor cores have to spare: with M = 128 tokens a tile of 32 KB takes them up to ~450 cycles, its
// bytes ~1400.  A score is then the sum of its term columns times the block's key scale; weights carry the
// block's value scale (a power of two) in their exponent, so no value is ever rescaled.
//
// Softmax, thread = token: with m the running reference of a row's (score + log2 of the value scale), a weight is
// 2^(s + log2 vs - m); m moves only when a tile exceeds it by 2^5 (then O^T in tensor memory is rescaled), which
// leaves e4m3's range room on both sides.  The denominator is kept per thread in fp32 with a reference of its
// own, because the value scale must not enter it.  One tile's chain of steps is longer than its bytes take, so there are
// two softmax warpgroups: up to 16 rows they take the even and the odd tiles, each with its own references and its own
// O^T; up to 32 rows (SPLIT) each takes 12 or 16 rows
// of every tile.
//
// A row's parts in different CTAs (kv8_line.cuh) are joined by a second kernel in a fixed order.
//
// Measured in graphs (8 KV heads, G = 4, bf16): one token over 128k 45-46 us with the join, 5.9 TB/s or 0.9 of the copy
// rate; 8 sequences of 80k (mean), 4 KV heads, G = 7: 107 us, 0.96; over 700 tokens 6.2 us, a chain of latencies.  With one softmax warpgroup the
// softmax was the bound: 58 us and 150 us.
#include "kv8_line.cuh"

namespace fathom {
namespace kv8 {
namespace {

constexpr int TERMS = 5;                         // e4m3 terms of a weight: 2^8 down to steps of 2^-25
constexpr int F16_UP = 7;                        // weights come to f16 times 2^7: up to 2^15, 11 bits down to 2^-21
constexpr int GROUP = 128;                       // threads of a softmax warpgroup
constexpr int THREADS = 2 * GROUP + 64;          // warps 0-3, 4-7: softmax; 8: loads; 9: products
constexpr int STAGE_BYTES = 2 * TILE * D;        // key tile, value tile
constexpr float SLACK = 5.0f;                    // a tile may exceed the reference by 2^5
constexpr float HEAD = 3.0f;                     // weights at the reference are 8: 2^(HEAD + SLACK) = 256 <= 448
constexpr int PIECE = 6;                         // tiles (~0.4 us each) that beginning and ending a piece takes: ~2.5 us
// Tiles up to which a row is whole in one CTA and not joined.  In a graph, whole against joined: one token of 32 KV heads,
// G = 7, over 1024 tokens 7.9 against 8.7 us; of 8 KV heads, G = 4, over 512 5.1 / 6.1, over 1024 6.7 / 6.1; drafts of 20
// rows over 384 10.2 / 10.3, over 1024 15.5 / 10.3 (there 3 tiles would be the rule).
constexpr int SHORT = 8;
constexpr int MAX_CTAS = 512;                    // shares that the join kernel has room for

constexpr int up16(int n) { return (n + 15) / 16 * 16; }

// NR: rows of a softmax thread; SPLIT: the two warpgroups have NR rows each, in NC = 16 columns of a term's RT.
template <int NR, int QT, bool SPLIT> struct Shape {
  static constexpr int ROWS = SPLIT ? 2 * NR : NR, NC = SPLIT ? 16 : NR, RT = SPLIT ? 2 * NC : NR;
  static constexpr int NQ = up16(RT * QT), NP = up16(RT * TERMS);
  static constexpr int COLS = 2 * NQ + (SPLIT ? 1 : 2) * NP;     // S^T of even and odd tiles, then O^T
  static constexpr int TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static_assert(COLS <= TMEM, "tensor memory");
  static constexpr int STAGES = SPLIT ? 5 : 6;
  // byte offsets in dynamic shared memory (1024-byte aligned operands first)
  static constexpr int Q = STAGES * STAGE_BYTES, P = Q + (NQ * D + 1023) / 1024 * 1024, END = P + 2 * NP * TILE;
  static constexpr int SMEM = END + 1024;        // room to align
};

// Weights as an MN-major operand without swizzle: 16 bytes of one token's columns, 8 tokens a 128-byte core matrix,
// the next 16 columns TILE * 16 bytes on.  A thread stores its token's columns in 16-byte pieces.
__device__ __forceinline__ uint64_t weight_operand(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(TILE * 16 >> 4) << 32 | 1ull << 46;
}

// 8 bytes if `there`.  (Written as a branch around a load, each row waited for the one before.)
__device__ __forceinline__ void load8(uint2& x, const void* p, bool there) {
  asm volatile("{ .reg .pred p; setp.ne.u32 p, %3, 0; @p ld.global.v2.u32 {%0, %1}, [%2]; }\n"
               : "+r"(x.x), "+r"(x.y)
               : "l"(p), "r"((uint32_t)there)
               : "memory");
}
template <typename T> __device__ __forceinline__ void unpack4(uint2 v, float (&x)[4]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(e[i]);
}

template <typename T, int NR, int QT, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) token_kernel(const __grid_constant__ CUtensorMap map,
                                                          const __grid_constant__ Args a) {
  using S = Shape<NR, QT, SPLIT>;
  constexpr int STAGES = S::STAGES, RT = S::RT, NC = S::NC, ROWS = S::ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = tc::smem_u32(smem);
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 10];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gave_up;
  __shared__ float s_rs[ROWS];                    // scale of a row's scores: 2^e log2(e) / sqrt(128)
  __shared__ float s_top[2][4][NR];              // a tile's largest s + log2 vs, by warpgroup and warp
  // at a row's end: references; denominators by warp; then the denominator, its reference, and what brings O^T there
  __shared__ float s_m[2][NR], s_lm[8][NR], s_l[8][NR], s_sum[ROWS], s_ref[ROWS], s_f[2][ROWS];
  __shared__ int64_t s_out[ROWS];                // where a row's output begins
  const uint32_t bar0 = tc::smem_u32(bars);
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8 * (STAGES + s); };
  const uint32_t B = bar0 + 16 * STAGES;
  auto s_full = [&](uint32_t k) { return B + 8 * k; };
  auto s_free = [&](uint32_t k) { return B + 16 + 8 * k; };
  auto p_full = [&](uint32_t k) { return B + 32 + 8 * k; };
  auto p_free = [&](uint32_t k) { return B + 48 + 8 * k; };
  const uint32_t q_full = B + 64, drain = B + 72;
  const int tid = threadIdx.x, lane = tid & 31, warp = (int)tc::uniform(tid >> 5);
  volatile int* gave_up = &s_gave_up;

  tc::wait_dependency();
  int count, share;
  const Place place = my_share<true>(a, &count, &share);
  Walk<true> w(a, place, count);
  if (warp == 8) {
    // ---- loads: the share's tiles in order, as stages come free.  They begin while the CTA still sets itself up.
    if (lane == 0) {
      for (int s = 0; s < STAGES; ++s) tc::mbar_init(full(s), 1), tc::mbar_init(empty(s), 1);
      for (int k = 0; k < 2; ++k)
        tc::mbar_init(s_full(k), 1), tc::mbar_init(s_free(k), SPLIT ? 8 : 4), tc::mbar_init(p_full(k), SPLIT ? 8 : 4),
            tc::mbar_init(p_free(k), 1);
      tc::mbar_init(q_full, 8);
      tc::mbar_init(drain, 1);
      tc::fence_mbar_init();
      s_gave_up = 0;
    }
    __syncwarp();
    tc::named_arrive(4, THREADS);
    if (lane == 0) {
      uint32_t i = 0;
      bool ok = true;
      while (ok && w.next()) {
        for (int tile = w.j0; tile < w.j1; ++tile, ++i) {
          const uint32_t s = i % STAGES;
          ok = tc::mbar_wait(empty(s), ((i / STAGES) & 1) ^ 1, gave_up);
          if (!ok) break;
          tc::mbar_expect_tx(full(s), STAGE_BYTES);
          tc::tma_load_3d(sbase + s * STAGE_BYTES, &map, 0, tile * TILE, w.bh, full(s));
          tc::tma_load_3d(sbase + s * STAGE_BYTES + TILE * D, &map, D, tile * TILE, w.bh, full(s));
        }
      }
      if (*gave_up) {          // copies in flight land before the CTA ends (bounded: the flag is up, so by time alone)
        for (uint32_t j = i > STAGES ? i - STAGES : 0; j < i; ++j) {
          const unsigned long long t0 = tc::now_ns();
          while (!tc::mbar_try(full(j % STAGES), (j / STAGES) & 1) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
        }
      }
    }
  } else if (warp == 9) {
    tc::tmem_alloc(tc::smem_u32(&s_tmem), S::TMEM);
    tc::fence_before();
    tc::named_sync(4, THREADS);
    tc::fence_after();
    // ---- products (the whole warp: elect_one): S^T of tile i, then O^T of tile i - 2, whose weights were made meanwhile
    constexpr uint32_t id_s = tc::instr(S::NQ, false, false), id_o = tc::instr(S::NP, true, true);
    const uint32_t tmu = tc::uniform(s_tmem);
    uint32_t seg = 0, ks = 0, vs = 0;             // rows begun: each fills q once; stages of the next S^T and O^T
    bool ok = true;
    auto scores = [&](uint32_t i) {
      const uint32_t k = i & 1;
      ok = ok && tc::mbar_wait(full(ks), (i / STAGES) & 1, gave_up);
      ok = ok && tc::mbar_wait(s_free(k), ((i >> 1) & 1) ^ 1, gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc::fence_after();
      const uint32_t ku = tc::uniform(k);
      const uint64_t dk = tc::operand(sbase + tc::uniform(ks) * STAGE_BYTES);
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)       // 32 dims a step: 32 bytes along the swizzled rows
          tc::mma_fp8(tmu + ku * S::NQ, dk + kk * 2, tc::operand(sbase + S::Q) + kk * 2, id_s, kk > 0);
        tc::mma_commit(s_full(ku));
      }
      __syncwarp();
      ks = ks + 1 == STAGES ? 0 : ks + 1;
    };
    auto values = [&](uint32_t i, bool accumulate) {
      const uint32_t k = i & 1;
      ok = ok && tc::mbar_wait(p_full(k), (i >> 1) & 1, gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc::fence_after();
      const uint32_t ku = tc::uniform(k), vu = tc::uniform(vs);
      const uint64_t dv = tc::operand(sbase + vu * STAGE_BYTES + TILE * D);
      const uint64_t dp = weight_operand(sbase + S::P + ku * S::NP * TILE);
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < TILE / 32; ++kk)    // 32 tokens a step: 4 groups of 8 value rows, 4 core matrices of weights
          tc::mma_fp8(tmu + 2 * S::NQ + (SPLIT ? 0 : ku * S::NP), dv + kk * (32 * D / 16), dp + kk * (4 * 128 / 16), id_o,
                      kk > 0 || accumulate);
        tc::mma_commit(empty(vu));
        tc::mma_commit(p_free(ku));
      }
      __syncwarp();
      vs = vs + 1 == STAGES ? 0 : vs + 1;
    };
    uint32_t i = 0;
    while (ok && w.next()) {
      ok = tc::mbar_wait(q_full, seg++ & 1, gave_up);
      const uint32_t i0 = i, n = w.j1 - w.j0;
      for (; i < i0 + n + 2 && ok; ++i) {
        if (i < i0 + n) scores(i);
        if (ok && i >= i0 + 2) values(i - 2, i >= i0 + (SPLIT ? 3 : 4));
      }
      i = i0 + n;
    }
    if (*gave_up && tc::elect_one()) {
      tc::mma_commit(drain);
      const unsigned long long t0 = tc::now_ns();
      while (!tc::mbar_try(drain, 0) && tc::now_ns() - t0 < tc::WAIT_LIMIT_NS) {}
    }
  } else {
    // ---- softmax: warpgroup g has the tiles i = g mod 2 of the share, or (SPLIT) rows g NR .. of every tile; thread = token
    // of the tile; lane of tensor memory = token of S^T, dim of O^T
    const int R = rows_of(a), late = (int)a.T - 1, g = warp >> 2, t = tid & (GROUP - 1);
    const int first = SPLIT ? g * NR : 0;         // this thread's rows: first + (0 .. NR - 1)
    // A warp brings every eighth row of q, a lane 4 dims of it; the share's first row ahead of everything else.
    constexpr int QR = (ROWS + 7) / 8;
    uint2 qv[QR] = {};
    auto load_q = [&]() {                         // rows are token-major: row = token * G + head
      const int64_t step = a.qt - a.G * a.qh;
      const T* const q0 = reinterpret_cast<const T*>(a.q) + w.b * a.qb + (int64_t)(w.bh - w.b * a.Hkv) * a.G * a.qh + lane * 4;
#pragma unroll
      for (int i = 0; i < QR; ++i) {
        const int r = warp + 8 * i;
        load8(qv[i], q0 + r * a.qh + (late ? div_small(r, a.inv_g) : 0) * step, r < R);
      }
    };
    bool more = w.next();
    if (more) load_q();
    for (int i = tid; i < (S::END - S::Q) / 16; i += 2 * GROUP)      // operand columns that no row writes stay 0
      reinterpret_cast<uint4*>(smem + S::Q)[i] = make_uint4(0, 0, 0, 0);
    tc::fence_async_smem();
    tc::fence_before();
    tc::named_sync(4, THREADS);
    tc::fence_after();
    tc::launch_dependents();
    const uint32_t tm = s_tmem;
    const uint32_t my = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tm_s = tm + (SPLIT ? g * NC : 0) + my, tm_o = tm_s + 2 * S::NQ;
    uint8_t* const pb = smem + S::P + t * 16;
    uint32_t i0 = 0;                              // the share's tiles before this row
    bool ok = true, bad = false;                  // ok: this thread's waits; bad: some thread's gave up
    while (more) {
      const int h = w.bh - w.b * a.Hkv, n = w.j1 - w.j0;
      // this row's queries as terms.  The products of the row before are complete (its O^T was read below), so its q
      // may go.
#pragma unroll
      for (int rr = 0; rr < QR; ++rr) {
        const int r = warp + 8 * rr;
        if (r >= R) break;
        float x[4];
        unpack4<T>(qv[rr], x);
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
          const int c = term * RT + (SPLIT ? r / NR * NC + r % NR : r);
          *reinterpret_cast<uint32_t*>(smem + S::Q + c * D + (((lane >> 2) ^ (c & 7)) << 4) + (lane & 3) * 4) = code;
          const float2 lo = kv8_decode2(code), hi = kv8_decode2(code >> 16);
          x[0] = (x[0] - lo.x) * 16.0f, x[1] = (x[1] - lo.y) * 16.0f;
          x[2] = (x[2] - hi.x) * 16.0f, x[3] = (x[3] - hi.y) * 16.0f;
        }
        if (lane == 0) s_rs[r] = pow2i(e2) * QSCALE;
      }
      tc::fence_async_smem();
      tc::named_sync(3, 2 * GROUP);
      if (lane == 0) tc::mbar_arrive(q_full);
      // a row's reference; its scale; this thread's denominator and that one's reference
      float m[NR], rs[NR], lm[NR], l[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r)
        m[r] = -INFINITY, lm[r] = -1e30f, l[r] = 0.0f, rs[r] = first + r < R ? s_rs[first + r] : 0.0f;
      const float2* sc = reinterpret_cast<const float2*>(a.scales) + (int64_t)w.bh * (a.cap / BLK);
      auto scale_of = [&](int tile) {
        const int tok = tile * TILE + t;
        uint2 x = make_uint2(0u, 0x3F800000u);    // 0 and 1
        load8(x, sc + tok / BLK, tok < w.end);
        return make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
      };
      constexpr uint32_t STEP = SPLIT ? 1 : 2;
      const uint32_t mine = SPLIT ? i0 : i0 + ((i0 ^ g) & 1);      // this warpgroup's first tile of the row
      float2 next_scale = scale_of(w.j0 + (int)(mine - i0));
      uint32_t i = mine;
      for (; i < i0 + n; i += STEP) {             // to the end also when a wait gave up: barriers stay in step
        const int tile = w.j0 + (int)(i - i0), tok = tile * TILE + t;
        const uint32_t use = i >> 1, k = SPLIT ? i & 1 : g;        // uses of the buffers before; the buffers
        const float2 ks = next_scale;
        next_scale = scale_of(tile + STEP);       // read ahead
        const float lv = (float)((int)(__float_as_uint(ks.y) >> 23) - 127);      // log2 of the value scale
        ok = ok && tc::mbar_wait(s_full(k), use & 1, gave_up);
        __syncwarp();
        tc::fence_after();
        float s[NR];
        {
          uint32_t c[QT][NC];
#pragma unroll
          for (int term = 0; term < QT; ++term) tc::Tmem<NC>::ld(tm_s + k * S::NQ + term * RT, c[term]);
          tc::wait_ld<QT * NC>(c[0]);
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(s_free(k));
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float v = __uint_as_float(c[QT - 1][r]);
#pragma unroll
            for (int term = QT - 2; term >= 0; --term) v = fmaf(v, 0.0625f, __uint_as_float(c[term][r]));
            s[r] = first + r < R ? v * (ks.x * rs[r]) : -INFINITY;
          }
        }
        // keys that a row does not see: past the end, or in the last T - 1 after its own
        if (tile * TILE + TILE > w.end - late) {
          const bool void_row = tok >= w.end;
          bool nan_v = false;
          uint4* vrow = reinterpret_cast<uint4*>(smem + (i % STAGES) * STAGE_BYTES + TILE * D + t * D);
          ok = ok && tc::mbar_wait(full(i % STAGES), (i / STAGES) & 1, gave_up);
          if (late > 0 && !void_row) {
            // the mask differs between rows here, and 0 * NaN would reach rows that do not see the key: a value row
            // with a NaN leaves the product, and the rows that see it become NaN by their denominators
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              const uint4 v = vrow[c];
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) nan_v = nan_v || __vcmpeq4(x[e] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
            }
          }
          if (SPLIT) tc::named_sync(5, 2 * GROUP);             // both warpgroups have looked at the row
          if (void_row || nan_v) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) vrow[c] = make_uint4(0, 0, 0, 0);
          }
          int room = div_small(first, a.inv_g), head = first - room * a.G;
          room += w.end - tok - late;                          // keys left to the row's token: seen if > 0
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            if (room <= 0) s[r] = -INFINITY;
            else if (nan_v && first + r < R) l[r] = __uint_as_float(0x7FFFFFFFu);
            if (++head == a.G) head = 0, ++room;
          }
          __syncwarp();
        }
        ok = ok && tc::mbar_wait(p_free(k), (use & 1) ^ 1, gave_up);   // the product that read this weight buffer
        bool above = !ok;
#pragma unroll
        for (int r = 0; r < NR; ++r) above = above || s[r] + lv > m[r] + SLACK;
        if (tc::named_or(1 + g, GROUP, above)) {
          // some row outgrew its reference: the tile's largest becomes every row's
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float mx = redux_max(s[r] + lv);
            if (lane == 0) s_top[g][warp & 3][r] = mx;
          }
          tc::named_sync(1 + g, GROUP);
          float f[NR];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float mx = fmaxf(fmaxf(s_top[g][0][r], s_top[g][1][r]), fmaxf(s_top[g][2][r], s_top[g][3][r]));
            mx = fmaxf(mx, m[r]);
            f[r] = m[r] == -INFINITY ? 0.0f : ex2(m[r] - mx);
            m[r] = mx;
          }
          tc::named_sync(1 + g, GROUP);
          if (i != mine) {
            // O^T of the tiles before is complete
            if (SPLIT) ok = ok && tc::mbar_wait(p_free(k ^ 1), ((i - 1) >> 1) & 1, gave_up);
            __syncwarp();
            tc::fence_after();
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
              uint32_t o[NC];
              tc::Tmem<NC>::ld(tm_o + (SPLIT ? 0 : g * S::NP) + term * RT, o);
              tc::wait_ld<NC>(o);
#pragma unroll
              for (int r = 0; r < NR; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * f[r]);
              tc::Tmem<NC>::st(tm_o + (SPLIT ? 0 : g * S::NP) + term * RT, o);
            }
            tc::wait_st();
          }
        }
        // weights as terms into the operand buffer, by way of f16: 11 bits, whose remainders after e4m3 are exact.  (More would
        // be lost in the outputs' 8 or 11: weights round independently.  fp16 drafts: 2.3e-4 off, in 32 bits 2.1e-4.)
        uint32_t codes[TERMS * NC / 4] = {};
#pragma unroll
        for (int r = 0; r < NR; r += 2) {
          float x[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float sv = s[r + e], mv = m[r + e];
            x[e] = mv == -INFINITY && !(sv != sv) ? 0.0f : ex2(sv + (lv - mv + (HEAD + F16_UP)));
            const float d = sv - lm[r + e], p = ex2(-fabsf(d));
            l[r + e] = d > 0.0f ? fmaf(l[r + e], p, 1.0f) : l[r + e] + p;
            lm[r + e] = fmaxf(lm[r + e], sv);
          }
          __half2 y = __floats2half2_rn(x[0], x[1]);
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            const float unit = (float)(1 << F16_UP) / (float)(1 << 4 * term);       // of this term in y
            const __half2 z = __hmul2(y, __float2half2_rn(1.0f / unit));
            const uint32_t code =
                __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&z), __NV_SATFINITE, __NV_E4M3);
            uint32_t& word = codes[(term * NC + r) / 4];
            word = (r & 2) ? word | code << 16 : code;
            const __half2_raw c = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)code, __NV_E4M3);
            y = __hfma2(*reinterpret_cast<const __half2*>(&c), __float2half2_rn(-unit), y);
          }
        }
        // columns as q's; with NC = 16 a term's rows are a 16-byte piece of their own
        constexpr int PIECES = SPLIT ? TERMS : S::NP / 16;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 4 * c + e;
            x[e] = at < TERMS * NC / 4 ? codes[at < TERMS * NC / 4 ? at : 0] : 0;
          }
          uint8_t* const at = pb + k * S::NP * TILE + (SPLIT ? 2 * c + g : c) * TILE * 16;
          *reinterpret_cast<uint4*>(at) = make_uint4(x[0], x[1], x[2], x[3]);
        }
        tc::fence_async_smem();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(k));
      }
      // the row's part (or whole): denominators over the threads, O^T out of tensor memory
      if (i != mine) ok = ok && tc::mbar_wait(p_free((i - STEP) & 1), ((i - STEP) >> 1) & 1, gave_up);
      __syncwarp();
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float mx = redux_max(lm[r]);
        const float sum = warp_sum(l[r] * ex2(lm[r] - mx));
        if (lane == 0) s_lm[warp][r] = mx, s_l[warp][r] = sum;
        if (t == 0) s_m[g][r] = m[r];
      }
      tc::fence_before();
      bad = tc::uniform(tc::named_or(3, 2 * GROUP, !ok));
      tc::fence_after();
      const Walk<true> now = w;
      more = w.next();
      if (more) load_q();                         // the next row's q, on its way while this one is finished
      const bool whole = now.j0 == 0 && now.j1 == now.n;
      float* const parts = a.part + ((int64_t)blockIdx.x + now.bh) * R * PART;
      if (tid < ROWS) {
        // the warps that have the row, and its place among their rows
        const int v0 = SPLIT ? tid / NR * 4 : 0, r = SPLIT ? tid % NR : tid;
        constexpr int NV = SPLIT ? 4 : 8;
        float mx = s_lm[v0][r], sum = 0.0f;
#pragma unroll
        for (int v = 1; v < NV; ++v) mx = fmaxf(mx, s_lm[v0 + v][r]);
#pragma unroll
        for (int v = 0; v < NV; ++v) sum = fmaf(s_l[v0 + v][r], ex2(s_lm[v0 + v][r] - mx), sum);
        s_sum[tid] = sum;
        s_ref[tid] = mx;
        const int tt = late ? div_small(tid, a.inv_g) : 0;
        s_out[tid] = now.b * a.ob + (int64_t)(h * a.G + tid - tt * a.G) * a.oh + tt * a.ot;
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;       // of parts too: a mean stays in range where a sum may not
        // O^T is relative to m - HEAD: both come to the denominator's reference.  A warpgroup that had no tile left its
        // columns as they were.
#pragma unroll
        for (int k = 0; k < (SPLIT ? 1 : 2); ++k) {
          const float m0 = s_m[SPLIT ? tid / NR : k][r];
          const bool none = (!SPLIT && n == 1 && k != (int)(i0 & 1)) || m0 == -INFINITY;
          s_f[k][tid] = (none ? 0.0f : exp2f(m0 - HEAD - mx)) * scale;       // (NaN where the denominator is)
        }
      }
      tc::named_sync(3, 2 * GROUP);
      // warpgroup g finishes its own rows, or of 4 rows r = g mod 2 (4 at a time: run once a row, small code is fast code)
#pragma unroll 1
      for (int r0 = 0; r0 < NR; r0 += 4) {
        constexpr int NO = SPLIT ? 1 : 2;         // accumulators that hold the row
        uint32_t c[NO][TERMS][4];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < NO; ++k) {
#pragma unroll
          for (int term = 0; term < TERMS; ++term) tc::Tmem<4>::ld(tm_o + k * S::NP + term * RT + r0, c[k][term]);
        }
        tc::wait_ld<NO * TERMS * 4>(c[0][0]);
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
          const int r = first + r0 + rr;
          if (r >= R || (!SPLIT && (rr & 1) != g)) continue;
          float x = 0.0f;
#pragma unroll
          for (int k = 0; k < NO; ++k) {
            float v = __uint_as_float(c[k][TERMS - 1][rr]);
#pragma unroll
            for (int term = TERMS - 2; term >= 0; --term) v = fmaf(v, 0.0625f, __uint_as_float(c[k][term][rr]));
            if (s_f[k][r] != 0.0f) x = fmaf(v, s_f[k][r], x);
          }
          if (bad) x = __uint_as_float(0x7FFFFFFFu);
          if (whole) {
            from_f32(x, reinterpret_cast<T*>(a.out) + s_out[r] + t);
          } else {
            parts[r * PART + t] = x;
            if (t == 0) parts[r * PART + D] = s_ref[r], parts[r * PART + D + 1] = s_sum[r];
          }
        }
      }
      tc::fence_before();
      tc::named_sync(3, 2 * GROUP);               // both warpgroups have read O^T: the next row may overwrite it
      i0 += n;
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 9) tc::tmem_free(s_tmem, S::TMEM);
  if (tid == 0 && s_gave_up) atomicAdd(a.timeouts, 1ull);
}

// Joins a row's parts: CTA = (bh, query row), thread = dim.  Rows of one part were written whole.
template <typename T>
__global__ void __launch_bounds__(D) token_join_kernel(const Args a, int ctas) {
  __shared__ int64_t s_before, s_total;
  __shared__ float s_m[MAX_CTAS], s_l[MAX_CTAS], s_e[MAX_CTAS], s_red[2][D / 32];
  tc::launch_dependents();
  const int R = rows_of(a), tid = threadIdx.x, lane = tid & 31;
  const int bh = blockIdx.y, r = blockIdx.x, b = div_small(bh, a.inv_hkv), h = bh - b * a.Hkv;
  const int nt = tiles_of<true>(a, seq_end(a, b), 0);
  if (a.end_dev && tid < 32) {
    // tiles of the sequences before b, and of all
    int64_t before = 0, total = 0;
    for (int j = tid; j < a.B; j += 32) {
      const int64_t x = (int64_t)tiles_of<true>(a, seq_end(a, j), 0) * a.Hkv;
      total += x;
      if (j < b) before += x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if (tid == 0) s_before = before, s_total = total;
  }
  __syncthreads();
  const int64_t share = a.share ? a.share : share_of(a, s_total, ctas);
  const int64_t first = a.share ? (int64_t)bh * a.stride : s_before + (int64_t)h * nt;
  const int c0 = (int)quotient(first, (int)share), n = (int)quotient(first + nt - 1, (int)share) - c0 + 1;
  tc::wait_dependency();                          // the parts are written; and nothing ends before they are
  if (n == 1) return;
  const float* part = a.part + ((int64_t)(c0 + bh) * R + r) * PART;
  const int64_t step = (int64_t)R * PART;
  // the first parts' dims are on their way while references and denominators are worked out
  constexpr int AHEAD = 20;
  float x[AHEAD];
#pragma unroll
  for (int p = 0; p < AHEAD; ++p) x[p] = part[min(p, n - 1) * step + tid];
  float M = -INFINITY;
  for (int p = tid; p < n; p += D) {
    const float2 ml = *reinterpret_cast<const float2*>(part + p * step + D);
    s_l[p] = ml.y;
    M = fmaxf(M, s_m[p] = ml.x);
  }
  M = warp_max(M);
  if (lane == 0) s_red[0][tid >> 5] = M;
  __syncthreads();
  M = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  float L = 0.0f;
  for (int p = tid; p < n; p += D) {
    const float e = s_l[p] * ex2(s_m[p] - M);
    s_e[p] = e;
    L += e;
  }
  L = warp_sum(L);
  if (lane == 0) s_red[1][tid >> 5] = L;
  __syncthreads();
  L = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  float O = 0.0f;                                 // parts are weighted means: each counts by its share of the denominator
#pragma unroll
  for (int p = 0; p < AHEAD; ++p)
    if (p < n) O = fmaf(x[p], s_e[p] * inv, O);
#pragma unroll 8
  for (int p = AHEAD; p < n; ++p) O = fmaf(part[p * step + tid], s_e[p] * inv, O);
  const int tt = div_small(r, a.inv_g), hq = h * a.G + r - tt * a.G;
  from_f32(O, reinterpret_cast<T*>(a.out) + b * a.ob + hq * a.oh + tt * a.ot + tid);
}

template <typename T, int NR, int QT, bool SPLIT>
int launch(const CUtensorMap& map, const Args& a, int ctas, cudaStream_t st) {
  using S = Shape<NR, QT, SPLIT>;
  static_assert(S::SMEM <= 224 * 1024, "shared memory");
  static std::atomic<uint64_t> told{0};
  const int r = allow_smem(token_kernel<T, NR, QT, SPLIT>, S::SMEM, told, "kv8_attend");
  if (r != FATHOM_OK) return r;
  const int e = launch_after(token_kernel<T, NR, QT, SPLIT>, dim3(ctas), THREADS, S::SMEM, st, "kv8_attend", map, a);
  if (e != FATHOM_OK || (a.share && a.share == a.stride)) return e;     // every row whole: nothing to join
  const dim3 rows((unsigned)(a.G * a.T), (unsigned)(a.B * a.Hkv));
  return launch_after(token_join_kernel<T>, rows, D, 0, st, "kv8_attend", a, ctas);
}

template <typename T, int QT>
int launch_rows(const CUtensorMap& map, const Args& a, int ctas, cudaStream_t st) {
  const int64_t R = a.G * a.T;
  if (R <= 4) return launch<T, 4, QT, false>(map, a, ctas, st);
  if (R <= 8) return launch<T, 8, QT, false>(map, a, ctas, st);
  if (R <= 16) return launch<T, 16, QT, false>(map, a, ctas, st);
  if (R <= 24) return launch<T, 12, QT, true>(map, a, ctas, st);      // 20 rows over 16k: with 16 per thread ~2.5 us more
  return launch<T, 16, QT, true>(map, a, ctas, st);
}

}  // namespace

size_t token_workspace(int64_t BH, int64_t R) { return (size_t)((sm_count() + BH) * R * PART * sizeof(float)); }

int token_attend(const CUtensorMap& map, Args a, int dtype, cudaStream_t st) {
  // one CTA per SM, but no more than there can be tiles
  const int64_t per = cdiv(a.end_dev ? a.cap : a.end, TILE), items = (int64_t)a.B * a.Hkv, tiles = items * (per > 1 ? per : 1);
  const int64_t sms = sm_count() < MAX_CTAS ? sm_count() : MAX_CTAS;
  const int ctas = plan_shares(a, (int)(tiles < sms ? tiles : sms), PIECE, SHORT, 1);
  return dtype == FATHOM_DTYPE_BF16 ? launch_rows<__nv_bfloat16, 2>(map, a, ctas, st)
                                    : launch_rows<__half, 3>(map, a, ctas, st);
}

}  // namespace kv8
}  // namespace fathom
