// The distinct rows among a KV head's picks, for caches in host memory: each is fetched once over the host link
// (attn.cu for bf16 rows, kv8_picks.cu for 8-bit ones).
#pragma once
#include "common.cuh"

namespace fathom {
namespace {

constexpr int DT = 1024;      // dedupe threads
constexpr int MAX_M = 16384;  // G*k per (batch, kv-head) handled by one dedupe CTA

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

__device__ uint32_t block_exclusive_scan(uint32_t v, uint32_t* s_warp, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const uint32_t w = lane < nw ? s_warp[lane] : 0u;
    uint32_t z = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    if (lane < nw) s_warp[lane] = z - w;
    if (lane == 31) s_warp[32] = z;
  }
  __syncthreads();
  const uint32_t res = s_warp[warp] + x - v;
  *total = s_warp[32];
  __syncthreads();
  return res;
}

constexpr uint32_t EMPTY = 0xFFFFFFFFu;
constexpr int MAX_TS = 32768;         // hash table slots (128 KB of shared memory; + M keys, 2 x NB bins)
constexpr int PICKS_PER_THREAD = MAX_M / DT;
constexpr int NB = 2048;              // rank buckets (high bits of the row index)
constexpr int MAX_PER = MAX_TS / DT;  // table slots per dedupe thread

__device__ __forceinline__ uint32_t hash_slot(uint32_t key, int log2ts) {
  return (key * 0x9E3779B1u) >> (32 - log2ts);
}

// One CTA per (batch, kv-head).  Every owned pick is inserted into an open-addressing table in
// shared memory (atomicCAS, linear probing; the table has at least twice as many slots as picks,
// so a probe sequence always ends at an empty slot or at its own key).  The distinct indices are
// then ranked in ascending order: a counting pass over NB buckets of their high bits, a block scan,
// a scatter into bucket order, and within each (small) bucket a count of the smaller keys.  The
// unique list is therefore sorted, so the gather walks the source in address order (fewer address
// translations per byte over the host link), and every rank is independent of the insert order.
// Each pick remembers its table slot and reads its rank.
__global__ void __launch_bounds__(DT) dedupe_kernel(const int64_t* __restrict__ idx, int64_t M, int64_t idx_lo,
                                                    int64_t idx_hi, int64_t row_limit, int log2ts, int bshift,
                                                    int32_t* __restrict__ slot,
                                                    int64_t* __restrict__ uniq, int32_t* __restrict__ ucount) {
  extern __shared__ uint32_t s_tab[];  // 1 << log2ts slots, then M keys in bucket order
  __shared__ uint32_t s_warp[33];
  __shared__ uint32_t s_bin[NB], s_cur[NB];
  const int64_t bh = blockIdx.x;
  const int TS = 1 << log2ts;
  uint32_t* s_sorted = s_tab + TS;
  for (int i = threadIdx.x; i < TS; i += blockDim.x) s_tab[i] = EMPTY;
  for (int b = threadIdx.x; b < NB; b += blockDim.x) s_bin[b] = 0u;
  __syncthreads();
  const int64_t* ib = idx + bh * M;
  int pos[PICKS_PER_THREAD];
  int64_t tv[PICKS_PER_THREAD];   // every pick load in flight before the first insert
#pragma unroll
  for (int u = 0; u < PICKS_PER_THREAD; ++u) {
    const int64_t i = threadIdx.x + (int64_t)u * DT;
    tv[u] = i < M ? ib[i] : -1;
  }
#pragma unroll
  for (int u = 0; u < PICKS_PER_THREAD; ++u) {
    const int64_t i = threadIdx.x + (int64_t)u * DT;
    pos[u] = -1;
    if (i < M) {
      const int64_t t = tv[u];
      if (t >= idx_lo && t < idx_hi && t - idx_lo < row_limit) {
        const uint32_t key = (uint32_t)(t - idx_lo);
        uint32_t h = hash_slot(key, log2ts);
        for (int probe = 0; probe < TS; ++probe) {
          const uint32_t old = atomicCAS(&s_tab[h], EMPTY, key);
          if (old == EMPTY || old == key) {
            pos[u] = (int)h;
            break;
          }
          h = (h + 1) & (TS - 1);
        }
      }
    }
  }
  __syncthreads();
  // ascending ranks of the distinct keys (each thread a contiguous chunk of the table)
  const int per = TS / DT > 0 ? TS / DT : 1;
  const int h0 = threadIdx.x * per;
  const int h1 = h0 + per < TS ? h0 + per : TS;
  for (int h = h0; h < h1; ++h)
    if (s_tab[h] != EMPTY) atomicAdd(&s_bin[s_tab[h] >> bshift], 1u);
  __syncthreads();
  uint32_t bsum = 0;   // bins 2t, 2t+1 of thread t (NB = 2 * DT)
  const uint32_t c0 = s_bin[2 * threadIdx.x], c1 = s_bin[2 * threadIdx.x + 1];
  uint32_t total;
  bsum = block_exclusive_scan(c0 + c1, s_warp, &total);
  s_bin[2 * threadIdx.x] = bsum;
  s_bin[2 * threadIdx.x + 1] = bsum + c0;
  s_cur[2 * threadIdx.x] = bsum;
  s_cur[2 * threadIdx.x + 1] = bsum + c0;
  __syncthreads();
  for (int h = h0; h < h1; ++h)
    if (s_tab[h] != EMPTY) s_sorted[atomicAdd(&s_cur[s_tab[h] >> bshift], 1u)] = s_tab[h];
  __syncthreads();   // s_cur[b] is now the end of bucket b
  uint32_t myrank[MAX_PER];
  int64_t* ul = uniq + bh * M;
  for (int h = h0; h < h1; ++h) {
    const uint32_t x = s_tab[h];
    if (x == EMPTY) continue;
    const uint32_t b = x >> bshift;
    uint32_t r = s_bin[b];
    for (uint32_t t = s_bin[b]; t < s_cur[b]; ++t) r += s_sorted[t] < x;
    myrank[h - h0] = r;
    ul[r] = (int64_t)x;
  }
  __syncthreads();   // every key read: the slots may now hold ranks
  for (int h = h0; h < h1; ++h)
    if (s_tab[h] != EMPTY) s_tab[h] = myrank[h - h0];
  __syncthreads();
  int32_t* sl = slot + bh * M;
#pragma unroll
  for (int u = 0; u < PICKS_PER_THREAD; ++u) {
    const int64_t i = threadIdx.x + (int64_t)u * DT;
    if (i < M) sl[i] = pos[u] >= 0 ? (int32_t)s_tab[pos[u]] : -1;
  }
  if (threadIdx.x == 0) ucount[bh] = (int32_t)total;
}

// Enqueues the dedupe of idx [BH][M]: slot [BH][M], uniq [BH][M], ucount [BH].
inline int launch_dedupe(const int64_t* idx, int64_t BH, int64_t M, int64_t idx_lo, int64_t idx_hi, int64_t row_limit,
                         int32_t* slot, int64_t* uniq, int32_t* ucount, cudaStream_t st) {
  int log2ts = 10;
  while ((1 << log2ts) < 2 * M) ++log2ts;           // load factor <= 1/2
  FATHOM_REQUIRE((1 << log2ts) <= MAX_TS, FATHOM_ERR_UNSUPPORTED, "decode_attention: too many picks");
  const size_t smem = sizeof(uint32_t) * (((size_t)1 << log2ts) + (size_t)M);   // table + keys in bucket order
  cudaFuncSetAttribute(dedupe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  int bshift = 0;   // NB buckets cover the readable rows [0, row_limit)
  while (((row_limit - 1) >> bshift) >= NB) ++bshift;
  dedupe_kernel<<<(unsigned)BH, DT, smem, st>>>(idx, M, idx_lo, idx_hi, row_limit, log2ts, bshift, slot, uniq, ucount);
  return FATHOM_OK;
}

}  // namespace
}  // namespace fathom
