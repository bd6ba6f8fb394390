// The work of the attention kernels over the whole 8-bit cache as a line of tiles, cut into equal shares.
//
// An item is up to 256 query rows (token-major pairs of token and head) of one cache row bh; its tiles are the 128-token
// stretches up to the last key that any of its rows sees.  Items follow each other by bh, then by row; CTA c of C
// takes tiles [c * share, (c + 1) * share) of the line, share = ceil(tiles / C), whatever the lengths are.  Where
// the host knows them, items may lie further apart than their tiles, so that no CTA has pieces of two.
#pragma once
#include "kv8_attn.cuh"
#include "tc.cuh"

namespace fathom {
namespace kv8 {

constexpr int TILE = 128;                    // tokens per tile
constexpr int ROWS = 256;                    // query rows per item

__device__ __forceinline__ int rows_of(const Args& a) { return a.G * (int)a.T; }
__device__ __forceinline__ int items_per_bh(const Args& a) { return (rows_of(a) - 1) / ROWS + 1; }

// Keys that row `row` (token-major) of a sequence with `end` tokens sees.
__device__ __forceinline__ int seen(const Args& a, int end, int row) { return end - ((int)a.T - 1) + row / a.G; }

// Tiles of item `it` of a row bh: up to its last row's last key, one at least.  ONE: every bh is known to be one item.
template <bool ONE = false> __device__ __forceinline__ int tiles_of(const Args& a, int end, int it) {
  if (ONE) return max(1, (end + TILE - 1) / TILE);
  const int last = min((int64_t)(it + 1) * ROWS, (int64_t)rows_of(a)) - 1;
  return max(1, (seen(a, end, last) + TILE - 1) / TILE);
}

// One warp: sum of f over [0, n); if at >= 0, also the first i whose running sum exceeds at (and the sum before it).
template <typename F> __device__ __forceinline__ int64_t warp_line(int n, int64_t at, int* where, int64_t* before, F f) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0;
  bool found = at < 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int64_t mine = i0 + lane < n ? f(i0 + lane) : 0;
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (!found) {
      const unsigned hit = __ballot_sync(0xffffffffu, total + x > at);
      if (hit) {
        const int l = __ffs(hit) - 1;
        *where = i0 + l;
        *before = total + __shfl_sync(0xffffffffu, x - mine, l);
        found = true;
      }
    }
    total += __shfl_sync(0xffffffffu, x, 31);
  }
  return total;
}

// One warp: tiles of the items of one bh of a sequence with `end` tokens; with at >= 0 also the item that holds tile `at`.
__device__ __forceinline__ int64_t bh_line(const Args& a, int end, int64_t at, int* it, int64_t* before) {
  const int per = items_per_bh(a);
  if (per == 1) {
    *it = 0, *before = 0;
    return tiles_of(a, end, 0);
  }
  return warp_line(per, at, it, before, [&](int i) { return (int64_t)tiles_of(a, end, i); });
}

struct Place {
  int item;      // bh * items_per_bh + it
  int tile;      // tile within the item
};

// One warp: tiles of all items, and the place of tile `at` of the line (if at >= 0 and the line is longer).
__device__ inline int64_t line(const Args& a, int64_t at, Place* place) {
  const int per = items_per_bh(a);
  int it = 0, b = 0;
  int64_t before = 0, total = 0, one = 0;
  if (!a.end_dev) {
    one = a.tiles_bh;
    total = one * a.Hkv * a.B;
    if (at < 0 || at >= total) return total;
    b = (int)(at / (one * a.Hkv));
    at -= b * one * a.Hkv;
  } else if (per == 1) {
    total = warp_line(a.B, at, &b, &before, [&](int i) { return (int64_t)tiles_of(a, seq_end(a, i), 0) * a.Hkv; });
    if (at < 0 || at >= total) return total;
    at -= before;
  } else {
    int64_t left = at;
    bool found = false;
    for (int i = 0; i < a.B; ++i) {
      const int64_t n = bh_line(a, seq_end(a, i), -1, &it, &before);
      if (!found && at >= 0 && left < n * a.Hkv) found = true, b = i, at = left;
      left -= n * a.Hkv;
      total += n * a.Hkv;
    }
    if (!found) return total;
  }
  const int end = seq_end(a, b);
  if (a.end_dev) one = bh_line(a, end, -1, &it, &before);
  const int h = (int)(at / one);
  at -= h * one;
  bh_line(a, end, at, &it, &before);
  *place = Place{(b * a.Hkv + h) * per + it, (int)(at - before)};
  return total;
}

// n / d for 0 <= n, d > 0: in 32 bits where n allows it (a 64-bit division is ~100 cycles longer).
__device__ __forceinline__ int64_t quotient(int64_t n, int d) {
  return n >> 32 ? n / d : (int64_t)((uint32_t)n / (uint32_t)d);
}

// Tiles per CTA where the device cuts the line: at least `least`, or an item's where those are fewer.
__device__ __forceinline__ int64_t share_of(const Args& a, int64_t total, int ctas) {
  const int64_t share = quotient(total + ctas - 1, ctas);
  return share >= a.least ? share : max(share, min((int64_t)a.least, quotient(total, a.B * a.Hkv * items_per_bh(a))));
}

// One warp: where this CTA's share begins, how many tiles it has (0 or less: none) and how many a CTA has at most.  A
// token's latency counts on this: the common forms, a plan or up to 32 sequences of one item per bh, take one pass.
template <bool ONE = false> __device__ inline Place my_share(const Args& a, int* count, int* per_cta) {
  const int lane = threadIdx.x & 31;
  Place p{0, 0};
  if (a.share) {
    const int64_t at = (int64_t)a.share * blockIdx.x;
    *per_cta = a.share;
    p.item = (int)quotient(at, a.stride);
    p.tile = (int)(at - (int64_t)p.item * a.stride);
    const int nt = tiles_of<ONE>(a, seq_end(a, 0), ONE ? 0 : p.item % items_per_bh(a));
    const bool apart = a.stride > nt || a.share == a.stride;       // no other item's tiles in this share
    *count = (int)min((int64_t)a.share, apart ? (int64_t)nt - p.tile : (int64_t)a.B * a.Hkv * nt - at);
    return p;
  }
  if ((ONE || items_per_bh(a) == 1) && a.B <= 32) {       // (ragged: equal lengths have a plan)
    const int nt = lane < a.B ? tiles_of<ONE>(a, seq_end(a, lane), 0) : 0;
    const int64_t mine = (int64_t)nt * a.Hkv;
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int64_t total = __shfl_sync(0xffffffffu, x, 31), share = share_of(a, total, gridDim.x);
    int64_t at = share * blockIdx.x;
    *per_cta = (int)share;
    *count = (int)min(share, total - at);
    if (*count <= 0) return p;
    const int b = __ffs(__ballot_sync(0xffffffffu, x > at)) - 1;     // the first sequence that ends past `at`
    at -= __shfl_sync(0xffffffffu, x - mine, b);
    const int n = __shfl_sync(0xffffffffu, nt, b), bh = (int)quotient(at, n);
    return Place{b * a.Hkv + bh, (int)(at - (int64_t)bh * n)};
  }
  const int64_t total = line(a, -1, &p), share = share_of(a, total, gridDim.x), first = share * blockIdx.x;
  *per_cta = (int)share;
  *count = (int)min(share, total - first);
  if (*count > 0) line(a, first, &p);
  return p;
}

// A share as its pieces of items, the same walk in every role; made by a converged warp and uniform as the compiler sees
// it, so that loops over it are.
template <bool ONE = false> struct Walk {
  const Args& a;
  int per, item, tile, left;
  int b, bh, it, end, n, j0, j1;   // item within bh; its sequence's tokens; its tiles; this piece's tiles [j0, j1)
  __device__ Walk(const Args& a_, const Place& p, int count)
      : a(a_), per(ONE ? 1 : items_per_bh(a_)), item(tc::uniform(p.item)), tile(tc::uniform(p.tile)),
        left(tc::uniform(max(count, 0))) {}
  // accumulators of 128 rows that the item needs
  __device__ int halves() const { return rows_of(a) - it * ROWS > ROWS / 2 ? 2 : 1; }
  __device__ bool next() {
    if (left <= 0) return false;
    bh = ONE ? item : item / per;
    it = item - bh * per;
    b = div_small(bh, a.inv_hkv);
    end = seq_end(a, b);
    n = tiles_of<ONE>(a, end, it);
    j0 = tile;
    j1 = min(n, j0 + left);
    left -= j1 - j0;
    ++item;
    tile = 0;
    return true;
  }
};

// Cuts the line for at most `most` CTAs at a time and returns the grid.  Where the host knows the lengths:
//  * items of at most `whole` tiles have a CTA each, and nothing is to be joined;
//  * else, where every bh is one item, the items follow each other, and a CTA may have pieces of two, or each has k CTAs of
//    its own: whichever takes the fewer tiles, beginning and ending a piece taking as long as `piece`.
// All other lines are left to the device.  Shares have at least `least` tiles.
inline int plan_shares(Args& a, int most, int piece, int whole, int least) {
  a.least = least;
  if (a.end_dev) return most;
  const int64_t per = (a.G * a.T - 1) / ROWS + 1;
  for (int64_t it = 0; it < per; ++it) {
    const int64_t rows = a.G * a.T, last = ((it + 1) * ROWS < rows ? (it + 1) * ROWS : rows) - 1;
    const int64_t see = a.end - (a.T - 1) + last / a.G;            // as tiles_of
    a.tiles_bh += see > TILE ? cdiv(see, TILE) : 1;
  }
  const int64_t items = (int64_t)a.B * a.Hkv * per, nt = a.end > TILE ? cdiv(a.end, TILE) : 1;   // of the longest
  if (nt <= whole) {
    a.share = a.stride = (int)nt;
    return (int)items;
  }
  if (per > 1) return most;
  const int64_t dense = cdiv(items * nt, most) > least ? cdiv(items * nt, most) : least;
  const int64_t fit = most / items, k = fit < cdiv(nt, least) ? fit : cdiv(nt, least);
  const bool apart = k >= 1 && cdiv(nt, k) <= dense + piece;
  a.share = (int)(apart ? cdiv(nt, k) : dense);
  a.stride = (int)(apart ? a.share * k : nt);
  return (int)cdiv(items * a.stride, a.share);
}

}  // namespace kv8
}  // namespace fathom
