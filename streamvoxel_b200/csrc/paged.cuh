// The paged cache and the division of its attention among CTAs, shared by the kernels that append to it and read it.
#pragma once

#include "common.cuh"

namespace svx {

// Host checks of a cache's shape and pointers; *shift = log2(page).
int check_cache(const svx_paged_cache* c, const char* who, int* shift);

namespace paged {

constexpr int kTile = 64;   // keys of a step; pages hold 16 * 2^i keys, so a page never straddles a 16-key slice

struct Params {
  const void* q;
  int64_t q_token, q_head;   // strides in elements
  const void *k, *v;         // pools [pages][kv_heads][page][dim]
  const int32_t *table, *lengths, *offsets;
  void* out;                 // [tokens][q_heads][dim]
  float* lse;                // [tokens][q_heads] or null
  uint32_t* status;          // [sequences] or null
  float* partial_o;          // [2 ctas][rows][dim]: unnormalised sums of a CTA's first and last unit where it has
  float2* partial_ml;        // [2 ctas][rows]: only a part of it; their exponent bases and sums of exponentials
  int32_t* join;             // [ctas][8]: the unit that each CTA ends for others (see Join)
  int tokens, sequences, q_heads, kv_heads, group, page_shift, pages, table_width, causal;
  float scale_log2;
  int unit_tokens;           // tokens of a unit
  int blocks;                // units of one (token tile, kv head): its group in parts of at most group_part heads
  int group_part;
  int tile_tokens, tile_rows;  // a unit's rows: tiles of tile_rows of them, tile_tokens tokens in each
  int rows;                  // rows of a partial
  int min_tiles;             // key tiles of a CTA at least
};

// The work is a line of 64-key tiles: for each sequence, each token tile j, each head h (kv head and part of its group),
// the tiles of the keys that the token tile can see (one at least, so that rows without keys are written too). CTA c
// takes an equal run of it, whatever the lengths are; a unit (sequence, j, h) that several CTAs share is joined by a
// second kernel, always in the same order.
struct Sequence {
  int row0, n, len;   // first row, new tokens, keys
};

__device__ __forceinline__ Sequence load_sequence(const Params& p, int s) {
  Sequence q;
  q.row0 = max(0, min(__ldg(p.offsets + s), p.tokens));
  q.n = max(0, min(__ldg(p.offsets + s + 1), p.tokens) - q.row0);
  q.len = max(0, min(__ldg(p.lengths + s), p.table_width << p.page_shift));
  return q;
}

// Keys that the last token of token tile j sees.
__device__ __forceinline__ int unit_limit(const Params& p, const Sequence& q, int j) {
  if (!p.causal) return q.len;
  return max(0, min(q.len, q.len - q.n + min((j + 1) * p.unit_tokens, q.n)));
}
__device__ __forceinline__ int unit_tiles(int limit) { return max(1, (limit + kTile - 1) / kTile); }
__device__ __forceinline__ int token_tiles(const Params& p, const Sequence& q) {
  return (q.n + p.unit_tokens - 1) / p.unit_tokens;
}

// sum of floor((a i + b) / m) over i in [0, n), a, b >= 0: the lattice points under a line, by Euclid's algorithm.
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t sum = 0;
  while (true) {
    if (a >= m) {
      sum += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += n * (b / m);
      b %= m;
    }
    const int64_t y = a * n + b;
    if (y < m) return sum;
    n = y / m;
    b = y % m;
    const int64_t t = m;
    m = a;
    a = t;
  }
}

// Key tiles of the first `count` token tiles of a sequence, for one head.
__device__ __forceinline__ int64_t tiles_before(const Params& p, const Sequence& q, int count) {
  if (!count) return 0;
  if (!p.causal) return (int64_t)count * unit_tiles(q.len);
  if (count == 1) return unit_tiles(unit_limit(p, q, 0));
  const int full = min(count, q.n / p.unit_tokens), base = q.len - q.n;
  // Token tiles that see at most one key tile, then a line of slope unit_tokens / 64, then the last, shorter one.
  const int ones = base >= kTile ? 0 : min(full, (kTile - base) / p.unit_tokens);
  int64_t sum = ones;
  if (full > ones)
    sum += floor_sum(full - ones, kTile, p.unit_tokens, (int64_t)base + (int64_t)(ones + 1) * p.unit_tokens + kTile - 1);
  if (count > full) sum += unit_tiles(unit_limit(p, q, full));
  return sum;
}

// Where a run of tiles begins.
struct Place {
  int64_t begin, end;   // run of the CTA on the line of tiles
  int64_t each;         // tiles of every CTA's run
  int s, j, h, t;
  int64_t unit;         // place of its unit's first tile
};

struct PlanShared {
  int64_t warp_sum[32];
  Place place;
};

// Fills sh.place for run `c` of `ctas`; all threads of the block call it.
template <int kThreads>
__device__ __forceinline__ void plan(const Params& p, int c, int ctas, PlanShared& sh) {
  const int heads = p.kv_heads * p.blocks;
  const int per = (p.sequences + kThreads - 1) / kThreads;
  const int s0 = min(p.sequences, (int)threadIdx.x * per), s1 = min(p.sequences, s0 + per);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) {
    const Sequence q = load_sequence(p, s);
    mine += tiles_before(p, q, token_tiles(p, q)) * heads;
  }
  int64_t sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane_id() >= d) sum += o;
  }
  if (lane_id() == 31) sh.warp_sum[warp_id()] = sum;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp_id()) before += sh.warp_sum[w];
    total += sh.warp_sum[w];
  }
  before += sum - mine;
  const int64_t each = max((int64_t)p.min_tiles, (total + ctas - 1) / ctas);
  const int64_t begin = min(total, each * c), end = min(total, begin + each);
  if (threadIdx.x == 0) {
    sh.place.begin = begin;
    sh.place.end = end;
    sh.place.each = each;
  }
  if (begin < end && begin >= before && begin < before + mine) {
    int64_t at = before;
    for (int s = s0; s < s1; ++s) {
      const Sequence q = load_sequence(p, s);
      const int tiles = token_tiles(p, q);
      const int64_t cost = tiles_before(p, q, tiles) * heads;
      if (begin < at + cost) {
        int lo = 0, hi = tiles - 1;   // the last token tile that begins at or before the place
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (at + tiles_before(p, q, mid) * heads <= begin) lo = mid; else hi = mid - 1;
        }
        at += tiles_before(p, q, lo) * heads;
        const int each_head = unit_tiles(unit_limit(p, q, lo));
        const int h = (int)((begin - at) / each_head);
        sh.place.s = s;
        sh.place.j = lo;
        sh.place.h = h;
        sh.place.unit = at + (int64_t)h * each_head;
        sh.place.t = (int)(begin - sh.place.unit);
        break;
      }
      at += cost;
    }
  }
  __syncthreads();
}

// A walk over units.
struct Cursor {
  int s, j, h, limit, tiles;
  Sequence q;
  __device__ __forceinline__ void set(const Params& p, int s_, int j_, int h_) {
    s = s_;
    j = j_;
    h = h_;
    q = load_sequence(p, s);
    limit = unit_limit(p, q, j);
    tiles = unit_tiles(limit);
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (++h < p.kv_heads * p.blocks) return;
    h = 0;
    if (++j >= token_tiles(p, q)) {
      j = 0;
      do {
        if (++s >= p.sequences) {
          s = p.sequences - 1;
          return;
        }
        q = load_sequence(p, s);
      } while (q.n == 0);
    }
    limit = unit_limit(p, q, j);
    tiles = unit_tiles(limit);
  }
};

// Left by CTA c for the joining kernel, where its run ends a unit that an earlier CTA began: the unit, the CTA that
// began it, and whether the unit was that CTA's first (partial slot 2 first) or its last (2 first + 1). The CTAs between
// hold their parts, like c, in their first slots.
struct Join {
  int valid, s, j, h, first, first_slot, pad0, pad1;
};

// The form for many rows (paged_tc.cu).
int chunk_launch(const Params& p, int dtype, int dim, int ctas, cudaStream_t stream);

}  // namespace paged
}  // namespace svx
