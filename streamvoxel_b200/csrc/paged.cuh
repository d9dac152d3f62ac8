// The paged cache and the division of its attention among CTAs, shared by the kernels that append to it and read it.
#pragma once

#include "common.cuh"

namespace svx {

// Host checks of a cache's shape and pointers; *shift = log2(page).
int check_cache(const svx_paged_cache* c, const char* who, int* shift);

namespace paged {

constexpr int kTile = 64;   // keys of a step; pages hold 16 * 2^i keys, so a page never straddles a 16-key slice

struct Join;

struct Params {
  const void* q;
  int64_t q_token, q_head;   // strides in elements
  const void *k, *v;         // pools [pages][kv_heads][page][dim]
  const int32_t *table, *lengths, *offsets;
  void* out;                 // [tokens][q_heads][dim]
  float* lse;                // [tokens][q_heads] or null
  uint32_t* status;          // [sequences] or null
  // Unnormalised sums of a CTA's first and last unit where it has only a part of it: [2 ctas][rows][dim] (few rows), or
  // [2 ctas][dim / 4][rows] groups of four columns (many rows); their exponent bases and sums of exponentials
  // [2 ctas][rows].
  float* partial_o;
  float2* partial_ml;
  Join* join;                // [ctas]: the unit that each CTA ends for others
  int tokens, sequences, q_heads, kv_heads, group, page_shift, pages, table_width, causal;
  float scale_log2;
  int unit_tokens;           // tokens of a unit
  int blocks;                // units of one (token tile, kv head): its group in parts of at most group_part heads
  int group_part;
  int tile_tokens, tile_rows;  // a unit's rows: tiles of tile_rows of them, tile_tokens tokens in each
  int rows;                  // rows of a partial
  int min_tiles;             // key tiles of a CTA at least
};

// The work is a line of 64-key tiles: for each sequence, each head h (kv head and part of its group), each token tile j,
// the tiles of the keys that the token tile can see (one at least, so that rows without keys are written too). A CTA takes
// an equal run of the line, whatever the lengths are; a unit (sequence, h, j) that several CTAs share is joined by a
// second kernel, always in the same order. Calls with several units for each CTA first deal whole units out in waves (CTA
// c takes units c, c + ctas, ...): the token tiles of one head then run side by side over the same keys, which come from
// memory once, and only the last units' tiles are divided into runs, whose lengths make every CTA's total equal.
// All arithmetic of the division is host code too, which the tests run.
#define SVX_HOST_DEVICE __host__ __device__ __forceinline__

SVX_HOST_DEVICE int32_t entry(const int32_t* at) {
#ifdef __CUDA_ARCH__
  return __ldg(at);
#else
  return *at;
#endif
}

struct Sequence {
  int row0, n, len;   // first row, new tokens, keys
};

SVX_HOST_DEVICE Sequence load_sequence(const Params& p, int s) {
  Sequence q;
  q.row0 = max(0, min(entry(p.offsets + s), p.tokens));
  q.n = max(0, min(entry(p.offsets + s + 1), p.tokens) - q.row0);
  q.len = max(0, min(entry(p.lengths + s), p.table_width << p.page_shift));
  return q;
}

// Keys that the last token of token tile j sees.
SVX_HOST_DEVICE int unit_limit(const Params& p, const Sequence& q, int j) {
  if (!p.causal) return q.len;
  return max(0, min(q.len, q.len - q.n + min((j + 1) * p.unit_tokens, q.n)));
}
SVX_HOST_DEVICE int unit_tiles(int limit) { return max(1, (limit + kTile - 1) / kTile); }
SVX_HOST_DEVICE int token_tiles(const Params& p, const Sequence& q) {
  return (q.n + p.unit_tokens - 1) / p.unit_tokens;
}

// x / y, mostly of values below 2^32.
SVX_HOST_DEVICE int64_t quotient(int64_t x, int64_t y) {
  return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

// sum of floor((a i + b) / 64) over i in [0, n), a, b >= 0: of the terms themselves, without their residues mod 64, which
// repeat every 64 / gcd(a, 64) terms; a whole period holds every residue that is b's mod the gcd once.
SVX_HOST_DEVICE int64_t floor_sum(int64_t n, int a, int64_t b) {
  const int g = (a & 63) ? (a & -a) : 64, period = 64 / g;
  const int64_t periods = n / period;
  int64_t residues = periods * ((int64_t)period * (b & (g - 1)) + g * (period * (period - 1) / 2));
  for (int i = 0; i < (int)(n - periods * period); ++i) residues += ((int64_t)a * i + b) & 63;
  return (a * (n * (n - 1) / 2) + b * n - residues) >> 6;
}

// Key tiles of the first `count` token tiles of a sequence, for one head.
SVX_HOST_DEVICE int64_t tiles_before(const Params& p, const Sequence& q, int count) {
  if (!count) return 0;
  if (!p.causal) return (int64_t)count * unit_tiles(q.len);
  if (count == 1) return unit_tiles(unit_limit(p, q, 0));
  const int full = min(count, q.n / p.unit_tokens), base = q.len - q.n;
  // Token tiles that see at most one key tile, then a line of slope unit_tokens / 64, then the last, shorter one.
  const int ones = base >= kTile ? 0 : min(full, (kTile - base) / p.unit_tokens);
  int64_t sum = ones;
  if (full > ones)
    sum += floor_sum(full - ones, p.unit_tokens, (int64_t)base + (int64_t)(ones + 1) * p.unit_tokens + kTile - 1);
  if (count > full) sum += unit_tiles(unit_limit(p, q, full));
  return sum;
}

// A CTA's share: units cta + k ctas for k < waves, then the run [begin, end) of the line of tiles.
struct Place {
  int waves;
  int s, j, h, t;       // where the run begins
  Sequence q;           // sequence s
  int count;            // its tiles
  int first, first_slot;  // for the join of the unit that the run begins inside of: see Join
};

struct PlanShared {
  int64_t warp_tiles[16], warp_units[16];   // of at most 512 threads
  Place place;
};

// Sum over the lanes up to this one.
__device__ __forceinline__ int64_t warp_scan(int64_t x) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane_id() >= d) x += o;
  }
  return x;
}

// Sums over the block of one value or (kBoth) two; *before: of the threads before this one.
template <int kThreads, bool kBoth>
__device__ __forceinline__ void block_scan(int64_t a, int64_t b, PlanShared& sh, int64_t* before_a, int64_t* before_b,
                                           int64_t* total_a, int64_t* total_b) {
  const int64_t sa = warp_scan(a), sb = kBoth ? warp_scan(b) : 0;
  __syncthreads();
  if (lane_id() == 31) {
    sh.warp_tiles[warp_id()] = sa;
    if (kBoth) sh.warp_units[warp_id()] = sb;
  }
  __syncthreads();
  *before_a = sa - a;
  *before_b = sb - b;
  *total_a = *total_b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t x = sh.warp_tiles[w];
    *before_a += w < warp_id() ? x : 0;
    *total_a += x;
    if (kBoth) {
      const int64_t y = sh.warp_units[w];
      *before_b += w < warp_id() ? y : 0;
      *total_b += y;
    }
  }
}

// A walk over units.
struct Cursor {
  int s, j, h, limit, tiles;
  Sequence q;
  SVX_HOST_DEVICE void see(const Params& p) {
    limit = unit_limit(p, q, j);
    tiles = unit_tiles(limit);
  }
  SVX_HOST_DEVICE void set(const Params& p, const Place& place) {
    s = place.s;
    j = place.j;
    h = place.h;
    q = place.q;
    see(p);
  }
  SVX_HOST_DEVICE void first(const Params& p) {
    s = j = h = 0;
    q = load_sequence(p, 0);
    see(p);
  }
  SVX_HOST_DEVICE void next(const Params& p) {
    if (++j >= token_tiles(p, q)) {
      j = 0;
      if (++h >= p.kv_heads * p.blocks) {
        h = 0;
        do {
          if (++s >= p.sequences) {
            s = p.sequences - 1;
            return;
          }
          q = load_sequence(p, s);
        } while (q.n == 0);
      }
    }
    see(p);
  }
  // On by `count` units; false past the last one.
  SVX_HOST_DEVICE bool skip(const Params& p, int64_t count) {
    const int heads = p.kv_heads * p.blocks;
    int per_head = token_tiles(p, q);
    int64_t at = (int64_t)h * per_head + j + count;
    while (at >= (int64_t)heads * per_head) {
      at -= (int64_t)heads * per_head;
      if (++s >= p.sequences) {
        s = p.sequences - 1;
        return false;
      }
      q = load_sequence(p, s);
      per_head = token_tiles(p, q);
    }
    h = (int)(at / per_head);
    j = (int)(at - (int64_t)h * per_head);
    see(p);
    return true;
  }
};

// Tiles and units of the sequences [s0, s1), all heads; *last: the last of them.
SVX_HOST_DEVICE void add_sequences(const Params& p, int s0, int s1, int64_t* tiles, int64_t* units, Sequence* last) {
  const int heads = p.kv_heads * p.blocks;
  *tiles = *units = 0;
  *last = Sequence{};
  for (int s = s0; s < s1; ++s) {
    const Sequence q = *last = load_sequence(p, s);
    const int n = token_tiles(p, q);
    *tiles += tiles_before(p, q, n) * heads;
    *units += (int64_t)n * heads;
  }
}

// Tiles of a CTA: an equal part of the line.
SVX_HOST_DEVICE int64_t equal_share(const Params& p, int64_t total, int ctas) {
  return max((int64_t)p.min_tiles, quotient(total + ctas - 1, ctas));
}

// Waves of whole units to begin with. The last wave and the rest stay for the runs. A step of `ctas` units reads every
// sequence that it passes, one after the other, so they are not to be many: from 16 units a sequence on, dealing pays
// (against none: 32 chunks of 250 tokens x 4 heads of 128 over 2000 older keys, 8 kv heads, 32 units each, 300 us against 320;
// 16 of 1000 x 96 over 4000, 32 each, 309 against 350; but 64 of 300 x 6 heads of 64, 32 each, 860 against 832). With 16 (64
// chunks of 125 x 4 of 128) it is even, 312 against 314.
SVX_HOST_DEVICE int most_waves(const Params& p, int64_t units_total, int ctas) {
  if (units_total < 2 * (int64_t)ctas || units_total < 16 * (int64_t)p.sequences) return 0;
  return (int)min(units_total / ctas - 1, (int64_t)1 << 20);
}

// Tiles of the units that CTA `c` takes whole.
SVX_HOST_DEVICE int64_t dealt_whole(const Params& p, int c, int ctas, int waves) {
  int64_t tiles = 0;
  Cursor u;
  u.first(p);
  bool ok = u.skip(p, c);
  for (int k = 0; ok && k < waves; ++k) {
    tiles += u.tiles;
    if (k + 1 < waves) ok = u.skip(p, ctas);
  }
  return tiles;
}

// Tiles of the run of a CTA that takes `dealt` tiles whole. full: the whole units of some CTA are an equal share already;
// every share is then a tile longer, so that no run before the line's end is empty. A run in the middle of a unit counts as
// one of its parts (Join), and an empty one would leave nothing where the joining kernel reads.
SVX_HOST_DEVICE int64_t run_length(int64_t each, int64_t dealt, bool full) { return each + (full ? 1 : 0) - dealt; }

// Where CTA c's run begins: tile `begin` of the line, which lies among the sequences [s0, s1); `before` tiles come before
// them and `last` is the last of them. line: the runs' begins where units are dealt out whole, null where every run is
// `each` tiles long.
SVX_HOST_DEVICE void find_place(const Params& p, int s0, int s1, const Sequence& last, int64_t before, int64_t begin,
                                int64_t each, int c, const int64_t* line, Place* place) {
  const int heads = p.kv_heads * p.blocks;
  int64_t at = before;
  for (int s = s0; s < s1; ++s) {
    const Sequence q = s + 1 < s1 ? load_sequence(p, s) : last;
    const int n = token_tiles(p, q);
    const int64_t head = tiles_before(p, q, n);
    if (begin < at + head * heads) {
      const int h = (int)quotient(begin - at, head);
      at += h * head;
      int lo = 0, hi = n - 1;   // the last token tile that begins at or before the place
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at + tiles_before(p, q, mid) <= begin) lo = mid; else hi = mid - 1;
      }
      at += tiles_before(p, q, lo);
      place->s = s;
      place->q = q;
      place->j = lo;
      place->h = h;
      place->t = (int)(begin - at);
      // The CTA whose run holds the unit's first tile.
      int first = (int)quotient(at, each);
      if (line) {
        first = 0;
        int top = c;
        while (first < top) {
          const int mid = (first + top + 1) >> 1;
          if (line[mid] <= at) first = mid; else top = mid - 1;
        }
      }
      place->first = first;
      place->first_slot = at == (line ? line[first] : first * each) ? 0 : 1;
      return;
    }
    at += head * heads;
  }
}

// Fills sh.place for CTA `c` of `ctas`; all threads of the block call it. kWaves: deal whole units out first where there
// are enough of them; `scratch` then holds 8 * ctas + 8 bytes of shared memory.
template <int kThreads, bool kWaves>
__device__ __forceinline__ void plan(const Params& p, int c, int ctas, PlanShared& sh, int64_t* scratch) {
  const int tid = threadIdx.x;
  // Up to 32 sequences: every warp adds them up for itself, a lane each, without the block's barriers.
  const bool few = p.sequences <= 32;
  const int id = few ? lane_id() : tid, per = few ? 1 : (p.sequences + kThreads - 1) / kThreads;
  const int s0 = min(p.sequences, id * per), s1 = min(p.sequences, s0 + per);
  int64_t tiles, units, before, units_before, total, units_total;
  Sequence last;
  add_sequences(p, s0, s1, &tiles, &units, &last);
  if (few) {
    before = warp_scan(tiles);
    units_before = kWaves ? warp_scan(units) : 0;
    total = __shfl_sync(0xffffffffu, before, 31);
    units_total = __shfl_sync(0xffffffffu, units_before, 31);
    before -= tiles;
  } else {
    block_scan<kThreads, kWaves>(tiles, units, sh, &before, &units_before, &total, &units_total);
  }
  const int64_t each = equal_share(p, total, ctas);
  int waves = kWaves ? most_waves(p, units_total, ctas) : 0;
  int64_t begin = min(total, each * c), end = min(total, begin + each);
  if (kWaves && waves) {
    // Tiles of the units that each CTA takes whole, which are not to be more than its share; then the runs that fill them
    // up to it.
    int64_t dealt;
    while (true) {
      dealt = waves && tid < ctas ? dealt_whole(p, tid, ctas, waves) : 0;
      if (!__syncthreads_or(dealt > each)) break;
      waves >>= 1;
    }
    const bool full = __syncthreads_or(tid < ctas && dealt == each);
    const int64_t need = tid < ctas ? run_length(each, dealt, full) : 0;   // waves == 0: equal runs of the whole line
    int64_t need_before, dealt_before, need_total, dealt_total;
    block_scan<kThreads, true>(need, dealt, sh, &need_before, &dealt_before, &need_total, &dealt_total);
    if (tid < ctas) scratch[tid] = min(total, dealt_total + need_before);
    if (tid == 0) scratch[ctas] = total;
    __syncthreads();
    begin = scratch[c];
    end = scratch[c + 1];
  }
  if (tid == 0) {
    sh.place.waves = waves;
    sh.place.count = (int)(end - begin);
  }
  if (begin < end && begin >= before && begin < before + tiles && (!few || tid < 32))
    find_place(p, s0, s1, last, before, begin, each, c, kWaves && waves ? scratch : nullptr, &sh.place);
  __syncthreads();
}

// A CTA's share, unit by unit: key tiles [t0, t1) of the unit at `at`; `part` counts the units of its run of the line (-1:
// a unit dealt out whole).
struct Walk {
  Cursor at;
  int t0, t1, waves, left, units, part;
  SVX_HOST_DEVICE Walk(const Params& p, const Place& place, int cta) {
    waves = place.waves;
    left = place.count;
    units = 0;
    part = -1;
    t0 = t1 = 0;
    if (waves) {
      at.first(p);
      at.skip(p, cta);
      t1 = at.tiles;
    } else {
      start_run(p, place);
    }
  }
  SVX_HOST_DEVICE void start_run(const Params& p, const Place& place) {
    if (left <= 0) return;
    part = 0;
    at.set(p, place);
    t0 = place.t;
    t1 = min(at.tiles, t0 + left);
  }
  SVX_HOST_DEVICE bool more() const { return waves > 0 || left > 0; }
  SVX_HOST_DEVICE bool whole() const { return t0 == 0 && t1 == at.tiles; }
  SVX_HOST_DEVICE void next(const Params& p, const Place& place, int ctas) {
    ++units;
    if (waves) {
      if (--waves) {
        at.skip(p, ctas);
        t1 = at.tiles;
      } else {
        start_run(p, place);
      }
      return;
    }
    left -= t1 - t0;
    if (left <= 0) return;
    ++part;
    at.next(p);
    t0 = 0;
    t1 = min(at.tiles, left);
  }
};

// Left by CTA c for the joining kernel, where its run ends a unit that an earlier CTA began: the unit's rows and heads,
// the CTA that began it, and whether the unit was that CTA's first of the line (partial slot 2 first) or its last
// (2 first + 1). The CTAs between hold their parts, like c, in their first slots: none of their runs is empty.
struct Join {
  int parts;               // 0: nothing to join
  int first, first_slot;
  int row, tokens;         // its tokens' first row, and their count
  int head, group;         // its first query head, and their count
  int pad;
  // The partial that holds part i.
  SVX_HOST_DEVICE int64_t slot(int i) const { return 2 * (int64_t)(first + i) + (i == 0 ? first_slot : 0); }
};

// The partial that CTA c leaves of the unit that is number `part` of its run; whether it ends that unit for others.
SVX_HOST_DEVICE int64_t partial_slot(int c, int part) { return 2 * (int64_t)c + (part > 0 ? 1 : 0); }
SVX_HOST_DEVICE bool ends_for_others(int part, bool whole, bool at_end) { return part == 0 && !whole && at_end; }

// The form for many rows (paged_tc.cu).
int chunk_launch(const Params& p, int dtype, int dim, int ctas, cudaStream_t stream);

}  // namespace paged
}  // namespace svx
