// The division of a batch of paged attention among CTAs, on the host: the arithmetic is that of the kernels (the host
// side of paged.cuh); only the sums over the threads of a block are loops here.
#include <algorithm>
#include <vector>

#include "paged.cuh"

using namespace svx::paged;

// shape: tokens, sequences, kv_heads, causal, unit_tokens, blocks, min_tiles, ctas, two_tiles (whole units are dealt out),
// page_shift, table_width, threads (which add up equal numbers of sequences each). segments: rows of 8 ints (cta, sequence, head, token tile, t0, t1, the unit's tiles, the partial
// that it leaves or -1); joins: rows of 5 (cta, parts, sequence, head, token tile) followed by `parts` partials. Returns
// the segments' count, -1 when one of the arrays is too small; counts[0] = ints of joins, counts[1] = waves.
extern "C" __attribute__((visibility("default"))) int paged_division(const int32_t* shape, const int32_t* lengths,
                                                                     const int32_t* offsets, int32_t* segments,
                                                                     int segment_rows, int32_t* joins, int join_ints,
                                                                     int32_t* counts) {
  Params p{};
  p.tokens = shape[0]; p.sequences = shape[1]; p.kv_heads = shape[2]; p.causal = shape[3]; p.unit_tokens = shape[4];
  p.blocks = shape[5]; p.min_tiles = shape[6]; p.page_shift = shape[9]; p.table_width = shape[10];
  p.lengths = lengths; p.offsets = offsets;
  const int ctas = shape[7];
  std::vector<int64_t> before(p.sequences + 1, 0), line(ctas + 1), dealt(ctas);
  int64_t units_total = 0;
  for (int s = 0; s < p.sequences; ++s) {
    int64_t tiles, units;
    Sequence last;
    add_sequences(p, s, s + 1, &tiles, &units, &last);
    before[s + 1] = before[s] + tiles;
    units_total += units;
  }
  const int64_t total = before[p.sequences], each = equal_share(p, total, ctas);
  int waves = shape[8] ? most_waves(p, units_total, ctas) : 0;
  int64_t most, dealt_total;
  while (true) {
    most = dealt_total = 0;
    for (int c = 0; c < ctas; ++c) {
      dealt[c] = waves ? dealt_whole(p, c, ctas, waves) : 0;
      dealt_total += dealt[c];
      most = dealt[c] > most ? dealt[c] : most;
    }
    if (most <= each) break;
    waves >>= 1;
  }
  int64_t at = dealt_total;
  for (int c = 0; c < ctas; ++c) {
    line[c] = at < total ? at : total;
    at += run_length(each, dealt[c], waves && most == each);
  }
  line[ctas] = total;
  counts[0] = 0;
  counts[1] = waves;
  int rows = 0;
  for (int c = 0; c < ctas; ++c) {
    Place place{};
    place.waves = waves;
    place.count = (int)(line[c + 1] - line[c]);
    if (place.count > 0) {
      const int per = (p.sequences + shape[11] - 1) / shape[11];
      int s0 = 0;
      while (before[std::min(p.sequences, s0 + per)] <= line[c]) s0 += per;
      const int s1 = std::min(p.sequences, s0 + per);
      int64_t tiles, units;
      Sequence last;
      add_sequences(p, s0, s1, &tiles, &units, &last);
      find_place(p, s0, s1, last, before[s0], line[c], each, c, waves ? line.data() : nullptr, &place);
    }
    for (Walk w(p, place, c); w.more(); w.next(p, place, ctas)) {
      if (rows == segment_rows) return -1;
      const bool whole = w.whole();
      const int32_t row[8] = {c, w.at.s, w.at.h, w.at.j, w.t0, w.t1, w.at.tiles, whole ? -1 : (int32_t)partial_slot(c, w.part)};
      for (int i = 0; i < 8; ++i) segments[8 * rows + i] = row[i];
      ++rows;
      if (!ends_for_others(w.part, whole, w.t1 == w.at.tiles)) continue;
      Join join{};
      join.parts = c - place.first + 1;
      join.first = place.first;
      join.first_slot = place.first_slot;
      if (counts[0] + 5 + join.parts > join_ints) return -1;
      int32_t* to = joins + counts[0];
      to[0] = c; to[1] = join.parts; to[2] = w.at.s; to[3] = w.at.h; to[4] = w.at.j;
      for (int i = 0; i < join.parts; ++i) to[5 + i] = (int32_t)join.slot(i);
      counts[0] += 5 + join.parts;
    }
  }
  return rows;
}
