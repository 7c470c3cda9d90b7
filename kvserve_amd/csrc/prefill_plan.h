// The prefill part's flat space of positions (see prefill_units in paged_attention.hip): plain
// integer functions of a sequence's lengths, shared by the kernels and compiled for the host by
// the test that compares them with a walk over every tile.
//
// A prefill-class sequence has R = q_len G query rows per kv head in ceil(R / PR) tiles of PR
// rows. Tile t occupies kTileCost + pre_tile_chunks positions: its fixed cost (query load, pipeline
// fill, output write), then the 32-key chunks its last row can see.
#pragma once
#include <stdint.h>

namespace kvh {

#ifndef KVH_PLAN_FN
#define KVH_PLAN_FN __device__ __forceinline__
#endif

constexpr int kPlanChunk = 32;  // keys of a chunk
// Fixed cost of a tile in chunk steps: each tile occupies kTileCost + chunks positions of the
// flat space, the first kTileCost virtual.
constexpr int kTileCost = 4;

// What the plan reads of a sequence: query rows R, the context before the step, the query
// length and the keys present (seq_len clamped to the block table's capacity).
struct PreSeq {
  int32_t R, q_len, kv_total;
  int64_t ctx;
};

// Chunks of tile t: those its last row can see, at least one so that every tile is visited
// and written.
KVH_PLAN_FN int pre_tile_chunks(const PreSeq& s, int G, int PR, int t) {
  const int end = PR * t + PR - 1, last = end < s.R - 1 ? end : s.R - 1;
  int64_t lim = s.ctx + last / G + 1;
  lim = lim < 0 ? 0 : (lim > s.kv_total ? s.kv_total : lim);
  const int c = (int)((lim + kPlanChunk - 1) / kPlanChunk);
  return c > 1 ? c : 1;
}

// floor(log2) of a power of two.
KVH_PLAN_FN int pre_log2(int x) { return __builtin_ctz((unsigned)x); }

// The greatest common divisor of two positive numbers.
KVH_PLAN_FN int pre_gcd(int a, int b) {
  while (b) {
    const int r = a % b;
    a = b;
    b = r;
  }
  return a;
}

// Positions of tiles 0 .. t - 1 of one kv head, t <= ceil(R / PR). With no clamped length, full
// tile i (from 1) sees ctx + ceil(PR i / G) keys, ceil((ctx G + PR i) / (32 G)) chunks, and the sum over
// i = 1 .. n splits into whole chunks per tile and a remainder that repeats after a few tiles: a few
// terms whatever the length of the prompt.
//  * step = PR / G where G divides PR: the remainder is that of (ctx + step i) / 32 and repeats every
//    32 / gcd(step, 32) tiles (2 at PR = 192, G = 4), with no division.
//  * step = 0, G does not divide PR (groups of 5, 7 or 10; of 3 and 6 at PR = 128): every 32 G /
//    gcd(PR, 32 G) tiles, at most G. A walk from the first tile instead made the search for a unit's
//    start quadratic in the prompt: 32768 tokens, G = 7, E4M3 caches, 11466 us against 8313.
// A clamped length is added tile by tile.
KVH_PLAN_FN int64_t pre_prefix(const PreSeq& s, int G, int PR, int step, int t) {
  if (t <= 0) return 0;
  int64_t n = (int64_t)kTileCost * t;
  if (s.ctx < 0 || s.ctx + s.q_len != s.kv_total) {
    for (int i = 0; i < t; ++i) n += pre_tile_chunks(s, G, PR, i);
    return n;
  }
  const int tiles = s.R / PR, full = t < tiles ? t : tiles;
  if (step > 0) {
    const int a = step / kPlanChunk, b = step % kPlanChunk;
    const int64_t e = s.ctx + kPlanChunk - 1;
    const int e0 = (int)(e % kPlanChunk);
    n += full * (e / kPlanChunk) + (int64_t)a * full * (full + 1) / 2;
    const int lp = pre_log2(kPlanChunk) - pre_log2(b ? b & -b : kPlanChunk);  // log2 of the period
    const int per = (b << lp) / kPlanChunk;
    for (int r = 1; r <= 1 << lp && r <= full; ++r) {  // tiles r, r + period, ... (1-based)
      const int64_t m = ((full - r) >> lp) + 1;
      n += m * ((e0 + b * r) / kPlanChunk) + per * (m * (m - 1) / 2);
    }
  } else {
    const int M = kPlanChunk * G, g = pre_gcd(PR, M), period = M / g, per = PR / g;
    const int a = PR / M, b = PR % M, whole = full / period, left = full % period;
    int q = 0, rem = (int)(s.ctx % kPlanChunk) * G + M - 1;  // below 2 M
    if (rem >= M) {
      rem -= M;
      q = 1;
    }
    n += full * (s.ctx / kPlanChunk);
    for (int r = 1; r <= period && r <= full; ++r) {  // tiles r, r + period, ...; q chunks of tile r
      q += a;
      rem += b;
      if (rem >= M) {
        rem -= M;
        ++q;
      }
      const int64_t m = whole + (r <= left);
      n += m * q + per * (m * (m - 1) / 2);
    }
  }
  if (t > full) n += (s.kv_total + kPlanChunk - 1) / kPlanChunk;  // the last, partly filled tile
  return n;
}

// A sliding window of WND keys with SNK sinks leaves out, behind the sinks' chunks, the chunks of tile t that end
// before its first row's window. (A tile's last row sees more than its first row's window skips: it keeps a chunk.)
KVH_PLAN_FN int pre_tile_skip(const PreSeq& s, int G, int PR, int WND, int SNK, int t) {
  int64_t lim = s.ctx + (int64_t)PR * t / G + 1;
  lim = lim < 0 ? 0 : (lim > s.kv_total ? s.kv_total : lim);
  const int64_t from = lim - WND, c = from / kPlanChunk - (SNK + kPlanChunk - 1) / kPlanChunk;
  return from > 0 && c > 0 ? (int)c : 0;
}

// The chunks that tiles 0 .. t - 1 leave out. With no clamped length tile i's are floor((A G + PR i) / (32 G)) where
// that is positive, A = ctx + 1 - WND - 32 ceil(SNK / 32): from the first tile i0 that leaves one out, the quotients of
// tiles a period apart (at most G tiles, as in pre_prefix) differ by a constant.
KVH_PLAN_FN int64_t pre_skips(const PreSeq& s, int G, int PR, int WND, int SNK, int t) {
  int64_t n = 0;
  if (s.ctx < 0 || s.ctx + s.q_len != s.kv_total) {
    for (int i = 0; i < t; ++i) n += pre_tile_skip(s, G, PR, WND, SNK, i);
    return n;
  }
  const int M = kPlanChunk * G;
  int64_t b = (s.ctx + 1 - WND - (int64_t)(SNK + kPlanChunk - 1) / kPlanChunk * kPlanChunk) * G;
  const int64_t i0 = b >= M ? 0 : (M - b + PR - 1) / PR;
  if (i0 >= t) return 0;
  b += PR * i0;
  const int tiles = t - (int)i0, g = pre_gcd(PR, M), period = M / g, per = PR / g;
  int64_t q = b / M;
  int rem = (int)(b % M);
  for (int r = 0; r < period && r < tiles; ++r) {  // tiles i0 + r, i0 + r + period, ...
    const int64_t m = (tiles - r + period - 1) / period;
    n += m * q + per * (m * (m - 1) / 2);
    q += PR / M;
    rem += PR % M;
    if (rem >= M) {
      rem -= M;
      ++q;
    }
  }
  return n;
}

// Whether the units of a windowed launch take whole tiles, each those whose middle (its first position + half of its
// positions) lies in the unit's range, instead of splitting tiles where ranges meet. A split tile's pieces are written in
// fp32 and read back by the merge, as long as kSplitCost chunk steps where all units hold pieces.
//  * Tiles alike, a full one's positions each (where its rows see a whole window): whole ones leave the last of a unit's
//    rounds part empty. Us split and whole, by the steps left empty (32 heads over 8 of 128, bf16; prompt and window): 2
//    (3000, 512) 76 and 57, 13 (12000, 1024) 260 and 238, 22 (8191, 1024) 194 and 182, 32 (4096, 1024) 108.9 and 110.4, 48
//    (8191, 2048) 275 and 293. Chunks over 4000 tokens: 20 (400, 512) 42 and 31, 29 (512, 1024) 41 and 50; on a third of the
//    units: 21 (40, 512) 26 and 30.
//  * Prompts of up to a few windows, whose first tiles are shorter (the mean is below 3/4 of a full one): where ranges
//    meet a unit is left with a tile too many, and a launch of few tiles with one that outlasts the ranges; half a full tile,
//    or what it is longer than a range. Three row tiles a wave, us split and whole by these steps: 67 (4600, 4096) 218 and
//    240, (5000, 4096) 234 and 283, (8000, 4096) 417 and 445, 35 (2500, 2048) 92 and 102, three prompts of (2000, 2048) 147 and 171,
//    26 (1400, 1024) 58 and 64, 19 (2000, 1024) 71 and 68, eight of (1000, 1024) 115 and 106, 11 eight of (500, 512) 56 and 49. Over
//    ranges of 9/4 full tiles and more that evens out, between the two units of a CU too, where every split still costs:
//    2.4 three of (3500, 2048) 299 and 284, 2.6 four of (3000, 2048) 332 and 301, 3.9 four of (5000, 4096) 820 and 794, but two of
//    (8000, 4096) 803 and 832, 5.4 sixteen of (2000, 2048) 641 and 599; 2.0 three of (4000, 4096) 434 and 478.
constexpr int kSplitCost = 26;

constexpr int pre_full_tile(int G, int PR, int WND, int SNK) {
  return kTileCost + (int)(((int64_t)WND + (PR + G - 1) / G + kPlanChunk - 1) / kPlanChunk + 1 +
                           ((int64_t)SNK + kPlanChunk - 1) / kPlanChunk);
}

// x / y of non-negative numbers, in 32 bits where they fit.
KVH_PLAN_FN int64_t pre_div(int64_t x, int64_t y) {
  return ((uint64_t)x | (uint64_t)y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

// `per` positions of tiles alike for each of `units` of the launch's `all` units; C positions over them.
KVH_PLAN_FN bool pre_whole_rounds(int64_t per, int64_t units, int64_t all, int tile) {
  const int64_t left = per - pre_div(per, tile) * tile;
  return left == 0 || (tile - left) * all <= kSplitCost * units;
}
KVH_PLAN_FN bool pre_whole_tiles(int64_t C, int64_t units, int64_t all, int tile) {
  return pre_whole_rounds(pre_div(C, units), units, all, tile);
}

// C positions of any `tiles` tiles. (Rounds that a range passes by a part of a position leave some units a tile more: the
// positions of a unit are rounded up.)
KVH_PLAN_FN bool pre_whole_tiles(int64_t C, int64_t tiles, int64_t units, int64_t all, int tile) {
  const int64_t per = pre_div(C + units - 1, units);
  if (4 * C >= 3 * tiles * tile) return pre_whole_rounds(per, units, all, tile);
  if (4 * C >= 9 * units * tile) return true;
  return (2 * per < tile ? tile - per : tile / 2) * all <= kSplitCost * units;
}

// What a unit of positions x .. x1 - 1 (x: where it stands in the tile, or before it) does with a tile of tw positions from
// beg on, where units take whole ones: nothing, as the unit before took it; take it; or end, as the next one does.
enum PreTurn { kPreSkip, kPreTake, kPreEnd };
KVH_PLAN_FN PreTurn pre_tile_turn(int64_t beg, int64_t tw, int64_t x, int64_t x1) {
  const int64_t mid = beg + tw / 2;
  return mid >= x1 ? kPreEnd : (mid >= x ? kPreTake : kPreSkip);
}

// 16-row tiles a wave takes under a window, 3 or 2, for `rows` query rows per kv head in `seqs` sequences: the cheaper by
// the above, with steps of 40 and 31 (a long prompt, window 4096: 936 us and 1060). Tiles of 2 fill a launch better that
// has few, or whose last round is part empty: (2000, 512) 49 us and 41, (4096, 1024) 109 and 94.5, chunks of 1000 and 900
// tokens over thousands, window 2048, 107 and 89, of 200 tokens, window 1024, 41 and 37; but (3000, 512) 57 and 63,
// (12000, 1024) 238 and 256. The contexts are not known on the host, so every tile counts as full; with the true lengths in
// their place the rule chose no better over 64 prompts and chunks of up to a few windows, 0.7% behind the faster number in
// the mean either way, furthest with four prompts of (1000, 1024), 68 us and 80.
inline int64_t pre_window_cost(int nt, int64_t rows, int64_t seqs, int Hkv, int G, int WND, int SNK, int64_t units) {
  const int64_t PR = 64 * nt, step = nt == 3 ? 40 : 31;
  const int64_t tiles = Hkv * ((rows + PR - 1) / PR + (seqs > 1 ? (seqs - 1) / 2 : 0));
  const int64_t tile = pre_full_tile(G, (int)PR, WND, SNK);
  const int64_t whole = (tiles + units - 1) / units * tile * step;
  const int64_t used = tiles * tile / 2 < units ? tiles * tile / 2 : units;
  const int64_t split = tiles * tile * step / units + kSplitCost * (nt == 3 ? 40 : 27) * used / units;  // (the pieces' rows)
  return whole < split ? whole : split;
}

inline int pre_window_nt(int64_t rows, int64_t seqs, int Hkv, int G, int WND, int SNK, int64_t units) {
  return pre_window_cost(2, rows, seqs, Hkv, G, WND, SNK, units) < pre_window_cost(3, rows, seqs, Hkv, G, WND, SNK, units)
             ? 2 : 3;
}

}  // namespace kvh
