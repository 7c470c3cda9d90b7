// How a product with a 4-bit weight is cut (linear4.hip): plain functions of its shape, also compiled for the host by the
// test that holds them to their limits.
#pragma once
#include <stdint.h>

namespace kvh {

constexpr int kW4Block = 128;  // k of a packed block

// A workgroup multiplies `rows` rows of x with wr groups of rt weight tiles; wk waves share a group's k, each s blocks of
// every chunk of wk s blocks; `splits` workgroups share the chunks.
struct Linear4Form {
  int rows, rt, wr, wk, s;
  int splits;
};

constexpr int linear4_chunk(const Linear4Form& f) { return f.wk * f.s; }
// Whether the waves that read the same x take turns at its groups' sums, four of them a group of weight rows (gated 64;
// 28672 x 4096: 33.5 us, so 30.7; two of them 8.6, 8.9 at (24; 16384 x 2048))
constexpr bool linear4_shares(const Linear4Form& f) { return f.wr >= 4 && f.rows > 16; }
constexpr int linear4_x(const Linear4Form& f) { return 2 * f.wk * f.s * f.rows * 2 * kW4Block; }
// LDS of a workgroup: two chunks of x with its sums over up to four groups a block, or the waves' sums
constexpr int linear4_lds(const Linear4Form& f) {
  const int x = linear4_x(f) + (linear4_shares(f) ? 2 * f.wk * f.s * 4 * f.rows * 4 : 0);
  const int sums = f.wr * f.wk * f.rt * ((f.rows + 15) / 16) * 1024;
  return x > sums ? x : sums;
}

// Times in us of (m rows of x; rows x columns of the weight), bf16, groups of 128, weights not in the caches; g: gated.
//  * Up to 16 rows of x: one tile a group as long as the tiles fit the CUs once ((1; 4096 x 4096) 5.2, with two tiles a wave
//    6.4), in sixteen slices of a long k ((8; 4096 x 14336) 10.9, in eight 11.8); two tiles behind that ((16; 6144 x 4096)
//    7.1, one 10.5), as long as they fit the CUs once ((16; 8192 x 4096) 7.2, two groups 8.6), then two groups, which share x
//    ((8; 8208 x 4096) 8.5, one group 11.2, (8; 9216 x 4096) 8.5 and 11.6, (8; 12288 x 4096) 8.7 and 11.9). From 1024
//    tiles on some CUs take two such workgroups and others one: four groups, one workgroup a CU, up to a full round of
//    them gated ((g 16; 16448 x 4096) 12.8, two groups 14.0, (g 8; 28736 x 4096) 14.1 and 15.1, (g 8; 32768 x 4096) 15.5 and
//    16.1), up to three quarters of one else, behind which the pairs are nearly even ((16; 16480 x 4096) 13.0 and 14.2,
//    (16; 20480 x 4096) 13.6 and 14.7, (1; 24576 x 2048) 8.6 and 9.1; but (1; 24576 x 4096) 14.4 and 13.9,
//    (8; 28672 x 4096) 15.9 and 14.8).
//  * More rows: workgroups of 32, 64, 128 or 256 weight rows, the fewest whose number fits the CUs once, in four slices of
//    k up to 64: (500; 2048 x 2048) 11.7 with 64, 16.0 with 128; (64; 12288 x 4096) 18.7, 22.1; (64; 6144 x 4096) 14.5 with
//    32, 15.3 with 64, 16.5 with 128. Each reads all of x: wider ones where that is more than 128 MB in all (at 128,
//    (64; 8192 x 4096), 16.1 with 32, 16.8 with 64), or 80 MB where they would be split besides ((250; 2048 x 8192) 21.1 with
//    128, 22.8 with 64; (48; 4096 x 8192) 14.8 with 64, 15.4 with 32). What they leave of the CUs is filled by splitting k,
//    four chunks at least each: (33; 2048 x 8192) 10.9 in four.
//  * Up to 32 rows eight slices in workgroups of 16 or 32 weight rows, as long as k is short ((20; 4096 x 4096) 8.1, 32 rows
//    8.9; (20; 6144 x 4096) 9.1, four slices 9.6).
//  * Where workgroups of 64 weight rows are too many, up to 48 rows of x take four tiles a wave in two groups for one round,
//    two in four groups for more ((g 32; 28672 x 4096) 19.6 and 21.4; (32; 128256 x 2048) 48.3 and 38.5).
//  * Past 64 rows of x the MFMAs and the codes' conversion bound it, which add up on this GPU: 256 weight rows and 64 of x
//    a workgroup where they fill it ((500; 6144 x 4096) 39.7, 128 rows 54.5; but (g 100; 16384 x 2048) 22.7 and 18.0).
inline Linear4Form linear4_form(int64_t tiles, int64_t blocks, int64_t m, bool glu) {
  if (m <= 16) {
    if (tiles <= 256 && !glu) {
      if (m > 8) return {16, 1, 1, 8, 2, 1};
      return blocks < 48 ? Linear4Form{8, 1, 1, 8, 2, 1} : Linear4Form{8, 1, 1, 16, 2, 1};
    }
    if (tiles <= 512 && !glu) return {16, 2, 1, 8, 2, 1};
    return tiles > 1024 && tiles <= (glu ? 2048 : 1536) ? Linear4Form{16, 2, 4, 4, 2, 1} : Linear4Form{16, 2, 2, 4, 2, 1};
  }
  if (m <= 32 && blocks < 48 && !glu) {
    if (tiles <= 256) return {32, 1, 1, 8, 1, 1};
    if (tiles < 512) return {32, 1, 2, 8, 1, 1};
  }
  const int rows = m <= 32 ? 32 : (m <= 48 ? 48 : 64);
  const int64_t mb = (m + 63) / 64;
  auto fits = [&](int64_t groups) {
    return groups <= 256 && groups * rows * blocks * 2 * kW4Block <= (groups > 128 ? 128 : 80) * (int64_t)(1 << 20);
  };
  Linear4Form f{rows, 2, 4, 2, 1, 1};
  if (!glu && fits((tiles + 1) / 2 * mb))
    f = {rows, 1, 2, 4, 1, 1};
  else if (fits((tiles + 3) / 4 * mb))
    f = {rows, 2, 2, 4, 1, 1};
  else if (m <= 48 && tiles > 1024 && tiles <= 2048)
    return {rows, 4, 2, 4, 1, 1};
  else if (m > 64 && (tiles + 15) / 16 * mb >= 150)
    return {64, 4, 4, 2, 1, 1};
  const int64_t groups = (tiles + f.rt * f.wr - 1) / (f.rt * f.wr) * mb, most = (blocks + f.wk - 1) / f.wk / 4;
  const int64_t z = 256 / groups < most ? 256 / groups : most;
  f.splits = z > 1 ? (int)z : 1;
  return f;
}

}  // namespace kvh
