// f8_choice.hpp - which kernel takes an 8-bit product, and in how many slices of K: a rule on sizes, the result's type and the chip, and nothing else (no
// HIP here: tests build it by itself and ask it).
#pragma once
#include <cstddef>
#include <cstdint>

namespace p0 {

enum F8Form {
  kF8TileSmall, kF8TileLow, kF8TileHalf, kF8TileLong, kF8TileWide,   // f8_tile_kernel, as kF8Shapes
  kF8Few32, kF8Few32w, kF8Few32x, kF8Few64,                          // f8_few_kernel past 16 rows, as kF8FewShapes
  kF8Few8, kF8Pairs4, kF8Pairs, kF8Few16b, kF8Few16,                 // up to 16
};
struct F8Choice {
  int form;     // -1: none takes as many outputs
  int slices;   // of K
};

// The rule past 16 rows: the form, and for a tile the slices of K (a power of two, as long as the slices' workgroups are no more than the CUs),
// with the least time by the figures below. The rule up to 16 rows is in f8_choice.
//
// Tiles: a round of workgroups takes its blocks of k, one after the other, and then its outputs; a slice's sums go through memory. The figures (us
// a block and a round) are fitted to 129 shapes of 17 to 4571 rows, 131 to 18216 outputs, 1 to 127 blocks, each tile and slicing measured on its
// own: the fastest by them is on average within 0.2% of the fastest measured, 5% at the worst (689 rows, 15753 outputs, 27 blocks, fp32: 97.8 for 93.1).
//   us, 16384 outputs x 2048 k   small   low   half   long   wide
//   64 rows, bf16                11.0    12.3  13.5   17.4   28.9
//   256 rows, bf16               36      22.1  17.1   21.3   33
//   1021 rows, bf16              137     89    55     45     37.8
//   1021 rows, fp32              199     134   91     75     -
//   slices (256 rows, 2048 outputs x 8192 k): low in 1 / 2 / 4 27.9 / 19.1 / 15.7, half in 8 21.3
constexpr int64_t kF8Groups = (1 << 23) - 1;   // workgroups of 512 threads: less than 2^32 threads
struct F8Shape {
  int bn, bm;
  float block, round;       // 16-bit results
  float block32, round32;   // fp32 results: half the matrix rate, conversions
};
constexpr F8Shape kF8Shapes[] = {{64, 64, 0.318f, 2.0f, 0.51f, 2.35f},     // kF8TileSmall
                                 {128, 64, 0.441f, 2.3f, 0.70f, 2.9f},     // kF8TileLow
                                 {128, 128, 0.613f, 2.65f, 0.97f, 3.6f},   // kF8TileHalf
                                 {128, 256, 1.032f, 3.9f, 1.50f, 6.0f},    // kF8TileLong
                                 {256, 256, 1.72f, 7.5f, 0.0f, 0.0f}};     // kF8TileWide: 16-bit results, no slices
// The kernel for few rows, ahead of the tiles, whose steps wait for each other, up to a few times as many workgroups as CUs: a round, then the longer of
// a wave's turns and of what a CU's workgroups ask for in all. Fitted to 255 shapes of 17 to 3330 rows; the choice among the first two and the tiles is
// on average within 1% of the fastest measured, 10% at the worst (512 rows, 1536 outputs x 1024 k). It is left out past 4 workgroups a CU (6 where results
// are fp32; 256 rows, 4096 x 2048: 32 x 32 9.4 us, tile 8.7), past one for 64 x 32 and 64 x 64 (1187 rows, 1541 x 9600: 51.6 in 64 x 64, tile 35.9), and,
// but for fp32, at weights past 64 MB, which stream better into tiles (64 rows, 9216 x 9216: 16 x 32 40, 32 x 32 32, tile 26; 17, fp32: 16 x 32 24, tile 34).
//   us: rows, outputs x k   16 x 32   32 x 32   64 x 32   64 x 64   tile
//   64, 2048 x 8192         7.2       8.4       -         -         11.5
//   64, 2048 x 2048         3.9       4.0       -         -         7.4
//   256, 512 x 2048         3.7       4.0       -         -         7.3
//   128, 4096 x 2048        9.9       5.7       -         -         8.7
//   1021, 2048 x 2048       36.6      16.6      -         -         11.1
//   256, 2048 x 8192        -         -         11.7      15.4      14.8
//   512, 2048 x 8192        -         -         20.8      17.3      21.1
//   the same, fp32          -         -         25.5      21.6      27.8
//   1021, 1024 x 4096       -         -         14.4      11.5      14.1
struct F8FewShape {
  int bn, bm, waves, per_cu;
  float round, turn, block, group;           // us: a round of workgroups, a turn of a wave, a block and a workgroup of each CU
  float round32, turn32, block32, group32;   // fp32 results
};
constexpr F8FewShape kF8FewShapes[] = {{16, 32, 8, 1, 0.41f, 0.486f, 0.060f, 0.09f, 0.53f, 0.62f, 0.05f, 0.0f},     // kF8Few32
                                       {32, 32, 8, 2, 0.0f, 0.60f, 0.085f, 0.41f, 0.0f, 0.665f, 0.10f, 0.55f},    // kF8Few32w
                                      {64, 32, 8, 1, 0.95f, 1.02f, 0.0f, 0.0f, 1.05f, 1.30f, 0.0f, 0.0f},        // kF8Few32x
                                      {64, 64, 8, 1, 3.0f, 1.45f, 0.0f, 0.0f, 3.5f, 1.94f, 0.0f, 0.0f}};         // kF8Few64
// M, N, blocks of 128 k; f32: fp32 results
inline F8Choice f8_choice(int64_t M, int64_t N, int blocks, bool f32, int cus, size_t part_floats) {
  if (M <= 16) {
    // Measured (us; rows, outputs x k). Up to 8 rows, pairs of 8 waves / of 4 / 16 outputs: 5, 2048 x 8192 5.1 / 5.6 / 7.3; 1, 9216 x 2048 6.9 / 6.0 / 5.5,
    // x 4096 10.2 / 9.1 / 10.2, x 8192 14.9 / 15.8 / 16.4; 1, 16384 x 2048 11.3 / 8.4 / 7.7, x 4096 15.5 / 12.7 / 14.8. Up to 16, 8 waves / 4: 16, 2048 x 8192
    // 6.0 / 7.6; 16, 9216 x 14720 33.3 / 33.8; 16, 16384 x 2048 9.2 / 8.1. Up to 16 blocks both are alike where there are few outputs
    const bool many = N > 18 * cus;   // workgroups of 8 outputs: more than two a CU
    if (M > 8) return {blocks <= 16 ? kF8Few16b : kF8Few16, 1};
    if (blocks <= 16) return {kF8Few8, 1};
    return {many && (blocks < 64 || N > 1 << 25) ? kF8Pairs4 : kF8Pairs, 1};   // (8 waves of 2^26 outputs: 2^32 threads)
  }
  float least = 0.0f;
  F8Choice best{-1, 1};
  for (int k = 0; k < (f32 ? 4 : 5); ++k) {
    const F8Shape& c = kF8Shapes[k];
    const int64_t tiles = (N + c.bn - 1) / c.bn * ((M + c.bm - 1) / c.bm);
    for (int n = 1; n <= 16; n *= 2) {
      if (n > 1 && (k == 4 || blocks / n < 4 || tiles * n > cus || (size_t)tiles * n * c.bn * c.bm > part_floats)) break;
      const int64_t groups = tiles * n, rounds = (groups + cus - 1) / cus;
      if (groups > kF8Groups) break;
      const float fill = groups < cus ? (float)groups / cus : 1.0f, alone = f32 ? 0.8f : 0.7f;   // a chip that is not full runs a little faster
      const float t = rounds * ((blocks + n - 1) / n * (f32 ? c.block32 : c.block) * (alone + (1.0f - alone) * fill) + (f32 ? c.round32 : c.round)) +
                      (n > 1 ? 3.0f + (f32 ? 0.26f : 0.23f) * n * (c.bn * c.bm / 4096) : 0.0f);
      if (best.form < 0 || t < least) { least = t; best = {k, n}; }
    }
  }
  for (int k = 0; k < 4; ++k) {
    const F8FewShape& c = kF8FewShapes[k];
    const int64_t groups = (N + c.bn - 1) / c.bn * ((M + c.bm - 1) / c.bm);
    if (groups > (k > 1 ? 1 : f32 ? 6 : 4) * cus || (!f32 && N * blocks > 1 << 19)) continue;
    const int rounds = (int)((groups + (int64_t)cus * c.per_cu - 1) / ((int64_t)cus * c.per_cu)), turns = (blocks + c.waves - 1) / c.waves;
    const float each = groups > cus ? (float)groups / cus : 1.0f, wait = rounds * turns * (f32 ? c.turn32 : c.turn),
                ask = each * blocks * (f32 ? c.block32 : c.block);
    const float t = rounds * (f32 ? c.round32 : c.round) + (wait > ask ? wait : ask) + each * (f32 ? c.group32 : c.group);
    if (best.form < 0 || t < least) { least = t; best = {kF8Few32 + k, 1}; }
  }
  if (best.slices > 1) {   // as many as have blocks
    const int each = (blocks + best.slices - 1) / best.slices;
    best.slices = (blocks + each - 1) / each;
  }
  return best;
}

}  // namespace p0
