// Which kernel, and which of its forms, a product with expert matrices takes
// and how expert choices are sorted: rules on sizes and types alone, in plain
// C++ (the tests check with them that every form is run).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace tinyoai_rule {

// What the rules see of a product.
struct Sizes {
  bool bf16;     // the matrices; else MXFP4
  int planes;    // of a row's values: bf16 1, fp16 2, fp32 3; 0: MXFP4 rows
  bool gate;     // (gate, up) pairs
  bool grouped;  // by offsets; else all rows with the one matrix
  int64_t experts, n, rows, cols;
};

inline int64_t groups(const Sizes &s) { return s.grouped ? std::min(s.experts, s.n) : 1; }
inline int64_t chunk_cols(const Sizes &s) { return s.bf16 ? 64 : 128; }
inline int64_t chunks(const Sizes &s) { return (s.cols + chunk_cols(s) - 1) / chunk_cols(s); }
inline int64_t stored_rows(const Sizes &s) { return ((s.rows + 15) / 16 * (s.gate ? 2 : 1) + 3) / 4 * 4 * 16; }

// ---------------------------------------------------------------- a few rows
constexpr int kMostChunks = 4;  // of a wave
// Whether the rows fill one or two column tiles (one, with sixteen waves), and
// the columns are no more than four chunks of sixteen waves (pairs and planes:
// of eight, or registers spill).
// 32 experts and more of large matrices: half of that on average. A group with more
// rows than the tiles hold is streamed again for each, by the few blocks that one
// expert has, so uneven groups cost much here, and little on the tiles of many rows.
// us, streamed and tiled, with 20 and with 32 operand columns a group (rows times
// planes), at random / of a popularity as 1 / i^1.5:
//   64 pairs of 1728 x 2560, MXFP4, fp32: 92 104 / 202 95, 100 112 / 319 115; bf16: 66 78 / 216 72,
//     93 81 / 345 95; MXFP4 rows: 54 54 / 120 51, 77 56 / 177 67;
//   128 of 512 x 512, MXFP4, fp32: 36 25 / 160 22, 42 26 / 256 27; BF16, bf16: 29 25 / 156 33, 46 27 / 241 36;
//   16 of 2560 x 1728, MXFP4, bf16: 14 20 / 24 20, 23 20 / 34 20; 8 pairs of 1728 x 2560, fp32: 18 24 / 25 24,
//     27 25 / 29 25; small, 32 of 256 x 1024, fp32: 10 14 / 14 14, 11 14 / 22 15.
inline bool few_rows(const Sizes &s) {
  const int waves = s.gate && s.planes ? 8 : 16;
  const bool large = groups(s) >= 32 && groups(s) * stored_rows(s) * s.cols > 1 << 25;
  return chunks(s) <= waves * kMostChunks &&
         s.n * std::max(s.planes, 1) <= groups(s) * (chunks(s) > 8 * kMostChunks || large ? 16 : 32);
}
struct Few {
  int waves, column_tiles, wave_chunks;
};
inline Few few_form(const Sizes &s) {
  // one column tile for a dense product of few rows; groups are uneven
  const bool two = s.n * std::max(s.planes, 1) > (s.grouped ? 4 : 16) * groups(s);
  if (chunks(s) > 8 * 4) return {16, 1, 4};
  return {8, two ? 2 : 1, chunks(s) > 8 * 3 ? 4 : 3};
}

// ---------------------------------------------------------------- many rows
// A chain of sums on the matrix cores rounds at every 16 columns of each plane
// (MXFP4 rows: 64), and its error grows with the root of its length: relative to
// float64, in the norm, fp32 rows times MXFP4 4.5e-7 at 2560 columns, 1.2e-6
// at 16384, 2.3e-6 at 65536. Long rows (chain_cols) go to totals a run of
// columns at a time: 2.8, 3.1 and 3.4e-7. Totals take as many registers as the
// sums, which costs the short rows 1 to 6%, and 21% where it leaves a CU fewer blocks
// (64 experts' pairs of MXFP4, bf16 rows).
constexpr int kRunBf16 = 1024, kRunMx = 8192;
// Columns of one chain, at most: for fp32 rows what keeps the error near that of
// fp32 sums of 512 columns (5e-7); bf16 rows' inputs are rounded to eight bits already.
constexpr int chain_cols(int planes) { return planes == 0 ? 65536 : planes == 1 ? 16384 : 8192 / planes; }
// Past these the totals' own chain counts: the smallest tiles, whose totals are doubles.
constexpr int kFloatTotals = 1 << 18;

// A weight's product whose smallest tiles leave half of the CUs without a block
// is cut over the columns, into parts of 8 steps at least, for a block a CU; the
// parts' sums are added by a launch of their own, which a short K does not repay
// (whole and in parts: fp32 rows, 128 x 1000, K = 4096, 33 and 17.6 us; 12 x 4096,
// K = 6912, 46 and 16; 48 x 2560, K = 2560, 22 and 16; 64 x 1024, K = 1024, 12.5
// and 12.7; MXFP4 rows, 100 x 500, K = 6912, 19 and 13.5; 400 x 1024, K = 2560,
// 11.3 and 13.1). The sums take 4 MiB at most.
inline int parts(const Sizes &s, int cus) {
  const int64_t step = s.planes ? 64 : 128, steps = (s.cols + step - 1) / step;
  if (s.grouped || s.gate || steps < 32) return 1;
  const int64_t blocks = (s.n + 31) / 32 * ((stored_rows(s) + 127) / 128);
  return (int)std::max<int64_t>(1, std::min<int64_t>(cus / blocks, steps / 8));
}

struct Tile {
  int bm, bn;
  bool runs;  // totals of runs
};
// The largest tiles that give most CUs a block, and of groups no taller than
// their rows need (BM x BN, measured at K = 2560; "rows" of each group on
// average):
//   6912 outputs, MXFP4 rows: 64 rows 8.1 us with 32 x 128, 12.3 with 64 x
//   256; 256 rows 10.3 with 64 x 128, 11.7 and 12.9; 1024 rows 19.5 with 64 x
//   256, 24.7 with 64 x 128; fp32 rows 25 and 47, 39 and 52, 98 and 112;
//   64 pairs of 1728: fp32, 16 rows: 124 with 32 x 128, 152 with 64 x 256,
//   64 rows: 270 and 248; MXFP4, 64 rows: 79 with 64 x 256, 78 with 128 x 256,
//   256 rows: 181 and 163;
//   BF16, 32 pairs: 32 rows 110 with 64 x 256, 113 with 128 x 256, 128 rows: 180
//   and 151.
// BF16 matrices and rows, 256 x 256 against 128 x 256: one block of either fills
// a CU, and the larger one takes 0.87 of the smaller's time for a product, so it
// is taken where its rounds of blocks are no more than half as many (groups have
// half a tile more on average). us, experts x rows of each:
//   rounds 1 and 2: 8 x 512 of 2560 x 1728, 49 and 57; 8 x 256 of 3584 x 4096, 89 and 102;
//     one of 4096, 4096 x 4096, 118 and 130; 4 and 8: 8 x 2048 of 3584 x 2560, 284 and 318;
//   rounds 2 and 3: 8 x 1024 of 2560 x 1728, 96 and 92; 8 x 400 of 5120 x 2560, 124 and 113;
//     2 and 2: 8 x 512 of 3584 x 2560, 123 and 90; 1 and 1: 4 x 1024 of 1792 x 4096, 84 and 64.
inline Tile tile(const Sizes &s, int ks, int cus) {
  const int64_t g = groups(s), rows = s.n / g, stored = stored_rows(s);
  auto fills = [&](int bm, int bn) { return g * ((rows + bm - 1) / bm) * ((stored + bn - 1) / bn) * 4 >= cus * 3; };
  const bool low = s.grouped && s.planes > 1 && rows <= 24;  // (one plane: the matrix's loads count for more)
  const int64_t chain = chain_cols(s.planes);
  if (s.cols <= kFloatTotals && !low && (fills(64, 256) || fills(64, 128))) {
    const bool runs = s.cols > chain;
    if (!runs) {  // (no registers for totals)
      auto rounds = [&](int bm) {
        const double tiles = g == 1 ? (double)((rows + bm - 1) / bm) : (double)rows / bm + 0.5;
        return std::ceil(g * tiles * (double)((stored + 255) / 256) / cus);
      };
      if (s.bf16 && s.planes == 1 && rows >= 256 && 2 * rounds(256) <= rounds(128)) return {256, 256, false};
      if (s.planes == 0 && rows >= 128 && fills(128, 256)) return {128, 256, false};
    }
    if (s.bf16 && rows >= 96 && fills(128, 256)) return {128, 256, runs};
    return {64, fills(64, 256) ? 256 : 128, runs};
  }
  // (a wave has four chains of sums, two of MXFP4 rows)
  return {32, 128, s.cols / ks > chain * (s.planes ? 4 : 2)};
}

// ---------------------------------------------------------------- routing
constexpr int kFewSlots = 256, kFewTokens = 32, kSortSlots = 8192;
enum class Sort { one_block, by_expert, by_tokens };
inline Sort sort_path(int64_t n, int64_t k) {
  return n <= kFewTokens && n * k <= kFewSlots ? Sort::one_block : n * k <= kSortSlots ? Sort::by_expert : Sort::by_tokens;
}
// Experts of a lane.
inline int lane_experts(int experts) { return experts <= 64 ? 1 : experts <= 128 ? 2 : experts <= 256 ? 4 : experts <= 512 ? 8 : 16; }

}  // namespace tinyoai_rule
