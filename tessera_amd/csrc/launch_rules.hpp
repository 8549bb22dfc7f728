// Rules that choose a launch's shape from a call's sizes.  Host logic only; no HIP calls.  (A constexpr function is
// device code's as well.)
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace qmm {

// ---- MXFP4, 17 fp32 rows and more: tiles whose steps of K workgroups share --------------------------------------
// Tiles of `rows` x `columns`, `tiles` of them; the (tile, step) units go to `groups` workgroups.  groups 0: not shared.
struct SharedTiles {
  uint32_t rows = 0, tiles = 0, groups = 0, columns = 256;
};
// First of the units of workgroup g.
constexpr uint64_t unit_bound(uint32_t g, uint32_t groups, uint32_t tiles, uint32_t steps) {
  return static_cast<uint64_t>(g) * (static_cast<uint64_t>(tiles) * steps) / groups;
}
// The workgroup that holds unit v: the last whose bound is not above it.
constexpr uint32_t unit_owner(uint64_t v, const SharedTiles& plan, uint32_t steps) {
  uint32_t g = static_cast<uint32_t>(v * plan.groups / (static_cast<uint64_t>(plan.tiles) * steps));
  while (g + 1u < plan.groups && unit_bound(g + 1u, plan.groups, plan.tiles, steps) <= v) ++g;
  return g;
}
// The piece of tile t that workgroup g holds is block g + t: along the units one of the two grows from piece to piece.
constexpr size_t shared_tiles_bytes(const SharedTiles& plan) {
  return plan.groups == 0u ? 0 : (static_cast<size_t>(plan.groups) + plan.tiles - 1u) * plan.rows * plan.columns * 4u;
}
// Rows a tile: the padding it takes decides.  Workgroups: as many as the chip holds, at least four units each.
// Tiles are shared where whole ones, small (128 x 64) or 256 x 256, leave much of the chip idle for long.  Sides measured
// (us, whole / shared): 17 rows of 6144 x 5120 57 / 42, 100 rows 69 / 54, 453 rows of 17408 x 5120 238 / 190, 1024 of 5120 x
// 17408 591 / 349, 640 of 4096 x 2048 55 / 48; but 2048 of 6144 x 5120 (192 tiles) 254 / 262, 1500 of 4000 x 1792 (14 steps)
// 73 / 83, 20 of 520 x 1024 19 / 21: the pieces cost a launch and twice their bytes, 64 MB of 256-row tiles where the chip
// is full of them.  With few steps that is more than small tiles lose which fill a round of a workgroup a CU, or of two:
// 256 rows of 2048 x 2048 34 / 45, 128 of 8192 x 2048 (128 small tiles) 33 / 38, but of 1024 x 2048 (16) 33 / 32, 512 of 8192
// x 2048 (512) 58 / 60, 512 of 4096 x 4096 (32 steps, 256 small tiles) 61 / 66, but 256 (128) 59 / 53.
constexpr SharedTiles shared_tiles(uint64_t m, uint64_t n, uint64_t steps, uint64_t cus) {
  if (m > 256 * cus || n > 256 * cus || steps < 16) return {};
  const uint64_t rows = m <= 64 ? 64 : (m + 127) / 128 * 128 < (m + 255) / 256 * 256 ? 128 : 256;
  const uint64_t tiles = (m + rows - 1) / rows * ((n + 255) / 256), small = (m + 127) / 128 * ((n + 63) / 64);
  if (tiles * 8 > cus * 5) return {};
  if (steps < 32 && rows == 128 && small <= cus && small * 8 > cus) return {};
  if (steps < 32 && rows == 256 && small <= 2 * cus) return {};
  if (steps < 40 && small * 8 >= cus * 7 && small <= cus) return {};
  const uint64_t room = cus * (rows == 64 ? 2 : 1), most = tiles * steps / 4;
  return {static_cast<uint32_t>(rows), static_cast<uint32_t>(tiles), static_cast<uint32_t>(room < most ? room : most)};
}

// ---- Q4_K, Q5_K and Q6_K on the tensor tile: tiles whose super-blocks workgroups share -----------------------------------
// Tiles of 128 x 128 whose (tile, super-block) units go to one workgroup a CU, at least two units each.  Whole tiles of
// 128 x 64 leave most CUs idle while a few walk all of K: 512 rows of 1024 x 5120 are 64 of them.  The pieces cost a launch
// and twice their bytes, so that with few super-blocks, or tiles that fill the chip, whole ones lead; `small` counts those, and
// the limits are sixteenths of the CUs.
// Q4_K, sides measured (us, whole / shared; rows x n x k, in brackets the small tiles).  `even`: every workgroup has as many
// units; otherwise some take two tiles' pieces, which counts where a tile has few; with several row tiles sharing leads
// all the same (500 x 1728 x 3072 (108) 30.6 / 28.9, 1000 x 1728 x 4096 (216) 40.8 / 39.1).  100 x 4096 x 2048 (64) 20.9 / 19.5, x 2304 22.6 /
// 23.6, x 2816 25.7 / 25.3; 100 x 5696 x 3072 (89) 27.4 / 27.6, x 6912 (108) 27.5 / 29.2, x 8192 (128, even) 27.4 / 26.3; 128 x 13888 x
// 4352 (217) 37 / 40, 256 x 8192 x 4096 (256, even) 38 / 36; 512 x 1024 x 5120 (64) 44 / 26, 512 x 6144 x 5120 (384) 64 / 59, 2048 x
// 6144 x 5120 (1536) 183 / 220; 256 x 5120 x 17408 (160) 126 / 84, 1024 (640) 316 / 267, 2048 (1280) 452 / 492.  Four row tiles and
// more whose small tiles fill two a CU: 500 x 7168 x 6144 (448) 76 / 82, but 256 x 14336 (448) 76 / 72, 500 x 8704 (544) 115 / 87.
// Up to 64 rows whole tiles are of 32 columns and 32 or 64 rows, with no padding, and start to take longer with more than a round of
// them: 17 rows of 2048 x 2048 (32) 14.6 / 15.1, 5120 x 3072 (80) 18.9 / 17.9, 6144 x 3072 (96) 18.9 / 20.7, 8192 x 5120 (128) 27.8 / 23.7,
// 10240 x 5120 (160) 29 / 30, 17408 x 5120 (272) 29.5 / 40, 12288 x 8192 (192) 43 / 41, 5120 x 17408 (80) 82 / 40; 64 rows of 4096 x
// 2048 (64) 18.7 / 16.8, 6144 x 3072 (96) 24.7 / 23.3, 7168 x 3072 (112) 24.8 / 25.5, 12288 x 4096 (192) 32 / 30.5, 14336 x 4096 (224) 32.4 /
// 32.7, 16384 x 5120 (256) 38 / 36, 20480 x 5120 (320) 39 / 46.
constexpr uint64_t shared_q4k_limit(uint64_t m, uint64_t steps, bool even) {
  if (m <= 32) return steps < 10 ? 0 : steps < 12 ? 2 : steps < 16 ? 4 : steps < 18 ? 6 : steps < 24 ? 8 : steps < 32 ? 10 : steps < 48 ? 12 : 14;
  if (steps < 12) return steps == 9 ? 3 : 4;
  if (m <= 64) return steps < 16 ? 6 : steps < 20 ? 12 : 16;
  if (steps < 16) return steps == 12 && m <= 256 && !even ? 5 : 8;
  return steps < 18 && m <= 384 && !even ? 12 : steps < 20 ? 16 : 40;
}
// Q5_K and Q6_K, whose whole tiles need no decode and go up to 256 x 256: 100 x 512 x 2048 (8) 22 / 19, 24 x 6144 x 2048 (96) 28 /
// 33; 200 x 2048 x 3072 (64) 33 / 28, 24 x 4096 x 3072 (64) 32 / 33, 384 x 4096 x 3072 (192) 36 / 38; 512 x 1024 x 5120 (64) 46 / 28,
// 512 x 6144 x 5120 (384) 80 / 79, 200 x 6144 x 5120 (192) 57 / 59; 512 x 3072 x 8192 (192) 66 / 75.
constexpr uint64_t shared_kquant_limit(uint64_t m, uint64_t steps) {
  return (steps < 12 ? 2 : steps < 16 ? 4 : steps < 20 ? 6 : 8) / (m <= 32 && steps < 20 ? 2 : 1);
}
constexpr SharedTiles shared_f16_tiles(uint64_t m, uint64_t n, uint64_t steps, uint64_t cus, bool q4k) {
  if (m > 256 * cus || n > 256 * cus || steps < 8) return {};
  const uint64_t tiles = (m + 127) / 128 * ((n + 127) / 128), small = (m + 127) / 128 * ((n + 63) / 64);
  if (small * 16 > cus * (q4k ? shared_q4k_limit(m, steps, tiles * steps % cus == 0) : shared_kquant_limit(m, steps))) return {};
  if (q4k && m > 384 && steps < 48 && small * 2 > cus * 3 && small <= 2 * cus) return {};
  const uint64_t units = tiles * steps / 2;
  return {128, static_cast<uint32_t>(tiles), static_cast<uint32_t>(cus < units ? cus : units), 128};
}

// ---- "ffn_gate_up_silu_q4k", more than 64 rows ----------------------------------------------------------------------
// Tiles of 256 rows and 128 columns of either matrix, from column 0 on; what they leave goes to tiles of 128 rows and 64.
// As in the single product, whole rounds of a tile a CU, and none where they fill less than half the chip.  Nor with 128
// rows or fewer, half of each tile being padding (us, small tiles / 256-row tiles, in brackets as two products: 17408 x 5120
// 103 / 138 (117)), nor with 257 to 384, half of the second ones, unless they fill three quarters of a round or all of it: 300
// rows of 17408 x 5120 (136 tiles) 209 / 233 (287), of 8192 x 4096 (64) 88 / 113 (107), of 12288 x 2048 (192) 74 / 70.
constexpr uint32_t gate_up_large_tiles(uint32_t m, uint32_t n, uint32_t cus) {
  const uint32_t tiles_m = (m + 255u) / 256u, tiles_n = (n + 127u) / 128u, tiles = tiles_m * tiles_n;
  if (m <= 128u || (m > 256u && m <= 384u && (tiles * 4u < cus * 3u || tiles > cus))) return 0;
  if (tiles > cus && tiles % cus != 0 && tiles % cus <= cus / 2) return tiles / cus * cus / tiles_m;
  return tiles < cus / 2 ? 0 : tiles_n;
}

// ---- Q5_K and Q6_K from 17 rows: both operands to fp16 -------------------------------------------------------------------
// RowsFirst: one launch, the rows' workgroups first.  RowsLast: the weights' first, so that the product finds the rows' copy where
// it was left last.  RowsTwice: rows first and read twice, since a row of more than 6144 held in registers leaves five wavefronts a
// SIMD also to the weights, where Q5_K's decode wants eight.  Apart: the weights, then the rows in a launch of their own.
// Sides measured in a whole feed forward of Q4_K gate and up with silu and this product (us, rows x hidden x inter).  Q6_K, first /
// last: 256 x 5120 x 17408 373 / 382 (the product alone, called again and again, 168 / 219), 512 534 / 536, 1024 812 / 783,
// 2048 x 4096 x 11008 708 / 672; but 2048 x 5120 x 6400 528 / 542, 1024 x 4096 x 8192 282 / 284, and the product of 2048 x 5120 x 5120
// 135 / 138.  Q5_K, first / twice / apart: 100 x 5120 x 17408 244 / 232 / 235, 256 375 / 380 (the product 168 / 213), 384 464 / 453 (186 /
// 230), 1024 838 / 834 / 799, 2048 x 4096 x 11008 716 / 725 / 685, 2048 x 5120 x 6400 537 / 542 / 548; the product of 33 x 24576 x 17408
// 693 / 638 / 638, of 512 x 24576 x 8192 409 / 381 / 378, of 33 x 512 x 12288 31.0 / 31.7 / 34.1: twice where the weights are most of it.
enum class KquantOperands { RowsFirst, RowsLast, RowsTwice, Apart };
constexpr KquantOperands kquant_operands(uint32_t m, uint32_t n, uint32_t k, uint32_t bits) {
  if (k <= 6144u || (bits == 6u && (m <= 512u || k <= 8192u))) return KquantOperands::RowsFirst;
  if (bits == 6u) return KquantOperands::RowsLast;
  if (m > 512u && k >= 8192u) return KquantOperands::Apart;
  return n >= uint64_t{24} * m ? KquantOperands::RowsTwice : KquantOperands::RowsFirst;
}

// ---- Q5_K and Q6_K from 17 rows: fp16 weights, decoded by the launch before ----------------------------------------------
// `large` tiles of 256 rows and `columns` columns, from column 0 on, for each 256 rows; the columns they leave go to tiles of
// 128 x 64.  Whole rounds of 256 columns, a tile a CU, and none where they fill less than half the chip.  Where the columns
// fit one round of narrower ones, the narrowest with which they still do: 2048 x 5120 as 216 tiles of 192 columns instead of
// 160 of 256 (515 -> 455 us at K = 17408).  But not with 64 rows or fewer, nor with 128 and a short K, which leave three
// quarters or half of those tiles empty (us, small tiles / 256 x 128): 64 rows of 24576 x 1024 30 / 39, of 32000 x 2048 58 / 68,
// 128 rows 34 / 40, 64 / 69; of 17408 x 5120 and 20000 x 5120 64 rows 97 / 95, 132 / 131, 128 rows 114 / 104, 143 / 135.
struct F16wTiles {
  uint32_t large, columns;
};
constexpr F16wTiles f16w_tiles(uint32_t m, uint32_t n, uint32_t k, uint32_t cus) {
  const uint32_t tiles_m = (m + 255u) / 256u;
  if (m > 128u || (m > 64u && k >= 4096u)) {
    for (uint32_t columns : {128u, 192u}) {
      const uint32_t tiles_n = (n + columns - 1u) / columns;
      if (tiles_m * tiles_n <= cus && tiles_m * tiles_n > cus / 2) return {tiles_n, columns};
    }
  }
  const uint32_t tiles_n = (n + 255u) / 256u, tiles = tiles_m * tiles_n;
  if (tiles > cus && tiles % cus != 0 && tiles % cus <= cus / 2) return {tiles / cus * cus / tiles_m, 256u};
  return {tiles < cus / 2 ? 0u : tiles_n, 256u};
}
// The order of the tiles.  Workgroups go round the XCDs, in the launch that decodes as here, so that along the columns an XCD
// finds part of the weights that it has written itself in its L2 (also with the rows' workgroups before the weights', whose count
// is the shift: 100, 101 and 103 rows of 16384 x 1024 25 us each, shares 32); an XCD's share of neighbouring tiles (xcd_tile) instead
// reads them once for several row tiles.  The first leads with one row tile, with up to three where the weights are small, and
// where small tiles are few (us, along / shares): 100 rows of 16384 x 1024 27 / 33, 256 rows 33 / 39, 300 of 6144 x 5120 70 /
// 84, 512 of 5120 x 17408 (320 small tiles) 286 / 324, 700 of 3072 x 1024 (288) 24 / 29; 256 rows of 17408 x 5120 161 / 151, of
// 12288 x 4096 (384) 78 / 76, 512 of 6144 x 5120 (384) 84 / 80.
constexpr bool f16w_tiles_as_decoded(uint32_t m, uint32_t n, uint32_t k, uint32_t cus, bool small) {
  return m <= 128u || (m <= 384u && static_cast<uint64_t>(n) * k <= (uint64_t{32} << 20)) ||
         (small && static_cast<uint64_t>((m + 127u) / 128u) * ((n + 63u) / 64u) * 4u <= cus * 5u);
}

// ---- "rope", "mrope" -------------------------------------------------------------------------------------------------
// Heads that share a thread's angle: eight from a wavefront a SIMD on (512 rows of 24 heads of 256 23 -> 7.5 us), of one head
// none, which would be read eight times (8193 rows of 64 5.7 / 6.2 us).
constexpr uint32_t rope_heads_a_thread(uint64_t rows, uint64_t heads, uint64_t pairs) {
  return heads > 1 && rows * heads * pairs >= 65536 ? 8 : 1;
}

// ---- "quantize_fp8_pack" ---------------------------------------------------------------------------------------------
// Workgroups of a row while the rows alone cannot fill the chip, at most sixteen, each finding the row's maximum for itself:
// of 256 threads one for 1024 columns, of 1024 one for 4096 where the row is long and there are many (us, 256 / 1024
// threads: 4 rows of 5120 3.3 / 3.5, of 8192 3.1 / 3.7, of 17408 3.6 / 4.0; 64 rows of 8192 3.6 / 4.0, 100 rows 4.5 / 4.1; 32
// of 17408 4.9 / 4.3, 200 rows 12 / 10).
struct PackShape {
  uint32_t per_row, threads;
};
constexpr PackShape pack_shape(uint64_t rows, uint64_t cols) {
  if (rows >= 256) return {1, 256};
  const uint32_t threads = cols <= 6144 || rows * cols <= (uint64_t{1} << 19) ? 256 : 1024;
  const uint64_t share = (cols + threads * 4 - 1) / (threads * 4);
  return {static_cast<uint32_t>(share < 16 ? share : 16), threads};
}

// ---- "attention" with many query rows -------------------------------------------------------------------------------
// How a call over an fp16 or a quantized cache runs: 0, the rows' kernel, a workgroup for up to eight heads of a row and
// key head; else the kernel that shares 64 keys at a time among 64 (row, head) pairs, in so many parts of the keys.  `keys`:
// how many a row sees at most; `padded`: the head size, 64, 128 or 256.
//
// The shorter of the estimated times, in us: a fixed part, then for the rows' kernel what a round of a workgroup a CU takes
// by its keys (four wavefronts up to 160 keys, eight beyond; where five take 129 to 160 keys they are up to a tenth faster than
// the estimate, and of 306 such calls none takes the longer way by more than 3 %), for the other what 64 keys take, and for its parts the
// second launch and the sums' way through memory.  Fitted to 1716 calls (17 to 512 rows, 17 to 2512 keys, 2 to 32 heads over
// 1 to 8 key heads of 64, 96, 128 and 256, fp16 and int8), which they meet within 4 % on average: one call of them
// takes the longer way by more than 5 %.  Rows' kernel / one part / parts: 64 rows of 24 heads over 4 of 256 on 564 keys 21 / 34 /
// 29, on 2064 48 / 95 / 42; 512 rows of 16 over 4 of 64 on 512 27 / 14 / 39; 64 of 8 over 8 of 128 on 64 7 / 10; 300 of 24
// over 4 of 256 on 2300 285 / 105.
struct AttentionCall {
  uint64_t rows, keys, heads, kv_heads, head_dim, padded;
  bool quantized;
};
constexpr uint64_t attention_pairs64(const AttentionCall& a) { return (a.rows * (a.heads / a.kv_heads) + 63) / 64 * a.kv_heads; }
// Bytes of `parts` parts: a sum of head_dim, the largest score and the sum of weights for each.
constexpr size_t attention_parts_size(uint64_t rows, uint64_t heads, uint64_t head_dim, uint64_t parts) {
  return parts < 2 ? 0 : static_cast<size_t>(rows * heads * parts * (head_dim + 2) * 4);
}
constexpr uint64_t attention_rule(const AttentionCall& a, uint64_t cus, uint64_t most_parts, size_t most_bytes) {
  const uint64_t units = attention_pairs64(a), tiles = (a.keys + 63) / 64;
  const uint64_t row_units = a.rows * a.kv_heads * ((a.heads / a.kv_heads + 7) / 8);
  uint64_t parts = cus / units < a.keys / 256 ? cus / units : a.keys / 256;
  if (parts > most_parts) parts = most_parts;
  while (parts > 1 && attention_parts_size(a.rows, a.heads, a.head_dim, parts) > most_bytes) --parts;

  const int size = a.padded == 64 ? 0 : a.padded == 128 ? 1 : 2;
  constexpr double kRowFixed[2][3] = {{5.2, 5.5, 5.3}, {5.3, 4.1, 5.3}}, kRowRound[2][3] = {{0.3, 0.65, 3.4}, {0.5, 3.1, 3.4}};
  constexpr double kRowKey[2][3] = {{0.0047, 0.0102, 0.0194}, {0.005, 0.0083, 0.0194}};
  constexpr double kTileFixed[3] = {6.1, 8.1, 12.8}, kTile[3] = {1.0, 1.32, 2.31}, kPartsMegabyte[3] = {1.07, 0.85, 0.79};
  constexpr double kPartsFixed = 2.5;
  const int wide = a.keys > 160 ? 1 : 0;
  const uint64_t row_rounds = (row_units + cus - 1) / cus, rounds = (units + cus - 1) / cus;
  const double key_us = kRowKey[wide][size] * (a.quantized ? 1.12 : 1.0);
  const double row_us = kRowFixed[wide][size] + (a.quantized ? 0.6 : 0.0) +
                        static_cast<double>(row_rounds) * (kRowRound[wide][size] + key_us * static_cast<double>(a.keys));
  const double tile = kTile[size] * (a.quantized ? 1.25 : 1.0);
  const double one_us = kTileFixed[size] + tile * static_cast<double>(rounds * tiles);
  if (parts > 1) {
    const uint64_t part_tiles = ((a.keys + parts - 1) / parts + 63) / 64;
    const double parts_us = kTileFixed[size] + kPartsFixed + tile * static_cast<double>(part_tiles) +
                            kPartsMegabyte[size] * static_cast<double>(a.rows * a.heads * parts * a.head_dim * 4) * 1e-6;
    if (parts_us <= one_us && parts_us < 0.98 * row_us) return parts;
  }
  return one_us < 0.98 * row_us ? 1 : 0;
}

// ---- "attention_tree" ------------------------------------------------------------------------------------------------
// How a call runs: a workgroup a row and key head, at most eight heads (sixteen over fp32 keys); or sixteen (row, head) pairs of a
// key head, fp32 keys only; or 64 that share their keys, 64 at a time (`tile`); and the parts of the keys.  The shortest of the
// estimated times, in us: a fixed part, the rounds of workgroups that the chip holds, each with a part of its own and what its
// keys take, and for parts the second launch and the sums' way through memory.  Fitted to 600 calls run in 9348 ways (1 to 64
// rows, 1 to 30000 keys, 1 to 64 heads over 1 to 8 key heads of 64 to 256, all kinds of cache; profiles/tree_rule_times.csv): the
// way taken is 1.6 % over the fastest of them on average, 5 % in nine calls of ten, 35 % at most.  A workgroup a row and key head /
// shared keys, each in its best number of parts: 1 row of 48 heads over 8 of 128 on 18168 4-bit keys 15 / 22, 10 rows of 12 heads
// over 2 of 64 on 62 5.8 / 7.1, 13 rows of 6 over 2 of 256 on 13892 fp16 keys 46 / 22, 59 rows of 24 over 4 of 128 on 11138
// 113 / 32; a row's heads / sixteen pairs / shared keys, fp32: 7 rows of 6 heads over 2 of 64 on 8199 12 / 11 / 15, 24 of 8 over 2 of 256
// on 71 15 / 20 / 16, 64 of 24 over 4 of 256 on 8192 428 / 220 / 87.
struct TreeCall {
  uint64_t rows, keys, heads, kv_heads, head_dim, padded;   // keys: that a row sees at most; padded: the head size, 64, 128 or 256
  bool fp32, quantized;
  bool by_rows, shared;                                     // which ways the call can take
};
struct TreeShape {
  bool tile;                                                // by the kernel of shared keys
  uint64_t pairs, parts;                                    // (row, head) pairs a workgroup
};
constexpr uint64_t tree_units(const TreeCall& a, uint64_t pairs) {
  return (a.rows * (a.heads / a.kv_heads) + pairs - 1) / pairs * a.kv_heads;
}
constexpr TreeShape tree_rule(const TreeCall& a, uint64_t cus, uint64_t most_parts, size_t most_bytes) {
  // at_once: workgroups a CU; whole: a round takes its time however few it holds (one workgroup fills the CU), else what it holds
  struct Times {
    double fixed, round, keys, quantized, at_once, parts, megabyte;
    bool whole;
    double pair = 0.0;
  };
  constexpr Times kRows[3] = {{4.7, 0.48, 0.0056, 1.23, 0.81, 2.6, 3.0, false},
                              {3.5, 2.76, 0.0089, 1.04, 0.76, 2.6, 1.1, false},
                              {2.35, 6.2, 0.0196, 1.02, 1.0, 3.2, 1.96, true}};
  constexpr Times kRowsF32[3] = {{4.57, 0.55, 0.0128, 1.0, 0.84, 3.0, 1.44, false, 0.017},
                                 {4.76, 1.48, 0.0245, 1.0, 0.76, 3.13, 2.3, false, 0.039},
                                 {3.59, 4.86, 0.0519, 1.0, 0.8, 3.74, 2.35, false, 0.19}};
  constexpr Times kTiles[3] = {{4.85, 0.27, 0.706, 1.36, 2.0, 3.0, 1.77, true},
                               {3.42, 2.55, 0.93, 1.35, 1.0, 3.05, 1.08, true},
                               {2.3, 5.6, 1.41, 1.29, 1.0, 4.3, 0.89, true}};
  constexpr Times kTilesF32[3] = {{4.0, 0.71, 2.13, 1.0, 2.0, 3.16, 1.71, true},
                                  {5.4, 0.4, 3.02, 1.0, 1.0, 3.16, 1.17, true},
                                  {7.9, 0.0, 4.98, 1.0, 1.0, 4.1, 1.05, true}};
  const int size = a.padded == 64 ? 0 : a.padded == 128 ? 1 : 2;
  const uint64_t group = a.heads / a.kv_heads, fit = a.fp32 ? 16 : 8, own = group < fit ? group : fit;
  TreeShape best{false, own, 1};
  double least = -1.0;
  for (uint64_t pairs : {own, uint64_t{16}, uint64_t{64}}) {
    const bool tile = pairs == 64;
    if (tile ? !a.shared : !a.by_rows || (pairs != own && (!a.fp32 || a.rows * group <= own))) continue;
    const Times& t = tile ? (a.fp32 ? kTilesF32[size] : kTiles[size]) : a.fp32 ? kRowsF32[size] : kRows[size];
    const uint64_t units = tree_units(a, pairs);
    const double slots = static_cast<double>(cus) * t.at_once;
    const uint64_t fill = static_cast<uint64_t>(slots) / units;        // parts that fill the chip
    for (uint64_t parts : {uint64_t{1}, uint64_t{2}, uint64_t{3}, uint64_t{4}, uint64_t{6}, uint64_t{8}, uint64_t{12}, uint64_t{16},
                           uint64_t{24}, uint64_t{32}, uint64_t{48}, uint64_t{64}, fill}) {
      if (parts == 0 || (parts > 1 && (parts > most_parts || a.keys / parts < 48))) continue;
      if (parts > 1 && attention_parts_size(a.rows, a.heads, a.head_dim, parts) > most_bytes) continue;
      const uint64_t each = (a.keys + parts - 1) / parts, groups = units * parts;
      double rounds = static_cast<double>(groups) / slots;
      if (t.whole) rounds = static_cast<double>((groups + static_cast<uint64_t>(slots) - 1) / static_cast<uint64_t>(slots));
      const double walk = t.keys * (a.quantized ? t.quantized : 1.0) * static_cast<double>(tile ? (each + 63) / 64 : each);
      double us = t.fixed + (rounds < 1.0 ? 1.0 : rounds) * (t.round + t.pair * static_cast<double>(pairs) + walk);
      if (parts > 1) us += t.parts + t.megabyte * static_cast<double>(a.rows * a.heads * parts * a.head_dim * 4) * 1e-6;
      if (least < 0.0 || us < least) least = us, best = TreeShape{tile, pairs, parts};
    }
  }
  return best;
}

// ---- "token_logprobs" ------------------------------------------------------------------------------------------------
// Threads of a workgroup: as many as eight entries each make a short row, 1024 where there is much to read, otherwise 512, whose
// barriers are shorter (us, 256 / 512 / 1024 threads: 512 rows of 1000 6.7 / 7.3 / 10.2, 512 of 4000 13.1 / 10.1 / 14.7, one of
// 131072 10.5 / 9.7 / 10.7, 128 of 131072 28.4 / 27.0 / 24.9, 512 of them 75 / 70 / 58.5, 4.6 TB/s).
// Tiles of a row a workgroup takes: the shortest time in tiles, the chip's threads full, each workgroup with one tile's time of
// its own, the second launch with two (128 rows of 131072 as 1, 4, 16 tiles a workgroup: 34 / 25 / 36 us).  Rows are shared where the
// shares of all of them fit `most` bytes and one launch; more rows fill the chip as they are.
constexpr uint32_t kLogprobEach = 8, kLogprobShares = 64;   // entries of a tile a thread; workgroups a row, at most
constexpr uint64_t kLogprobRows = uint64_t{1} << 14;        // rows of a launch: so many workgroups of 1024 threads, 64 a row, stay a grid
struct LogprobPlan {
  uint32_t threads, width, tiles, shares;                   // columns of a tile, a multiple of four; tiles a workgroup; workgroups a row
};
// What the shares of `rows` rows take: three sums and top_k keys each.
constexpr size_t logprob_bytes(const LogprobPlan& plan, uint64_t rows, uint64_t top_k) {
  return plan.shares < 2 ? 0 : static_cast<size_t>(rows * plan.shares * (12u + 8u * top_k));
}
constexpr LogprobPlan logprob_plan(uint64_t rows, uint64_t vocab, uint64_t top_k, uint64_t cus, size_t most) {
  const uint32_t threads = vocab <= 2048u ? 256u : vocab <= 4096u || rows * vocab <= (1u << 20) ? 512u : 1024u;
  const uint64_t padded = vocab + (vocab % 4u == 0 ? 0u : 3u);      // rows that begin anywhere are read from the 16 bytes before
  const uint64_t widest = uint64_t{threads} * kLogprobEach, all = (padded + widest - 1u) / widest;
  const uint64_t slots = cus * (2048u / threads);
  LogprobPlan best{threads, 0, static_cast<uint32_t>(all), 1};
  if (rows <= kLogprobRows) {
    uint64_t least = (rows + slots - 1) / slots * (all + 1);
    for (uint64_t tiles = (all + kLogprobShares - 1) / kLogprobShares, last = tiles + 64u; tiles < all && tiles < last; ++tiles) {
      const uint64_t shares = (all + tiles - 1) / tiles, cost = (rows * shares + slots - 1) / slots * (tiles + 1) + 2;
      const LogprobPlan plan{threads, 0, static_cast<uint32_t>(tiles), static_cast<uint32_t>(shares)};
      if (cost < least && logprob_bytes(plan, rows, top_k) <= most) least = cost, best = plan;
    }
  }
  // all tiles of a row about as wide
  const uint64_t tiles = uint64_t{best.tiles} * best.shares, width = ((padded + tiles - 1u) / tiles + 3u) / 4u * 4u;
  best.width = static_cast<uint32_t>(width < widest ? width : widest);
  return best;
}

// ---- "attention_pages" -----------------------------------------------------------------------------------------------
// A unit is `columns` (row, head) pairs of a key head in a sequence: one unit a sequence where 16, 32 or 64 hold all, else 128 each.
struct PagesCall {
  uint64_t rows, sequences, group, kv_heads, head_dim, max_rows, max_len, window, sinks;      // group: queries' heads to a key head
};
struct PagesShape {
  uint64_t columns, parts, part_tiles;                        // parts of a unit's positions, tiles each
  uint64_t even;                                              // workgroups that share all tiles evenly; 0: a workgroup a part
  uint64_t waves;                                             // wavefronts a workgroup, where columns are few
};
constexpr uint32_t kPagePartsMost = 1024;                     // that the merge takes
// Positions of a tile, as a power of two: 64, or 32 where a tile's codes and the sums are more registers together than a
// wavefront has with another on its SIMD (heads of 256, as the register limit has it: 48 sequences 91 us with 64 and one
// wavefront, 88 with 32 and two).
constexpr uint32_t pages_log_tile(uint64_t head_dim, uint64_t columns) {
  return columns >= 64 || (columns == 16 && head_dim <= 128) ? 6 : 5;
}
// To begin a head in an even split costs what so many tiles do (of 64 positions 2, 4, 6, 9, 12: 35.4, 33.4, 31.2, 33.7, 36.4
// us for windows of 4096 in 8 sequences of 8 heads, and within 2 % for 48 sequences of all lengths).
constexpr uint32_t begin_tiles(uint32_t log_tile) { return 6u << (6u - log_tile); }
constexpr uint64_t pages_units(const PagesCall& c, uint64_t columns) {
  const uint64_t of_row = (c.group + columns - 1) / columns, of_sequence = (c.max_rows * c.group + columns - 1) / columns;
  uint64_t most = c.rows * c.group / columns + c.sequences;
  for (const uint64_t other : {c.rows * of_row, c.sequences * of_sequence}) most = other < most ? other : most;
  return most;
}
// Columns of a unit that can be there; tiles that it walks at most.
constexpr uint64_t pages_stored(const PagesCall& c, uint64_t columns) { return c.max_rows * c.group < columns ? c.max_rows * c.group : columns; }
constexpr uint64_t pages_tiles(const PagesCall& c, uint64_t columns) {
  const uint64_t tile = uint64_t{1} << pages_log_tile(c.head_dim, columns), all = (c.max_len + tile - 1) / tile;
  const uint64_t some = (c.sinks + tile - 1) / tile + (c.window + c.max_rows + tile - 1) / tile + 1;
  return c.window == 0 || all < some ? all : some;
}
// What the parts leave for the merge: for each column their result, its reference and its weights' sum.
constexpr size_t pages_bytes(const PagesCall& c, const PagesShape& shape) {
  const uint64_t places = shape.even != 0 ? 2 * shape.even : shape.parts < 2 ? 0 : pages_units(c, shape.columns) * c.kv_heads * shape.parts;
  return static_cast<size_t>(places * pages_stored(c, shape.columns) * (c.head_dim + 2) * 4);
}
// Few columns: one workgroup a head of a sequence, or parts of four tiles where all of those are on the chip at once, or an
// even split.  A split costs the merge and its launch, each of its runs a start; one workgroup has the longest sequence's time.
// us, one workgroup / parts: a sequence of 4 heads of 64, 500 positions 7.3 / 11.3, 1500 11.0 / 11.4, 2000 13 / 12; 8 heads of
// 128, 400 10.4 / 13.2, 1000 13.7 / 13.2; 4 heads of 256, 250 11.8 / 14.0, 500 14.9 / 14.0.  One / even split, sequences of all
// lengths up to the stated one: 40 of 8 heads of 128, 2000 29 / 32, 3000 51 / 41; 128 of them, 3000 92 / 99, 5000 142 / 141, 8000
// 215 / 205; 48 of 4 heads of 256, 1500 27 / 31, 3000 52 / 46, 8000 124 / 88; 200 of them, 3000 147 / 151, 5000 225 / 211.
// Many columns: 64 where they hold all, else 128 (though 65 pairs fill half of those).  us, 64 / 128 columns, int8, heads of 64, 128 and 256 (8, 8 and
// 4 key heads; E4M3 within 8 % but for 190 / 182 of the first): 2 x 1500 rows of 6 queries on 1000 positions 254 / 199, 321 / 299, 298 / 263; 4 x
// 512 of 4 on 4000 258 / 207, 319 / 273, 273 / 231; 64 x 13 of 5 on 1000 77 / 60, 96 / 82, 93 / 70; 8 x 15 of 6 on 3000 53 / 48, 70 / 66, 55 / 50.  They
// cost where units of 128 leave CUs idle and parts of theirs do not fit or do not pay: 8 x 50 of 4 on 3000 93 / 92, 102 / 98, 96 / 141; 32 x 15 of
// 6 on 2000 72 / 108, 90 / 77, 78 / 104; 400 of 4 alone 34 / 36, 38 / 37, 31 / 37.
// Parts only where the units are fewer than two a CU, as if two workgroups were on a CU at once.  So they are of 256 threads; of 512 threads (heads
// over 64 in 128 columns, over 128 in 64) it is one.  (`most`: bytes that the parts may take.)
constexpr PagesShape pages_rule(const PagesCall& c, uint64_t cus, size_t most) {
  const uint64_t pairs = c.max_rows * c.group, columns = pairs <= 16 ? 16 : pairs <= 32 && c.head_dim <= 128 ? 32 : pairs <= 64 ? 64 : 128;
  const uint64_t tiles = pages_tiles(c, columns), groups = pages_units(c, columns) * c.kv_heads, log_tile = pages_log_tile(c.head_dim, columns);
  const uint64_t resident = 2 * cus < kPagePartsMost ? 2 * cus : kPagePartsMost;
  const PagesShape one{columns, 1, tiles, 0, columns < 64 && groups <= cus ? 8u : 4u};
  if (groups * pages_stored(c, columns) >= (1u << 24)) return one;      // (the merge has a workgroup a column: a grid of fewer than 2^32 threads)
  if (columns < 64) {
    const uint64_t parts = (tiles + 3) / 4, of_64 = tiles >> (6 - log_tile);
    const PagesShape each{columns, parts, 4, 0, 4};
    if (groups * parts <= resident) {
      return parts < 2 || of_64 <= (c.head_dim <= 64 ? 24 : c.head_dim <= 128 ? 12 : 6) || pages_bytes(c, each) > most ? one : each;
    }
    if (of_64 <= 32 || of_64 <= 38 * groups / resident) return one;
    // As many workgroups as are on the chip at once, or as leave no more than there is room for: of 16 MB 504 of 512 where all of 32 columns
    // of 128, 508 where all of 16 of 256 are there.
    const PagesShape even{columns, 1, tiles, 1, 4};
    const uint64_t room = most / pages_bytes(c, even), runs = room < resident ? room : resident;
    return c.sequences * c.kv_heads * (tiles + begin_tiles(5)) < (1u << 30) && runs != 0 ? PagesShape{columns, 1, tiles, runs, 4} : one;      // (32-bit sums)
  }
  uint64_t parts = groups >= 2 * cus ? 1 : 2 * cus / groups;
  if (parts > 256) parts = 256;
  if (parts > (tiles + 3) / 4) parts = (tiles + 3) / 4;
  for (; parts > 1; --parts) {
    const uint64_t each = (tiles + parts - 1) / parts;
    const PagesShape shape{columns, (tiles + each - 1) / each, each, 0, 4};
    if (shape.parts > 1 && pages_bytes(c, shape) <= most) return shape;
  }
  return one;
}

// ---- "attention_combine" ---------------------------------------------------------------------------------------------
// Wavefronts of a (row, head): sixteen where there are few and many parts, four where the rows fill the chip by themselves or
// sixteen parts are all that there are, one where its four are and that does not make a lane's run long with few rows (us, 1 /
// 4 / 16 wavefronts: 24 rows of 256 over 4 parts 3.3 / 2.9 / 3.2, over 64 15 / 6.9 / 6.0; 12288 rows of 64 over 2 parts 5.4 / 10 / 39,
// of 256 over 8 26 / 25 / 55).
constexpr uint32_t combine_waves(uint64_t rows, uint64_t head_dim, uint64_t parts) {
  if (parts <= 4 && (rows >= 1024 || head_dim <= 64 || parts == 1)) return 1;
  return parts <= 16 || rows > 256 ? 4 : 16;
}

}  // namespace qmm
