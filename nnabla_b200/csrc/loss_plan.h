// The arithmetic of a head's products on the host: tiles, pieces, and where a call's scratch holds what. No CUDA, so that it can
// be gone through for any size and number of SMs without a GPU.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

namespace nb200 {

inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Scratch for a call, in parts that begin at 256-byte boundaries.
struct Parts {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

// Time of a tile in cycles of an SM: 512 MMA cycles a K block of a pair's 256 x 256 tile, 204 of a 128 x 64 one (51 an
// instruction, for its operands' reads; 32 by its products); its epilogue at least.
inline int64_t loss_tile_cycles(int64_t kblocks, bool pair) {
  return std::max<int64_t>((pair ? 512 : 204) * kblocks, pair ? 4500 : 2000);
}

// Whether a launch's tiles take less time as pairs of SMs' 256 x 256 ones than as 128 x 64 ones: the mean tile, in whole rounds.
struct TileCount {
  int64_t M, N, kblocks;
  int64_t splits = 1; // tiles along K, each of kblocks
};
inline bool pays_pairs(std::initializer_list<TileCount> products, int sms) {
  int64_t pair_tiles = 0, single_tiles = 0, pair_work = 0, single_work = 0;
  for (const TileCount &p : products) {
    const int64_t pairs = ((p.M + 255) / 256) * ((p.N + 255) / 256) * p.splits;
    const int64_t singles = ((p.M + 127) / 128) * ((p.N + 63) / 64) * p.splits;
    pair_tiles += pairs, single_tiles += singles;
    pair_work += pairs * loss_tile_cycles(p.kblocks, true);
    single_work += singles * loss_tile_cycles(p.kblocks, false);
  }
  auto time = [](int64_t work, int64_t tiles, int64_t units) {
    return tiles == 0 ? 0 : (tiles + units - 1) / units * (work / tiles);
  };
  return time(pair_work, pair_tiles, sms / 2) <= time(single_work, single_tiles, sms);
}

// Whether an fp32 head takes W as it lies, its pieces made between memory and the tensor cores, in 128 x 128 tiles: with one tile
// of rows, which makes each piece once a product, and a W of 32 MB or more. The pieces of a smaller one stay in L2, where laying
// them out costs less than the finer tiles, which make no pieces, gain (loss and gradients of 64 rows, us, laid out and as it
// lies: [512, 1000] 50 and 80, [128, 40000] 90 and 95, [777, 10007] 140 and 128, [512, 20000] 149 and 135, [2048, 20000] 510 and
// 322, [4096, 131071] 6399 and 3353).
constexpr int kSplitTile = 128;
inline bool loss_splits(int64_t rows, int64_t size, int64_t classes) {
  return rows <= kSplitTile && size * classes >= 8 << 20;
}

// Two products' tiles on `units`: the first's dealt out one by one, and of the second's this many to each of the units that got
// one more of the first's, the rest to the others, so that the last one ends first.
inline int64_t extra_tiles(int64_t first, int64_t second, int64_t first_cycles, int64_t second_cycles, int64_t units) {
  const int64_t more = first % units;
  if (more == 0 || second == 0)
    return 0;
  // With n tiles the former end at first_cycles + n second_cycles, which grows, the others at rounds(n) second_cycles, which
  // falls: the best lies where the two cross, found by halves.
  auto rounds = [&](int64_t n) {
    return (std::max<int64_t>(0, second - more * n) + units - more - 1) / (units - more);
  };
  int64_t n = 0, top = (second + more - 1) / more; // rounds(top) is 0
  while (n < top) {
    const int64_t half = (n + top) / 2;
    if (first_cycles + half * second_cycles >= rounds(half) * second_cycles)
      top = half;
    else
      n = half + 1;
  }
  if (n == 0 || first_cycles + n * second_cycles < rounds(n - 1) * second_cycles)
    return n;
  // the fewest with as many rounds as n - 1 leaves
  return std::max<int64_t>(0, (second - rounds(n - 1) * (units - more) + more - 1) / more);
}

// The rows of a matrix in slabs, each of whose column sums a block makes for itself (256 columns a block).
constexpr int kSumColumns = 256;
struct Slabs {
  int64_t rows, count; // of a slab; slabs
};
inline Slabs column_slabs(int64_t all_rows, int64_t columns, int sms) {
  const int64_t wide = (columns + kSumColumns - 1) / kSumColumns;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>((all_rows + 31) / 32, 4 * sms / wide));
  const int64_t rows = (all_rows + most - 1) / most;
  return {rows, (all_rows + rows - 1) / rows};
}

// Both gradients of a head of few rows in one pass over W (few_rows.cuh): blocks of kFewBlock classes by `slab` rows of W, which
// lie `step` apart.
constexpr int kFewGradThreads = 256, kFewBlock = 8 * kFewGradThreads;
constexpr int kFewWalk = 32; // rows of W between two exchanges of the warps' sums
struct FewGradients {
  int64_t columns; // blocks of classes; with `shift` one more, for the rows' ends
  int64_t slab, blocks; // rows of W a block; blocks along them
  // (with a third as many blocks, some one and a half rounds of them, [8, 4096] . [4096, 131071] fp32 1002 us, not 907)
  // shift: rows of W that begin up to vec - 1 values behind a 16-byte boundary, and so do the blocks of classes
  FewGradients(int64_t size, int64_t classes, int vec, bool shift, int sms) {
    const int64_t step = shift ? vec : 1, each = (size + step - 1) / step, walks = (each + kFewWalk - 1) / kFewWalk;
    columns = (classes + (shift ? vec - 1 : 0) + kFewBlock - 1) / kFewBlock + (shift ? 1 : 0);
    const int64_t slabs = std::min(walks, (12 * sms + columns * step - 1) / (columns * step));
    slab = (walks + slabs - 1) / slabs * kFewWalk;
    blocks = step * ((each + slab - 1) / slab);
  }
};

// A head's gradients on the tensor cores: the pieces of the classes, the tiles and parts of K of the products, and what of it
// lies where in the scratch. `planes`: three bf16 pieces an fp32 value, or one of 16 bits.
struct HeadGradients {
  int planes;
  int64_t rows, size, classes;
  int64_t piece;        // classes at a time, a multiple of 256; the last piece has what is left
  bool pieces;          // more than one
  bool pair_grad, pair; // tiles of G, of dx and dW
  bool split;           // W as it lies; `pair` is then dW's alone
  int dx_splits, dx_blocks, dw_splits, dw_blocks; // parts of K, K blocks of each
  bool direct;          // dx without sums of its own
  int64_t ld_dx;        // of dx's own sums
  Slabs db; // of G's rows, the same ones for every piece: with fewer classes a piece of its own would have more of them
  // of the scratch: the operands, G [planes][rows][piece], its scale, fp32 sums [dx_splits][rows][ld_dx],
  // [dw_splits][size][piece], [db.count][piece]
  size_t at_x, at_w, at_g, at_scale, at_dx, at_dw, at_db, bytes;

  int64_t classes_at(int64_t c0) const { return std::min(piece, classes - c0); }

  HeadGradients(int64_t rows_, int64_t size_, int64_t classes_, bool f32, bool dx, bool dw, bool with_db, bool accum_dx,
                size_t x_bytes, size_t w_bytes, int sms)
      : planes(f32 ? 3 : 1), rows(rows_), size(size_), classes(classes_) {
    // A piece's G is 64 MB: both products read it from L2, and their tiles are rounds enough to leave few SMs idle.
    piece = std::max<int64_t>(256, (int64_t)(1 << 25) / planes / rows);
    const int64_t count = (classes + piece - 1) / piece;
    piece = up((classes + count - 1) / count, 256);
    pieces = piece < classes;
    const int64_t size_blocks = (size + 63) / 64, row_blocks = (rows + 63) / 64, piece_blocks = (std::min(piece, classes) + 63) / 64;
    split = f32 && loss_splits(rows, size, classes);
    pair_grad = pays_pairs({{rows, piece, size_blocks}}, sms);
    pair = pays_pairs({{dw ? size : 0, piece, row_blocks}, {dx && !split ? rows : 0, size, piece_blocks}}, sms);
    // A product with few tiles and a long K (dx of few rows, dW of many) has it in up to 16 parts, each with sums of its own that
    // add_parts joins, until a tile is a third of an SM's share at most.
    const int64_t tile_m = pair ? 256 : 128, tile_n = pair ? 256 : 64, units = pair ? sms / 2 : sms;
    const int64_t dw_tiles = dw ? (size + tile_m - 1) / tile_m * ((piece + tile_n - 1) / tile_n) : 0;
    const int64_t dx_tiles = dx ? (rows + tile_m - 1) / tile_m * ((size + tile_n - 1) / tile_n) : 0;
    const int64_t share = std::max<int64_t>(8, (dw_tiles * row_blocks + dx_tiles * piece_blocks) / (3 * units));
    auto cut = [&](int64_t tiles, int64_t blocks, int &splits, int &split_blocks) {
      splits = 1;
      while (splits < 16 && tiles * splits < 4 * units && blocks > share * splits)
        splits *= 2;
      split_blocks = (int)((blocks + splits - 1) / splits);
      splits = (int)((blocks + split_blocks - 1) / split_blocks); // no empty part (a last, smaller piece may leave some)
    };
    cut(dx_tiles, piece_blocks, dx_splits, dx_blocks);
    cut(dw_tiles, row_blocks, dw_splits, dw_blocks);
    if (split && dx) { // (its tiles are the last launch: two rounds of them, of eight K blocks at least)
      const int64_t tiles = (size + kSplitTile - 1) / kSplitTile;
      dx_splits = (int)std::max<int64_t>(1, std::min<int64_t>({piece_blocks / 8, 2 * sms / tiles, 64}));
      dx_blocks = (int)((piece_blocks + dx_splits - 1) / dx_splits);
      dx_splits = (int)((piece_blocks + dx_blocks - 1) / dx_blocks);
    }
    direct = dx_splits == 1 && (!pieces || (f32 && !accum_dx));
    ld_dx = up(size, 4);
    db = column_slabs(planes * rows, piece, sms);
    Parts parts;
    at_x = parts.take(x_bytes), at_w = parts.take(w_bytes);
    at_g = parts.take((size_t)planes * rows * piece * 2), at_scale = parts.take(12);
    at_dx = parts.take(dx && !direct ? (size_t)dx_splits * rows * ld_dx * 4 : 0);
    at_dw = parts.take(dw && dw_splits > 1 ? (size_t)dw_splits * size * piece * 4 : 0);
    at_db = parts.take(with_db ? (size_t)db.count * piece * 4 : 0);
    bytes = parts.bytes;
  }
};

} // namespace nb200
