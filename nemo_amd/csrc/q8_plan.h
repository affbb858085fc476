// q8_plan.h -- which kernel a product of 8-bit rows runs on, and its launch: plain C++ (no HIP), so that the rules and limits can be checked
// on the CPU for sizes that no test can hold.
#ifndef Q8_PLAN_H
#define Q8_PLAN_H

#include <stddef.h>
#include <stdint.h>

constexpr int Q8_PR = 256;                             // rows per workgroup of the short-row kernel, at most
constexpr size_t Q8_MAX_BLOCKS = (1u << 24) - 1;       // 256 threads each: a launch holds fewer than 2^32 threads
// Rows of an operand, at most: the kernels count them in an int, up to 1023 past the last one (the last wave's of the score's 1024).
constexpr int32_t Q8_MAX_ROWS = 0x7fffffff - 1023;
// Row length of a result, at most: a lane's place behind the first of 32 rows and 64 columns, (4 n_cols + 62) numbers of up to 4 bytes, has
// to fit 32 bits in the kernels' stores.
constexpr int32_t Q8_MAX_COLS = 1 << 27;

enum Q8Kernel { Q8_FEW, Q8_SHORT, Q8_LONG };
enum Q8Refusal { Q8_FITS, Q8_WIDE, Q8_MANY };  // more than Q8_MAX_COLS columns; more workgroups than a launch holds

struct Q8Problem {
  int32_t M, n_seg;    // rows, segments they are cut into
  int ragged;          // the cuts are anywhere (offsets on the device); else one segment
  int32_t n_cols, K;
  int out_bytes;       // of a number of the result
  int n_cu;
};
struct Q8Plan {
  Q8Refusal refusal;
  Q8Kernel kernel;
  unsigned grid_x, grid_y;
  size_t tiles, cuts;  // of rows, of columns
  int across;          // few: waves of a workgroup side by side
  int split;           // few: the waves deal the blocks of a row among them
  int wc, rt;          // short: waves over different columns; row tiles of a workgroup
};

inline bool q8_rows_fit(int64_t n) { return n <= Q8_MAX_ROWS; }
// Tiles of tm rows that cover the rows, wherever the cuts are (one segment: no more than its own).
inline size_t q8_tiles(const Q8Problem &p, size_t tm) { return ((size_t)p.M + tm - 1) / tm + (p.ragged ? (size_t)p.n_seg : 0); }

inline Q8Plan q8_plan(const Q8Problem &p) {
  Q8Plan r = {};
  if (p.n_cols > Q8_MAX_COLS) {
    r.refusal = Q8_WIDE;
    return r;
  }
  const size_t chunks = ((size_t)p.n_cols + 127) / 128, cus = (size_t)p.n_cu;
  const int nb = (p.K + 127) / 128;
  // One wave for 32 x 32 in three cases (f32 results, us; in brackets with the kernels below, which also take what does not fit its grid):
  // - Up to 32 columns: 262144 x 16 x 128 10.8 (18.8), x 32 12.3 (19.1), x 48 21.8 (19.8); x 16 x 512 36.6 (42.5), x 32 39.2 (45.3), x 48 69.8
  //   (47.5); 100000 x 32 x 2048 46.9 (63.1), x 48 76.3 (64.8).
  // - So few rows that 32 x 128 products a workgroup make at most 3 workgroups for 2 compute units: 1000 x 1000 x 128 on the device alone 4.3 (5.7),
  //   300 x 8000 x 128 7.1 (6.1).
  // - Fewer than 64 rows a segment on average: 256 segments of 8 x 1000 x 128 15.2 (16.4), of 32 17.6 (19.9), of 48 26.2 (23.9), of 64 33.7 (31.6).
  //   What it does not see: with K = 512 it loses at any length (of 8 49.9 (43.4), of 48 95.5 (54.5)), and where most segments are empty
  //   (12 of 2000 rows among 600 x 128 52 (67), but among 3000 319 (195), x 512 1198 (356)).
  if (p.n_cols <= 32 || 2 * q8_tiles(p, 32) * chunks <= 3 * cus || (size_t)p.M < 64 * (size_t)p.n_seg) {
    r.kernel = Q8_FEW;
    r.split = nb > 2;
    r.across = p.n_cols <= 32 ? 1 : 4;
    r.tiles = q8_tiles(p, r.split ? 32 : 128 / r.across);
    r.cuts = r.split ? ((size_t)p.n_cols + 31) / 32 : r.across == 1 ? 1 : chunks;
    if (r.tiles <= Q8_MAX_BLOCKS && r.cuts <= 65535) {
      r.grid_x = (unsigned)r.tiles;
      r.grid_y = (unsigned)r.cuts;
      return r;
    }
  }
  size_t blocks;
  if (nb == 1) {
    // Short rows: 8 waves over 512 columns of a bf16 result (wc = 8), over half of them in f32, two to the same columns: 1 KB of a row
    // either way.  (262144 rows x 1095 x 128, whose rows begin anywhere in a line: f32 312 us with wc = 8, 242 with 4; bf16 186 and 204; x 1088,
    // whole lines: f32 227 and 214, bf16 125 and 155.)  Fewer where there are fewer columns.  As many rows to a workgroup, up to 128 (f32) or
    // 256, as still give a workgroup to every compute unit (8000 x 1088 f32: 128 rows 11.2 us, 64 11.6, 32 13.8; 262144 x 1088 f32: 213,
    // 317, 378).
    r.kernel = Q8_SHORT;
    r.wc = p.out_bytes == 4 ? 4 : 8;
    while (r.wc > 1 && p.n_cols <= 64 * (r.wc / 2)) r.wc /= 2;
    r.cuts = ((size_t)p.n_cols + 64 * r.wc - 1) / ((size_t)64 * r.wc);
    r.rt = (p.out_bytes == 4 ? Q8_PR / 2 : Q8_PR) / 32;
    while (r.rt > 8 / r.wc && r.rt > 1 && q8_tiles(p, 32 * r.rt) * r.cuts < cus) r.rt /= 2;
    r.tiles = q8_tiles(p, 32 * r.rt);
    blocks = (r.tiles * r.cuts + 7) / 8 * 8;
    if (blocks > (1u << 23) - 1) r.refusal = Q8_MANY;  // 512 threads each
  } else {
    r.kernel = Q8_LONG;
    r.tiles = q8_tiles(p, 128);
    r.cuts = chunks;
    blocks = (r.tiles * r.cuts + 7) / 8 * 8;
    if (blocks > Q8_MAX_BLOCKS) r.refusal = Q8_MANY;
  }
  r.grid_x = (unsigned)blocks;
  r.grid_y = 1;
  return r;
}

#endif  // Q8_PLAN_H
