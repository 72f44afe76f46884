// Which kernels the token rows of a 4-bit product run in.  Host code only.
#pragma once

#include <algorithm>
#include <cstdint>

#define MXG_CUS 256

// The kernel of few rows against the tile kernel (128 x 128 tiles, one workgroup for 128 outputs whatever the rows); us in a graph,
// codes in, N x K at 1 / 32 / 64 rows:
//   5,120 x 512      2.8 / 3.1 / 4.1    to  5.2 / 5.3 / 5.5      13,824 x 2,048    5.7 / 7.1 / 11.2   to  8.2 / 8.4 / 8.8
//   5,120 x 2,048    4.3 / 5.1 / 6.5    to  7.9 / 8.1 / 8.5      16,384 x 2,048    5.7 / 7.2 / 11.2   to  8.4 / 8.5 / 9.0
//   5,120 x 5,120    6.1 / 8.0 / 10.7   to 13.0 / 13.4 / 14.0    13,824 x 5,120   11.2 / 16.4 / 22.4  to 15.5 / 16.7 / 18.1
//   8,192 x 5,120    6.5 / 8.0 / 10.7   to 13.3 / 13.6 / 14.2    16,384 x 5,120   11.7 / 16.5 / 22.9  to 17.3 / 17.8 / 19.3
//   5,120 x 13,824  14.0 / 18.8 / 25.2  to 29.0 / 30.4 / 32.9    13,824 x 13,824  25.8 / 37.5 / 49.1  to 33.8 / 34.9 / 36.7
//   8,192 x 13,824  13.9 / 21.4 / 25.9  to 29.8 / 30.9 / 33.6    20,480 x 5,120   14.5 / 22.7 / 32.0  to 17.6 / 19.3 / 20.4
//   30,720 x 512     4.4 / 5.2 / 8.3    to  6.3 / 6.5 / 6.9      30,720 x 5,120   18.9 / 29.8 / 42.5  to 19.7 / 21.2 / 23.4
// Many outputs fill the chip with tiles, whose lines are read whole.  (The rule leaves out k: single rows of many outputs and
// short ones would still gain, 32 rows of 13,824 x 13,824 lose.)
inline bool mx_rows_takes(int64_t M, int64_t N) { return (M <= 32 && N <= 16384) || (M <= 64 && N <= 8192); }

// A launch takes rounds of one tile a CU.  Measured (us, one round): a 256 x 256 tile 1.6 a group and 1 to 4 besides, GELU 3.4; a
// 128 x 128 tile 0.56 a group and 2.5, GELU 0.5; a launch 4.5.  In units of 0.56 us.
inline double mx_rounds(int64_t tiles) { return (double)((tiles + MXG_CUS - 1) / MXG_CUS); }
inline double mx_big_time(int64_t tiles, int groups, bool gelu) { return mx_rounds(tiles) * (2.9 * groups + 4 + 6 * gelu); }
inline double mx_small_time(int64_t tiles, int groups, bool gelu) { return mx_rounds(tiles) * (groups + 4.5 + 1 * gelu); }

// How many of the first rows run in 256 x 256 tiles: all, none, or those of whole rounds.  The others run in 128 x 128 tiles or,
// behind large ones, in the kernel of few rows where it takes them.  All three measured (large tiles, small ones, whole rounds and
// the rest; us, M x N x K): 512 x 5,120 x 4,096 24.3, 12.7, -; 1,560 x 5,120 x 5,120 32.0, 41.3, -; 3,120 x 5,120 x 5,120 67.1,
// 57.2, 54.7; 9,360 x 2,000 x 5,120 71.0, 72.4, 61.7; 14,040 x 5,120 x 13,824 454.9, 597.0, 450.3; 65,520 x 5,120 x 5,120 817,
// 1,154, 822.
inline int64_t mx_large_rows(int64_t M, int64_t cols, int groups, bool gelu) {
  const int64_t n_big = (cols + 255) / 256, n_small = (cols + 127) / 128, m_big = (M + 255) / 256;
  auto small = [&](int64_t rows) { return mx_small_time(n_small * ((rows + 127) / 128), groups, gelu); };
  const int64_t split = std::min<int64_t>(n_big * m_big / MXG_CUS * MXG_CUS / n_big, m_big - 1) * 256;   // rows that whole rounds take
  const double t_big = mx_big_time(n_big * m_big, groups, gelu), t_small = small(M);
  const double t_split = split > 0 ? mx_big_time(n_big * (split / 256), groups, gelu) + small(M - split) + 8 : t_big + 1;
  if (t_small <= t_big && t_small <= t_split) return 0;
  return t_big <= t_split ? M : split;
}
