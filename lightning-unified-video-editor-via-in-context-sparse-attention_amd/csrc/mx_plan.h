// Which kernels the token rows of a 4-bit product run in.  Host code only.
#pragma once

#include <algorithm>
#include <cstdint>

#define MXG_CUS 256

// The kernel of few rows against the tile kernel (128 x 128 tiles, one workgroup for 128 outputs whatever the rows; us, codes in,
// N x K): 5,120 x 5,120 at 1 / 32 / 64 rows 8.9 / 8.5 / 10.6 to 12.9 / 13.5 / 13.6; 5,120 x 13,824 11.1 / 15.7 / 22.8 to
// 27.0 / 27.1 / 27.4; 13,824 x 5,120 10.0 / 12.9 / 22.8 to 13.1 / 13.5 / 14.5; 30,720 x 5,120 at 1 / 4 / 16 rows 19.7 / 20.7 /
// 25.1 to 18.9 / 18.9 / 19.2, 20,480 x 5,120 15.7 / 16.4 / 19.0 to 13.5 / 13.5 / 13.7: many outputs fill the chip with tiles,
// whose lines are read whole.
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
