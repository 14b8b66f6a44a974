// Which kernel serves a microscaled product, and how.  Host code alone, without
// HIP, so a program without a GPU can ask too.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace nsd {

constexpr int kMxBlock = 32;         // values under one scale
constexpr int kMxTileK = 128;        // k of a tile
constexpr int kMxTile4 = 1024;       // bytes of a tile's 4-bit codes
constexpr int kMxTile8 = 2048;       // and of its 8-bit codes
constexpr int kMxScaleTile = 256;    // scale bytes of 16 rows x 4 tiles of k

constexpr int64_t mx_row_tiles(int64_t rows) { return (rows + 15) / 16; }
constexpr int64_t mx_k_tiles(int64_t n_in) { return (n_in + kMxTileK - 1) / kMxTileK; }

constexpr int kMxWaves = 4;      // of a workgroup of the stream kernel
constexpr int kMxFp16Tiles = 4;  // row tiles that it takes as fp16

enum MxKernel { kMxStream, kMxTile128x256, kMxTile128 };
struct MxConfig {
  MxKernel kernel = kMxStream;  // a shape of mx_tile_kernel, or mx_stream_kernel with
  int mt = 1, jw = 1, splits = 1;
  bool fp16 = false;  // reads x as it is
  bool nt = false;    // the weight past the caches
};

// Stream kernels that exist: 1 to 8 row tiles by 1, 2, 3, 4 or 6 column tiles
// (gated: the even ones), x as fp16 up to kMxFp16Tiles, and with the weight past
// the caches these.  Rows as fp16 pay below some 130 steps of a workgroup alone
// (2.6 us of cutting against 20 ns a step), so of the weights that large only
// wide groups over one row tile take them.
constexpr bool mx_stream_nt(int mt, int jw, bool fp16) { return !fp16 || (mt == 1 && jw == 6); }

// Which kernel serves a product, and how: the cheapest by a model of each one's
// time in ns.  Its constants are fitted to sweeps and order the choices; they are
// no rates of one unit, and nothing in it stands for the memory (16 x 4096 ->
// 151936 takes 59 us, 31 by the model).  Against every choice at 134 shapes (1 to
// 8192 rows, ten weights from 1024 x 1024 to 151936 x 4096), GPU time with the
// weight called again and again and among others together: rows given in blocks
// 0.3% off the best on the average and 14% at worst, fp16 rows 1.4% and 38%.
//
// The stream kernel:
//   - A compute unit takes in weight and x together, however they mix, a KB in
//     11 ns where two workgroups share it or it has one to run, in 18 where
//     one's registers leave no room for another.  (Measured 9 out of the L2, 16
//     with the weight out of the last-level cache, 24 among other weights.)
//   - A workgroup's end, its sums through LDS and its stores, takes 175 ns a
//     tile (measured 140 to 200).
//   - x as fp16 is more bytes to every workgroup and 39 ns of cutting a step
//     and row tile, and saves the pass that cuts it once, 2.6 us.  From 33 rows
//     on that is what the host takes to launch it, more than the device does:
//     33, 48 and 64 x 1024 -> 1024 take 6.9, 7.6 and 9.1 us a call against 9.7,
//     9.8 and 9.9 with the pass, but in a graph 6.9, 7.8 and 9.3 against 6.3,
//     6.2 and 6.7.  (33 x 2080 -> 18993 loses either way: 12.4 against 10.0 us a
//     call, 13 against 10 in a graph.)
// The tile kernel: a step of 128 k takes a workgroup of 128 x 256 900 ns alone on
// its compute unit, two of them 1430; of 128 x 128 425 and 780.  (One of 256 x
// 256, eight waves, takes as long as two of 128 x 256 and was no faster where
// its tiles come out even, 105 us for 8192 x 4096 -> 4096 either way.)
// Splits of k cost a pass that adds them, 2.1 us and their bytes, at 3 TB/s the
// stream kernel's, whose stores are runs of 64 bytes, and 4.6 the other's; they
// serve rows of whole vectors.  (The 128 x 256 tile has none: what it serves
// fills the device without.)
constexpr double kMxCutNs = 2600.0;

inline double mx_split_ns(int splits, int64_t n_rows, int64_t n, double bytes_per_ns) {
  return splits == 1 ? 0.0 : 2100.0 + (double)splits * n_rows * n * 8 / bytes_per_ns;
}

inline double choose_stream(MxConfig& best, double least, int64_t n_rows, int64_t n, int64_t T, bool gated,
                            bool quantised, int cus) {
  const int64_t row_tiles = mx_row_tiles(n_rows), chunks = (row_tiles + 7) / 8;
  const int mt = (int)((row_tiles + chunks - 1) / chunks);
  const int64_t out_tiles = (n + 15) / 16;
  for (int fp16 = 0; fp16 <= (!quantised && row_tiles <= kMxFp16Tiles ? 1 : 0); ++fp16)
    for (int jw : {1, 2, 3, 4, 6}) {
      if (gated && jw % 2) continue;
      const int p = gated ? jw / 2 : jw;
      const int64_t groups = (out_tiles + p - 1) / p * chunks;
      const bool two = 4 * jw * mt + (fp16 ? 34 : 18) * mt + 11 * jw + 12 <= 252;
      for (int splits : {1, 2, 3, 4, 6, 8}) {
        if (splits > 1 && (gated || n % 8 || T < kMxWaves * splits)) break;  // a wave has a step at least
        const int64_t wgs = groups * splits;
        const double rounds = wgs <= 2 * cus ? (double)((wgs + cus - 1) / cus) : (double)wgs / cus + 0.5;
        const double steps = (double)((T + splits - 1) / splits);
        const double x_kb = fp16 ? n_rows * 0.25 : 2.0 * mt;  // rows of fp16 that do not exist are not fetched
        const double t = 2700.0 + mx_split_ns(splits, n_rows, n, 3000.0) + (fp16 || quantised ? 0.0 : kMxCutNs) +
                         rounds * (steps * ((jw + x_kb) * (wgs > cus && !two ? 18.0 : 11.0) + (fp16 ? 39.0 * mt : 0.0)) +
                                   jw * mt * 175.0);
        if (t < least) {
          least = t;
          best = MxConfig{};
          best.mt = mt;
          best.jw = jw;
          best.splits = splits;
          best.fp16 = fp16 != 0;
        }
      }
    }
  return least;
}

inline double choose_tile(MxConfig& best, double least, int64_t n_rows, int64_t n, int64_t T, bool gated,
                          bool quantised, int cus) {
  for (MxKernel kernel : {kMxTile128x256, kMxTile128}) {
    const bool wide = kernel == kMxTile128x256;
    const int64_t columns = (wide ? 256 : 128) / (gated ? 2 : 1);
    const int64_t tiles = (n_rows + 127) / 128 * ((n + columns - 1) / columns);
    for (int splits : {1, 2, 3, 4, 6, 8}) {
      if (splits > 1 && (wide || gated || n % 8 || (T + 3) / 4 < splits)) break;
      const int64_t wgs = tiles * splits, full = wgs / (2 * cus), rest = wgs - full * 2 * cus;
      const double one = wide ? 900.0 : 425.0, two = wide ? 1430.0 : 780.0;
      const double steps = splits == 1 ? (double)T : 4.0 * (((T + 3) / 4 + splits - 1) / splits);
      const double t = 3300.0 + mx_split_ns(splits, n_rows, n, 4600.0) + (quantised ? 0.0 : kMxCutNs) +
                       steps * (full * two + (rest == 0 ? 0.0 : rest <= cus ? one : two)) +
                       (double)(full + (rest > 0)) * (wide ? 1900.0 : 860.0);
      if (t < least) {
        least = t;
        best = MxConfig{};
        best.kernel = kernel;
        best.splits = splits;
      }
    }
  }
  return least;
}

// n_rows, n and T at least 1.
inline MxConfig choose_mx(int64_t n_rows, int64_t n, int64_t T, bool gated, bool quantised, int cus) {
  // The choice of a shape, not worked out anew every call (1.5 us of a decode
  // step's 7): the last ones of this thread.
  struct Chosen {
    int64_t n_rows = -1, n = 0, T = 0;
    int kind = 0, cus = 0;
    MxConfig config;
  };
  static thread_local Chosen kept[64];
  const int kind = gated * 2 + quantised;
  Chosen& c = kept[(uint64_t)(n_rows * 31 + n * 7 + T * 3 + kind) % 64];
  if (c.n_rows == n_rows && c.n == n && c.T == T && c.kind == kind && c.cus == cus) return c.config;
  MxConfig best;
  double least = choose_stream(best, 1e300, n_rows, n, T, gated, quantised, cus);
  choose_tile(best, least, n_rows, n, T, gated, quantised, cus);
  // A weight that the 256 MB last-level cache cannot keep from call to call
  // streams faster past it: 311 MB, one, 16 and 80 rows 57 -> 53, 61 -> 57 and
  // 112 -> 106 us.  One that it keeps, called again and again, slower: 7.0 -> 9.4 (34
  // MB, 16 rows), 24 -> 25 (134), 39 -> 42 (235).  Among other weights past the
  // caches is faster from 34 MB on, 11.0 -> 10.5, 29 -> 27 and 48 -> 43.
  best.nt = best.kernel == kMxStream && mx_stream_nt(best.mt, best.jw, best.fp16) &&
            (double)((n + 15) / 16) * (gated ? 2 : 1) * T * kMxTile4 > 192e6;
  c = Chosen{n_rows, n, T, kind, cus, best};
  return best;
}

}  // namespace nsd
