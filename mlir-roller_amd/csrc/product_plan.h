// Which tile a matrix product gets and over how many workgroups the K steps of a tile are shared out: host
// arithmetic only, by a model of the time each choice takes.
#ifndef PRODUCT_PLAN_H
#define PRODUCT_PLAN_H

#include <cstddef>

namespace product {

// What a tile costs on one compute unit, in microseconds: `step` per K step of 128 bytes, `fixed` for first
// loads and epilogue, `once` for the launch.  Fitted to 3588 timings of 339 products that store their sums and
// nothing else (32 to 8192 rows, 64 to 11000 columns, K 64 to 11000, three sets of operands in turn, most of which
// the 256 MB cache before the memory holds; K-major and row-major operands; whole tiles, all split, the last round
// split; some ms of work at a time): there it is off by 13 % (16 bits) and 7 % (32 bits) rms, and what it chooses is on
// average 1 %, at worst 19 %, slower than the fastest choice timed.
// It ranks tiles of one product and does not foretell times.  It has no term for the memory, for what an epilogue
// reads and writes besides the result, or for the clock that the card keeps under a long load, which are much the same
// for every tile; products that are bound by those take up to 2.8 times as long as it says (24 tokens, gate and up weights
// of 134 MB: 12.6 us by the model, 25 of the memory; 4096 x 4096 update, B X with X in fp32: 70 and 134).  Rounds are
// counted by CUs also for the tiles of which a CU holds two or three.
// The large tiles have the higher rate where they fill the CUs (4096^3 in bf16: 103 us with 256 x 256 tiles,
// 113 with 192, 120 with 128, 191 with 64); the small ones where the others would not (1024 x 1920 x 5000:
// 118, 65, 49 and 46 us unsplit), and 192 x 192 makes the lower triangle of 4096 x 4096 253 tiles for 256 CUs.
struct TileCost {
  int bm, bn;   // tile of the product (gated: bn / 2 result columns)
  float step16, fixed16, once16;   // 16-bit operands
  float step32, fixed32, once32;   // 32-bit operands
};

constexpr int XCDS = 8;
constexpr int kFewRowsTile = 4;   // for products of K-major operands only
constexpr TileCost kTiles[] = {
    {256, 256, 0.957f, 8.8f, 0.0f, 6.879f, 8.5f, 0.0f},
    {192, 192, 0.598f, 7.9f, 0.0f, 3.940f, 7.6f, 0.8f},
    {128, 128, 0.340f, 5.1f, 0.0f, 1.748f, 4.5f, 0.8f},
    {64, 64, 0.175f, 1.0f, 2.6f, 0.439f, 0.8f, 2.4f},
    {32, 64, 0.138f, 0.5f, 3.3f, 0.414f, 0.0f, 3.9f},
};
// What splitting costs, microseconds: the workgroup that adds a tile up waits once for every piece ...
constexpr float kJoinPiece = 0.55f;
constexpr float kPieceBytes = 4.0e6f;       // ... and the pieces are written and read, so many bytes per microsecond
constexpr float kClearLaunch = 3.0f;        // a launch that clears the arrival counters, where no other does
constexpr int kMaxSplits = 16;
constexpr int kMaxArrivals = 4096;          // tiles of a split product
constexpr size_t kMaxPieces = (size_t)1 << 29;
constexpr long kMaxGroups = 0xffffff;       // workgroups of a launch (below 2^32 threads)

struct Plan {
  float time;   // microseconds, by the model
  int tile, splits, steps_per_split;
  int whole;    // tiles that are not split, all of them if splits is 1
  size_t piece_bytes;
};

inline Plan plan_product(int elem_bytes, int gated, int segs, int sym, int M_out, int N_out, int K, int batch, int compute_units, int tiles_end, int max_splits = kMaxSplits) {
  Plan best = {};
  const int kstep = 128 / elem_bytes;
  const int steps = (K + kstep - 1) / kstep * segs;
  for (int t = 0; t < tiles_end; ++t) {
    const TileCost& c = kTiles[t];
    const int out_n = gated ? c.bn / 2 : c.bn;
    const long nbm = ((long)M_out + c.bm - 1) / c.bm, nbn = ((long)N_out + out_n - 1) / out_n;
    const long tiles = (sym ? nbm * (nbm + 1) / 2 : nbm * nbn) * batch;
    const float step = elem_bytes == 2 ? c.step16 : c.step32, fixed = elem_bytes == 2 ? c.fixed16 : c.fixed32, once = elem_bytes == 2 ? c.once16 : c.once32;
    // All tiles split alike; or those of full rounds whole, and only what would be a last, partly filled round
    // shared out over the CUs.
    const long rounds = tiles / compute_units * compute_units;
    for (int splits = 1; splits <= max_splits; splits *= 2) {
      const int per = (steps + splits - 1) / splits;
      // (every split has two steps at least; the largest tile is not split)
      if (splits > 1 && (t == 0 || per < 2 || (long)(splits - 1) * per >= steps)) break;
      for (int tail = 0; tail < 2; ++tail) {
        const long whole = splits == 1 ? tiles : tail ? rounds : 0;
        if (tail && (splits == 1 || whole == 0 || whole == tiles || compute_units % XCDS != 0)) continue;
        const size_t pieces = (size_t)(tiles - whole) * splits * c.bm * c.bn * 4;
        if (pieces > kMaxPieces || tiles - whole > kMaxArrivals) continue;
        // (the largest tile stays in any case: what is too much for it is refused)
        if (t != 0 && whole + (tiles - whole) * splits > kMaxGroups) continue;
        const long alone = (whole + compute_units - 1) / compute_units, shared = ((tiles - whole) * splits + compute_units - 1) / compute_units;
        float time = once + alone * (steps * step + fixed) + shared * (per * step + fixed);
        if (splits > 1) time += kJoinPiece * splits + 2.0f * pieces / kPieceBytes;
        if (best.time == 0.0f || time < best.time) best = {time, t, splits, per, (int)whole, pieces};
      }
    }
  }
  return best;
}

// Pitch, in elements, of an internal matrix with rows of `cols`: an odd number of 128-byte lines.  Rows that
// start inside a line cost an extra line per 128 bytes read (measured: 15 instead of 30 TB/s out of the L2),
// and rows a power of two apart crowd the same memory channels (4.4 instead of 6.2 TB/s out of memory).
inline int line_pitch(int elem_bytes, int cols) {
  const int per_line = 128 / elem_bytes, lines = (cols + per_line - 1) / per_line;
  return (lines | 1) * per_line;
}

}  // namespace product

#endif
