// Which tile a matrix product gets and over how many workgroups the K steps of a tile are shared out: host
// arithmetic only, by a model of the time each choice takes.
#ifndef PRODUCT_PLAN_H
#define PRODUCT_PLAN_H

#include <cstddef>

namespace product {

struct TileCost {
  int bm, bn;       // tile of the product (gated: bn / 2 result columns)
  int per_cu;       // workgroups that share a CU
  float rate;       // share of the matrix rate that a full CU reaches in the K loop
  float step_floor; // cycles one K step takes at least: the round trip of its loads
  float fixed;      // cycles per workgroup outside the K loop (first loads, epilogue)
};

constexpr TileCost kTiles[] = {
    {256, 256, 1, 0.80f, 1500.0f, 9000.0f},
    {192, 192, 1, 0.75f, 1500.0f, 7000.0f},
    {128, 128, 2, 0.60f, 1200.0f, 5000.0f},
    {64, 64, 4, 0.35f, 1000.0f, 3500.0f},
};

struct Plan {
  int tile, splits, steps_per_split;
  size_t slab_bytes;
};

inline Plan plan_product(int elem_bytes, int gated, int segs, int sym, int M_out, int N_out, int K, int batch, int compute_units) {
  Plan best = {};
  float best_time = 0.0f;
  const int kstep = 128 / elem_bytes;
  const int steps = (K + kstep - 1) / kstep * segs;
  const float flops_per_cycle = elem_bytes == 2 ? 4096.0f : 256.0f;   // of one CU
  for (int t = 0; t < 4; ++t) {
    const TileCost& c = kTiles[t];
    const long nbm = ((long)M_out + c.bm - 1) / c.bm, nbn = ((long)N_out + (gated ? c.bn / 2 : c.bn) - 1) / (gated ? c.bn / 2 : c.bn);
    const long tiles = (sym ? nbm * (nbm + 1) / 2 : nbm * nbn) * batch;
    const float step = 2.0f * c.bm * c.bn * kstep / flops_per_cycle / c.rate;   // alone on a CU at full rate
    for (int splits = 1; splits <= 32; splits *= 2) {
      const int per = (steps + splits - 1) / splits;
      if (splits > 1 && (per < 4 || (long)(splits - 1) * per >= steps)) break;
      const long groups = tiles * splits;
      const long slots = (long)compute_units * c.per_cu;
      const long full = groups / slots, rest = groups % slots;
      const float slots_f = (float)c.per_cu;
      auto round = [&](float resident) {   // workgroups resident per CU
        const float s = step * resident > c.step_floor ? step * resident : c.step_floor;
        return per * s + c.fixed;
      };
      float time = full * round(slots_f);
      if (rest) time += round((float)((rest + compute_units - 1) / compute_units));
      const size_t slab = splits > 1 ? (size_t)splits * batch * (gated ? 2 : 1) * M_out * ((N_out + 3) / 4 * 4) * 4 : 0;
      // slabs: written once, read once, about 1.7 KB a cycle, and one more launch
      if (splits > 1) time += 2.0f * slab / 1700.0f + 6000.0f;
      if (slab > ((size_t)1 << 30)) break;
      if (best_time == 0.0f || time < best_time) {
        best_time = time;
        best.tile = t;
        best.splits = splits;
        best.steps_per_split = per;
        best.slab_bytes = slab;
      }
    }
  }
  return best;
}

}  // namespace product

#endif
