// Host side of the matrix-product engine: which tile a product gets, whether its K steps are shared out,
// and the launches.  Used by the translation units that instantiate kernels (ffn.hip, orthogonalize.hip).
#ifndef PRODUCT_LAUNCH_H
#define PRODUCT_LAUNCH_H

#include "product_ops.h"
#include "product_plan.h"
#include "roller_hip.h"
#include "roller_internal.h"

#define PT_TRY(expr)              \
  do {                            \
    const int rc_ = (expr);       \
    if (rc_) return rc_;          \
  } while (0)

namespace product {

template <class... Params, class... Args>
int launch(void (*kernel)(Params...), const char* what, dim3 grid, int threads, hipStream_t stream, Args... args) {
  // (the arguments converted to the kernel's parameter types, then their addresses)
  return [&](Params... p) {
    void* ptrs[] = {(void*)&p...};
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3(threads), ptrs, 0, stream);
    return e == hipSuccess ? RL_OK : rl_hip_fail(e, what);
  }(args...);
}

inline unsigned blocks_for(long items) {
  const long n = (items + 255) / 256;
  return (unsigned)(n < 1 ? 1 : n > 8192 ? 8192 : n);
}

// Tile k of kTiles (product_plan.h): BM x BN, wave tile, workgroups per CU.
template <int K>
struct tile;
template <> struct tile<0> { static constexpr int BM = 256, BN = 256, WM = 128, WN = 128, PER_CU = 1, BUFS = 2; };
template <> struct tile<1> { static constexpr int BM = 192, BN = 192, WM = 96, WN = 96, PER_CU = 1, BUFS = 3; };
template <> struct tile<2> { static constexpr int BM = 128, BN = 128, WM = 64, WN = 64, PER_CU = 1, BUFS = 4; };
template <> struct tile<3> { static constexpr int BM = 64, BN = 64, WM = 32, WN = 32, PER_CU = 2, BUFS = 4; };

template <int K, class T, int A_KM, int B_KM, int GATED, int SEGS, int SYM, class Epi>
int launch_tile(const Problem& p, const Partial& part, const Epi& epi, int batch, hipStream_t stream, const char* what) {
  typedef tile<K> t;
  // a gated wave tile of 32 or 96 columns is 16 or 48 of each kind: blocks of 16
  typedef Shape<T, t::BM, t::BN, t::WM, t::WN, A_KM, B_KM, GATED, SEGS, SYM, t::PER_CU, (GATED && t::WN / 2 % 32 != 0) ? 16 : 32, t::BUFS> S;
  const long nbm = (p.M_out + S::BM - 1) / S::BM, nbn = (p.N_out + S::OUT_N - 1) / S::OUT_N;
  const long groups = (SYM ? nbm * (nbm + 1) / 2 : nbm * nbn) * p.splits;
  if (groups > 0xffffff) return rl_fail(RL_ERR_INVALID_ARG, "%s: %ld workgroups are more than one launch takes", what, groups);
  return launch(tile_kernel<S, Epi>, what, dim3((unsigned)groups, 1, batch), S::NT, stream, p, part, epi);
}

// The product `p` (extents, operands) with epilogue `epi`: tile and split by plan(), slabs of a split one
// from `room` (plan().slab_bytes of it).
template <class T, int A_KM, int B_KM, int GATED, int SEGS, int SYM, class Epi>
int run_product(Problem p, const Epi& epi, int batch, void* room, hipStream_t stream, int compute_units, const char* what) {
  const Plan plan = plan_product(sizeof(T), GATED, SEGS, SYM, p.M_out, p.N_out, p.K, batch, compute_units);
  p.splits = plan.splits;
  p.steps_per_split = plan.steps_per_split;
  Partial part = {};
  part.slab = (float*)room;
  part.pitch = (p.N_out + 3) / 4 * 4;
  part.slab_size = (long)p.M_out * part.pitch;
  part.per_split = batch * (GATED ? 2 : 1);
  switch (plan.tile) {
    case 0: PT_TRY((launch_tile<0, T, A_KM, B_KM, GATED, SEGS, SYM>(p, part, epi, batch, stream, what))); break;
    case 1: PT_TRY((launch_tile<1, T, A_KM, B_KM, GATED, SEGS, SYM>(p, part, epi, batch, stream, what))); break;
    case 2: PT_TRY((launch_tile<2, T, A_KM, B_KM, GATED, SEGS, SYM>(p, part, epi, batch, stream, what))); break;
    default: PT_TRY((launch_tile<3, T, A_KM, B_KM, GATED, SEGS, SYM>(p, part, epi, batch, stream, what))); break;
  }
  if (p.splits == 1) return RL_OK;
  const long quads = (long)p.M_out * (part.pitch / 4);
  return launch(join_kernel<Epi, GATED != 0>, what, dim3(blocks_for(quads), 1, batch), 256, stream, part, p.splits,
                SYM ? kTiles[plan.tile].bm : 0, p.M_out, p.N_out, epi);
}

}  // namespace product

#endif
