// Host side of the matrix-product engine: which tile a product gets, whether its K steps are shared out,
// and the launches.  Used by the translation units that instantiate kernels (ffn.hip, orthogonalize.hip).
#ifndef PRODUCT_LAUNCH_H
#define PRODUCT_LAUNCH_H

#include <atomic>

#include "product_ops.h"
#include "product_plan.h"
#include "roller_hip.h"
#include "roller_internal.h"

#define PT_TRY(...)               \
  do {                            \
    const int rc_ = (__VA_ARGS__); \
    if (rc_) return rc_;          \
  } while (0)

namespace product {

// (the arguments converted to the kernel's parameter types, then their addresses)
template <class... Params, class... Args>
int launch_function(hipFunction_t f, void (*)(Params...), const char* what, dim3 grid, int threads, hipStream_t stream, Args... args) {
  return [&](Params... p) {
    void* ptrs[] = {(void*)&p...};
    const hipError_t e = hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, threads, 1, 1, 0, stream, ptrs, nullptr);
    return e == hipSuccess ? RL_OK : rl_hip_fail(e, what);
  }(args...);
}

// Launches KERNEL.  Its function is looked up once: a launch by symbol looks it up every time, which a call of
// two short kernels notices.
template <auto KERNEL, class... Args>
int launch(const char* what, dim3 grid, int threads, hipStream_t stream, Args... args) {
  static std::atomic<hipFunction_t> known{nullptr};
  hipFunction_t f = known.load(std::memory_order_relaxed);
  if (!f) {
    const hipError_t e = hipGetFuncBySymbol(&f, (const void*)KERNEL);
    if (e != hipSuccess) return rl_hip_fail(e, what);
    known.store(f, std::memory_order_relaxed);
  }
  return launch_function(f, KERNEL, what, grid, threads, stream, args...);
}

inline unsigned blocks_for(long items) {
  const long n = (items + 255) / 256;
  return (unsigned)(n < 1 ? 1 : n > 8192 ? 8192 : n);
}

// Tile k of kTiles (product_plan.h) for elements of ES bytes: BM x BN, wave tile, workgroups per CU, LDS buffers.
// Three of the 64 x 64 tiles fit a CU with three buffers each, two with four.  With 32 bits, where the matrix units
// are the limit, three are faster (333 x 5462 x 1001: 39 us, 44 with two); with 16 bits a step is too short for
// the loads of two (200 x 2880 x 7680: 30 us, 23 with two workgroups and four buffers).
template <int K, int ES>
struct tile;
template <int ES> struct tile<0, ES> { static constexpr int BM = 256, BN = 256, WM = 128, WN = 128, PER_CU = 1, BUFS = 2; };
template <int ES> struct tile<1, ES> { static constexpr int BM = 192, BN = 192, WM = 96, WN = 96, PER_CU = 1, BUFS = 3; };
template <int ES> struct tile<2, ES> { static constexpr int BM = 128, BN = 128, WM = 64, WN = 64, PER_CU = 1, BUFS = 4; };
template <int ES> struct tile<3, ES> { static constexpr int BM = 64, BN = 64, WM = 32, WN = 32, PER_CU = ES == 4 ? 3 : 2, BUFS = ES == 4 ? 3 : 4; };
template <int ES> struct tile<4, ES> { static constexpr int BM = 32, BN = 64, WM = 32, WN = 32, PER_CU = 3, BUFS = 4; };

template <int K, class T, int A_KM, int B_KM, int GATED, int SEGS, int SYM, class Epi>
int launch_tile(const Problem& p, const Epi& epi, int batch, hipStream_t stream, const char* what) {
  typedef tile<K, sizeof(T)> t;
  // Blocks of 32 x 32, or of 16 x 16 where 32 do not fit: gated wave tiles of 32 or 96 columns are 16 or 48 of
  // each kind, and the few-rows tile has two blocks of 16 rows.
  constexpr int MI = K == kFewRowsTile || (GATED && t::WN / 2 % 32 != 0) ? 16 : 32;
  typedef Shape<T, t::BM, t::BN, t::WM, t::WN, A_KM, B_KM, GATED, SEGS, SYM, t::PER_CU, MI, t::BUFS> S;
  static_assert(t::BM == kTiles[K].bm && t::BN == kTiles[K].bn, "the plan's tiles");
  const long nbm = (p.M_out + S::BM - 1) / S::BM, nbn = (p.N_out + S::OUT_N - 1) / S::OUT_N;
  const long tiles = (SYM ? nbm * (nbm + 1) / 2 : nbm * nbn) * batch, groups = p.whole + (tiles - p.whole) * p.splits;
  if (groups > kMaxGroups) return rl_fail(RL_ERR_INVALID_ARG, "%s: %ld workgroups are more than one launch takes", what, groups);
  return launch<tile_kernel<S, Epi>>(what, dim3((unsigned)groups), S::NT, stream, p, epi);
}

// Arrival counters of the products of one call, in its workspace: two sets that take turns.  Every product
// clears the other set for the next one, whether it uses its own or not.  `ready`: the set whose turn it is
// has been cleared, by the product before or by another kernel of the call; a first product that gains more
// from splitting than that costs launches a kernel for it.
struct Arrivals {
  unsigned* set[2];
  bool ready;
  int turn = 0;
};
constexpr size_t kArrivalBytes = 2 * kMaxArrivals * sizeof(unsigned);
inline Arrivals arrivals_at(void* room, bool ready) { return {{(unsigned*)room, (unsigned*)room + kMaxArrivals}, ready}; }

// Which tiles a product may take: the few-rows tile exists for K-major operands.
template <int A_KM, int B_KM, int SEGS, int SYM>
constexpr int tiles_end() { return A_KM && B_KM && !SYM && SEGS == 1 ? kFewRowsTile + 1 : kFewRowsTile; }

// Fills in p's split by `plan` and takes this product's turn of the arrival counters.
inline int take_plan(Problem& p, const Plan& plan, void* room, Arrivals& arrivals, hipStream_t stream) {
  p.splits = plan.splits;
  p.steps_per_split = plan.steps_per_split;
  p.whole = plan.whole;
  p.pieces = (float*)room;
  p.arrivals = arrivals.set[arrivals.turn];
  arrivals.turn ^= 1;
  p.clear = arrivals.set[arrivals.turn];
  p.n_clear = kMaxArrivals;
  if (p.splits > 1 && !arrivals.ready)
    PT_TRY(launch<zero_kernel<unsigned>>("clearing arrival counters", dim3(kMaxArrivals / 256), 256, stream, p.arrivals, kMaxArrivals, 1, kMaxArrivals));
  arrivals.ready = true;
  return RL_OK;
}

// The plan of a product of these forms.
template <class T, int A_KM, int B_KM, int GATED, int SEGS, int SYM>
Plan plan_for(int M_out, int N_out, int K, int batch, int compute_units, int max_splits = kMaxSplits) {
  return plan_product(sizeof(T), GATED, SEGS, SYM, M_out, N_out, K, batch, compute_units, tiles_end<A_KM, B_KM, SEGS, SYM>(), max_splits);
}

// The product `p` (extents, operands) with epilogue `epi` by `plan`; pieces of split tiles in `room`
// (piece_bytes of the plan).
template <class T, int A_KM, int B_KM, int GATED, int SEGS, int SYM, class Epi>
int run_product(Problem p, Plan plan, const Epi& epi, int batch, void* room, Arrivals& arrivals, hipStream_t stream, int compute_units, const char* what) {
  if (plan.splits > 1 && !arrivals.ready) {
    const Plan whole = plan_for<T, A_KM, B_KM, GATED, SEGS, SYM>(p.M_out, p.N_out, p.K, batch, compute_units, 1);
    if (whole.time < plan.time + kClearLaunch) plan = whole;
  }
  PT_TRY(take_plan(p, plan, room, arrivals, stream));
  switch (plan.tile) {
    case 0: return launch_tile<0, T, A_KM, B_KM, GATED, SEGS, SYM>(p, epi, batch, stream, what);
    case 1: return launch_tile<1, T, A_KM, B_KM, GATED, SEGS, SYM>(p, epi, batch, stream, what);
    case 2: return launch_tile<2, T, A_KM, B_KM, GATED, SEGS, SYM>(p, epi, batch, stream, what);
    case 3: return launch_tile<3, T, A_KM, B_KM, GATED, SEGS, SYM>(p, epi, batch, stream, what);
    default: break;
  }
  if constexpr (tiles_end<A_KM, B_KM, SEGS, SYM>() > kFewRowsTile) return launch_tile<kFewRowsTile, T, A_KM, B_KM, GATED, SEGS, SYM>(p, epi, batch, stream, what);
  else return RL_OK;
}

}  // namespace product

#endif
