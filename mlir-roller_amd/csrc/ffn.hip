// The gated feed-forward block, for one element type (FFN_TYPE 0: fp32, 1: fp16, 2: bf16).
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T                        x[T,D], Wg[F,D], Wu[F,D], Wd[D,F]
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Two products forward (gate and up share their operand x and come out of one kernel, which also makes h)
// and four backward (dh with dg and du made on the accumulators; dx as one sum over both pairs; dWg and dWu
// as the two batch entries of one launch; dWd).  h, dg and du are rounded once to the element type, since
// the next product's matrix instructions read that type (in fp16 dg and du times a power of two, product_ops.h);
// everything else between the inputs and the outputs is fp32, g and u included, which the forward pass keeps for the
// backward pass.
//
// With up to 16 tokens the forward pass does little but read the weights; it takes few_rows_kernel instead of
// the tile engine, and with 16-bit types h stays in fp32 there (the second product splits it in two).
#include "product_launch.h"
#include "roller_ffn.h"

namespace {

using namespace product;

#if FFN_TYPE == 0
typedef float T;
#define FFN_TABLE rl_ffn_f32
#elif FFN_TYPE == 1
typedef half_t T;
#define FFN_TABLE rl_ffn_f16
#else
typedef bf16_t T;
#define FFN_TABLE rl_ffn_bf16
#endif

constexpr int ES = sizeof(T), PER = 16 / ES;
constexpr int FEW = 16;       // tokens up to which the forward products take few_rows_kernel,
constexpr int FEW_ODD = 64;   // and with rows at odd places, which the tile engine would need packed copies of
constexpr int EXACT_TOKENS = ES == 2 ? FEW : 0;   // tokens up to which h goes into the second product unrounded

int pitch_of(int n) { return line_pitch(ES, n); }

// The tile engine loads dword-aligned rows; 16-bit rows at odd places are packed first, or with few tokens
// multiplied by few_rows_kernel.
bool aligned(const FfnMatrix& m) { return (uintptr_t)m.p % 4 == 0 && (long)m.ld * ES % 4 == 0; }

class Carver {
 public:
  explicit Carver(char* base) : base_(base) {}
  char* take(size_t bytes) {
    char* p = base_ ? base_ + used_ : nullptr;
    used_ += ffn_round(bytes);
    return p;
  }
  size_t used() const { return used_; }

 private:
  char* base_;
  size_t used_ = 0;
};

// Space for a packed copy, if one is needed.
T* pack_space(Carver& room, int rows, int cols, bool need) {
  return need ? (T*)room.take((size_t)rows * pitch_of(cols) * ES) : nullptr;
}

int pack(FfnMatrix& m, int rows, int cols, T* space, hipStream_t stream) {
  if (!space) return RL_OK;
  const int pitch = pitch_of(cols);
  PT_TRY(launch<pack_kernel<T>>("packing an operand", dim3(blocks_for((long)rows * (pitch / PER))), 256, stream, (const T*)m.p, m.ld, rows, cols, space, pitch));
  m = {space, pitch};
  return RL_OK;
}

int vec_ok(const void* p, int ld) { return (uintptr_t)p % (4 * ES) == 0 && ld % 4 == 0; }

template <int SCALED = 0>
Store<T, SCALED> store(void* c, int ldc, int N) {
  Store<T, SCALED> s = {};
  s.c[0] = s.c[1] = (T*)c;
  s.ldc = s.ldc1 = ldc;
  s.N = N;
  s.vec = vec_ok(c, ldc);
  return s;
}

Problem problem(const void* a, int lda, const void* b, int ldb, int M, int N, int K, int M_out, int N_out) {
  Problem p = {};
  p.a[0] = a;
  p.b[0] = b;
  p.lda = lda;
  p.ldb = p.ldb1 = ldb;
  p.M = M;
  p.N = N;
  p.K = K;
  p.M_out = M_out;
  p.N_out = N_out;
  return p;
}

size_t larger(size_t a, size_t b) { return a > b ? a : b; }

Plan plan_up(const FfnCall& c) { return plan_for<T, 1, 1, 1, 1, 0>(c.T, c.F, c.D, 1, c.compute_units); }
Plan plan_down(const FfnCall& c) { return plan_for<T, 1, 1, 0, 1, 0>(c.T, c.D, c.F, 1, c.compute_units); }
Plan plan_dw_down(const FfnCall& c) { return plan_for<T, 0, 0, 0, 1, 0>(c.D, c.F, c.T, 1, c.compute_units); }
Plan plan_dh(const FfnCall& c) { return plan_for<T, 1, 0, 0, 1, 0>(c.T, c.F, c.D, 1, c.compute_units); }
Plan plan_dx(const FfnCall& c) { return plan_for<T, 1, 0, 0, 2, 0>(c.T, c.D, c.F, 1, c.compute_units); }
Plan plan_dw(const FfnCall& c) { return plan_for<T, 0, 0, 0, 1, 0>(c.F, c.D, c.T, 2, c.compute_units); }

void plans(const FfnCall& c, Plan out[6]) {
  out[0] = plan_up(c);
  out[1] = plan_down(c);
  out[2] = plan_dw_down(c);
  out[3] = plan_dh(c);
  out[4] = plan_dx(c);
  out[5] = plan_dw(c);
}

// ---- forward ----

struct ForwardRoom {
  T *x, *w_gate, *w_up, *w_down, *h;
  float* h32;
  char *arrivals, *pieces;
  Plan up, down;
  bool few_up, few_down;   // takes few_rows_kernel
  size_t bytes;
};

ForwardRoom forward_carve(const FfnCall& c, bool unaligned) {
  Carver room(c.room);
  ForwardRoom r = {};
  const FfnSaved s = ffn_saved(ES, c.T, c.F);
  r.few_up = c.T <= FEW || (c.T <= FEW_ODD && !(aligned(c.x) && aligned(c.w_gate) && aligned(c.w_up)));
  r.few_down = c.T <= FEW || (c.T <= FEW_ODD && !aligned(c.w_down));
  if (c.T <= EXACT_TOKENS) {
    r.h32 = (float*)room.take((size_t)c.T * s.pitch * 4);
  } else if (!c.saved) {
    r.h = (T*)room.take((size_t)c.T * s.pitch * ES);
  }
  // (with 17 to 64 tokens the same room whatever the alignment, which a query does not know)
  if (c.T > FEW) {
    const bool pack = c.T > FEW_ODD;
    r.x = pack_space(room, c.T, c.D, pack && (unaligned || !aligned(c.x)));
    r.w_gate = pack_space(room, c.F, c.D, pack && (unaligned || !aligned(c.w_gate)));
    r.w_up = pack_space(room, c.F, c.D, pack && (unaligned || !aligned(c.w_up)));
    r.w_down = pack_space(room, c.D, c.F, pack && (unaligned || !aligned(c.w_down)));
    r.arrivals = room.take(kArrivalBytes);
    r.up = plan_up(c);
    r.down = plan_down(c);
    r.pieces = room.take(larger(r.up.piece_bytes, r.down.piece_bytes));
  }
  r.bytes = room.used();
  return r;
}

// A product of few tokens: x (SPLIT: in fp32) with the rows of w0, GATED: and w1.
template <int GATED, int SPLIT, class Epi>
int few_rows(const FfnCall& c, const void* x, int ldx, const FfnMatrix& w0, const FfnMatrix& w1, int N, int K, const Epi& epi, const char* what) {
  auto as = [&](auto blocks, auto parts) -> int {
    constexpr int BLOCKS = decltype(blocks)::value, PARTS = decltype(parts)::value, ROWS = 16 / PARTS;
    const int groups = (N + ROWS - 1) / ROWS;
    // Enough waves to keep the memory busy from every CU: up to 16 share the K of a workgroup's rows, none with
    // fewer than 256 bytes of each part of a row.
    int waves = 1;
    while (waves < 16 && (long)groups * waves < 16L * c.compute_units && K / PARTS * ES >= 512 * waves) waves *= 2;
    return launch<few_rows_kernel<T, BLOCKS, PARTS, GATED, SPLIT, Epi>>(what, dim3(groups), 64 * waves, c.stream, (const typename x_type<T, SPLIT>::type*)x, ldx, (const T*)w0.p, w0.ld, (const T*)w1.p, w1.ld, c.T,
                                                                        N, K, epi);
  };
  if (c.T <= 4) return as(int_c<1>{}, int_c<4>{});
  if (c.T <= 8) return as(int_c<1>{}, int_c<2>{});
  if (c.T <= 16) return as(int_c<1>{}, int_c<1>{});
  if constexpr (SPLIT) return RL_ERR_INTERNAL;   // (no more than EXACT_TOKENS)
  else return c.T <= 32 ? as(int_c<2>{}, int_c<1>{}) : as(int_c<4>{}, int_c<1>{});
}

size_t forward_room(const FfnCall& c, bool unaligned) { return forward_carve(c, unaligned).bytes; }

template <int KIND>
int forward_as(const FfnCall& call) {
  FfnCall c = call;
  const ForwardRoom r = forward_carve(c, false);
  const FfnSaved s = ffn_saved(ES, c.T, c.F);
  GatedForward<T, KIND> gated = {};
  gated.h = c.saved ? (T*)((char*)c.saved + s.h) : r.h;
  gated.g = c.saved ? (float*)((char*)c.saved + s.g) : nullptr;
  gated.u = c.saved ? (float*)((char*)c.saved + s.u) : nullptr;
  gated.pitch = s.pitch;
  const Store<T> out = store(c.y, c.ldy, c.D);
  gated.h32 = r.h32;
  PT_TRY(pack(c.x, c.T, c.D, r.x, c.stream));
  PT_TRY(pack(c.w_gate, c.F, c.D, r.w_gate, c.stream));
  PT_TRY(pack(c.w_up, c.F, c.D, r.w_up, c.stream));
  PT_TRY(pack(c.w_down, c.D, c.F, r.w_down, c.stream));
  Arrivals arrivals = arrivals_at(r.arrivals, false);
  if (r.few_up) {
    PT_TRY((few_rows<1, 0>(c, c.x.p, c.x.ld, c.w_gate, c.w_up, c.F, c.D, gated, "ffn: gate and up")));
  } else {
    Problem up = problem(c.x.p, c.x.ld, c.w_gate.p, c.w_gate.ld, c.T, c.F, c.D, c.T, c.F);
    up.b[1] = c.w_up.p;
    up.ldb1 = c.w_up.ld;
    PT_TRY((run_product<T, 1, 1, 1, 1, 0>(up, r.up, gated, 1, r.pieces, arrivals, c.stream, c.compute_units, "ffn: gate and up")));
  }
  if (r.few_down) {
    if constexpr (EXACT_TOKENS != 0) {
      if (r.h32) return few_rows<0, 1>(c, r.h32, s.pitch, c.w_down, {}, c.D, c.F, out, "ffn: down");
    }
    return few_rows<0, 0>(c, gated.h, s.pitch, c.w_down, {}, c.D, c.F, out, "ffn: down");
  }
  const Problem down = problem(gated.h, s.pitch, c.w_down.p, c.w_down.ld, c.T, c.D, c.F, c.T, c.D);
  return run_product<T, 1, 1, 0, 1, 0>(down, r.down, out, 1, r.pieces, arrivals, c.stream, c.compute_units, "ffn: down");
}

int forward(const FfnCall& c) {
  return c.activation == ACT_SILU ? forward_as<ACT_SILU>(c) : c.activation == ACT_GELU ? forward_as<ACT_GELU>(c) : forward_as<ACT_GELU_TANH>(c);
}

// ---- backward ----

struct BackwardRoom {
  T *dy, *x, *w_gate, *w_up, *w_down, *dg, *du;
  unsigned* peaks;   // of dy, fp16
  char *arrivals, *pieces;
  Plan dw_down, dh, dx, dw;   // (dw: gate and up)
  size_t bytes;
};

BackwardRoom backward_carve(const FfnCall& c, bool unaligned) {
  Carver room(c.room);
  BackwardRoom r = {};
  const FfnSaved s = ffn_saved(ES, c.T, c.F);
  const size_t n = (size_t)c.T * s.pitch * ES;
  // (dg and du directly behind each other: the two batch entries of one product)
  r.dg = (T*)room.take(2 * n);
  r.du = r.dg ? r.dg + (size_t)c.T * s.pitch : nullptr;
  r.dy = pack_space(room, c.T, c.D, unaligned || !aligned(c.dy));
  r.x = pack_space(room, c.T, c.D, unaligned || !aligned(c.x));
  // dx reads both weights with one leading dimension
  const bool weights = unaligned || !aligned(c.w_gate) || !aligned(c.w_up) || c.w_gate.ld != c.w_up.ld;
  r.w_gate = pack_space(room, c.F, c.D, weights);
  r.w_up = pack_space(room, c.F, c.D, weights);
  r.w_down = pack_space(room, c.D, c.F, unaligned || !aligned(c.w_down));
  if (is_scaled<T>()) r.peaks = (unsigned*)room.take(PEAKS * sizeof(unsigned));
  r.arrivals = room.take(kArrivalBytes);
  r.dw_down = plan_dw_down(c);
  r.dh = plan_dh(c);
  r.dx = plan_dx(c);
  r.dw = plan_dw(c);
  const size_t pieces = larger(larger(r.dw_down.piece_bytes, r.dh.piece_bytes), larger(r.dx.piece_bytes, r.dw.piece_bytes));
  r.pieces = room.take(pieces);
  r.bytes = room.used();
  return r;
}

size_t backward_room(const FfnCall& c, bool unaligned) { return backward_carve(c, unaligned).bytes; }

int zero(void* p, int ld, int rows, int cols, hipStream_t stream) {
  return launch<zero_kernel<T>>("ffn: zero gradient", dim3(blocks_for((long)rows * cols)), 256, stream, (T*)p, ld, rows, cols);
}

template <int KIND>
int gated_backward(const FfnCall& c, const BackwardRoom& r, const FfnSaved& s, const Problem& dh, Arrivals& arrivals) {
  GatedBackward<T, KIND> gated = {};
  gated.g = (const float*)((char*)c.saved + s.g);
  gated.u = (const float*)((char*)c.saved + s.u);
  gated.dg = r.dg;
  gated.du = r.du;
  gated.pitch = s.pitch;
  gated.peaks = r.peaks;
  return run_product<T, 1, 0, 0, 1, 0>(dh, r.dh, gated, 1, r.pieces, arrivals, c.stream, c.compute_units, "ffn: dh");
}

int backward(const FfnCall& call) {
  FfnCall c = call;
  if (c.T == 0) {   // no tokens: the gradients of the weights are zero
    if (c.dw_gate) PT_TRY(zero(c.dw_gate, c.ld_dw_gate, c.F, c.D, c.stream));
    if (c.dw_up) PT_TRY(zero(c.dw_up, c.ld_dw_up, c.F, c.D, c.stream));
    if (c.dw_down) PT_TRY(zero(c.dw_down, c.ld_dw_down, c.D, c.F, c.stream));
    return RL_OK;
  }
  const BackwardRoom r = backward_carve(c, false);
  const FfnSaved s = ffn_saved(ES, c.T, c.F);
  const T* h = (const T*)((char*)c.saved + s.h);
  const bool scaled = is_scaled<T>() && (c.dx || c.dw_gate);
  Arrivals arrivals = arrivals_at(r.arrivals, scaled);   // (cleared by peak_kernel)
  if constexpr (is_scaled<T>()) {
    if (scaled) {
      int lanes = 1;   // per row of dy, 16 bytes each
      while (lanes < 64 && lanes * PER < c.D) lanes *= 2;
      PT_TRY(launch<peak_kernel<T>>("ffn: largest gradient", dim3(PEAKS), 256, c.stream, (const T*)c.dy.p, c.dy.ld, c.T, c.D, lanes, r.peaks, arrivals.set[0], kMaxArrivals));
    }
  }
  PT_TRY(pack(c.dy, c.T, c.D, r.dy, c.stream));
  if (c.dw_down) {
    const Problem p = problem(c.dy.p, c.dy.ld, h, s.pitch, c.D, c.F, c.T, c.D, c.F);
    PT_TRY((run_product<T, 0, 0, 0, 1, 0>(p, r.dw_down, store(c.dw_down, c.ld_dw_down, c.F), 1, r.pieces, arrivals, c.stream, c.compute_units, "ffn: dw_down")));
  }
  if (!c.dx && !c.dw_gate) return RL_OK;
  PT_TRY(pack(c.w_down, c.D, c.F, r.w_down, c.stream));
  const Problem dh = problem(c.dy.p, c.dy.ld, c.w_down.p, c.w_down.ld, c.T, c.F, c.D, c.T, c.F);
  switch (c.activation) {
    case ACT_SILU: PT_TRY(gated_backward<ACT_SILU>(c, r, s, dh, arrivals)); break;
    case ACT_GELU: PT_TRY(gated_backward<ACT_GELU>(c, r, s, dh, arrivals)); break;
    default: PT_TRY(gated_backward<ACT_GELU_TANH>(c, r, s, dh, arrivals)); break;
  }
  if (c.dx) {
    PT_TRY(pack(c.w_gate, c.F, c.D, r.w_gate, c.stream));
    PT_TRY(pack(c.w_up, c.F, c.D, r.w_up, c.stream));
    Problem p = problem(r.dg, s.pitch, c.w_gate.p, c.w_gate.ld, c.T, c.D, c.F, c.T, c.D);
    p.a[1] = r.du;
    p.b[1] = c.w_up.p;
    auto out = store<is_scaled<T>()>(c.dx, c.ld_dx, c.D);
    out.peaks = r.peaks;
    PT_TRY((run_product<T, 1, 0, 0, 2, 0>(p, r.dx, out, 1, r.pieces, arrivals, c.stream, c.compute_units, "ffn: dx")));
  }
  if (c.dw_gate) {
    PT_TRY(pack(c.x, c.T, c.D, r.x, c.stream));
    Problem p = problem(r.dg, s.pitch, c.x.p, c.x.ld, c.F, c.D, c.T, c.F, c.D);
    p.batch_a = (long)c.T * s.pitch;
    auto out = store<is_scaled<T>()>(c.dw_gate, c.ld_dw_gate, c.D);
    out.c[1] = (T*)c.dw_up;
    out.ldc1 = c.ld_dw_up;
    out.peaks = r.peaks;
    out.vec = out.vec && vec_ok(c.dw_up, c.ld_dw_up);
    PT_TRY((run_product<T, 0, 0, 0, 1, 0>(p, r.dw, out, 2, r.pieces, arrivals, c.stream, c.compute_units, "ffn: dw_gate and dw_up")));
  }
  return RL_OK;
}

}  // namespace

FfnType FFN_TABLE() { return {plans, forward_room, backward_room, forward, backward}; }
