// The feed-forward block between its C entry points (roller_products.cpp) and its kernels (ffn.hip, one
// object per element type).  Internal to libroller_hip.so.
#ifndef ROLLER_FFN_H
#define ROLLER_FFN_H

#include <hip/hip_runtime_api.h>

#include <cstddef>

#include "product_plan.h"

struct FfnMatrix {
  const void* p;
  int ld;
};

struct FfnCall {
  int activation, T, D, F;
  FfnMatrix x, w_gate, w_up, w_down;   // inputs
  FfnMatrix dy;                        // backward
  void *y, *dx, *dw_gate, *dw_up, *dw_down;   // outputs; gradients may be NULL
  int ldy, ld_dx, ld_dw_gate, ld_dw_up, ld_dw_down;
  void* saved;                         // forward: may be NULL
  char* room;
  hipStream_t stream;
  int compute_units;
};

// Bytes of the three kept buffers (h in the element type, g and u in fp32), each T x pitch.
struct FfnSaved {
  int pitch;               // elements from row to row
  size_t h, g, u, total;   // offsets
};
inline size_t ffn_round(size_t n) { return (n + 255) / 256 * 256; }
inline FfnSaved ffn_saved(int es, int T, int F) {
  FfnSaved s;
  s.pitch = product::line_pitch(es, F);
  const size_t n = (size_t)T * s.pitch;
  s.h = 0;
  s.g = ffn_round(n * es);
  s.u = s.g + ffn_round(n * 4);
  s.total = s.u + ffn_round(n * 4);
  return s;
}

// One set of functions per element type.  `room` sizes count packed copies only where the call needs them:
// the matrices of `c` decide (pointers and leading dimensions; for a size question with `unaligned`, all).
struct FfnType {
  void (*plans)(const FfnCall& c, product::Plan out[6]);   // gate and up, down, dw_down, dh, dx, dw_gate and dw_up
  size_t (*forward_room)(const FfnCall& c, bool unaligned);
  size_t (*backward_room)(const FfnCall& c, bool unaligned);
  int (*forward)(const FfnCall& c);
  int (*backward)(const FfnCall& c);
};
__attribute__((visibility("hidden"))) FfnType rl_ffn_f32();
__attribute__((visibility("hidden"))) FfnType rl_ffn_f16();
__attribute__((visibility("hidden"))) FfnType rl_ffn_bf16();

#endif
