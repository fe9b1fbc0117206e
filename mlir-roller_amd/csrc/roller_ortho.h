// Newton-Schulz orthogonalisation between its C entry points (roller_products.cpp) and its kernels
// (orthogonalize.hip).  Internal to libroller_hip.so.
#ifndef ROLLER_ORTHO_H
#define ROLLER_ORTHO_H

#include <hip/hip_runtime_api.h>

#include <cstddef>

#include "product_plan.h"

struct OrthoCall {
  int dtype, rows, cols, batch, steps;
  const float* coefficients;   // steps x (a, b, c), host memory
  float eps, scale;
  const void* g;
  void* o;
  int ldg, ldo;
  long stride_g, stride_o;
  char* room;
  hipStream_t stream;
  int compute_units;
};

__attribute__((visibility("hidden"))) size_t rl_ortho_room(const OrthoCall& c);
__attribute__((visibility("hidden"))) void rl_ortho_plans(const OrthoCall& c, product::Plan out[3]);
__attribute__((visibility("hidden"))) int rl_ortho_run(const OrthoCall& c);

#endif
