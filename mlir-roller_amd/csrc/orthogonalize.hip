// Newton-Schulz orthogonalisation of a matrix or a stack of them:
//   X0 = G / (||G||_F + eps);   A = X X^T, B = b A + c A^2, X <- a X + B X   (steps times);   O = scale X
// with X the shorter side by the longer one (a tall G is worked on transposed).  A, A^2 and B are symmetric:
// only the tiles on and below the diagonal are computed, and those below it leave twice.
//
// Precision.  The iteration multiplies the small directions of X by a (3.4 by default) in every step, and
// with them the rounding errors of what is multiplied: with bf16 operands the result is 1 to 20 % off, in
// 16-bit bf16 outputs that can hold 0.17 %.  So X is kept in fp32, and
//   * bf16 matrices: the operands of the products are fp16 (11 bits instead of 8; |X| and |A| are bounded, so
//     the range does not matter), and the diagonals of A and B, the one place where A and B are not small
//     and whose errors add up along the rows of X, never pass through them:
//       (A^2)_ij = (Ao^2)_ij + (D_i + D_j) Ao_ij + [i = j] D_i^2      Ao = A without its diagonal D
//       X <- (a + diag(B)) X + Bo X                                    Bo = B without its diagonal
//     which leaves an error of 0.02 to 0.1 % of the norm, under the rounding of the output.
//   * fp16 and fp32 matrices: the products run on fp32 operands.
#include "product_launch.h"
#include "roller_ortho.h"

namespace {

using namespace product;

// fp16 operands are scaled by 2^8: entries of a normalised X of n columns are around n^-1/2, and what is
// below 2^-14 would lose bits as a subnormal.
template <class Op> constexpr float kScale = sizeof(Op) == 2 ? 256.0f : 1.0f;

// ---- norm and first X -------------------------------------------------------------------------------

constexpr int NORM_BLOCKS = 256;

template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* G, int ld, long stride, int rows, int cols, double* partial, unsigned* clear, int n_clear) {
  if (blockIdx.y == 0)   // the arrival counters of the first product
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n_clear; i += gridDim.x * 256) clear[i] = 0;
  const T* g = G + blockIdx.y * stride;
  double sum = 0.0;   // (fp64: squares of entries beyond 1.8e19 overflow fp32)
  for (long r = blockIdx.x * 4L + threadIdx.x / 64; r < rows; r += gridDim.x * 4L)   // 64 lanes per row
    for (int c = threadIdx.x % 64; c < cols; c += 64) {
      const double v = (double)(float)g[r * ld + c];
      sum += v * v;
    }
  __shared__ double sums[256];
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int w = 128; w > 0; w /= 2) {
    if ((int)threadIdx.x < w) sums[threadIdx.x] += sums[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) partial[blockIdx.y * gridDim.x + blockIdx.x] = sums[0];
}

// X0 in fp32 and as an operand, 64 x 64 elements per workgroup, transposed if G is tall; zeros behind the
// rows' ends up to whole chunks.
template <class T, class Op>
__global__ __launch_bounds__(256) void first_kernel(const T* G, int ld, long stride, int tall, const double* partial, int n_partial, float eps, int s, int l, int l8, int pitch, long x_stride, float* X, Op* Xop) {
  __shared__ double total[256];
  __shared__ float patch[64][65];
  const int t = threadIdx.x;
  total[t] = t < n_partial ? partial[blockIdx.z * n_partial + t] : 0.0;
  __syncthreads();
  for (int w = 128; w > 0; w /= 2) {
    if (t < w) total[t] += total[t + w];
    __syncthreads();
  }
  const float norm = (float)sqrt(total[0]) + eps;
  const T* g = G + blockIdx.z * stride;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  if (tall) {
    for (int i = t / 64; i < 64; i += 4) {
      const int c = c0 + i, r = r0 + t % 64;   // element (r, c) of X is G[c][r]
      patch[t % 64][i] = c < l && r < s ? (float)g[(long)c * ld + r] : 0.0f;
    }
    __syncthreads();
  }
  for (int i = t / 64; i < 64; i += 4) {
    const int r = r0 + i, c = c0 + t % 64;
    if (r >= s || c >= l8) continue;
    float v = tall ? patch[i][t % 64] : c < l ? (float)g[(long)r * ld + c] : 0.0f;
    v = v / norm;
    const long at = blockIdx.z * x_stride + (long)r * pitch + c;
    X[at] = v;
    if constexpr (sizeof(Op) == 2) Xop[at] = (Op)(v * kScale<Op>);
  }
}

// O = scale X for a tall matrix: the transpose of X, 64 x 64 elements per workgroup.
template <class T>
__global__ __launch_bounds__(256) void transposed_out_kernel(const float* X, int s, int l, int pitch, long x_stride, float scale, T* O, int ldo, long stride) {
  __shared__ float patch[64][65];
  const int t = threadIdx.x, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  for (int i = t / 64; i < 64; i += 4)
    if (r0 + i < s && c0 + t % 64 < l) patch[i][t % 64] = X[blockIdx.z * x_stride + (long)(r0 + i) * pitch + c0 + t % 64];
  __syncthreads();
  for (int i = t / 64; i < 64; i += 4)
    if (c0 + i < l && r0 + t % 64 < s) O[blockIdx.z * stride + (long)(c0 + i) * ldo + r0 + t % 64] = (T)(patch[t % 64][i] * scale);
}

// O = scale X without a step (steps = 0), and for a wide matrix whose last step ran elsewhere.
template <class T>
__global__ __launch_bounds__(256) void out_kernel(const float* X, int s, int l, int pitch, long x_stride, float scale, T* O, int ldo, long stride) {
  const float* x = X + blockIdx.z * x_stride;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)s * l; i += gridDim.x * 256L)
    O[blockIdx.z * stride + i / l * ldo + i % l] = (T)(x[i / l * pitch + i % l] * scale);
}

// ---- epilogues --------------------------------------------------------------------------------------

// Both halves of a symmetric matrix without its diagonal, and the diagonal: the buffers that one product
// writes and the next ones read.
template <class Op>
struct Symmetric {
  Op* off;        // [rows][pitch]
  float* diag;    // [pitch]
  int rows, pitch;
  __device__ __forceinline__ Symmetric of(int batch) const {
    Symmetric o = *this;
    o.off += (long)batch * rows * pitch;
    o.diag += (long)batch * pitch;
    return o;
  }
  __device__ __forceinline__ void put(int m, int n, v4f v, bool ok) const {
    v4f x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (ok && m == n + e) diag[m] = v[e];
      x[e] = m == n + e ? 0.0f : v[e] * kScale<Op>;
    }
    if (ok) store4(off + (long)m * pitch + n, x);
  }
};

// A = X X^T
template <class Op>
struct Gram {
  Symmetric<Op> A;
  __device__ __forceinline__ Gram at(int batch) const { return {A.of(batch)}; }
  struct In {};
  __device__ __forceinline__ In get(int, int) const { return {}; }
  __device__ __forceinline__ void put(int m, int n, v4f v, In, bool ok) const { A.put(m, n, v * (1.0f / (kScale<Op> * kScale<Op>)), ok); }
};

// B = b A + c A^2, from the product of Ao with itself
template <class Op>
struct Polynomial {
  Symmetric<Op> A, B;
  float b, c;
  __device__ __forceinline__ Polynomial at(int batch) const { return {A.of(batch), B.of(batch), b, c}; }
  struct In {
    v4f ao, dn;
    float dm;
  };
  __device__ __forceinline__ In get(int m, int n) const { return {load4(A.off + (long)m * A.pitch + n), *(const v4f*)(A.diag + n), A.diag[m]}; }
  __device__ __forceinline__ void put(int m, int n, v4f v, In in, bool ok) const {
    const v4f ao = in.ao * (1.0f / kScale<Op>), dn = in.dn;
    const float dm = in.dm;
    v4f x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float sq = v[e] * (1.0f / (kScale<Op> * kScale<Op>));
      x[e] = m == n + e ? b * dm + c * (sq + dm * dm) : b * ao[e] + c * (sq + (dm + dn[e]) * ao[e]);
    }
    B.put(m, n, x, ok);
  }
};

// X <- (a + diag(B)) X + Bo X; the last step of a wide matrix writes the output instead
template <class T, class Op>
struct Update {
  const float *from, *diag;
  float* to;
  Op* op;
  int pitch, diag_pitch;
  long stride;
  float a, scale;
  T* out;         // NULL: X goes on
  int ldo, l, vec;
  long out_stride;
  __device__ __forceinline__ Update at(int batch) const {
    Update o = *this;
    o.from += batch * stride;
    o.to += batch * stride;
    if (o.op) o.op += batch * stride;
    if (o.out) o.out += batch * out_stride;
    o.diag += (long)batch * diag_pitch;
    return o;
  }
  struct In {
    v4f x;
    float d;
  };
  __device__ __forceinline__ In get(int m, int n) const { return {*(const v4f*)(from + (long)m * pitch + n), diag[m]}; }
  __device__ __forceinline__ void put(int m, int n, v4f v, In in, bool ok) const {
    const long i = (long)m * pitch + n;
    const v4f x = in.x * (a + in.d) + v * (1.0f / (kScale<Op> * kScale<Op>));
    if (!ok) return;
    if (out) {
      T* o = out + (long)m * ldo + n;
      if (vec && n + 3 < l) {
        store4(o, x * scale);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < l) o[e] = (T)(x[e] * scale);
      }
      return;
    }
    *(v4f*)(to + i) = x;
    if constexpr (sizeof(Op) == 2) store4(op + i, x * kScale<Op>);
  }
};

// ---- host -------------------------------------------------------------------------------------------

struct Room {
  float* x[2];     // X in fp32 (fp32 operands: the two take turns; fp16: the first)
  half_t* op[2];   // X as an operand, taking turns (fp16 operands)
  void *ao, *bo;
  float *da, *db;
  double* partial;
  char *arrivals, *pieces;
  int s, l;        // sides of X
  int l8, s8;      // the same up to whole chunks: columns written
  int pitch, sq;   // elements from row to row of X, and of A and B
  size_t bytes;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

template <class Op>
Room carve(const OrthoCall& c) {
  Room r = {};
  char* base = c.room;
  size_t used = 0;
  auto take = [&](size_t n) {
    char* p = base ? base + used : nullptr;
    used += up256(n);
    return p;
  };
  r.s = c.rows < c.cols ? c.rows : c.cols;
  r.l = c.rows < c.cols ? c.cols : c.rows;
  r.l8 = (r.l + 7) / 8 * 8;
  r.s8 = (r.s + 7) / 8 * 8;
  r.pitch = line_pitch(sizeof(Op), r.l);
  r.sq = line_pitch(sizeof(Op), r.s);
  const size_t x = (size_t)c.batch * r.s * r.pitch, q = (size_t)c.batch * r.s8 * r.sq;
  r.x[0] = (float*)take(x * 4);
  if (sizeof(Op) == 2) {
    r.op[0] = (half_t*)take(x * 2);
    r.op[1] = (half_t*)take(x * 2);
  } else {
    r.x[1] = (float*)take(x * 4);
  }
  r.ao = take(q * sizeof(Op));
  r.bo = take(q * sizeof(Op));
  r.da = (float*)take((size_t)c.batch * r.sq * 4);
  r.db = (float*)take((size_t)c.batch * r.sq * 4);
  r.partial = (double*)take((size_t)c.batch * NORM_BLOCKS * 8);
  const size_t gram = plan_product(sizeof(Op), 0, 1, 1, r.s8, r.s8, r.l, c.batch, c.compute_units).piece_bytes;
  const size_t poly = plan_product(sizeof(Op), 0, 1, 1, r.s8, r.s8, r.s, c.batch, c.compute_units).piece_bytes;
  const size_t update = plan_product(sizeof(Op), 0, 1, 0, r.s, r.l8, r.s, c.batch, c.compute_units).piece_bytes;
  size_t pieces = gram > poly ? gram : poly;
  pieces = pieces > update ? pieces : update;
  r.arrivals = take(kArrivalBytes);
  r.pieces = take(pieces);
  r.bytes = used;
  return r;
}

template <class T, class Op>
int run(const OrthoCall& c) {
  const Room r = carve<Op>(c);
  const int tall = c.rows > c.cols;
  const long x_stride = (long)r.s * r.pitch;
  Arrivals arrivals = arrivals_at(r.arrivals, true);   // (by norm_kernel)
  const int blocks = c.rows < 4 * NORM_BLOCKS ? (c.rows + 3) / 4 : NORM_BLOCKS;
  PT_TRY(launch(norm_kernel<T>, "orthogonalize: norm", dim3(blocks, c.batch), 256, c.stream, (const T*)c.g, c.ldg, c.stride_g, c.rows, c.cols, r.partial, arrivals.set[0], kMaxArrivals));
  PT_TRY(launch(first_kernel<T, Op>, "orthogonalize: first X", dim3((r.l8 + 63) / 64, (r.s + 63) / 64, c.batch), 256, c.stream, (const T*)c.g, c.ldg, c.stride_g, tall, (const double*)r.partial, blocks, c.eps,
                r.s, r.l, r.l8, r.pitch, x_stride, r.x[0], (Op*)r.op[0]));
  const int vec = (uintptr_t)c.o % (4 * sizeof(T)) == 0 && c.ldo % 4 == 0 && c.stride_o % 4 == 0;
  int cur = 0;
  for (int k = 0; k < c.steps; ++k) {
    const float *coefficients = c.coefficients + 3 * k, a = coefficients[0], b = coefficients[1], cc = coefficients[2];
    const bool last = k + 1 == c.steps && !tall;
    const Op* x = sizeof(Op) == 2 ? (const Op*)r.op[cur] : (const Op*)r.x[cur];
    Problem p = {};
    p.a[0] = p.b[0] = x;
    p.lda = p.ldb = p.ldb1 = r.pitch;
    p.M = p.N = r.s;
    p.M_out = p.N_out = r.s8;
    p.K = r.l;
    p.batch_a = p.batch_b = x_stride;
    Symmetric<Op> A = {(Op*)r.ao, r.da, r.s8, r.sq}, B = {(Op*)r.bo, r.db, r.s8, r.sq};
    PT_TRY((run_product<Op, 1, 1, 0, 1, 1>(p, Gram<Op>{A}, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: X X^T")));
    p.a[0] = p.b[0] = r.ao;
    p.lda = p.ldb = p.ldb1 = r.sq;
    p.K = r.s;
    p.batch_a = p.batch_b = (long)r.s8 * r.sq;
    PT_TRY((run_product<Op, 1, 1, 0, 1, 1>(p, Polynomial<Op>{A, B, b, cc}, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: A A")));
    const int next = 1 - cur;
    Update<T, Op> u = {};
    u.from = sizeof(Op) == 2 ? r.x[0] : r.x[cur];
    u.to = sizeof(Op) == 2 ? r.x[0] : r.x[next];
    u.op = (Op*)r.op[next];
    u.diag = r.db;
    u.pitch = r.pitch;
    u.diag_pitch = r.sq;
    u.stride = x_stride;
    u.a = a;
    u.scale = c.scale;
    u.out = last ? (T*)c.o : nullptr;
    u.ldo = c.ldo;
    u.l = r.l;
    u.vec = vec;
    u.out_stride = c.stride_o;
    p.a[0] = r.bo;
    p.b[0] = x;
    p.ldb = p.ldb1 = r.pitch;
    p.N = r.l;
    p.M_out = r.s;
    p.N_out = r.l8;
    p.batch_b = x_stride;
    PT_TRY((run_product<Op, 1, 0, 0, 1, 0>(p, u, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: B X")));
    cur = next;
  }
  const float* x = sizeof(Op) == 2 ? r.x[0] : r.x[cur];
  if (tall)
    return launch(transposed_out_kernel<T>, "orthogonalize: output", dim3((r.l + 63) / 64, (r.s + 63) / 64, c.batch), 256, c.stream, x, r.s, r.l, r.pitch, x_stride, c.scale, (T*)c.o, c.ldo, c.stride_o);
  if (c.steps == 0)
    return launch(out_kernel<T>, "orthogonalize: output", dim3(blocks_for((long)r.s * r.l), 1, c.batch), 256, c.stream, x, r.s, r.l, r.pitch, x_stride, c.scale, (T*)c.o, c.ldo, c.stride_o);
  return RL_OK;
}

}  // namespace

size_t rl_ortho_room(const OrthoCall& c) { return c.dtype == RL_BF16 ? carve<half_t>(c).bytes : carve<float>(c).bytes; }

int rl_ortho_run(const OrthoCall& c) {
  if (c.dtype == RL_BF16) return run<bf16_t, half_t>(c);
  if (c.dtype == RL_F16) return run<half_t, float>(c);
  return run<float, float>(c);
}
