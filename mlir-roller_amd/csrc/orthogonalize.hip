// Newton-Schulz orthogonalisation of a matrix or a stack of them:
//   X0 = G / (||G||_F + eps);   A = X X^T, B = b A + c A^2, X <- a X + B X   (steps times);   O = scale X
// with X the shorter side by the longer one (a tall G is worked on transposed).  A, A^2 and B are symmetric:
// only the tiles on and below the diagonal are computed, and those below it leave twice.
//
// Precision.  The iteration multiplies the small directions of X by a (3.4 by default) in every step, and
// with them the rounding errors of what is multiplied: with bf16 operands the result is 1 to 20 % off, in
// 16-bit bf16 outputs that can hold 0.17 %.  So X is kept in fp32, and the operands of the products are fp16
// (11 bits instead of 8; |X| and |A| are bounded, so the range does not matter):
//   * The diagonals of A and B, the one place where they are not small and whose errors add up along the rows
//     of X, never pass through 16 bits:
//       (A^2)_ij = (Ao^2)_ij + (D_i + D_j) Ao_ij + [i = j] D_i^2      Ao = A without its diagonal D
//       X <- (a + diag(B)) X + Bo X                                    Bo = B without its diagonal
//   * bf16 matrices: one fp16 number per operand element, which leaves an error of 0.02 to 0.1 % of the norm,
//     under the rounding of the output.
//   * fp16 and fp32 matrices: two, high part and remainder (22 bits), and three of their four products,
//     hi hi + hi lo + lo hi, as three segments of one K loop: an error of some 10^-6 of the norm (1.3e-6 at
//     509 x 1023; fp32 products in the plain form 2.4e-6), at a third of the fp16 rate instead of a sixteenth.
#include "product_launch.h"
#include "roller_ortho.h"

namespace {

using namespace product;

// Operands are scaled by 2^9: entries of a normalised X of n columns are around n^-1/2, and what is below
// 2^-14 (or a remainder below 2^-25) would lose bits as a subnormal.
typedef half_t Op;
constexpr float kScale = 512.0f, kUnscale = 1.0f / (kScale * kScale);

// Writes four elements of an operand: to[0 ..], and with two parts the remainders `parts` elements further on.
template <int PARTS>
PT_DEV void put_operand(Op* to, long parts, v4f v) {
  const v4f x = v * kScale;
  const typename vec4<Op>::type hi = round4<Op>(x);
  *(typename vec4<Op>::type*)to = hi;
  if constexpr (PARTS == 2) store4(to + parts, v4f{x[0] - (float)hi[0], x[1] - (float)hi[1], x[2] - (float)hi[2], x[3] - (float)hi[3]});
}
template <int PARTS>
PT_DEV v4f get_operand(const Op* at, long parts) {
  v4f v = load4(at);
  if constexpr (PARTS == 2) v += load4(at + parts);
  return v * (1.0f / kScale);
}

// ---- norm and first X -------------------------------------------------------------------------------

constexpr int NORM_BLOCKS = 256;   // (first_kernel adds up one partial sum per thread)

// Partial sums of squares: 16-byte loads, four at a time (4096 x 4096 in bf16: 12 us; element by element, 111).

template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* G, int ld, long stride, int rows, int cols, double* partial, unsigned* clear, int n_clear) {
  if (blockIdx.y == 0)   // the arrival counters of the first product
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n_clear; i += gridDim.x * 256) clear[i] = 0;
  const T* g = G + blockIdx.y * stride;
  constexpr int PER = 16 / sizeof(T), UNROLL = 4;
  typedef T chunk __attribute__((ext_vector_type(PER)));
  double part[PER] = {};   // (fp64: squares of entries beyond 1.8e19 overflow fp32)
  const int chunks = (cols + PER - 1) / PER;
  for (long r = blockIdx.x * 4L + threadIdx.x / 64; r < rows; r += gridDim.x * 4L)   // 64 lanes per row
    for (int c = threadIdx.x % 64; c < chunks; c += 64 * UNROLL) {
      chunk v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) v[u] = __builtin_bit_cast(chunk, chunk_at(g + r * ld, (c + 64 * u) * PER, cols));   // (zeros past the end)
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int e = 0; e < PER; ++e) part[e] += (double)(float)v[u][e] * (double)(float)v[u][e];
    }
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < PER; ++e) sum += part[e];
  __shared__ double sums[256];
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int w = 128; w > 0; w /= 2) {
    if ((int)threadIdx.x < w) sums[threadIdx.x] += sums[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) partial[blockIdx.y * gridDim.x + blockIdx.x] = sums[0];
}

// X0 in fp32 and as an operand, 64 x 64 elements per workgroup, transposed if G is tall; zeros behind
// the ends of rows and columns up to whole patches.
template <class T, int PARTS>
__global__ __launch_bounds__(256) void first_kernel(const T* G, int ld, long stride, int tall, const double* partial, int n_partial, float eps, int s, int l, int pitch, long x_stride, float* X, Op* Xop, long parts) {
  __shared__ double total[256];
  __shared__ float patch[64][65];
  const int t = threadIdx.x;
  total[t] = t < n_partial ? partial[blockIdx.z * n_partial + t] : 0.0;
  __syncthreads();
  for (int w = 128; w > 0; w /= 2) {
    if (t < w) total[t] += total[t + w];
    __syncthreads();
  }
  const double inv = 1.0 / (sqrt(total[0]) + (double)eps);   // (a norm beyond fp32 is no infinity here)
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
    float v = tall ? patch[i][t % 64] : c < l && r < s ? (float)g[(long)r * ld + c] : 0.0f;
    v = (float)((double)v * inv);
    const long at = blockIdx.z * x_stride + (long)r * pitch + c;
    X[at] = v;
    const Op hi = (Op)(v * kScale);
    Xop[at] = hi;
    if constexpr (PARTS == 2) Xop[parts + at] = (Op)(v * kScale - (float)hi);
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

// O = scale X without a step (steps = 0) for a matrix that is not tall; with steps the last one writes O.
template <class T>
__global__ __launch_bounds__(256) void out_kernel(const float* X, int s, int l, int pitch, long x_stride, float scale, T* O, int ldo, long stride) {
  const float* x = X + blockIdx.z * x_stride;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)s * l; i += gridDim.x * 256L)
    O[blockIdx.z * stride + i / l * ldo + i % l] = (T)(x[i / l * pitch + i % l] * scale);
}

// ---- epilogues --------------------------------------------------------------------------------------

// A symmetric matrix without its diagonal, and the diagonal: the buffers that one product writes and the next
// ones read.
template <int PARTS>
struct Symmetric {
  Op* off;        // [rows][pitch]
  float* diag;    // [pitch]
  int rows, pitch;
  long parts;     // from the high parts to the remainders
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
      x[e] = m == n + e ? 0.0f : v[e];
    }
    if (ok) put_operand<PARTS>(off + (long)m * pitch + n, parts, x);
  }
};

// A = X X^T
template <int PARTS>
struct Gram {
  Symmetric<PARTS> A;
  __device__ __forceinline__ Gram at(int batch) const { return {A.of(batch)}; }
  struct In {};
  __device__ __forceinline__ In get(int, int) const { return {}; }
  __device__ __forceinline__ v4f value(int, int, v4f v, In) const { return v * kUnscale; }
  __device__ __forceinline__ void put(int m, int n, v4f v, bool ok) const { A.put(m, n, v, ok); }
};

// B = b A + c A^2, from the product of Ao with itself
template <int PARTS>
struct Polynomial {
  Symmetric<PARTS> A, B;
  float b, c;
  __device__ __forceinline__ Polynomial at(int batch) const { return {A.of(batch), B.of(batch), b, c}; }
  struct In {
    v4f ao, dn;
    float dm;
  };
  __device__ __forceinline__ In get(int m, int n) const { return {get_operand<PARTS>(A.off + (long)m * A.pitch + n, A.parts), *(const v4f*)(A.diag + n), A.diag[m]}; }
  __device__ __forceinline__ v4f value(int m, int n, v4f v, In in) const {
    v4f x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float sq = v[e] * kUnscale;
      x[e] = m == n + e ? b * in.dm + c * (sq + in.dm * in.dm) : b * in.ao[e] + c * (sq + (in.dm + in.dn[e]) * in.ao[e]);
    }
    return x;
  }
  __device__ __forceinline__ void put(int m, int n, v4f v, bool ok) const { B.put(m, n, v, ok); }
};

// X <- (a + diag(B)) X + Bo X, in place (every element is read and written by one lane); the last step of a
// wide matrix writes the output instead
template <class T, int PARTS>
struct Update {
  float* x;
  const float* diag;
  Op* op;
  long parts;
  int pitch, diag_pitch;
  long stride;
  float a, scale;
  T* out;         // NULL: X goes on
  int ldo, s, l, vec;
  long out_stride;
  __device__ __forceinline__ Update at(int batch) const {
    Update o = *this;
    o.x += batch * stride;
    o.op += batch * stride;
    if (o.out) o.out += batch * out_stride;
    o.diag += (long)batch * diag_pitch;
    return o;
  }
  struct In {
    v4f x;
    float d;
  };
  __device__ __forceinline__ In get(int m, int n) const { return {*(const v4f*)(x + (long)m * pitch + n), diag[m]}; }
  __device__ __forceinline__ void put(int m, int n, v4f v, In in, bool ok) const {
    const long i = (long)m * pitch + n;
    const v4f y = in.x * (a + in.d) + v * kUnscale;
    if (!ok) return;
    if (out) {
      if (m >= s) return;
      T* o = out + (long)m * ldo + n;
      if (vec && n + 3 < l) {
        store4(o, y * scale);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < l) o[e] = (T)(y[e] * scale);
      }
      return;
    }
    *(v4f*)(x + i) = y;
    put_operand<PARTS>(op + i, parts, y);
  }
};

// ---- host -------------------------------------------------------------------------------------------

struct Room {
  float* x;        // X in fp32
  Op* op[2];       // X as an operand, taking turns
  Op *ao, *bo;
  float *da, *db;
  double* partial;
  char *arrivals, *pieces;
  Plan gram, poly, update;
  int s, l;        // sides of X
  int l64, s64;    // the same up to whole K steps: rows and columns that exist, zeros beyond s and l
  int pitch, sq;   // elements from row to row of X, and of A and B
  long x_parts, sq_parts;   // from the high parts of an operand to the remainders
  size_t bytes;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

template <int PARTS>
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
  r.l64 = (r.l + 63) / 64 * 64;
  r.s64 = (r.s + 63) / 64 * 64;
  r.pitch = line_pitch(sizeof(Op), r.l);
  r.sq = line_pitch(sizeof(Op), r.s);
  r.x_parts = (long)c.batch * r.s64 * r.pitch;
  r.sq_parts = (long)c.batch * r.s64 * r.sq;
  r.x = (float*)take((size_t)r.x_parts * 4);
  r.op[0] = (Op*)take((size_t)r.x_parts * sizeof(Op) * PARTS);
  r.op[1] = (Op*)take((size_t)r.x_parts * sizeof(Op) * PARTS);
  r.ao = (Op*)take((size_t)r.sq_parts * sizeof(Op) * PARTS);
  r.bo = (Op*)take((size_t)r.sq_parts * sizeof(Op) * PARTS);
  r.da = (float*)take((size_t)c.batch * r.sq * 4);
  r.db = (float*)take((size_t)c.batch * r.sq * 4);
  r.partial = (double*)take((size_t)c.batch * NORM_BLOCKS * 8);
  constexpr int SEGS = PARTS == 2 ? 3 : 1;
  r.gram = plan_for<Op, 1, 1, 0, SEGS, 1>(r.s64, r.s64, r.l64, c.batch, c.compute_units);
  r.poly = plan_for<Op, 1, 1, 0, SEGS, 1>(r.s64, r.s64, r.s64, c.batch, c.compute_units);
  r.update = plan_for<Op, 1, 0, 0, SEGS, 0>(r.s64, r.l64, r.s64, c.batch, c.compute_units);
  size_t pieces = r.gram.piece_bytes > r.poly.piece_bytes ? r.gram.piece_bytes : r.poly.piece_bytes;
  pieces = pieces > r.update.piece_bytes ? pieces : r.update.piece_bytes;
  r.arrivals = take(kArrivalBytes);
  r.pieces = take(pieces);
  r.bytes = used;
  return r;
}

// The operands a b^T of a product: with two parts the segments hi hi, hi lo, lo hi.
template <int PARTS>
Problem problem(const Op* a, long a_parts, int lda, const Op* b, long b_parts, int ldb) {
  Problem p = {};
  p.a[0] = a;
  p.b[0] = b;
  if (PARTS == 2) {
    p.a[1] = a;
    p.b[1] = b + b_parts;
    p.a[2] = a + a_parts;
    p.b[2] = b;
  }
  p.lda = lda;
  p.ldb = p.ldb1 = ldb;
  return p;
}

template <class T, int PARTS>
int run(const OrthoCall& c) {
  constexpr int SEGS = PARTS == 2 ? 3 : 1;
  const Room r = carve<PARTS>(c);
  const int tall = c.rows > c.cols;
  const long x_stride = (long)r.s64 * r.pitch;
  Arrivals arrivals = arrivals_at(r.arrivals, true);   // (by norm_kernel)
  const int blocks = c.rows < 4 * NORM_BLOCKS ? (c.rows + 3) / 4 : NORM_BLOCKS;
  PT_TRY(launch<norm_kernel<T>>("orthogonalize: norm", dim3(blocks, c.batch), 256, c.stream, (const T*)c.g, c.ldg, c.stride_g, c.rows, c.cols, r.partial, arrivals.set[0], kMaxArrivals));
  PT_TRY(launch<first_kernel<T, PARTS>>("orthogonalize: first X", dim3(r.l64 / 64, r.s64 / 64, c.batch), 256, c.stream, (const T*)c.g, c.ldg, c.stride_g, tall, (const double*)r.partial, blocks, c.eps,
                r.s, r.l, r.pitch, x_stride, r.x, r.op[0], r.x_parts));
  const int vec = (uintptr_t)c.o % (4 * sizeof(T)) == 0 && c.ldo % 4 == 0 && c.stride_o % 4 == 0;
  const Symmetric<PARTS> A = {r.ao, r.da, r.s64, r.sq, r.sq_parts}, B = {r.bo, r.db, r.s64, r.sq, r.sq_parts};
  for (int k = 0; k < c.steps; ++k) {
    const Op* x = r.op[k % 2];
    Problem p = problem<PARTS>(x, r.x_parts, r.pitch, x, r.x_parts, r.pitch);
    p.M = p.N = p.M_out = p.N_out = r.s64;
    p.K = r.l64;
    p.batch_a = p.batch_b = x_stride;
    PT_TRY((run_product<Op, 1, 1, 0, SEGS, 1>(p, r.gram, Gram<PARTS>{A}, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: X X^T")));
    p = problem<PARTS>(r.ao, r.sq_parts, r.sq, r.ao, r.sq_parts, r.sq);
    p.M = p.N = p.M_out = p.N_out = p.K = r.s64;
    p.batch_a = p.batch_b = (long)r.s64 * r.sq;
    PT_TRY((run_product<Op, 1, 1, 0, SEGS, 1>(p, r.poly, Polynomial<PARTS>{A, B, c.coefficients[3 * k + 1], c.coefficients[3 * k + 2]}, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: A A")));
    Update<T, PARTS> u = {};
    u.x = r.x;
    u.diag = r.db;
    u.op = r.op[1 - k % 2];
    u.parts = r.x_parts;
    u.pitch = r.pitch;
    u.diag_pitch = r.sq;
    u.stride = x_stride;
    u.a = c.coefficients[3 * k];
    u.scale = c.scale;
    u.out = k + 1 == c.steps && !tall ? (T*)c.o : nullptr;
    u.ldo = c.ldo;
    u.s = r.s;
    u.l = r.l;
    u.vec = vec;
    u.out_stride = c.stride_o;
    p = problem<PARTS>(r.bo, r.sq_parts, r.sq, x, r.x_parts, r.pitch);
    p.M = p.M_out = p.K = r.s64;
    p.N = p.N_out = r.l64;
    p.batch_a = (long)r.s64 * r.sq;
    p.batch_b = x_stride;
    PT_TRY((run_product<Op, 1, 0, 0, SEGS, 0>(p, r.update, u, c.batch, r.pieces, arrivals, c.stream, c.compute_units, "orthogonalize: B X")));
  }
  if (tall)
    return launch<transposed_out_kernel<T>>("orthogonalize: output", dim3((r.l + 63) / 64, (r.s + 63) / 64, c.batch), 256, c.stream, (const float*)r.x, r.s, r.l, r.pitch, x_stride, c.scale, (T*)c.o, c.ldo, c.stride_o);
  if (c.steps == 0)
    return launch<out_kernel<T>>("orthogonalize: output", dim3(blocks_for((long)r.s * r.l), 1, c.batch), 256, c.stream, (const float*)r.x, r.s, r.l, r.pitch, x_stride, c.scale, (T*)c.o, c.ldo, c.stride_o);
  return RL_OK;
}

}  // namespace

size_t rl_ortho_room(const OrthoCall& c) { return c.dtype == RL_BF16 ? carve<1>(c).bytes : carve<2>(c).bytes; }

int rl_ortho_run(const OrthoCall& c) {
  if (c.dtype == RL_BF16) return run<bf16_t, 1>(c);
  if (c.dtype == RL_F16) return run<half_t, 2>(c);
  return run<float, 2>(c);
}

void rl_ortho_plans(const OrthoCall& c, Plan out[3]) {
  const Room r = c.dtype == RL_BF16 ? carve<1>(c) : carve<2>(c);
  out[0] = r.gram;
  out[1] = r.poly;
  out[2] = r.update;
}
