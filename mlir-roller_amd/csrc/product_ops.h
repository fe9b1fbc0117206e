// What follows a product: the epilogues of the matrix-product engine (product_tile.h) for the gated
// feed-forward block and for Newton-Schulz orthogonalisation, and the small kernels around them.
//
// An epilogue is a struct with at(batch), which picks the buffers of a batch entry, get(m, n), which
// loads what it needs besides the product, and put(m, n, v, in, ok): four consecutive columns n .. n+3 of row
// m, n a multiple of 4 (gated products: put(m, n, gate, up, in, ok)), stored if ok.  Of a symmetric product
// value(m, n, v, in) is what v becomes and put(m, n, value, ok) stores it, once as it is and once mirrored.

#ifndef PRODUCT_OPS_H
#define PRODUCT_OPS_H

#include "product_tile.h"

namespace product {

template <class T>
struct vec4;
template <> struct vec4<float> { typedef v4f type; };
template <> struct vec4<half_t> { typedef _Float16 type __attribute__((ext_vector_type(4))); };
template <> struct vec4<bf16_t> { typedef __bf16 type __attribute__((ext_vector_type(4))); };

// One rounding, to nearest even, from fp32 to the stored type.
template <class T>
PT_DEV typename vec4<T>::type round4(v4f v) {
  typename vec4<T>::type o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
  return o;
}

// Internal buffers: pitch a multiple of 4 elements, 16-byte aligned.
template <class T>
PT_DEV void store4(T* at, v4f v) { *(typename vec4<T>::type*)at = round4<T>(v); }
template <class T>
PT_DEV v4f load4(const T* at) {
  const typename vec4<T>::type x = *(const typename vec4<T>::type*)at;
  return v4f{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}

// ---- activations ------------------------------------------------------------------------------------
// Kept in fp32 throughout.  1 / (1 + 2^(-z log2 e)) from the exponential and the reciprocal of the
// hardware, 1 ulp each: the ends are exact (0 and 1), NaN stays NaN.

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

PT_DEV float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }

constexpr float GELU_2C = 1.5957691216f, GELU_C1 = 0.044715f;   // 2 sqrt(2 / pi)

// (1 + erf(g / sqrt 2)) / 2, as erfc of the other sign: 1 + erf has no digits left far below zero (at -5 the activation
// would be 4 % off, at -6 zero).
PT_DEV float normal_below(float g) { return 0.5f * erfcf(-0.70710678f * g); }

template <int KIND>
PT_DEV float act(float g) {
  if constexpr (KIND == ACT_SILU) return g * sigmoid(g);
  if constexpr (KIND == ACT_GELU) return g * normal_below(g);
  return g * sigmoid(GELU_2C * (g + GELU_C1 * g * g * g));   // (1 + tanh z) / 2 = sigmoid(2 z)
}

// The activation and its slope.  The factors that grow with g stand beside ones that are zero in fp32 where they
// would overflow (the sigmoid from -104 down, earlier the density of gelu and the sigmoid of gelu_tanh), so they are
// taken of g cut to +-128.
template <int KIND>
PT_DEV void act_slope(float g, float& a, float& slope) {
  const float c = fminf(fmaxf(g, -128.0f), 128.0f);
  if constexpr (KIND == ACT_SILU) {
    const float s = sigmoid(g);
    a = g * s;
    slope = s * (1.0f + c * (1.0f - s));
  } else if constexpr (KIND == ACT_GELU) {
    const float s = normal_below(g);
    a = g * s;
    slope = s + c * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * c * c);
  } else {
    const float s = sigmoid(GELU_2C * (g + GELU_C1 * g * g * g));
    a = g * s;
    slope = s + c * s * (1.0f - s) * GELU_2C * (1.0f + 3.0f * GELU_C1 * c * c);
  }
}

// ---- the scale of fp16 gradients --------------------------------------------------------------------
// dg and du are operands of two further products and have the element type.  In fp16 a number below 2^-14 has fewer
// than 11 bits, and that is where the gradients of an unscaled loss are (dy of 1e-6: dW_gate 3 % off).  So they are
// held times 2^k, and the products made of them leave times 2^-k.  k >= 0 is the least that brings the largest
// finite |dy| to 2^-6: dg and du around 2^-9 then have all their bits, and they reach infinity at 2^21 to 2^22 times
// that |dy|.  From |dy| = 2^-6 on k is 0.  (bf16 has the exponents of fp32.)

constexpr int PEAKS = 256;   // workgroups of peak_kernel

template <class T>
constexpr bool is_scaled() { return __is_same(T, half_t); }

// 2^k (SIGN 1) or 2^-k (SIGN -1) by the peaks of dy, each of which is a fp16 magnitude's bits.  By whole waves.
template <int SIGN>
PT_DEV float power_of_peaks(const unsigned* peaks) {
  const v4u four = *(const v4u*)(peaks + 4 * (threadIdx.x & 63));
  unsigned peak = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) peak = four[e] > peak ? four[e] : peak;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    const unsigned other = __shfl_xor(peak, d);
    peak = other > peak ? other : peak;
  }
  const float value = (float)__builtin_bit_cast(half_t, (unsigned short)__builtin_amdgcn_readfirstlane(peak));
  const int exponent = (int)(__builtin_bit_cast(unsigned, value) >> 23) - 127;
  const int k = value > 0.0f && exponent < -6 ? -6 - exponent : 0;   // (18 at most)
  return __builtin_bit_cast(float, (unsigned)(127 + SIGN * k) << 23);
}

// ---- epilogues --------------------------------------------------------------------------------------

// C = acc, in a caller's matrix: any leading dimension and alignment.  SCALED: an operand was held times 2^k, and C is
// 2^-k acc.
template <class T, int SCALED = 0>
struct Store {
  T* c[2];      // one per batch entry
  int ldc, ldc1, N;
  int vec;      // rows of 4 elements are aligned
  const unsigned* peaks;   // SCALED: of the dy that k is by
  float scale;             // (by at)
  __device__ __forceinline__ Store at(int batch) const {
    Store o = *this;
    if (batch) {
      o.c[0] = c[1];
      o.ldc = ldc1;
    }
    if constexpr (SCALED) o.scale = power_of_peaks<-1>(peaks);
    return o;
  }
  struct In {};
  __device__ __forceinline__ In get(int, int) const { return {}; }
  __device__ __forceinline__ void put(int m, int n, v4f v, In, bool ok) const {
    if (!ok) return;
    if constexpr (SCALED) v *= scale;
    T* to = c[0] + (long)m * ldc + n;
    if (vec && n + 3 < N) {
      store4(to, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) to[e] = (T)v[e];
    }
  }
};

// h = act(g) u; for a later backward pass g and u as well, unrounded (a gradient made of g and u rounded
// to 16 bits would carry two or three roundings where it now carries its own).
template <class T, int KIND>
struct GatedForward {
  T* h;           // NULL: only h32
  float* h32;     // h unrounded, NULL: not needed
  float *g, *u;   // NULL: not kept
  int pitch;
  __device__ __forceinline__ GatedForward at(int) const { return *this; }
  struct In {};
  __device__ __forceinline__ In get(int, int) const { return {}; }
  __device__ __forceinline__ void put(int m, int n, v4f gate, v4f up, In, bool ok) const {
    const long i = (long)m * pitch + n;
    v4f o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = act<KIND>(gate[e]) * up[e];
    if (!ok) return;
    if (h) store4(h + i, o);
    if (h32) *(v4f*)(h32 + i) = o;
    if (g) {
      *(v4f*)(g + i) = gate;
      *(v4f*)(u + i) = up;
    }
  }
};

// From dh: dg = dh u act'(g), du = dh act(g), in fp16 times 2^k.
template <class T, int KIND>
struct GatedBackward {
  const float *g, *u;
  T *dg, *du;
  int pitch;
  const unsigned* peaks;   // fp16: of dy
  float scale;             // (by at)
  __device__ __forceinline__ GatedBackward at(int) const {
    GatedBackward o = *this;
    if constexpr (is_scaled<T>()) o.scale = power_of_peaks<1>(peaks);
    return o;
  }
  struct In {
    v4f gate, up;
  };
  __device__ __forceinline__ In get(int m, int n) const {
    const long i = (long)m * pitch + n;
    return {*(const v4f*)(g + i), *(const v4f*)(u + i)};
  }
  __device__ __forceinline__ void put(int m, int n, v4f dh, In in, bool ok) const {
    const long i = (long)m * pitch + n;
    if constexpr (is_scaled<T>()) dh *= scale;
    v4f x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a, slope;
      act_slope<KIND>(in.gate[e], a, slope);
      x[e] = dh[e] * in.up[e] * slope;
      y[e] = dh[e] * a;
    }
    if (!ok) return;
    store4(dg + i, x);
    store4(du + i, y);
  }
};

// ---- small kernels ----------------------------------------------------------------------------------

// 16 bytes from any element on: loaded whole, at the alignment of their type, and at the end of a row element by
// element.
template <class T>
PT_DEV v4u whole_chunk(const T* at) {
  v4u v;
  __builtin_memcpy(&v, __builtin_assume_aligned(at, sizeof(T)), 16);
  return v;
}
template <class T>
PT_DEV v4u chunk_at(const T* row, int k, int K) {
  constexpr int PER = 16 / sizeof(T);
  if (k + PER <= K) return whole_chunk(row + k);
  typedef T chunk __attribute__((ext_vector_type(PER)));
  chunk v;
#pragma unroll
  for (int e = 0; e < PER; ++e) v[e] = k + e < K ? row[k + e] : (T)0.0f;
  return __builtin_bit_cast(v4u, v);
}

// Copies a matrix whose rows are not dword-aligned (16-bit elements at odd places) into one whose rows are,
// with zeros up to the pitch.
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, int ld, int rows, int cols, T* dst, int pitch) {
  constexpr int PER = 16 / sizeof(T);
  const int chunks = pitch / PER;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)rows * chunks; i += gridDim.x * 256L) {
    const int r = (int)(i / chunks), c = (int)(i % chunks) * PER;
    *(v4u*)(dst + (long)r * pitch + c) = chunk_at(src + (long)r * ld, c, cols);
  }
}

// The largest finite |element| of each of PEAKS shares of a fp16 matrix, as the bits of a magnitude, which are in the order
// of the numbers; zeros in `clear`.  `lanes` lanes, a power of two, read a row side by side.
template <class T>
__global__ __launch_bounds__(256) void peak_kernel(const T* src, int ld, int rows, int cols, int lanes, unsigned* peaks, unsigned* clear, int n_clear) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n_clear; i += gridDim.x * 256) clear[i] = 0;
  constexpr int PER = 16 / sizeof(T), UNROLL = 4;
  const int chunks = (cols + PER - 1) / PER, side = 256 / lanes;
  unsigned peak = 0;
  for (long r = (long)blockIdx.x * side + threadIdx.x / lanes; r < rows; r += (long)gridDim.x * side)
    for (int c = threadIdx.x % lanes; c < chunks; c += lanes * UNROLL) {
      v4u v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) v[u] = chunk_at(src + r * ld, (c + lanes * u) * PER, cols);   // (zeros past the end)
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const unsigned bits = v[u][e / 2] >> (e % 2 * 16) & 0x7fff;
          peak = bits < 0x7c00 && bits > peak ? bits : peak;
        }
    }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    const unsigned other = __shfl_xor(peak, d);
    peak = other > peak ? other : peak;
  }
  __shared__ unsigned waves[4];
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = peak;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < 4; ++w) peak = waves[w] > peak ? waves[w] : peak;
    peaks[blockIdx.x] = peak;
  }
}

// rows x cols zeros (the gradient of a weight over no tokens).
template <class T>
__global__ __launch_bounds__(256) void zero_kernel(T* c, int ld, int rows, int cols) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)rows * cols; i += gridDim.x * 256L) c[i / cols * ld + i % cols] = (T)0;
}

// ---- few rows ---------------------------------------------------------------------------------------
// A product with at most 16 * BLOCKS rows of x, whose time is that of reading the weights once.  A workgroup owns
// ROWS = 16 / PARTS weight rows (GATED: as many gate and up rows) and its waves share out K; weights go from
// memory straight into the MFMA's registers, so that all of a small problem's bytes can be asked for at once
// (the tile engine has at most three K steps on their way: with one token and weights 4096 x 1024 it took 8.6 us
// for the gate and up product where this kernel takes 5.8); no LDS until the waves' sums are added up.
//
// PARTS = 2 or 4: with few tokens the 16 x 16 block of an MFMA holds that many parts of K side by side, part q in
// rows and columns 16 / PARTS * q and on; of the products of all parts with all parts only the diagonal blocks
// are used.  A workgroup then owns fewer weight rows, and there are more of them (1024 rows of 4096 elements: 64
// workgroups of 16 rows for 256 CUs, or 256 of 4: 8.9 us against 4.7).  The parts are 64-byte pieces that lie side
// by side, so a load takes 128 or 256 bytes of a row: one token, weights of 4096 x 12288, 57 us; with the
// quarters of K as parts, 64.
//
// Rows may start at any element (chunk_at).
//
// SPLIT: x is fp32 although the weights have 16 bits.  Each of its elements then goes into the product as
// the sum of two of 16 bits, high part and remainder: twice the matrix instructions, which are idle anyway,
// and no rounding of x that the result could show.  What the type cannot hold becomes an infinity, as by rounding,
// without a remainder (infinity less infinity would make it a NaN).
template <class T, int SPLIT>
struct x_type { typedef T type; };
template <class T>
struct x_type<T, 1> { typedef float type; };

template <class T>
PT_DEV void split_chunk(const float* x, v4u& hi, v4u& lo) {
  typedef T chunk __attribute__((ext_vector_type(8)));
  chunk h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = (T)x[e];
    const float rest = x[e] - (float)h[e];
    l[e] = (T)(fabsf(rest) <= fabsf(x[e]) ? rest : 0.0f);
  }
  hi = __builtin_bit_cast(v4u, h);
  lo = __builtin_bit_cast(v4u, l);
}

template <class T, int BLOCKS, int PARTS, int GATED, int SPLIT, class Epi>
__global__ __launch_bounds__(1024) void few_rows_kernel(const typename x_type<T, SPLIT>::type* x, int ldx, const T* w0, int ldw0, const T* w1, int ldw1, int M, int N, int K, const Epi epi) {
  static_assert(PARTS == 1 || BLOCKS == 1, "parts share one block");
  constexpr int PER = 16 / sizeof(T), W = GATED ? 2 : 1, UNROLL = BLOCKS == 1 ? 8 : BLOCKS == 2 ? 4 : 2, ROWS = 16 / PARTS;
  const int waves = blockDim.x / 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * ROWS, row = n0 + lr % ROWS < N ? n0 + lr % ROWS : N - 1;   // (a row past the end is not stored)
  const T* wr[2] = {w0 + (long)row * ldw0, GATED ? w1 + (long)row * ldw1 : nullptr};
  typedef typename x_type<T, SPLIT>::type X;
  const X* xr[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    const int m = 16 * b + lr % ROWS;
    xr[b] = x + (long)(m < M ? m : M - 1) * ldx;
  }

  v4f acc[W][BLOCKS];
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) acc[w][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  // the waves take turns at groups of UNROLL x PARTS x 64 bytes
  constexpr int GROUP = UNROLL * PARTS * 4 * PER, XV = SPLIT ? 2 : 1;   // XV: 16-byte loads per chunk of x
  const int part = (lr / ROWS * 4 + lg) * PER;
  for (int k0 = wave * GROUP; k0 < K; k0 += waves * GROUP) {
    v4u wv[W][UNROLL], xv[BLOCKS][UNROLL][XV];
    const bool whole = k0 + GROUP <= K;
#pragma unroll
    for (int t = 0; t < UNROLL; ++t) {
      const int k = k0 + t * (PARTS * 4 * PER) + part;
#pragma unroll
      for (int w = 0; w < W; ++w) wv[w][t] = whole ? whole_chunk(wr[w] + k) : chunk_at(wr[w], k, K);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int v = 0; v < XV; ++v) xv[b][t][v] = whole ? whole_chunk(xr[b] + k + 4 * v) : chunk_at(xr[b], k + 4 * v, K);
    }
#pragma unroll
    for (int t = 0; t < UNROLL; ++t)
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        v4u hi = xv[b][t][0], lo;
        if constexpr (SPLIT) {
          float f[8];
          __builtin_memcpy(f, &xv[b][t][0], 16);
          __builtin_memcpy(f + 4, &xv[b][t][XV - 1], 16);
          split_chunk<T>(f, hi, lo);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          acc[w][b] = mma<T, 16>::run(wv[w][t], hi, acc[w][b]);
          if constexpr (SPLIT) acc[w][b] = mma<T, 16>::run(wv[w][t], lo, acc[w][b]);
        }
      }
  }

  // the waves' sums, added in wave order, and the parts' in part order, block after block by the first wave
  __shared__ v4f sums[W][16][64];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    if (b) __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) sums[w][wave][lane] = acc[w][b];
    __syncthreads();
    if (wave != 0 || lane >= 64 / (PARTS * PARTS)) continue;
    // lane of part 0 that holds columns 4 * quad .. of row m
    const int quad = PARTS == 1 ? lane >> 4 : PARTS == 2 ? lane >> 3 : 0, m = 16 * b + lane % ROWS, n = n0 + 4 * quad;
    v4f total[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      total[w] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      for (int s = 0; s < waves; ++s)
#pragma unroll
        for (int q = 0; q < PARTS; ++q) total[w] += sums[w][s][16 * (ROWS / 4 * q + quad) + ROWS * q + lane % ROWS];
    }
    if (m >= M || n >= N) continue;
    // (columns past the last weight row hold copies of its products: padding of h, or not stored)
    const auto out = epi.at(0);
    if constexpr (GATED) {
      out.put(m, n, total[0], total[W - 1], out.get(m, n), true);
    } else {
      out.put(m, n, total[0], out.get(m, n), true);
    }
  }
}

}  // namespace product

#endif
