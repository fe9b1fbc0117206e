// The matrix-product engine behind the feed-forward block and the orthogonalisation (gfx950, CDNA4):
// one workgroup per tile of the result, bf16 / fp16 / fp32 operands, fp32 accumulators, and an
// epilogue that is a template argument, so that what follows a product happens on the accumulators.
//
//   acc[m][n] = sum over segments s, sum over k:  A_s[m][k] * B_s[n][k]
//
// Each operand is stored either with k contiguous (A[M][lda >= K], "K-major") or with its rows
// contiguous (At[K][lda >= M], "row-major in k"), which covers x W^T, dy W and dy^T x without a
// transposed copy of anything.
//
// Layout.  A K step is 128 bytes of k: 64 elements of 16 bits, 32 of 32 bits.  Both forms arrive in
// LDS by buffer loads that write LDS directly, 16 bytes per lane; a wave's load lands as 64
// consecutive 16-byte chunks, so rows are not padded but their chunks are XOR-permuted on the load
// side (each lane chooses which global chunk it fetches), and the reads apply the same permutation:
//   * K-major tile [rows][128 bytes]: chunk c of row r sits at c ^ ((r / 2) % 8).  A lane reads one
//     chunk (8 or 4 consecutive k of its row) with ds_read_b128; the 16 rows of a lane group then
//     cover 16 distinct 16-byte bank groups.
//   * row-major tile [64 or 32 k][rows]: of 16-bit operands a lane group reads a 4 (k) x 16 (rows)
//     patch with ds_read_b64_tr_b16, which hands every lane 4 consecutive k of one row; two of those
//     make the same 8 k that a K-major chunk holds.  Of 32-bit operands a lane reads its four k one
//     by one.  The chunk permutation by k (mn_swizzle) keeps both free of bank conflicts.
// An MFMA sums over its k slots and only A and B have to agree on which k sits in which slot, so the
// 32-bit path feeds the four floats of a chunk to four v_mfma_f32_16x16x4_f32.
//
// The operands go into the MFMA in swapped order (B as the first), which computes the transposed
// block: a lane then holds four consecutive columns of one row of the result, and stores are
// vectors.
//
// The K loop is software pipelined over two to four LDS buffers: the loads of the next steps are in
// flight while a step is multiplied, and the fragments of the next MFMAs are read beside the current
// ones, also across the barrier between steps.

#ifndef PRODUCT_TILE_H
#define PRODUCT_TILE_H

#include <hip/hip_runtime.h>

#include "product_plan.h"

#define PT_DEV static __device__ __forceinline__

namespace product {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 half_t;
typedef __bf16 bf16_t;

constexpr unsigned OOB = 0x80000000u;   // beyond every resource: a load there returns 0 and touches no memory
constexpr int STEP_BYTES = 128;         // bytes of k per K step

template <int V>
struct int_c {
  static constexpr int value = V;
};

// Buffer resource over `bytes` from p, or over nothing: a load beyond it returns 0 and touches no memory.
PT_DEV v4u resource(const void* p, bool live, unsigned bytes) {
  const unsigned long at = (unsigned long)p;
  return v4u{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, live ? bytes : 0u, 0x00020000u};
}
// What is left of a matrix, in whole dwords, 2 GiB at most.
PT_DEV unsigned dwords_of(long bytes) { return bytes > 0x7ffffffcL ? 0x7ffffffcu : ((unsigned)bytes + 3u) & ~3u; }

#if __HIP_DEVICE_COMPILE__
// 16 bytes per lane from `off` of the resource to LDS, lane by lane from `lds_at` on.  Written out, because
// the compiler waits for a builtin load of this kind to land before it issues any ds_read_b64_tr_b16, to
// whatever address; the K loop waits where a buffer changes hands.  The instruction has no register
// result.  Before it m0 needs one wait state, and a resource register that the vector unit has written (as a
// readlane does where scalar registers are short) five, which the compiler does not see to in front of
// written-out code.
PT_DEV void load_to_lds(v4u rsrc, unsigned lds_at, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_at), "v"(off), "s"(rsrc) : "m0");
}
// Waits until at most n of this wave's loads are outstanding (vmcnt is split over bits 3:0 and 15:14).
#define wait_loads(n) __builtin_amdgcn_s_waitcnt(0x0f70 | ((n) & 0xf) | (((n) >> 4) << 14))
#endif

// One 16-byte fragment of each operand into an accumulator block of MI x MI.
typedef float v16f __attribute__((ext_vector_type(16)));
template <int MI>
struct block;
template <>
struct block<16> { typedef v4f type; };
template <>
struct block<32> { typedef v16f type; };

template <class T, int MI>
struct mma {
  static constexpr int PER_FRAG = sizeof(T) == 4 ? 4 : 1;
  typedef typename block<MI>::type acc_t;
  // part t of PER_FRAG
  PT_DEV acc_t part(int t, v4u a, v4u b, acc_t c) {
    if constexpr (sizeof(T) == 4) {
      const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
      if constexpr (MI == 16) return __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
      else return __builtin_amdgcn_mfma_f32_32x32x2f32(x[t], y[t], c, 0, 0, 0);
    } else if constexpr (__is_same(T, half_t)) {
      const v8h x = __builtin_bit_cast(v8h, a), y = __builtin_bit_cast(v8h, b);
      if constexpr (MI == 16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
      else return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    } else {
      const v8b x = __builtin_bit_cast(v8b, a), y = __builtin_bit_cast(v8b, b);
      if constexpr (MI == 16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
      else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }
  }
  PT_DEV acc_t run(v4u a, v4u b, acc_t c) {
#pragma unroll
    for (int t = 0; t < PER_FRAG; ++t) c = part(t, a, b, c);
    return c;
  }
};

// Permutation of the 16-byte chunks of row k of a row-major tile whose rows are ROW_BYTES long (XOR-ed
// onto the chunk number).
//   16 bits: half a wave reads 64 bytes (32 rows of the product) from each of the rows k .. k+3; the four
//   must lie in four different quarters of the 256 bytes that the banks span.  Where a row is an odd multiple
//   of 128 bytes (tiles of 64 and 192), every second row differs from its neighbour by its own length already;
//   and its number of chunks allows no permutation beyond groups of eight.
//   32 bits: half a wave reads 128 bytes of one row, which covers the 32 banks of a 32-bit read as it is.
template <int ES, int ROW_BYTES>
PT_DEV constexpr int mn_swizzle(int k) {
  static_assert(ROW_BYTES % 128 == 0, "tiles are multiples of 64 rows of 16 bits");
  if constexpr (ES == 4) {
    return 0;
  } else if constexpr (ROW_BYTES % 256 == 0) {
    return (k & 3) * 4;
  } else {
    return ((k >> 1) & 1) * 4;
  }
}

#if __HIP_DEVICE_COMPILE__
// LDS by address (a kernel's one __shared__ array starts at 0)
template <class V>
PT_DEV V lds_read(unsigned at) {
  return *(const __attribute__((address_space(3))) V*)at;
}

template <class V>
PT_DEV void lds_write(unsigned at, V v) {
  *(__attribute__((address_space(3))) V*)at = v;
}

// Address, within a row-major tile with rows of ROW_BYTES, of what a lane reads of the 32 rows from `row0`.
// 16 bits: the 16 lanes of a group address a patch of 4 k x 16 rows, lane q its row q / 4 at 4 elements from
// 4 * (q % 4); k = 8 * (lane / 32).  32 bits: element lane % 32 of k = 4 * (lane / 32).
template <int ES, int ROW_BYTES>
PT_DEV unsigned rows_at(int row0, int lane) {
  if constexpr (ES == 2) {
    const int q = lane % 16, k = 8 * (lane / 32) + q / 4, chunk = (row0 + (lane & 16)) / 8 + (q & 3) / 2;
    return k * ROW_BYTES + (chunk ^ mn_swizzle<ES, ROW_BYTES>(k)) * 16 + (q & 1) * 8;
  } else {
    return 4 * (lane / 32) * ROW_BYTES + (row0 + lane % 32) * 4;
  }
}

// The lane's fragment from there: 8 (16 bits) or 4 (32 bits) consecutive k of its row.  The permutation
// is the same for the k that follow within the fragment.
template <int ES, int ROW_BYTES>
PT_DEV v4u read_rows(unsigned at) {
  if constexpr (ES == 2) {
    typedef __attribute__((address_space(3))) v4s* tr_ptr;
    const v2u lo = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at));
    const v2u hi = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 4 * ROW_BYTES)));
    return v4u{lo.x, lo.y, hi.x, hi.y};
  } else {
    return v4u{lds_read<unsigned>(at), lds_read<unsigned>(at + ROW_BYTES), lds_read<unsigned>(at + 2 * ROW_BYTES), lds_read<unsigned>(at + 3 * ROW_BYTES)};
  }
}

#endif

// What a launch is about.  Extents and leading dimensions in elements.
struct Problem {
  const void* a[3];   // one per K segment
  const void* b[3];   // one per K segment; GATED: gate and up weights of the one segment
  int lda, ldb, ldb1; // (ldb1: leading dimension of the up weights)
  int M, N, K;        // GATED: N counts columns of the product, each made of a gate and an up column
  int M_out, N_out;   // rows and columns handed to the epilogue (those beyond M and N are zeros)
  long batch_a, batch_b;
  // A tile's K steps may be shared out over workgroups.  Each then leaves its accumulators in `pieces`,
  // and the one that finds the tile's arrival counter at splits - 1 adds them up in split order, whoever
  // that is, so results do not depend on timing.  `arrivals` is zero when the launch starts; the launch
  // before it on the stream sees to that (clear, n_clear).  The first `whole` tiles (a multiple of the number of
  // XCDs) have a workgroup each, the others `splits`.
  int splits, steps_per_split, whole;
  float* pieces;
  unsigned *arrivals, *clear;
  int n_clear;
};

// Tile shape, operand forms and options of one kernel.
//   A_KM, B_KM  K-major (1) or row-major in k (0)
//   GATED       the tile's columns are BN/2 gate columns and the same BN/2 up columns, laid out so that
//               a lane has both of a column (accumulator blocks j and j + TN/2)
//   SEGS        K segments
//   SYM         the result is symmetric: only the tiles on and below the diagonal are computed, and those
//               below it leave twice, as they are and transposed (M_out = N_out, a multiple of 4)
template <class T_, int BM_, int BN_, int WM_, int WN_, int A_KM_, int B_KM_, int GATED_ = 0, int SEGS_ = 1, int SYM_ = 0, int PER_CU_ = 1, int MI_ = 32, int BUFS_ = 2>
struct Shape {
  typedef T_ T;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, A_KM = A_KM_, B_KM = B_KM_, GATED = GATED_, SEGS = SEGS_, SYM = SYM_;
  static constexpr int PER_CU = PER_CU_;   // workgroups that should fit a CU
  // Quarters of a step's loads that are issued a step ahead.  More wait out more latency, fewer crowd the
  // end of a step less (8192^3 in bf16, K-major operands, 0 to 4: 1275, 1340, 1367, 1332, 1300 TFLOP/s).
  static constexpr int TAIL_LOADS = 2;
  static constexpr int NWM = BM / WM, NWN = BN / WN, WAVES = NWM * NWN, NT = 64 * WAVES;
  static constexpr int ES = sizeof(T), KSTEP = STEP_BYTES / ES;
  static constexpr int MI = MI_, TM = WM / MI, TN = WN / MI;
  static constexpr int ROUNDS = MI / 8;               // fragment rounds per K step: each takes 64 / MI of its 8 chunks
  static constexpr int A_BYTES = BM * STEP_BYTES, B_BYTES = BN * STEP_BYTES;
  static constexpr int BUFS = BUFS_, LDS_BYTES = BUFS * (A_BYTES + B_BYTES);
  static constexpr int A_LOADS = BM * 8 / NT, B_LOADS = BN * 8 / NT;
  static constexpr bool SPLIT = BM * BN <= 192 * 192;   // K steps may be shared out (the registers of 256 x 256 leave no room to)
  static constexpr int OUT_N = GATED ? BN / 2 : BN;   // result columns per tile
  // Tiles for few rows stream B once.  Groups of neighbours then start at different K steps: rows a power of two
  // apart would otherwise be read at the same place of a row by everybody at once, which crowds the same memory
  // channels (24 rows, B of 16384 rows of 8192 bytes, 32 x 64 tiles: 30.9 us, 25.8 with every tile at a step of
  // its own, 23.6 with every eighth; 4096 rows of 16384 bytes in four splits: 20.0, 17.1, 19.1).
  static constexpr bool ROTATE = BM <= 64 && A_KM && B_KM && SEGS == 1 && !SYM;
  static_assert(BM % WM == 0 && BN % WN == 0 && WM % MI == 0 && WN % MI == 0, "tile");
  static_assert((BM * 8) % NT == 0 && (BN * 8) % NT == 0, "whole loads per thread");
  static_assert(!GATED || ((WN / 2) % MI == 0 && B_KM), "gate and up halves of a wave tile");
  static_assert(!SYM || BM == BN, "square tiles");
  static_assert(BUFS >= 2 && BUFS <= 4, "LDS buffers");
  static_assert(MI == 32 || (A_KM && B_KM), "row-major tiles are read 32 rows at a time");
};

// Tile of a workgroup: every XCD gets a contiguous run of the tile order (workgroups are dealt to the
// XCDs round-robin), and the order walks panels of 8 tile rows, so that neighbours share operand panels
// in their L2.
PT_DEV int xcd_order(int pid, int n) {
  const int per = (n + XCDS - 1) / XCDS;
  int tall = n % XCDS;
  if (tall == 0) tall = XCDS;
  const int xcd = pid % XCDS, loc = pid / XCDS;
  return xcd < tall ? xcd * per + loc : tall * per + (xcd - tall) * (per - 1) + loc;
}

PT_DEV void panel_tile(int pid, int nbm, int nbn, int& tm, int& tn) {
  constexpr int GROUP = 8;
  const int width = GROUP * nbn, first = pid / width * GROUP;
  const int rows = nbm - first < GROUP ? nbm - first : GROUP;
  tm = first + pid % width % rows;
  tn = pid % width / rows;
}

// Tile number p of the lower triangle of n x n tiles, in panels of 8 tile rows: a panel's full columns one
// after the other, 8 tiles each, then the triangle at its end, row by row.
PT_DEV void triangle_tile(int p, int n, int& tm, int& tn) {
  constexpr int GROUP = 8;
  int g = 0, height = n < GROUP ? n : GROUP;
  for (;;) {   // (a few panels)
    const int size = GROUP * g * height + height * (height + 1) / 2;
    if (p < size) break;
    p -= size;
    ++g;
    height = n - GROUP * g < GROUP ? n - GROUP * g : GROUP;
  }
  if (p < GROUP * g * height) {
    tm = GROUP * g + p % height;
    tn = p / height;
    return;
  }
  p -= GROUP * g * height;
  int r = 0;
  while (p > r) p -= ++r;
  tm = GROUP * g + r;
  tn = GROUP * g + p;
}

// Cache policy of the pieces of a split tile: sc0 and sc1, coherent across the device's L2 caches, so that
// neither side writes back or invalidates a cache that holds the operands.
constexpr int COHERENT = 0x11;

template <class S, class Epi>
__global__ __launch_bounds__(S::NT, S::PER_CU * S::WAVES / 4 > 0 ? S::PER_CU * S::WAVES / 4 : 1) void tile_kernel(const Problem p, const Epi epi) {
#if __HIP_DEVICE_COMPILE__   // (the host pass needs the kernel's name only)
  typedef typename S::T T;
  constexpr int ES = S::ES, TM = S::TM, TN = S::TN, NT = S::NT;
  __shared__ __attribute__((aligned(1024))) char lds[S::LDS_BYTES];
  typedef __attribute__((address_space(3))) void* lds_ptr;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm0 = (wave / S::NWN) * S::WM, wn0 = (wave % S::NWN) * S::WN;
  constexpr int MI = S::MI, ROUNDS = S::ROUNDS;
  const int lr = lane % MI, lg = lane / MI;   // row of a block; k group

  const int nbm = (p.M_out + S::BM - 1) / S::BM, nbn = (p.N_out + S::OUT_N - 1) / S::OUT_N;
  const int tiles = S::SYM ? nbm * (nbm + 1) / 2 : nbm * nbn;
  // Tiles are numbered through the batch; workgroups are those of the whole tiles, then splits * the other
  // tiles, in this order: a run of either shares operands.
  int pid, split = 0;
  const bool shared = (int)blockIdx.x >= p.whole;
  if (shared) {
    const int others = (gridDim.x - p.whole) / p.splits;
    pid = xcd_order(blockIdx.x - p.whole, gridDim.x - p.whole);
    split = pid / others;
    pid += p.whole - split * others;
  } else {
    pid = xcd_order(blockIdx.x, p.whole);
  }
  const int shared_tile = pid - p.whole, batch = pid / tiles;
  pid -= batch * tiles;
  int tile_m, tile_n;
  if constexpr (S::SYM) {
    triangle_tile(pid, nbm, tile_m, tile_n);
  } else {
    panel_tile(pid, nbm, nbn, tile_m, tile_n);
  }
  const int m0 = tile_m * S::BM, n0 = tile_n * S::OUT_N;

  // (unsigned: there may be almost 2^32 threads; where the step wraps around it goes back by 256 or more, and ends)
  for (unsigned i = blockIdx.x * NT + tid; i < (unsigned)p.n_clear; i += gridDim.x * NT) p.clear[i] = 0;

  // K steps of this workgroup.  A segment is a whole number of steps: its last step is cut by K.
  const int seg_steps = (p.K + S::KSTEP - 1) / S::KSTEP;
  const int first_step = split * p.steps_per_split;
  const int all_steps = seg_steps * S::SEGS;
  const int last_step = shared && first_step + p.steps_per_split < all_steps ? first_step + p.steps_per_split : all_steps;
  const int KT = last_step - first_step;
  // (more rows of tiles share B in the L2, which takes a common start)
  const int start = S::ROTATE && nbm <= 4 && KT > 0 ? (shared ? tile_n : tile_n / 8) % KT : 0;

  // ---- what each lane fetches: offsets from the tile's first element, fixed through the K loop ----
  unsigned a_off[S::A_LOADS], b_off[S::B_LOADS];
  int a_k;   // K-major: first k of the lane's chunks within a step, the same for every load
  // K-major: unit u is chunk (u % 8) ^ ((row / 2) % 8) of row u / 8; the rows of a lane's loads are NT / 8
  // apart, a multiple of 16, so the chunk is the same for all of them.
  static_assert(NT % 128 == 0 || (!S::A_KM && !S::B_KM), "the chunk of a lane's K-major loads is the same for all");
  const int km_chunk = (tid & 7) ^ ((tid >> 4) & 7);
  a_k = km_chunk * (16 / ES);
#pragma unroll
  for (int i = 0; i < S::A_LOADS; ++i) {
    const int u = tid + i * NT;
    if constexpr (S::A_KM) {
      const int row = u / 8;
      a_off[i] = m0 + row < p.M ? (unsigned)(row * p.lda * ES + km_chunk * 16) : OOB;
    } else {
      constexpr int CU = S::BM * ES / 16;
      const int k = u / CU, c = (u % CU) ^ mn_swizzle<ES, S::BM * ES>(k);
      a_off[i] = m0 + c * (16 / ES) < p.M ? (unsigned)(k * p.lda * ES + c * 16) : OOB;
    }
  }
#pragma unroll
  for (int i = 0; i < S::B_LOADS; ++i) {
    const int u = tid + i * NT;
    if constexpr (S::B_KM) {
      const int row = u / 8;
      if constexpr (S::GATED) {
        // rows [0, WN/2) of a wave's part of the B tile are gate columns, the rest the same up columns
        const int col = row / S::WN * (S::WN / 2) + row % (S::WN / 2), ld = row % S::WN < S::WN / 2 ? p.ldb : p.ldb1;
        b_off[i] = n0 + col < p.N ? (unsigned)(col * ld * ES + km_chunk * 16) : OOB;
      } else {
        b_off[i] = n0 + row < p.N ? (unsigned)(row * p.ldb * ES + km_chunk * 16) : OOB;
      }
    } else {
      constexpr int CU = S::BN * ES / 16;
      const int k = u / CU, c = (u % CU) ^ mn_swizzle<ES, S::BN * ES>(k);
      b_off[i] = n0 + c * (16 / ES) < p.N ? (unsigned)(k * p.ldb * ES + c * 16) : OOB;
    }
  }

  const long a_tile = (S::A_KM ? (long)m0 * p.lda : (long)m0) + batch * p.batch_a;
  const long b_tile = (S::B_KM ? (long)n0 * p.ldb : (long)n0) + batch * p.batch_b;
  const long b_tile1 = (long)n0 * p.ldb1 + batch * p.batch_b;
  const long a_step = S::A_KM ? S::KSTEP : (long)S::KSTEP * p.lda;   // elements per K step
  const long b_step = S::B_KM ? S::KSTEP : (long)S::KSTEP * p.ldb;

  // bytes from the tile's first element to the matrix's end
  const long a_end = ((S::A_KM ? (long)(p.M - 1 - m0) * p.lda + p.K : (long)(p.K - 1) * p.lda + p.M - m0)) * ES;
  const long b_end = ((S::B_KM ? (long)(p.N - 1 - n0) * p.ldb + p.K : (long)(p.K - 1) * p.ldb + p.N - n0)) * ES;

  // Operand bases of K step kt (of this workgroup).  A step at or beyond KT gets empty resources.  KTEST: the
  // step may be the last, in which a chunk can reach past the matrix's last element.
  struct source {
    v4u a, b, b1;   // (b1: the up weights)
    int k_left;     // of K, from the step's first k on
  };
  auto source_of = [&](auto ktest, int kt) __attribute__((always_inline)) {
    constexpr bool KTEST = decltype(ktest)::value;
    const bool live = kt < KT;
    int step = first_step + (live ? kt : 0), seg = 0;
    if constexpr (S::ROTATE) step += start < KT - (live ? kt : 0) ? start : start - KT;
    if constexpr (S::SEGS > 1) {
      if (step >= seg_steps) { step -= seg_steps; seg = 1; }
      if constexpr (S::SEGS > 2) {
        if (step >= seg_steps) { step -= seg_steps; seg = 2; }
      }
    }
    const T* ap = (const T*)(S::SEGS > 1 && seg == 1 ? p.a[1] : S::SEGS > 2 && seg == 2 ? p.a[2] : p.a[0]) + a_tile + step * a_step;
    const T* bp = (const T*)(S::SEGS > 1 && seg == 1 ? p.b[1] : S::SEGS > 2 && seg == 2 ? p.b[2] : p.b[0]) + b_tile + step * b_step;
    source s;
    s.a = resource(ap, live, KTEST ? dwords_of(a_end - step * a_step * ES) : 0x7fffffffu);
    s.b = resource(bp, live, KTEST ? dwords_of(b_end - step * b_step * ES) : 0x7fffffffu);
    if constexpr (S::GATED) s.b1 = resource((const T*)p.b[1] + b_tile1 + step * S::KSTEP, live, KTEST ? dwords_of(((long)(p.N - 1 - n0) * p.ldb1 + p.K - step * S::KSTEP) * ES) : 0x7fffffffu);
    s.k_left = p.K - step * S::KSTEP;
    return s;
  };
  // Issues load i of a step (the loads of A, then those of B) into LDS buffer `buf`.  KTEST: the step may be
  // one that K cuts short.
  const unsigned lds0 = (unsigned)(unsigned long)(lds_ptr)lds;
  auto load = [&](auto ktest, const source& s, int buf, int i) __attribute__((always_inline)) {
    constexpr bool KTEST = decltype(ktest)::value;
    if (i < S::A_LOADS) {
      unsigned off = a_off[i];
      if constexpr (KTEST) off = (S::A_KM ? a_k : (tid + i * NT) / (S::BM * ES / 16)) < s.k_left ? off : OOB;
      load_to_lds(s.a, lds0 + buf * S::A_BYTES + (i * NT + wave * 64) * 16, off);
    } else {
      i -= S::A_LOADS;
      unsigned off = b_off[i];
      if constexpr (KTEST) off = (S::B_KM ? a_k : (tid + i * NT) / (S::BN * ES / 16)) < s.k_left ? off : OOB;
      // (GATED: the 8 rows of a wave's load are all gate or all up)
      const bool up = S::GATED && (i * (NT / 8) + wave * 8) % S::WN >= S::WN / 2;
      load_to_lds(up ? s.b1 : s.b, lds0 + S::BUFS * S::A_BYTES + buf * S::B_BYTES + (i * NT + wave * 64) * 16, off);
    }
  };

  // ---- fragments ----
  struct frags {
    v4u a[TM], b[TN];
  };
  // LDS addresses: one register per operand and half step (K-major) or per operand and block (row-major);
  // everything else about a read is an immediate offset.  The registers are opaque to the compiler, which
  // would otherwise fold the offsets of all reads into addresses of their own, one register each.
  unsigned a_at[S::A_KM ? ROUNDS : TM], b_at[S::B_KM ? ROUNDS : TN];
  auto opaque = [](unsigned& v) __attribute__((always_inline)) { asm volatile("" : "+v"(v)); };
  if constexpr (S::A_KM) {
#pragma unroll
    for (int h = 0; h < ROUNDS; ++h) {
      a_at[h] = (wm0 + lr) * STEP_BYTES + ((64 / MI * h + lg) ^ ((lr >> 1) & 7)) * 16;
      opaque(a_at[h]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      a_at[i] = rows_at<ES, S::BM * ES>(wm0 + MI * i, lane);
      opaque(a_at[i]);
    }
  }
  if constexpr (S::B_KM) {
#pragma unroll
    for (int h = 0; h < ROUNDS; ++h) {
      b_at[h] = S::BUFS * S::A_BYTES + (wn0 + lr) * STEP_BYTES + ((64 / MI * h + lg) ^ ((lr >> 1) & 7)) * 16;
      opaque(b_at[h]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      b_at[j] = S::BUFS * S::A_BYTES + rows_at<ES, S::BN * ES>(wn0 + MI * j, lane);
      opaque(b_at[j]);
    }
  }
  // Fragment i of a round: blocks of A and B in the order in which the MFMAs ask for them.
  auto read = [&](frags& f, auto buf_c, auto round_c, int i) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value, round = decltype(round_c)::value;
    if (i == 0 || i > TN) {
      if (i) i -= TN;
      if constexpr (S::A_KM) {
        f.a[i] = lds_read<v4u>(a_at[round] + (buf * S::A_BYTES + i * MI * STEP_BYTES));
      } else {
        f.a[i] = read_rows<ES, S::BM * ES>(a_at[i] + (buf * S::A_BYTES + round * (S::KSTEP / ROUNDS) * S::BM * ES));
      }
    } else {
      i -= 1;
      if constexpr (S::B_KM) {
        f.b[i] = lds_read<v4u>(b_at[round] + (buf * S::B_BYTES + i * MI * STEP_BYTES));
      } else {
        f.b[i] = read_rows<ES, S::BN * ES>(b_at[i] + (buf * S::B_BYTES + round * (S::KSTEP / ROUNDS) * S::BN * ES));
      }
    }
  };

  typename mma<T, MI>::acc_t acc[TM][TN];
  constexpr int REGS = MI * MI / 64;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < REGS; ++r) acc[i][j][r] = 0.0f;

  auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };

  // ---- K loop ----
  // A step is ROUNDS rounds of G slots; a round multiplies one set of fragments while the next set is read.
  // Buffer `cur` holds step kt, and the steps up to kt + BUFS - 1 are on their way into the others: of the
  // last of them the first TAIL loads were issued at the end of step kt - 1, the others go out in the first
  // two rounds.  A quarter into the last round the step's own reads are over and kt + 1 must have landed:
  // the workgroup meets, reads the first fragments of kt + 1 and sends the first loads of kt + BUFS into
  // `cur`.
  // The order of instructions is the order written here (sched_barrier between the slots, one MFMA each, four
  // with 32-bit operands): reads and loads are spread over the MFMAs, which run meanwhile; issued in a bunch
  // they hold up the MFMAs behind them.
  constexpr int PARTS = mma<T, MI>::PER_FRAG, G = TM * TN, FRAGS = TM + TN, L = S::A_LOADS + S::B_LOADS;
  constexpr int BUFS = S::BUFS, EARLY = G / 4, TAIL = L * S::TAIL_LOADS / 4;
  auto slot_mfma = [&](const frags& f, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int e = t * PARTS; e < (t + 1) * PARTS; ++e) {
      const int i = e % G / TN, j = e % TN;
      acc[i][j] = mma<T, MI>::part(e / G, f.b[j], f.a[i], acc[i][j]);
    }
  };
  // The steps that K cuts short are the last ones of the segments.  Where K ends inside a chunk of a K-major
  // operand, what the chunk brought from behind K (the next row's first elements, or nobody's) is overwritten
  // with zeros in LDS once it has landed.
  constexpr int PER = 16 / ES;
  const bool whole = p.K % S::KSTEP == 0 && (S::A_KM || p.M % PER == 0) && (S::B_KM || p.N % PER == 0);
  const bool ragged = p.K % PER != 0;
  const int rotated_cut = last_step == seg_steps ? KT - 1 - start : KT;   // ROTATE: where the last step of K comes
  auto is_cut = [&](int kt) __attribute__((always_inline)) { return S::ROTATE ? kt == rotated_cut : kt < KT && (first_step + kt + 1) % seg_steps == 0; };
  auto zero_tails = [&](int buf) __attribute__((always_inline)) {
    const int left = p.K % S::KSTEP;
    if (a_k < left && a_k + PER > left) {
      if constexpr (S::A_KM) {
#pragma unroll 1
        for (int i = 0; i < S::A_LOADS; ++i)
          for (int e = left - a_k; e < PER; ++e) lds_write<T>(buf * S::A_BYTES + (tid + i * NT) * 16 + e * ES, (T)0.0f);
      }
      if constexpr (S::B_KM) {
#pragma unroll 1
        for (int i = 0; i < S::B_LOADS; ++i)
          for (int e = left - a_k; e < PER; ++e) lds_write<T>(BUFS * S::A_BYTES + buf * S::B_BYTES + (tid + i * NT) * 16 + e * ES, (T)0.0f);
      }
    }
    __syncthreads();
  };
  if (KT > 0) {
    frags f[2];
    {
#pragma unroll
      for (int b = 0; b < BUFS; ++b) {
        const source s = source_of(int_c<1>{}, b);
#pragma unroll
        for (int i = 0; i < (b + 1 < BUFS ? L : TAIL); ++i) load(int_c<1>{}, s, b, i);
      }
    }
    wait_loads((BUFS - 2) * L + TAIL);   // step 0 has landed
    __syncthreads();
    if (ragged && is_cut(0)) zero_tails(0);
#pragma unroll
    for (int i = 0; i < FRAGS; ++i) read(f[0], int_c<0>{}, int_c<0>{}, i);
    fence();
    auto step = [&](auto ktest, auto cur_c, int kt) __attribute__((always_inline)) {
      constexpr int cur = decltype(cur_c)::value;
      {
        const source next = source_of(ktest, kt + BUFS - 1);
        constexpr int into = (cur + BUFS - 1) % BUFS;
        auto round = [&](auto round_c) __attribute__((always_inline)) {
          constexpr int r = decltype(round_c)::value;
          constexpr int FROM = TAIL + (r < 2 ? r : 2) * (L - TAIL) / 2, TO = TAIL + (r < 1 ? r + 1 : 2) * (L - TAIL) / 2;
#pragma unroll
          for (int t = 0; t < G; ++t) {
            slot_mfma(f[r & 1], t);
#pragma unroll
            for (int i = t * FRAGS / G; i < (t + 1) * FRAGS / G; ++i) read(f[(r + 1) & 1], cur_c, int_c<r + 1>{}, i);
#pragma unroll
            for (int i = FROM + t * (TO - FROM) / G; i < FROM + (t + 1) * (TO - FROM) / G; ++i) load(ktest, next, into, i);
            fence();
          }
        };
        round(int_c<0>{});
        if constexpr (ROUNDS == 4) {
          round(int_c<ROUNDS - 3>{});
          round(int_c<ROUNDS - 2>{});
        } else {
#pragma unroll
          for (int i = TAIL + (L - TAIL) / 2; i < L; ++i) load(ktest, next, into, i);
        }
      }
#pragma unroll
      for (int t = 0; t < EARLY; ++t) slot_mfma(f[1], t);
      fence();
      wait_loads((BUFS - 2) * L);   // kt + 1 has landed
      __syncthreads();
      if constexpr (decltype(ktest)::value) {
        if (ragged && is_cut(kt + 1)) zero_tails((cur + 1) % BUFS);
      }
      fence();
      const source next = source_of(ktest, kt + BUFS);
      constexpr int REST = G - EARLY;
#pragma unroll
      for (int t = 0; t < REST; ++t) {
        slot_mfma(f[1], EARLY + t);
#pragma unroll
        for (int i = t * FRAGS / REST; i < (t + 1) * FRAGS / REST; ++i) read(f[0], int_c<(cur + 1) % BUFS>{}, int_c<0>{}, i);
#pragma unroll
        for (int i = t * TAIL / REST; i < (t + 1) * TAIL / REST; ++i) load(ktest, next, cur, i);
        fence();
      }
    };
    // Passes of BUFS steps: without the tests as long as the pass's loads and reads (up to step kt + 2 BUFS) stay
    // clear of a cut step, with them around one.
    int kt = 0;
    auto pass = [&](auto ktest) __attribute__((always_inline)) {
      step(ktest, int_c<0>{}, kt);
      step(ktest, int_c<1>{}, kt + 1);
      if constexpr (BUFS > 2) step(ktest, int_c<2 % BUFS>{}, kt + 2);
      if constexpr (BUFS > 3) step(ktest, int_c<3 % BUFS>{}, kt + 3);
      kt += BUFS;
    };
    if constexpr (S::ROTATE) {
      const int free = whole ? KT : rotated_cut - BUFS;
      while (kt + BUFS <= KT && kt + BUFS <= free) pass(int_c<0>{});
      while (kt + BUFS <= KT && kt <= rotated_cut) pass(int_c<1>{});
      while (kt + BUFS <= KT) pass(int_c<0>{});
    } else if constexpr (S::SEGS == 1) {
      const int free = whole ? KT : seg_steps - 1 - first_step - BUFS;   // passes that end at or before it
      while (kt + BUFS <= KT && kt + BUFS <= free) pass(int_c<0>{});
      while (kt + BUFS <= KT) pass(int_c<1>{});
    } else {
      for (int cut = seg_steps - 1 - first_step % seg_steps; kt + BUFS <= KT; cut += seg_steps) {
        const int free = whole ? KT : cut - BUFS;
        while (kt + BUFS <= KT && kt + BUFS <= free) pass(int_c<0>{});
        while (kt + BUFS <= KT && kt <= cut) pass(int_c<1>{});
      }
    }
    if (kt < KT) step(int_c<1>{}, int_c<0>{}, kt);
    if constexpr (BUFS > 2) {
      if (kt + 1 < KT) step(int_c<1>{}, int_c<1>{}, kt + 1);
    }
    if constexpr (BUFS > 3) {
      if (kt + 2 < KT) step(int_c<1>{}, int_c<2>{}, kt + 2);
    }
    wait_loads(0);   // the empty requests past the end have drained
  }

  __syncthreads();   // the K loop is done with the LDS

  // ---- a shared tile: leave the accumulators, and the last one in adds them up ----
  if constexpr (S::SPLIT) if (shared) {
    constexpr int QUADS = REGS / 4;
    const long tile = shared_tile;
    float* const pieces = p.pieces + tile * p.splits * (S::BM * S::BN);
    {
      const __amdgpu_buffer_rsrc_t mine = __builtin_amdgcn_make_buffer_rsrc(pieces + (long)split * (S::BM * S::BN), 0, S::BM * S::BN * 4, 0x00020000);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < QUADS; ++q)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]}), mine,
                                                   (unsigned)((((i * TN + j) * QUADS + q) * NT + tid) * 16), 0, COHERENT);
        fence();
      }
    }
    wait_loads(0);   // (stores count as well: the piece has arrived in memory)
    __syncthreads();
    if (tid == 0) lds_write(0u, __hip_atomic_fetch_add(&p.arrivals[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(lds_read<unsigned>(0u)) != (unsigned)p.splits - 1) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      for (int s = 0; s < p.splits; ++s) {
        const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(pieces + (long)s * (S::BM * S::BN), 0, S::BM * S::BN * 4, 0x00020000);
        v4f v[TN][QUADS];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < QUADS; ++q)
            v[j][q] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(from, (unsigned)((((i * TN + j) * QUADS + q) * NT + tid) * 16), 0, COHERENT));
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = s == 0 ? v[j][q][e] : acc[i][j][4 * q + e] + v[j][q][e];
      }
      fence();
    }
  }
  // ---- every accumulator leaves once ----
  // Through LDS, which the K loop has left: each wave writes a row of its blocks there (its own part, so
  // no wave waits for another) and reads it back row by row, four columns a lane.  Stores and the
  // epilogue's own loads are then whole stretches of a row, and its code is a loop instead of a copy per
  // accumulator.  Rows are padded by 16 bytes: the 16-byte writes of the lanes of a block go to
  // consecutive rows.
  constexpr int PITCH = S::WN + 4;
  static_assert(S::WAVES * MI * PITCH * 4 <= S::LDS_BYTES, "a row of blocks per wave fits the LDS");
  const unsigned mine = wave * (MI * PITCH * 4);
  const unsigned to = mine + (lr * PITCH + 4 * lg) * 4;
  const auto out = epi.at(batch);
  // (what one lane writes another reads; the LDS serves a wave's accesses in their order, which the compiler has to keep)
  auto lanes_meet = []() __attribute__((always_inline)) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); };
  {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      lanes_meet();
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < REGS / 4; ++q)   // registers 4q .. 4q+3: columns 256 / MI * q + 4 * lg and on of the block
          lds_write(to + (j * MI + 256 / MI * q) * 4, v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]});
      lanes_meet();
      const int mb = m0 + wm0 + i * MI;
      constexpr int COLS = S::GATED ? S::WN / 2 : S::WN, PER_ROW = COLS / 4, UNITS = MI * PER_ROW;   // 4 columns a unit
      const int nb = n0 + (S::GATED ? (wave % S::NWN) * (S::WN / 2) : wn0);
      typedef typename Epi::In In;
      constexpr int PER_LANE = UNITS / 64, MOST = sizeof(In) > 32 ? 4 : 8;
      constexpr int BATCH = PER_LANE <= MOST ? PER_LANE : PER_LANE % MOST == 0 ? MOST : PER_LANE % 6 == 0 ? 6 : 4;
      static_assert(UNITS % 64 == 0 && PER_LANE % BATCH == 0, "whole batches");
      // The epilogue's loads for BATCH units first (of the nearest unit that exists), then their results:
      // the loads wait for memory together, and nothing but the stores is conditional.
      auto units = [&](auto transposed) __attribute__((always_inline)) {
        constexpr bool TR = decltype(transposed)::value;
        constexpr int PER = TR ? MI / 4 : PER_ROW;
        const int m_last = p.M_out - 1, n_last = (p.N_out - 1) / 4 * 4;
#pragma unroll 1
        for (int u0 = lane; u0 < UNITS; u0 += 64 * BATCH) {
          In in[BATCH];
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            const int u = u0 + 64 * k, m = (TR ? nb : mb) + u / PER, n = (TR ? mb : nb) + u % PER * 4;
            if constexpr (!TR) in[k] = out.get(m < m_last ? m : m_last, n < n_last ? n : n_last);
          }
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            const int u = u0 + 64 * k, r = u / PER, c = u % PER * 4, m = (TR ? nb : mb) + r, n = (TR ? mb : nb) + c;
            const bool ok = m <= m_last && n <= n_last;
            const unsigned from = mine + (TR ? c * PITCH + r : r * PITCH + c) * 4;
            if constexpr (S::GATED) {
              out.put(m, n, lds_read<v4f>(from), lds_read<v4f>(from + S::WN / 2 * 4), in[k], ok);
            } else if constexpr (S::SYM) {
              if constexpr (TR) {
                out.put(m, n, v4f{lds_read<float>(from), lds_read<float>(from + PITCH * 4), lds_read<float>(from + PITCH * 8), lds_read<float>(from + PITCH * 12)}, ok);
              } else {
                const v4f v = out.value(m, n, lds_read<v4f>(from), in[k]);
                lds_write(from, v);
                out.put(m, n, v, ok);
              }
            } else {
              out.put(m, n, lds_read<v4f>(from), in[k], ok);
            }
          }
        }
      };
      units(int_c<0>{});
      // the mirror image of a tile below the diagonal, of the values that have just left: four rows of one column
      // a unit
      if constexpr (S::SYM) {
        if (tile_m != tile_n) {
          lanes_meet();
          units(int_c<1>{});
        }
      }
    }
  }
#endif
}

}  // namespace product

#endif
