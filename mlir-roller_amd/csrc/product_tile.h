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
// The K loop is software pipelined over two LDS buffers: the loads of step k+1 are in flight while
// step k is multiplied, the fragments of the next 128-byte half are read beside the MFMAs of the
// current one, also across the barrier between steps.

#ifndef PRODUCT_TILE_H
#define PRODUCT_TILE_H

#include <hip/hip_runtime.h>

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
constexpr int XCDS = 8;

template <int V>
struct int_c {
  static constexpr int value = V;
};

PT_DEV __amdgpu_buffer_rsrc_t live_rsrc(const void* p, bool live) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, live ? 0x7fffffff : 0, 0x00020000);
}

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
  PT_DEV acc_t run(v4u a, v4u b, acc_t c) {
    if constexpr (sizeof(T) == 4) {
      const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (MI == 16) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
        else c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[t], y[t], c, 0, 0, 0);
      }
      return c;
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
};

// Permutation of the 16-byte chunks of row k of a row-major tile whose rows are ROW_BYTES long (XOR-ed
// onto the chunk number).
//   16 bits: half a wave reads 64 bytes (32 rows of the product) from each of the rows k .. k+3; the four
//   must lie in four different quarters of the 256 bytes that the banks span.  A row of 128 bytes already
//   differs from its neighbour by its own length.
//   32 bits: half a wave reads 128 bytes of one row, which covers the 32 banks of a 32-bit read as it is.
template <int ES, int ROW_BYTES>
PT_DEV constexpr int mn_swizzle(int k) {
  if constexpr (ES == 4) {
    return 0;
  } else if constexpr (ROW_BYTES >= 256) {
    return (k & 3) * 4;
  } else {
    static_assert(ROW_BYTES == 128, "tiles are at least 64 rows of 16 bits");
    return ((k >> 1) & 1) * 4;
  }
}

#if __HIP_DEVICE_COMPILE__
// LDS by address (a kernel's one __shared__ array starts at 0)
template <class V>
PT_DEV V lds_read(unsigned at) {
  return *(const __attribute__((address_space(3))) V*)at;
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
  int M_out, N_out;   // rows and columns handed to the epilogue (those beyond M and N are zeros: the padding
                      // of a buffer that a later product reads as K-major)
  long batch_a, batch_b;
  int splits, steps_per_split;   // workgroups that share a tile's K steps, and how many each takes
};

// Tile shape, operand forms and options of one kernel.
//   A_KM, B_KM  K-major (1) or row-major in k (0)
//   GATED       the tile's columns are BN/2 gate columns and the same BN/2 up columns, laid out so that
//               a lane has both of a column (accumulator blocks j and j + TN/2)
//   SEGS        K segments
//   SYM         the result is symmetric: only the tiles on and below the diagonal exist
template <class T_, int BM_, int BN_, int WM_, int WN_, int A_KM_, int B_KM_, int GATED_ = 0, int SEGS_ = 1, int SYM_ = 0, int PER_CU_ = 1, int MI_ = 32>
struct Shape {
  typedef T_ T;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, A_KM = A_KM_, B_KM = B_KM_, GATED = GATED_, SEGS = SEGS_, SYM = SYM_;
  static constexpr int PER_CU = PER_CU_;   // workgroups that should fit a CU
  static constexpr int NWM = BM / WM, NWN = BN / WN, WAVES = NWM * NWN, NT = 64 * WAVES;
  static constexpr int ES = sizeof(T), KSTEP = STEP_BYTES / ES;
  static constexpr int MI = MI_, TM = WM / MI, TN = WN / MI;
  static constexpr int ROUNDS = MI / 8;               // fragment rounds per K step: each takes 64 / MI of its 8 chunks
  static constexpr int A_BYTES = BM * STEP_BYTES, B_BYTES = BN * STEP_BYTES;
  static constexpr int LDS_BYTES = 2 * (A_BYTES + B_BYTES);
  static constexpr int A_LOADS = BM * 8 / NT, B_LOADS = BN * 8 / NT;
  static constexpr int OUT_N = GATED ? BN / 2 : BN;   // result columns per tile
  static_assert(BM % WM == 0 && BN % WN == 0 && WM % MI == 0 && WN % MI == 0, "tile");
  static_assert((BM * 8) % NT == 0 && (BN * 8) % NT == 0, "whole loads per thread");
  static_assert(!GATED || ((WN / 2) % MI == 0 && B_KM), "gate and up halves of a wave tile");
  static_assert(!SYM || BM == BN, "square tiles");
  static_assert(MI == 32 || (A_KM && B_KM), "row-major tiles are read 32 rows at a time");
};

// Orders the next NM MFMAs and NO instructions of class MASK evenly (0x100 LDS read, 0x020 global read).
template <int NM, int NO, int MASK>
PT_DEV void interleave() {
  if constexpr (NM > 0) {
    constexpr int q = NO / NM, rem = NO % NM;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i < rem) {
        __builtin_amdgcn_sched_group_barrier(MASK, q + 1, 0);
      } else if (q > 0) {
        __builtin_amdgcn_sched_group_barrier(MASK, q > 0 ? q : 1, 0);
      }
    }
  }
}

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

// tile number p of the lower triangle, row by row: (p's row, column)
PT_DEV void triangle_tile(int p, int& tm, int& tn) {
  int r = (int)((__builtin_sqrtf(8.0f * (float)p + 1.0f) - 1.0f) * 0.5f);
  while ((long)(r + 1) * (r + 2) / 2 <= p) ++r;
  while ((long)r * (r + 1) / 2 > p) --r;
  tm = r;
  tn = p - (int)((long)r * (r + 1) / 2);
}

// Part of a split product: fp32, one slab of rows x pitch per split and batch entry (GATED: two, gate and up).
struct Partial {
  float* slab;
  int pitch;
  long slab_size;   // rows * pitch
  int per_split;    // slabs per split
  __device__ __forceinline__ Partial at(int batch, int split) const {
    Partial o = *this;
    o.slab += ((long)split * per_split + batch) * slab_size;
    return o;
  }
  __device__ __forceinline__ void put(int m, int n, v4f v) const { *(v4f*)(slab + (long)m * pitch + n) = v; }
  __device__ __forceinline__ void put(int m, int n, v4f gate, v4f up) const {
    put(m, n, gate);
    *(v4f*)(slab + slab_size + (long)m * pitch + n) = up;
  }
};

template <class S, class Epi>
__global__ __launch_bounds__(S::NT, S::PER_CU * S::WAVES / 4 > 0 ? S::PER_CU * S::WAVES / 4 : 1) void tile_kernel(const Problem p, const Partial partial, const Epi epi) {
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
  int pid = blockIdx.x;
  const int split = pid / tiles;                 // (grid.x = tiles * splits)
  pid = xcd_order(pid - split * tiles, tiles);
  int tile_m, tile_n;
  if constexpr (S::SYM) {
    triangle_tile(pid, tile_m, tile_n);
  } else {
    panel_tile(pid, nbm, nbn, tile_m, tile_n);
  }
  const int m0 = tile_m * S::BM, n0 = tile_n * S::OUT_N;
  const int batch = blockIdx.z;

  // K steps of this workgroup.  A segment is a whole number of steps: its last step is cut by K.
  const int seg_steps = (p.K + S::KSTEP - 1) / S::KSTEP;
  const int first_step = split * p.steps_per_split;
  const int all_steps = seg_steps * S::SEGS;
  const int last_step = first_step + p.steps_per_split < all_steps ? first_step + p.steps_per_split : all_steps;
  const int KT = last_step - first_step;

  // ---- what each lane fetches: offsets from the tile's first element, fixed through the K loop ----
  unsigned a_off[S::A_LOADS], b_off[S::B_LOADS];
  int a_k, b_k[1];   // first k of the lane's chunks within a step (K-major: the same for every load of the lane)
  // K-major: unit u is chunk (u % 8) ^ ((row / 2) % 8) of row u / 8; the rows of a lane's loads are NT / 8
  // apart, a multiple of 16, so the chunk is the same for all of them.
  static_assert(NT % 128 == 0 || (!S::A_KM && !S::B_KM), "the chunk of a lane's K-major loads is the same for all");
  const int km_chunk = (tid & 7) ^ ((tid >> 4) & 7);
  a_k = b_k[0] = km_chunk * (16 / ES);
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

  // Issues the loads of K step kt (of this workgroup) into LDS buffer `buf`.  KTEST: the step may be one
  // that K cuts short.  A step at or beyond KT gets an empty resource: zeros, no memory touched.
  auto fetch = [&](auto ktest, int kt, int buf) __attribute__((always_inline)) {
    constexpr bool KTEST = decltype(ktest)::value;
    const bool live = kt < KT;
    int step = first_step + (live ? kt : 0), seg = 0;
    if constexpr (S::SEGS > 1) {
      if (step >= seg_steps) { step -= seg_steps; seg = 1; }
      if constexpr (S::SEGS > 2) {
        if (step >= seg_steps) { step -= seg_steps; seg = 2; }
      }
    }
    const T* ap = (const T*)(S::SEGS > 1 && seg == 1 ? p.a[1] : S::SEGS > 2 && seg == 2 ? p.a[2] : p.a[0]) + a_tile + step * a_step;
    const T* bp = (const T*)(S::SEGS > 1 && seg == 1 ? p.b[1] : S::SEGS > 2 && seg == 2 ? p.b[2] : p.b[0]) + b_tile + step * b_step;
    const __amdgpu_buffer_rsrc_t ar = live_rsrc(ap, live), br = live_rsrc(bp, live);
    const int k_left = p.K - step * S::KSTEP;
    char* As = lds + buf * S::A_BYTES;
    char* Bs = lds + 2 * S::A_BYTES + buf * S::B_BYTES;
#pragma unroll
    for (int i = 0; i < S::A_LOADS; ++i) {
      unsigned off = a_off[i];
      if constexpr (KTEST) {
        if constexpr (S::A_KM) {
          off = a_k < k_left ? off : OOB;
        } else {
          off = (tid + i * NT) / (S::BM * ES / 16) < k_left ? off : OOB;
        }
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, (lds_ptr)(As + (i * NT + wave * 64) * 16), 16, off, 0, 0, 0);
    }
    __amdgpu_buffer_rsrc_t br1 = br;
    if constexpr (S::GATED) br1 = live_rsrc((const T*)p.b[1] + b_tile1 + step * S::KSTEP, live);
#pragma unroll
    for (int i = 0; i < S::B_LOADS; ++i) {
      unsigned off = b_off[i];
      if constexpr (KTEST) {
        if constexpr (S::B_KM) {
          off = b_k[0] < k_left ? off : OOB;
        } else {
          off = (tid + i * NT) / (S::BN * ES / 16) < k_left ? off : OOB;
        }
      }
      if constexpr (S::GATED) {
        const int row = i * (NT / 8) + wave * 8;   // the 8 rows of this wave's load are all gate or all up
        __builtin_amdgcn_raw_ptr_buffer_load_lds(row % S::WN < S::WN / 2 ? br : br1, (lds_ptr)(Bs + (i * NT + wave * 64) * 16), 16, off, 0, 0, 0);
      } else {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(br, (lds_ptr)(Bs + (i * NT + wave * 64) * 16), 16, off, 0, 0, 0);
      }
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
      b_at[h] = 2 * S::A_BYTES + (wn0 + lr) * STEP_BYTES + ((64 / MI * h + lg) ^ ((lr >> 1) & 7)) * 16;
      opaque(b_at[h]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      b_at[j] = 2 * S::A_BYTES + rows_at<ES, S::BN * ES>(wn0 + MI * j, lane);
      opaque(b_at[j]);
    }
  }
  auto read = [&](frags& f, auto buf_c, auto round_c) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value, round = decltype(round_c)::value;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if constexpr (S::A_KM) {
        f.a[i] = lds_read<v4u>(a_at[round] + (buf * S::A_BYTES + i * MI * STEP_BYTES));
      } else {
        f.a[i] = read_rows<ES, S::BM * ES>(a_at[i] + (buf * S::A_BYTES + round * (S::KSTEP / ROUNDS) * S::BM * ES));
      }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if constexpr (S::B_KM) {
        f.b[j] = lds_read<v4u>(b_at[round] + (buf * S::B_BYTES + j * MI * STEP_BYTES));
      } else {
        f.b[j] = read_rows<ES, S::BN * ES>(b_at[j] + (buf * S::B_BYTES + round * (S::KSTEP / ROUNDS) * S::BN * ES));
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
  auto multiply = [&](const frags& f, int i0, int i1) __attribute__((always_inline)) {
#pragma unroll
    for (int i = i0; i < i1; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma<T, MI>::run(f.b[j], f.a[i], acc[i][j]);
  };

  // ---- K loop ----
  constexpr int G = TM * TN * mma<T, MI>::PER_FRAG;                // MFMAs per round
  constexpr int RA = S::A_KM ? TM : TM * (ES == 2 ? 2 : 4), RB = S::B_KM ? TN : TN * (ES == 2 ? 2 : 4);
  constexpr int R = RA + RB, L = S::A_LOADS + S::B_LOADS;
  constexpr int EARLY = TM >= 4 ? TM / 4 : 0;                      // block rows multiplied before the barrier
  if (KT > 0) {
    frags f[2];
    fetch(int_c<1>{}, 0, 0);
    fetch(int_c<1>{}, 1, 1);
    __builtin_amdgcn_s_waitcnt(0x0f70 | (L & 0xf) | ((L >> 4) << 14));   // vmcnt <= L: step 0 has landed
    __syncthreads();
    read(f[0], int_c<0>{}, int_c<0>{});
    auto step = [&](auto ktest, auto cur_c, int kt) __attribute__((always_inline)) {
      constexpr int cur = decltype(cur_c)::value;
      read(f[1], cur_c, int_c<1>{});
      multiply(f[0], 0, TM);
      if constexpr (ROUNDS == 4) {
        read(f[0], cur_c, int_c<2 % ROUNDS>{});
        multiply(f[1], 0, TM);
        read(f[1], cur_c, int_c<3 % ROUNDS>{});
        multiply(f[0], 0, TM);
      }
#pragma unroll
      for (int r = 1; r < ROUNDS; ++r) interleave<G, R, 0x100>();
      multiply(f[1], 0, EARLY);
      interleave<G * EARLY / TM, 0, 0x100>();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt 0: step kt + 1 has landed
      __syncthreads();
      read(f[0], int_c<1 - cur>{}, int_c<0>{});
      fetch(ktest, kt + 2, cur);
      multiply(f[1], EARLY, TM);
      constexpr int REST = G - G * EARLY / TM;
      interleave<(R < REST ? R : REST), R, 0x100>();
      if constexpr (REST > R) interleave<REST - R, L, 0x020>();
      __builtin_amdgcn_sched_barrier(0);
    };
    int kt = 0;
    // steps whose fetch (of kt + 2) cannot be cut short by the end of K (of any segment)
    const int cut_free = p.K % S::KSTEP == 0 ? KT : (S::SEGS > 1 ? 0 : (last_step == seg_steps ? KT - 3 : KT));
    for (; kt + 1 < KT && kt + 1 < cut_free; kt += 2) {
      step(int_c<0>{}, int_c<0>{}, kt);
      step(int_c<0>{}, int_c<1>{}, kt + 1);
    }
    for (; kt + 1 < KT; kt += 2) {
      step(int_c<1>{}, int_c<0>{}, kt);
      step(int_c<1>{}, int_c<1>{}, kt + 1);
    }
    if (kt < KT) step(int_c<1>{}, int_c<0>{}, kt);
    __builtin_amdgcn_s_waitcnt(0x0f70);   // the empty requests past the end have drained
  }

  // ---- every accumulator leaves once: row m, columns n to n + 3 ----
  auto leave = [&](auto out) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + wm0 + i * MI + lr;
#pragma unroll
      for (int j = 0; j < (S::GATED ? TN / 2 : TN); ++j)
#pragma unroll
        for (int q = 0; q < REGS / 4; ++q) {
          // registers 4q .. 4q+3 of lane group lg: columns 256 / MI * q + 4 * lg and on of the block
          const int col = j * MI + 256 / MI * q + 4 * lg;
          auto four = [&](int jj) __attribute__((always_inline)) { return v4f{acc[i][jj][4 * q], acc[i][jj][4 * q + 1], acc[i][jj][4 * q + 2], acc[i][jj][4 * q + 3]}; };
          if constexpr (S::GATED) {
            const int n = n0 + (wave % S::NWN) * (S::WN / 2) + col;
            if (m < p.M_out && n < p.N_out) out.put(m, n, four(j), four(j + TN / 2));
          } else {
            const int n = n0 + wn0 + col;
            if (m < p.M_out && n < p.N_out) out.put(m, n, four(j));
          }
        }
    }
  };
  if (p.splits > 1) {
    leave(partial.at(batch, split));
  } else {
    leave(epi.at(batch, 0));
  }
#endif
}

}  // namespace product

#endif
