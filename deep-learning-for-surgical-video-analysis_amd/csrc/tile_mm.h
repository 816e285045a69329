// Tiled matrix product of the token-block operators (gated_ffn.hip, gemm_i8.hip):
//
//   acc[m][n] = sum_k A(m, k) B(n, k)        T = bf16, f16, float (f32 sums) or int8 (int32 sums)
//
// Each operand is stored along the reduction ("row": [m][k]) or across it ("col": [k][m]), so one kernel serves
// x W^T (row, row), dP W (row, col) and dP^T x (col, col).  A stage holds 128 bytes of k for every row of the tile
// whatever T is (64 / 32 / 128 values of k), and a lane's share of an MFMA step is always one 16-byte chunk of k:
//   16-bit: mfma 16x16x32, 8 values; int8: mfma 16x16x64, 16 values; f32: four mfma 16x16x4, value s of every
//   lane's chunk in step s (A and B agree on which k that is, so the sum is the same set of products).
// Col operands: 16-bit tiles are read back transposed by ds_read_b64_tr_b16 (as in wgrad_pk.hip), f32 by ds_read_b32.
//
// Staging: LDS-DMA (global_load_lds_dwordx4) into a ring of NS stages, one barrier a stage: a wave waits for its own
// DMA of stage t, the barrier makes everyone's visible and ends the reads of stage t - 1, whose slot is then filled
// with stage t + NS - 1 while stage t is multiplied.  16-byte chunks are XOR-swizzled on the source address so that
// fragment reads are free of bank conflicts.
//
// The MFMA is issued as B x A: a lane holds 4 consecutive n of one m, which the epilogue stores as one piece.
#pragma once
#include "svk_common.h"
#include <type_traits>

namespace svk {
namespace mm {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* las_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

static __device__ __attribute__((aligned(16))) uint4 g_zero[4];   // what a chunk past the end of K reads

// 16-byte LDS-DMA per lane: from sbase + voff (or a full address), to lds + 16 * lane
__device__ __forceinline__ void dma16s(const char* sbase, uint32_t voff, uint32_t lds) {
  const uint64_t b = reinterpret_cast<uint64_t>(sbase);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  sbase = reinterpret_cast<const char*>(((uint64_t)hi << 32) | (uint64_t)lo);
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}

template <typename T> struct Acc { typedef f32x4 t; };
template <> struct Acc<int8_t> { typedef i32x4 t; };

// one 64-byte step of k: a, b = the lane's 16-byte chunks
template <typename T>
__device__ __forceinline__ typename Acc<T>::t step(i32x4 b, i32x4 a, typename Acc<T>::t c) {
  if constexpr (__is_same(T, int8_t)) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, c, 0, 0, 0);
  } else if constexpr (__is_same(T, float)) {
    const f32x4 fb = __builtin_bit_cast(f32x4, b), fa = __builtin_bit_cast(f32x4, a);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[s], fa[s], c, 0, 0, 0);
    return c;
  } else {
    return mfma16x16x32(__builtin_bit_cast(v8_t<T>, b), __builtin_bit_cast(v8_t<T>, a), c);
  }
}

struct Args {
  const char *A, *B;
  long lda, ldb;        // bytes between rows
  int M, N;             // rows (row operands) or columns (col operands) of A and B that exist (row operand B: 32-bit
                        // byte offsets, N * ldb < 2^32; A and col operands: 256 rows of 32-bit offsets a tile)
  int K;                // reduction length in values; row operands: K * sizeof(T) % 16 == 0
  int ntm, ntn;         // tiles
  int nk, parts;        // stages in all; parts of the reduction (blockIdx.y), nk / parts stages each, rounded up
};

template <int BM_, int BN_, int WGM_, int WGN_, int NS_, int OCC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NS = NS_, OCC = OCC_;
  static constexpr int NT = 64 * WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int A_LD = A_BYTES / (NT * 16), B_LD = B_BYTES / (NT * 16), LD = A_LD + B_LD;
  static_assert(A_BYTES % (NT * 16) == 0 && B_BYTES % (NT * 16) == 0, "whole DMA rounds");
  static_assert(NS * STAGE <= 160 * 1024 && NS >= 2 && NS <= 4, "LDS ring");
};

// chunk swizzle of row r of a col image of RB bytes a row: the 8 rows x 2 chunks of a 32-lane half of a transposed read
// (16-bit: rows 8 g + q, then + 4) land in distinct banks; f32: rows 4 g + s of one ds_read_b32 in distinct 64-byte
// pieces.  A row's chunks stay within the row: RB / 16 of them.
template <typename T, int RB> __device__ __forceinline__ int col_swz(int r) {
  if constexpr (sizeof(T) == 2 && RB >= 256) return ((r & 3) << 1) | (((r >> 3) & 1) << 3);
  else if constexpr (sizeof(T) == 2) return (((r >> 1) & 1) << 1) | (((r >> 3) & 1) << 2);
  else return ((r >> 2) & 3) << 2;
}

// XCD-aware tile order: workgroup ids are dealt round-robin to the 8 XCDs, so consecutive tiles go to one XCD's L2;
// within it 8 row tiles are walked before the next column tile, for operand reuse
__device__ __forceinline__ void tile_of(int bid, int ntm, int ntn, int& tm, int& tn) {
  const int n = ntm * ntn, xcd = bid & 7, q = n >> 3, r = n & 7;
  const int p = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
  const int G = 8, per = G * ntn, grp = p / per, in = p - grp * per;
  const int g = min(G, ntm - grp * G);
  tm = grp * G + in % g;
  tn = in / g;
}

// Epi: static int row(int r, int tile): the B row of tile-local row r (row operands: which weight row it is);
//      operator()(acc, m, n, ...) writes the tile
template <typename T, class C, bool ACOL, bool BCOL, class Epi>
__global__ __launch_bounds__(C::NT, C::OCC) void tile_mm(Args p, Epi epi) {
  constexpr int ES = sizeof(T), BK = 128 / ES;
  constexpr int TM = C::TM, TN = C::TN, NS = C::NS;
  typedef typename Acc<T>::t acc_t;
  static_assert(!(ACOL || BCOL) || ES >= 2, "col operands: 16 / 32-bit");
  static_assert((C::BM * ES >= 128 && C::BN * ES >= 128) || !(ACOL || BCOL), "col images: rows of 8 chunks or more");
  __shared__ __attribute__((aligned(1024))) char smem[NS * C::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int fr = lane & 15, fq = lane >> 4;
  int tm, tn;
  tile_of(blockIdx.x, p.ntm, p.ntn, tm, tn);
  const int per = (p.nk + p.parts - 1) / p.parts;
  const int k0 = blockIdx.y * per, k1 = min(k0 + per, p.nk);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(las_ptr)smem;

  // DMA plan: instruction i of this wave fills 1 KiB = rows of the stage image.  Row operands: 8 rows of 128 bytes;
  // col operands: 1024 / (tile bytes a row of k) rows of k.
  constexpr int ARB = ACOL ? C::BM * ES : 128, BRB = BCOL ? C::BN * ES : 128;      // image row bytes
  uint32_t offA[C::A_LD], offB[C::B_LD];
  const char* baseA = p.A + (ACOL ? (long)tm * C::BM * ES : (long)tm * C::BM * p.lda);
  const char* baseB = p.B + (BCOL ? (long)tn * C::BN * ES : 0);
  auto img = [&](int i, int rb, int& row, int& slot) {          // image row and chunk slot of this lane's 16 bytes
    const int at = (wave + i * (C::NT / 64)) * 1024 + lane * 16;
    row = at / rb;
    slot = (at % rb) >> 4;
  };
#pragma unroll
  for (int i = 0; i < C::A_LD; ++i) {
    int r, s;
    img(i, ARB, r, s);
    if constexpr (ACOL) {
      const int last = (p.M * ES - 1) / 16 - tm * (C::BM * ES / 16);   // last chunk of the row that exists
      offA[i] = (uint32_t)r * (uint32_t)p.lda + min(s ^ col_swz<T, ARB>(r), last) * 16;
    } else {
      offA[i] = (uint32_t)min(r, p.M - 1 - tm * C::BM) * (uint32_t)p.lda + ((s ^ (r & 7)) << 4);
    }
  }
#pragma unroll
  for (int i = 0; i < C::B_LD; ++i) {
    int r, s;
    img(i, BRB, r, s);
    if constexpr (BCOL) {
      const int last = (p.N * ES - 1) / 16 - tn * (C::BN * ES / 16);
      offB[i] = (uint32_t)r * (uint32_t)p.ldb + min(s ^ col_swz<T, BRB>(r), last) * 16;
    } else {
      offB[i] = (uint32_t)epi.template row<C>(r, tn) * (uint32_t)p.ldb + ((s ^ (r & 7)) << 4);   // by the epilogue's map
    }
  }
  const char* zero = reinterpret_cast<const char*>(g_zero);
  auto issue = [&](int kt) {
    const uint32_t sa = lds0 + ((kt - k0) % NS) * C::STAGE, sb = sa + C::A_BYTES;
    const bool tail = (kt + 1) * BK > p.K;
#pragma unroll
    for (int i = 0; i < C::A_LD; ++i) {
      const uint32_t dst = sa + (wave + i * (C::NT / 64)) * 1024;
      const char* src = baseA + (ACOL ? (long)kt * BK * p.lda : (long)kt * 128);
      if (!tail) dma16s(src, offA[i], dst);
      else {
        int r, s;
        img(i, ARB, r, s);
        const int k = kt * BK + (ACOL ? r : (s ^ (r & 7)) * (16 / ES));
        dma16(k < p.K ? src + offA[i] : zero, dst);
      }
    }
#pragma unroll
    for (int i = 0; i < C::B_LD; ++i) {
      const uint32_t dst = sb + (wave + i * (C::NT / 64)) * 1024;
      const char* src = baseB + (BCOL ? (long)kt * BK * p.ldb : (long)kt * 128);
      if (!tail) dma16s(src, offB[i], dst);
      else {
        int r, s;
        img(i, BRB, r, s);
        const int k = kt * BK + (BCOL ? r : (s ^ (r & 7)) * (16 / ES));
        dma16(k < p.K ? src + offB[i] : zero, dst);
      }
    }
  };

  acc_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = acc_t{0, 0, 0, 0};

  // the lane's 16-byte chunk of k (step ks) of row `row0 + fr` of an operand image
  auto frag = [&](const char* im, int row0, int ks, auto COL_, auto RB_) -> i32x4 {
    constexpr bool COL = decltype(COL_)::value;
    constexpr int rb = decltype(RB_)::value;           // bytes of an image row
    if constexpr (!COL) {
      const int r = row0 + fr;
      return *reinterpret_cast<const i32x4*>(im + r * 128 + (((ks * 4 + fq) ^ (r & 7)) << 4));
    } else if constexpr (ES == 2) {
      // lane 4 q + c of a 16-lane group addresses row q, columns 4 c ..: the group's lane i receives column i
      const int q = fr >> 2, c = fr & 3;
      s16x4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = ks * 32 + fq * 8 + h * 4 + q, col = row0 + c * 4;
        const char* at = im + r * rb + (((col >> 3) ^ col_swz<T, rb>(r)) << 4) + ((col >> 2) & 1) * 8;
        v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(las_ptr)at);
      }
      return __builtin_bit_cast(i32x4, s16x8{v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w});
    } else {
      i32x4 v;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int r = ks * 16 + fq * 4 + s, col = row0 + fr;
        v[s] = *reinterpret_cast<const int*>(im + r * rb + (((col >> 2) ^ col_swz<T, rb>(r)) << 4) + (col & 3) * 4);
      }
      return v;
    }
  };

#pragma unroll
  for (int t = 0; t < NS - 1; ++t)
    if (k0 + t < k1) issue(k0 + t);
  for (int kt = k0; kt < k1; ++kt) {
    const int later = min(k1 - 1 - kt, NS - 2);                 // stages issued after this one
    if (NS > 3 && later == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C::LD) : "memory");
    else if (NS > 2 && later == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::LD) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + NS - 1 < k1) issue(kt + NS - 1);
    const char* ia = smem + ((kt - k0) % NS) * C::STAGE;
    const char* ib = ia + C::A_BYTES;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x4 fa[TM], fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = frag(ib, wn * C::WN + j * 16, ks, std::integral_constant<bool, BCOL>{}, std::integral_constant<int, BRB>{});
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = frag(ia, wm * C::WM + i * 16, ks, std::integral_constant<bool, ACOL>{}, std::integral_constant<int, ARB>{});
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = step<T>(fb[j], fa[i], acc[i][j]);
    }
  }
  epi.template write<C>(acc, tm * C::BM + wm * C::WM + fr, tn, wn, fq);
}

// 16 (or fewer, at the end) token rows against the weights: each weight value is read once, straight into
// registers, and the reduction is split over the workgroup's waves and joined in LDS.  MT blocks of 16 tokens, 2
// blocks of 16 weight rows (the epilogue's map names them).  VEC: rows 16-byte aligned and whole 16-byte chunks;
// otherwise chunks are put together value by value.
constexpr int SK_WAVES = 8;

template <typename T, bool VEC>
__device__ __forceinline__ i32x4 load_chunk(const char* row, long kb, long kbytes) {
  constexpr int ES = sizeof(T);
  if constexpr (VEC) {
    return kb < kbytes ? *reinterpret_cast<const i32x4*>(row + kb) : i32x4{0, 0, 0, 0};
  } else {
    // 32-bit storage of the chunk's values, taken one by one
    union { i32x4 v; T e[16 / ES]; } u;
    u.v = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i)
      if (kb + i * ES < kbytes) u.e[i] = *reinterpret_cast<const T*>(row + kb + i * ES);
    return u.v;
  }
}

template <typename T, int MT, bool VEC, class Epi>
__global__ __launch_bounds__(64 * SK_WAVES) void skinny_mm(Args p, Epi epi) {
  typedef typename Acc<T>::t acc_t;
  constexpr int U = VEC ? 4 : 1;                                // 64-byte steps in flight
  typedef std::conditional_t<std::is_same<T, int8_t>::value, int, float> sum_t;
  __shared__ sum_t red[SK_WAVES][MT][2][16][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const long kbytes = (long)p.K * sizeof(T);
  const char* rb[2];
  const char* ra[MT];
#pragma unroll
  for (int j = 0; j < 2; ++j) rb[j] = p.B + (long)epi.skinny_row(blockIdx.x, j, fr) * p.ldb;
#pragma unroll
  for (int i = 0; i < MT; ++i) ra[i] = p.A + (long)min(i * 16 + fr, p.M - 1) * p.lda;
  acc_t acc[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
  for (long kb = (long)wave * 64 * U; kb < kbytes; kb += (long)SK_WAVES * 64 * U) {
    i32x4 fb[U][2], fa[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long k = kb + u * 64 + fq * 16;
#pragma unroll
      for (int j = 0; j < 2; ++j) fb[u][j] = load_chunk<T, VEC>(rb[j], k, kbytes);
#pragma unroll
      for (int i = 0; i < MT; ++i) fa[u][i] = load_chunk<T, VEC>(ra[i], k, kbytes);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = step<T>(fb[u][j], fa[u][i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][i][j][fr][fq * 4 + e] = acc[i][j][e];
  __syncthreads();
  for (int t = tid; t < MT * 256; t += 64 * SK_WAVES) {
    const int i = t >> 8, m = (t >> 4) & 15, n = t & 15;
    sum_t v[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < SK_WAVES; ++w) v[j] += red[w][i][j][m][n];
    if (i * 16 + m < p.M) epi.skinny_write(blockIdx.x, i * 16 + m, n, v[0], v[1]);
  }
}

// copy of rows of `width` values into rows of `ld` values (a multiple of 16 bytes), the rest filled with zeros: what
// the tiled kernels read where a row operand's length or address is no whole number of 16-byte chunks
template <typename T>
__global__ __launch_bounds__(256) void pad_rows(const T* __restrict__ X, long ldx, T* __restrict__ Y, long ld, long rows,
                                                int width) {
  const long total = rows * ld;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long r = i / ld, c = i - r * ld;
    Y[i] = c < width ? X[r * ldx + c] : T(0);
  }
}

inline long up16(long bytes) { return (bytes + 15) & ~15L; }
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace mm
}  // namespace svk
