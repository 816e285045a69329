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
// Staging: LDS-DMA (buffer_load ... lds, 16 bytes a lane) into a ring of NS stages.  A stage is two MFMA steps of 64
// bytes of k; the fragments of one step are read while the other's are multiplied, so the LDS reads run under the MFMAs.
// The stage's one barrier stands between its two steps: by then every wave holds the second step's fragments in
// registers and its own DMA of the next stage has landed, so behind it the next stage can be read and this stage's slot
// filled again.  That DMA is dealt between the MFMAs of the second step (issued in one go it held the wave's MFMAs up:
// 16384 x 11264 x 2048 in bf16 went from 755 to 707 us with the persistent form below).
// The lane offsets of the DMA are the same for every tile and stage; a tile or a stage is a descriptor's base, and its
// range check gives zeros for rows past the end, so there is no branch and no address arithmetic in the loop.
//
// Persistent: the grid walks a stream of (tile, stage) and the DMA runs NS stages ahead of the products across tile
// ends, so a tile's first stages are there when the last tile's results are written.  Results of the 256 x 256 tiles
// are stored past the L2 (they are larger than it, and evicted the operands: 664 -> 631 us at the size above).
// What is left (618 us, 1223 TFLOP/s; 1336 at 8192^3, where a plain library product reaches 1442): every CU writes its
// tile at the same time, about 6 us a tile that nothing covers.
//
// The MFMA is issued as B x A: a lane holds 4 consecutive n of one m; pairs of 16-column blocks of a row operand B are
// interleaved by fours, so that two blocks hold 8 consecutive n, one 16-byte store of a 16-bit type.
#pragma once
#include "svk_common.h"
#include <type_traits>

namespace svk {
namespace mm {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* las_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t OUTSIDE = 0xFFFFFFF0u;      // a lane offset past every descriptor's range: reads zeros

// buffer descriptor of the `left` bytes behind base (32-bit offsets; reads past them give zeros)
__device__ __forceinline__ i32x4 descriptor(const char* base, long left) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const uint32_t n = left <= 0 ? 0u : (left > 0xFFFFFF00L ? 0xFFFFFF00u : (uint32_t)left);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(b >> 32) & 0xFFFFu));
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;                           // raw 32-bit data
  return r;
}
// 16 bytes a lane from the descriptor's base + voff to LDS lds + 16 * lane
__device__ __forceinline__ void dma16(i32x4 r, uint32_t voff, uint32_t lds) {
  // (m0 is told as clobbered rather than kept and put back: two scalar instructions a piece, 1.2 % of a large product)
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "s"(lds) : "memory", "m0");
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
  long abytes, bbytes;  // bytes from A (B) to the end of its last row
  int M, K;             // token rows (skinny_mm); reduction length in values
  int ntm, ntn;         // tiles
  int nk, parts;        // stages of the reduction; parts it is split into, nk / parts stages each, rounded up, none empty
};

template <int BM_, int BN_, int WGM_, int WGN_, int NS_, int OCC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NS = NS_, OCC = OCC_;
  static constexpr int NT = 64 * WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int A_LD = A_BYTES / (NT * 16), B_LD = B_BYTES / (NT * 16), LD = A_LD + B_LD;
  static constexpr bool NONTEMPORAL = BM >= 256;
  static_assert(A_BYTES % (NT * 16) == 0 && B_BYTES % (NT * 16) == 0, "whole DMA rounds");
  static_assert(NS * STAGE <= 160 * 1024 && NS >= 2 && (NS - 1) * LD <= 63, "LDS ring, wait counter");
};

// chunk swizzle of row r of a col image of RB bytes a row: the 8 rows x 2 chunks of a 32-lane half of a transposed read
// (16-bit: rows 8 g + q, then + 4) land in distinct banks; f32: rows 4 g + s of one ds_read_b32 in distinct 64-byte
// pieces.  A row's chunks stay within the row: RB / 16 of them.
template <typename T, int RB> __device__ __forceinline__ int col_swz(int r) {
  if constexpr (sizeof(T) == 2 && RB >= 256) return ((r & 3) << 1) | (((r >> 3) & 1) << 3);
  else if constexpr (sizeof(T) == 2) return (((r >> 1) & 1) << 1) | (((r >> 3) & 1) << 2);
  else return ((r >> 2) & 3) << 2;
}

// XCD-aware tile order: workgroups are dealt round-robin to the 8 XCDs, so consecutive tiles go to one XCD's L2; within
// it 4 row tiles are walked before the next column tile, for operand reuse (2, 4, 8: within 1 %; 16: 3 % slower)
__device__ __forceinline__ void tile_of(int bid, int ntm, int ntn, int& tm, int& tn) {
  const int n = ntm * ntn, xcd = bid & 7, q = n >> 3, r = n & 7;
  const int p = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
  const int G = 4, per = G * ntn, grp = p / per, in = p - grp * per;
  const int g = min(G, ntm - grp * G);
  tm = grp * G + in % g;
  tn = in / g;
}

// W consecutive values of a row: one store (of any alignment) where all W exist, else one by one.  NTS: past the L2
template <typename T, int W, bool NTS>
__device__ __forceinline__ void put(T* at, const float* v, int n) {
  T o[W];
#pragma unroll
  for (int e = 0; e < W; ++e) o[e] = from_f<T>(v[e]);
  typedef uint32_t vec __attribute__((ext_vector_type(W * sizeof(T) / 4)));
  typedef vec anywhere __attribute__((aligned(2)));
  if (n >= W) {
    vec w;
    __builtin_memcpy(&w, o, sizeof(w));
    if constexpr (NTS) __builtin_nontemporal_store(w, reinterpret_cast<anywhere*>(at));
    else *reinterpret_cast<anywhere*>(at) = w;
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < n) at[e] = o[e];
  }
}

// position of tile-local B row r among the columns of its 32-column group: blocks of 16 interleaved by fours
__device__ __forceinline__ int pair_col(int r) { return (r & ~31) + 8 * ((r >> 2) & 3) + 4 * ((r >> 4) & 1) + (r & 3); }

// GELU (erf form) for results of 16 bits: relu(x) - |x| erfc(|x| / sqrt 2) / 2 with erfc by Abramowitz & Stegun 7.1.26
// (|error| <= 1.5e-7): erfc(z) = t q(t) exp(-z^2), t = 1 / (1 + c z).  12 plain and 2 transcendental instructions; the
// epilogues of short reductions are bound by them.  The result is off by 0.75e-7 |x| at most: under half a step down to
// x = -3.5 in f16 and -5 in bf16.  Further down it is not (f16 1.9 half steps at -4.2, of a result of 6e-5; bf16 1.8 at -6
// and 3.2 at -7, of results of 1e-8 and less), where x (1 + erf) / 2 in f32 has lost more: all of its digits from -5.5 on.
__device__ __forceinline__ float gelu16(float x) {
  constexpr float c = 0.3275911f * 0.70710678118654752f, s = -0.5f;
  const float t = __builtin_amdgcn_rcpf(fmaf(c, fabsf(x), 1.0f));
  float q = fmaf(s * 1.061405429f, t, s * -1.453152027f);
  q = fmaf(q, t, s * 1.421413741f);
  q = fmaf(q, t, s * -0.284496736f);
  q = fmaf(q, t, s * 0.254829592f);
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);                // -x^2 / 2 * log2(e)
  // medians: |x| bounded (infinity times t = 0 is no number), and x where it is positive; one instruction each
  return fmaf(__builtin_amdgcn_fmed3f(fabsf(x), 0.f, 1e4f) * t * q, e, __builtin_amdgcn_fmed3f(x, 0.f, INFINITY));
}

// Epi (row operand B): uint32_t offset<C>(r, ldb): bytes from the tile's first row to B row r of the tile;
//                      long first<C>(tn): the tile's first row
//      write<C>(acc, m, tn, wn, fq, part): stores the tile; acc[i][j]: row m + 16 i, columns 4 fq .. of block j
//      M: its rows;  skip(rows): begins that many rows later
template <typename T, class C, bool ACOL, bool BCOL, class Epi>
__global__ __launch_bounds__(C::NT, C::OCC) void tile_mm(Args p, Epi epi) {
  constexpr int ES = sizeof(T), BK = 128 / ES;
  constexpr int TM = C::TM, TN = C::TN, NS = C::NS;
  typedef typename Acc<T>::t acc_t;
  static_assert(!(ACOL || BCOL) || (ES >= 2 && C::BM * ES >= 128 && C::BN * ES >= 128), "col operands: 16 / 32-bit, rows of 8 chunks or more");
  __shared__ __attribute__((aligned(1024))) char smem[NS * C::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int fr = lane & 15, fq = lane >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(las_ptr)smem;
  constexpr int ARB = ACOL ? C::BM * ES : 128, BRB = BCOL ? C::BN * ES : 128;      // image row bytes
  const int units = p.ntm * p.ntn * p.parts, per = (p.nk + p.parts - 1) / p.parts;
  const int stride = gridDim.x;
  if ((int)blockIdx.x >= units) return;

  // DMA piece q of a stage: 1 KiB a wave of A's image, of B's from q = A_LD on
  uint32_t offs[C::LD];
#pragma unroll
  for (int q = 0; q < C::LD; ++q) {
    const bool isA = q < C::A_LD;
    const int rb = isA ? ARB : BRB, at = (wave + (isA ? q : q - C::A_LD) * (C::NT / 64)) * 1024 + lane * 16;
    const int r = at / rb, s = (at % rb) >> 4;                  // image row, chunk slot
    if (isA) offs[q] = (uint32_t)r * (uint32_t)p.lda + (ACOL ? s ^ col_swz<T, ARB>(r) : s ^ (r & 7)) * 16;
    else if constexpr (BCOL) offs[q] = (uint32_t)r * (uint32_t)p.ldb + (s ^ col_swz<T, BRB>(r)) * 16;
    else offs[q] = epi.template offset<C>(r, (uint32_t)p.ldb) + (s ^ (r & 7)) * 16;
  }
  const int kin = ((lane & 7) ^ (lane >> 3)) * (16 / ES);       // first k, within the stage, of a row operand's chunk

  // the DMA's place in the stream: unit, stage, ring slot; its operand bases and the bytes behind them
  int du = blockIdx.x, dkt = 0, dend = 0, dslot = 0;
  const char *dA = nullptr, *dB = nullptr;
  long lA = 0, lB = 0;
  const long stepA = ACOL ? (long)BK * p.lda : 128, stepB = BCOL ? (long)BK * p.ldb : 128;
  auto start = [&]() {
    int tm, tn;
    const int t = du / p.parts, part = du - t * p.parts;
    tile_of(t, p.ntm, p.ntn, tm, tn);
    dkt = part * per;
    dend = min(dkt + per, p.nk);
    const long oa = (ACOL ? (long)tm * C::BM * ES : (long)tm * C::BM * p.lda) + dkt * stepA;
    long ob;
    if constexpr (BCOL) ob = (long)tn * C::BN * ES + dkt * stepB;
    else ob = epi.template first<C>(tn) * p.ldb + dkt * stepB;
    dA = p.A + oa;
    dB = p.B + ob;
    lA = p.abytes - oa;
    lB = p.bbytes - ob;
  };
  i32x4 ra, rb;
  uint32_t dlds = 0;
  auto aim = [&]() {                                            // past the end of the stream: reads nothing
    const bool live = du < units;
    ra = descriptor(dA, live ? lA : 0);
    rb = descriptor(dB, live ? lB : 0);
    dlds = lds0 + dslot * C::STAGE;
  };
  auto piece = [&](int q) {                                     // q: a constant once unrolled
    const bool isA = q < C::A_LD, col = isA ? ACOL : BCOL;
    const uint32_t off = col || dkt * BK + kin < p.K ? offs[q] : OUTSIDE;
    dma16(isA ? ra : rb, off, dlds + (isA ? 0 : C::A_BYTES) + (wave + (isA ? q : q - C::A_LD) * (C::NT / 64)) * 1024);
  };
  auto next = [&]() {
    dslot = dslot + 1 == NS ? 0 : dslot + 1;
    if (du >= units) return;
    if (++dkt < dend) {
      dA += stepA;
      lA -= stepA;
      dB += stepB;
      lB -= stepB;
    } else {
      du += stride;
      if (du < units) start();
    }
  };

  // the lane's 16-byte chunk of k (step ks) of row `row0 + fr` of an operand image
  auto frag = [&](const char* im, int row0, int ks, auto COL_, auto RB_) -> i32x4 {
    constexpr bool COL = decltype(COL_)::value;
    constexpr int rowb = decltype(RB_)::value;
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
        const char* at = im + r * rowb + (((col >> 3) ^ col_swz<T, rowb>(r)) << 4) + ((col >> 2) & 1) * 8;
        v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(las_ptr)at);
      }
      return __builtin_bit_cast(i32x4, s16x8{v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w});
    } else {
      i32x4 v;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int r = ks * 16 + fq * 4 + s, col = row0 + fr;
        v[s] = *reinterpret_cast<const int*>(im + r * rowb + (((col >> 2) ^ col_swz<T, rowb>(r)) << 4) + (col & 3) * 4);
      }
      return v;
    }
  };
  struct Frags { i32x4 a[TM], b[TN]; };
  auto read = [&](Frags& f, int slot, int ks) {
    const char* ia = smem + slot * C::STAGE;
    const char* ib = ia + C::A_BYTES;
#pragma unroll
    for (int j = 0; j < TN; ++j)
      f.b[j] = frag(ib, wn * C::WN + j * 16, ks, std::integral_constant<bool, BCOL>{}, std::integral_constant<int, BRB>{});
#pragma unroll
    for (int i = 0; i < TM; ++i)
      f.a[i] = frag(ia, wm * C::WM + i * 16, ks, std::integral_constant<bool, ACOL>{}, std::integral_constant<int, ARB>{});
  };
  acc_t acc[TM][TN];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
  };
  constexpr int PER = 2 * ((C::LD + TM - 1) / TM);              // pieces behind a row of MFMAs: the first half of the rows
  auto mul = [&](const Frags& f, auto ISSUE_) {
    constexpr bool ISSUE = decltype(ISSUE_)::value;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = step<T>(f.b[j], f.a[i], acc[i][j]);
      if constexpr (ISSUE) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = i * PER; q < (i + 1) * PER; ++q)
          if (q < C::LD) piece(q);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  start();
#pragma unroll
  for (int t = 0; t < NS; ++t) {
    aim();
#pragma unroll
    for (int q = 0; q < C::LD; ++q) piece(q);
    next();
  }
  Frags f0, f1;
  clear();
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * C::LD) : "memory");
  read(f0, 0, 0);
  int slot = 0;
  for (int u = blockIdx.x; u < units; u += stride) {
    const int t = u / p.parts, part = u - t * p.parts;
    const int n = min(per, p.nk - part * per);
    for (int k = 0; k < n; ++k) {
      // the compiler counts LDS reads to 15 only; told here that all of f0 (below: f1) has arrived, it does not wait for
      // reads that were issued behind them (col operands: up to 24 a step)
      __builtin_amdgcn_s_waitcnt(0xC07F);                       // lgkmcnt(0)
      read(f1, slot, 1);
      mul(f0, std::false_type{});
      // stages behind the next one may be in flight; an epilogue's stores only make the wait longer
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * C::LD) : "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("s_barrier" ::: "memory");
      slot = slot + 1 == NS ? 0 : slot + 1;
      aim();
      if (k + 1 < n) read(f0, slot, 0);                         // at a tile's end behind the epilogue: its registers
      __builtin_amdgcn_sched_barrier(0);
      mul(f1, std::true_type{});
      next();
    }
    int tm, tn;
    tile_of(t, p.ntm, p.ntn, tm, tn);
    epi.template write<C>(acc, tm * C::BM + wm * C::WM + fr, tn, wn, fq, part);
    clear();
    read(f0, slot, 0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // no DMA outlives the workgroup's LDS
}

using Big = Tile<256, 256, 2, 4, 2, 2>;        // one workgroup a CU
using Mid = Tile<128, 128, 2, 2, 2, 2>;        // two
using Small = Tile<64, 64, 2, 2, 3, 3>;        // three

// Which tile, and into how many parts the reduction is split where `most` allows it (parts are f32 slabs that another
// kernel joins).  A CU works off its tiles at `step` us a stage with its residents together, but no stage of one tile in
// less than `alone` us; `end` us a tile for its results.  Fitted over 100 to 50176 rows, 192 to 11264 results, 64 to 2048
// values of k (profiles/token_ops/choices.txt): the choice is the best of the three tiles or within 10 % of it at 359 of
// 388 sizes, within 20 % at 381 (bf16, 256-, 128-, 64-wide: 1500 x 1024 x 2 x 5632 55, 51, 66 us, chosen 48; 6000 x 2048 x
// 2 x 1024 52, 61, 90, chosen 60; 100 x 2048 x 2 x 340 45, 28, 14, chosen 14).  `end` is one number a type: it does not know
// the activation, kept projections, a residual or rows that are no whole lines, and it is there that the choice is wrong
// by more (8 bits, 50176 x 64 with 680 results in f16: 45 us, 128-wide 27).
// Where the last round of tiles would leave most CUs idle, the rows behind the whole rounds are taken by a second launch
// with smaller tiles (352 tiles of 256 for 256 CUs, dW of 8192 tokens: 421 -> 388 us).
struct Plan { int tile, parts; long rows; int rest; };          // the first `rows` rows with `tile`, the others with `rest`
struct Rate { double alone, step, end; };
template <typename T>
inline Plan plan_tiles(long m, long n, long nk, long most) {
  constexpr Rate r16[3] = {{1.33, 1.5, 4.0}, {0.54, 0.47, 1.3}, {0.235, 0.2, 0.5}};
  constexpr Rate r8[3] = {{1.1, 1.5, 8.0}, {0.5, 0.45, 2.2}, {0.21, 0.2, 0.7}};
  constexpr Rate r32[3] = {{7.3, 7.3, 4.0}, {2.1, 2.0, 1.3}, {0.72, 0.54, 0.5}};
  const Rate* rates = sizeof(T) == 4 ? r32 : (sizeof(T) == 1 ? r8 : r16);
  auto cost = [&](int c, long rows, long parts, long per) {
    const long side = 256 >> c;
    const double tiles = (double)((rows + side - 1) / side) * (double)((n + side - 1) / side);
    const double each = ceil(tiles * (double)parts / 256.0);
    return (double)per * fmax(rates[c].alone, each * rates[c].step) + each * rates[c].end;
  };
  Plan best{2, 1, m, 2};
  double least = 1e30;
  for (int c = 0; c < 3; ++c) {
    for (long parts = 1; parts <= most && (parts == 1 || nk >= 4 * parts); parts *= 2) {
      const long per = (nk + parts - 1) / parts, real = (nk + per - 1) / per;      // no empty part
      double t = cost(c, m, real, per);
      if (real > 1) t += 4.0 + (double)m * (double)n * 4.0 * (double)(real + 1) / 4e6;        // the slabs and their join
      if (t < least) {
        least = t;
        best = Plan{c, (int)real, m, c};
      }
    }
    const long side = 256 >> c, ntn = (n + side - 1) / side, rounds = (m + side - 1) / side * ntn / 256;
    const long rows = rounds * 256 / ntn * side;                // rows of the whole rounds
    if (rows <= 0 || rows >= m) continue;
    for (int d = c + 1; d < 3; ++d) {
      const double t = cost(c, rows, 1, nk) + 3.0 + cost(d, m - rows, 1, nk);
      if (t < least) {
        least = t;
        best = Plan{c, 1, rows, d};
      }
    }
  }
  return best;
}

// a plan as the host queries tell it: tile side, parts, rows, tile side of the rows behind them (0: none)
inline void tell(const Plan& plan, long m, long* out) {
  out[0] = 256 >> plan.tile;
  out[1] = plan.parts;
  out[2] = plan.rows;
  out[3] = plan.rows < m ? 256 >> plan.rest : 0;
}
inline void tell_few(long m, long* out) {         // the few-token kernel has no tiles
  out[0] = out[3] = 0;
  out[1] = 1;
  out[2] = m;
}

struct Slots { int cus, per; };
template <class K>
static Slots slots_of(K* fn, int threads) {
  int dev = 0, cus = 0, per = 0;
  (void)hipGetDevice(&dev);
  (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  (void)hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, reinterpret_cast<const void*>(fn), threads, 0);
  return Slots{cus > 0 ? cus : 1, per > 0 ? per : 1};
}

template <typename T, class C, bool AC, bool BC, class Epi>
static int launch_tiles(Args p, long m, long n, const Epi& epi, hipStream_t st, const char* name) {
  p.ntm = (int)((m + C::BM - 1) / C::BM);
  p.ntn = (int)((n + C::BN - 1) / C::BN);
  const long units = (long)p.ntm * p.ntn * p.parts;
  if (units > 0x7fffffffL) { set_error("%s: too many tiles", name); return SVK_EUNSUPPORTED; }
  static const Slots slots = slots_of(&tile_mm<T, C, AC, BC, Epi>, C::NT);
  const long all = (long)slots.cus * slots.per, grid = units < all ? units : all;
  // a grid that does not fill the chip is spread over the CUs by asking for LDS that keeps the others off (left alone
  // the dispatcher puts two workgroups on one CU beside idle ones: 176 tiles took as long as 352)
  const long want = (grid + slots.cus - 1) / slots.cus, lds = (long)C::NS * C::STAGE;
  long extra = 0;
  if (want < slots.per) extra = ((160 * 1024 / (want + 1) + 512) / 512) * 512 - lds;
  hipLaunchKernelGGL((tile_mm<T, C, AC, BC, Epi>), dim3((unsigned)grid), dim3(C::NT), (unsigned)(extra > 0 ? extra : 0), st, p, epi);
  set_last_kernel(name);
  return check_launch(name);
}
template <typename T, bool AC, bool BC, class Epi>
static int launch_plan(const Plan& plan, Args p, long m, long n, Epi epi, hipStream_t st, const char* name) {
  auto go = [&](int tile, long rows) -> int {
    if (tile == 0) return launch_tiles<T, Big, AC, BC>(p, rows, n, epi, st, name);
    if (tile == 1) return launch_tiles<T, Mid, AC, BC>(p, rows, n, epi, st, name);
    return launch_tiles<T, Small, AC, BC>(p, rows, n, epi, st, name);
  };
  p.parts = plan.parts;
  const long last = epi.M;
  epi.M = (int)plan.rows;
  if (int rc = go(plan.tile, plan.rows)) return rc;
  if (plan.rows >= m) return SVK_OK;
  // the rest: the operand and the results from row plan.rows on
  const long skip = AC ? plan.rows * (long)sizeof(T) : plan.rows * p.lda;
  p.A += skip;
  p.abytes -= skip;
  epi.M = (int)(last - plan.rows);
  epi.skip(plan.rows);
  return go(plan.rest, m - plan.rows);
}
template <typename T> inline int stages(long k) { return (int)((k * (long)sizeof(T) + 127) / 128); }

// Few token rows against the weights: each weight value is read once, straight into registers, and the reduction is
// split over the workgroup's waves and joined in LDS.  MT blocks of 16 tokens, NB blocks of 16 weight rows a workgroup
// (the epilogue's map names them, `epi.per` results).  Rows of any alignment and length.  Bound by the weights' bytes, and below some MiB by one trip to memory.
constexpr int SK_WAVES = 8;
// up to which it runs (us of it | of the tiles, weights of several copies in turn from memory: 2048 -> 2 x 5632 in bf16 1 token
// 13.4 | 17.5, 32 17.6 | 18.1, 48 20.8 | 18.2, 64 21.8 | 18.9; 2048 -> 2 x 340 64 tokens 11.9 | 14.1; 512 -> 2 x 2048 in f32
// 8.8 | 14.9; 8 bits 4096 -> 8192 18.2 | 17.4, 2048 -> 2048 7.5 | 8.7: at 64 tokens ahead but for the widest weights)
constexpr int SKINNY_M = 64;

// 16 bytes of a row from byte kb on, zeros past its end; rows of any alignment (the hardware reads 16 bytes anywhere)
typedef i32x4 any_i32x4 __attribute__((aligned(1)));
template <typename T>
__device__ __forceinline__ i32x4 load_chunk(const char* row, long kb, long kbytes) {
  constexpr int ES = sizeof(T);
  if (kb + 16 <= kbytes) return *reinterpret_cast<const any_i32x4*>(row + kb);
  union { i32x4 v; T e[16 / ES]; } u;
  u.v = i32x4{0, 0, 0, 0};
  if (kb < kbytes)
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i)
      if (kb + i * ES < kbytes) u.e[i] = *reinterpret_cast<const T*>(row + kb + i * ES);
  return u.v;
}

// ENDS: rows that end inside a 16-byte chunk
template <typename T, int MT, int NB, bool ENDS, class Epi>
__global__ __launch_bounds__(64 * SK_WAVES) void skinny_mm(Args p, Epi epi) {
  typedef typename Acc<T>::t acc_t;
  constexpr int U = MT + NB <= 2 ? 8 : (MT + NB <= 5 ? 4 : 2);  // 64-byte steps in flight
  typedef std::conditional_t<std::is_same<T, int8_t>::value, int, float> sum_t;
  __shared__ sum_t red[SK_WAVES][MT][NB][16][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const long kbytes = (long)p.K * sizeof(T);
  const char* rb[NB];
  const char* ra[MT];
#pragma unroll
  for (int j = 0; j < NB; ++j) rb[j] = p.B + (long)epi.skinny_row(blockIdx.x, j * 16 + fr) * p.ldb;
#pragma unroll
  for (int i = 0; i < MT; ++i) ra[i] = p.A + (long)min(i * 16 + fr, p.M - 1) * p.lda;
  acc_t acc[MT][NB];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
  for (long kb = (long)wave * 64 * U; kb < kbytes; kb += (long)SK_WAVES * 64 * U) {
    i32x4 fb[U][NB], fa[U][MT];
    auto load = [&](auto E) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long k = kb + u * 64 + fq * 16;
        auto get = [&](const char* row) {
          if constexpr (decltype(E)::value) return load_chunk<T>(row, k, kbytes);
          else return k < kbytes ? *reinterpret_cast<const any_i32x4*>(row + k) : i32x4{0, 0, 0, 0};
        };
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[u][j] = get(rb[j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[u][i] = get(ra[i]);
      }
    };
    if (ENDS && kb + U * 64 > kbytes) load(std::true_type{});      // the turn in which the rows end
    else load(std::false_type{});
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = step<T>(fb[u][j], fa[u][i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][i][j][fr][fq * 4 + e] = acc[i][j][e];
  __syncthreads();
  auto sum = [&](int m, int r) {                                // the waves' parts, in order
    sum_t v = 0;
#pragma unroll
    for (int w = 0; w < SK_WAVES; ++w) v += red[w][m >> 4][r >> 4][m & 15][r & 15];
    return v;
  };
  for (int t = tid; t < p.M * epi.per; t += 64 * SK_WAVES) {
    const int m = t / epi.per, n = t - m * epi.per;
    epi.skinny_write(blockIdx.x, m, n, sum(m, n), Epi::PAIR ? sum(m, n + epi.per) : sum_t(0));
  }
}

// `results` of a row, epi.per a workgroup and WPR weight rows each: as many as give the 256 CUs one workgroup each (the
// tokens are read once a workgroup, the weights evenly), 16 to 64 weight rows
// (2 x 5632 rows of 2048 in bf16, 16 tokens: 32 rows a workgroup 15.5, 16 rows 14, 44 rows 11.3 us: 46 MB of weights at
// 4.1 TB/s)
template <typename T, int MT, int WPR, class Epi>
static int launch_skinny(const Args& p, long results, Epi epi, hipStream_t st, const char* name) {
  long per = (results + 255) / 256;
  per = per < 16 / WPR ? 16 / WPR : (per > 64 / WPR ? 64 / WPR : per);
  epi.per = (int)per;
  const dim3 grid((unsigned)((results + per - 1) / per)), block(64 * SK_WAVES);
  auto go = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if (p.K * sizeof(T) % 16) hipLaunchKernelGGL((skinny_mm<T, MT, NB, true, Epi>), grid, block, 0, st, p, epi);
    else hipLaunchKernelGGL((skinny_mm<T, MT, NB, false, Epi>), grid, block, 0, st, p, epi);
    set_last_kernel(name);
    return check_launch(name);
  };
  switch ((per * WPR + 15) / 16) {
    case 1: return go(std::integral_constant<int, 1>{});
    case 2: return go(std::integral_constant<int, 2>{});
    case 3: return go(std::integral_constant<int, 3>{});
    default: return go(std::integral_constant<int, 4>{});
  }
}
template <typename T, int WPR, class Epi>
static int few_tokens(const Args& p, long results, const Epi& epi, hipStream_t st, const char* name) {
  if (p.M <= 16) return launch_skinny<T, 1, WPR>(p, results, epi, st, name);
  if (p.M <= 32) return launch_skinny<T, 2, WPR>(p, results, epi, st, name);
  return launch_skinny<T, 4, WPR>(p, results, epi, st, name);
}

// copy of rows into rows of whole 16-byte chunks, the last filled up with zeros: what the tiled kernels read where a row
// operand's length or address is no whole number of chunks.  A chunk a thread, rows read at any alignment (value by value
// it took longer than the product: 315 x 3930 x 4240 in 8 bits 72 us in all, by chunks 63; 38 with the tokens quantised 8 values a lane too)
template <typename T>
__global__ __launch_bounds__(256) void pad_rows(const char* __restrict__ X, long ldx, char* __restrict__ Y, long rows, long kbytes) {
  const long chunks = (kbytes + 15) / 16, total = rows * chunks;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long r = total <= 0x7fffffffL ? (uint32_t)i / (uint32_t)chunks : i / chunks, c = i - r * chunks;
    *reinterpret_cast<i32x4*>(Y + i * 16) = load_chunk<T>(X + r * ldx, c * 16, kbytes);
  }
}
// ldx: bytes between the rows of X
template <typename T>
static int pad(const void* X, long ldx, void* Y, long rows, long kbytes, hipStream_t st) {
  const long blocks = (rows * ((kbytes + 15) / 16) + 255) / 256;
  hipLaunchKernelGGL((pad_rows<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, (const char*)X, ldx, (char*)Y, rows, kbytes);
  return check_launch("pad_rows");
}

// rows that may be stored past the L2: whole 64-byte lines.  Lines that two tiles share cost there what they would not in the
// L2 (8-bit products of 50176 x 320 with 680 results in f16, rows of 21.25 lines: 77 us, 43 through the L2; 16384 x 1024 with
// 1000: 47 and 31; 50176 x 320 x 2 x 856 in bf16: 93 and 87); whole lines gain by it (16384 x 4096 with 8192: 446 us, 473
// through the L2; with 8224: 491 and 539).  Long reductions are within 3 % either way
inline bool whole_lines(const void* p, long ld_bytes, long row_bytes) {
  return (((uintptr_t)p | (uintptr_t)ld_bytes | (uintptr_t)row_bytes) & 63) == 0;
}
inline long up16(long bytes) { return (bytes + 15) & ~15L; }
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace mm
}  // namespace svk
