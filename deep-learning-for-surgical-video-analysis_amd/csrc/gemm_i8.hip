// Matrix product in 8-bit integers with a scale for each token and each output channel (svk_gemm_i8), and the
// quantisation of token rows that feeds it (svk_quant_rows):
//
//   s[m] = max_k |x[m, k]| / 127,  q[m, k] = round(x[m, k] / s[m])            (ties to even; a row of zeros: s = 0, q = 0)
//   C[m, n] = act((sum_k qa[m, k] qw[n, k]) sa[m] sw[n] + bias[n]) + R[m, n]
//
// The integer sums are exact (int32: K <= 131072 for codes of -128 .. 127); everything behind them is f32, rounded once.
// A row with an infinity or a NaN gets the scale NaN and codes of zero: its outputs are NaN, not quietly wrong.
// tile_mm.h with int8 operands: mfma 16x16x64 at twice the 16-bit rate and half the bytes.
#include "tile_mm.h"
#include <algorithm>
#include <type_traits>

namespace svk {
namespace i8 {
using namespace mm;

// one wave a row; NCH chunks of 8 values a lane kept in registers (0: read twice)
template <typename T, int NCH, bool VEC>
__global__ __launch_bounds__(256) void quant_rows(const T* __restrict__ X, long ldx, int8_t* __restrict__ Q, long ldq,
                                                  float* __restrict__ S, long M, int K) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= M) return;
  const T* x = X + row * ldx;
  int8_t* q = Q + row * ldq;
  float top = 0.f;
  bool fine = true;
  auto see = [&](float v) {
    top = fmaxf(top, fabsf(v));
    fine = fine && fabsf(v) < INFINITY;
  };
  auto code = [&](float v, float s) { return (int)rintf(fminf(fmaxf(v / s, -127.f), 127.f)); };
  if constexpr (VEC) {
    const int nch = K >> 3;
    float v[NCH > 0 ? NCH : 1][8];
    auto load = [&](int ch, float* o) {
      T t[8];
#pragma unroll
      for (int p = 0; p < (int)sizeof(T) / 2; ++p)
        reinterpret_cast<uint4*>(t)[p] = reinterpret_cast<const uint4*>(x + (long)ch * 8)[p];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = to_f(t[e]);
    };
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (lane + 64 * i < nch) {
          load(lane + 64 * i, v[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) see(v[i][e]);
        }
    } else {
      for (int ch = lane; ch < nch; ch += 64) {
        load(ch, v[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) see(v[0][e]);
      }
    }
    top = wave_max(top);
    fine = __all(fine);
    const float s = fine ? top / 127.f : NAN;
    if (lane == 0) S[row] = s;
    auto store = [&](int ch, const float* o) {
      uint32_t w[2] = {0u, 0u};
      if (s > 0.f)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= ((uint32_t)code(o[e], s) & 255u) << (8 * (e & 3));
      *reinterpret_cast<uint2*>(q + (long)ch * 8) = uint2{w[0], w[1]};
    };
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (lane + 64 * i < nch) store(lane + 64 * i, v[i]);
    } else {
      for (int ch = lane; ch < nch; ch += 64) {
        load(ch, v[0]);
        store(ch, v[0]);
      }
    }
  } else {
    for (int k = lane; k < K; k += 64) see(to_f(x[k]));
    top = wave_max(top);
    fine = __all(fine);
    const float s = fine ? top / 127.f : NAN;
    if (lane == 0) S[row] = s;
    for (int k = lane; k < K; k += 64) q[k] = s > 0.f ? (int8_t)code(to_f(x[k]), s) : 0;
  }
}

// ACT: none, GELU, or -1: `act`, chosen while running
template <typename T, int ACT>
struct ScaleEpi {
  const float *sa, *sw, *bias;
  const T* R; long ldr;
  T* y; long ldy;
  int M, N, act;

  __device__ __forceinline__ float value(int acc, float a, float w, float b) const {
    const float v = (float)acc * a * w + b;
    if constexpr (sizeof(T) == 4) return apply_act(v, ACT < 0 ? act : ACT);
    else return apply_act_fast(v, ACT < 0 ? act : ACT);
  }
  template <class C> __device__ __forceinline__ long first(int tn) const { return (long)tn * C::BN; }
  template <class C> __device__ __forceinline__ uint32_t offset(int r, uint32_t ldb) const { return (uint32_t)pair_col(r) * ldb; }
  __device__ __forceinline__ int skinny_row(int bid, int j, int fr) const { return min(bid * 32 + j * 16 + fr, N - 1); }
  __device__ __forceinline__ void skinny_write(int bid, int m, int n, int v0, int v1) const {
    one(m, bid * 32 + n, v0);
    one(m, bid * 32 + 16 + n, v1);
  }
  __device__ __forceinline__ void one(int m, int n, int acc) const {
    if (n >= N) return;
    float v = value(acc, sa[m], sw[n], bias ? bias[n] : 0.f);
    if (R) v += to_f(R[(long)m * ldr + n]);
    y[(long)m * ldy + n] = from_f<T>(v);
  }
  template <class C, typename A>
  __device__ __forceinline__ void write(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq, int) const {
    constexpr int NW = 8 * sizeof(T) / 4;
    typedef uint32_t vec __attribute__((ext_vector_type(NW)));
    typedef vec anywhere __attribute__((aligned(2)));
    float a[C::TM];
#pragma unroll
    for (int i = 0; i < C::TM; ++i) a[i] = sa[min(m0 + i * 16, M - 1)];
#pragma unroll
    for (int j = 0; j < C::TN; j += 2) {
      const int n = tn * C::BN + wn * C::WN + j * 16 + fq * 8, left = N - n;
      if (left <= 0) continue;
      float w[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = min(n + e, N - 1);
        w[e] = sw[c];
        b[e] = bias ? bias[c] : 0.f;
      }
      // the residual of the next rows is read before these rows are stored: read behind a store it would wait for that
      // store (R may be Y itself: every value is read before it is written, by the same lane)
      constexpr int RB = C::TM >= 4 ? 8 / (int)sizeof(T) : C::TM;  // rows in hand: 16 registers
      vec r[2][RB];
      auto fetch = [&](int i0, vec* o) {
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const T* at = R + (long)min(m0 + (i0 + i) * 16, M - 1) * ldr + n;
          if (left >= 8) o[i] = *reinterpret_cast<const anywhere*>(at);
          else {
            T t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = at[min(e, left - 1)];
            __builtin_memcpy(&o[i], t, sizeof(vec));
          }
        }
      };
      if (R) fetch(0, r[0]);
#pragma unroll
      for (int i0 = 0; i0 < C::TM; i0 += RB) {
        if (R && i0 + RB < C::TM) fetch(i0 + RB, r[(i0 / RB + 1) & 1]);
#pragma unroll
        for (int i = i0; i < i0 + RB; ++i) {
          const int m = m0 + i * 16;
          float v[8];
          T t[8];
          if (R) __builtin_memcpy(t, &r[(i0 / RB) & 1][i - i0], sizeof(vec));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = value(acc[i][j + e / 4][e % 4], a[i], w[e], b[e]);
            if (R) v[e] += to_f(t[e]);
          }
          if (m < M) put<T, 8, C::NONTEMPORAL>(y + (long)m * ldy + n, v, left);
          __builtin_amdgcn_sched_barrier(0);                    // one row at a time: fewer registers
        }
      }
    }
  }
};

using Big = Tile<256, 256, 2, 4, 2, 2>;
using Mid = Tile<128, 128, 2, 2, 2, 2>;
using Small = Tile<64, 64, 2, 2, 4, 2>;
template <typename T, int MT>
static int go_skinny(const Args& p, bool vec, const ScaleEpi<T, -1>& epi, hipStream_t st) {
  const int blocks = (epi.N + 31) / 32;
  if (vec) hipLaunchKernelGGL((skinny_mm<int8_t, MT, true, ScaleEpi<T, -1>>), dim3(blocks), dim3(64 * SK_WAVES), 0, st, p, epi);
  else hipLaunchKernelGGL((skinny_mm<int8_t, MT, false, ScaleEpi<T, -1>>), dim3(blocks), dim3(64 * SK_WAVES), 0, st, p, epi);
  set_last_kernel("gemm_i8_skinny");
  return check_launch("gemm_i8_skinny");
}

static bool rows_ok(const void* p, long ld, long K) { return al16(p) && ld % 16 == 0 && K % 16 == 0; }
static bool bad_dims(long M, long N, long K) {
  return M < 0 || N <= 0 || K <= 0 || M > 0x7fffff00L || N > 0x7fffff00L || K > 131072;
}

}  // namespace i8
}  // namespace svk

using namespace svk;
using namespace svk::i8;

extern "C" int svk_quant_rows(int dtype, const void* X, long ldx, void* Q, long ldq, float* S, long M, long K, void* stream) {
  if (M < 0 || K <= 0 || M > 0x7fffff00L || K > 0x7fffff00L || !X || !Q || !S || ldx < K || ldq < K) { set_error("svk_quant_rows: bad args"); return SVK_EINVAL; }
  if (M == 0) return SVK_OK;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((M + 3) / 4)), block(256);
  SVK_DISPATCH_DTYPE(dtype, T, {
    const T* x = (const T*)X;
    int8_t* q = (int8_t*)Q;
    const bool vec = K % 8 == 0 && al16(X) && ldx * (long)sizeof(T) % 16 == 0 && ((uintptr_t)Q & 7) == 0 && ldq % 8 == 0;
    if (!vec) hipLaunchKernelGGL((quant_rows<T, 0, false>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    else if (K <= 512) hipLaunchKernelGGL((quant_rows<T, 1, true>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    else if (K <= 1024) hipLaunchKernelGGL((quant_rows<T, 2, true>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    else if (K <= 2048) hipLaunchKernelGGL((quant_rows<T, 4, true>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    else if (K <= 4096) hipLaunchKernelGGL((quant_rows<T, 8, true>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    else hipLaunchKernelGGL((quant_rows<T, 0, true>), grid, block, 0, st, x, ldx, q, ldq, S, M, (int)K);
    return check_launch("quant_rows");
  });
}

extern "C" long svk_gemm_i8_workspace(const void* A, long lda, const void* W, long ldw, long M, long N, long K) {
  if (bad_dims(M, N, K) || M <= SKINNY_M) return 0;
  const long ldk = up16(K);
  return (rows_ok(A, lda, K) ? 0 : M * ldk) + (rows_ok(W, ldw, K) ? 0 : N * ldk);
}

extern "C" int svk_gemm_i8(int dtype, const void* A, long lda, const float* sa, const void* W, long ldw, const float* sw,
                           const float* bias, const void* R, long ldr, void* Y, long ldy, long M, long N, long K, int act,
                           void* ws, long ws_bytes, void* stream) {
  if (!A || !sa || !W || !sw || !Y || bad_dims(M, N, K) || lda < K || ldw < K || ldy < N || (R && ldr < N) ||
      act < SVK_ACT_NONE || act > SVK_ACT_TANH) {
    set_error("svk_gemm_i8: bad args (K up to 131072)");
    return SVK_EINVAL;
  }
  const long ldk = up16(K);
  if (N * std::max(ldw, ldk) >= (1L << 32) || 256 * std::max(lda, ldk) >= (1L << 32)) {
    set_error("svk_gemm_i8: weights or 256 rows of a of 4 GiB or more");
    return SVK_EUNSUPPORTED;
  }
  if (ws_bytes < svk_gemm_i8_workspace(A, lda, W, ldw, M, N, K)) { set_error("svk_gemm_i8: workspace too small"); return SVK_EINVAL; }
  if (M == 0) return SVK_OK;
  hipStream_t st = (hipStream_t)stream;
  SVK_DISPATCH_DTYPE(dtype, T, {
    Args p{(const char*)A, (const char*)W, lda, ldw, 0, 0, (int)M, (int)K, 0, 0, 0, 1};
    if (M <= SKINNY_M) {
      const bool vec = rows_ok(A, lda, K) && rows_ok(W, ldw, K);
      ScaleEpi<T, -1> epi{sa, sw, bias, (const T*)R, ldr, (T*)Y, ldy, (int)M, (int)N, act};
      return M <= 16 ? go_skinny<T, 1>(p, vec, epi, st) : go_skinny<T, 2>(p, vec, epi, st);
    }
    char* at = (char*)ws;
    auto pad = [&](const void* X, long ld, long rows) {
      const unsigned blocks = (unsigned)std::min<long>((rows * ldk + 255) / 256, 8192);
      hipLaunchKernelGGL((pad_rows<int8_t>), dim3(blocks), dim3(256), 0, st, (const int8_t*)X, ld, (int8_t*)at, ldk, rows, (int)K);
      return check_launch("pad_rows");
    };
    if (!rows_ok(A, lda, K)) {
      if (int rc = pad(A, lda, M)) return rc;
      p.A = at;
      p.lda = ldk;
      at += M * ldk;
      p.K = (int)ldk;
    }
    if (!rows_ok(W, ldw, K)) {
      if (int rc = pad(W, ldw, N)) return rc;
      p.B = at;
      p.ldb = ldk;
      p.K = (int)ldk;
    }
    p.nk = (p.K + 127) / 128;
    p.abytes = (M - 1) * p.lda + p.K;
    p.bbytes = (N - 1) * p.ldb + p.K;
    auto tiles = [&](long b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
    auto run = [&](auto act_c) {
      ScaleEpi<T, decltype(act_c)::value> epi{sa, sw, bias, (const T*)R, ldr, (T*)Y, ldy, (int)M, (int)N, act};
      if (tiles(256) >= 200) return launch_tiles<int8_t, Big, false, false>(p, M, N, epi, st, "gemm_i8");
      if (tiles(128) >= 200) return launch_tiles<int8_t, Mid, false, false>(p, M, N, epi, st, "gemm_i8");
      return launch_tiles<int8_t, Small, false, false>(p, M, N, epi, st, "gemm_i8");
    };
    if (act == SVK_ACT_NONE) return run(std::integral_constant<int, SVK_ACT_NONE>{});
    if (act == SVK_ACT_GELU) return run(std::integral_constant<int, SVK_ACT_GELU>{});
    return run(std::integral_constant<int, -1>{});
  });
}
