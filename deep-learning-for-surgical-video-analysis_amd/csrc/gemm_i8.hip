// Matrix product in 8-bit integers with a scale for each token and each output channel (svk_gemm_i8), and the
// quantisation of token rows that feeds it (svk_quant_rows):
//
//   s[m] = max_k |x[m, k]| (1 / 127),  q[m, k] = round(x[m, k] / s[m])        (ties to even; a row of zeros: s = 0, q = 0)
//   C[m, n] = act((sum_k qa[m, k] qw[n, k]) sa[m] sw[n] + bias[n]) + R[m, n]
//
// The integer sums are exact (int32: K <= 131071, 2^31 / 128^2 less one); everything behind them is f32, rounded once.
// A row with an infinity or a NaN gets the scale NaN and codes of zero: its outputs are NaN, not quietly wrong.
// tile_mm.h with int8 operands: mfma 16x16x64 at twice the 16-bit rate and half the bytes.
#include "tile_mm.h"
#include <algorithm>
#include <type_traits>

namespace svk {
namespace i8 {
using namespace mm;

// largest of the 64 lanes' values, in every lane
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  auto over = [&](auto C) { v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(C)::value, 0xF, 0xF, true)); };
  over(std::integral_constant<int, 0xB1>{});                    // lanes 1 0 3 2 of each four
  over(std::integral_constant<int, 0x4E>{});                    // lanes 2 3 0 1
  over(std::integral_constant<int, 0x141>{});                   // each eight mirrored
  over(std::integral_constant<int, 0x140>{});                   // each sixteen mirrored
  return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
             max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// RW rows a wave, read before the first is reduced; NCH chunks of 8 values a lane and row kept in registers (0: read
// twice).
// The largest magnitude is found on the bits without the sign, whose order as integers is that of the magnitudes (an
// infinity or a NaN comes out largest).  A code is the correctly rounded quotient x / s, rounded to an integer: with r the
// correctly rounded 1 / s and y = x r, the residual x - y s is exact in one fma, and y + residual * r is the correctly
// rounded quotient (Markstein); 1.5 * 2^23 added to it leaves the nearest integer, ties to even, in the last byte.  Four
// instructions a value; the division, a rounding and two clamps each, and one row a wave, took 12544 rows of 512 in f16
// 11.0 us, this 9.6; 16384 rows of 4096 in bf16 46 and 33 us (201 MB at 6.1 TB/s).  (x * (127 / max) would take one, but decides the
// many exact ties of 16-bit values another way than x / s.)
template <typename T, int NCH, int RW>
__global__ __launch_bounds__(256) void quant_rows(const T* __restrict__ X, long ldx, int8_t* __restrict__ Q, long ldq,
                                                  float* __restrict__ S, long M, int K) {
  const int lane = threadIdx.x & 63;
  const long row0 = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RW;
  if (row0 >= M) return;
  constexpr int W = 2 * sizeof(T);                              // words of 8 values
  float s, inv;
  // the scale from the largest magnitude (times the f32 1 / 127: what torch's x.abs().amax(-1) / 127 is on the GPU, so the
  // codes are those of that expression; a true division differs by a step in one row of 20, and with it decided 1 of 14000
  // codes of bf16 tokens the other way), and its reciprocal; 0 where the scale is so small that the residual would
  // underflow (then codes come from the division), or is no finite number, or 0 (codes of 0)
  auto scale = [&](long row, float top) {
    s = top < INFINITY ? top * (1.f / 127.f) : NAN;
    inv = s >= 1e-30f ? 1.f / s : 0.f;
    if (lane == 0) S[row] = s;
  };
  auto code = [&](float v) -> uint32_t {
    if (inv > 0.f) {
      const float y = v * inv;
      return __float_as_uint(fmaf(fmaf(-y, s, v), inv, y) + 12582912.f) & 255u;
    }
    if (s > 0.f) return (uint32_t)(int)rintf(fminf(fmaxf(v / s, -127.f), 127.f)) & 255u;
    return 0u;
  };
  const int nch = (K + 7) >> 3;
  uint32_t v[RW][NCH > 0 ? NCH : 1][W], top[W];
  auto load = [&](long row, int ch, uint32_t* o) {             // rows of any alignment; zeros past their end
    const T* at = X + row * ldx + (long)ch * 8;
    if (ch * 8 + 8 <= K) {
#pragma unroll
      for (int p = 0; p < W / 4; ++p) {
        const i32x4 w = reinterpret_cast<const any_i32x4*>(at)[p];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[p * 4 + e] = (uint32_t)w[e];
      }
    } else {
      union { T t[8]; uint32_t w[W]; } u;
#pragma unroll
      for (int w = 0; w < W; ++w) u.w[w] = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (ch * 8 + e < K) u.t[e] = at[e];
#pragma unroll
      for (int w = 0; w < W; ++w) o[w] = u.w[w];
    }
  };
  auto see = [&](const uint32_t* o) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if constexpr (sizeof(T) == 2)
        top[w] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top[w]), __builtin_bit_cast(u16x2, o[w] & 0x7FFF7FFFu)));
      else top[w] = max(top[w], o[w] & 0x7FFFFFFFu);
    }
  };
  auto store = [&](long row, int ch, const uint32_t* o) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f;
        if constexpr (sizeof(T) == 4) f = __uint_as_float(o[h * 4 + e]);
        else {
          const f32x2 two = unpack2<T>(o[h * 2 + e / 2]);
          f = e & 1 ? two.y : two.x;
        }
        c[e] = code(f);
      }
      w[h] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    }
    int8_t* at = Q + row * ldq + (long)ch * 8;
    typedef uint32_t two __attribute__((ext_vector_type(2)));
    typedef two any_two __attribute__((aligned(1)));
    if (ch * 8 + 8 <= K) *reinterpret_cast<any_two*>(at) = two{w[0], w[1]};
    else
      for (int e = 0; ch * 8 + e < K; ++e) at[e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
  };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (lane + 64 * i < nch) load(min(row0 + r, M - 1), lane + 64 * i, v[r][i]);
  }
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const long row = row0 + r;
    if (row >= M) return;
#pragma unroll
    for (int w = 0; w < W; ++w) top[w] = 0u;
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (lane + 64 * i < nch) see(v[r][i]);
    } else {
      for (int ch = lane; ch < nch; ch += 64) {
        load(row, ch, v[0][0]);
        see(v[0][0]);
      }
    }
    uint32_t m = 0u;
#pragma unroll
    for (int w = 0; w < W; ++w) m = max(m, sizeof(T) == 2 ? max(top[w] & 0xFFFFu, top[w] >> 16) : top[w]);
    m = wave_umax(m);
    if constexpr (sizeof(T) == 4) scale(row, __uint_as_float(m));
    else scale(row, unpack2<T>(m).x);
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (lane + 64 * i < nch) store(row, lane + 64 * i, v[r][i]);
    } else {
      for (int ch = lane; ch < nch; ch += 64) {
        load(row, ch, v[0][0]);
        store(row, ch, v[0][0]);
      }
    }
  }
}

// ACT: none, GELU, ReLU, or -1: `act`, chosen while running
template <typename T, int ACT>
struct ScaleEpi {
  const float *sa, *sw, *bias;
  const T* R; long ldr;
  T* y; long ldy;
  int M, N, act, per;
  bool past;              // rows of y are whole lines
  void skip(long rows) {
    sa += rows;
    if (R) R += rows * ldr;
    y += rows * ldy;
  }

  __device__ __forceinline__ float value(int acc, float a, float w, float b) const {
    const float v = (float)acc * a * w + b;
    const int f = ACT < 0 ? act : ACT;
    if (f == SVK_ACT_RELU) return v < 0.f ? 0.f : v;            // NaN stays NaN
    if constexpr (sizeof(T) == 4) return apply_act(v, f);
    else return f == SVK_ACT_GELU ? gelu16(v) : apply_act_fast(v, f);
  }
  template <class C> __device__ __forceinline__ long first(int tn) const { return (long)tn * C::BN; }
  template <class C> __device__ __forceinline__ uint32_t offset(int r, uint32_t ldb) const { return (uint32_t)pair_col(r) * ldb; }
  static constexpr bool PAIR = false;
  __device__ __forceinline__ int skinny_row(int bid, int r) const { return min(bid * per + min(r, per - 1), N - 1); }
  __device__ __forceinline__ void skinny_write(int bid, int m, int i, int acc, int) const {
    const int n = bid * per + i;
    if (n >= N) return;
    float v = value(acc, sa[m], sw[n], bias ? bias[n] : 0.f);
    if (R) v += to_f(R[(long)m * ldr + n]);
    y[(long)m * ldy + n] = from_f<T>(v);
  }
  template <class C, typename A>
  __device__ __forceinline__ void write(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq, int) const {
    if (C::NONTEMPORAL && past) rows_of<C, true>(acc, m0, tn, wn, fq);
    else rows_of<C, false>(acc, m0, tn, wn, fq);
  }
  template <class C, bool NTS, typename A>
  __device__ __forceinline__ void rows_of(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq) const {
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
          if (m < M) put<T, 8, NTS>(y + (long)m * ldy + n, v, left);
          __builtin_amdgcn_sched_barrier(0);                    // one row at a time: fewer registers
        }
      }
    }
  }
};

// rows that the tiled kernel can read as they are: aligned, and of whole chunks.  Tokens may end inside a chunk where the
// weights (or their copy) hold zeros there: whatever lies behind the codes is a finite integer and is multiplied by zero.
// (An aligned chunk that holds a code lies in that code's page.)
static bool rows_ok(const void* p, long ld, long K) { return al16(p) && ld % 16 == 0 && K % 16 == 0; }
static bool tokens_ok(const void* p, long ld, long K) { return al16(p) && ld % 16 == 0 && ld >= up16(K); }
static bool bad_dims(long M, long N, long K) {
  return M < 0 || N <= 0 || K <= 0 || M > 0x7fffff00L || N > 0x7fffff00L || K > 131071;
}

inline Plan plan_of(long M, long N, long K) { return plan_tiles<int8_t>(M, N, stages<int8_t>(K), 1); }

}  // namespace i8
}  // namespace svk

using namespace svk;
using namespace svk::i8;

extern "C" int svk_quant_rows(int dtype, const void* X, long ldx, void* Q, long ldq, float* S, long M, long K, void* stream) {
  if (M < 0 || K <= 0 || M > 0x7fffff00L || K > 0x7fffff00L || !X || !Q || !S || ldx < K || ldq < K) { set_error("svk_quant_rows: bad args"); return SVK_EINVAL; }
  if (M == 0) return SVK_OK;
  hipStream_t st = (hipStream_t)stream;
  SVK_DISPATCH_DTYPE(dtype, T, {
    const T* x = (const T*)X;
    int8_t* q = (int8_t*)Q;
    auto go = [&](auto nch, auto rw) {
      constexpr int RW = decltype(rw)::value;
      for (long m = 0; m < M; m += 1L << 25) {                  // a launch has under 2^32 threads, 64 a row here
        const long rows = std::min(M - m, 1L << 25);
        hipLaunchKernelGGL((quant_rows<T, decltype(nch)::value, RW>), dim3((unsigned)((rows + 4 * RW - 1) / (4 * RW))),
                           dim3(256), 0, st, x + m * ldx, ldx, q + m * ldq, ldq, S + m, rows, (int)K);
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    // short rows of 16 bits in numbers: four a wave, whose loads are under way together (one row a wave | four, us, tokens
    // past every cache: 4096 x 512 in bf16 4.6 | 4.9, 6144 5.6 | 5.4, 12544 10.4 | 8.6, 12544 x 128 7.6 | 5.7; f32 12544 x
    // 512 11.3 | 14.2; two rows of 1024 in bf16 a wave 11.5 | 12.9)
    if (K <= 512) {
      if constexpr (sizeof(T) == 2) M >= 6144 ? go(I1{}, I4{}) : go(I1{}, I1{});
      else go(I1{}, I1{});
    } else if (K <= 1024) go(I2{}, I1{});
    else if (K <= 2048) go(I4{}, I1{});
    else if (K <= 4096) go(std::integral_constant<int, 8>{}, I1{});
    else go(I0{}, I1{});
    return check_launch("quant_rows");
  });
}

extern "C" long svk_gemm_i8_workspace(const void* A, long lda, const void* W, long ldw, long M, long N, long K) {
  if (bad_dims(M, N, K) || M <= SKINNY_M) return 0;
  const long ldk = up16(K);
  return (tokens_ok(A, lda, K) ? 0 : M * ldk) + (rows_ok(W, ldw, K) ? 0 : N * ldk);
}

extern "C" int svk_gemm_i8_plan(long M, long N, long K, long* plan) {
  if (bad_dims(M, N, K) || M == 0 || !plan) { set_error("svk_gemm_i8_plan: bad args"); return SVK_EINVAL; }
  if (M <= SKINNY_M) tell_few(M, plan);
  else tell(plan_of(M, N, K), M, plan);
  return SVK_OK;
}

extern "C" int svk_gemm_i8(int dtype, const void* A, long lda, const float* sa, const void* W, long ldw, const float* sw,
                           const float* bias, const void* R, long ldr, void* Y, long ldy, long M, long N, long K, int act,
                           void* ws, long ws_bytes, void* stream) {
  if (!A || !sa || !W || !sw || !Y || bad_dims(M, N, K) || lda < K || ldw < K || ldy < N || (R && ldr < N) ||
      act < SVK_ACT_NONE || act > SVK_ACT_TANH) {
    set_error("svk_gemm_i8: bad args (K up to 131071)");
    return SVK_EINVAL;
  }
  const long ldk = up16(K);
  if (N * std::max(ldw, ldk) >= (1L << 32) || 256 * std::max(lda, ldk) >= (1L << 32)) {
    set_error("svk_gemm_i8: weights or 256 rows of a of 4 GiB or more");
    return SVK_EUNSUPPORTED;
  }
  const long need = svk_gemm_i8_workspace(A, lda, W, ldw, M, N, K);
  if (need && (!ws || !al16(ws) || ws_bytes < need)) { set_error("svk_gemm_i8: workspace too small or misaligned"); return SVK_EINVAL; }
  if (M == 0) return SVK_OK;
  hipStream_t st = (hipStream_t)stream;
  SVK_DISPATCH_DTYPE(dtype, T, {
    const bool past = whole_lines(Y, ldy * (long)sizeof(T), N * (long)sizeof(T));
    Args p{(const char*)A, (const char*)W, lda, ldw, 0, 0, (int)M, (int)K, 0, 0, 0, 1};
    if (M <= SKINNY_M) {
      ScaleEpi<T, -1> epi{sa, sw, bias, (const T*)R, ldr, (T*)Y, ldy, (int)M, (int)N, act, 0, past};
      return few_tokens<int8_t, 1>(p, N, epi, st, "gemm_i8_few");
    }
    char* at = (char*)ws;
    if (!tokens_ok(A, lda, K)) {
      if (int rc = pad<int8_t>(A, lda, at, M, K, st)) return rc;
      p.A = at;
      p.lda = ldk;
      at += M * ldk;
    }
    p.K = (int)ldk;                                 // whole chunks
    if (!rows_ok(W, ldw, K)) {
      if (int rc = pad<int8_t>(W, ldw, at, N, K, st)) return rc;
      p.B = at;
      p.ldb = ldk;
    }
    p.nk = stages<int8_t>(p.K);
    p.abytes = (M - 1) * p.lda + p.K;
    p.bbytes = (N - 1) * p.ldb + p.K;
    const Plan plan = plan_of(M, N, K);
    auto run = [&](auto act_c) {
      ScaleEpi<T, decltype(act_c)::value> epi{sa, sw, bias, (const T*)R, ldr, (T*)Y, ldy, (int)M, (int)N, act, 0, past};
      return launch_plan<int8_t, false, false>(plan, p, M, N, epi, st, "gemm_i8");
    };
    if (act == SVK_ACT_NONE) return run(std::integral_constant<int, SVK_ACT_NONE>{});
    if (act == SVK_ACT_GELU) return run(std::integral_constant<int, SVK_ACT_GELU>{});
    if (act == SVK_ACT_RELU) return run(std::integral_constant<int, SVK_ACT_RELU>{});
    return run(std::integral_constant<int, -1>{});
  });
}
