// Gated feed-forward block (svk_gated_ffn): both projections, the activation and the product in one kernel
//
//   h[m, c] = act(sum_k x[m, k] Wg[c, k] + bg[c]) * (sum_k x[m, k] Wu[c, k] + bu[c])
//
// and its backward pass.  The two weight matrices are one stacked [2H, K] (gate rows, then up rows).  The B rows of a
// tile are taken alternately from the two halves, so that a wave's accumulators hold the gate and the up value of the
// same (m, c) in the same lane: the product is formed in f32 registers, and the [M, 2H] projections never exist in
// memory unless the caller keeps them for the backward pass (rounded to the storage type, once).
//
// Backward, from the kept projections g, u and dh:
//   dg = dh u act'(g),  du = dh act(g)   (gated_dpre: f32, rounded once to the storage type: operands of the products;
//                                         the bias gradient sums the unrounded values in f32)
//   dx = [dg | du] [Wg; Wu],  dW = [dg | du]^T x   (tile_mm.h, col operands: no transposed copies)
// Every sum has a fixed order: results do not change from run to run.
#include "tile_mm.h"
#include <algorithm>
#include <type_traits>

namespace svk {
namespace gf {
using namespace mm;

// act(g); 16-bit results take the short forms: SiLU to a relative 2^-21, far under half a step of either type, GELU as
// gelu16 says
template <typename T>
__device__ __forceinline__ float glu_act(float g, int act) {
  if (act == SVK_GLU_SILU) {
    if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g));
    else return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
  }
  if (act == SVK_GLU_GELU) {
    if constexpr (sizeof(T) == 4) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    else return gelu16(g);
  }
  return g > 0.f ? g : (g <= 0.f ? 0.f : g);     // NaN stays NaN
}
// act(g) and act'(g) of a kept projection.  Where it left f16's range it is an infinity: act(-inf) is 0, act' there 0 or 1
// (from 1e4 on act' is 0 or 1 in f32 as well); NaN stays NaN
template <typename T>
__device__ __forceinline__ void glu_grad(float g, int act, float& a, float& d) {
  g = g < -1e4f && act != SVK_GLU_RELU ? -1e4f : g;
  const float b = g > 1e4f ? 1e4f : g;
  if (act == SVK_GLU_SILU) {
    float s;
    if constexpr (sizeof(T) == 4) s = 1.0f / (1.0f + expf(-g));
    else s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
    a = g * s;
    d = s * (1.0f + b * (1.0f - s));
  } else if (act == SVK_GLU_GELU) {
    const float p = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    a = g * p;
    d = p + b * 0.3989422804014327f * expf(-0.5f * b * b);
  } else {
    a = g > 0.f ? g : (g <= 0.f ? 0.f : g);
    d = g > 0.f ? 1.f : 0.f;
  }
}

// ACT: the activation, or -1: `act`, chosen while running (few tokens)
template <typename T, int ACT>
struct GateEpi {
  T* h; long ldh;
  T* pre;                 // [M, 2H] contiguous, or null
  const float* bias;      // [2H] or null
  int M, H, act, per;
  bool past;              // rows of h and pre are whole lines
  void skip(long rows) {
    h += rows * ldh;
    if (pre) pre += rows * 2 * H;
  }

  __device__ __forceinline__ float activate(float g) const { return glu_act<T>(g, ACT < 0 ? act : ACT); }
  // a wave's columns: half gate, half up rows of the same hidden channels; the pairs of blocks interleaved where each
  // half has two
  template <class C> static constexpr int width() { return C::TN >= 4 ? 8 : 4; }
  template <class C> __device__ __forceinline__ long first(int tn) const { return (long)tn * (C::BN / 2); }
  template <class C> __device__ __forceinline__ uint32_t offset(int r, uint32_t ldb) const {
    const int in = r % C::WN, up = in >= C::WN / 2, c = in - up * (C::WN / 2);
    return (uint32_t)(r / C::WN * (C::WN / 2) + (width<C>() == 8 ? pair_col(c) : c) + up * H) * ldb;
  }
  // few tokens: `per` gate rows, then the up rows of the same channels
  static constexpr bool PAIR = true;
  __device__ __forceinline__ int skinny_row(int bid, int r) const {
    const int up = r >= per;
    return min(bid * per + min(r - up * per, per - 1), H - 1) + up * H;
  }
  __device__ __forceinline__ void skinny_write(int bid, int m, int n, float g, float u) const {
    const int c = bid * per + n;
    if (c >= H) return;
    if (bias) {
      g += bias[c];
      u += bias[H + c];
    }
    if (pre) {
      pre[(long)m * 2 * H + c] = from_f<T>(g);
      pre[(long)m * 2 * H + H + c] = from_f<T>(u);
    }
    h[(long)m * ldh + c] = from_f<T>(activate(g) * u);
  }
  template <class C, typename A>
  __device__ __forceinline__ void write(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq, int) const {
    if (C::NONTEMPORAL && past) rows_of<C, true>(acc, m0, tn, wn, fq);
    else rows_of<C, false>(acc, m0, tn, wn, fq);
  }
  template <class C, bool NTS, typename A>
  __device__ __forceinline__ void rows_of(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq) const {
    constexpr int TG = C::TN / 2, W = width<C>(), S = W / 4;
    static_assert(C::TN % 2 == 0 && TG % S == 0, "a wave's columns are half gate, half up");
#pragma unroll
    for (int j = 0; j < TG; j += S) {
      const int c = tn * (C::BN / 2) + wn * (C::WN / 2) + j * 16 + fq * W, left = H - c;
      if (left <= 0) continue;
      float bg[W], bu[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int at = min(c + e, H - 1);
        bg[e] = bias ? bias[at] : 0.f;
        bu[e] = bias ? bias[H + at] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int m = m0 + i * 16;
        if (m >= M) continue;
        float g[W], u[W], o[W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          g[e] = acc[i][j + e / 4][e % 4] + bg[e];
          u[e] = acc[i][j + TG + e / 4][e % 4] + bu[e];
          o[e] = activate(g[e]) * u[e];
        }
        if (pre) {
          put<T, W, NTS>(pre + (long)m * 2 * H + c, g, left);
          put<T, W, NTS>(pre + (long)m * 2 * H + H + c, u, left);
        }
        put<T, W, NTS>(h + (long)m * ldh + c, o, left);
      }
    }
  }
};

// v += the first n (of 4) values at `at`
__device__ __forceinline__ void add_to(float* v, const float* at, int n) {
  typedef f32x4 anywhere __attribute__((aligned(4)));
  if (n >= 4) {
    const f32x4 o = *reinterpret_cast<const anywhere*>(at);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += o[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] += at[e];
  }
}

// plain product of a col operand B: rounded to T; or (ADD) added in f32 to y; or an f32 slab of one part of the reduction
template <typename T, bool ADD>
struct PlainEpi {
  typedef std::conditional_t<ADD, float, T> out_t;
  out_t* y; long ldy;
  float* slab;            // [parts][M][N], or null
  int M, N;
  bool past;              // rows of y are whole lines
  void skip(long rows) { y += rows * ldy; }      // never with slabs
  template <class C, typename A>
  __device__ __forceinline__ void write(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq, int part) const {
    if (C::NONTEMPORAL && past) rows_of<C, true>(acc, m0, tn, wn, fq, part);
    else rows_of<C, false>(acc, m0, tn, wn, fq, part);
  }
  template <class C, bool NTS, typename A>
  __device__ __forceinline__ void rows_of(A (&acc)[C::TM][C::TN], int m0, int tn, int wn, int fq, int part) const {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int n = tn * C::BN + wn * C::WN + j * 16 + fq * 4, left = N - n;
      if (left <= 0) continue;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int m = m0 + i * 16;
        if (m >= M) continue;
        float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        if (slab) {
          put<float, 4, false>(slab + ((long)part * M + m) * N + n, v, left);
          continue;
        }
        out_t* at = y + (long)m * ldy + n;
        if constexpr (ADD) add_to(v, at, left);
        put<out_t, 4, NTS>(at, v, left);
      }
    }
  }
};

// The joins of the backward pass, one launch: results whose reduction was split, y[m][n] = sum of the parts' f32 slabs in
// order, and the bias gradient, db[c] = sum of the row blocks' sums.  The first workgroups join dx, then come dW's, then the bias's.
struct Slabs {
  const float* S;         // [parts][M][N]
  void* y; long ldy;
  int parts, M, N, blocks;        // workgroups that join it
  bool add;               // y is f32 and added to
};
constexpr int JOIN = 4;   // values a thread
template <typename T, bool ADD>
__device__ __forceinline__ void join_slabs(const Slabs& j, int block) {
  const long total = (long)j.M * j.N;
  T* y = static_cast<T*>(j.y);
  for (long i = ((long)block * 256 + threadIdx.x) * JOIN; i < total; i += (long)j.blocks * 256 * JOIN) {
    float v[JOIN] = {0.f, 0.f, 0.f, 0.f};
    if (total % JOIN == 0) {
      for (int s = 0; s < j.parts; ++s) {
        const f32x4 p = *reinterpret_cast<const f32x4*>(j.S + s * total + i);
#pragma unroll
        for (int e = 0; e < JOIN; ++e) v[e] += p[e];
      }
    } else {
      for (int s = 0; s < j.parts; ++s)
#pragma unroll
        for (int e = 0; e < JOIN; ++e)
          if (i + e < total) v[e] += j.S[s * total + i + e];
    }
    const long m = i / j.N;
    const int n = (int)(i - m * j.N);
    if (n + JOIN <= j.N) {
      if constexpr (ADD) add_to(v, y + m * j.ldy + n, JOIN);
      put<T, JOIN, false>(y + m * j.ldy + n, v, JOIN);
    } else {
#pragma unroll
      for (int e = 0; e < JOIN; ++e)
        if (i + e < total) {
          T* at = y + (i + e) / j.N * j.ldy + (i + e) % j.N;
          if constexpr (ADD) v[e] += *at;
          *at = from_f<T>(v[e]);
        }
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void join_all(Slabs x, Slabs w, const float* __restrict__ S, int rows, float* __restrict__ db,
                                                int N, bool add) {
  int b = blockIdx.x;
  if (b < x.blocks) return join_slabs<T, false>(x, b);
  b -= x.blocks;
  if (b < w.blocks) return w.add ? join_slabs<float, true>(w, b) : join_slabs<T, false>(w, b);
  b -= w.blocks;
  // 16 columns a workgroup, 16 threads a column
  __shared__ float part[16][17];
  const int cl = threadIdx.x & 15, t = threadIdx.x >> 4, c = b * 16 + cl;
  float v = 0.f;
  if (c < N)
    for (int r = t; r < rows; r += 16) v += S[(long)r * N + c];
  part[t][cl] = v;
  __syncthreads();
  if (t == 0 && c < N) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][cl];
    db[c] = add ? db[c] + s : s;
  }
}

// dg, du from the kept projections: D [M][ld] = dg | du | zeros up to ld; S [row blocks][2H] = their column sums over
// a block of rows, f32, before the rounding.  4 waves a workgroup, 64 * V columns, rows dealt to the waves in turn.
template <typename T>
__global__ __launch_bounds__(256) void gated_dpre(const T* __restrict__ pre, const T* __restrict__ dh, long lddh,
                                                  T* __restrict__ D, long ld, float* __restrict__ S, int M, int H, int act, int rows) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float sum[2][4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.y * 64 + lane) * V;
  const long r0 = (long)blockIdx.x * rows, r1 = min(r0 + rows, (long)M);
  const int nc = H - c;                       // columns that exist from c on
  float sg[V], su[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sg[e] = su[e] = 0.f;
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef vec anywhere __attribute__((aligned(sizeof(T))));
  auto get = [&](const T* p) -> vec {         // V columns at any alignment, zeros past the last
    if (nc >= V) return *reinterpret_cast<const anywhere*>(p);
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < nc ? p[e] : from_f<T>(0.f);
    return v;
  };
  auto set = [&](T* p, const vec& v) {
    if (nc >= V) *reinterpret_cast<anywhere*>(p) = v;
    else
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < nc) p[e] = v[e];
  };
  for (long r = r0 + wave; r < r1; r += 4) {
    if (nc > 0) {
      const vec g = get(pre + r * 2 * H + c), u = get(pre + r * 2 * H + H + c), d = get(dh + r * lddh + c);
      float dg[V], du[V];
      bool nan = false;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a, da;
        glu_grad<T>(to_f(g[e]), act, a, da);
        dg[e] = to_f(d[e]) * to_f(u[e]) * da;
        du[e] = to_f(d[e]) * a;
        nan |= __builtin_isunordered(dg[e], du[e]);
      }
      // a dh of 0, and an act' of 0 under a finite dh, win over an infinity (a projection kept past f16's range, whose f32
      // value the forward pass multiplied by 0; dh u past f32's range); NaN passes.  Looked at where a product is NaN only
      // (at every value it took 2 us more of the 11 that 1470 x 856 take in f32, so 0.2)
      if (nan) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float a, da;
          glu_grad<T>(to_f(g[e]), act, a, da);
          const float f = to_f(d[e]), v = to_f(u[e]);
          if (v == v && (f == 0.f ? da == da : da == 0.f && fabsf(f) < INFINITY)) dg[e] = 0.f;
          if (f == 0.f && a == a) du[e] = 0.f;
        }
      }
      vec og, ou;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        og[e] = from_f<T>(dg[e]);
        ou[e] = from_f<T>(du[e]);
        sg[e] += dg[e];
        su[e] += du[e];
      }
      set(D + r * ld + c, og);
      set(D + r * ld + H + c, ou);
    }
    // the padding of the row, by the last column block
    if (blockIdx.y == gridDim.y - 1 && 2 * H + lane < ld) D[r * ld + 2 * H + lane] = from_f<T>(0.f);
  }
  if (!S) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sum[0][wave][lane * V + e] = sg[e];
    sum[1][wave][lane * V + e] = su[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 64 * V; i += 256) {
    const int half = i / (64 * V), k = i % (64 * V), col = blockIdx.y * 64 * V + k;
    if (col < H) S[(long)blockIdx.x * 2 * H + half * H + col] = (sum[half][0][k] + sum[half][1][k]) + (sum[half][2][k] + sum[half][3][k]);
  }
}

// rows a workgroup of gated_dpre: 64, fewer where that leaves CUs idle (16: 4 a wave), more where the launch would have
// 2^32 threads
inline int dpre_rows(long m, long h) { return m >= 1L << 29 ? 1024 : (m * h >= 1L << 23 ? 64 : 16); }

// workspace of the backward pass: [dpre][x padded][w padded][bias partials][slabs of dx][slabs of dW]
struct BwdWs {
  long ldd, dpre, x, w, sums, xslabs, wslabs, total;
  int rows;
  Plan px{2, 1, 0, 2}, pw{2, 1, 0, 2};
  BwdWs(long es, long M, long H, long K, bool padx, bool db, bool dx, bool dw) {
    auto plan = [&](long m, long n, long k) {
      return es == 4 ? plan_tiles<float>(m, n, stages<float>(k), 64) : plan_tiles<bf16>(m, n, stages<bf16>(k), 64);
    };
    ldd = up16(2 * H * es) / es;
    dpre = up16(M * ldd * es);
    const long ldk = up16(K * es);
    x = padx ? up16(M * ldk) : 0;
    w = padx ? up16(2 * H * ldk) : 0;
    rows = dpre_rows(M, H);
    sums = db ? up16((M + rows - 1) / rows * 2 * H * 4) : 0;
    if (dx && M) px = plan(M, K, 2 * H);
    if (dw && M) pw = plan(2 * H, K, M);      // (no tokens: nothing to plan)
    xslabs = px.parts > 1 ? up16(px.parts * M * K * 4) : 0;
    wslabs = pw.parts > 1 ? up16(pw.parts * 2 * H * K * 4) : 0;
    total = dpre + x + w + sums + xslabs + wslabs;
  }
};

// (a row that is padded to whole 16-byte pieces has as many stages)
template <typename T>
inline Plan forward_plan(long M, long H, long K) { return plan_tiles<T>(M, 2 * H, stages<T>(K), 1); }

static bool bad_dims(long M, long H, long K) {
  // 32-bit row and column counts inside a kernel; 65535 column blocks of gated_dpre
  return M < 0 || H <= 0 || K <= 0 || M > 0x7fffff00L || H > 4000000L || K > 0x1fffff00L;
}

static int es_of(int dtype) { return dtype == SVK_F32 ? 4 : (dtype == SVK_BF16 || dtype == SVK_F16 ? 2 : 0); }

}  // namespace gf
}  // namespace svk

using namespace svk;
using namespace svk::gf;

// rows that the tiled kernels can read as they are
static bool rows_ok(const void* p, long ld, long width, long es) { return al16(p) && ld * es % 16 == 0 && width * es % 16 == 0; }

extern "C" long svk_gated_ffn_workspace(int dtype, const void* X, long ldx, const void* W, long ldw, long M, long H, long K) {
  const long es = es_of(dtype);
  if (!es || bad_dims(M, H, K) || M <= SKINNY_M) return 0;
  const long ldk = up16(K * es);
  return (rows_ok(X, ldx, K, es) ? 0 : M * ldk) + (rows_ok(W, ldw, K, es) ? 0 : 2 * H * ldk);
}

extern "C" int svk_gated_ffn_plan(int dtype, int product, long M, long H, long K, long* plan) {
  const long es = es_of(dtype);
  if (!es || bad_dims(M, H, K) || M == 0 || product < 0 || product > 2 || !plan) { set_error("svk_gated_ffn_plan: bad args"); return SVK_EINVAL; }
  if (product == 0) {
    if (M <= SKINNY_M) tell_few(M, plan);
    else tell(es == 4 ? forward_plan<float>(M, H, K) : forward_plan<bf16>(M, H, K), M, plan);
    return SVK_OK;
  }
  const BwdWs ws(es, M, H, K, false, false, product == 1, product == 2);
  if (product == 1) tell(ws.px, M, plan);
  else tell(ws.pw, 2 * H, plan);
  return SVK_OK;
}

extern "C" int svk_gated_ffn(int dtype, const void* X, long ldx, const void* W, long ldw, const float* bias, void* Hout,
                             long ldh, void* pre, long M, long H, long K, int act, void* ws, long ws_bytes, void* stream) {
  const long es = es_of(dtype);
  if (!es) { set_error("svk_gated_ffn: unsupported dtype %d", dtype); return SVK_EINVAL; }
  if (!X || !W || !Hout || bad_dims(M, H, K) || ldx < K || ldw < K || ldh < H || act < SVK_GLU_SILU || act > SVK_GLU_RELU) {
    set_error("svk_gated_ffn: bad args");
    return SVK_EINVAL;
  }
  const long ldk = up16(K * es);
  if (2 * H * std::max(ldw * es, ldk) >= (1L << 32) || 256 * std::max(ldx * es, ldk) >= (1L << 32)) {
    set_error("svk_gated_ffn: weights or 256 rows of x of 4 GiB or more");
    return SVK_EUNSUPPORTED;
  }
  const long need = svk_gated_ffn_workspace(dtype, X, ldx, W, ldw, M, H, K);
  if (need && (!ws || !al16(ws) || ws_bytes < need)) { set_error("svk_gated_ffn: workspace too small or misaligned"); return SVK_EINVAL; }
  if (M == 0) return SVK_OK;
  hipStream_t st = (hipStream_t)stream;
  SVK_DISPATCH_DTYPE(dtype, T, {
    const bool past = whole_lines(Hout, ldh * es, H * es) && (!pre || whole_lines(pre, 0, 0));
    Args p{(const char*)X, (const char*)W, ldx * es, ldw * es, 0, 0, (int)M, (int)K, 0, 0, 0, 1};
    if (M <= SKINNY_M) {
      GateEpi<T, -1> epi{(T*)Hout, ldh, (T*)pre, bias, (int)M, (int)H, act, 0, past};
      return few_tokens<T, 2>(p, H, epi, st, "gated_ffn_few");
    }
    char* at = (char*)ws;
    if (!rows_ok(X, ldx, K, es)) {
      if (int rc = pad<T>(X, ldx * es, at, M, K * es, st)) return rc;
      p.A = at;
      p.lda = ldk;
      at += M * ldk;
      p.K = (int)(ldk / es);
    }
    if (!rows_ok(W, ldw, K, es)) {
      if (int rc = pad<T>(W, ldw * es, at, 2 * H, K * es, st)) return rc;
      p.B = at;
      p.ldb = ldk;
      p.K = (int)(ldk / es);
    }
    p.abytes = (M - 1) * p.lda + p.K * es;
    p.bbytes = (2 * H - 1) * p.ldb + p.K * es;
    p.nk = stages<T>(p.K);
    const Plan plan = forward_plan<T>(M, H, K);
    auto run = [&](auto act_c) {
      GateEpi<T, decltype(act_c)::value> epi{(T*)Hout, ldh, (T*)pre, bias, (int)M, (int)H, act, 0, past};
      return launch_plan<T, false, false>(plan, p, M, 2 * H, epi, st, "gated_ffn");
    };
    if (act == SVK_GLU_SILU) return run(std::integral_constant<int, SVK_GLU_SILU>{});
    if (act == SVK_GLU_GELU) return run(std::integral_constant<int, SVK_GLU_GELU>{});
    return run(std::integral_constant<int, SVK_GLU_RELU>{});
  });
}

extern "C" long svk_gated_ffn_bwd_workspace(int dtype, const void* X, long ldx, const void* W, long ldw, long M, long H,
                                            long K, int want_dx, int want_dw, int want_db) {
  const long es = es_of(dtype);
  if (!es || bad_dims(M, H, K) || M == 0) return 0;
  const bool padx = !rows_ok(X, ldx, K, es) || !rows_ok(W, ldw, K, es);
  return BwdWs(es, M, H, K, padx, want_db, want_dx, want_dw).total;
}

// add: SVK_ADD_DW (dW is f32), SVK_ADD_DB
static int backward(int dtype, const void* X, long ldx, const void* W, long ldw, const void* pre, const void* dH, long lddh,
                    void* dX, long lddx, void* dW, float* db, int add, long M, long H, long K, int act, void* ws, long ws_bytes,
                    void* stream) {
  const long es = es_of(dtype);
  if (!es) { set_error("svk_gated_ffn_bwd: unsupported dtype %d", dtype); return SVK_EINVAL; }
  if (!X || !W || !pre || !dH || bad_dims(M, H, K) || ldx < K || ldw < K || lddh < H || (dX && lddx < K) ||
      act < SVK_GLU_SILU || act > SVK_GLU_RELU) {
    set_error("svk_gated_ffn_bwd: bad args");
    return SVK_EINVAL;
  }
  const long ldk = up16(K * es);
  if (256 * std::max(std::max(ldx, ldw) * es, std::max(ldk, up16(2 * H * es))) >= (1L << 32)) {
    set_error("svk_gated_ffn_bwd: 256 rows of 4 GiB or more");
    return SVK_EUNSUPPORTED;
  }
  const bool padx = !rows_ok(X, ldx, K, es) || !rows_ok(W, ldw, K, es);
  const BwdWs need(es, M, H, K, padx, db, dX, dW);
  if (M && (!ws || !al16(ws) || ws_bytes < need.total)) { set_error("svk_gated_ffn_bwd: workspace too small or misaligned"); return SVK_EINVAL; }
  hipStream_t st = (hipStream_t)stream;
  const bool add_w = add & SVK_ADD_DW, add_b = add & SVK_ADD_DB;
  SVK_DISPATCH_DTYPE(dtype, T, {
    auto blocks_of = [](long values) { return (int)std::min<long>((values + 256 * JOIN - 1) / (256 * JOIN), 4096); };
    Slabs jx{};
    Slabs jw{};
    const int db_blocks = db && (M || !add_b) ? (int)((2 * H + 15) / 16) : 0;
    auto join = [&](const float* sums, int rows) -> int {
      const int all = jx.blocks + jw.blocks + db_blocks;
      if (!all) return SVK_OK;
      hipLaunchKernelGGL((join_all<T>), dim3((unsigned)all), dim3(256), 0, st, jx, jw, sums, rows, db, (int)(2 * H), add_b);
      return check_launch("join_all");
    };
    if (M == 0) {                                   // no tokens: the sums are empty
      if (dW && !add_w) jw = Slabs{nullptr, dW, K, 0, (int)(2 * H), (int)K, blocks_of(2 * H * K), false};
      return join(nullptr, 0);
    }
    char* at = (char*)ws;
    T* D = (T*)at;
    at += need.dpre;
    const char *Xr = (const char*)X, *Wr = (const char*)W;
    long ldxb = ldx * es, ldwb = ldw * es;
    const long kb = padx ? ldk : K * es;            // bytes of a row of either
    if (padx) {
      if (int rc = pad<T>(X, ldx * es, at, M, K * es, st)) return rc;
      Xr = at;
      ldxb = ldk;
      at += need.x;
      if (int rc = pad<T>(W, ldw * es, at, 2 * H, K * es, st)) return rc;
      Wr = at;
      ldwb = ldk;
      at += need.w;
    }
    float* sums = db ? (float*)at : nullptr;
    at += need.sums;
    const int rowblocks = (int)((M + need.rows - 1) / need.rows);
    constexpr int V = 16 / (int)sizeof(T);
    hipLaunchKernelGGL((gated_dpre<T>), dim3(rowblocks, (unsigned)((H + 64 * V - 1) / (64 * V))), dim3(256), 0, st,
                       (const T*)pre, (const T*)dH, lddh, D, need.ldd, sums, (int)M, (int)H, act, need.rows);
    if (int rc = check_launch("gated_dpre")) return rc;
    // y [m, n]; where its reduction is split, the parts' slabs, joined below
    auto product = [&](auto ac, auto addc, Plan plan, Args p, void* y, long ldy, long m, long n, Slabs& j, const char* name) -> int {
      typedef PlainEpi<T, decltype(addc)::value> Epi;
      constexpr long out = sizeof(typename Epi::out_t);
      p.nk = stages<T>(p.K);
      float* slabs = plan.parts > 1 ? (float*)at : nullptr;
      Epi epi{(typename Epi::out_t*)y, ldy, slabs, (int)m, (int)n, whole_lines(y, ldy * out, n * out)};
      if (slabs) {
        j = Slabs{slabs, y, ldy, plan.parts, (int)m, (int)n, blocks_of(m * n), decltype(addc)::value};
        at += up16(plan.parts * m * n * 4);
      }
      return launch_plan<T, decltype(ac)::value, true>(plan, p, m, n, epi, st, name);
    };
    const long Db = M * need.ldd * es;
    // the padding of D is zero and rows of W past 2H read as zero, so dx's reduction runs over whole chunks
    if (dX)
      if (int rc = product(std::false_type{}, std::false_type{}, need.px,
                           Args{(const char*)D, Wr, need.ldd * es, ldwb, Db, (2 * H - 1) * ldwb + kb, 0, (int)(2 * H), 0, 0, 0, 1},
                           dX, lddx, M, K, jx, "gated_ffn_dx")) return rc;
    if (dW) {
      const Args a{(const char*)D, Xr, need.ldd * es, ldxb, Db, (M - 1) * ldxb + kb, 0, (int)M, 0, 0, 0, 1};
      if (int rc = add_w ? product(std::true_type{}, std::true_type{}, need.pw, a, dW, K, 2 * H, K, jw, "gated_ffn_dw")
                         : product(std::true_type{}, std::false_type{}, need.pw, a, dW, K, 2 * H, K, jw, "gated_ffn_dw")) return rc;
    }
    return join(sums, rowblocks);
  });
}

extern "C" int svk_gated_ffn_bwd(int dtype, const void* X, long ldx, const void* W, long ldw, const void* pre,
                                 const void* dH, long lddh, void* dX, long lddx, void* dW, float* db, long M, long H, long K,
                                 int act, void* ws, long ws_bytes, void* stream) {
  return backward(dtype, X, ldx, W, ldw, pre, dH, lddh, dX, lddx, dW, db, 0, M, H, K, act, ws, ws_bytes, stream);
}

extern "C" int svk_gated_ffn_bwd_add(int dtype, const void* X, long ldx, const void* W, long ldw, const void* pre,
                                     const void* dH, long lddh, void* dX, long lddx, void* dW, float* db, int add, long M,
                                     long H, long K, int act, void* ws, long ws_bytes, void* stream) {
  if (add & ~(SVK_ADD_DW | SVK_ADD_DB)) { set_error("svk_gated_ffn_bwd: unknown bits in add"); return SVK_EINVAL; }
  return backward(dtype, X, ldx, W, ldw, pre, dH, lddh, dX, lddx, dW, db, add, M, H, K, act, ws, ws_bytes, stream);
}
