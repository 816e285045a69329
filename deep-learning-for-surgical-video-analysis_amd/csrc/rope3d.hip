// Rotary positions with three axes (svk_rope3d): tokens of a video carry (time, row, column), and pair i of every head
// is turned by th = pos[axis(i)] f_i:
//
//   (x, y) -> (x cos th - y sin th, x sin th + y cos th)
//
// Pairs are (i, i + R) of the first 2R channels of a head (halves) or (2i, 2i + 1) (interleaved); channels from 2R on
// pass unchanged.  The gradient turns by -th: the same kernel with the sine's sign changed.
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there (a frame number of 1e5 times f = 1 has no
// useful fraction left in f32), the sine and cosine of the reduced angle in f32.  A workgroup forms the R pairs of its
// tokens once, in LDS, for all heads of q and k: 2 R sines a token against (Hq + Hk) hd values moved.
// Bound by HBM: q and k are read once and written once, as 16-byte pieces.
#include "svk_common.h"
#include <algorithm>
#include <type_traits>

namespace svk {
namespace rope {

struct Map {
  const char* x;
  char* y;
  long ldx, sbx, ldy, sby;      // values between tokens / batches
  int heads;
};
struct RopeArgs {
  Map q, k;                     // k.heads == 0: no k
  const char* pos;
  long ldp, sbp;                // values between tokens / batches (sbp 0: one table for all)
  const double* freqs;
  int nt, nh, R, hd, N, tokens, tpb;
  bool apart;                   // the outputs are not the inputs
  float sign;
};

// n values (V where n >= V) of any alignment
template <typename T, int V>
__device__ __forceinline__ void get(const T* p, int n, float* v) {
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef vec anywhere __attribute__((aligned(sizeof(T))));
  if (n >= V) {
    const vec w = *reinterpret_cast<const anywhere*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = to_f(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < n ? to_f(p[e]) : 0.f;
  }
}
// A value's last rounding in f32, kept apart from the conversion: the compiler fuses the two into one instruction with one
// rounding (v_fma_mixlo_f16) for some of a piece's pairs and not for others, and a pair's bits must not depend on where it
// lies (pieces overlap).  The same time.
template <typename T>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (std::is_same<T, f16>::value) asm("" : "+v"(v));
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void set(T* p, int n, const float* v) {
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef vec anywhere __attribute__((aligned(sizeof(T))));
  if (n >= V) {
    vec w;
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = from_f<T>(rounded<T>(v[e]));
    *reinterpret_cast<anywhere*>(p) = w;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) p[e] = from_f<T>(rounded<T>(v[e]));
  }
}

// A unit: V channels, 16 bytes (V pairs of the halves layout: two pieces), fewer at the end of a part of the head (WHOLE:
// nowhere).  Pieces need no alignment (pairs 19 apart in heads of 72, 161 MB: 41 us, value by value 142).
template <typename T, typename P, bool IL, bool WHOLE>
__global__ __launch_bounds__(256) void rope3d(RopeArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ float2 cs[];                                // [tokens of the workgroup][R]: cos, sin
  const int t0 = blockIdx.x * a.tpb, nt = min(a.tpb, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * a.R; i += 256) {
    const int t = i / a.R, r = i - t * a.R, tok = t0 + t, b = tok / a.N, n = tok - b * a.N;
    const int ax = r < a.nt ? 0 : (r < a.nt + a.nh ? 1 : 2);
    const double p = (double)reinterpret_cast<const P*>(a.pos)[b * a.sbp + n * a.ldp + ax];
    double turns = p * a.freqs[r] * 0.15915494309189533577;     // 1 / 2 pi
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = float2{c, a.sign * s};
  }
  __syncthreads();
  const int part = IL ? 2 * a.R : a.R, rot = (part + V - 1) / V;       // units of a head's rotated part
  const int uph = rot + (a.hd - 2 * a.R + V - 1) / V, upt = uph * (a.q.heads + a.k.heads);
  for (int u = threadIdx.x; u < nt * upt; u += 256) {
    const int t = u / upt, v = u - t * upt;
    int h = v / uph;
    const int w = v - h * uph, tok = t0 + t, b = tok / a.N, n = tok - b * a.N;
    const bool isk = h >= a.q.heads;
    const Map& m = isk ? a.k : a.q;
    h -= isk ? a.q.heads : 0;
    const T* x = reinterpret_cast<const T*>(m.x) + b * m.sbx + n * m.ldx + (long)h * a.hd;
    T* y = reinterpret_cast<T*>(m.y) + b * m.sby + n * m.ldy + (long)h * a.hd;
    const float2* z = cs + t * a.R;
    float p[V], q[V], o[V];
    if (w >= rot) {                                             // past the pairs: the values themselves
      if (x == y) continue;                                     // in place: there already
      int c = 2 * a.R + (w - rot) * V;
      if (!WHOLE && c + V > a.hd && a.hd - V >= 2 * a.R) c = a.hd - V;       // the last piece: a whole one that overlaps
      const int left = a.hd - c;
      typedef uint32_t four __attribute__((ext_vector_type(4)));
      typedef four anywhere __attribute__((aligned(2)));
      if (WHOLE || left >= V) *reinterpret_cast<anywhere*>(y + c) = *reinterpret_cast<const anywhere*>(x + c);
      else
        for (int e = 0; e < left; ++e) y[c + e] = x[c + e];
      continue;
    }
    int c = w * V;
    // the last piece of the rotated part: a whole one that overlaps the one before, unless that is being turned in place
    if (!WHOLE && a.apart && c + V > part && part >= V) c = part - V;
    if constexpr (IL) {
      get<T, V>(x + c, WHOLE ? V : part - c, p);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 r = z[WHOLE ? (c + e) >> 1 : min((c + e) >> 1, a.R - 1)];
        o[e] = p[e] * r.x - p[e + 1] * r.y;
        o[e + 1] = p[e] * r.y + p[e + 1] * r.x;
      }
      set<T, V>(y + c, WHOLE ? V : part - c, o);
    } else {
      get<T, V>(x + c, WHOLE ? V : part - c, p);
      get<T, V>(x + a.R + c, WHOLE ? V : part - c, q);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 r = z[WHOLE ? c + e : min(c + e, a.R - 1)];
        const float f = p[e], g = q[e];
        o[e] = f * r.x - g * r.y;
        q[e] = f * r.y + g * r.x;
      }
      set<T, V>(y + c, WHOLE ? V : part - c, o);
      set<T, V>(y + a.R + c, WHOLE ? V : part - c, q);
    }
  }
}

template <typename T, typename P>
static int launch(const RopeArgs& a, bool il, hipStream_t st) {
  const dim3 grid((unsigned)((a.tokens + a.tpb - 1) / a.tpb)), block(256);
  const size_t lds = (size_t)a.tpb * a.R * sizeof(float2);
  constexpr int V = 16 / (int)sizeof(T);
  const bool whole = (il ? 2 * a.R : a.R) % V == 0 && (a.hd - 2 * a.R) % V == 0;
  if (il && whole) hipLaunchKernelGGL((rope3d<T, P, true, true>), grid, block, lds, st, a);
  else if (il) hipLaunchKernelGGL((rope3d<T, P, true, false>), grid, block, lds, st, a);
  else if (whole) hipLaunchKernelGGL((rope3d<T, P, false, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((rope3d<T, P, false, false>), grid, block, lds, st, a);
  return check_launch("rope3d");
}

}  // namespace rope
}  // namespace svk

using namespace svk;
using namespace svk::rope;

extern "C" int svk_rope3d(int dtype, const void* Q, long ldq, long sbq, void* Qo, long ldqo, long sbqo, int heads,
                          const void* K, long ldk, long sbk, void* Ko, long ldko, long sbko, int kv_heads, const void* pos,
                          int pos_type, long ldp, long sbp, const double* freqs, int nt, int nh, int nw, int hd, int B, int N,
                          int interleaved, int inverse, void* stream) {
  const long Rl = (long)nt + nh + nw;
  const int R = (int)Rl;
  if (!Q || !Qo || heads <= 0 || kv_heads < 0 || (kv_heads && (!K || !Ko)) || !pos || !freqs || nt < 0 || nh < 0 || nw < 0 ||
      Rl < 1 || 2 * Rl > hd || B < 0 || N < 0 || (pos_type != SVK_POS_I32 && pos_type != SVK_POS_I64 && pos_type != SVK_POS_F32)) {
    set_error("svk_rope3d: bad args");
    return SVK_EINVAL;
  }
  if (hd > 4096 || (long)heads + kv_heads > 65536 || (long)B * N > 0x7fff0000L) {
    set_error("svk_rope3d: head width over 4096, over 65536 heads or over 2^31 tokens");
    return SVK_EUNSUPPORTED;
  }
  if (B == 0 || N == 0) return SVK_OK;
  // in place with the same strides only, and neither output in the other's input (read by other threads meanwhile)
  auto moved = [&](const void* in, long ld, long sb, const void* out, long ldo, long sbo) {
    return in == out && ((N > 1 && ld != ldo) || (B > 1 && sb != sbo));
  };
  if (moved(Q, ldq, sbq, Qo, ldqo, sbqo) ||
      (kv_heads && (Qo == K || Ko == Q || Qo == Ko || moved(K, ldk, sbk, Ko, ldko, sbko)))) {
    set_error("svk_rope3d: an output overlaps an input or the other output");
    return SVK_EINVAL;
  }
  SVK_DISPATCH_DTYPE(dtype, T, {
    RopeArgs a{};
    a.q = Map{(const char*)Q, (char*)Qo, ldq, sbq, ldqo, sbqo, heads};
    if (kv_heads) a.k = Map{(const char*)K, (char*)Ko, ldk, sbk, ldko, sbko, kv_heads};
    a.pos = (const char*)pos;
    a.ldp = ldp; a.sbp = sbp; a.freqs = freqs;
    a.nt = nt; a.nh = nh; a.R = R; a.hd = hd; a.N = N; a.tokens = B * N;
    a.apart = Qo != Q && (!kv_heads || Ko != K);
    a.sign = inverse ? -1.f : 1.f;
    constexpr int V = 16 / (int)sizeof(T);
    // about 1024 units (4 a thread) a workgroup, fewer where that would leave CUs idle; the table within 32 KiB of LDS
    const long upt = (long)(heads + kv_heads) * ((hd + V - 1) / V);
    long tpb = std::min<long>(std::max<long>(1, 1024 / upt), std::max<long>(1, a.tokens / 2048));
    tpb = std::max<long>(1, std::min<long>(tpb, 4096 / R));
    a.tpb = (int)std::max<long>(tpb, ((long)a.tokens + (1L << 23) - 1) >> 23);   // a launch has under 2^32 threads
    if ((long)a.tpb * R > 8192) { set_error("svk_rope3d: too many tokens of so many pairs"); return SVK_EUNSUPPORTED; }
    if (pos_type == SVK_POS_I32) return launch<T, int>(a, interleaved, (hipStream_t)stream);
    if (pos_type == SVK_POS_I64) return launch<T, long>(a, interleaved, (hipStream_t)stream);
    return launch<T, float>(a, interleaved, (hipStream_t)stream);
  });
}
