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
// Bound by HBM: q and k are read once and written once, as 16-byte pieces where rows allow it.
#include "svk_common.h"
#include <algorithm>

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
  float sign;
};

// V channels a unit (a pair of V-channel pieces in the halves layout's rotated part)
template <typename T, typename P, int V, bool IL>
__global__ __launch_bounds__(256) void rope3d(RopeArgs a) {
  extern __shared__ float2 cs[];                                // [tokens of the workgroup][R]: cos, sin
  typedef T vec __attribute__((ext_vector_type(V)));
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
  const int rot = IL ? 2 * a.R / V : a.R / V;                   // units of a head's rotated part
  const int uph = rot + (a.hd - 2 * a.R) / V, upt = uph * (a.q.heads + a.k.heads);
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
    if (w >= rot) {
      const int c = 2 * a.R + (w - rot) * V;
      *reinterpret_cast<vec*>(y + c) = *reinterpret_cast<const vec*>(x + c);
    } else if constexpr (IL) {
      const int c = w * V;
      const vec p = *reinterpret_cast<const vec*>(x + c);
      vec o;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 r = z[(c + e) >> 1];
        const float f = to_f(p[e]), g = to_f(p[e + 1]);
        o[e] = from_f<T>(f * r.x - g * r.y);
        o[e + 1] = from_f<T>(f * r.y + g * r.x);
      }
      *reinterpret_cast<vec*>(y + c) = o;
    } else {
      const int c = w * V;
      const vec p = *reinterpret_cast<const vec*>(x + c), q = *reinterpret_cast<const vec*>(x + a.R + c);
      vec o, s;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 r = z[c + e];
        const float f = to_f(p[e]), g = to_f(q[e]);
        o[e] = from_f<T>(f * r.x - g * r.y);
        s[e] = from_f<T>(f * r.y + g * r.x);
      }
      *reinterpret_cast<vec*>(y + c) = o;
      *reinterpret_cast<vec*>(y + a.R + c) = s;
    }
  }
}

template <typename T, typename P>
static int launch(const RopeArgs& a, bool vec, bool il, hipStream_t st) {
  const dim3 grid((unsigned)((a.tokens + a.tpb - 1) / a.tpb)), block(256);
  const size_t lds = (size_t)a.tpb * a.R * sizeof(float2);
  constexpr int V = 16 / (int)sizeof(T);
  if (vec && il) hipLaunchKernelGGL((rope3d<T, P, V, true>), grid, block, lds, st, a);
  else if (vec) hipLaunchKernelGGL((rope3d<T, P, V, false>), grid, block, lds, st, a);
  else if (il) hipLaunchKernelGGL((rope3d<T, P, 2, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((rope3d<T, P, 1, false>), grid, block, lds, st, a);
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
  const int R = nt + nh + nw;
  if (!Q || !Qo || heads <= 0 || kv_heads < 0 || (kv_heads && (!K || !Ko)) || !pos || !freqs || nt < 0 || nh < 0 || nw < 0 ||
      R < 1 || 2 * (long)R > hd || B < 0 || N < 0 || (pos_type != SVK_POS_I32 && pos_type != SVK_POS_I64 && pos_type != SVK_POS_F32)) {
    set_error("svk_rope3d: bad args");
    return SVK_EINVAL;
  }
  if (hd > 4096 || (long)heads + kv_heads > 65536 || (long)B * N > 0x7fff0000L) {
    set_error("svk_rope3d: head width over 4096, over 65536 heads or over 2^31 tokens");
    return SVK_EUNSUPPORTED;
  }
  if (B == 0 || N == 0) return SVK_OK;
  SVK_DISPATCH_DTYPE(dtype, T, {
    RopeArgs a{};
    a.q = Map{(const char*)Q, (char*)Qo, ldq, sbq, ldqo, sbqo, heads};
    if (kv_heads) a.k = Map{(const char*)K, (char*)Ko, ldk, sbk, ldko, sbko, kv_heads};
    a.pos = (const char*)pos;
    a.ldp = ldp; a.sbp = sbp; a.freqs = freqs;
    a.nt = nt; a.nh = nh; a.R = R; a.hd = hd; a.N = N; a.tokens = B * N;
    a.sign = inverse ? -1.f : 1.f;
    constexpr int V = 16 / (int)sizeof(T);
    auto ok = [&](const Map& m) {
      return !m.heads || (((((uintptr_t)m.x) | ((uintptr_t)m.y)) & 15) == 0 && (m.ldx | m.sbx | m.ldy | m.sby) % V == 0);
    };
    const bool vec = hd % V == 0 && (interleaved ? 2 * R : R) % V == 0 && (hd - 2 * R) % V == 0 && ok(a.q) && ok(a.k);
    // interleaved pairs are moved two values at a time where 16-byte pieces do not fit; that needs even rows
    auto even = [&](const Map& m) {
      return !m.heads || (((((uintptr_t)m.x) | ((uintptr_t)m.y)) & (2 * sizeof(T) - 1)) == 0 && (m.ldx | m.sbx | m.ldy | m.sby) % 2 == 0);
    };
    if (interleaved && !vec && !(hd % 2 == 0 && even(a.q) && even(a.k))) {
      set_error("svk_rope3d: interleaved pairs need an even head width, even strides and pair-aligned pointers");
      return SVK_EUNSUPPORTED;
    }
    // about 1024 units (4 a thread) a workgroup, fewer where that would leave CUs idle; the table within 32 KiB of LDS
    const long upt = (long)(heads + kv_heads) * (vec ? hd / V : hd);
    long tpb = std::min<long>(std::max<long>(1, 1024 / upt), std::max<long>(1, a.tokens / 2048));
    a.tpb = (int)std::max<long>(1, std::min<long>(tpb, 4096 / R));
    if (pos_type == SVK_POS_I32) return launch<T, int>(a, vec, interleaved, (hipStream_t)stream);
    if (pos_type == SVK_POS_I64) return launch<T, long>(a, vec, interleaved, (hipStream_t)stream);
    return launch<T, float>(a, vec, interleaved, (hipStream_t)stream);
  });
}
