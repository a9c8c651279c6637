// Rotary embedding over several position axes for gfx950.
//
// Pair j of a head's features (R = sum of the sections; pairs (j, j + R), or
// (2j, 2j + 1) interleaved) turns by position[axis(j)] * inv_freq[j]; features
// from 2R on pass through.  The backward is the turn by the negative angle.
//
// Bound by memory: one read and one write of x.  A token's R cosines and sines
// are computed once, in LDS, for all its heads; the angle in turns is reduced
// with products in two doubles, so that any 64-bit position keeps fp32's
// precision.  A thread's first piece of x is on its way while the angles are
// computed, and each next one while the last is turned: 3 x 8191 tokens of 12
// heads of 128 bf16 features 36 us, 4.2 TB/s (without this, and with 8-byte
// pieces where pairs are side by side, 48).
#include "common.h"

namespace uttt {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxAxes = 8;
constexpr int kRotPairs = 2048;   // cosines and sines of a workgroup's tokens, 16 KiB
constexpr int kRotTokens = 256;   // tokens of a workgroup at most

struct RotArgs {
  const void* x;
  int64_t x_sb, x_sl, x_sh;
  const void* pos;
  int pos64;
  int64_t p_sb, p_sl, p_sa;
  const float* freq;
  int ends[kMaxAxes];   // pairs up to and with each axis
  int axes, B, L, H, D, R, tokens;   // tokens of a workgroup
  float sign;
  void* y;              // [B, L, H, D]
};

// V elements of one type at a time
template <class TT, int V>
struct Vec {
  using S = typename TT::S;
  __device__ __forceinline__ static void load(const S* p, float (&v)[V]) {
    S w[V];
    __builtin_memcpy(w, __builtin_assume_aligned(p, V * sizeof(S) > 16 ? 16 : V * sizeof(S)), sizeof w);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = TT::load(w[i]);
  }
  __device__ __forceinline__ static void store(S* p, const float (&v)[V]) {
    S w[V];
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = TT::store(v[i]);
    __builtin_memcpy(__builtin_assume_aligned(p, V * sizeof(S) > 16 ? 16 : V * sizeof(S)), w, sizeof w);
  }
};

// p f / pi without whole turns, in [-1, 1], to 2^-106 of |p f|: f / pi and its
// product with p in two doubles each.
__device__ __forceinline__ double half_turns(double p, double f) {
  constexpr double kInvPi = 0x1.45f306dc9c883p-2, kInvPiLow = -0x1.6b01ec5417056p-56;
  const double fh = f * kInvPi, fl = __builtin_fma(f, kInvPiLow, __builtin_fma(f, kInvPi, -fh));
  const double h = p * fh, l = __builtin_fma(p, fl, __builtin_fma(p, fh, -h));
  const double x = (h - 2.0 * rint(0.5 * h)) + l;
  return x - 2.0 * rint(0.5 * x);
}

template <class TT, int V, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotary_axes_kernel(RotArgs a) {
  using S = typename TT::S;
  __shared__ float cs[kRotPairs], sn[kRotPairs];
  __shared__ int64_t xat[kRotTokens], pat[kRotTokens];   // tokens' places in x and in the positions
  const int64_t first = (int64_t)blockIdx.x * a.tokens, all = (int64_t)a.B * a.L;
  const int nt = (int)min((int64_t)a.tokens, all - first);
  for (int t = threadIdx.x; t < nt; t += kRotThreads) {
    const uint32_t b = (uint32_t)(first + t) / (uint32_t)a.L, l = (uint32_t)(first + t) - b * (uint32_t)a.L;
    xat[t] = b * a.x_sb + l * a.x_sl;
    pat[t] = b * a.p_sb + l * a.p_sl;
  }
  __syncthreads();
  // A piece is 2V features of a token's head: V pairs, or after the pairs
  // features that pass through (turned by 0).  The next of a thread is
  // kRotThreads further on, by sums and carries, and is loaded a piece ahead.
  const int rp = a.R / V, per = (a.D + 2 * V - 1) / (2 * V);
  const int dth = kRotThreads / per, de = kRotThreads - dth * per, dt = dth / a.H, dh = dth - dt * a.H;
  struct Piece {
    int t, h, e;
    float u[V], w[V];
  };
  // first features of a piece's two halves, and whether it has the second
  const auto at_u = [&](int e) { return INTER ? 2 * V * e : e < rp ? V * e : 2 * V * e; };
  const auto at_w = [&](int e) { return INTER ? 2 * V * e + V : e < rp ? a.R + V * e : 2 * V * e + V; };
  const auto load = [&](Piece& p) {
    if (p.t >= nt) return;
    const S* x = static_cast<const S*>(a.x) + xat[p.t] + p.h * a.x_sh;
    Vec<TT, V>::load(x + at_u(p.e), p.u);
    if (at_w(p.e) < a.D) Vec<TT, V>::load(x + at_w(p.e), p.w);
  };
  Piece next;
  const int th = threadIdx.x / per;
  next.e = threadIdx.x - th * per;
  next.t = th / a.H;
  next.h = th - next.t * a.H;
  load(next);
  for (int i = threadIdx.x; i < nt * a.R; i += kRotThreads) {
    const int t = i / a.R, j = i - t * a.R;
    int axis = 0;
    while (j >= a.ends[axis]) ++axis;
    const int64_t at = pat[t] + axis * a.p_sa;
    const double f = (double)a.freq[j];
    double half;
    if (a.pos64) {
      const int64_t p = static_cast<const int64_t*>(a.pos)[at];
      half = half_turns((double)(p >> 32) * 4294967296.0, f) + half_turns((double)(uint32_t)p, f);
      half -= 2.0 * rint(0.5 * half);
    } else {
      half = half_turns((double)static_cast<const int32_t*>(a.pos)[at], f);
    }
    float s, c;
    sincospif((float)half, &s, &c);
    cs[i] = c;
    sn[i] = a.sign * s;
  }
  __syncthreads();
  while (next.t < nt) {
    Piece p = next;
    next.e += de;
    next.h += dh;
    next.t += dt;
    if (next.e >= per) next.e -= per, ++next.h;
    if (next.h >= a.H) next.h -= a.H, ++next.t;
    load(next);
    if (p.e < rp) {
      const float *c = cs + p.t * a.R + V * p.e, *s = sn + p.t * a.R + V * p.e;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (INTER) {   // pairs 0 .. V/2-1 of the piece in u, the others in w
          float& m = 2 * k < V ? p.u[2 * k] : p.w[2 * k - V];
          float& o = 2 * k + 1 < V ? p.u[2 * k + 1] : p.w[2 * k + 1 - V];
          const float x = m, y = o;
          m = x * c[k] - y * s[k];
          o = x * s[k] + y * c[k];
        } else {
          const float x = p.u[k], y = p.w[k];
          p.u[k] = x * c[k] - y * s[k];
          p.w[k] = x * s[k] + y * c[k];
        }
      }
    }
    S* y = static_cast<S*>(a.y) + ((first + p.t) * a.H + p.h) * a.D;
    Vec<TT, V>::store(y + at_u(p.e), p.u);
    if (at_w(p.e) < a.D) Vec<TT, V>::store(y + at_w(p.e), p.w);
  }
}

template <class TT, int V>
void launch_rotary_as(const RotArgs& a, bool inter, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)a.B * a.L + a.tokens - 1) / a.tokens));
  if (inter) hipLaunchKernelGGL((rotary_axes_kernel<TT, V, true>), grid, dim3(kRotThreads), 0, st, a);
  else hipLaunchKernelGGL((rotary_axes_kernel<TT, V, false>), grid, dim3(kRotThreads), 0, st, a);
}

template <class TT>
int launch_rotary(RotArgs a, bool inter, hipStream_t st) {
  constexpr int V = 16 / sizeof(typename TT::S);
  // v pairs at a time: whole pieces, aligned throughout.  2 x 8191 tokens, 12
  // heads, read from memory: 16-byte pieces 2.9 TB/s, 8-byte ones (120 features,
  // 60 pairs) 2.5, single features (100 and 41) 1.7.
  const auto fits = [&](int v) {
    const int size = sizeof(typename TT::S), bytes = size * v;
    return a.R % v == 0 && (a.D * size) % bytes == 0 && (a.x_sb * size) % bytes == 0 &&
           (a.x_sl * size) % bytes == 0 && (a.x_sh * size) % bytes == 0 &&
           (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % bytes == 0;
  };
  // about four pieces a thread, and cosines that fit
  const int64_t pieces = (int64_t)a.H * a.D / (2 * V);
  int64_t tokens = pieces ? (4 * kRotThreads) / pieces : kRotTokens;
  tokens = tokens < 1 ? 1 : tokens > kRotTokens ? kRotTokens : tokens;
  if (tokens > kRotPairs / a.R) tokens = kRotPairs / a.R;
  const int64_t all = (int64_t)a.B * a.L;
  if (all / tokens < 1024) tokens = (all + 1023) / 1024 < tokens ? (all + 1023) / 1024 : tokens;
  a.tokens = (int)tokens;
  UTTT_REQUIRE((all + tokens - 1) / tokens * kRotThreads < (1LL << 32),
               "rotary_axes: too many tokens of %d features for one launch", a.H * a.D);
  if (fits(V)) launch_rotary_as<TT, V>(a, inter, st);
  else if (fits(V / 2)) launch_rotary_as<TT, V / 2>(a, inter, st);
  else launch_rotary_as<TT, 1>(a, inter, st);
  return check_launch("rotary_axes");
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_rotary_axes(const void* x, int dtype, const int64_t* x_strides, int B, int L,
                                int H, int D, const void* positions, int positions_int64,
                                const int64_t* position_strides, const float* inv_freq,
                                const int* sections, int axes, int interleaved, int inverse,
                                void* out, void* stream) {
  const char* what = "uttt_rotary_axes";
  UTTT_REQUIRE(B >= 0 && L >= 0 && H >= 0 && D >= 0, "%s: bad sizes B=%d L=%d H=%d D=%d", what, B, L, H, D);
  UTTT_REQUIRE(axes >= 1 && axes <= kMaxAxes && sections, "%s: %d axes, 1 to %d are built", what, axes,
               kMaxAxes);
  UTTT_REQUIRE(dtype_bytes(dtype) != 0, "%s: dtype code %d", what, dtype);
  RotArgs a{};
  int64_t R = 0;
  for (int i = 0; i < axes; ++i) {
    UTTT_REQUIRE(sections[i] >= 0, "%s: section %d", what, sections[i]);
    R += sections[i];
    UTTT_REQUIRE(R <= kRotPairs, "%s: more than %d pairs", what, kRotPairs);
    a.ends[i] = (int)R;
  }
  UTTT_REQUIRE(R >= 1 && 2 * R <= D, "%s: %lld pairs in %d features", what, (long long)R, D);
  UTTT_REQUIRE((int64_t)B * L < (1LL << 31) && (int64_t)H * D < (1LL << 24), "%s: too many tokens or features",
               what);
  if (B == 0 || L == 0 || H == 0) return UTTT_OK;
  UTTT_REQUIRE(x && x_strides && positions && position_strides && inv_freq && out, "%s: null pointer", what);
  a.x = x;
  a.x_sb = x_strides[0]; a.x_sl = x_strides[1]; a.x_sh = x_strides[2];
  a.pos = positions;
  a.pos64 = positions_int64;
  a.p_sb = position_strides[0]; a.p_sl = position_strides[1]; a.p_sa = position_strides[2];
  a.freq = inv_freq;
  a.axes = axes; a.B = B; a.L = L; a.H = H; a.D = D; a.R = (int)R;
  a.sign = inverse ? -1.0f : 1.0f;
  a.y = out;
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return launch_rotary<TT>(a, interleaved != 0, as_stream(stream)));
  return UTTT_OK;
}
