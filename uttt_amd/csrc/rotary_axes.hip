// Rotary embedding over several position axes for gfx950.
//
// Pair j of a head's features (R = sum of the sections; pairs (j, j + R), or
// (2j, 2j + 1) interleaved) turns by position[axis(j)] * inv_freq[j]; features
// from 2R on pass through.  The backward is the turn by the negative angle.
//
// Bound by memory: one read and one write of x.  A token's R cosines and sines
// are computed once, in LDS, for all its heads; the angle in turns is reduced
// in 64 bits, so that positions of any size keep fp32's precision.
#include "common.h"

namespace uttt {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxAxes = 8;
constexpr int kRotPairs = 2048;   // cosines and sines of a workgroup's tokens, 16 KiB

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

template <class TT, int V, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotary_axes_kernel(RotArgs a) {
  using S = typename TT::S;
  __shared__ float cs[kRotPairs], sn[kRotPairs];
  const int64_t first = (int64_t)blockIdx.x * a.tokens, all = (int64_t)a.B * a.L;
  const int nt = (int)min((int64_t)a.tokens, all - first);
  for (int i = threadIdx.x; i < nt * a.R; i += kRotThreads) {
    const int t = i / a.R, j = i - t * a.R;
    int axis = 0;
    while (j >= a.ends[axis]) ++axis;
    const int64_t b = (first + t) / a.L, l = (first + t) - b * a.L;
    const int64_t at = b * a.p_sb + l * a.p_sl + axis * a.p_sa;
    const double p = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at]
                             : (double)static_cast<const int32_t*>(a.pos)[at];
    double half = p * (double)a.freq[j] * 0.31830988618379067154;   // angle / pi
    half -= 2.0 * rint(0.5 * half);
    float s, c;
    sincospif((float)half, &s, &c);
    cs[i] = c;
    sn[i] = a.sign * s;
  }
  __syncthreads();
  // rotated pieces, V pairs each, then the features that pass through
  const int rp = a.R / V, rest = (a.D - 2 * a.R) / V, per = rp + rest;
  const int n = nt * a.H * per;
  for (int i = threadIdx.x; i < n; i += kRotThreads) {
    const int th = i / per, e = i - th * per, t = th / a.H, h = th - t * a.H;
    const int64_t b = (first + t) / a.L, l = (first + t) - b * a.L;
    const S* x = static_cast<const S*>(a.x) + b * a.x_sb + l * a.x_sl + h * a.x_sh;
    S* y = static_cast<S*>(a.y) + ((first + t) * a.H + h) * a.D;
    float u[V], w[V], c[V], s[V];
    if (e >= rp) {
      const int f = 2 * a.R + (e - rp) * V;
      Vec<TT, V>::load(x + f, u);
      Vec<TT, V>::store(y + f, u);
      continue;
    }
    const int j = e * V;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      c[k] = cs[t * a.R + j + k];
      s[k] = sn[t * a.R + j + k];
    }
    if constexpr (INTER) {
      float p[2 * V];
      Vec<TT, 2 * V>::load(x + 2 * j, p);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float m = p[2 * k], o = p[2 * k + 1];
        p[2 * k] = m * c[k] - o * s[k];
        p[2 * k + 1] = m * s[k] + o * c[k];
      }
      Vec<TT, 2 * V>::store(y + 2 * j, p);
    } else {
      Vec<TT, V>::load(x + j, u);
      Vec<TT, V>::load(x + a.R + j, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float m = u[k], o = w[k];
        u[k] = m * c[k] - o * s[k];
        w[k] = m * s[k] + o * c[k];
      }
      Vec<TT, V>::store(y + j, u);
      Vec<TT, V>::store(y + a.R + j, w);
    }
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
  const int size = sizeof(typename TT::S);
  const auto fits = [&](int v) {   // v pairs at a time, whole aligned pieces throughout
    const int bytes = v * size > 16 ? 16 : v * size;
    return a.R % v == 0 && a.D % v == 0 && (a.D * size) % bytes == 0 && (a.x_sb * size) % bytes == 0 &&
           (a.x_sl * size) % bytes == 0 && (a.x_sh * size) % bytes == 0 &&
           (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % bytes == 0;
  };
  // about four pieces a thread, and cosines that fit
  const int64_t pieces = (int64_t)a.H * a.D / (2 * V);
  int64_t tokens = pieces ? (4 * kRotThreads) / pieces : 1;
  tokens = tokens < 1 ? 1 : tokens;
  if (tokens > kRotPairs / a.R) tokens = kRotPairs / a.R;
  const int64_t all = (int64_t)a.B * a.L;
  if (all / tokens < 1024) tokens = (all + 1023) / 1024 < tokens ? (all + 1023) / 1024 : tokens;
  a.tokens = (int)tokens;
  if (inter ? a.R % (V / 2) == 0 && fits(V / 2) && a.D % (V / 2) == 0 && a.D * size % 16 == 0 &&
                  a.x_sb * size % 16 == 0 && a.x_sl * size % 16 == 0 && a.x_sh * size % 16 == 0 &&
                  (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % 16 == 0
            : fits(V)) {
    if (inter) launch_rotary_as<TT, V / 2>(a, true, st);
    else launch_rotary_as<TT, V>(a, false, st);
  } else {
    launch_rotary_as<TT, 1>(a, inter, st);
  }
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
