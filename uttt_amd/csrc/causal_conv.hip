// The short causal convolution per channel for gfx950, over sequences with its
// backward and token by token:
//   p_t = b + sum_k w[k] x_{t-W+1+k},  y_t = p_t or p_t sigmoid(p_t)
// where the W - 1 inputs before a sequence's first one are its initial state.
// With dp_t = dy_t act'(p_t): dx_t = sum_k w[k] dp_{t+W-1-k}, dw[k] = sum_t dp_t
// x_{t-W+1+k}, db = sum_t dp_t, and the initial state's gradient is dx before the
// first token.
//
// Bound by memory: the forward reads x and writes y, the backward reads x and
// dy and writes dx.  A thread walks over a run of tokens with four channels (one
// where rows do not allow it), its window of W inputs in registers, the loads of
// several tokens ahead of their use; the W - 1 tokens around a run are read
// twice, from cache.  The backward computes p again and keeps the W unfinished
// dx in registers too.  16 x 2048 tokens of 1536 channels, W = 4, bf16, silu:
// forward 49 us (200 MB, 4.1 TB/s), backward 80 (300 MB, 3.8 TB/s), where 36
// vector instructions an element take 77 % of the CUs' time beside the memory, and
// the sums over the workgroups 4; with eight channels a thread, half the waves, 87
// and 142.
#include "rows.h"
#include "state_space.h"

namespace uttt {
namespace ssm {
namespace {

constexpr int kConvThreads = 256;
constexpr int kMinWidth = 2, kMaxWidth = 8;

struct ConvArgs {
  Seqs seqs;
  int D, R, nruns, nvec;
  const void* x;
  int64_t x_sb, x_st;
  const void *w, *b, *h0;   // [D, W], [D] or null, [nseq, W - 1, D] or null
  int w_dtype, b_dtype, act;
  void *y, *hT;             // [B, T, D]; [nseq, W - 1, D] or null
  // backward
  const void *dy, *dhT;
  int64_t dy_sb, dy_st;
  void *dx, *dh0;
  float *part_w, *part_b;   // [blocks, D, W], [blocks, D] or null
};

template <class TT, int V>
struct Piece {
  typename TT::S v[V];
  __device__ __forceinline__ void load(const typename TT::S* p) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, sizeof v), sizeof v);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const { return TT::load(v[i]); }
};

// Zeros for the tokens of no sequence, `first` of kLooseRuns places: one thread
// writes every eighth one's channels in turn (2000 tokens of 1536 channels in a
// buffer of 16 384: 629 us, the full buffer 29).
template <class TT, int V>
__device__ __forceinline__ void zero_loose(const Seqs& s, void* out, int D, int d, int first) {
  const float none[V] = {};
  for (int i = first;; i += kLooseRuns) {
    const int t = loose_token(s, i);
    if (t < 0) return;
    store_piece<TT, V>(static_cast<typename TT::S*>(out) + (int64_t)t * D + d, none);
  }
}

template <int W, int V>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int d, float (&w)[W][V], float (&b)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][i] = load_any(a.w, a.w_dtype, (int64_t)(d + i) * W + k);
    b[i] = a.b ? load_any(a.b, a.b_dtype, d + i) : 0.0f;
  }
}
// The inputs before token t0 of a sequence, the oldest first.
template <class TT, int W, int V>
__device__ __forceinline__ void load_window(const ConvArgs& a, const Run& r, int t0, const typename TT::S* xp, int d,
                                            float (&win)[W][V]) {
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    const int t = t0 - (W - 1) + k;
    Piece<TT, V> v;
    v.zero();
    if (t >= 0) v.load(xp + (int64_t)t * a.x_st);
    else if (a.h0) v.load(static_cast<const typename TT::S*>(a.h0) + ((int64_t)r.seq * (W - 1) + t + W - 1) * a.D + d);
#pragma unroll
    for (int i = 0; i < V; ++i) win[k][i] = v.get(i);
  }
}
template <int W, int V>
__device__ __forceinline__ void push(float (&win)[W][V]) {
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
}

template <class TT, int W, int V>
__global__ __launch_bounds__(kConvThreads) void conv_fwd_kernel(ConvArgs a) {
  using S = typename TT::S;
  constexpr int U = 8;   // tokens that are loaded ahead
  const uint32_t id = blockIdx.x * kConvThreads + threadIdx.x;
  const int at = id / (uint32_t)a.nvec, d = (int)(id % (uint32_t)a.nvec) * V;
  if (at >= a.nruns) {
    if (a.seqs.cu && at < a.nruns + kLooseRuns) zero_loose<TT, V>(a.seqs, a.y, a.D, d, at - a.nruns);
    return;
  }
  const Run r = run_of(a.seqs, at, a.R);
  if (r.seq < 0) return;
  const int t0 = r.c * a.R, n = min(a.R, r.len - t0);
  const S* xp = static_cast<const S*>(a.x) + r.b * a.x_sb + r.tok0 * a.x_st + d;
  S* yp = static_cast<S*>(a.y) + ((int64_t)r.b * a.seqs.T + r.tok0 + t0) * a.D + d;
  float w[W][V], b[V], win[W][V];
  load_weights<W, V>(a, d, w, b);
  load_window<TT, W, V>(a, r, t0, xp, d, win);
  xp += (int64_t)t0 * a.x_st;
  auto token = [&](const Piece<TT, V>& x) {
    float p[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      win[W - 1][i] = x.get(i);
      p[i] = b[i];
#pragma unroll
      for (int k = 0; k < W; ++k) p[i] = __builtin_fmaf(w[k][i], win[k][i], p[i]);
    }
    if (a.act)
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] *= sigmoid_for<TT>(p[i]);
    store_piece<TT, V>(yp, p);
    yp += a.D;
    push<W, V>(win);
  };
  Piece<TT, V> next[U];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next[u].load(xp);
      xp += a.x_st;
    }
  };
  if (n >= U) load();
  int t = 0;
#pragma unroll 1
  for (; t + U <= n; t += U) {
    Piece<TT, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = next[u];
    if (t + 2 * U <= n) load();
#pragma unroll
    for (int u = 0; u < U; ++u) token(x[u]);
  }
#pragma unroll 1
  for (; t < n; ++t) {
    Piece<TT, V> x;
    x.load(xp);
    xp += a.x_st;
    token(x);
  }
  if (a.hT && t0 + n >= r.len)
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      store_piece<TT, V>(static_cast<S*>(a.hT) + ((int64_t)r.seq * (W - 1) + k) * a.D + d, win[k]);
}

// A workgroup: 32 pieces of channels by 8 runs, whose sums for dw and db it
// adds, run by run.
constexpr int kBwdPieces = 32, kBwdRuns = kConvThreads / kBwdPieces;

template <class TT, int W, int V>
__global__ __launch_bounds__(kConvThreads) void conv_bwd_kernel(ConvArgs a) {
  using S = typename TT::S;
  constexpr int U = 4;   // tokens that are loaded ahead
  __shared__ float red[kBwdRuns][kBwdPieces * V];
  const int nvb = (a.nvec + kBwdPieces - 1) / kBwdPieces;
  const int blk = blockIdx.x / nvb;
  const int vec = (int)(blockIdx.x % nvb) * kBwdPieces + threadIdx.x % kBwdPieces, d = vec * V;
  const int slot = threadIdx.x / kBwdPieces, at = blk * kBwdRuns + slot;
  float dw[W][V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][i] = 0.0f;
  }
  Run r;
  r.seq = -1;
  if (vec < a.nvec) {
    if (at < a.nruns) r = run_of(a.seqs, at, a.R);
    else if (a.seqs.cu && at < a.nruns + kLooseRuns) zero_loose<TT, V>(a.seqs, a.dx, a.D, d, at - a.nruns);
  }
  if (r.seq >= 0) {
    const int t0 = r.c * a.R, t1 = min(t0 + a.R, r.len);
    const S* xp = static_cast<const S*>(a.x) + r.b * a.x_sb + r.tok0 * a.x_st + d;
    const S* gp = static_cast<const S*>(a.dy) + r.b * a.dy_sb + r.tok0 * a.dy_st + d;
    S* op = static_cast<S*>(a.dx) + ((int64_t)r.b * a.seqs.T + r.tok0) * a.D + d;
    float w[W][V], b[V], win[W][V], acc[W][V];
    load_weights<W, V>(a, d, w, b);
    load_window<TT, W, V>(a, r, t0, xp, d, win);
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][i] = 0.0f;
    // Token t: of the run itself (own) or behind it, in which case it only ends
    // the dx of the run's last tokens; behind the sequence's end there is none.
    auto token = [&](const Piece<TT, V>& x, const Piece<TT, V>& g, bool own) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        win[W - 1][i] = x.get(i);
        float dp = g.get(i);
        if (a.act) {
          float p = b[i];
#pragma unroll
          for (int k = 0; k < W; ++k) p = __builtin_fmaf(w[k][i], win[k][i], p);
          const float s = sigmoid_for<TT>(p);
          dp *= s * __builtin_fmaf(p, 1.0f - s, 1.0f);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k][i] = __builtin_fmaf(w[k][i], dp, acc[k][i]);
        if (own) {
          db[i] += dp;
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k][i] = __builtin_fmaf(dp, win[k][i], dw[k][i]);
        }
      }
    };
    auto step = [&]() {
      push<W, V>(win);
      push<W, V>(acc);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[W - 1][i] = 0.0f;
    };
    // with what the final state adds, and positions before the first token
    auto checked = [&](int t) {
      if (t < r.len) {
        Piece<TT, V> x, g;
        x.load(xp + (int64_t)t * a.x_st);
        g.load(gp + (int64_t)t * a.dy_st);
        token(x, g, t < t1);
      }
      const int done = t - (W - 1), kept = done - (r.len - (W - 1));   // whose dx ends here; its place in the final state
      if (done >= t0 || (done < 0 && t0 == 0)) {
        if (a.dhT && kept >= 0) {
          Piece<TT, V> e;
          e.load(static_cast<const S*>(a.dhT) + ((int64_t)r.seq * (W - 1) + kept) * a.D + d);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[0][i] += e.get(i);
        }
        if (done >= 0) store_piece<TT, V>(op + (int64_t)done * a.D, acc[0]);
        else if (a.dh0)
          store_piece<TT, V>(static_cast<S*>(a.dh0) + ((int64_t)r.seq * (W - 1) + done + W - 1) * a.D + d, acc[0]);
      }
      step();
    };
    const int end = t1 + W - 1;   // the last token of the run is done with the W - 1 behind it
    int t = t0;
#pragma unroll 1
    for (; t < end && t < t0 + W - 1; ++t) checked(t);
    // from here to the run's last token one position ends with each, before the final state
    Piece<TT, V> nx[U], ng[U];
    auto load = [&](int t) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        nx[u].load(xp + (int64_t)(t + u) * a.x_st);
        ng[u].load(gp + (int64_t)(t + u) * a.dy_st);
      }
    };
    if (t + U <= t1) load(t);
#pragma unroll 1
    for (; t + U <= t1; t += U) {
      Piece<TT, V> x[U], g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = nx[u];
        g[u] = ng[u];
      }
      if (t + 2 * U <= t1) load(t + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        token(x[u], g[u], true);
        store_piece<TT, V>(op + (int64_t)(t + u - (W - 1)) * a.D, acc[0]);
        step();
      }
    }
#pragma unroll 1
    for (; t < end; ++t) checked(t);
  }
  if (!a.part_w && !a.part_b) return;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) red[slot][threadIdx.x % kBwdPieces * V + i] = k < W ? dw[k < W ? k : 0][i] : db[i];
    __syncthreads();
    if (threadIdx.x >= kBwdPieces * V) continue;
    const int e = (int)(blockIdx.x % nvb) * kBwdPieces * V + threadIdx.x;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < kBwdRuns; ++s) sum += red[s][threadIdx.x];
    if (e >= a.D) continue;
    if (k < W) {
      if (a.part_w) a.part_w[((int64_t)blk * a.D + e) * W + k] = sum;
    } else if (a.part_b) {
      a.part_b[(int64_t)blk * a.D + e] = sum;
    }
  }
}

// ------------------------------------------------------------ by tokens ----
struct ConvStepArgs {
  const void* x;
  int64_t x_sb, x_st;
  const void *w, *b;
  int w_dtype, b_dtype, act, B, T, D, slots;
  void* state;             // [slots, W - 1, D], slots s_slot apart
  int64_t s_slot;
  const void* idx;
  int idx64;
  void* y;                 // [B, T, D]
};

template <class TT, int W>
__global__ __launch_bounds__(kConvThreads) void conv_step_kernel(ConvStepArgs a) {
  using S = typename TT::S;
  const int ncb = (a.D + kConvThreads - 1) / kConvThreads;
  const int d = (int)(blockIdx.x % ncb) * kConvThreads + threadIdx.x;
  Rows rows{a.idx, a.idx64, a.B, a.slots};
  int b = blockIdx.x / ncb;
  const int64_t slot = rows.slot_of(b);
  const bool live = d < a.D;
  if (slot < 0) {   // a padded row: zeros, no state
    if (live)
      for (int t = 0; t < a.T; ++t) static_cast<S*>(a.y)[((int64_t)b * a.T + t) * a.D + d] = TT::store(0.0f);
    return;
  }
  S* sp = static_cast<S*>(a.state) + slot * a.s_slot + d;
  float win[W] = {}, w[W] = {}, bias = 0.0f;
  if (live) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k] = TT::load(sp[(int64_t)k * a.D]);
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = load_any(a.w, a.w_dtype, (int64_t)d * W + k);
    if (a.b) bias = load_any(a.b, a.b_dtype, d);
  }
  const int others = rows.others<kConvThreads>(b, slot);
  if (others & 1) return;   // an earlier row's workgroup takes this one up
  for (;;) {
    if (live)
      for (int t = 0; t < a.T; ++t) {
        win[W - 1] = TT::load(static_cast<const S*>(a.x)[b * a.x_sb + t * a.x_st + d]);
        float p = bias;
#pragma unroll
        for (int k = 0; k < W; ++k) p = __builtin_fmaf(w[k], win[k], p);
        if (a.act) p *= sigmoid(p);
        static_cast<S*>(a.y)[((int64_t)b * a.T + t) * a.D + d] = TT::store(p);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) win[k] = win[k + 1];
      }
    if (!(others & 2)) break;
    b = rows.next_of<kConvThreads>(b, slot);
    if (b >= a.B) break;
  }
  if (live)
#pragma unroll
    for (int k = 0; k < W - 1; ++k) sp[(int64_t)k * a.D] = TT::store(win[k]);
}

// --------------------------------------------------------------- launches --
#define UTTT_WIDTH_SWITCH(W, WW, ...)                       \
  switch (W) {                                              \
    case 2: { constexpr int WW = 2; __VA_ARGS__; } break;   \
    case 3: { constexpr int WW = 3; __VA_ARGS__; } break;   \
    case 4: { constexpr int WW = 4; __VA_ARGS__; } break;   \
    case 5: { constexpr int WW = 5; __VA_ARGS__; } break;   \
    case 6: { constexpr int WW = 6; __VA_ARGS__; } break;   \
    case 7: { constexpr int WW = 7; __VA_ARGS__; } break;   \
    default: { constexpr int WW = 8; __VA_ARGS__; } break;  \
  }

// Whether rows hold whole pieces of four elements.
bool whole_pieces(const ConvArgs& a, int size) {
  uintptr_t all = 0;
  for (const void* p : {a.x, (const void*)a.y, a.h0, (const void*)a.hT, a.dy, (const void*)a.dx, a.dhT, (const void*)a.dh0})
    all |= reinterpret_cast<uintptr_t>(p);
  const int64_t rows = a.D | a.x_sb | a.x_st | a.dy_sb | a.dy_st;
  return ((all | (uintptr_t)(rows * size)) & (uintptr_t)(4 * size - 1)) == 0;
}

int64_t fwd_threads(const ConvArgs& a) {
  return ((int64_t)a.nruns + (a.seqs.cu ? kLooseRuns : 0)) * a.nvec;
}
int64_t bwd_run_blocks(const Seqs& s, int R) {
  return (run_count(s, R) + (s.cu ? kLooseRuns : 0) + kBwdRuns - 1) / kBwdRuns;
}
constexpr int kBwdRun = 32;   // tokens of a backward's run

template <class TT, int V>
int launch_conv(ConvArgs a, int W, bool bwd, hipStream_t st) {
  a.nvec = (a.D + V - 1) / V;
  if (!bwd) {
    // 32 tokens a run where that makes work enough, so that the window is read
    // again seldom
    a.R = run_count(a.seqs, 32) * a.nvec >= 1 << 17 ? 32 : 8;
    a.nruns = (int)run_count(a.seqs, a.R);
    const int64_t n = fwd_threads(a);
    UTTT_REQUIRE(run_count(a.seqs, a.R) < (1 << 30) && n < (1LL << 31), "causal_conv: too many tokens and channels");
    UTTT_WIDTH_SWITCH(W, WW,
                      hipLaunchKernelGGL((conv_fwd_kernel<TT, WW, V>), dim3((unsigned)((n + kConvThreads - 1) / kConvThreads)),
                                         dim3(kConvThreads), 0, st, a));
    return check_launch("causal_conv");
  }
  a.R = kBwdRun;
  a.nruns = (int)run_count(a.seqs, a.R);
  const int64_t blocks = bwd_run_blocks(a.seqs, a.R) * ((a.nvec + kBwdPieces - 1) / kBwdPieces);
  UTTT_REQUIRE(run_count(a.seqs, a.R) < (1 << 30) && blocks < (1LL << 24), "causal_conv: too many tokens and channels");
  UTTT_WIDTH_SWITCH(W, WW, hipLaunchKernelGGL((conv_bwd_kernel<TT, WW, V>), dim3((unsigned)blocks), dim3(kConvThreads), 0,
                                              st, a));
  return check_launch("causal_conv_bwd");
}

template <class TT>
int conv_any(const ConvArgs& a, int W, bool bwd, hipStream_t st) {
  return whole_pieces(a, sizeof(typename TT::S)) ? launch_conv<TT, 4>(a, W, bwd, st) : launch_conv<TT, 1>(a, W, bwd, st);
}

int conv_check(const ConvArgs& a, int W, int dtype, const char* what) {
  UTTT_REQUIRE(seqs_ok(a.seqs) && a.seqs.T < (1 << 30) && a.seqs.nseq < (1 << 30), "%s: bad sizes B=%d T=%d nseq=%d",
               what, a.seqs.B, a.seqs.T, a.seqs.nseq);
  UTTT_REQUIRE(a.D >= 1 && a.D < (1 << 28), "%s: D=%d", what, a.D);
  UTTT_REQUIRE(W >= kMinWidth && W <= kMaxWidth, "%s: W=%d must be %d to %d", what, W, kMinWidth, kMaxWidth);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(a.w_dtype) && dtype_bytes(a.b_dtype), "%s: dtype codes %d, %d, %d",
               what, dtype, a.w_dtype, a.b_dtype);
  UTTT_REQUIRE(a.w && (a.x || a.seqs.T == 0), "%s: null pointer", what);
  return UTTT_OK;
}

}  // namespace
}  // namespace ssm
}  // namespace uttt

using namespace uttt;
using namespace uttt::ssm;

extern "C" int uttt_causal_conv_fwd(const void* x, const int64_t* x_strides, int dtype, const void* weight,
                                    int weight_dtype, const void* bias, int bias_dtype, int silu,
                                    const void* initial_state, const void* cu_seqlens, int cu_is_int64, int B, int T,
                                    int nseq, int D, int W, void* out, void* final_state, void* stream) {
  const char* what = "uttt_causal_conv_fwd";
  ConvArgs a{};
  a.seqs = Seqs{cu_seqlens, cu_is_int64, B, T, nseq};
  a.D = D; a.x = x; a.w = weight; a.b = bias; a.h0 = initial_state;
  a.w_dtype = weight_dtype; a.b_dtype = bias_dtype; a.act = silu;
  a.y = out; a.hT = final_state;
  if (const int rc = conv_check(a, W, dtype, what)) return rc;
  UTTT_REQUIRE(x_strides && (out || T == 0), "%s: null pointer", what);
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return conv_any<TT>(a, W, false, as_stream(stream)));
  return UTTT_OK;
}

extern "C" size_t uttt_causal_conv_bwd_workspace_bytes(int B, int T, int nseq, int packed, int D, int W) {
  const Seqs s{packed ? uttt_last_error() : nullptr, 0, B, T, nseq};   // a stand-in, not read
  if (!seqs_ok(s) || D < 1 || W < kMinWidth || W > kMaxWidth) return 0;
  return (size_t)bwd_run_blocks(s, kBwdRun) * D * (W + 1) * 4;
}

extern "C" int uttt_causal_conv_bwd(const void* x, const int64_t* x_strides, int dtype, const void* weight,
                                    int weight_dtype, const void* bias, int bias_dtype, int silu,
                                    const void* initial_state, const void* cu_seqlens, int cu_is_int64, int B, int T,
                                    int nseq, int D, int W, const void* dout, const int64_t* dout_strides,
                                    const void* dfinal_state, void* dx, void* dweight, void* dbias,
                                    void* dinitial_state, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "uttt_causal_conv_bwd";
  ConvArgs a{};
  a.seqs = Seqs{cu_seqlens, cu_is_int64, B, T, nseq};
  a.D = D; a.x = x; a.w = weight; a.b = bias; a.h0 = initial_state;
  a.w_dtype = weight_dtype; a.b_dtype = bias_dtype; a.act = silu;
  a.dy = dout; a.dhT = dfinal_state; a.dx = dx; a.dh0 = dinitial_state;
  if (const int rc = conv_check(a, W, dtype, what)) return rc;
  UTTT_REQUIRE(x_strides && dout_strides && (T == 0 || (dout && dx)), "%s: null pointer", what);
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  a.dy_sb = dout_strides[0]; a.dy_st = dout_strides[1];
  const size_t need = uttt_causal_conv_bwd_workspace_bytes(B, T, nseq, cu_seqlens != nullptr, D, W);
  UTTT_REQUIRE((!dweight && !dbias) || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, %zu needed",
               what, workspace_bytes, need);
  const int64_t blocks = bwd_run_blocks(a.seqs, kBwdRun);
  float* w = static_cast<float*>(workspace);
  a.part_w = dweight ? w : nullptr;
  a.part_b = dbias ? w + (size_t)blocks * D * W : nullptr;
  const hipStream_t st = as_stream(stream);
  int rc = UTTT_OK;
  switch (dtype) {
    case UTTT_F32: rc = conv_any<F32T>(a, W, true, st); break;
    case UTTT_BF16: rc = conv_any<BF16T>(a, W, true, st); break;
    default: rc = conv_any<F16T>(a, W, true, st); break;
  }
  if (rc) return rc;
  return launch_sums(blocks, {{a.part_w, (int64_t)D * W, dweight, weight_dtype}, {a.part_b, D, dbias, bias_dtype}}, st, what);
}

extern "C" int uttt_causal_conv_step(const void* x, const int64_t* x_strides, int dtype, const void* weight,
                                     int weight_dtype, const void* bias, int bias_dtype, int silu, int B, int T, int D,
                                     int W, void* state, int64_t state_stride, int slots, const void* indices,
                                     int indices_int64, void* out, void* stream) {
  const char* what = "uttt_causal_conv_step";
  UTTT_REQUIRE(B >= 0 && T >= 0 && D >= 1 && slots >= 0, "%s: bad sizes B=%d T=%d D=%d slots=%d", what, B, T, D, slots);
  UTTT_REQUIRE(W >= kMinWidth && W <= kMaxWidth, "%s: W=%d must be %d to %d", what, W, kMinWidth, kMaxWidth);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(weight_dtype) && dtype_bytes(bias_dtype), "%s: dtype codes %d, %d, %d",
               what, dtype, weight_dtype, bias_dtype);
  UTTT_REQUIRE(indices || B <= slots, "%s: %d rows without indices, %d slots", what, B, slots);
  const int64_t blocks = (int64_t)B * ((D + kConvThreads - 1) / kConvThreads);
  UTTT_REQUIRE(blocks < (1LL << 24), "%s: too many rows and channels", what);
  if (B == 0 || T == 0) return UTTT_OK;
  UTTT_REQUIRE(x && x_strides && weight && out && (state || slots == 0), "%s: null pointer", what);
  UTTT_REQUIRE(state_stride >= (int64_t)(W - 1) * D, "%s: states %lld elements apart", what, (long long)state_stride);
  const ConvStepArgs a{x, x_strides[0], x_strides[1], weight, bias, weight_dtype, bias_dtype, silu, B, T, D, slots,
                       state, state_stride, indices, indices_int64, out};
  const hipStream_t st = as_stream(stream);
  UTTT_DTYPE_SWITCH_LR(dtype, TT, UTTT_WIDTH_SWITCH(W, WW,
      hipLaunchKernelGGL((conv_step_kernel<TT, WW>), dim3((unsigned)blocks), dim3(kConvThreads), 0, st, a)));
  return check_launch(what);
}
