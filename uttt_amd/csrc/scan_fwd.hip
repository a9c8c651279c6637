// The selective state space scan over sequences for gfx950 (formulas and
// layout: scan.h).
//
// Along one sequence the recurrence is a chain, so sequences are cut into runs
// that are worked on side by side: what a run adds to a state of zeros and the
// sum of its steps (local pass), the runs joined, h' = e^{A sum dt} h + end
// (one thread a state), and the runs again from the states they start with.
#include "scan.h"

namespace uttt {
namespace ssm {
namespace {

template <class TT, int LN, bool LOCAL>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanArgs a) {
  using S = typename TT::S;
  using M = Geo<LN>;
  constexpr int CS = M::CS, CB = M::CB, NP = M::NP, EPT = M::EPT, BPT = M::BPT;
  __shared__ float sU[kTile][CB], sDt[kTile][CB], sY[LOCAL ? 1 : kTile][CB];
  __shared__ float4 sB[kTile][LN], sC[LOCAL ? 1 : kTile][LN];
  const int tid = threadIdx.x;
  const int c = tid % CB, tq = tid / CB;   // the element column that this thread loads and stores
  Place p;
  if (!p.init(a, CB)) {
    // the workgroups past the last run: zeros for the tokens of no sequence
    if (!LOCAL && a.seqs.cu && (int)(blockIdx.x / (a.G * a.ncb)) >= a.nruns && c < p.nc)
      for (int i = tq;; i += M::TPP) {
        const int t = loose_token(a.seqs, i);
        if (t < 0) break;
        static_cast<S*>(a.out)[(int64_t)t * a.D + p.d0 + c] = TT::store(0.0f);
      }
    return;
  }
  if (LOCAL && p.t0 + p.n >= p.run.len) return;   // nothing follows it
  const int at = p.run.base + p.run.c;
  const int64_t tok = p.run.tok0 + p.t0;
  const bool live = c < p.nc;
  const S* xp = static_cast<const S*>(a.x) + p.run.b * a.x_sb + tok * a.x_st + p.d0 + c;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + tok * a.z_st + p.d0 + c;
  const int64_t dt_at = p.run.b * a.dt_sb + tok * a.dt_st + p.d0 + c;
  const S* Bp = static_cast<const S*>(a.Bm) + p.run.b * a.B_sb + tok * a.B_st + p.g * a.B_sg;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + tok * a.C_st + p.g * a.C_sg;
  const float bias = live && a.bias ? a.bias[p.d0 + c] : 0.0f;
  const float skip = !LOCAL && live && a.Dskip ? a.Dskip[p.d0 + c] : 0.0f;
  const bool gate = !LOCAL && a.z != nullptr;

  const int wave = tid >> 6, lane = tid & 63, ln = lane % LN;
  const int ch = wave * M::WC + lane / LN * CS;   // first channel of this lane
  float h[CS][4], A2[CS][4];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const bool on = ch + s < p.nc;
    const int64_t row = p.d0 + ch + s;
    unpack(on ? load_states(a.A + row * a.N, 4 * ln, a.N) : make_float4(0, 0, 0, 0), A2[s]);
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[s][j] = log2_rate(A2[s][j]);
    float4 v = make_float4(0, 0, 0, 0);
    if (!LOCAL && on) {
      if (p.run.c > 0) v = load_states(a.starts + ((int64_t)at * a.D + row) * a.N, 4 * ln, a.N);
      else if (a.h0) v = load_states(a.h0 + ((int64_t)p.run.seq * a.D + row) * a.N, 4 * ln, a.N);
    }
    unpack(v, h[s]);
  }

  S rx[EPT], rz[EPT], rB[BPT], rC[BPT];
  uint32_t rdt[EPT];
  auto load_tile = [&](int tt) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int t = tt + tq + i * M::TPP;
      rx[i] = rz[i] = S(0);
      rdt[i] = 0;
      if (live && t < p.n) {
        rx[i] = xp[(int64_t)t * a.x_st];
        rdt[i] = load_bits(a.dt, a.dt_dtype, dt_at + (int64_t)t * a.dt_st);
        if (gate) rz[i] = zp[(int64_t)t * a.z_st];
      }
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads, t = tt + e / NP, n = e % NP;
      rB[i] = rC[i] = S(0);
      if (e < kTile * NP && t < p.n && n < a.N) {
        rB[i] = Bp[(int64_t)t * a.B_st + n];
        if (!LOCAL) rC[i] = Cp[(int64_t)t * a.C_st + n];
      }
    }
  };
  float sum_dt = 0.0f;
  load_tile(0);
  const int64_t tile0 = a.hs ? first_run(a.seqs, p.run.seq, kTile) + p.t0 / kTile : 0;
  for (int tt = 0; tt < p.n; tt += kTile) {
    float x[EPT], z[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      float dt = 0.0f;
      x[i] = TT::load(rx[i]);
      z[i] = TT::load(rz[i]);
      if (tt + tl < p.n) {
        dt = widen(rdt[i], a.dt_dtype) + bias;
        if (a.soft) dt = softplus(dt);
      }
      sum_dt += dt;
      sDt[tl][c] = dt;
      sU[tl][c] = dt * x[i];
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads;
      if (e < kTile * NP) {
        reinterpret_cast<float*>(sB)[e] = TT::load(rB[i]);
        if (!LOCAL) reinterpret_cast<float*>(sC)[e] = TT::load(rC[i]);
      }
    }
    __syncthreads();
    if (tt + kTile < p.n) load_tile(tt + kTile);
    if (!LOCAL && a.hs) {
#pragma unroll
      for (int s = 0; s < CS; ++s)
        if (ch + s < p.nc)
          store_states(a.hs + ((tile0 + tt / kTile) * a.D + p.d0 + ch + s) * a.N, 4 * ln, a.N,
                       make_float4(h[s][0], h[s][1], h[s][2], h[s][3]));
    }
#pragma unroll
    for (int t = 0; t < kTile; ++t) {
      float b[4], cc[4];
      unpack(sB[t][ln], b);
      if (!LOCAL) unpack(sC[t][ln], cc);
#pragma unroll
      for (int s = 0; s < CS; ++s) {
        const float dt = sDt[t][ch + s], u = sU[t][ch + s];
        float y = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[s][j] = __builtin_fmaf(exp2_hw(dt * A2[s][j]), h[s][j], u * b[j]);
          if (!LOCAL) y = __builtin_fmaf(cc[j], h[s][j], y);
        }
        if (!LOCAL) {
          y = sum_lanes<LN>(y);
          if (ln == 0) sY[t][ch + s] = y;
        }
      }
    }
    __syncthreads();
    if (LOCAL) continue;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      if (!live || tt + tl >= p.n) continue;
      float y = __builtin_fmaf(skip, x[i], sY[tl][c]);
      if (gate) y *= z[i] * sigmoid(z[i]);
      static_cast<S*>(a.out)[((int64_t)p.run.b * a.seqs.T + tok + tt + tl) * a.D + p.d0 + c] = TT::store(y);
    }
  }
  float* to = LOCAL ? a.ends + (int64_t)at * a.D * a.N
              : a.hT && p.t0 + p.n >= p.run.len ? a.hT + (int64_t)p.run.seq * a.D * a.N : nullptr;
  if (to)
#pragma unroll
    for (int s = 0; s < CS; ++s)
      if (ch + s < p.nc)
        store_states(to + (int64_t)(p.d0 + ch + s) * a.N, 4 * ln, a.N,
                     make_float4(h[s][0], h[s][1], h[s][2], h[s][3]));
  if (LOCAL) {
    float* red = &sU[0][0];   // the last tile is read
    red[tid] = sum_dt;
    __syncthreads();
    if (tq == 0 && live) {
#pragma unroll
      for (int i = 1; i < M::TPP; ++i) sum_dt += red[c + i * CB];
      a.decay[(int64_t)at * a.D + p.d0 + c] = sum_dt;
    }
  }
}

// The states that a sequence's runs start with, from the second on.
__global__ __launch_bounds__(kScanThreads) void scan_join_kernel(ScanArgs a, const float* __restrict__ ends,
                                                                 const float* __restrict__ decay,
                                                                 float* __restrict__ starts) {
  const int64_t e = (int64_t)blockIdx.x * kScanThreads + threadIdx.x, M = (int64_t)a.D * a.N;
  if (e >= M * a.seqs.nseq) return;
  const int seq = (int)(e / M);
  const int64_t at = e % M, d = at / a.N;
  const Run r = span_of(a.seqs, seq, a.R);
  const int runs = (int)(((int64_t)r.len + a.R - 1) / a.R);
  const float A2 = log2_rate(a.A[at]);
  float h = a.h0 ? a.h0[e] : 0.0f;
#pragma unroll 8
  for (int c = 1; c < runs; ++c) {
    const int64_t i = r.base + c - 1;
    h = __builtin_fmaf(exp2_hw(decay[i * a.D + d] * A2), h, ends[i * M + at]);
    starts[(i + 1) * M + at] = h;
  }
}

template <class TT, int LN>
int launch_fwd_as(const ScanArgs& a, hipStream_t st) {
  const unsigned per = (unsigned)(a.G * a.ncb), blocks = (unsigned)a.nruns * per;
  if (a.ends) {
    hipLaunchKernelGGL((scan_fwd_kernel<TT, LN, true>), dim3(blocks), dim3(kScanThreads), 0, st, a);
    const int64_t states = (int64_t)a.seqs.nseq * a.D * a.N;
    hipLaunchKernelGGL(scan_join_kernel, dim3((unsigned)((states + kScanThreads - 1) / kScanThreads)),
                       dim3(kScanThreads), 0, st, a, a.ends, a.decay, a.starts);
  }
  hipLaunchKernelGGL((scan_fwd_kernel<TT, LN, false>), dim3(blocks + (a.seqs.cu ? per : 0)), dim3(kScanThreads), 0,
                     st, a);
  return check_launch("selective_scan");
}

template <class TT>
int launch_fwd(const ScanArgs& a, hipStream_t st) {
  switch (scan_lanes(a.N)) {
    case 1: return launch_fwd_as<TT, 1>(a, st);
    case 2: return launch_fwd_as<TT, 2>(a, st);
    case 4: return launch_fwd_as<TT, 4>(a, st);
    case 8: return launch_fwd_as<TT, 8>(a, st);
    default: return launch_fwd_as<TT, 16>(a, st);
  }
}

constexpr int kFwdBlocks = 1024;   // workgroups that are wanted at once

}  // namespace

// A sequence that no cut would help is one run.
void scan_runs(ScanArgs& a, int want) {
  a.Dg = a.D / a.G;
  const int cb = scan_width(a.N);
  a.ncb = (a.Dg + cb - 1) / cb;
  const int64_t per = (int64_t)a.G * a.ncb, tokens = (int64_t)a.seqs.B * a.seqs.T;
  const int64_t runs = (want + per - 1) / per;       // wanted over all tokens
  int64_t R = (tokens + runs - 1) / runs;
  if (R < 4 * kTile) R = 4 * kTile;
  if (!a.seqs.cu) {                                  // equal runs
    const int64_t k = R < a.seqs.T ? (a.seqs.T + R - 1) / R : 1;
    R = (a.seqs.T + k - 1) / k;
  }
  if (R > a.seqs.T) R = a.seqs.T;
  R = (R + kTile - 1) / kTile * kTile;
  a.R = (int)(R < kTile ? kTile : R);
  a.nruns = (int)run_count(a.seqs, a.R);
}

int scan_check(const ScanArgs& a, int dtype, const char* what) {
  UTTT_REQUIRE(seqs_ok(a.seqs) && a.seqs.T < (1 << 30) && a.seqs.nseq < (1 << 30),
               "%s: bad sizes B=%d T=%d nseq=%d", what, a.seqs.B, a.seqs.T, a.seqs.nseq);
  UTTT_REQUIRE(a.D >= 1 && a.G >= 1 && a.D % a.G == 0, "%s: D=%d must be a multiple of G=%d", what, a.D, a.G);
  UTTT_REQUIRE(a.N >= 1 && a.N <= kMaxStates, "%s: N=%d must be at most %d", what, a.N, kMaxStates);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(a.dt_dtype), "%s: dtype codes %d, %d", what, dtype, a.dt_dtype);
  const bool empty = a.seqs.T == 0;
  UTTT_REQUIRE(a.A && (empty || (a.x && a.dt && a.Bm && a.Cm)), "%s: null pointer", what);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.h0) |
                         reinterpret_cast<uintptr_t>(a.hT) | reinterpret_cast<uintptr_t>(a.dhT) |
                         reinterpret_cast<uintptr_t>(a.dh0) | reinterpret_cast<uintptr_t>(a.hs);
  UTTT_REQUIRE((rows & 15u) == 0, "%s: A and the states must be 16-byte aligned", what);
  return UTTT_OK;
}

bool scan_fits(const ScanArgs& a) {   // a launch has fewer than 2^32 threads
  const int64_t runs = run_count(a.seqs, a.R), states = (int64_t)a.seqs.nseq * a.D * a.N;
  return runs < (1 << 30) && (runs + 1) * a.G * a.ncb < (1LL << 24) && states < (1LL << 31);
}

namespace {
size_t fwd_bytes(const ScanArgs& a) {
  const bool whole = a.R >= a.seqs.T;
  return whole ? 0 : (size_t)a.nruns * a.D * (2 * (size_t)a.N + 1) * 4;
}
}  // namespace

}  // namespace ssm
}  // namespace uttt

using namespace uttt;
using namespace uttt::ssm;

extern "C" int uttt_selective_scan_tiles(int B, int T, int nseq, int packed) {
  const Seqs s{packed ? uttt_last_error() : nullptr, 0, B, T, nseq};   // a stand-in, not read
  return seqs_ok(s) ? (int)run_count(s, kTile) : 0;
}

extern "C" size_t uttt_selective_scan_fwd_workspace_bytes(int B, int T, int nseq, int packed, int D, int N, int G) {
  ScanArgs a{};
  a.seqs = Seqs{packed ? &a : nullptr, 0, B, T, nseq};
  a.D = D; a.N = N; a.G = G;
  if (!seqs_ok(a.seqs) || D < 1 || G < 1 || D % G || N < 1 || N > kMaxStates) return 0;
  scan_runs(a, kFwdBlocks);
  return fwd_bytes(a);
}

extern "C" int uttt_selective_scan_fwd(const void* x, const int64_t* x_strides, int dtype, const void* dt,
                                       const int64_t* dt_strides, int dt_dtype, const float* A, const void* Bm,
                                       const int64_t* B_strides, const void* Cm, const int64_t* C_strides,
                                       const float* skip, const void* gate, const int64_t* gate_strides,
                                       const float* dt_bias, int dt_softplus, const float* initial_state,
                                       const void* cu_seqlens, int cu_is_int64, int B, int T, int nseq, int D,
                                       int N, int G, void* out, float* final_state, float* tile_states,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "uttt_selective_scan_fwd";
  ScanArgs a{};
  a.seqs = Seqs{cu_seqlens, cu_is_int64, B, T, nseq};
  a.D = D; a.N = N; a.G = G;
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = gate;
  a.dt_dtype = dt_dtype; a.soft = dt_softplus;
  a.A = A; a.Dskip = skip; a.bias = dt_bias; a.h0 = initial_state;
  a.out = out; a.hT = final_state; a.hs = tile_states;
  if (const int rc = scan_check(a, dtype, what)) return rc;
  UTTT_REQUIRE(x_strides && dt_strides && B_strides && C_strides && (gate_strides || !gate) && (out || T == 0),
               "%s: null pointer", what);
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  a.dt_sb = dt_strides[0]; a.dt_st = dt_strides[1];
  a.B_sb = B_strides[0]; a.B_st = B_strides[1]; a.B_sg = B_strides[2];
  a.C_sb = C_strides[0]; a.C_st = C_strides[1]; a.C_sg = C_strides[2];
  if (gate) { a.z_sb = gate_strides[0]; a.z_st = gate_strides[1]; }
  scan_runs(a, kFwdBlocks);
  UTTT_REQUIRE(scan_fits(a), "%s: too many sequences, channels or states", what);
  const size_t need = fwd_bytes(a);
  UTTT_REQUIRE(!need || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, %zu needed", what,
               workspace_bytes, need);
  if (need) {
    UTTT_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned", what);
    a.ends = static_cast<float*>(workspace);
    a.starts = a.ends + (size_t)a.nruns * D * N;
    a.decay = a.starts + (size_t)a.nruns * D * N;
  }
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return launch_fwd<TT>(a, as_stream(stream)));
  return UTTT_OK;
}
