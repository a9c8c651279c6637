// The selective state space scan over sequences for gfx950 (formulas and
// layout: scan.h).
//
// Along one sequence the recurrence is a chain, so sequences are cut into runs
// that are worked on side by side: what a run adds to a state of zeros and the
// sum of its steps (local pass), the runs joined, h' = e^{A sum dt} h + end
// (one thread a state), and the runs again from the states they start with.
//
// A lane has one channel with all its states in registers, so that x, dt, z and y
// go from memory to the lane and back without a detour, steps and gates are
// computed once, and no sum crosses lanes; B and C of 16 tokens are widened into
// LDS a tile ahead and read by all lanes at once.  Bound by vector instructions:
// per state a product, an exponential (as long as two others), three more; some
// 50 for a token's step, gate and conversions, at 16 states 145 in all.  Four
// waves a SIMD issue them nearly without a gap (7 registers are spilled with a gate
// at 9 to 16 states); one alone takes 7 cycles each.
// 16 x 2048 tokens of 1536 channels, 16 states, bf16, gated: local pass 167 us,
// joins 13, outputs with the kept states 233 (600 MB, 2.6 TB/s).  With four lanes
// to a channel and two channels a lane, everything through LDS: 262 and 560 us.
#include <math.h>

#include "scan.h"

namespace uttt {
namespace ssm {
namespace {

template <class TT, class DT, int NP, bool LOCAL, bool GATE>
__global__ __launch_bounds__(kScanThreads, fwd_waves(NP)) void scan_fwd_kernel(ScanArgs a) {
  using S = typename TT::S;
  using SD = typename DT::S;
  __shared__ float4 sB[2][kTile][NP / 4], sC[2][LOCAL ? 1 : kTile][NP / 4];
  const int tid = threadIdx.x;
  Place p;
  if (!p.init(a, kScanThreads)) {
    if (!LOCAL && a.seqs.cu) {   // the workgroups past the last run: zeros for the tokens of no sequence
      const int first = (int)(blockIdx.x / (a.G * a.ncb)) - a.nruns;
      if (first >= 0 && tid < p.nc)
        for (int i = first;; i += kLooseRuns) {
          const int t = loose_token(a.seqs, i);
          if (t < 0) break;
          static_cast<S*>(a.out)[(int64_t)t * a.D + p.d0 + tid] = TT::store(0.0f);
        }
    }
    return;
  }
  if (LOCAL && p.t0 + p.n >= p.run.len) return;   // nothing follows it
  const int at = p.run.base + p.run.c;
  const int64_t tok = p.run.tok0 + p.t0;
  // a lane without a channel does the last one's work again, a wave without any none
  const bool busy = (tid & ~(kWave - 1)) < p.nc;
  const uint32_t c = min(tid, p.nc - 1), d = p.d0 + c;
  const S* xp = static_cast<const S*>(a.x) + p.run.b * a.x_sb + tok * a.x_st + p.d0;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + tok * a.z_st + p.d0;
  const SD* tp = static_cast<const SD*>(a.dt) + p.run.b * a.dt_sb + tok * a.dt_st + p.d0;
  const S* Bp = static_cast<const S*>(a.Bm) + p.run.b * a.B_sb + tok * a.B_st + p.g * a.B_sg;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + tok * a.C_st + p.g * a.C_sg;
  S* yp = static_cast<S*>(a.out) + ((int64_t)p.run.b * a.seqs.T + tok) * a.D + p.d0;
  const float bias = a.bias ? a.bias[d] : 0.0f;
  const float skip = !LOCAL && a.Dskip ? a.Dskip[d] : 0.0f;
  const bool soft = a.soft;

  float h[NP], A2[NP];
  load_row<NP>(a.A + (int64_t)d * a.N, a.N, A2);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    A2[j] = log2_rate(A2[j]);
    h[j] = 0.0f;
  }
  if (!LOCAL) {
    if (p.run.c > 0) load_kept<NP>(a.starts + (int64_t)at * NP * a.D, a.D, d, h);
    else if (a.h0) load_row<NP>(a.h0 + ((int64_t)p.run.seq * a.D + d) * a.N, a.N, h);
  }
  float sum_dt = 0.0f;
  // A token's step and what it writes; the states through a token with B and C at
  // q, and the sum over them; what comes of it.
  auto grow = [&](S xbits, SD dtbits, float& x, float& dt) {
    const float raw = DT::load(dtbits) + bias, grown = softplus(raw);
    x = TT::load(xbits);
    dt = soft ? grown : raw;
    if (LOCAL) sum_dt += dt;
  };
  auto states = [&](const float4* qB, const float4* qC, float dt, float u) {
    float y[4] = {};
#pragma unroll
    for (int q = 0; q < NP / 4; ++q) {
      float b[4], cc[4];
      unpack(qB[q], b);
      if (!LOCAL) unpack(qC[q], cc);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& hj = h[4 * q + j];
        hj = __builtin_fmaf(exp2_hw(dt * A2[4 * q + j]), hj, u * b[j]);
        if (!LOCAL) y[j] = __builtin_fmaf(cc[j], hj, y[j]);
      }
    }
    return (y[0] + y[1]) + (y[2] + y[3]);
  };
  auto finish = [&](float sum, float x, S zbits) {
    float v = __builtin_fmaf(skip, x, sum);
    if (GATE) {
      const float z = TT::load(zbits);
      v *= z * sigmoid_for<TT>(z);
    }
    return v;
  };

  constexpr int U = 4;   // tokens whose x, dt and z are loaded ahead
  S rx[U], rz[U];
  SD rdt[U];
  auto load = [&]() {    // the next U tokens'
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rx[i] = xp[c];
      xp += a.x_st;
      rdt[i] = tp[c];
      tp += a.dt_st;
      if (GATE) {
        rz[i] = zp[c];
        zp += a.z_st;
      }
    }
  };
  float* keep = a.hs ? a.hs + ((int64_t)first_run(a.seqs, p.run.seq, kTile) + p.t0 / kTile) * NP * a.D : nullptr;
  const int whole = p.n / U * U;
  Rows16<TT, NP> rB, rC;
  if (p.n > 0) {
    rB.load(Bp, (uint32_t)a.B_st, min(p.n, kTile), a.N);
    if (!LOCAL) rC.load(Cp, (uint32_t)a.C_st, min(p.n, kTile), a.N);
    if (busy && whole) load();
    rB.write(sB[0][0], p.n, a.N);
    if (!LOCAL) rC.write(sC[0][0], p.n, a.N);
  }
  __syncthreads();
  for (int tt = 0; tt < p.n; tt += kTile) {
    const int buf = tt / kTile & 1, left = p.n - tt - kTile;   // tokens behind the tile
    if (left > 0) {
      Bp += kTile * a.B_st;
      Cp += kTile * a.C_st;
      rB.load(Bp, (uint32_t)a.B_st, min(left, kTile), a.N);
      if (!LOCAL) rC.load(Cp, (uint32_t)a.C_st, min(left, kTile), a.N);
    }
    if (busy) {
      if (!LOCAL && keep) {
        store_kept<NP>(keep, a.D, d, h);
        keep += (int64_t)NP * a.D;
      }
      const float4 *qB = sB[buf][0], *qC = sC[LOCAL ? 0 : buf][0];
      int t = tt;
#pragma unroll 1
      for (; t < min(tt + kTile, whole); t += U) {
        // the steps of all U tokens, the states through one after another, the outputs
        // of all U: chains of one token stand beside those of the others
        S z[U];
        float x[U], dt[U], y[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          grow(rx[i], rdt[i], x[i], dt[i]);
          z[i] = rz[i];
        }
        if (t + 2 * U <= p.n) load();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          y[i] = states(qB, qC, dt[i], dt[i] * x[i]);
          qB += NP / 4;
          qC += NP / 4;
          // without it decays of many tokens ahead are computed and spilled
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!LOCAL)
#pragma unroll
          for (int i = 0; i < U; ++i) {
            yp[c] = TT::store(finish(y[i], x[i], z[i]));
            yp += a.D;
          }
      }
      if (left <= 0)   // the last few
#pragma unroll 1
        for (; t < p.n; ++t) {
          float x, dt;
          grow(xp[c], tp[c], x, dt);
          const float y = states(qB, qC, dt, dt * x);
          if (!LOCAL) yp[c] = TT::store(finish(y, x, GATE ? zp[c] : S(0)));
          xp += a.x_st;
          tp += a.dt_st;
          if (GATE) zp += a.z_st;
          qB += NP / 4;
          qC += NP / 4;
          yp += a.D;
        }
    }
    if (left > 0) {
      rB.write(sB[buf ^ 1][0], left, a.N);
      if (!LOCAL) rC.write(sC[LOCAL ? 0 : buf ^ 1][0], left, a.N);
    }
    __syncthreads();
  }
  if (!busy) return;
  if (LOCAL) {
    store_kept<NP>(a.ends + (int64_t)at * NP * a.D, a.D, d, h);
    a.decay[(int64_t)at * a.D + d] = sum_dt;
  } else if (a.hT && p.t0 + p.n >= p.run.len) {
    store_row<NP>(a.hT + ((int64_t)p.run.seq * a.D + d) * a.N, a.N, h);
  }
}

// The states that a sequence's runs start with, from the second on.
__global__ __launch_bounds__(kScanThreads) void scan_join_kernel(ScanArgs a, int keep, const float* __restrict__ ends,
                                                                 const float* __restrict__ decay,
                                                                 float* __restrict__ starts) {
  const int64_t e = (int64_t)blockIdx.x * kScanThreads + threadIdx.x, K = (int64_t)a.D * keep;   // K: states kept of a run
  if (e >= K * a.seqs.nseq) return;
  const int seq = (int)(e / K);
  const int64_t in = e % K, d = in % a.D, n = in / a.D;
  const bool real = n < a.N;   // the others stay zero
  const int64_t own = d * a.N + n, M = (int64_t)a.D * a.N;   // as the caller holds it
  const Run r = span_of(a.seqs, seq, a.R);
  const int runs = (int)(((int64_t)r.len + a.R - 1) / a.R);
  const float A2 = real ? log2_rate(a.A[own]) : 0.0f;
  float h = a.h0 && real ? a.h0[seq * M + own] : 0.0f;
#pragma unroll 8
  for (int c = 1; c < runs; ++c) {
    const int64_t i = r.base + c - 1;
    h = through_run(decay[i * a.D + d] * A2, h, ends[i * K + in]);
    starts[(i + 1) * K + in] = h;
  }
}

template <class TT, class DT, int NP>
int launch_fwd_as(const ScanArgs& a, hipStream_t st) {
  const unsigned per = (unsigned)(a.G * a.ncb), blocks = (unsigned)a.nruns * per;
  const dim3 threads(kScanThreads), all(blocks + (a.seqs.cu ? kLooseRuns * per : 0));
  if (a.ends) {
    hipLaunchKernelGGL((scan_fwd_kernel<TT, DT, NP, true, false>), dim3(blocks), threads, 0, st, a);
    const int64_t states = (int64_t)a.seqs.nseq * a.D * kept_states(a.N);
    hipLaunchKernelGGL(scan_join_kernel, dim3((unsigned)((states + kScanThreads - 1) / kScanThreads)),
                       dim3(kScanThreads), 0, st, a, NP, a.ends, a.decay, a.starts);
  }
  if (a.z) hipLaunchKernelGGL((scan_fwd_kernel<TT, DT, NP, false, true>), all, threads, 0, st, a);
  else hipLaunchKernelGGL((scan_fwd_kernel<TT, DT, NP, false, false>), all, threads, 0, st, a);
  return check_launch("selective_scan");
}

template <class TT, class DT>
int launch_fwd(const ScanArgs& a, hipStream_t st) {
  if (a.N <= 4) return launch_fwd_as<TT, DT, 4>(a, st);
  if (a.N <= 8) return launch_fwd_as<TT, DT, 8>(a, st);
  if (a.N <= 16) return launch_fwd_as<TT, DT, 16>(a, st);
  if (a.N <= 32) return launch_fwd_as<TT, DT, 32>(a, st);
  return launch_fwd_as<TT, DT, 64>(a, st);
}

void fwd_runs(ScanArgs& a) { scan_runs(a, kScanThreads, kWanted, 0.48, 0.3, 0.65); }

}  // namespace

// Runs: as many as make `wanted` workgroups, kWanted or, of half the width, twice
// that: three or four rounds of them backward and one and a half forward (16 x 2048 tokens of 1536 channels, both directions: 1024
// 1540 us, 1536 1460, twice as many 1515: shorter runs are evener, but more to
// join, and the kernels were a tenth slower when this was measured); where
// there are fewer, a call is a chain of R tokens twice, half a microsecond each,
// and of T / R joins, a tenth each, so that runs are no shorter than sqrt(T / 10)
// tokens (300 tokens of 1536 channels of 16 states: runs of 64 65 us, of 16 36).
// Whole sequences where that takes less: a token's workgroup `chain` us alone and
// `busy` / 256 on a full card, runs a second pass of `extra` of the first, a launch,
// the joins, and what is kept of each written and read (256 sequences of 64 tokens
// of 256 channels: whole 39 us, 16-token runs 77).  Up to three packed sequences
// count as long as all tokens; more always go by runs, as the host knows no length
// (64 of 64 tokens, 1536 channels, 16 states: packed 87 us, as a batch 51).
void scan_runs(ScanArgs& a, int width, int wanted, double chain, double busy, double extra) {
  const Seqs& s = a.seqs;
  a.Dg = a.D / a.G;
  a.ncb = (a.Dg + width - 1) / width;
  const int64_t T = s.T, per = (int64_t)a.G * a.ncb, seqs = s.cu ? 1 : s.nseq;   // that share the workgroups
  int64_t runs = wanted / (per * seqs);                          // of a sequence, of all packed tokens
  if (s.cu && runs > s.nseq + 1) runs -= s.nseq;                  // a sequence has one run more than whole ones
  const int64_t least = (int64_t)(sqrt((double)T / 10) / kTile + 1) * kTile;
  if (runs > (T + least - 1) / least) runs = (T + least - 1) / least;
  if (runs < 1) runs = 1;
  const auto tiles = [](int64_t n) { return n < kTile ? kTile : (n + kTile - 1) / kTile * kTile; };
  const int64_t whole = tiles(T);
  a.R = (int)tiles((T + runs - 1) / runs);
  if (a.R < whole && (!s.cu || s.nseq <= 3)) {
    const double work = (double)s.B * T * per * busy / 256, kept = (double)a.D * kept_states(a.N) * 16 / 4e6;
    const auto pass = [&](double R) { return work > R * chain ? work : R * chain; };
    const double split = (1 + extra) * pass(a.R) + 12 + 0.1 * T / a.R + ((double)s.B * T / a.R + s.nseq) * kept;
    if (pass((double)T) < split) a.R = (int)whole;
  }
  a.nruns = (int)run_count(s, a.R);
}

int scan_check(const ScanArgs& a, int dtype, const char* what) {
  UTTT_REQUIRE(seqs_ok(a.seqs) && a.seqs.T < (1 << 30) && a.seqs.nseq < (1 << 30),
               "%s: bad sizes B=%d T=%d nseq=%d", what, a.seqs.B, a.seqs.T, a.seqs.nseq);
  UTTT_REQUIRE(a.D >= 1 && a.G >= 1 && a.D % a.G == 0, "%s: D=%d must be a multiple of G=%d", what, a.D, a.G);
  UTTT_REQUIRE(a.D <= 1 << 24, "%s: D=%d must be at most 2^24", what, a.D);
  UTTT_REQUIRE(a.N >= 1 && a.N <= kMaxStates, "%s: N=%d must be at most %d", what, a.N, kMaxStates);
  UTTT_REQUIRE(dtype_bytes(dtype) && (a.dt_dtype == UTTT_F32 || a.dt_dtype == dtype), "%s: dtype codes %d, %d", what,
               dtype, a.dt_dtype);
  // offsets within a tile are 32 bits
  for (const int64_t st : {a.x_st, a.dt_st, a.z_st, a.B_st, a.C_st, a.do_st})
    UTTT_REQUIRE(st >= 0 && st < (1 << 24), "%s: %lld elements between tokens", what, (long long)st);
  const bool empty = a.seqs.T == 0;
  UTTT_REQUIRE(a.A && (empty || (a.x && a.dt && a.Bm && a.Cm)), "%s: null pointer", what);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.h0) |
                         reinterpret_cast<uintptr_t>(a.hT) | reinterpret_cast<uintptr_t>(a.dhT) |
                         reinterpret_cast<uintptr_t>(a.dh0) | reinterpret_cast<uintptr_t>(a.hs);
  UTTT_REQUIRE((rows & 15u) == 0, "%s: A and the states must be 16-byte aligned", what);
  return UTTT_OK;
}

bool scan_fits(const ScanArgs& a) {   // a launch has fewer than 2^32 threads
  const int64_t runs = run_count(a.seqs, a.R), states = (int64_t)a.seqs.nseq * a.D * kept_states(a.N);
  return runs < (1 << 30) && (runs + kLooseRuns) * a.G * a.ncb < (1LL << 24) && states < (1LL << 31);
}

namespace {
size_t fwd_bytes(const ScanArgs& a) {
  const bool whole = a.R >= a.seqs.T;
  return whole ? 0 : (size_t)a.nruns * a.D * (2 * (size_t)kept_states(a.N) + 1) * 4;
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
  fwd_runs(a);
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
  UTTT_REQUIRE(x_strides && dt_strides && B_strides && C_strides && (gate_strides || !gate) && (out || T == 0),
               "%s: null pointer", what);
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  a.dt_sb = dt_strides[0]; a.dt_st = dt_strides[1];
  a.B_sb = B_strides[0]; a.B_st = B_strides[1]; a.B_sg = B_strides[2];
  a.C_sb = C_strides[0]; a.C_st = C_strides[1]; a.C_sg = C_strides[2];
  if (gate) { a.z_sb = gate_strides[0]; a.z_st = gate_strides[1]; }
  if (const int rc = scan_check(a, dtype, what)) return rc;
  fwd_runs(a);
  UTTT_REQUIRE(scan_fits(a), "%s: too many sequences, channels or states", what);
  const size_t need = fwd_bytes(a);
  UTTT_REQUIRE(!need || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, %zu needed", what,
               workspace_bytes, need);
  if (need) {
    UTTT_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned", what);
    a.ends = static_cast<float*>(workspace);
    a.starts = a.ends + (size_t)a.nruns * D * kept_states(N);
    a.decay = a.starts + (size_t)a.nruns * D * kept_states(N);
  }
  const hipStream_t st = as_stream(stream);
  UTTT_DTYPE_SWITCH_LR(dtype, TT,
                       return dt_dtype == UTTT_F32 ? launch_fwd<TT, F32T>(a, st) : launch_fwd<TT, TT>(a, st));
  return UTTT_OK;
}
