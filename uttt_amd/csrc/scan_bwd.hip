// The selective state space scan's backward for gfx950 (the forward: scan.h).
// With dy_t = dout_t silu(z_t) and the adjoint of h_t
//   q_t = C_t dy_t + e^{dt_{t+1} A} q_{t+1}          (behind the last token dhT)
// and w_t = q_t e^{dt_t A} h_{t-1} per state:
//   dC_t = sum_d dy_t h_t,  dB_t = sum_d q_t dt_t x_t,  du_t = sum_n q_t B_t
//   d dt_t = sum_n A w_t + du_t x_t,  dA = sum_t dt_t w_t,  dx_t = du_t dt_t + Dskip dy_t
//   dDskip = sum_t dy_t x_t,  dz_t = dout_t y_t silu'(z_t),  dh0 = e^{dt_0 A} q_0
// The forward kept the state at every 16th token.  A tile of 16 is run forward
// from there, the states of half of it at a time staying in registers, and then
// backward.  As in the forward the sequences are cut into runs: the adjoint that a
// run adds at its start (local pass, a lane per channel), the runs joined from the
// last to the first, and the gradients.
//
// Sums over channels (dB, dC) are added by lane, over a wave's lanes with
// permutations (halves, rows of 16 and lanes of a row exchange what the other
// needs: 16 instructions for 8 sums of 64), over its workgroup's waves in LDS, and
// over the workgroups of a token by a launch of its own; sums over tokens (dA,
// dDskip, d bias) by 256 tokens, by run and then by a launch.  All in a fixed order.
//
// Bound by vector instructions, about 3500 for 16 tokens of 32 channels of 16
// states (11 a state backward, 6 forward), at two waves a SIMD, whose 256 registers
// the states of half a tile, a tile's loads ahead and the sums fill (15 or 16 are
// spilled with a gate at 9 to 16 states, 19 to 24 in long runs, none in the others
// of up to 32).  Up to 4
// states a workgroup has 256 channels, whose tile takes 117 KB of LDS: one stands on
// a CU, one wave a SIMD (16 x 2048 tokens of 1536 channels, both directions: 4
// states 780 us, 8 states 862, 16 states 1267).  16 x 2048
// tokens of 1536 channels, 16 states, bf16, gated: local pass 208 us, joins 9,
// gradients 780 (1.3 GB), dB and dC 12, the other sums 7.  All 16 tokens' states in
// registers (spilled) and sums through LDS: 2284; one channel a lane at three waves
// a SIMD: 803; writes of sums by one lane of a channel only, under masks: 860.
// Beyond 32 states a channel takes 16 lanes, and a lane one channel with the
// states of a whole tile, three waves a SIMD (8 x 1024 tokens of 1536 channels, 64
// states, bf16, gated, both directions, without the folds of long runs below: 1153
// us, with two channels and half tiles 1321; 8 x 2048 tokens of 32 states: 1295 and
// 1214), for twice as many partial
// sums of dB and dC: 16 channels a workgroup make 96 of them there, 403 MB.
#include "scan.h"

namespace uttt {
namespace ssm {
namespace {

// What a run adds to the adjoint at its start, and the sum of its steps: a lane
// per channel, as in the forward.
template <class TT, class DT, int NP, bool GATE>
__global__ __launch_bounds__(kScanThreads, fwd_waves(NP)) void scan_adjoint_kernel(ScanArgs a) {
  using S = typename TT::S;
  using SD = typename DT::S;
  __shared__ float4 sC[2][kTile][NP / 4];
  const int tid = threadIdx.x;
  Place p;
  if (!p.init(a, kScanThreads) || p.run.c == 0) return;   // nothing comes before the first one
  const int at = p.run.base + p.run.c;
  const int last = (p.n - 1) / kTile * kTile;             // it has tokens
  const int64_t tok = p.run.tok0 + p.t0, end = tok + p.n - 1;
  const bool busy = (tid & ~(kWave - 1)) < p.nc;
  const uint32_t c = min(tid, p.nc - 1), d = p.d0 + c;
  const SD* tp = static_cast<const SD*>(a.dt) + p.run.b * a.dt_sb + end * a.dt_st + p.d0;
  const S* gp = static_cast<const S*>(a.dout) + p.run.b * a.do_sb + end * a.do_st + p.d0;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + end * a.z_st + p.d0;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + (tok + last) * a.C_st + p.g * a.C_sg;
  const float bias = a.bias ? a.bias[d] : 0.0f;
  const bool soft = a.soft;
  float q[NP], A2[NP];
  load_row<NP>(a.A + (int64_t)d * a.N, a.N, A2);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    A2[j] = log2_rate(A2[j]);
    q[j] = 0.0f;
  }
  float sum_dt = 0.0f;
  auto token = [&](const float4* qC, S gbits, SD dtbits, S zbits) {
    const float raw = DT::load(dtbits) + bias, grown = softplus(raw), dt = soft ? grown : raw;
    float dy = TT::load(gbits);
    if (GATE) {
      const float z = TT::load(zbits);
      dy *= z * sigmoid(z);
    }
    sum_dt += dt;
#pragma unroll
    for (int k = 0; k < NP / 4; ++k) {
      float cc[4];
      unpack(qC[k], cc);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q[4 * k + j] = exp2_hw(dt * A2[4 * k + j]) * __builtin_fmaf(cc[j], dy, q[4 * k + j]);
    }
  };
  auto back = [&]() {
    tp -= a.dt_st;
    gp -= a.do_st;
    if (GATE) zp -= a.z_st;
  };
  constexpr int U = 4;   // tokens that are loaded ahead
  S rg[U], rz[U];
  SD rdt[U];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rg[i] = gp[c];
      rdt[i] = tp[c];
      if (GATE) rz[i] = zp[c];
      back();
    }
  };
  Rows16<TT, NP> rC;
  rC.load(Cp, (uint32_t)a.C_st, p.n - last, a.N);
  rC.write(sC[0][0], p.n - last, a.N);
  __syncthreads();
  int t = p.n, buf = 0;
  for (int tt = last; tt >= 0; tt -= kTile, buf ^= 1) {
    if (tt > 0) {
      Cp -= kTile * a.C_st;
      rC.load(Cp, (uint32_t)a.C_st, kTile, a.N);
    }
    if (busy) {
      const float4* qC = sC[buf][0] + (t - tt) * (NP / 4);
      if (tt == last) {   // the last few, and the first loads
#pragma unroll 1
        for (; t % U; --t) {
          qC -= NP / 4;
          token(qC, gp[c], tp[c], GATE ? zp[c] : S(0));
          back();
        }
        if (t > 0) load();
      }
#pragma unroll 1
      for (; t > tt; t -= U) {
        S g[U], z[U];
        SD dt[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          g[i] = rg[i];
          dt[i] = rdt[i];
          z[i] = rz[i];
        }
        if (t > U) load();
#pragma unroll
        for (int i = 0; i < U; ++i) {
          qC -= NP / 4;
          token(qC, g[i], dt[i], z[i]);
          __builtin_amdgcn_sched_barrier(0);   // as in the forward
        }
      }
    }
    if (tt > 0) rC.write(sC[buf ^ 1][0], kTile, a.N);
    __syncthreads();
  }
  if (!busy) return;
  store_kept<NP>(a.ends + (int64_t)at * NP * a.D, a.D, d, q);
  a.decay[(int64_t)at * a.D + d] = sum_dt;
}

// The adjoint behind each run of a sequence but the last.
__global__ __launch_bounds__(kScanThreads) void scan_join_back_kernel(ScanArgs a, int keep, const float* __restrict__ ends,
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
  float q = a.dhT && real ? a.dhT[seq * M + own] : 0.0f;
#pragma unroll 8
  for (int c = runs - 1; c > 0; --c) {
    const int64_t i = r.base + c;
    q = through_run(decay[i * a.D + d] * A2, q, ends[i * K + in]);
    starts[(i - 1) * K + in] = q;
  }
}

// Sums over the tokens of a run longer than kFold (LONG) are added up every kFold
// tokens into two floats, a sum and what its rounding left out, so that the errors
// of dA, dDskip and d bias do not grow with the run: 16384 steps of 0.1 added one
// by one were off by 2770 half ulps.  A kernel of its own, as the others' registers
// leave no room for it: with folds everywhere 16 x 2048 tokens of 1536 channels, 16
// states, both directions, take 1292 us, not 1267; runs of 1024 tokens with them
// 1205 us, without 1168 (8 x 1024, 1536 channels, 64 states), and 5450, without
// 5330 (64 x 4096, 768 channels, 16 states).
constexpr int kFold = 256;
__device__ __host__ __forceinline__ int64_t part_rows(const ScanArgs& a) {
  return (int64_t)a.nruns * (a.R > kFold ? 2 : 1);
}
// had += v; returns what its rounding left out.
__device__ __forceinline__ float add_exactly(float& had, float v) {
  const float sum = had + v, back = sum - had;
  const float rest = (had - (sum - back)) + (v - back);
  had = sum;
  return rest;
}

template <int LN>
struct BwdLds {
  using M = Geo<LN>;
  float u[kTile][M::CB], dt[kTile][M::CB], dy[kTile][M::CB];   // u: then du
  float aw[kTile][M::CB], y[kTile][M::CB];                     // sums over the states
  float slope[kTile][M::CB], dgate[kTile][M::CB];              // of the step by its input; dout silu'(z)
  float4 B[kTile][LN], C[kTile][LN];
  float sum[4][kTile][2][M::NP];   // dB and dC, by wave
};

// a + (lane ^ 32's) in the lower 32 lanes, b's in the upper ones.
__device__ __forceinline__ float halves_add(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// a + (lane ^ 16's) in lanes 0..15 and 32..47, b's in the others.
__device__ __forceinline__ float rows_add(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over the lanes of a row of 16 that are LN apart, in all of them.
template <int LN>
__device__ __forceinline__ float sum_apart(float x) {
  if constexpr (LN < 16) x = dpp_add<0x128>(x);   // rotations by 8, 4, 2, 1
  if constexpr (LN < 8) x = dpp_add<0x124>(x);
  if constexpr (LN < 4) x = dpp_add<0x122>(x);
  if constexpr (LN < 2) x = dpp_add<0x121>(x);
  asm volatile("" : "+v"(x));   // as in sum_lanes
  return x;
}

template <class TT, class DT, int LN, bool GATE, bool LONG>
__global__ __launch_bounds__(kScanThreads, LN < 16 ? 2 : 3) void scan_bwd_kernel(ScanArgs a) {
  using S = typename TT::S;
  using SD = typename DT::S;
  using M = Geo<LN>;
  using L = BwdLds<LN>;
  constexpr int CS = M::CS, CB = M::CB, NP = M::NP, EPT = M::EPT, BPT = M::BPT, HT = M::HT;
  __shared__ L lds;
  const int tid = threadIdx.x, c = tid % CB, tq = tid / CB;
  Place p;
  const bool found = p.init(a, CB);
  const int num = blockIdx.x / (a.G * a.ncb);   // of the run, found or not
  const bool live = c < p.nc;
  const int wave = tid >> 6, lane = tid & 63, ln = lane % LN;
  const int ch = wave * M::WC + lane / LN * CS;
  if (!found) {
    if (num < a.nruns) {   // no run of this number: it adds nothing
#pragma unroll
      for (int s = 0; s < CS; ++s)
        if (ch + s < p.nc)
          store_states(a.part_A + ((int64_t)num * a.D + p.d0 + ch + s) * a.N, 4 * ln, a.N, make_float4(0, 0, 0, 0));
      if (live && tq == 0) {
        if (a.part_D) a.part_D[(int64_t)num * a.D + p.d0 + c] = 0.0f;
        if (a.part_bias) a.part_bias[(int64_t)num * a.D + p.d0 + c] = 0.0f;
      }
      if (LONG) {   // the rest of its sums
        const int64_t low = (int64_t)a.nruns * a.D;
#pragma unroll
        for (int s = 0; s < CS; ++s)
          if (ch + s < p.nc)
            store_states(a.part_A + (low + (int64_t)num * a.D + p.d0 + ch + s) * a.N, 4 * ln, a.N, make_float4(0, 0, 0, 0));
        if (live && tq == 0) {
          if (a.part_D) a.part_D[low + (int64_t)num * a.D + p.d0 + c] = 0.0f;
          if (a.part_bias) a.part_bias[low + (int64_t)num * a.D + p.d0 + c] = 0.0f;
        }
      }
    } else {   // the tokens of no sequence
      for (int i = num - a.nruns;; i += kLooseRuns) {
        const int t = loose_token(a.seqs, i);
        if (t < 0) break;
        if (live && tq == 0) {
          const int64_t e = (int64_t)t * a.D + p.d0 + c;
          static_cast<S*>(a.dx)[e] = TT::store(0.0f);
          static_cast<SD*>(a.ddt)[e] = DT::store(0.0f);
          if (GATE) static_cast<S*>(a.dz)[e] = TT::store(0.0f);
        }
        const int64_t row = ((int64_t)(p.d0 - p.g * a.Dg) / CB * a.seqs.T + t) * 2;
        for (int n = tid; n < 2 * a.N; n += kScanThreads)
          a.part_bc[((row + n / a.N) * a.G + p.g) * a.N + n % a.N] = 0.0f;
      }
    }
    return;
  }
  const int64_t tok = p.run.tok0 + p.t0;
  const int cl = live ? c : p.nc - 1;   // loads of a thread without a channel are the last one's
  const S* xp = static_cast<const S*>(a.x) + p.run.b * a.x_sb + tok * a.x_st + p.d0;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + tok * a.z_st + p.d0;
  const S* gp = static_cast<const S*>(a.dout) + p.run.b * a.do_sb + tok * a.do_st + p.d0;
  const SD* tp = static_cast<const SD*>(a.dt) + p.run.b * a.dt_sb + tok * a.dt_st + p.d0;
  const S* Bp = static_cast<const S*>(a.Bm) + p.run.b * a.B_sb + tok * a.B_st + p.g * a.B_sg;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + tok * a.C_st + p.g * a.C_sg;
  const int64_t out0 = ((int64_t)p.run.b * a.seqs.T + tok) * a.D + p.d0;
  const float bias = a.bias ? a.bias[p.d0 + cl] : 0.0f;
  const float skip = a.Dskip ? a.Dskip[p.d0 + cl] : 0.0f;
  const bool soft = a.soft;

  float A2[CS][4], q[CS][4], dA[CS][4];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const bool on = ch + s < p.nc;
    const int64_t row = p.d0 + ch + s;
    unpack(on ? load_states(a.A + row * a.N, 4 * ln, a.N) : make_float4(0, 0, 0, 0), A2[s]);
    float4 v = make_float4(0, 0, 0, 0);
    if (on) {
      if (p.t0 + p.n < p.run.len) {
        const float* from = a.starts + ((int64_t)num * NP + 4 * ln) * a.D + row;
        v = make_float4(from[0], from[a.D], from[2 * (int64_t)a.D], from[3 * (int64_t)a.D]);
      } else if (a.dhT) v = load_states(a.dhT + ((int64_t)p.run.seq * a.D + row) * a.N, 4 * ln, a.N);
    }
    unpack(v, q[s]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      A2[s][j] = log2_rate(A2[s][j]);
      dA[s][j] = 0.0f;
    }
  }
  const int64_t tile0 = first_run(a.seqs, p.run.seq, kTile) + p.t0 / kTile;
  float sum_D = 0.0f, sum_bias = 0.0f;
  const bool busy = wave * M::WC < p.nc;   // a wave without channels adds nothing
  if (!busy)
    for (int e = lane; e < kTile * 2 * NP; e += kWave) (&lds.sum[wave][0][0][0])[e] = 0.0f;

  // What a tile reads, a tile ahead.  Tokens behind the run's last are loaded as
  // the last and count for nothing.
  S rx[EPT], rg[EPT], rz[EPT], rB[BPT], rC[BPT];
  SD rdt[EPT];
  float rh[CS][4];
  auto load_tile = [&](int tt) {
    const int most = min(p.n - 1 - tt, kTile - 1);
    const S *x0 = xp + tt * a.x_st, *g0 = gp + tt * a.do_st, *z0 = zp + tt * a.z_st;
    const SD* t0 = tp + tt * a.dt_st;
    const S *B0 = Bp + tt * a.B_st, *C0 = Cp + tt * a.C_st;
    // within a tile 32 bits hold any offset
    const uint32_t xs = (uint32_t)a.x_st, gs = (uint32_t)a.do_st, zs = (uint32_t)a.z_st, ts = (uint32_t)a.dt_st;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint32_t t = (uint32_t)min(tq + i * M::TPP, most);
      rx[i] = x0[t * xs + cl];
      rg[i] = g0[t * gs + cl];
      rdt[i] = t0[t * ts + cl];
      if (GATE) rz[i] = z0[t * zs + cl];
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads;
      const uint32_t t = (uint32_t)min(e / NP, most), n = (uint32_t)min(e % NP, a.N - 1);
      rB[i] = B0[t * (uint32_t)a.B_st + n];
      rC[i] = C0[t * (uint32_t)a.C_st + n];
    }
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        rh[s][j] = (a.hs + (tile0 + tt / kTile) * NP * a.D + p.d0)[(uint32_t)((4 * ln + j) * a.D + min(ch + s, p.nc - 1))];
  };

  // One token forward.
  auto forward = [&](int t, const float (&from)[CS][4], float (&to)[CS][4]) {
    float b[4];
    unpack(lds.B[t][ln], b);
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      const float dts = lds.dt[t][ch + s], u = lds.u[t][ch + s];
#pragma unroll
      for (int j = 0; j < 4; ++j) to[s][j] = __builtin_fmaf(exp2_hw(dts * A2[s][j]), from[s][j], u * b[j]);
    }
  };
  // What a token's backward step reads, a token ahead.
  struct Token {
    float b[4], c[4], dt[CS], u[CS], dy[CS];
  };
  auto read = [&](int t, Token& k) {
    unpack(lds.B[t][ln], k.b);
    unpack(lds.C[t][ln], k.c);
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      k.dt[s] = lds.dt[t][ch + s];
      k.u[s] = lds.u[t][ch + s];
      k.dy[s] = lds.dy[t][ch + s];
    }
  };
  // One token backward, from the states before and behind it.
  auto backward = [&](int t, const Token& k, const float (&before)[CS][4], const float (&h)[CS][4]) {
    float db[4] = {}, dc[4] = {}, y[CS] = {}, du[CS] = {}, aw[CS] = {};
#pragma unroll
    for (int s = 0; s < CS; ++s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float qj = __builtin_fmaf(k.c[j], k.dy[s], q[s][j]);
        if (GATE) y[s] = __builtin_fmaf(k.c[j], h[s][j], y[s]);
        dc[j] = __builtin_fmaf(k.dy[s], h[s][j], dc[j]);
        db[j] = __builtin_fmaf(qj, k.u[s], db[j]);
        du[s] = __builtin_fmaf(qj, k.b[j], du[s]);
        q[s][j] = exp2_hw(k.dt[s] * A2[s][j]) * qj;
        const float w = q[s][j] * before[s][j];
        aw[s] = __builtin_fmaf(A2[s][j], w, aw[s]);
        dA[s][j] = __builtin_fmaf(k.dt[s], w, dA[s][j]);
      }
      if (GATE) y[s] = sum_lanes<LN>(y[s]);
      du[s] = sum_lanes<LN>(du[s]);
      aw[s] = sum_lanes<LN>(aw[s]) * kLn2;
    }
    // over the wave's channels: rows of 16 lanes end with dB 0 1, dB 2 3, dC 0 1, dC 2 3
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = halves_add(db[j], dc[j]);
    const float v0 = sum_apart<LN>(rows_add(v[0], v[2])), v1 = sum_apart<LN>(rows_add(v[1], v[3]));
#pragma unroll
      for (int s = 0; s < CS; ++s) {   // lanes of a channel the same
        lds.u[t][ch + s] = du[s];
        lds.aw[t][ch + s] = aw[s];
        if (GATE) lds.y[t][ch + s] = y[s];
      }
    *reinterpret_cast<float2*>(&lds.sum[wave][t][lane >> 5][4 * ln + (lane >> 3 & 2)]) = make_float2(v0, v1);
  };

  // The sums of up to kFold tokens into a long run's.
  auto fold = [&](bool first) {
    int id = tid;
    asm volatile("" : "+v"(id));   // addresses are computed here and hold no registers before
    const int fc = id % CB, fq = id / CB, fn = (id & 63) % LN, f0 = (id >> 6) * M::WC + (id & 63) / LN * CS;
    const int64_t low = (int64_t)a.nruns * a.D;   // what rounding left out stands so far behind
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      if (f0 + s < p.nc) {
        float* to = a.part_A + ((int64_t)num * a.D + p.d0 + f0 + s) * a.N;
        float had[4] = {}, rest[4] = {};
        if (!first) {
          unpack(load_states(to, 4 * fn, a.N), had);
          unpack(load_states(to + low * a.N, 4 * fn, a.N), rest);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) rest[j] += add_exactly(had[j], dA[s][j]);
        store_states(to, 4 * fn, a.N, make_float4(had[0], had[1], had[2], had[3]));
        store_states(to + low * a.N, 4 * fn, a.N, make_float4(rest[0], rest[1], rest[2], rest[3]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) dA[s][j] = 0.0f;
    }
    float* red = &lds.u[0][0];
    red[id] = sum_D;
    red[kScanThreads + id] = sum_bias;
    sum_D = sum_bias = 0.0f;
    __syncthreads();
    if (fq == 0 && fc < p.nc)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float* to = k ? a.part_bias : a.part_D;
        if (!to) continue;
        to += (int64_t)num * a.D + p.d0 + fc;
        float v = red[k * kScanThreads + fc];
#pragma unroll
        for (int i = 1; i < M::TPP; ++i) v += red[k * kScanThreads + fc + i * CB];
        float had = first ? 0.0f : *to, rest = first ? 0.0f : to[low];
        rest += add_exactly(had, v);
        *to = had;
        to[low] = rest;
      }
    __syncthreads();
  };

  if (p.n > 0) load_tile((p.n - 1) / kTile * kTile);
  for (int tt = p.n > 0 ? (p.n - 1) / kTile * kTile : -1; tt >= 0; tt -= kTile) {
    const int nt = min(kTile, p.n - tt);
    S x[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      const bool in = tl < nt && live;
      x[i] = rx[i];
      const float raw = DT::load(rdt[i]) + bias, g = TT::load(rg[i]);
      float slope, dy = g;
      const float grown = softplus(raw, slope), dt = soft ? grown : raw;
      if (GATE) {
        const float z = TT::load(rz[i]), s = sigmoid(z);
        dy = g * (z * s);
        lds.dgate[tl][c] = g * s * __builtin_fmaf(z, 1.0f - s, 1.0f);
      }
      lds.slope[tl][c] = soft ? slope : 1.0f;
      lds.dt[tl][c] = in ? dt : 0.0f;
      lds.u[tl][c] = in ? dt * TT::load(x[i]) : 0.0f;
      lds.dy[tl][c] = in ? dy : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads;
      if (e < kTile * NP) {
        const bool in = e / NP < nt && e % NP < a.N;
        reinterpret_cast<float*>(lds.B)[e] = in ? TT::load(rB[i]) : 0.0f;
        reinterpret_cast<float*>(lds.C)[e] = in ? TT::load(rC[i]) : 0.0f;
      }
    }
    float h0[CS][4], h8[CS][4];
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) h0[s][j] = ch + s < p.nc ? rh[s][j] : 0.0f;
    __syncthreads();
    if (tt > 0) load_tile(tt - kTile);
    // the tile's second half from the state in its middle, then the first, or the
    // tile as a whole: the states of HT tokens stay in registers
    if (busy) {
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) h8[s][j] = h0[s][j];
#pragma unroll
    for (int t = 0; t < kTile - HT; ++t) forward(t, h8, h8);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int half = kTile / HT - 1; half >= 0; --half) {
      const int t0 = half * HT;
      float h[HT][CS][4];
#pragma unroll
      for (int t = 0; t < HT; ++t) forward(t0 + t, t ? h[t ? t - 1 : 0] : half ? h8 : h0, h[t]);
      Token now, next;
      read(t0 + HT - 1, now);
#pragma unroll
      for (int t = HT - 1; t >= 0; --t) {
        if (t) read(t0 + t - 1, next);
        if (t0 + t < nt) backward(t0 + t, now, t ? h[t ? t - 1 : 0] : half ? h8 : h0, h[t]);
        now = next;
        __builtin_amdgcn_sched_barrier(0);   // as in the forward
      }
    }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      if (!live || tl >= nt) continue;
      const int64_t e = out0 + (int64_t)(tt + tl) * a.D + c;
      const float du = lds.u[tl][c], dy = lds.dy[tl][c], xf = TT::load(x[i]);
      const float ddt = __builtin_fmaf(du, xf, lds.aw[tl][c]) * lds.slope[tl][c];
      static_cast<S*>(a.dx)[e] = TT::store(__builtin_fmaf(du, lds.dt[tl][c], skip * dy));
      static_cast<SD*>(a.ddt)[e] = DT::store(ddt);
      if (GATE) static_cast<S*>(a.dz)[e] = TT::store(lds.dgate[tl][c] * __builtin_fmaf(skip, xf, lds.y[tl][c]));
      sum_D = __builtin_fmaf(dy, xf, sum_D);
      sum_bias += ddt;
    }
    const int64_t row0 = ((int64_t)(p.d0 - p.g * a.Dg) / CB * a.seqs.B + p.run.b) * a.seqs.T + tok + tt;
    for (int e = tid; e < nt * 2 * NP; e += kScanThreads) {
      const int tl = e / (2 * NP), k = e / NP % 2, n = e % NP;
      if (n >= a.N) continue;
      const float* s = &lds.sum[0][0][0][0] + e;
      constexpr int W = kTile * 2 * NP;
      a.part_bc[(((row0 + tl) * 2 + k) * a.G + p.g) * a.N + n] = (s[0] + s[W]) + (s[2 * W] + s[3 * W]);
    }
    __syncthreads();   // the next tile takes its place
    if (LONG && tt > 0 && tt % kFold == 0) fold(tt + kFold >= p.n);
  }
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    if (ch + s >= p.nc) continue;
    const int64_t row = p.d0 + ch + s;
    if (!LONG)
      store_states(a.part_A + ((int64_t)num * a.D + row) * a.N, 4 * ln, a.N,
                   make_float4(dA[s][0], dA[s][1], dA[s][2], dA[s][3]));
    if (a.dh0 && p.run.c == 0)
      store_states(a.dh0 + ((int64_t)p.run.seq * a.D + row) * a.N, 4 * ln, a.N,
                   make_float4(q[s][0], q[s][1], q[s][2], q[s][3]));
  }
  if (LONG) {
    fold(p.n <= kFold);
    return;
  }
  float* red = &lds.u[0][0];
  red[tid] = sum_D;
  red[kScanThreads + tid] = sum_bias;
  __syncthreads();
  if (tq == 0 && live) {
#pragma unroll
    for (int i = 1; i < M::TPP; ++i) {
      sum_D += red[c + i * CB];
      sum_bias += red[kScanThreads + c + i * CB];
    }
    if (a.part_D) a.part_D[(int64_t)num * a.D + p.d0 + c] = sum_D;
    if (a.part_bias) a.part_bias[(int64_t)num * a.D + p.d0 + c] = sum_bias;
  }
}

// dB and dC [rows, G, N] of the workgroups' sums [ncb, rows, 2, G, N].
__global__ __launch_bounds__(256) void scan_bc_kernel(const float* __restrict__ part, int ncb, int64_t rows, int GN,
                                                      int dtype, void* dB, void* dC) {
  const int64_t M = rows * 2 * GN;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < M; e += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
#pragma unroll 4
    for (int i = 0; i < ncb; ++i) v += part[(int64_t)i * M + e];
    const int64_t row = e / (2 * GN);
    const int in = (int)(e - row * 2 * GN);
    store_any(in < GN ? dB : dC, dtype, row * GN + (in < GN ? in : in - GN), v);
  }
}

constexpr int kSumSlices = 16, kMostSums = 3;
struct SumArgs {
  Sum sum[kMostSums];
  int64_t first[kMostSums + 1];   // workgroups' numbers: 16 columns each
};
// 16 columns by 16 slices of the rows.
__global__ __launch_bounds__(256) void sums_kernel(int64_t n, SumArgs a) {
  __shared__ double red[kSumSlices][17];
  const int c = threadIdx.x & 15, s = threadIdx.x >> 4;
  for (int64_t blk = blockIdx.x; blk < a.first[kMostSums]; blk += gridDim.x) {
    const int k = blk < a.first[1] ? 0 : blk < a.first[2] ? 1 : 2;
    const int64_t M = a.sum[k].M, e = (blk - a.first[k]) * 16 + c;
    const float* part = a.sum[k].part;
    double v = 0.0;
    if (e < M)
#pragma unroll 8
      for (int64_t i = s; i < n; i += kSumSlices) v += (double)part[i * M + e];
    __syncthreads();   // the columns before are read
    red[s][c] = v;
    __syncthreads();
    if (s == 0 && e < M) {
#pragma unroll
      for (int i = 1; i < kSumSlices; ++i) v += red[i][c];
      store_any(a.sum[k].out, a.sum[k].dtype, e, (float)v);
    }
  }
}

template <class TT, class DT, int LN, bool GATE>
int launch_bwd_gated(const ScanArgs& a, hipStream_t st) {
  const unsigned per = (unsigned)(a.G * a.ncb), blocks = (unsigned)a.nruns * per;
  if (a.ends) {
    ScanArgs b = a;
    b.ncb = (a.Dg + kScanThreads - 1) / kScanThreads;
    hipLaunchKernelGGL((scan_adjoint_kernel<TT, DT, 4 * LN, GATE>), dim3((unsigned)a.nruns * (unsigned)(a.G * b.ncb)),
                       dim3(kScanThreads), 0, st, b);
    const int64_t states = (int64_t)a.seqs.nseq * a.D * kept_states(a.N);
    hipLaunchKernelGGL(scan_join_back_kernel, dim3((unsigned)((states + kScanThreads - 1) / kScanThreads)),
                       dim3(kScanThreads), 0, st, a, 4 * LN, a.ends, a.decay, a.starts);
  }
  const dim3 all(blocks + (a.seqs.cu ? kLooseRuns * per : 0));
  if (a.R > kFold) hipLaunchKernelGGL((scan_bwd_kernel<TT, DT, LN, GATE, true>), all, dim3(kScanThreads), 0, st, a);
  else hipLaunchKernelGGL((scan_bwd_kernel<TT, DT, LN, GATE, false>), all, dim3(kScanThreads), 0, st, a);
  return check_launch("selective_scan_bwd");
}
template <class TT, class DT, int LN>
int launch_bwd_as(const ScanArgs& a, hipStream_t st) {
  return a.z ? launch_bwd_gated<TT, DT, LN, true>(a, st) : launch_bwd_gated<TT, DT, LN, false>(a, st);
}

template <class TT, class DT>
int launch_bwd(const ScanArgs& a, hipStream_t st) {
  switch (scan_lanes(a.N)) {
    case 1: return launch_bwd_as<TT, DT, 1>(a, st);
    case 2: return launch_bwd_as<TT, DT, 2>(a, st);
    case 4: return launch_bwd_as<TT, DT, 4>(a, st);
    case 8: return launch_bwd_as<TT, DT, 8>(a, st);
    default: return launch_bwd_as<TT, DT, 16>(a, st);
  }
}

void bwd_runs(ScanArgs& a) {
  const int narrow = scan_lanes(a.N) == 16 ? 2 : 1;   // half the channels, and the time, of a workgroup
  scan_runs(a, scan_width(a.N), kWanted * narrow, 0.8, 0.5 / narrow, 0.3);
}

// Floats of the workspace's parts.
struct Parts {
  size_t joins, A, D, bias, bc;
  size_t bytes() const { return (joins + A + D + bias + bc) * 4; }
};
Parts bwd_parts(const ScanArgs& a) {
  const size_t sums = (size_t)part_rows(a) * a.D;
  Parts p{};
  p.joins = a.R >= a.seqs.T ? 0 : (2 * (size_t)kept_states(a.N) + 1) * a.nruns * a.D;
  p.A = sums * a.N;
  p.D = p.bias = sums;
  p.bc = (size_t)a.ncb * a.seqs.B * a.seqs.T * 2 * a.G * a.N;
  const auto whole = [](size_t& n) { n = (n + 3) / 4 * 4; };   // each starts on 16 bytes
  whole(p.joins); whole(p.A); whole(p.D); whole(p.bias); whole(p.bc);
  return p;
}

}  // namespace

int launch_sums(int64_t n, std::initializer_list<Sum> sums, hipStream_t st, const char* what) {
  SumArgs a{};
  int k = 0;
  for (const Sum& s : sums) {
    a.sum[k] = s;
    a.first[k + 1] = a.first[k] + (s.part ? (s.M + 15) / 16 : 0);
    ++k;
  }
  for (; k < kMostSums; ++k) a.first[k + 1] = a.first[k];
  const int64_t blocks = a.first[kMostSums];
  if (blocks == 0) return UTTT_OK;
  hipLaunchKernelGGL(sums_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, st, n, a);
  return check_launch(what);
}

}  // namespace ssm
}  // namespace uttt

using namespace uttt;
using namespace uttt::ssm;

extern "C" size_t uttt_selective_scan_bwd_workspace_bytes(int B, int T, int nseq, int packed, int D, int N, int G) {
  ScanArgs a{};
  a.seqs = Seqs{packed ? &a : nullptr, 0, B, T, nseq};
  a.D = D; a.N = N; a.G = G;
  if (!seqs_ok(a.seqs) || D < 1 || G < 1 || D % G || N < 1 || N > kMaxStates) return 0;
  bwd_runs(a);
  return bwd_parts(a).bytes();
}

extern "C" int uttt_selective_scan_bwd(const void* x, const int64_t* x_strides, int dtype, const void* dt,
                                       const int64_t* dt_strides, int dt_dtype, const float* A, const void* Bm,
                                       const int64_t* B_strides, const void* Cm, const int64_t* C_strides,
                                       const float* skip, const void* gate, const int64_t* gate_strides,
                                       const float* dt_bias, int dt_softplus, const void* cu_seqlens,
                                       int cu_is_int64, int B, int T, int nseq, int D, int N, int G,
                                       const float* tile_states, const void* dout, const int64_t* dout_strides,
                                       const float* dfinal_state, void* dx, void* ddt, float* dA, void* dB, void* dC,
                                       float* dskip, void* dgate, float* ddt_bias, float* dinitial_state,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "uttt_selective_scan_bwd";
  ScanArgs a{};
  a.seqs = Seqs{cu_seqlens, cu_is_int64, B, T, nseq};
  a.D = D; a.N = N; a.G = G;
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = gate;
  a.dt_dtype = dt_dtype; a.soft = dt_softplus;
  a.A = A; a.Dskip = skip; a.bias = dt_bias;
  a.hs = const_cast<float*>(tile_states);
  a.dout = dout; a.dhT = dfinal_state;
  a.dx = dx; a.ddt = ddt; a.dz = dgate; a.dh0 = dinitial_state;
  UTTT_REQUIRE(x_strides && dt_strides && B_strides && C_strides && dout_strides && (gate_strides || !gate),
               "%s: null strides", what);
  UTTT_REQUIRE(dA && (T == 0 || (tile_states && dout && dx && ddt && dB && dC && (dgate || !gate))),
               "%s: null pointer", what);
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  a.dt_sb = dt_strides[0]; a.dt_st = dt_strides[1];
  a.B_sb = B_strides[0]; a.B_st = B_strides[1]; a.B_sg = B_strides[2];
  a.C_sb = C_strides[0]; a.C_st = C_strides[1]; a.C_sg = C_strides[2];
  a.do_sb = dout_strides[0]; a.do_st = dout_strides[1];
  if (gate) { a.z_sb = gate_strides[0]; a.z_st = gate_strides[1]; }
  if (const int rc = scan_check(a, dtype, what)) return rc;
  bwd_runs(a);
  UTTT_REQUIRE(scan_fits(a), "%s: too many sequences, channels or states", what);
  const Parts parts = bwd_parts(a);
  UTTT_REQUIRE(workspace && workspace_bytes >= parts.bytes() && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
               "%s: workspace of %zu bytes, %zu needed on 16", what, workspace_bytes, parts.bytes());
  float* w = static_cast<float*>(workspace);
  if (parts.joins) {
    a.ends = w;
    a.starts = a.ends + (size_t)a.nruns * D * kept_states(N);
    a.decay = a.starts + (size_t)a.nruns * D * kept_states(N);
  }
  a.part_A = w += parts.joins;
  w += parts.A;
  a.part_D = dskip ? w : nullptr;
  w += parts.D;
  a.part_bias = ddt_bias ? w : nullptr;
  a.part_bc = w + parts.bias;
  const hipStream_t st = as_stream(stream);
  int rc = UTTT_OK;
  switch (dtype) {
    case UTTT_F32: rc = launch_bwd<F32T, F32T>(a, st); break;
    case UTTT_BF16: rc = dt_dtype == UTTT_F32 ? launch_bwd<BF16T, F32T>(a, st) : launch_bwd<BF16T, BF16T>(a, st); break;
    default: rc = dt_dtype == UTTT_F32 ? launch_bwd<F16T, F32T>(a, st) : launch_bwd<F16T, F16T>(a, st); break;
  }
  if (rc) return rc;
  const int64_t rows = (int64_t)B * T;
  if (rows) {
    const int64_t n = (rows * 2 * G * N + 255) / 256;
    hipLaunchKernelGGL(scan_bc_kernel, dim3((unsigned)(n < 4096 ? n : 4096)), dim3(256), 0, st, a.part_bc, a.ncb, rows,
                       G * N, dtype, dB, dC);
  }
  return launch_sums(part_rows(a), {{a.part_A, (int64_t)D * N, dA, UTTT_F32}, {a.part_D, D, dskip, UTTT_F32},
                               {a.part_bias, D, ddt_bias, UTTT_F32}}, st, what);
}
