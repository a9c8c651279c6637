// The selective state space scan's backward for gfx950 (the forward: scan.h).
// With dy_t = dout_t silu(z_t) and the adjoint of h_t
//   q_t = C_t dy_t + e^{dt_{t+1} A} q_{t+1}          (behind the last token dhT)
// and w_t = q_t e^{dt_t A} h_{t-1} per state:
//   dC_t = sum_d dy_t h_t,  dB_t = sum_d q_t dt_t x_t,  du_t = sum_n q_t B_t
//   d dt_t = sum_n A w_t + du_t x_t,  dA = sum_t dt_t w_t,  dx_t = du_t dt_t + Dskip dy_t
//   dDskip = sum_t dy_t x_t,  dz_t = dout_t y_t silu'(z_t),  dh0 = e^{dt_0 A} q_0
// The forward kept the state at every 16th token; a tile is run forward from
// it, its 16 states staying in registers, and then backward.  As in the forward
// the sequences are cut into runs: the adjoint that a run adds at its start
// (local pass), the runs joined from the last to the first, and the gradients.
//
// Sums over channels (dB, dC) are added by lane, over a wave's lanes through
// LDS, over its workgroup's waves, and over the workgroups of a token by a
// launch of its own; sums over tokens (dA, dDskip, d bias) by run and then by a
// launch.  All in a fixed order.
#include "scan.h"

namespace uttt {
namespace ssm {
namespace {

// What a run adds to the adjoint at its start, and the sum of its steps.
template <class TT, int LN>
__global__ __launch_bounds__(kScanThreads) void scan_adjoint_kernel(ScanArgs a) {
  using S = typename TT::S;
  using M = Geo<LN>;
  constexpr int CS = M::CS, CB = M::CB, NP = M::NP, EPT = M::EPT, BPT = M::BPT;
  __shared__ float sDy[kTile][CB], sDt[kTile][CB];
  __shared__ float4 sC[kTile][LN];
  const int tid = threadIdx.x, c = tid % CB, tq = tid / CB;
  Place p;
  if (!p.init(a, CB) || p.run.c == 0) return;   // nothing comes before the first one
  const int at = p.run.base + p.run.c;
  const int64_t tok = p.run.tok0 + p.t0;
  const bool live = c < p.nc;
  const int64_t dt_at = p.run.b * a.dt_sb + tok * a.dt_st + p.d0 + c;
  const S* gp = static_cast<const S*>(a.dout) + p.run.b * a.do_sb + tok * a.do_st + p.d0 + c;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + tok * a.z_st + p.d0 + c;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + tok * a.C_st + p.g * a.C_sg;
  const float bias = live && a.bias ? a.bias[p.d0 + c] : 0.0f;
  const int wave = tid >> 6, lane = tid & 63, ln = lane % LN;
  const int ch = wave * M::WC + lane / LN * CS;
  float q[CS][4], A2[CS][4];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    unpack(ch + s < p.nc ? load_states(a.A + (int64_t)(p.d0 + ch + s) * a.N, 4 * ln, a.N) : make_float4(0, 0, 0, 0),
           A2[s]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      A2[s][j] = log2_rate(A2[s][j]);
      q[s][j] = 0.0f;
    }
  }
  S rg[EPT], rz[EPT], rC[BPT];
  uint32_t rdt[EPT];
  auto load_tile = [&](int tt) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int t = tt + tq + i * M::TPP;
      rg[i] = rz[i] = S(0);
      rdt[i] = 0;
      if (live && t < p.n) {
        rg[i] = gp[(int64_t)t * a.do_st];
        rdt[i] = load_bits(a.dt, a.dt_dtype, dt_at + (int64_t)t * a.dt_st);
        if (a.z) rz[i] = zp[(int64_t)t * a.z_st];
      }
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads, t = tt + e / NP, n = e % NP;
      rC[i] = e < kTile * NP && t < p.n && n < a.N ? Cp[(int64_t)t * a.C_st + n] : S(0);
    }
  };
  float sum_dt = 0.0f;
  const int last = (p.n - 1) / kTile * kTile;   // a run has tokens, or it is the first
  load_tile(last);
  for (int tt = last; tt >= 0; tt -= kTile) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      float dt = 0.0f, dy = TT::load(rg[i]);
      if (a.z) {
        const float z = TT::load(rz[i]);
        dy *= z * sigmoid(z);
      }
      if (tt + tl < p.n) {
        dt = widen(rdt[i], a.dt_dtype) + bias;
        if (a.soft) dt = softplus(dt);
      }
      sum_dt += dt;
      sDt[tl][c] = dt;
      sDy[tl][c] = dy;
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const int e = tid + i * kScanThreads;
      if (e < kTile * NP) reinterpret_cast<float*>(sC)[e] = TT::load(rC[i]);
    }
    __syncthreads();
    if (tt > 0) load_tile(tt - kTile);
#pragma unroll
    for (int t = kTile - 1; t >= 0; --t) {
      float cc[4];
      unpack(sC[t][ln], cc);
#pragma unroll
      for (int s = 0; s < CS; ++s) {
        const float dt = sDt[t][ch + s], dy = sDy[t][ch + s];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[s][j] = exp2_hw(dt * A2[s][j]) * __builtin_fmaf(cc[j], dy, q[s][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int s = 0; s < CS; ++s)
    if (ch + s < p.nc)
      store_states(a.ends + ((int64_t)at * a.D + p.d0 + ch + s) * a.N, 4 * ln, a.N,
                   make_float4(q[s][0], q[s][1], q[s][2], q[s][3]));
  float* red = &sDt[0][0];
  red[tid] = sum_dt;
  __syncthreads();
  if (tq == 0 && live) {
#pragma unroll
    for (int i = 1; i < M::TPP; ++i) sum_dt += red[c + i * CB];
    a.decay[(int64_t)at * a.D + p.d0 + c] = sum_dt;
  }
}

// The adjoint behind each run of a sequence but the last.
__global__ __launch_bounds__(kScanThreads) void scan_join_back_kernel(ScanArgs a, const float* __restrict__ ends,
                                                                      const float* __restrict__ decay,
                                                                      float* __restrict__ starts) {
  const int64_t e = (int64_t)blockIdx.x * kScanThreads + threadIdx.x, M = (int64_t)a.D * a.N;
  if (e >= M * a.seqs.nseq) return;
  const int seq = (int)(e / M);
  const int64_t at = e % M, d = at / a.N;
  const Run r = span_of(a.seqs, seq, a.R);
  const int runs = (int)(((int64_t)r.len + a.R - 1) / a.R);
  const float A2 = log2_rate(a.A[at]);
  float q = a.dhT ? a.dhT[e] : 0.0f;
#pragma unroll 8
  for (int c = runs - 1; c > 0; --c) {
    const int64_t i = r.base + c;
    q = __builtin_fmaf(exp2_hw(decay[i * a.D + d] * A2), q, ends[i * M + at]);
    starts[(i - 1) * M + at] = q;
  }
}

template <int LN>
struct BwdLds {
  using M = Geo<LN>;
  static constexpr int kGroup = 4;        // tokens whose sums over lanes are taken together
  static constexpr int kRow = 64 + 4;     // float4 of one token's dB or dC, four to leave the banks
  float u[kTile][M::CB], dt[kTile][M::CB], dy[kTile][M::CB];   // then du, sum A w, y
  float4 B[kTile][LN], C[kTile][LN];
  float4 red[4][kGroup * 2][kRow];        // by wave
  float4 sum[4][kTile][2][LN];
};

template <class TT, int LN>
__global__ __launch_bounds__(kScanThreads, 2) void scan_bwd_kernel(ScanArgs a) {
  using S = typename TT::S;
  using M = Geo<LN>;
  using L = BwdLds<LN>;
  constexpr int CS = M::CS, CB = M::CB, NP = M::NP, EPT = M::EPT, BPT = M::BPT;
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
    } else {   // the tokens of no sequence
      for (int i = tq;; i += M::TPP) {
        const int t = loose_token(a.seqs, i);
        if (t < 0) break;
        if (live) {
          const int64_t e = (int64_t)t * a.D + p.d0 + c;
          static_cast<S*>(a.dx)[e] = TT::store(0.0f);
          store_any(a.ddt, a.dt_dtype, e, 0.0f);
          if (a.z) static_cast<S*>(a.dz)[e] = TT::store(0.0f);
        }
        const int64_t row = ((int64_t)(p.d0 - p.g * a.Dg) / CB * a.seqs.T + t) * 2;
        for (int n = c; n < 2 * a.N; n += CB)
          a.part_bc[((row + n / a.N) * a.G + p.g) * a.N + n % a.N] = 0.0f;
      }
    }
    return;
  }
  const int64_t tok = p.run.tok0 + p.t0;
  const S* xp = static_cast<const S*>(a.x) + p.run.b * a.x_sb + tok * a.x_st + p.d0 + c;
  const S* zp = static_cast<const S*>(a.z) + p.run.b * a.z_sb + tok * a.z_st + p.d0 + c;
  const S* gp = static_cast<const S*>(a.dout) + p.run.b * a.do_sb + tok * a.do_st + p.d0 + c;
  const int64_t dt_at = p.run.b * a.dt_sb + tok * a.dt_st + p.d0 + c;
  const S* Bp = static_cast<const S*>(a.Bm) + p.run.b * a.B_sb + tok * a.B_st + p.g * a.B_sg;
  const S* Cp = static_cast<const S*>(a.Cm) + p.run.b * a.C_sb + tok * a.C_st + p.g * a.C_sg;
  const int64_t out0 = ((int64_t)p.run.b * a.seqs.T + tok) * a.D + p.d0 + c;
  const float bias = live && a.bias ? a.bias[p.d0 + c] : 0.0f;
  const float skip = live && a.Dskip ? a.Dskip[p.d0 + c] : 0.0f;

  float A2[CS][4], q[CS][4], dA[CS][4];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const bool on = ch + s < p.nc;
    const int64_t row = p.d0 + ch + s;
    unpack(on ? load_states(a.A + row * a.N, 4 * ln, a.N) : make_float4(0, 0, 0, 0), A2[s]);
    float4 v = make_float4(0, 0, 0, 0);
    if (on) {
      if (p.t0 + p.n < p.run.len) v = load_states(a.starts + ((int64_t)num * a.D + row) * a.N, 4 * ln, a.N);
      else if (a.dhT) v = load_states(a.dhT + ((int64_t)p.run.seq * a.D + row) * a.N, 4 * ln, a.N);
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

  for (int tt = p.n > 0 ? (p.n - 1) / kTile * kTile : -1; tt >= 0; tt -= kTile) {
    const int nt = min(kTile, p.n - tt);
    float x[EPT], dt[EPT], dy[EPT], slope[EPT], dgate[EPT];   // slope: of the step by its input
    {
      S rx[EPT], rg[EPT], rz[EPT], rB[BPT], rC[BPT];
      uint32_t rdt[EPT];
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int tl = tq + i * M::TPP;
        rx[i] = rg[i] = rz[i] = S(0);
        rdt[i] = 0;
        if (live && tl < nt) {
          rx[i] = xp[(int64_t)(tt + tl) * a.x_st];
          rg[i] = gp[(int64_t)(tt + tl) * a.do_st];
          rdt[i] = load_bits(a.dt, a.dt_dtype, dt_at + (int64_t)(tt + tl) * a.dt_st);
          if (a.z) rz[i] = zp[(int64_t)(tt + tl) * a.z_st];
        }
      }
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const int e = tid + i * kScanThreads, tl = e / NP, n = e % NP;
        rB[i] = rC[i] = S(0);
        if (e < kTile * NP && tl < nt && n < a.N) {
          rB[i] = Bp[(int64_t)(tt + tl) * a.B_st + n];
          rC[i] = Cp[(int64_t)(tt + tl) * a.C_st + n];
        }
      }
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int tl = tq + i * M::TPP;
        x[i] = TT::load(rx[i]);
        const float raw = widen(rdt[i], a.dt_dtype) + bias, g = TT::load(rg[i]);
        dt[i] = tl < nt ? a.soft ? softplus(raw) : raw : 0.0f;
        slope[i] = a.soft ? sigmoid(raw) : 1.0f;
        dy[i] = g;
        dgate[i] = 0.0f;
        if (a.z) {
          const float z = TT::load(rz[i]), s = sigmoid(z);
          dy[i] = g * (z * s);
          dgate[i] = g * s * __builtin_fmaf(z, 1.0f - s, 1.0f);
        }
        lds.dt[tl][c] = dt[i];
        lds.u[tl][c] = dt[i] * x[i];
        lds.dy[tl][c] = dy[i];
      }
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const int e = tid + i * kScanThreads;
        if (e < kTile * NP) {
          reinterpret_cast<float*>(lds.B)[e] = TT::load(rB[i]);
          reinterpret_cast<float*>(lds.C)[e] = TT::load(rC[i]);
        }
      }
    }
    __syncthreads();
    float h0[CS][4], h[kTile][CS][4];
#pragma unroll
    for (int s = 0; s < CS; ++s)
      unpack(ch + s < p.nc ? load_states(a.hs + ((tile0 + tt / kTile) * a.D + p.d0 + ch + s) * a.N, 4 * ln, a.N)
                           : make_float4(0, 0, 0, 0),
             h0[s]);
#pragma unroll
    for (int t = 0; t < kTile; ++t) {
      float b[4];
      unpack(lds.B[t][ln], b);
#pragma unroll
      for (int s = 0; s < CS; ++s) {
        const float dts = lds.dt[t][ch + s], u = lds.u[t][ch + s];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          h[t][s][j] = __builtin_fmaf(exp2_hw(dts * A2[s][j]), t ? h[t - 1][s][j] : h0[s][j], u * b[j]);
      }
    }
#pragma unroll
    for (int t = kTile - 1; t >= 0; --t) {
      float b[4], cc[4], db[4] = {}, dc[4] = {};
      if (t < nt) {   // behind the run's end there is nothing
        unpack(lds.B[t][ln], b);
        unpack(lds.C[t][ln], cc);
#pragma unroll
        for (int s = 0; s < CS; ++s) {
          const float dts = lds.dt[t][ch + s], u = lds.u[t][ch + s], g = lds.dy[t][ch + s];
          float y = 0.0f, du = 0.0f, aw = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float qj = __builtin_fmaf(cc[j], g, q[s][j]);
            y = __builtin_fmaf(cc[j], h[t][s][j], y);
            dc[j] = __builtin_fmaf(g, h[t][s][j], dc[j]);
            db[j] = __builtin_fmaf(qj, u, db[j]);
            du = __builtin_fmaf(qj, b[j], du);
            q[s][j] = exp2_hw(dts * A2[s][j]) * qj;
            const float w = q[s][j] * (t ? h[t - 1][s][j] : h0[s][j]);
            aw = __builtin_fmaf(A2[s][j], w, aw);
            dA[s][j] = __builtin_fmaf(dts, w, dA[s][j]);
          }
          y = sum_lanes<LN>(y);
          du = sum_lanes<LN>(du);
          aw = sum_lanes<LN>(aw);
          if (ln == 0) {
            lds.u[t][ch + s] = du;
            lds.dt[t][ch + s] = aw * kLn2;
            lds.dy[t][ch + s] = y;
          }
        }
      }
      lds.red[wave][t % L::kGroup * 2][lane] = make_float4(db[0], db[1], db[2], db[3]);
      lds.red[wave][t % L::kGroup * 2 + 1][lane] = make_float4(dc[0], dc[1], dc[2], dc[3]);
      if (t % L::kGroup == 0) {   // the wave's lanes of equal states added, 8 values a lane
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        constexpr int OUT = 2 * L::kGroup * LN;            // float4 sums
        constexpr int PER = OUT > 64 ? 1 : 64 / OUT;       // lanes that share one
        constexpr int EACH = 64 / LN / PER;                // values that a lane adds
#pragma unroll
        for (int o0 = 0; o0 < OUT; o0 += 64) {
          const int o = o0 + lane % (OUT < 64 ? OUT : 64), part = OUT < 64 ? lane / OUT : 0;
          const int row = o / LN, l = o % LN;
          float v[4] = {};
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            const float4 r = lds.red[wave][row][(part * EACH + i) * LN + l];
            v[0] += r.x; v[1] += r.y; v[2] += r.z; v[3] += r.w;
          }
#pragma unroll
          for (int d = OUT; d < 64; d <<= 1)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], d);
          if (part == 0) lds.sum[wave][t + row / 2][row % 2][l] = make_float4(v[0], v[1], v[2], v[3]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tl = tq + i * M::TPP;
      if (!live || tl >= nt) continue;
      const int64_t e = out0 + (int64_t)(tt + tl) * a.D;
      const float du = lds.u[tl][c];
      const float ddt = __builtin_fmaf(du, x[i], lds.dt[tl][c]) * slope[i];
      static_cast<S*>(a.dx)[e] = TT::store(__builtin_fmaf(du, dt[i], skip * dy[i]));
      store_any(a.ddt, a.dt_dtype, e, ddt);
      if (a.z) static_cast<S*>(a.dz)[e] = TT::store(dgate[i] * __builtin_fmaf(skip, x[i], lds.dy[tl][c]));
      sum_D = __builtin_fmaf(dy[i], x[i], sum_D);
      sum_bias += ddt;
    }
    const int64_t row0 = ((int64_t)(p.d0 - p.g * a.Dg) / CB * a.seqs.B + p.run.b) * a.seqs.T + tok + tt;
    for (int e = tid; e < nt * 2 * NP; e += kScanThreads) {
      const int tl = e / (2 * NP), k = e / NP % 2, n = e % NP;
      if (n >= a.N) continue;
      const float* s = reinterpret_cast<const float*>(lds.sum) + e;
      constexpr int W = kTile * 2 * NP;
      a.part_bc[(((row0 + tl) * 2 + k) * a.G + p.g) * a.N + n] = (s[0] + s[W]) + (s[2 * W] + s[3 * W]);
    }
    __syncthreads();   // the next tile takes its place
  }
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    if (ch + s >= p.nc) continue;
    const int64_t row = p.d0 + ch + s;
    store_states(a.part_A + ((int64_t)num * a.D + row) * a.N, 4 * ln, a.N,
                 make_float4(dA[s][0], dA[s][1], dA[s][2], dA[s][3]));
    if (a.dh0 && p.run.c == 0)
      store_states(a.dh0 + ((int64_t)p.run.seq * a.D + row) * a.N, 4 * ln, a.N,
                   make_float4(q[s][0], q[s][1], q[s][2], q[s][3]));
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

constexpr int kSumSlices = 16;
// 16 columns by 16 slices of the rows.
__global__ __launch_bounds__(256) void sums_kernel(const float* __restrict__ part, int64_t n, int64_t M, void* out,
                                                   int dtype) {
  __shared__ double red[kSumSlices][17];
  const int c = threadIdx.x & 15, s = threadIdx.x >> 4;
  for (int64_t base = (int64_t)blockIdx.x * 16; base < M; base += (int64_t)gridDim.x * 16) {
    const int64_t e = base + c;
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
      store_any(out, dtype, e, (float)v);
    }
  }
}

template <class TT, int LN>
int launch_bwd_as(const ScanArgs& a, hipStream_t st) {
  const unsigned per = (unsigned)(a.G * a.ncb), blocks = (unsigned)a.nruns * per;
  if (a.ends) {
    hipLaunchKernelGGL((scan_adjoint_kernel<TT, LN>), dim3(blocks), dim3(kScanThreads), 0, st, a);
    const int64_t states = (int64_t)a.seqs.nseq * a.D * a.N;
    hipLaunchKernelGGL(scan_join_back_kernel, dim3((unsigned)((states + kScanThreads - 1) / kScanThreads)),
                       dim3(kScanThreads), 0, st, a, a.ends, a.decay, a.starts);
  }
  hipLaunchKernelGGL((scan_bwd_kernel<TT, LN>), dim3(blocks + (a.seqs.cu ? per : 0)), dim3(kScanThreads), 0, st, a);
  return check_launch("selective_scan_bwd");
}

template <class TT>
int launch_bwd(const ScanArgs& a, hipStream_t st) {
  switch (scan_lanes(a.N)) {
    case 1: return launch_bwd_as<TT, 1>(a, st);
    case 2: return launch_bwd_as<TT, 2>(a, st);
    case 4: return launch_bwd_as<TT, 4>(a, st);
    case 8: return launch_bwd_as<TT, 8>(a, st);
    default: return launch_bwd_as<TT, 16>(a, st);
  }
}

constexpr int kBwdBlocks = 512;   // workgroups that are wanted at once

// Floats of the workspace's parts.
struct Parts {
  size_t joins, A, D, bias, bc;
  size_t bytes() const { return (joins + A + D + bias + bc) * 4; }
};
Parts bwd_parts(const ScanArgs& a) {
  const size_t states = (size_t)a.nruns * a.D * a.N, chans = (size_t)a.nruns * a.D;
  Parts p{};
  p.joins = a.R >= a.seqs.T ? 0 : 2 * states + chans;
  p.A = states;
  p.D = p.bias = chans;
  p.bc = (size_t)a.ncb * a.seqs.B * a.seqs.T * 2 * a.G * a.N;
  const auto whole = [](size_t& n) { n = (n + 3) / 4 * 4; };   // each starts on 16 bytes
  whole(p.joins); whole(p.A); whole(p.D); whole(p.bias); whole(p.bc);
  return p;
}

}  // namespace

int launch_sums(const float* part, int64_t n, int64_t M, void* out, int dtype, hipStream_t st, const char* what) {
  const int64_t blocks = (M + 15) / 16;
  hipLaunchKernelGGL(sums_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, st, part, n, M,
                     out, dtype);
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
  scan_runs(a, kBwdBlocks);
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
  if (const int rc = scan_check(a, dtype, what)) return rc;
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
  scan_runs(a, kBwdBlocks);
  UTTT_REQUIRE(scan_fits(a), "%s: too many sequences, channels or states", what);
  const Parts parts = bwd_parts(a);
  UTTT_REQUIRE(workspace && workspace_bytes >= parts.bytes() && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
               "%s: workspace of %zu bytes, %zu needed on 16", what, workspace_bytes, parts.bytes());
  float* w = static_cast<float*>(workspace);
  if (parts.joins) {
    a.ends = w;
    a.starts = a.ends + (size_t)a.nruns * D * N;
    a.decay = a.starts + (size_t)a.nruns * D * N;
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
    case UTTT_F32: rc = launch_bwd<F32T>(a, st); break;
    case UTTT_BF16: rc = launch_bwd<BF16T>(a, st); break;
    default: rc = launch_bwd<F16T>(a, st); break;
  }
  if (rc) return rc;
  const int64_t rows = (int64_t)B * T;
  if (rows) {
    const int64_t n = (rows * 2 * G * N + 255) / 256;
    hipLaunchKernelGGL(scan_bc_kernel, dim3((unsigned)(n < 4096 ? n : 4096)), dim3(256), 0, st, a.part_bc, a.ncb, rows,
                       G * N, dtype, dB, dC);
  }
  rc = launch_sums(a.part_A, a.nruns, (int64_t)D * N, dA, UTTT_F32, st, what);
  if (!rc && dskip) rc = launch_sums(a.part_D, a.nruns, D, dskip, UTTT_F32, st, what);
  if (!rc && ddt_bias) rc = launch_sums(a.part_bias, a.nruns, D, ddt_bias, UTTT_F32, st, what);
  return rc;
}
