// Backward of the chunked gated delta rule (formulas, precision and fragment
// layout in delta.h): a scan over each sequence's chunks from the last to the
// first, which carries the state's gradient and leaves dS', dR and dV, then a
// pass over all chunks at once for the gradients of q, k, g and beta.
//
// With dP = dO U^T, dA = -dR U^T, D = s E dP (j <= i), M = b_i E dA (j < i):
//   dQ = s gam dO S0^T + D K
//   dK = D^T Q + e^{G_C - G} U dS'^T - b gam dR S0^T + (M + M^T) K
//   db_i = dR_i.v_i - gam_i k_i.(S0 dR_i) + sum_j (M_ij / b_i) k_i.k_j
// A decay g_t scales every product across it, so with X = D qk + M kk
// (elementwise; qk = q_i.k_j, kk = k_i.k_j)
//   dg_t = sum_{j < t <= i} X_ij + sum_{i >= t} (s gam q.(S0 dO) - b gam k.(S0 dR))_i
//        + sum_{j < t} (e^{G_C - G} k.(dS' U))_j + gam_C <S0, dS'>
// a sum without cancelling terms, where differences of running sums of o.do
// and v.dv would lose a strong decay's small gradient.
//
// Measured, 16 x 2048 tokens, 12 heads of 128 by 128, 16-bit gates: scan 395 us
// (0.7 GB stored, 0.63 loaded: 3.4 TB/s), gradients 565 us (2 GB from and to
// memory, 0.6 once more from cache).
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

template <int KS, int NT>
struct ScanBwdLds {
  uint8_t S[3][KS * NT * 1024];   // dS', in three parts as the others
  uint8_t G[2 * NT * 1024];       // dO
  uint8_t U[3][2 * NT * 1024];    // dU
  uint8_t H[3][2 * NT * 1024];    // s gam dO
  uint8_t E[3][2 * NT * 1024];    // -b gam dR
  f32x4 R[4][NT][64];             // dR in fp32, as its waves' lanes hold it
};

template <int NT>
__device__ __forceinline__ uint32_t put_at(int wave, int r, int q) {
  return (wave >> 1) * NT * 1024 + (wave & 1) * 512 + (r + 16 * (q >> 1)) * 16 + (q & 1) * 8;
}

// The state's waves: dR = T^T dU, 16 tokens each, and a quarter of dS's features
// each.  While the others work on dU they store dS' and add Q^T (s gam dO).
template <int KS, int NT>
__device__ __forceinline__ void scan_bwd_state(const Args& a, const Scan& s, int wave, int lane,
                                               ScanBwdLds<KS, NT>& lds) {
  constexpr int FT = (2 * KS + 3) / 4;
  const int r = lane & 15, q = lane >> 4, col = s.col0 + NT * r;
  const uint32_t dead = miss_from(col, a.Dv), put_tok = put_at<NT>(wave, r, q);
  const uint32_t put = (r + 16 * (q >> 1)) * 16 + (q & 1) * 8;
  const auto get = [&](const uint8_t* buf, int f) {
    return *reinterpret_cast<const bf16x8*>(buf + f * 1024 + lane * 16);
  };

  f32x4 S[FT][NT];   // dS'
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int feat = 16 * (wave * FT + f) + 4 * q + i;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        S[f][n][i] = a.dhT && col < a.Dv && feat < a.Dk
                         ? a.dhT[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] : 0.0f;
    }

  bf16x8 qtf[FT][2], tf[2][3], ktf[FT][2];
  f32x4 bg;
  float gc;
  // Operands of the chunk before: pointers that go along, at first those of the
  // last chunk.  `left`: tokens from the chunk on to the sequence's end; 0
  // before its first chunk.
  const int lastc = s.nc - 1;
  const uint8_t* trip = a.tri + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kTriBwdBytes;
  const int64_t trans_at = ((int64_t)(s.c0 + lastc) * a.Hk + s.hk) * (4 * KS * 1024);
  const uint8_t *ktp = a.kt + trans_at, *qtp = a.qt + trans_at;
  const float* scp = a.scal + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kScal;
  const auto load_t = [&](int left) {
    const Rsrc tr = buffer_at(trip), sr = buffer_at(scp);
    const uint32_t at = lane * 16 | miss_from(0, left), s_at = 4 * (16 * wave + 4 * q) | miss_from(0, left);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      // step 0 of the lower tiles is zero and not stored: step 1 again, unused
      const int f = upper_frag(wave, wave < 2 ? ks : 1);
#pragma unroll
      for (int k = 0; k < 3; ++k) tf[ks][k] = load_frag(tr, at, (k * kTFrags + f) * 1024);
    }
    bg = load_f4(sr, s_at) * load_f4(sr, s_at, 8 * kC);
    scp -= a.Hv * kScal;
    trip -= (int64_t)a.Hv * kTriBwdBytes;
  };
  const auto load_trans = [&](int left, const uint8_t*& p, bf16x8 (&x)[FT][2]) {
    const Rsrc tr = buffer_at(p);
    const uint32_t at = lane * 16 | miss_from(0, left);
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (wave * FT + f < 2 * KS) x[f][t] = load_frag(tr, at, (2 * (wave * FT + f) + t) * 1024);
    p -= (int64_t)a.Hk * (4 * KS * 1024);
  };
  const auto load_qt = [&](int left) {
    gc = load_f1(buffer_at(scp), 4 * (kC - 1) | miss_from(0, left));
    load_trans(left, qtp, qtf);
  };
  float* dsp = a.ds + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * a.Dk * a.Dv;
  const auto put_state = [&]() {
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const int tile = wave * FT + f;
      if (tile < 2 * KS)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const Parts3 p = parts3_of(S[f][n]);
          const uint32_t at = ((tile >> 1) * NT + n) * 1024 + (tile & 1) * 512 + put;
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.S[k] + at) = p.p[k];
        }
    }
  };
  const auto save_state = [&]() {
    const Rsrc sr = buffer_at(dsp);
#pragma unroll
    for (int f = 0; f < FT; ++f)
      if (wave * FT + f < 2 * KS)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int feat = 16 * (wave * FT + f) + 4 * q + i;
          store_row<NT>(sr, 4 * (feat * a.Dv + col) | dead | miss_from(feat, a.Dk), S[f], i);
        }
    dsp -= (int64_t)a.Hv * a.Dk * a.Dv;
  };

  const int first_left = s.len - lastc * kC;
  if (lastc >= 0) {
    load_qt(first_left);
    load_t(first_left);
    load_trans(first_left, ktp, ktf);
    put_state();
    settle();
    lds_barrier();   // dO is in LDS, for the other waves
  }
  for (int c = lastc; c >= 0; --c) {
    const int next = c > 0 ? kC : 0;
    lds_barrier();   // dS' and s gam dO are in LDS
    save_state();
    // dS0 = gam_C dS' + Q^T (s gam dO) - K^T (b gam dR): the first product here
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int n = 0; n < NT; ++n) S[f][n] *= gc;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const bf16x8 h = get(lds.H[k], t * NT + n);
#pragma unroll
          for (int f = 0; f < FT; ++f)
            if (wave * FT + f < 2 * KS) S[f][n] = mfma(qtf[f][t], h, S[f][n]);
        }
      }
    load_qt(next);
    lds_barrier();   // dU is in LDS
    f32x4 R[NT] = {};   // dR = T^T dU
    {
      f32x4 R2[NT] = {}, R3[NT] = {};   // the products below 2^-7, below 2^-15 of the first
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (ks >= wave >> 1)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bf16x8 u1 = get(lds.U[0], ks * NT + n), u2 = get(lds.U[1], ks * NT + n), u3 = get(lds.U[2], ks * NT + n);
            R[n] = mfma(tf[ks][0], u1, R[n]);
            R2[n] = mfma(tf[ks][1], u1, R2[n]);
            R3[n] = mfma(tf[ks][2], u1, R3[n]);
            R2[n] = mfma(tf[ks][0], u2, R2[n]);
            R3[n] = mfma(tf[ks][1], u2, R3[n]);
            R3[n] = mfma(tf[ks][0], u3, R3[n]);
          }
#pragma unroll
      for (int n = 0; n < NT; ++n) R[n] += R2[n] + R3[n];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const Parts3 p = parts3_of(-bg * R[n]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.E[k] + put_tok + n * 1024) = p.p[k];
      lds.R[wave][n][lane] = R[n];
    }
    load_t(next);
    lds_barrier();   // b gam dR is in LDS
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const bf16x8 e = get(lds.E[k], t * NT + n);
#pragma unroll
          for (int f = 0; f < FT; ++f)
            if (wave * FT + f < 2 * KS) S[f][n] = mfma(ktf[f][t], e, S[f][n]);
        }
      }
    if (c > 0) put_state();
    load_trans(next, ktp, ktf);
  }
  if (a.dh0 && col < a.Dv) {
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int feat = 16 * (wave * FT + f) + 4 * q + i;
        if (feat < a.Dk)
#pragma unroll
          for (int n = 0; n < NT; ++n) a.dh0[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] = S[f][n][i];
      }
  }
}

// The tokens' waves, 16 tokens each: dU = e^{G_C - G} K dS' + P^T dO, its second
// term and s gam dO a chunk before they are needed, and dR and dV on their way
// to memory.
template <int KS, int NT>
__device__ __forceinline__ void scan_bwd_tokens(const Args& a, const Scan& s, int wave, int lane,
                                                ScanBwdLds<KS, NT>& lds) {
  const int r = lane & 15, q = lane >> 4, col = s.col0 + NT * r;
  const uint32_t dead = miss_from(col, a.Dv), put_tok = put_at<NT>(wave, r, q);
  bf16x8 kf[KS], pf[2][3];
  f32x4 ge, gam, bt;
  Cols<NT> gr[4];
  const int lastc = s.nc - 1;
  // K: rows of the caller's tensor, or their fragments
  const bool copies = a.kf != nullptr;
  const int64_t copy_step = (int64_t)a.Hk * (4 * KS * 1024);
  const uint8_t* kp = copies ? a.kf + (s.c0 + lastc) * copy_step + s.hk * (4 * KS * 1024)
                             : reinterpret_cast<const uint8_t*>(a.k + s.b * a.k_sb + s.hk * a.k_sh +
                                                                (s.tok0 + (int64_t)lastc * kC) * a.k_st);
  const int64_t k_step = copies ? copy_step : 2 * kC * a.k_st;
  const uint32_t krow = copies ? wave * KS * 1024 + lane * 16 : 2 * ((16 * wave + r) * (uint32_t)a.k_st + 8 * q);
  const uint32_t along = copies ? 1024 : 64;
  const uint32_t last_half = miss_from(32 * (KS - 1) + 8 * q, a.Dk), before_half = miss_from(32 * (KS - 2) + 8 * q, a.Dk);
  const uint16_t* gp = a.dout + s.b * a.do_sb + s.hv * a.do_sh + (s.tok0 + (int64_t)lastc * kC) * a.do_st;
  const uint8_t* trip = a.tri + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kTriBwdBytes;
  const float* gamp = a.scal + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kScal;   // goes with dO
  const float *betap = gamp, *gep = gamp;                                         // with dR, with K
  const uint32_t grow = 2 * ((16 * wave + 4 * q) * (uint32_t)a.do_st + col);
  int64_t out_at = (((int64_t)s.b * a.T + s.tok0 + (int64_t)lastc * kC + 16 * wave) * a.Hv + s.hv) * a.Dv;
  const auto load_k = [&](int left) {
    const uint32_t miss = miss_from(16 * wave + r, left);
    const Rsrc kr = buffer_at(kp);
    ge = load_f4(buffer_at(gep), 4 * (16 * wave + 4 * q) | miss_from(0, left), 4 * kC);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      kf[ks] = load_frag(kr, krow | miss | (ks == KS - 1 ? last_half : ks == KS - 2 ? before_half : 0), along * ks);
    gep -= a.Hv * kScal;
    kp -= k_step;
  };
  const auto load_do = [&](int left) {
    const Rsrc gr_ = buffer_at(gp);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      gr[i].load(gr_, (grow + 2 * i * (uint32_t)a.do_st) | dead | miss_from(16 * wave + 4 * q + i, left));
    gam = load_f4(buffer_at(gamp), 4 * (16 * wave + 4 * q) | miss_from(0, left));
    gamp -= a.Hv * kScal;
    gp -= kC * a.do_st;
  };
  const auto load_p = [&](int left) {
    const Rsrc tr = buffer_at(trip);
    const uint32_t at = lane * 16 | miss_from(0, left);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int f = kPFrag + upper_frag(wave, wave < 2 ? ks : 1);
#pragma unroll
      for (int k = 0; k < 3; ++k) pf[ks][k] = load_frag(tr, at, (k * kTFrags + f) * 1024);
    }
    trip -= (int64_t)a.Hv * kTriBwdBytes;
  };
  const auto load_beta = [&](int left) {
    bt = load_f4(buffer_at(betap), 4 * (16 * wave + 4 * q) | miss_from(0, left), 8 * kC);
    betap -= a.Hv * kScal;
  };
  const auto get = [&](const uint8_t* buf, int f) {
    return *reinterpret_cast<const bf16x8*>(buf + f * 1024 + lane * 16);
  };
  const auto put_do = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const u32x2 g = {gr[0].half(n) | (gr[1].half(n) << 16), gr[2].half(n) | (gr[3].half(n) << 16)};
      *reinterpret_cast<u32x2*>(lds.G + put_tok + n * 1024) = g;
    }
  };
  f32x4 Z[NT];   // P^T dO
  const auto make_z = [&]() {
    f32x4 Z2[NT] = {}, Z3[NT] = {};
#pragma unroll
    for (int n = 0; n < NT; ++n) Z[n] = f32x4{};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (ks >= wave >> 1)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 g = *reinterpret_cast<const bf16x8*>(lds.G + (ks * NT + n) * 1024 + lane * 16);
          Z[n] = mfma(pf[ks][0], g, Z[n]);
          Z2[n] = mfma(pf[ks][1], g, Z2[n]);
          Z3[n] = mfma(pf[ks][2], g, Z3[n]);
        }
#pragma unroll
    for (int n = 0; n < NT; ++n) Z[n] += Z2[n] + Z3[n];
  };
  const auto put_h = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 g;
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = gr[i].get(n);
      const Parts3 p = parts3_of(g * (gam * a.scale));
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.H[k] + put_tok + n * 1024) = p.p[k];
    }
  };

  // dO and P are a chunk ahead of K and beta
  const int first_left = s.len - lastc * kC;
  if (lastc >= 0) {
    load_do(first_left);
    load_p(first_left);
    load_k(first_left);
    load_beta(first_left);
    settle();
    put_do();
    lds_barrier();   // dO is in LDS
    make_z();
    put_h();
    const int next = lastc > 0 ? kC : 0;
    load_do(next);
    load_p(next);
    settle();
  }
  for (int c = lastc; c >= 0; --c) {
    const int left = s.len - c * kC, next = c > 0 ? kC : 0, later = c > 1 ? kC : 0;
    lds_barrier();   // dS' and s gam dO are in LDS
    {
      f32x4 X[NT] = {}, X2[NT] = {}, X3[NT] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          X[n] = mfma(kf[ks], get(lds.S[0], ks * NT + n), X[n]);
          X2[n] = mfma(kf[ks], get(lds.S[1], ks * NT + n), X2[n]);
          X3[n] = mfma(kf[ks], get(lds.S[2], ks * NT + n), X3[n]);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const Parts3 p = parts3_of(ge * (X[n] + (X2[n] + X3[n])) + Z[n]);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.U[k] + put_tok + n * 1024) = p.p[k];
      }
    }
    put_do();        // of the chunk before
    lds_barrier();   // dU and dO are in LDS, s gam dO read
    load_k(next);
    make_z();
    put_h();
    load_p(later);
    load_do(later);
    lds_barrier();   // dR is in LDS
    {
      const Rsrc vr = buffer_at(a.dv + out_at), rr = buffer_at(a.dr + out_at);
      f32x4 R[NT];
      u32x2 v[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        R[n] = lds.R[wave][n][lane];
        v[n] = round_of(bt * R[n]);
      }
      load_beta(next);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = (4 * q + i) * (uint32_t)(a.Hv * a.Dv) + col;
        const uint32_t none = dead | miss_from(16 * wave + 4 * q + i, left);
        store_row<NT>(vr, 2 * at | none, v, i);
        store_row<NT>(rr, 4 * at | none, R, i);
      }
      out_at -= (int64_t)kC * a.Hv * a.Dv;
    }
  }
}

// The forward scan's geometry and division of work (delta_fwd.hip), from the
// last chunk to the first.
template <int KS, int NT>
__global__ __launch_bounds__(512) void delta_scan_bwd_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) ScanBwdLds<KS, NT> lds;
  Scan s;
  if (!s.init(a, 16 * NT)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (wave < 4) scan_bwd_state<KS, NT>(a, s, wave, lane, lds);
  else scan_bwd_tokens<KS, NT>(a, s, wave & 3, lane, lds);
}

// One chunk of one key head, its value heads one after another so that the
// shared gradients of q and k are added in registers, in a fixed order.  Each
// of the 2 KS waves has one 16-feature tile of the [64, Dk] products; the
// first PW also have a 16-token row tile and CT column tiles of the [64, 64]
// ones.  The rows of dO, dR and U pass through LDS 32 columns at a time (every
// wave reads all of them), loaded a step ahead; S0 and dS' go straight to the
// wave that has their features.  It is bound by memory (S0, dS', U and dR are
// 4 bytes an element) and its latency, so that registers (128) and LDS are
// kept to what lets two workgroups of eight waves share a CU: the products
// with dS' come in a second pass, when those with S0 and the [64, 64] ones are
// done, which reads U and S0 (for <S0, dS'>) once more from cache.  With all
// of them in one pass and one workgroup a CU 6144 chunks of 128 x 128 took 745
// us, with two workgroups and the registers spilled 1129, as it is now 565.
// D, M and M^T go through LDS a part at a time; the second is 34 us of that.  PARTS: bf16 parts
// of U, S0, dR, dS' and X, 3 where g or beta is fp32 and its gradient shows what a
// third holds, 2 where both are 16-bit.
constexpr int grads_waves(int KS, bool shared, int parts) {   // per SIMD, at least
  return KS == 8 ? 4 : KS == 6 ? 3 : shared || (parts == 3 && KS < 4) ? 2 : 4;
}

template <int KS, bool SHARED, int PARTS>
__global__ __launch_bounds__(128 * KS, grads_waves(KS, SHARED, PARTS)) void delta_grads_kernel(Args a) {
  constexpr int NW = 2 * KS, PW = NW >= 16 ? 16 : NW >= 8 ? 8 : 4, CT = 16 / PW;
  constexpr int LX = kC + 4, LM = kC + 8, LO = 32 * KS + 8;
  constexpr int kThreads = 64 * NW, kStage = (1 + 2 * PARTS) * 4 * 1024;   // dO, dR's parts, U's: 4 fragments each
  constexpr int kHalves = PARTS == 2 ? 2 : 1;                 // the stage twice, where two workgroups share a CU
  constexpr int kMats = 3 * kC * LM * 2;                      // D, D^T, M + M^T; before them X
  constexpr int kRows = 3 * NW * kC * 4, kOut = kC * LO * 2;
  constexpr int kPair = 8 * KS * 1024;                         // K and Q fragments
  constexpr int kBig = kHalves * kStage > kMats + kRows ? kHalves * kStage : kMats + kRows;
  constexpr int kBuf = kBig > kPair ? kBig : kPair;
  __shared__ __attribute__((aligned(16))) uint8_t trans[NW][4 * 1024];   // a wave's K^T and Q^T fragments
  __shared__ __attribute__((aligned(16))) uint8_t buf[kBuf > kOut ? kBuf : kOut];
  __shared__ __attribute__((aligned(16))) float Sc[kScal];
  __shared__ float bsum[PW][16], zsum[PW][kC], rvs[kC], dots[NW];
  __shared__ int bad;   // the first column of X that is not finite
  float* Xl = reinterpret_cast<float*>(buf);
  __bf16* Dl = reinterpret_cast<__bf16*>(buf);
  __bf16* DTl = Dl + kC * LM;
  __bf16* Nl = DTl + kC * LM;
  float* rows = reinterpret_cast<float*>(buf + kMats);   // [3][NW][kC]: q.(S0 dO), k.(S0 dR), k.(dS' U)
  const int c = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk;
  const Chunk ch = chunk_of(a, c);
  if (ch.seq < 0) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r0 = lane & 15, q0 = lane >> 4;
  const int rw = wave & 3, cw = (wave >> 2) * CT;   // the wave's row tile, first column tile
  const int group = a.Hv / a.Hk;
  const uint16_t* kp = a.k + ch.b * a.k_sb + ch.t0 * a.k_st + hk * a.k_sh;
  const uint16_t* qp = a.q + ch.b * a.q_sb + ch.t0 * a.q_st + hk * a.q_sh;
  {
    const int64_t at = ((int64_t)c * a.Hk + hk) * (4 * KS * 1024) + wave * 2048 + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<bf16x8*>(trans[wave] + i * 1024 + lane * 16) =
          *reinterpret_cast<const bf16x8*>(a.kt + at + i * 1024);
      *reinterpret_cast<bf16x8*>(trans[wave] + (2 + i) * 1024 + lane * 16) =
          *reinterpret_cast<const bf16x8*>(a.qt + at + i * 1024);
    }
  }
  f32x4 dQ[4] = {}, dK[4] = {};
  const int64_t orow = (int64_t)a.Hv * a.Dv, tok = (int64_t)ch.b * a.T + ch.t0;
  const int hv_end = SHARED ? (hk + 1) * group : hk + 1;
  for (int hv = SHARED ? hk * group : hk; hv < hv_end; ++hv) {
    // Behind this the compiler takes r and q for new values in every turn: the
    // some 60 offsets and masks made of them, kept over the loop, would be
    // spilled for the products' registers.
    int r = r0, q = q0;
    asm volatile("" : "+v"(r), "+v"(q));
    const int feat = 16 * wave + r;
    if (tid == 0) bad = kC;
    for (int i = tid; i < kScal; i += kThreads) Sc[i] = a.scal[((size_t)c * a.Hv + hv) * kScal + i];
    const int64_t oat = tok * orow + (int64_t)hv * a.Dv;
    const uint16_t* gp = a.dout + ch.b * a.do_sb + ch.t0 * a.do_st + hv * a.do_sh;
    const Rsrc vp = buffer_at(a.v + ch.b * a.v_sb + ch.t0 * a.v_st + hv * a.v_sh);
    const int64_t sat = ((int64_t)c * a.Hv + hv) * a.Dk * a.Dv;
    const Rsrc sp = buffer_at(a.s0 + sat), dp = buffer_at(a.ds + sat);
    const uint32_t srow = 4 * (feat * a.Dv + 8 * q) | miss_from(feat, a.Dk);
    // Rows of 16 tokens by 32 columns to LDS, 16 bytes a lane at a time: four
    // fragments of dO, then eight half ones each of dR and U in fp32.  Wave w has
    // pieces w, w + NW, .. of `count` from `from` on.
    u32x4 st[(20 + NW - 1) / NW];
    const auto load_rows = [&](int e0, int from, int count) {
#pragma unroll
      for (int i = 0; i < (20 + NW - 1) / NW; ++i) {
        const int f = i * NW + wave, g = from + f;
        if (f < count) {
          const int tile = g < 4 ? g : (g >> 1) & 3, half = g < 4 ? 0 : 4 * (g & 1);
          const uint32_t miss = miss_from(16 * tile + r, ch.n) | miss_from(e0 + 8 * q, a.Dv);
          const uint32_t col = e0 + 8 * q + half;
          const Rsrc p = g < 4 ? buffer_at(gp + 16 * tile * a.do_st)
                               : buffer_at((g < 12 ? a.dr : a.u) + oat + 16 * tile * orow);
          const uint32_t at = g < 4 ? 2 * (r * (uint32_t)a.do_st + col) : 4 * (r * (uint32_t)orow + col);
          st[i] = __builtin_amdgcn_raw_buffer_load_b128(p, at | miss, 0, 0);
        }
      }
    };
    const auto put_rows = [&](uint8_t* stage, int from, int count) {
#pragma unroll
      for (int i = 0; i < (20 + NW - 1) / NW; ++i) {
        const int f = i * NW + wave, g = from + f;
        if (f < count) {
          if (g < 4) {
            *reinterpret_cast<u32x4*>(stage + g * 1024 + lane * 16) = st[i];
          } else {   // part k of dR or U behind the parts before it; of U alone from the start
            const int base = from ? 0 : g < 12 ? 4 : 4 + 4 * PARTS;
            const Parts3 x = parts3_of(__builtin_bit_cast(f32x4, st[i]));
#pragma unroll
            for (int k = 0; k < PARTS; ++k)
              *reinterpret_cast<u32x2*>(stage + (base + 4 * k + ((g >> 1) & 3)) * 1024 + lane * 16 + 8 * (g & 1)) = x.p[k];
          }
        }
      }
    };
    struct Eight {
      f32x4 a, b;
    };
    const auto load_state = [&](Rsrc p, int e0) {
      const uint32_t at = (srow + 4 * e0) | miss_from(e0 + 8 * q, a.Dv);
      return Eight{load_f4(p, at), load_f4(p, at, 16)};
    };
    // a wave's own 16 x 16 products, of which the diagonal is wanted
    const auto diagonal = [&](f32x4 x) {
      float d = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) d += 4 * q + i == r ? x[i] : 0.0f;
      return d;
    };
    f32x4 EQ[4] = {}, ER[4] = {}, dP[CT] = {}, dA[CT] = {}, rv = {};
    {
      bf16x8 vf;
      const auto load_v = [&](int e0) {
        const int t = 16 * rw + r;
        vf = load_frag(vp, 2 * (t * (uint32_t)a.v_st + e0 + 8 * q) | miss_from(t, ch.n) | miss_from(e0 + 8 * q, a.Dv));
      };
      load_rows(0, 0, 20);
      Eight s8 = load_state(sp, 0);
      if (wave < 4) load_v(0);
      int half = 0;
      for (int e0 = 0; e0 < a.Dv; e0 += 32, half ^= kHalves - 1) {
        uint8_t* stage = buf + half * kStage;
        if (kHalves == 1 && e0 > 0) lds_barrier();   // the step before is read
        put_rows(stage, 0, 20);
        load_rows(e0 + 32, 0, 20);   // past Dv: nothing is read
        lds_barrier();               // the step's rows are in LDS; the other half is free after the next one
        const auto row = [&](int which, int rt) {   // 0: dO, then the parts of dR, of U
          return *reinterpret_cast<const bf16x8*>(stage + (4 * which + rt) * 1024 + lane * 16);
        };
        bf16x8 sf[PARTS];
        split8(s8.a, s8.b, sf);
        s8 = load_state(sp, e0 + 32);
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          const bf16x8 g = row(0, rt);
#pragma unroll
          for (int k = 0; k < PARTS; ++k) EQ[rt] = mfma(g, sf[k], EQ[rt]);
#pragma unroll
          for (int j = 0; j < PARTS; ++j) {
            const bf16x8 x = row(1 + j, rt);
#pragma unroll
            for (int k = 0; j + k < PARTS; ++k) ER[rt] = mfma(x, sf[k], ER[rt]);
          }
        }
        if (wave < PW) {
          const bf16x8 gw = row(0, rw);
          bf16x8 x[PARTS];
#pragma unroll
          for (int j = 0; j < PARTS; ++j) x[j] = row(1 + j, rw);
          if (wave < 4) {   // dR.v
#pragma unroll
            for (int j = 0; j < PARTS; ++j) rv = mfma(x[j], vf, rv);
            load_v(e0 + 32);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
              const bf16x8 u = row(1 + PARTS + k, cw + c);
              dP[c] = mfma(gw, u, dP[c]);
#pragma unroll
              for (int j = 0; j + k < PARTS; ++j) dA[c] = mfma(x[j], u, dA[c]);
            }
        }
      }
    }
    lds_barrier();   // every wave is done with the staged rows
    asm volatile("" : "+v"(r), "+v"(q));
    // kk = K K^T and qk = Q K^T, the chunk's rows through LDS
    f32x4 kk[CT] = {}, qk[CT] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = i * NW + wave, ks = f >> 3, t = 16 * (f & 3) + r, e = 32 * ks + 8 * q;
      const uint32_t st = (uint32_t)(f & 4 ? a.q_st : a.k_st);
      *reinterpret_cast<bf16x8*>(buf + f * 1024 + lane * 16) =
          load_frag(buffer_at(f & 4 ? qp : kp), 2 * (t * st + e) | miss_from(t, ch.n) | miss_from(e, a.Dk));
    }
    lds_barrier();
    if (wave < PW) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const auto row = [&](int f) { return *reinterpret_cast<const bf16x8*>(buf + (8 * ks + f) * 1024 + lane * 16); };
        const bf16x8 ka = row(rw), qa = row(4 + rw);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          const bf16x8 kb = row(cw + x);
          kk[x] = mfma(ka, kb, kk[x]);
          qk[x] = mfma(qa, kb, qk[x]);
        }
      }
    }
    lds_barrier();
    asm volatile("" : "+v"(r), "+v"(q));
    // X; dP and dA become D and M
    if (wave < PW) {
      if (wave < 4) {
        const float d = diagonal(rv);   // of column r, in one of the four lanes that have it
        if (r >> 2 == q) rvs[16 * rw + r] = d;
      }
      f32x4 bs = {};
      float zero = 0.0f;   // NaN where some X is not finite
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const int j = 16 * (cw + x) + r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * rw + 4 * q + i;
          const float E = row >= j ? __expf((Sc[3 * kC + row] - Sc[3 * kC + j]) +
                                            (Sc[4 * kC + row] - Sc[4 * kC + j])) : 0.0f;
          const float D = row >= j ? a.scale * E * dP[x][i] : 0.0f;
          const float m = row > j ? -E * dA[x][i] : 0.0f;
          const float M = Sc[2 * kC + row] * m;
          bs[i] = __builtin_fmaf(m, kk[x][i], bs[i]);
          const float xv = D * qk[x][i] + M * kk[x][i];
          Xl[row * LX + j] = xv;
          zero = __builtin_fmaf(xv, 0.0f, zero);
          dP[x][i] = D;
          dA[x][i] = M;
        }
      }
      // An X that is not finite comes from a U of token j that is not.  It is left
      // out of the sums over j < t, whose product multiplies zeros with it, and dg
      // is NaN behind j.
      if (__builtin_expect(zero != 0.0f, 0))
        for (int x = 0; x < CT; ++x)
          for (int i = 0; i < 4; ++i) {
            const int j = 16 * (cw + x) + r;
            float* xp = Xl + (16 * rw + 4 * q + i) * LX + j;
            if (*xp * 0.0f != 0.0f) {
              *xp = 0.0f;
              atomicMin(&bad, j);
            }
          }
#pragma unroll
      for (int i = 0; i < 4; ++i) bs[i] = sum16(bs[i]);
      if (r == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) bsum[wave][4 * q + i] = bs[i];
    }
    // Rows' products with q (which = 1) or k (0), a wave's features' share of them
    const auto row_products = [&](int which, int slot, int rt, f32x4 x) {
      const uint8_t* tp = trans[wave] + 2048 * which + (rt >> 1) * 1024 +
                          ((2 * (rt & 1) + (q >> 1)) * 16 + r) * 16 + (q & 1) * 8;
      const u32x2 w = *reinterpret_cast<const u32x2*>(tp);
      f32x4 s;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[i] = sum16(x[i] * __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16));
      if (r == 0) *reinterpret_cast<f32x4*>(rows + (slot * NW + wave) * kC + 16 * rt + 4 * q) = s;
    };
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      row_products(1, 0, rt, EQ[rt]);
      row_products(0, 1, rt, ER[rt]);
      const f32x4 gam = *reinterpret_cast<const f32x4*>(Sc + 16 * rt + 4 * q);
      const f32x4 bt = *reinterpret_cast<const f32x4*>(Sc + 2 * kC + 16 * rt + 4 * q);
      const f32x4 nq = a.scale * gam * EQ[rt], nk = -bt * gam * ER[rt];
      dQ[rt] = SHARED ? dQ[rt] + nq : nq;
      dK[rt] = SHARED ? dK[rt] + nk : nk;
    }
    lds_barrier();
    asm volatile("" : "+v"(r), "+v"(q));
    // sum_{j < t} X_ij as a product with the strictly upper ones
    if (wave < PW) {
      f32x4 Z[CT] = {};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const float* xp = Xl + (16 * rw + r) * LX + 32 * ks + 8 * q;
        bf16x8 xf[PARTS];
        split8(*reinterpret_cast<const f32x4*>(xp), *reinterpret_cast<const f32x4*>(xp + 4), xf);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          const int below = 16 * (cw + x) + r - (32 * ks + 8 * q);   // ones in places under it
          u32x4 ones;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ones[i] = 2 * i + 1 < below ? 0x3f803f80u : 2 * i < below ? 0x3f80u : 0u;
#pragma unroll
          for (int k = 0; k < PARTS; ++k) Z[x] = mfma(xf[k], __builtin_bit_cast(bf16x8, ones), Z[x]);
        }
      }
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const int t = 16 * (cw + x) + r;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) z += 16 * rw + 4 * q + i >= t ? Z[x][i] : 0.0f;
        z += __shfl_xor(z, 16);
        z += __shfl_xor(z, 32);
        if (q == 0) zsum[wave][t] = z;
      }
    }
    lds_barrier();   // X is read: D, D^T and M + M^T take its place
    // dQ += D K, dK += D^T Q + (M + M^T) K, the matrices in two bf16 parts, one
    // after the other through LDS
    Eight s8, d8;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (wave < PW) {
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          const int j = 16 * (cw + x) + r, row0 = 16 * rw + 4 * q;
          const u32x2 d = round_of(dP[x]), m = round_of(dA[x]);
          *reinterpret_cast<u32x2*>(DTl + j * LM + row0) = d;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = row0 + i;
            const uint32_t dw = i & 1 ? d[i >> 1] & 0xffff0000u : d[i >> 1] << 16;
            const uint32_t mw = i & 1 ? m[i >> 1] & 0xffff0000u : m[i >> 1] << 16;
            reinterpret_cast<uint16_t*>(Dl)[row * LM + j] = (uint16_t)(dw >> 16);
            if (row >= j) {   // M is zero on the diagonal
              reinterpret_cast<uint16_t*>(Nl)[row * LM + j] = (uint16_t)(mw >> 16);
              reinterpret_cast<uint16_t*>(Nl)[j * LM + row] = (uint16_t)(mw >> 16);
            }
            dP[x][i] -= __uint_as_float(dw);
            dA[x][i] -= __uint_as_float(mw);
          }
        }
      }
      lds_barrier();
      if (part == 1) {   // for the second pass
        load_rows(0, 12, 8);
        s8 = load_state(sp, 0);
        d8 = load_state(dp, 0);
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const bf16x8 kb = *reinterpret_cast<const bf16x8*>(trans[wave] + ks * 1024 + lane * 16);
        const bf16x8 qb = *reinterpret_cast<const bf16x8*>(trans[wave] + (2 + ks) * 1024 + lane * 16);
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          const int o = (16 * rt + r) * LM + 32 * ks + 8 * q;
          if (ks == 0 || rt >= 2) dQ[rt] = mfma(*reinterpret_cast<const bf16x8*>(Dl + o), kb, dQ[rt]);
          if (ks == 1 || rt < 2) dK[rt] = mfma(*reinterpret_cast<const bf16x8*>(DTl + o), qb, dK[rt]);
          dK[rt] = mfma(*reinterpret_cast<const bf16x8*>(Nl + o), kb, dK[rt]);
        }
      }
      lds_barrier();   // every wave is done with the 64 x 64 matrices
    }
    // the second pass: U dS'^T and <S0, dS'>
    f32x4 EU[4] = {}, dot = {};
    {
      int half = 0;
      for (int e0 = 0; e0 < a.Dv; e0 += 32, half ^= 1) {
        uint8_t* stage = buf + half * 4 * PARTS * 1024;
        put_rows(stage, 12, 8);
        load_rows(e0 + 32, 12, 8);
        lds_barrier();
        bf16x8 sf[PARTS], df[PARTS];
        split8(d8.a, d8.b, df);
        d8 = load_state(dp, e0 + 32);
#pragma unroll
        for (int rt = 0; rt < 4; ++rt)
#pragma unroll
          for (int j = 0; j < PARTS; ++j) {
            const bf16x8 u = *reinterpret_cast<const bf16x8*>(stage + (4 * j + rt) * 1024 + lane * 16);
#pragma unroll
            for (int k = 0; j + k < PARTS; ++k) EU[rt] = mfma(u, df[k], EU[rt]);
          }
        split8(s8.a, s8.b, sf);
        s8 = load_state(sp, e0 + 32);
#pragma unroll
        for (int j = 0; j < PARTS; ++j)
#pragma unroll
          for (int k = 0; j + k < PARTS; ++k) dot = mfma(sf[j], df[k], dot);
      }
    }
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      row_products(0, 2, rt, EU[rt]);
      dK[rt] += *reinterpret_cast<const f32x4*>(Sc + kC + 16 * rt + 4 * q) * EU[rt];
    }
    {
      float d = sum16(diagonal(dot));
      d += __shfl_xor(d, 16);
      d += __shfl_xor(d, 32);
      if (lane == 0) dots[wave] = d;
    }
    lds_barrier();
    if (wave == NW - 1) {   // lane = token
      float s[3] = {};
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int w = 0; w < NW; ++w) s[i] += rows[(i * NW + w) * kC + lane];
      const float gam = Sc[lane], ge = Sc[kC + lane], bt = Sc[2 * kC + lane];
      const float after = a.scale * gam * s[0] - bt * gam * s[1];   // of tokens t and later
      const float before = ge * s[2];                                // of tokens before t
      float suf = after, pre = before;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const float x = __shfl_down(suf, d), y = __shfl_up(pre, d);
        if (lane + d < 64) suf += x;
        if (lane >= d) pre += y;
      }
      pre = __shfl_up(pre, 1);
      if (lane == 0) pre = 0.0f;
      float all = 0.0f, z = 0.0f, b = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) all += dots[w];
      // column t's sums are with the waves of its column tile, row i's with those of its row tile
#pragma unroll
      for (int w = 0; w < 4; ++w) z += zsum[w + 4 * ((lane >> 4) / CT)][lane];
#pragma unroll
      for (int w = 0; w < PW / 4; ++w) b += bsum[(lane >> 4) + 4 * w][lane & 15];
      if (lane < ch.n) {
        const int64_t at = (tok + lane) * a.Hv + hv;
        store_any(a.dg, a.g_dtype, at, lane > bad ? __builtin_nanf("") : z + suf + pre + Sc[kC - 1] * all);
        store_any(a.dbeta, a.beta_dtype, at, rvs[lane] - gam * s[1] + b);
      }
    }
    lds_barrier();   // LDS is free for the next head, or for the results
  }
  // through LDS to whole rows
  __bf16* Ol = reinterpret_cast<__bf16*>(buf);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which) lds_barrier();
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        Ol[(16 * rt + 4 * q0 + i) * LO + 16 * wave + r0] = (__bf16)(which ? dK[rt][i] : dQ[rt][i]);
    lds_barrier();
    uint16_t* out = (which ? a.dk : a.dq) + (tok * a.Hk + hk) * a.Dk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = i * kThreads + tid, t = p / (4 * KS), e = 8 * (p % (4 * KS));
      if (t < ch.n && e < a.Dk)
        *reinterpret_cast<u32x4*>(out + (int64_t)t * a.Hk * a.Dk + e) =
            *reinterpret_cast<const u32x4*>(Ol + t * LO + e);
    }
  }
}

template <int KS>
int launch_bwd(const Args& a, hipStream_t st) {
  switch (scan_tiles(a, true)) {
    case 1:
      hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 1>), dim3((unsigned)scan_blocks(a, 16)), dim3(512), 0, st, a);
      break;
    case 2:
      hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 2>), dim3((unsigned)scan_blocks(a, 32)), dim3(512), 0, st, a);
      break;
    default:
      if constexpr (scan_widest(KS, true) == 4)
        hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 4>), dim3((unsigned)scan_blocks(a, 64)), dim3(512), 0, st, a);
  }
  if (const int rc = check_launch("delta_scan_bwd")) return rc;
  if (a.nchunks == 0) return UTTT_OK;
  const dim3 grid((unsigned)((int64_t)a.nchunks * a.Hk));
  const bool shared = a.Hv > a.Hk, exact = a.g_dtype == UTTT_F32 || a.beta_dtype == UTTT_F32;
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(128 * KS), 0, st, a); };
  if (shared) exact ? launch(delta_grads_kernel<KS, true, 3>) : launch(delta_grads_kernel<KS, true, 2>);
  else exact ? launch(delta_grads_kernel<KS, false, 3>) : launch(delta_grads_kernel<KS, false, 2>);
  return check_launch("delta_grads");
}

}  // namespace
}  // namespace delta
}  // namespace uttt

using namespace uttt;
using namespace uttt::delta;

extern "C" int uttt_gated_delta_bwd(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, const void* g, int g_dtype,
                                    const void* beta, int beta_dtype, const void* cu_seqlens,
                                    int cu_is_int64, int B, int T, int nseq, int Hk, int Hv, int Dk,
                                    int Dv, float scale, const void* u_saved, const void* s_saved,
                                    const void* dout, const int64_t* do_strides,
                                    const float* dfinal_state, void* dq, void* dk, void* dv, void* dg,
                                    void* dbeta, float* dinitial_state, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* what = "uttt_gated_delta_bwd";
  UTTT_REQUIRE(q_strides && k_strides && v_strides && do_strides, "%s: null strides", what);
  const bool packed = cu_seqlens != nullptr;
  Args a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_sb = q_strides[0]; a.q_st = q_strides[1]; a.q_sh = q_strides[2];
  a.k_sb = k_strides[0]; a.k_st = k_strides[1]; a.k_sh = k_strides[2];
  a.v_sb = v_strides[0]; a.v_st = v_strides[1]; a.v_sh = v_strides[2];
  a.do_sb = do_strides[0]; a.do_st = do_strides[1]; a.do_sh = do_strides[2];
  a.g = g; a.beta = beta; a.g_dtype = g_dtype; a.beta_dtype = beta_dtype;
  a.B = B; a.T = T; a.Hk = Hk; a.Hv = Hv; a.Dk = Dk; a.Dv = Dv; a.nseq = nseq;
  a.cps = (T + kC - 1) / kC;
  a.scale = scale;
  if (const int rc = check_args(a, B, packed, true, what)) return rc;
  a.nchunks = chunk_slots(B, T, nseq, packed);
  UTTT_REQUIRE(T == 0 || (u_saved && s_saved && dout && dq && dk && dv && dg && dbeta), "%s: null pointer", what);
  for (const void* p : {u_saved, s_saved, dout, (const void*)dq, (const void*)dk, (const void*)dv,
                        (const void*)workspace})
    UTTT_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15u) == 0, "%s: tensors must be 16-byte aligned", what);
  UTTT_REQUIRE(a.do_sb % 8 == 0 && a.do_st % 8 == 0 && a.do_sh % 8 == 0 && a.do_sb >= 0 && a.do_st >= 0 &&
                   a.do_sh >= 0 && a.do_st < (1 << 23),
               "%s: strides of the output's gradient are not multiples of 8, or too large", what);
  const Workspace w = workspace_of(B, T, nseq, Hk, Hv, Dk, Dv, packed, true);
  UTTT_REQUIRE(w.total == 0 || (workspace && workspace_bytes >= w.total),
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, w.total);
  bind_workspace(a, w, static_cast<uint8_t*>(workspace), packed, true);
  a.u = static_cast<float*>(const_cast<void*>(u_saved));
  a.s0 = static_cast<float*>(const_cast<void*>(s_saved));
  a.dout = static_cast<const uint16_t*>(dout);
  a.dhT = dfinal_state;
  a.dh0 = dinitial_state;
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.dg = dg;
  a.dbeta = dbeta;
  const hipStream_t st = as_stream(stream);
  if (packed)
    if (const int rc = launch_table(cu_seqlens, cu_is_int64, nseq, T, a.nchunks,
                                    const_cast<int4*>(a.table), const_cast<int4*>(a.seqs), st))
      return rc;
  if (a.nchunks > 0)
    if (const int rc = launch_prep(a, true, st)) return rc;
  UTTT_DELTA_STEPS(steps_of(Dk), KS, return launch_bwd<KS>(a, st));
  return UTTT_OK;
}
