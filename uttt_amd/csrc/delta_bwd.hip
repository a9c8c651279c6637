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
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

// The forward scan's division of work (delta_fwd.hip), from the last chunk to
// the first; a wave has 16 tokens of dU and dR and a quarter of dS's features.
template <int KS, int NT>
__global__ __launch_bounds__(256) void delta_scan_bwd_kernel(Args a) {
  constexpr int FT = (2 * KS + 3) / 4;
  __shared__ __attribute__((aligned(16))) uint8_t Sb[2][KS * NT * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t Gb[2 * NT * 1024];      // dO
  __shared__ __attribute__((aligned(16))) uint8_t Ub[2][2 * NT * 1024];   // dU
  __shared__ __attribute__((aligned(16))) uint8_t Hb[2][2 * NT * 1024];   // s gam dO
  __shared__ __attribute__((aligned(16))) uint8_t Eb[2][2 * NT * 1024];   // -b gam dR
  Scan s;
  if (!s.init(a, 16 * NT)) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int col = s.col0 + NT * r;
  const bool live = col < a.Dv;
  const uint32_t dead = miss_from(col, a.Dv);
  const uint32_t put = (r + 16 * (q >> 1)) * 16 + (q & 1) * 8;
  const uint32_t put_tok = (wave >> 1) * NT * 1024 + (wave & 1) * 512 + put;
  const auto put_tile = [&](uint8_t (*buf)[2 * NT * 1024], int n, const Parts& p) {
    *reinterpret_cast<u32x2*>(buf[0] + put_tok + n * 1024) = p.hi;
    *reinterpret_cast<u32x2*>(buf[1] + put_tok + n * 1024) = p.lo;
  };
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
        S[f][n][i] = a.dhT && live && feat < a.Dk
                         ? a.dhT[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] : 0.0f;
    }

  bf16x8 kf[KS], tf[2][2], pf[2][2], ktf[FT][2], qtf[FT][2];
  f32x4 gam, ge, bt;
  float gc;
  Cols<NT> gr[4];
  // Operands of the chunk before: pointers that go along, at first those of the last chunk.
  const int lastc = s.nc - 1;
  const int64_t crow = (int64_t)s.b * a.T + s.tok0 + (int64_t)lastc * kC;
  const uint16_t* kp = a.k + s.b * a.k_sb + s.hk * a.k_sh + (s.tok0 + (int64_t)lastc * kC) * a.k_st;
  const uint16_t* gp = a.dout + s.b * a.do_sb + s.hv * a.do_sh + (s.tok0 + (int64_t)lastc * kC) * a.do_st;
  const uint8_t* trip = a.tri + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kTriBytes;
  const int64_t trans_at = ((int64_t)(s.c0 + lastc) * a.Hk + s.hk) * (4 * KS * 1024);
  const uint8_t *ktp = a.kt + trans_at, *qtp = a.qt + trans_at;
  const float* scp = a.scal + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * kScal;
  const uint32_t krow = 2 * ((16 * wave + r) * (uint32_t)a.k_st + 8 * q);
  const uint32_t grow = 2 * ((16 * wave + 4 * q) * (uint32_t)a.do_st + col);
  const uint32_t orow = 2 * ((16 * wave + 4 * q) * (uint32_t)(a.Hv * a.Dv) + col);
  const uint32_t last_half = miss_from(32 * (KS - 1) + 8 * q, a.Dk), before_half = miss_from(32 * (KS - 2) + 8 * q, a.Dk);
  // `left`: tokens from the chunk on to the sequence's end; 0 before its first chunk
  const auto load_k = [&](int left) {
    const uint32_t miss = miss_from(16 * wave + r, left);
    const Rsrc kr = buffer_at(kp);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      kf[ks] = load_frag(kr, (krow + 64 * ks) | miss | (ks == KS - 1 ? last_half : ks == KS - 2 ? before_half : 0));
    ge = load_f4(buffer_at(scp), 4 * (16 * wave + 4 * q) | miss_from(0, left), 4 * kC);
    kp -= kC * a.k_st;
  };
  const auto load_do = [&](int left) {
    const Rsrc gr_ = buffer_at(gp);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      gr[i].load(gr_, (grow + 2 * i * (uint32_t)a.do_st) | dead | miss_from(16 * wave + 4 * q + i, left));
    gp -= kC * a.do_st;
  };
  const auto load_tri = [&](int left, int which, bf16x8 (&x)[2][2]) {
    const Rsrc tr = buffer_at(trip);
    const uint32_t at = lane * 16 | miss_from(0, left);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      // step 0 of the lower tiles is zero and not stored: step 1 again, unused
      const int f = 2 * which * kTFrags + upper_frag(wave, wave < 2 ? ks : 1);
      x[ks][0] = load_frag(tr, at, f * 1024);
      x[ks][1] = load_frag(tr, at, (kTFrags + f) * 1024);
    }
    if (!which) {
      const Rsrc sr = buffer_at(scp);
      const uint32_t s_at = 4 * (16 * wave + 4 * q) | miss_from(0, left);
      gam = load_f4(sr, s_at);
      bt = load_f4(sr, s_at, 8 * kC);
      gc = load_f1(sr, 4 * (kC - 1) | miss_from(0, left));
      scp -= a.Hv * kScal;
      trip -= (int64_t)a.Hv * kTriBytes;
    }
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
  // dS' to LDS and memory, dO to LDS
  uint16_t* dsp = a.ds + ((int64_t)(s.c0 + lastc) * a.Hv + s.hv) * 2 * a.Dk * a.Dv;
  const auto put_state = [&]() {
    const Rsrc sr = buffer_at(dsp);
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const int tile = wave * FT + f;
      if (tile < 2 * KS) {
        u32x2 hi[NT], lo[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const Parts p = parts_of(S[f][n]);
          const uint32_t at = ((tile >> 1) * NT + n) * 1024 + (tile & 1) * 512 + put;
          *reinterpret_cast<u32x2*>(Sb[0] + at) = hi[n] = p.hi;
          *reinterpret_cast<u32x2*>(Sb[1] + at) = lo[n] = p.lo;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int feat = 16 * tile + 4 * q + i;
          const uint32_t at = 2 * (feat * a.Dv + col) | dead | miss_from(feat, a.Dk);
          store_row<NT>(sr, at, hi, i);
          store_row<NT>(sr, at, lo, i, 2 * (uint32_t)(a.Dk * a.Dv));
        }
      }
    }
    dsp -= (int64_t)a.Hv * 2 * a.Dk * a.Dv;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const u32x2 g = {gr[0].half(n) | (gr[1].half(n) << 16), gr[2].half(n) | (gr[3].half(n) << 16)};
      *reinterpret_cast<u32x2*>(Gb + put_tok + n * 1024) = g;
    }
  };

  const int first_left = s.len - lastc * kC;
  if (lastc >= 0) {
    load_do(first_left);
    load_k(first_left);
    load_tri(first_left, 1, pf);
    load_tri(first_left, 0, tf);
    load_trans(first_left, qtp, qtf);
    load_trans(first_left, ktp, ktf);
    put_state();
    settle();
  }
  const int64_t plane = (int64_t)a.B * a.T * a.Hv * a.Dv;
  int64_t out_at = (crow * a.Hv + s.hv) * a.Dv;
  for (int c = lastc; c >= 0; --c) {
    const int left = s.len - c * kC, next = c > 0 ? kC : 0;
    lds_barrier();   // dS' and dO are in LDS
    // dU = e^{G_C - G} K dS' + P^T dO
    {
      f32x4 X[NT] = {}, X2[NT] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          X[n] = mfma(kf[ks], get(Sb[0], ks * NT + n), X[n]);
          X2[n] = mfma(kf[ks], get(Sb[1], ks * NT + n), X2[n]);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        X[n] = ge * (X[n] + X2[n]);
        X2[n] = f32x4{};
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (ks >= wave >> 1)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bf16x8 g = get(Gb, ks * NT + n);
            X[n] = mfma(pf[ks][0], g, X[n]);
            X2[n] = mfma(pf[ks][1], g, X2[n]);
          }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        put_tile(Ub, n, parts_of(X[n] + X2[n]));
        f32x4 g;
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = gr[i].get(n);
        put_tile(Hb, n, parts_of(g * (gam * a.scale)));
      }
    }
    load_do(next);
    load_k(next);
    load_tri(next, 1, pf);
    lds_barrier();   // dU and s gam dO are in LDS
    f32x4 R[NT] = {};   // dR = T^T dU
    {
      f32x4 R2[NT] = {};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (ks >= wave >> 1)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bf16x8 hi = get(Ub[0], ks * NT + n), lo = get(Ub[1], ks * NT + n);
            R[n] = mfma(tf[ks][0], hi, R[n]);
            R2[n] = mfma(tf[ks][1], hi, R2[n]);
            R2[n] = mfma(tf[ks][0], lo, R2[n]);
          }
#pragma unroll
      for (int n = 0; n < NT; ++n) R[n] += R2[n];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) put_tile(Eb, n, parts_of(-(bt * gam) * R[n]));
    // dS0 = gam_C dS' + Q^T (s gam dO) - K^T (b gam dR): the first product here
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int n = 0; n < NT; ++n) S[f][n] *= gc;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8 hi = get(Hb[0], t * NT + n), lo = get(Hb[1], t * NT + n);
#pragma unroll
        for (int f = 0; f < FT; ++f)
          if (wave * FT + f < 2 * KS) {
            S[f][n] = mfma(qtf[f][t], hi, S[f][n]);
            S[f][n] = mfma(qtf[f][t], lo, S[f][n]);
          }
      }
    load_trans(next, qtp, qtf);
    {
      const Rsrc vr = buffer_at(a.dv + out_at), hr = buffer_at(a.dr + out_at), lr = buffer_at(a.dr + plane + out_at);
      u32x2 v[NT], hi[NT], lo[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const Parts p = parts_of(R[n]);
        hi[n] = p.hi;
        lo[n] = p.lo;
        v[n] = round_of(bt * R[n]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = (orow + 2 * i * (uint32_t)(a.Hv * a.Dv)) | dead | miss_from(16 * wave + 4 * q + i, left);
        store_row<NT>(vr, at, v, i);
        store_row<NT>(hr, at, hi, i);
        store_row<NT>(lr, at, lo, i);
      }
      out_at -= (int64_t)kC * a.Hv * a.Dv;
    }
    load_tri(next, 0, tf);
    lds_barrier();   // b gam dR is in LDS
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8 hi = get(Eb[0], t * NT + n), lo = get(Eb[1], t * NT + n);
#pragma unroll
        for (int f = 0; f < FT; ++f)
          if (wave * FT + f < 2 * KS) {
            S[f][n] = mfma(ktf[f][t], hi, S[f][n]);
            S[f][n] = mfma(ktf[f][t], lo, S[f][n]);
          }
      }
    load_trans(next, ktp, ktf);
    if (c > 0) put_state();
  }
  if (a.dh0 && live) {
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

// One chunk of one key head, its value heads one after another so that the
// shared gradients of q and k are added in registers, in a fixed order.  NW
// waves: each has FT 16-feature tiles of the [64, Dk] products, and a 16-token
// row tile with CT column tiles of the [64, 64] ones.  The rows of dO, dR and U
// pass through LDS 32 columns at a time (every wave reads all of them), loaded
// a step ahead; S0 and dS' go straight to the wave that has their features.
template <int KS, int NW>
__global__ __launch_bounds__(64 * NW) void delta_grads_kernel(Args a) {
  constexpr int LD = 32 * KS + 8, FT = (2 * KS + NW - 1) / NW, CT = 16 / NW, LX = kC + 4, LM = kC + 8;
  constexpr int kThreads = 64 * NW, kStage = 5 * 4 * 1024;   // dO, dR hi, lo, U hi, lo: 4 fragments each
  constexpr int kMats = kC * LX * 4 + 3 * kC * LM * 2;
  __shared__ __attribute__((aligned(16))) uint16_t Kl[kC * LD];
  __shared__ __attribute__((aligned(16))) uint16_t Ql[kC * LD];
  __shared__ __attribute__((aligned(16))) uint8_t buf[kMats > 2 * kStage ? kMats : 2 * kStage];
  __shared__ __attribute__((aligned(16))) float Sc[kScal];
  __shared__ float rows[3][NW][kC];   // per wave: q.(S0 dO), k.(S0 dR), k.(dS' U)
  __shared__ float bsum[NW][16], zsum[NW][kC], rvs[kC], dots[NW];
  float* Xl = reinterpret_cast<float*>(buf);
  __bf16* Dl = reinterpret_cast<__bf16*>(buf + kC * LX * 4);   // D, D^T, M + M^T
  __bf16* DTl = Dl + kC * LM;
  __bf16* Nl = DTl + kC * LM;
  const int c = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk;
  const Chunk ch = chunk_of(a, c);
  if (ch.seq < 0) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int rw = wave & 3, cw = (wave >> 2) * CT;   // the wave's row tile, first column tile
  const int group = a.Hv / a.Hk;
  {
    const Rsrc kp = buffer_at(a.k + ch.b * a.k_sb + ch.t0 * a.k_st + hk * a.k_sh);
    const Rsrc qp = buffer_at(a.q + ch.b * a.q_sb + ch.t0 * a.q_st + hk * a.q_sh);
    for (int p = tid; p < kC * 4 * KS; p += kThreads) {
      const int t = p / (4 * KS), e = 8 * (p % (4 * KS));
      const uint32_t miss = miss_from(t, ch.n) | miss_from(e, a.Dk);
      *reinterpret_cast<bf16x8*>(Kl + t * LD + e) = load_frag(kp, 2 * (t * (uint32_t)a.k_st + e) | miss);
      *reinterpret_cast<bf16x8*>(Ql + t * LD + e) = load_frag(qp, 2 * (t * (uint32_t)a.q_st + e) | miss);
    }
  }
  __syncthreads();
  f32x4 kk[CT] = {}, qk[CT] = {};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = 32 * ks + 8 * q;
    const bf16x8 ka = *reinterpret_cast<const bf16x8*>(Kl + (16 * rw + r) * LD + e);
    const bf16x8 qa = *reinterpret_cast<const bf16x8*>(Ql + (16 * rw + r) * LD + e);
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const bf16x8 kb = *reinterpret_cast<const bf16x8*>(Kl + (16 * (cw + x) + r) * LD + e);
      kk[x] = mfma(ka, kb, kk[x]);
      qk[x] = mfma(qa, kb, qk[x]);
    }
  }
  f32x4 dQ[4][FT] = {}, dK[4][FT] = {};
  const int64_t orow = (int64_t)a.Hv * a.Dv, tok = (int64_t)ch.b * a.T + ch.t0;
  const int64_t plane = (int64_t)a.B * a.T * orow;
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    for (int i = tid; i < kScal; i += kThreads) Sc[i] = a.scal[((size_t)c * a.Hv + hv) * kScal + i];
    const int64_t oat = tok * orow + (int64_t)hv * a.Dv;
    const Rsrc src[5] = {buffer_at(a.dout + ch.b * a.do_sb + ch.t0 * a.do_st + hv * a.do_sh),
                         buffer_at(a.dr + oat), buffer_at(a.dr + plane + oat),
                         buffer_at(a.u + oat), buffer_at(a.u + plane + oat)};
    const Rsrc vp = buffer_at(a.v + ch.b * a.v_sb + ch.t0 * a.v_st + hv * a.v_sh);
    const int64_t sat = ((int64_t)c * a.Hv + hv) * 2 * a.Dk * a.Dv;
    const Rsrc sp = buffer_at(a.s0 + sat), dp = buffer_at(a.ds + sat);
    const uint32_t lo_at = 2 * (uint32_t)(a.Dk * a.Dv);
    // wave w stages fragments w, w + NW, ... of the 20 of a step
    constexpr int kMine = (20 + NW - 1) / NW;
    bf16x8 st[kMine], sh[FT], sl[FT], dh[FT], dl[FT], vf;
    const auto load_step = [&](int e0) {
      const int e = e0 + 8 * q;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int f = i * NW + wave;
        if (f < 20) {
          const int t = 16 * (f & 3) + r;
          const uint32_t ld = f < 4 ? (uint32_t)a.do_st : (uint32_t)orow;
          const Rsrc p = f < 4 ? src[0] : f < 8 ? src[1] : f < 12 ? src[2] : f < 16 ? src[3] : src[4];
          st[i] = load_frag(p, 2 * (t * ld + e) | miss_from(t, ch.n) | miss_from(e, a.Dv));
        }
      }
#pragma unroll
      for (int x = 0; x < FT; ++x) {
        const int feat = 16 * (wave * FT + x) + r;
        const uint32_t at = 2 * (feat * a.Dv + e) | miss_from(feat, a.Dk) | miss_from(e, a.Dv);
        sh[x] = load_frag(sp, at);
        sl[x] = load_frag(sp, at, lo_at);
        dh[x] = load_frag(dp, at);
        dl[x] = load_frag(dp, at, lo_at);
      }
      if (wave < 4) {
        const int t = 16 * rw + r;
        vf = load_frag(vp, 2 * (t * (uint32_t)a.v_st + e) | miss_from(t, ch.n) | miss_from(e, a.Dv));
      }
    };
    f32x4 EQ[4][FT] = {}, ER[4][FT] = {}, EU[4][FT] = {}, dP[CT] = {}, dA[CT] = {};
    float dot = 0.0f, rv = 0.0f;
    load_step(0);
    int half = 0;
    for (int e0 = 0; e0 < a.Dv; e0 += 32, half ^= 1) {
      uint8_t* stage = buf + half * kStage;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (i * NW + wave < 20)
          *reinterpret_cast<bf16x8*>(stage + (i * NW + wave) * 1024 + lane * 16) = st[i];
      bf16x8 s0h[FT], s0l[FT], dsh[FT], dsl[FT];
#pragma unroll
      for (int x = 0; x < FT; ++x) {
        s0h[x] = sh[x];
        s0l[x] = sl[x];
        dsh[x] = dh[x];
        dsl[x] = dl[x];
      }
      const bf16x8 vv = vf;
      load_step(e0 + 32);   // past Dv: nothing is read
      lds_barrier();        // the step's rows are in LDS; the other half is free after the next one
      const auto row = [&](int which, int rt) {
        return *reinterpret_cast<const bf16x8*>(stage + (4 * which + rt) * 1024 + lane * 16);
      };
#pragma unroll
      for (int x = 0; x < FT; ++x)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          dot = __builtin_fmaf((float)s0h[x][i] + (float)s0l[x][i], (float)dsh[x][i] + (float)dsl[x][i], dot);
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
        const bf16x8 g = row(0, rt), rh = row(1, rt), rl = row(2, rt), uh = row(3, rt), ul = row(4, rt);
#pragma unroll
        for (int x = 0; x < FT; ++x) {
          EQ[rt][x] = mfma(g, s0h[x], EQ[rt][x]);
          ER[rt][x] = mfma(rh, s0h[x], ER[rt][x]);
          EU[rt][x] = mfma(uh, dsh[x], EU[rt][x]);
          EQ[rt][x] = mfma(g, s0l[x], EQ[rt][x]);
          ER[rt][x] = mfma(rh, s0l[x], ER[rt][x]);
          EU[rt][x] = mfma(uh, dsl[x], EU[rt][x]);
          ER[rt][x] = mfma(rl, s0h[x], ER[rt][x]);
          EU[rt][x] = mfma(ul, dsh[x], EU[rt][x]);
        }
      }
      const bf16x8 gw = row(0, rw), rh = row(1, rw), rl = row(2, rw);
      if (wave < 4)
#pragma unroll
        for (int i = 0; i < 8; ++i) rv = __builtin_fmaf((float)rh[i] + (float)rl[i], (float)vv[i], rv);
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const bf16x8 uh = row(3, cw + x), ul = row(4, cw + x);
        dP[x] = mfma(gw, uh, dP[x]);
        dA[x] = mfma(rh, uh, dA[x]);
        dP[x] = mfma(gw, ul, dP[x]);
        dA[x] = mfma(rh, ul, dA[x]);
        dA[x] = mfma(rl, uh, dA[x]);
      }
    }
    lds_barrier();   // every wave is done with the staged rows
    rv += __shfl_xor(rv, 16);
    rv += __shfl_xor(rv, 32);
    if (wave < 4 && q == 0) rvs[16 * rw + r] = rv;   // dR.v
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) dot += __shfl_xor(dot, d);
    if (lane == 0) dots[wave] = dot;
    // the 64 x 64 matrices
    f32x4 bs = {};
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const int j = 16 * (cw + x) + r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * rw + 4 * q + i;
        const float E = row >= j ? __expf((Sc[3 * kC + row] - Sc[3 * kC + j]) +
                                          (Sc[4 * kC + row] - Sc[4 * kC + j])) : 0.0f;
        const float D = a.scale * E * dP[x][i];
        const float m = row > j ? -E * dA[x][i] : 0.0f;
        const float M = Sc[2 * kC + row] * m;
        bs[i] = __builtin_fmaf(m, kk[x][i], bs[i]);
        Xl[row * LX + j] = D * qk[x][i] + M * kk[x][i];
        Dl[row * LM + j] = (__bf16)D;
        DTl[j * LM + row] = (__bf16)D;
        if (row > j) {
          Nl[row * LM + j] = (__bf16)M;
          Nl[j * LM + row] = (__bf16)M;
        } else if (row == j) {
          Nl[row * LM + j] = (__bf16)0.0f;
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) bs[i] += __shfl_xor(bs[i], d);
    if (r == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) bsum[wave][4 * q + i] = bs[i];
    // the [64, Dk] products, and their rows' products with q and k
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
      const int t0 = 16 * rt + 4 * q;
      const f32x4 gam = *reinterpret_cast<const f32x4*>(Sc + t0);
      const f32x4 ge = *reinterpret_cast<const f32x4*>(Sc + kC + t0);
      const f32x4 bt = *reinterpret_cast<const f32x4*>(Sc + 2 * kC + t0);
      f32x4 s1 = {}, s2 = {}, s3 = {};
#pragma unroll
      for (int x = 0; x < FT; ++x) {
        const int f = wave * FT + x, feat = 16 * f + r;
        if (f < 2 * KS)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float kv = bf16_to_f32(Kl[(t0 + i) * LD + feat]);
            const float qv = bf16_to_f32(Ql[(t0 + i) * LD + feat]);
            s1[i] = __builtin_fmaf(EQ[rt][x][i], qv, s1[i]);
            s2[i] = __builtin_fmaf(ER[rt][x][i], kv, s2[i]);
            s3[i] = __builtin_fmaf(EU[rt][x][i], kv, s3[i]);
          }
        dQ[rt][x] += a.scale * gam * EQ[rt][x];
        dK[rt][x] += ge * EU[rt][x] - bt * gam * ER[rt][x];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          s1[i] += __shfl_xor(s1[i], d);
          s2[i] += __shfl_xor(s2[i], d);
          s3[i] += __shfl_xor(s3[i], d);
        }
        if (r == 0) {
          rows[0][wave][t0 + i] = s1[i];
          rows[1][wave][t0 + i] = s2[i];
          rows[2][wave][t0 + i] = s3[i];
        }
      }
    }
    __syncthreads();
    // sum_{j < t} X_ij as a product with the strictly upper ones, X in two bf16 parts
    f32x4 Z[CT] = {};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const float* xp = Xl + (16 * rw + r) * LX + 32 * ks + 8 * q;
      bf16x8 hi, lo;
      split8(*reinterpret_cast<const f32x4*>(xp), *reinterpret_cast<const f32x4*>(xp + 4), hi, lo);
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        bf16x8 ones;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          ones[i] = (__bf16)(32 * ks + 8 * q + i < 16 * (cw + x) + r ? 1.0f : 0.0f);
        Z[x] = mfma(hi, ones, Z[x]);
        Z[x] = mfma(lo, ones, Z[x]);
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
    // dQ += D K, dK += D^T Q + (M + M^T) K
#pragma unroll
    for (int x = 0; x < FT; ++x) {
      const int f = wave * FT + x;
      if (f < 2 * KS) {
        const size_t at = ((size_t)c * a.Hk + hk) * (4 * KS) * 1024 + (size_t)f * 2048 + lane * 16;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const bf16x8 kb = *reinterpret_cast<const bf16x8*>(a.kt + at + ks * 1024);
          const bf16x8 qb = *reinterpret_cast<const bf16x8*>(a.qt + at + ks * 1024);
#pragma unroll
          for (int rt = 0; rt < 4; ++rt) {
            const int o = (16 * rt + r) * LM + 32 * ks + 8 * q;
            if (ks == 0 || rt >= 2)
              dQ[rt][x] = mfma(*reinterpret_cast<const bf16x8*>(Dl + o), kb, dQ[rt][x]);
            if (ks == 1 || rt < 2)
              dK[rt][x] = mfma(*reinterpret_cast<const bf16x8*>(DTl + o), qb, dK[rt][x]);
            dK[rt][x] = mfma(*reinterpret_cast<const bf16x8*>(Nl + o), kb, dK[rt][x]);
          }
        }
      }
    }
    __syncthreads();
    if (wave == 0) {   // lane = token
      float s[3] = {};
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int w = 0; w < NW; ++w) s[i] += rows[i][w][lane];
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
      for (int w = 0; w < NW / 4; ++w) b += bsum[(lane >> 4) + 4 * w][lane & 15];
      if (lane < ch.n) {
        const int64_t at = (tok + lane) * a.Hv + hv;
        store_any(a.dg, a.g_dtype, at, z + suf + pre + Sc[kC - 1] * all);
        store_any(a.dbeta, a.beta_dtype, at, rvs[lane] - gam * s[1] + b);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int rt = 0; rt < 4; ++rt)
#pragma unroll
    for (int x = 0; x < FT; ++x) {
      const int feat = 16 * (wave * FT + x) + r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * rt + 4 * q + i;
        if (t < ch.n && feat < a.Dk) {
          const int64_t at = ((tok + t) * a.Hk + hk) * a.Dk + feat;
          a.dq[at] = f32_to_bf16(dQ[rt][x][i]);
          a.dk[at] = f32_to_bf16(dK[rt][x][i]);
        }
      }
    }
}

template <int KS>
int launch_bwd(const Args& a, hipStream_t st) {
  switch (scan_tiles(a)) {
    case 1:
      hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 1>), dim3(scan_blocks(a, 16)), dim3(256), 0, st, a);
      break;
    case 2:
      hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 2>), dim3(scan_blocks(a, 32)), dim3(256), 0, st, a);
      break;
    default:
      hipLaunchKernelGGL((delta_scan_bwd_kernel<KS, 4>), dim3(scan_blocks(a, 64)), dim3(256), 0, st, a);
  }
  if (const int rc = check_launch("delta_scan_bwd")) return rc;
  if (a.nchunks == 0) return UTTT_OK;
  constexpr int NW = KS == 2 ? 4 : 8;
  hipLaunchKernelGGL((delta_grads_kernel<KS, NW>), dim3((unsigned)((int64_t)a.nchunks * a.Hk)), dim3(64 * NW),
                     0, st, a);
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
  if (const int rc = check_args(a, B, packed, what)) return rc;
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
  a.u = static_cast<uint16_t*>(const_cast<void*>(u_saved));
  a.s0 = static_cast<uint16_t*>(const_cast<void*>(s_saved));
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
