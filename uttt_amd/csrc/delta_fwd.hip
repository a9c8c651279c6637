// Forward of the chunked gated delta rule: the scan over each sequence's
// chunks (formulas, precision and fragment layout in delta.h).
//
// A workgroup owns 16 NT value columns of one head of one sequence and walks
// its chunks in order, with two kinds of waves.  Four have the tokens, 16 each:
// X = K S0 and R = b (V - gam X), then O = s gam Q S0 + P U.  Four have the
// state: U = T R, 16 tokens each, and S' = gam_C S0 + K^T (e^{G_C - G} U), a
// quarter of the features each, which stay in registers from the first chunk to
// the last.  The chain R, U, S' bounds a chunk, so what is off it stands where
// the other kind works on it: the state's waves load the next chunk's operands
// and store what a backward will read while R is made, the others have Q S0
// while U is made and P U while S' is.  An operand fragment (K, Q, T, P, K^T) is
// read by one wave, straight into its registers and a chunk ahead; S, R and U
// pass through LDS, from the wave that made them to all: three barriers a chunk.
//
// Values that are not finite.  U = T R and P U multiply the zeros above the
// diagonal with later tokens' R and U, and a zero by an infinity is NaN.  So an R
// that is not finite goes in as zero, and what becomes of it is put in behind the
// products: NaN in its column from its token on, in the outputs, in U as saved
// and in what goes to the state.  With ordinary values that is one test of R and
// two of a flag a chunk (one sequence of 8192 tokens, 16 heads of 64 by 64, whose
// chunks are the shortest: scan 105 -> 113 us with operands in two parts; other
// scans 0 to 1 %).
//
// Measured: one sequence of 4096 tokens, 4 heads of 192 by 192, 97 us (1.5 us a
// chunk); 16 x 2048 tokens, 12 heads of 128 by 128, with U and S0 stored for a
// backward, 383 us: 0.7 GB of stores and 0.6 GB of loads at 3.4 TB/s (a copy
// reaches 5.1).  The third part of the operands is 15 to 20 % of a scan that a
// chunk's chain bounds: with two 80 us and 348.  With T and K^T loaded where their
// last value was used, not a whole chunk ahead, the first takes 15 us more.
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

// LDS of a scan's workgroup: operand fragments (32 contracted rows x 16
// columns, 1 KiB) of each bf16 part.
template <int KS, int NT>
struct ScanLds {
  uint8_t S[3][KS * NT * 1024];
  uint8_t R[3][2 * NT * 1024];
  uint8_t U[2][2 * NT * 1024];
  uint8_t E[3][2 * NT * 1024];   // e^{G_C - G} U
  int first[NT][16];             // a column's first token in the chunk whose R is not finite
  int bad;                       // whether there is one
};

// NaN in rows from `first` on.
__device__ __forceinline__ void spoil(f32x4& x, int row, int first) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (row + i >= first) x[i] = __builtin_nanf("");
}

// What both kinds of waves know of their place.
struct Lane {
  int wave, lane, r, q, col;   // wave: its row tile; col: the lane's first column
  uint32_t dead;               // kNoRow where the column is none
  uint32_t last_half, before_half;   // kNoRow where the last two steps' features are none
};

// The state's waves: U = T R and S' = gam_C S0 + K^T (e^{G_C - G} U).  While the
// others work on R they load the next chunk's operands and store what a
// backward will read.
template <int KS, int NT, bool SAVE>
__device__ __forceinline__ void scan_state(const Args& a, const Scan& s, const Lane& l, ScanLds<KS, NT>& lds) {
  constexpr int FT = (2 * KS + 3) / 4;   // 16-feature tiles of a wave
  const int wave = l.wave, r = l.r, q = l.q, col = l.col;
  const uint32_t dead = l.dead;
  const uint32_t put = (r + 16 * (q >> 1)) * 16 + (q & 1) * 8;   // 4 rows of a tile in a fragment
  const uint32_t put_tok = (wave >> 1) * NT * 1024 + (wave & 1) * 512 + put;
  const auto get = [&](const uint8_t* buf, int f) {
    return *reinterpret_cast<const bf16x8*>(buf + f * 1024 + l.lane * 16);
  };

  f32x4 S[FT][NT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int feat = 16 * (wave * FT + f) + 4 * q + i;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        S[f][n][i] = a.h0 && col < a.Dv && feat < a.Dk
                         ? a.h0[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] : 0.0f;
    }

  // Operands of this chunk, and of the next on their way.  With 64 accumulators
  // a lane there are no registers for K^T twice: it is then loaded for this
  // chunk while R is made.
  constexpr bool kAhead = FT * NT < 16;
  struct Ops {
    bf16x8 t[2][3], kt[FT][2];
    f32x4 ge;
    float gc;
  };
  Ops now, coming;
  const uint8_t* trip = a.tri + ((size_t)s.c0 * a.Hv + s.hv) * kTriBytes;
  const uint8_t* ktp = a.kt + ((size_t)s.c0 * a.Hk + s.hk) * (4 * KS * 1024);
  const float* scp = a.scal + ((size_t)s.c0 * a.Hv + s.hv) * kScal;
  const auto load = [&](int left, Ops& o) {
    const uint32_t none = miss_from(0, left), at = l.lane * 16 | none;
    const Rsrc tr = buffer_at(trip), sr = buffer_at(scp);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      // step 1 of the upper tiles is zero and not stored: step 0 again, unused
      const int f = lower_frag(wave, wave < 2 ? 0 : ks);
#pragma unroll
      for (int k = 0; k < 3; ++k) o.t[ks][k] = load_frag(tr, at, (k * kTFrags + f) * 1024);
    }
    o.ge = load_f4(sr, 4 * (16 * wave + 4 * q) | none, 4 * kC);
    o.gc = load_f1(sr, 4 * (kC - 1) | none);
    trip += (size_t)a.Hv * kTriBytes;
    scp += a.Hv * kScal;
  };
  const auto load_kt = [&](int left, Ops& o) {
    const uint32_t at = l.lane * 16 | miss_from(0, left);
    const Rsrc kr = buffer_at(ktp);
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (wave * FT + f < 2 * KS) o.kt[f][t] = load_frag(kr, at, (2 * (wave * FT + f) + t) * 1024);
    ktp += (size_t)a.Hk * (4 * KS * 1024);
  };
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
  float* s0p = SAVE ? a.s0 + ((int64_t)s.c0 * a.Hv + s.hv) * a.Dk * a.Dv : nullptr;
  const auto save_state = [&]() {
    const Rsrc sr = buffer_at(s0p);
#pragma unroll
    for (int f = 0; f < FT; ++f)
      if (wave * FT + f < 2 * KS)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int feat = 16 * (wave * FT + f) + 4 * q + i;
          store_row<NT>(sr, 4 * (feat * a.Dv + col) | dead | miss_from(feat, a.Dk), S[f], i);
        }
    s0p += (int64_t)a.Hv * a.Dk * a.Dv;
  };
  const int64_t token = (int64_t)a.Hv * a.Dv;
  float* up = SAVE ? a.u + ((int64_t)s.b * a.T + s.tok0 + 16 * wave) * token + s.hv * a.Dv : nullptr;
  const auto save_u = [&](const f32x4 (&U)[NT], int left) {
    const Rsrc ur = buffer_at(up);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store_row<NT>(ur, 4 * ((4 * q + i) * (uint32_t)token + col) | dead | miss_from(16 * wave + 4 * q + i, left), U, i);
    up += kC * token;
  };

  if (s.len > 0) {
    load(s.len, coming);
    if constexpr (kAhead) load_kt(s.len, coming);
    put_state();
    settle();
  }
  for (int left = s.len; left > 0; left -= kC) {
    lds_barrier();   // S0 is in LDS
    now = coming;
    if constexpr (!kAhead) load_kt(left, now);
    load(left - kC, coming);
    if constexpr (kAhead) load_kt(left - kC, coming);
    if constexpr (SAVE) save_state();
    lds_barrier();   // R is in LDS
    int bad = lds.bad;
    f32x4 U[NT] = {};
    {
      f32x4 U2[NT] = {}, U3[NT] = {};   // the products below 2^-7, below 2^-15 of the first
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (ks <= wave >> 1)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bf16x8 r1 = get(lds.R[0], ks * NT + n), r2 = get(lds.R[1], ks * NT + n), r3 = get(lds.R[2], ks * NT + n);
            U[n] = mfma(now.t[ks][0], r1, U[n]);
            U2[n] = mfma(now.t[ks][1], r1, U2[n]);
            U3[n] = mfma(now.t[ks][2], r1, U3[n]);
            U2[n] = mfma(now.t[ks][0], r2, U2[n]);
            U3[n] = mfma(now.t[ks][1], r2, U3[n]);
            U3[n] = mfma(now.t[ks][0], r3, U3[n]);
          }
      asm volatile("" : "+v"(bad));   // read with R, not when U is made
#pragma unroll
      for (int n = 0; n < NT; ++n) U[n] += U2[n] + U3[n];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const Parts p = parts_of(U[n]);
      *reinterpret_cast<u32x2*>(lds.U[0] + put_tok + n * 1024) = p.hi;
      *reinterpret_cast<u32x2*>(lds.U[1] + put_tok + n * 1024) = p.lo;
    }
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(bad), 0))
#pragma unroll
      for (int n = 0; n < NT; ++n) spoil(U[n], 16 * wave + 4 * q, lds.first[n][r]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const Parts3 p = parts3_of(now.ge * U[n]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.E[k] + put_tok + n * 1024) = p.p[k];
    }
    lds_barrier();   // U is in LDS
    // S' = gam_C S0 + K^T (e^{G_C - G} U)
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int n = 0; n < NT; ++n) S[f][n] *= now.gc;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const bf16x8 e = get(lds.E[k], t * NT + n);
#pragma unroll
          for (int f = 0; f < FT; ++f)
            if (wave * FT + f < 2 * KS) S[f][n] = mfma(now.kt[f][t], e, S[f][n]);
        }
      }
    if (left > kC) put_state();
    if constexpr (SAVE) save_u(U, left);
  }
  if (a.hT && col < a.Dv) {
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int feat = 16 * (wave * FT + f) + 4 * q + i;
        if (feat < a.Dk)
#pragma unroll
          for (int n = 0; n < NT; ++n) a.hT[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] = S[f][n][i];
      }
  }
}

// The tokens' waves: R = b (V - gam K S0) and O = s gam Q S0 + P U.
template <int KS, int NT>
__device__ __forceinline__ void scan_tokens(const Args& a, const Scan& s, const Lane& l, ScanLds<KS, NT>& lds) {
  // With one tile there are registers to read S0's first two parts from LDS once
  // for both products (4096 tokens, 4 heads of 192, with two parts: 85 -> 79 us).
  constexpr bool kHold = NT == 1;
  constexpr int kHeld = kHold ? KS : 1;
  const int wave = l.wave, q = l.q;
  const uint32_t put_tok = (wave >> 1) * NT * 1024 + (wave & 1) * 512 + (l.r + 16 * (q >> 1)) * 16 + (q & 1) * 8;
  const auto get = [&](const uint8_t* buf, int f) {
    return *reinterpret_cast<const bf16x8*>(buf + f * 1024 + l.lane * 16);
  };
  bf16x8 kf[KS], qf[KS], pf[2][2];
  f32x4 gam, bt;
  Cols<NT> vr[4];
  // Operands of the next chunk: pointers that go along, per-lane offsets that
  // stay, and the bit that masks rows past the sequence.  Each is loaded where
  // its last value was used, in the order of use, which is the order in which
  // loads are waited for.
  // K and Q: rows of the caller's tensors, or their fragments (delta_prep.hip)
  const bool copies = a.kf != nullptr;
  const int64_t copy_at = ((int64_t)s.c0 * a.Hk + s.hk) * (4 * KS * 1024), copy_step = (int64_t)a.Hk * (4 * KS * 1024);
  const uint8_t* kp = copies ? a.kf + copy_at
                             : reinterpret_cast<const uint8_t*>(a.k + s.b * a.k_sb + s.hk * a.k_sh + s.tok0 * a.k_st);
  const uint8_t* qp = copies ? a.qf + copy_at
                             : reinterpret_cast<const uint8_t*>(a.q + s.b * a.q_sb + s.hk * a.q_sh + s.tok0 * a.q_st);
  const int64_t k_step = copies ? copy_step : 2 * kC * a.k_st, q_step = copies ? copy_step : 2 * kC * a.q_st;
  const uint32_t in_copy = wave * KS * 1024 + l.lane * 16, along = copies ? 1024 : 64;
  const uint32_t krow = copies ? in_copy : 2 * ((16 * wave + l.r) * (uint32_t)a.k_st + 8 * q);
  const uint32_t qrow = copies ? in_copy : 2 * ((16 * wave + l.r) * (uint32_t)a.q_st + 8 * q);
  const uint16_t* vp = a.v + s.b * a.v_sb + s.hv * a.v_sh + s.tok0 * a.v_st;
  const uint8_t* trip = a.tri + ((size_t)s.c0 * a.Hv + s.hv) * kTriBytes;
  const float* scp = a.scal + ((size_t)s.c0 * a.Hv + s.hv) * kScal;
  uint16_t* op = a.o + (((int64_t)s.b * a.T + s.tok0) * a.Hv + s.hv) * a.Dv;
  const uint32_t vrow = 2 * ((16 * wave + 4 * q) * (uint32_t)a.v_st + l.col);
  const uint32_t orow = 2 * ((16 * wave + 4 * q) * (uint32_t)(a.Hv * a.Dv) + l.col);
  const auto half_miss = [&](int ks) { return ks == KS - 1 ? l.last_half : ks == KS - 2 ? l.before_half : 0; };
  const auto load_k = [&](int left) {
    const uint32_t miss = miss_from(16 * wave + l.r, left), at = 4 * (16 * wave + 4 * q) | miss_from(0, left);
    const Rsrc kr = buffer_at(kp), vr_ = buffer_at(vp), sr = buffer_at(scp);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = load_frag(kr, krow | miss | half_miss(ks), along * ks);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      vr[i].load(vr_, (vrow + 2 * i * (uint32_t)a.v_st) | l.dead | miss_from(16 * wave + 4 * q + i, left));
    gam = load_f4(sr, at);
    bt = load_f4(sr, at, 8 * kC);
    kp += k_step;
    vp += kC * a.v_st;
    scp += a.Hv * kScal;
  };
  const auto load_q = [&](int left) {
    const uint32_t miss = miss_from(16 * wave + l.r, left);
    const Rsrc qr = buffer_at(qp);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_frag(qr, qrow | miss | half_miss(ks), along * ks);
    qp += q_step;
  };
  const auto load_p = [&](int left) {
    const Rsrc tr = buffer_at(trip);
    const uint32_t at = l.lane * 16 | miss_from(0, left);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int f = kPFrag + lower_frag(wave, wave < 2 ? 0 : ks);
      pf[ks][0] = load_frag(tr, at, f * 1024);
      pf[ks][1] = load_frag(tr, at, (kTFrags + f) * 1024);
    }
    trip += (size_t)a.Hv * kTriBytes;
  };
  if (s.len > 0) {
    load_k(s.len);
    load_q(s.len);
    load_p(s.len);
    settle();
  }
  for (int left = s.len; left > 0; left -= kC) {
    lds_barrier();   // S0 is in LDS
    bf16x8 held[kHeld][2];
    const auto state = [&](int part, int f) { return kHold ? held[f < kHeld ? f : 0][part] : get(lds.S[part], f); };
    if constexpr (kHold) {
#pragma unroll
      for (int f = 0; f < kHeld; ++f) {
        held[f][0] = get(lds.S[0], f);
        held[f][1] = get(lds.S[1], f);
      }
    }
    {
      f32x4 X[NT] = {}, X2[NT] = {}, X3[NT] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          X[n] = mfma(kf[ks], state(0, ks * NT + n), X[n]);
          X2[n] = mfma(kf[ks], state(1, ks * NT + n), X2[n]);
          X3[n] = mfma(kf[ks], get(lds.S[2], ks * NT + n), X3[n]);
        }
      // rows behind the sequence's end have b = 0 and V = 0
      f32x4 zero = {};   // NaN where some value is not finite
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = vr[i].get(n);
        X[n] = bt * (v - gam * (X[n] + (X2[n] + X3[n])));
        const Parts3 p = parts3_of(X[n]);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(lds.R[k] + put_tok + n * 1024) = p.p[k];
        zero += X[n] * 0.0f;
      }
      if (__builtin_expect(__any((zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.0f), 0)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (X[n][i] * 0.0f != 0.0f) {
#pragma unroll
              for (int k = 0; k < 3; ++k) *reinterpret_cast<uint16_t*>(lds.R[k] + put_tok + n * 1024 + 2 * i) = 0;
              atomicMin(&lds.first[n][l.r], 16 * wave + 4 * q + i);
            }
        lds.bad = 1;
      }
    }
    const f32x4 sgam = gam * a.scale;
    lds_barrier();   // R is in LDS
    int next = left - kC;
    asm volatile("" : "+s"(next));   // offsets of the next loads: here, not in front of the barrier
    load_k(next);
    f32x4 O[NT] = {}, O2[NT] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        O[n] = mfma(qf[ks], state(0, ks * NT + n), O[n]);
        O2[n] = mfma(qf[ks], state(1, ks * NT + n), O2[n]);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      O[n] = (O[n] + O2[n]) * sgam;
      O2[n] = f32x4{};
    }
    lds_barrier();   // U is in LDS, and nobody reads S0 any more
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (ks <= wave >> 1)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 hi = get(lds.U[0], ks * NT + n), lo = get(lds.U[1], ks * NT + n);
          O[n] = mfma(pf[ks][0], hi, O[n]);
          O2[n] = mfma(pf[ks][1], hi, O2[n]);
          O2[n] = mfma(pf[ks][0], lo, O2[n]);
        }
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(lds.bad), 0))
#pragma unroll
      for (int n = 0; n < NT; ++n) spoil(O[n], 16 * wave + 4 * q, lds.first[n][l.r]);
    load_q(next);
    load_p(next);
    const Rsrc orsrc = buffer_at(op);
    u32x2 ow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) ow[n] = round_of(O[n] + O2[n]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store_row<NT>(orsrc, (orow + 2 * i * (uint32_t)(a.Hv * a.Dv)) | l.dead | miss_from(16 * wave + 4 * q + i, left), ow, i);
    op += (int64_t)kC * a.Hv * a.Dv;
  }
}

// The smallest variants keep to the 128 registers with which two workgroups
// share a CU.
template <int KS, int NT, bool SAVE>
__global__ __launch_bounds__(512, KS * NT <= 2 ? 4 : 2) void delta_scan_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) ScanLds<KS, NT> lds;
  Scan s;
  if (!s.init(a, 16 * NT)) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4, col = s.col0 + NT * r;
  if (wave == 4 && q == 0) {   // one of the waves that write it
#pragma unroll
    for (int n = 0; n < NT; ++n) lds.first[n][r] = kC;
    lds.bad = 0;
  }
  const Lane l{wave & 3, lane, r, q, col, miss_from(col, a.Dv), miss_from(32 * (KS - 1) + 8 * q, a.Dk),
               miss_from(32 * (KS - 2) + 8 * q, a.Dk)};
  if (wave < 4) scan_state<KS, NT, SAVE>(a, s, l, lds);
  else scan_tokens<KS, NT>(a, s, l, lds);
}

template <int KS, int NT>
void launch_scan_as(const Args& a, hipStream_t st) {
  const dim3 grid((unsigned)scan_blocks(a, 16 * NT));
  if (a.s0) hipLaunchKernelGGL((delta_scan_kernel<KS, NT, true>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((delta_scan_kernel<KS, NT, false>), grid, dim3(512), 0, st, a);
}

int launch_scan(const Args& a, hipStream_t st) {
  UTTT_DELTA_STEPS(steps_of(a.Dk), KS, switch (scan_tiles(a, false)) {
    case 1: launch_scan_as<KS, 1>(a, st); break;
    case 2: launch_scan_as<KS, 2>(a, st); break;
    default: if constexpr (scan_widest(KS, false) == 4) launch_scan_as<KS, 4>(a, st);
  });
  return check_launch("delta_scan");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int check_args(const Args& a, int B, bool packed, bool backward, const char* what) {
  UTTT_REQUIRE(B >= 1 && a.T >= 0 && a.nseq >= 1 && a.Hk >= 1 && a.Hv >= 1,
               "%s: bad sizes B=%d T=%d sequences=%d Hk=%d Hv=%d", what, B, a.T, a.nseq, a.Hk, a.Hv);
  UTTT_REQUIRE(a.Hv % a.Hk == 0, "%s: Hv=%d must be a multiple of Hk=%d", what, a.Hv, a.Hk);
  UTTT_REQUIRE(a.Dk >= 8 && a.Dk <= 256 && a.Dk % 8 == 0, "%s: Dk=%d must be a multiple of 8 up to 256",
               what, a.Dk);
  UTTT_REQUIRE(a.Dv >= 8 && a.Dv <= 65536 && a.Dv % 8 == 0,
               "%s: Dv=%d must be a multiple of 8 up to 65536", what, a.Dv);
  UTTT_REQUIRE(packed ? B == 1 : a.nseq == B, "%s: %d sequences in a batch of %d", what, a.nseq, B);
  const int64_t slots = chunk_slots(B, a.T, a.nseq, packed);
  // a launch has fewer than 2^32 threads: of a chunk and key head (operands,
  // gradients), of a workgroup of the scans
  const int64_t chunk = backward && steps_of(a.Dk) > 2 ? 128 * steps_of(a.Dk) : 256;
  const int64_t scans = scan_blocks(a, 16 * scan_tiles(a.T, a.nseq, a.Hv, a.Dk, a.Dv, packed, backward, backward));
  UTTT_REQUIRE(slots >= 0 && slots * a.Hv < (1LL << 31) && slots * a.Hk * chunk < (1LL << 32) &&
                   scans * 512 < (1LL << 32),
               "%s: too many chunks and heads for one launch", what);
  UTTT_REQUIRE(a.T == 0 || (a.q && a.k && a.v && a.g && a.beta), "%s: null pointer", what);
  UTTT_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v), "%s: q, k and v must be 16-byte aligned",
               what);
  for (const int64_t s : {a.q_sb, a.q_st, a.q_sh, a.k_sb, a.k_st, a.k_sh, a.v_sb, a.v_st, a.v_sh})
    UTTT_REQUIRE(s % 8 == 0 && s >= 0, "%s: stride %lld of q, k or v is not a multiple of 8", what,
                 (long long)s);
  // a chunk's rows are addressed by 31-bit byte offsets
  for (const int64_t s : {a.q_st, a.k_st, a.v_st, (int64_t)a.Hv * a.Dv})
    UTTT_REQUIRE(s < (1 << 23), "%s: %lld elements from token to token, at most 2^23 are built", what,
                 (long long)s);
  for (const int dt : {a.g_dtype, a.beta_dtype})
    UTTT_REQUIRE(dtype_bytes(dt) != 0, "%s: dtype code %d", what, dt);
  return UTTT_OK;
}

}  // namespace delta
}  // namespace uttt

using namespace uttt;
using namespace uttt::delta;

extern "C" size_t uttt_gated_delta_workspace_bytes(int B, int T, int nseq, int Hk, int Hv, int Dk,
                                                   int Dv, int packed, int backward) {
  if (B < 1 || T < 0 || nseq < 1 || Hk < 1 || Hv < 1 || Dk < 1 || Dk > 256 || Dv < 1 ||
      chunk_slots(B, T, nseq, packed != 0) < 0)
    return 0;
  return workspace_of(B, T, nseq, Hk, Hv, Dk, Dv, packed != 0, backward != 0).total;
}

extern "C" int uttt_gated_delta_chunks(int B, int T, int nseq, int packed) {
  return B < 1 || T < 0 || nseq < 1 ? -1 : chunk_slots(B, T, nseq, packed != 0);
}

extern "C" int uttt_gated_delta_fwd(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, const void* g, int g_dtype,
                                    const void* beta, int beta_dtype, const void* cu_seqlens,
                                    int cu_is_int64, int B, int T, int nseq, int Hk, int Hv, int Dk,
                                    int Dv, float scale, const float* initial_state, void* out,
                                    float* final_state, void* u_saved, void* s_saved,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "uttt_gated_delta_fwd";
  UTTT_REQUIRE(q_strides && k_strides && v_strides, "%s: null strides", what);
  const bool packed = cu_seqlens != nullptr;
  Args a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_sb = q_strides[0]; a.q_st = q_strides[1]; a.q_sh = q_strides[2];
  a.k_sb = k_strides[0]; a.k_st = k_strides[1]; a.k_sh = k_strides[2];
  a.v_sb = v_strides[0]; a.v_st = v_strides[1]; a.v_sh = v_strides[2];
  a.g = g; a.beta = beta; a.g_dtype = g_dtype; a.beta_dtype = beta_dtype;
  a.B = B; a.T = T; a.Hk = Hk; a.Hv = Hv; a.Dk = Dk; a.Dv = Dv; a.nseq = nseq;
  a.cps = (T + kC - 1) / kC;
  a.scale = scale;
  if (const int rc = check_args(a, B, packed, false, what)) return rc;
  a.nchunks = chunk_slots(B, T, nseq, packed);
  UTTT_REQUIRE(out || T == 0, "%s: null output", what);
  UTTT_REQUIRE(aligned16(out) && aligned16(u_saved) && aligned16(s_saved) && aligned16(workspace),
               "%s: tensors must be 16-byte aligned", what);
  UTTT_REQUIRE(T == 0 || (u_saved == nullptr) == (s_saved == nullptr), "%s: save both U and S or neither", what);
  const Workspace w = workspace_of(B, T, nseq, Hk, Hv, Dk, Dv, packed, false);
  UTTT_REQUIRE(w.total == 0 || (workspace && workspace_bytes >= w.total),
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, w.total);
  bind_workspace(a, w, static_cast<uint8_t*>(workspace), packed, false);
  a.h0 = initial_state;
  a.hT = final_state;
  a.o = static_cast<uint16_t*>(out);
  a.u = static_cast<float*>(u_saved);
  a.s0 = static_cast<float*>(s_saved);
  const hipStream_t st = as_stream(stream);
  if (packed)
    if (const int rc = launch_table(cu_seqlens, cu_is_int64, nseq, T, a.nchunks,
                                    const_cast<int4*>(a.table), const_cast<int4*>(a.seqs), st))
      return rc;
  if (a.nchunks > 0)
    if (const int rc = launch_prep(a, false, st)) return rc;
  return launch_scan(a, st);
}
