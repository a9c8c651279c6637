// Forward of the chunked gated delta rule: the scan over each sequence's
// chunks (formulas, precision and fragment layout in delta.h).
//
// A workgroup of four waves owns 16 NT value columns of one head of one
// sequence and walks its chunks in order.  Each wave has a quarter of every
// product's rows: 16 tokens of X = K S0, of U = T R and of O, and a quarter of
// the state's features, which stay in its registers from the first chunk to
// the last.  So an operand fragment (K, Q, T, P, K^T) is read by one wave,
// straight into its registers and a chunk ahead, and only S, R and U pass
// through LDS, from the wave that made them to all four: three barriers a
// chunk.  With one wave for all rows of 16 columns instead, and the fragments
// in LDS for four such waves, a chunk took 4.9 us (79 chunks of 128 x 128).
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

template <int KS, int NT, bool SAVE>
__global__ __launch_bounds__(256) void delta_scan_kernel(Args a) {
  constexpr int FT = (2 * KS + 3) / 4;   // 16-feature tiles of a wave
  __shared__ __attribute__((aligned(16))) uint8_t Sb[2][KS * NT * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t Rb[2][2 * NT * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t Ub[2][2 * NT * 1024];   // U
  __shared__ __attribute__((aligned(16))) uint8_t Eb[2][2 * NT * 1024];   // e^{G_C - G} U
  Scan s;
  if (!s.init(a, 16 * NT)) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int col = s.col0 + NT * r;   // the lane's first column
  const bool live = col < a.Dv;
  const uint32_t put = (r + 16 * (q >> 1)) * 16 + (q & 1) * 8;   // 4 rows of a tile in a fragment
  const auto put_tile = [&](uint8_t (*buf)[2 * NT * 1024], int n, f32x4 x) {
    bf16x4 hi, lo;
    split4(x, hi, lo);
    const uint32_t at = ((wave >> 1) * NT + n) * 1024 + (wave & 1) * 512 + put;
    *reinterpret_cast<bf16x4*>(buf[0] + at) = hi;
    *reinterpret_cast<bf16x4*>(buf[1] + at) = lo;
  };
  const auto get = [&](const uint8_t* buf, int f) {
    return *reinterpret_cast<const bf16x8*>(buf + f * 1024 + lane * 16);
  };

  f32x4 S[FT][NT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int feat = 16 * (wave * FT + f) + 4 * q + i;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        S[f][n][i] = a.h0 && live && feat < a.Dk
                         ? a.h0[((int64_t)s.head * a.Dk + feat) * a.Dv + col + n] : 0.0f;
    }

  bf16x8 kf[KS], qf[KS], tf[2][2], pf[2][2], ktf[FT][2];
  f32x4 gam, ge, bt;
  float gc;
  Cols<NT> vr[4];
  // The loads of chunk c's operands; past the last chunk they repeat it.
  const auto load_rows = [&](int c) {
    c = min(c, s.nc - 1);
    const int n = min(kC, s.len - c * kC), t = 16 * wave + r;
    const Rsrc kp = buffer_at(a.k + s.b * a.k_sb + s.hk * a.k_sh + (s.tok0 + (int64_t)c * kC) * a.k_st);
    const Rsrc qp = buffer_at(a.q + s.b * a.q_sb + s.hk * a.q_sh + (s.tok0 + (int64_t)c * kC) * a.q_st);
    const Rsrc vp = buffer_at(a.v + s.b * a.v_sb + s.hv * a.v_sh + (s.tok0 + (int64_t)c * kC) * a.v_st);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int e = 32 * ks + 8 * q;
      const bool ok = t < n && e < a.Dk;
      kf[ks] = load_frag(kp, ok ? 2 * (t * (uint32_t)a.k_st + e) : kNoRow);
      qf[ks] = load_frag(qp, ok ? 2 * (t * (uint32_t)a.q_st + e) : kNoRow);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tv = 16 * wave + 4 * q + i;
      vr[i].load(vp, tv < n && live ? 2 * (tv * (uint32_t)a.v_st + col) : kNoRow);
    }
  };
  const auto load_scal = [&](int c) {
    const float* sc = a.scal + ((size_t)(s.c0 + min(c, s.nc - 1)) * a.Hv + s.hv) * kScal;
    const int t = 16 * wave + 4 * q;
    gam = *reinterpret_cast<const f32x4*>(sc + t);
    ge = *reinterpret_cast<const f32x4*>(sc + kC + t);
    bt = *reinterpret_cast<const f32x4*>(sc + 2 * kC + t);
    gc = sc[kC - 1];
  };
  const auto load_tri = [&](int c, int which, bf16x8 (&x)[2][2]) {
    const uint8_t* p = a.tri + ((size_t)(s.c0 + min(c, s.nc - 1)) * a.Hv + s.hv) * kTriBytes +
                       which * 2 * kTFrags * 1024 + lane * 16;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      // step 1 of the upper tiles is zero and not stored: step 0 again, unused
      const int f = lower_frag(wave, wave < 2 ? 0 : ks);
      x[ks][0] = *reinterpret_cast<const bf16x8*>(p + f * 1024);
      x[ks][1] = *reinterpret_cast<const bf16x8*>(p + (kTFrags + f) * 1024);
    }
  };
  const auto load_kt = [&](int c) {
    const uint8_t* p = a.kt + ((size_t)(s.c0 + min(c, s.nc - 1)) * a.Hk + s.hk) * (4 * KS) * 1024 + lane * 16;
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (wave * FT + f < 2 * KS)
          ktf[f][t] = *reinterpret_cast<const bf16x8*>(p + (2 * (wave * FT + f) + t) * 1024);
  };
  // the state's parts to LDS, and of a chunk that a backward will read to memory
  const auto put_state = [&](int c) {
    Rsrc sp;
    if constexpr (SAVE) sp = buffer_at(a.s0 + ((int64_t)(s.c0 + c) * a.Hv + s.hv) * 2 * a.Dk * a.Dv);
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const int tile = wave * FT + f;
      if (tile < 2 * KS) {
        bf16x4 hi[NT], lo[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          split4(S[f][n], hi[n], lo[n]);
          const uint32_t at = ((tile >> 1) * NT + n) * 1024 + (tile & 1) * 512 + put;
          *reinterpret_cast<bf16x4*>(Sb[0] + at) = hi[n];
          *reinterpret_cast<bf16x4*>(Sb[1] + at) = lo[n];
        }
        if constexpr (SAVE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int feat = 16 * tile + 4 * q + i;
            const uint32_t at = live && feat < a.Dk ? 2 * (feat * a.Dv + col) : kNoRow;
            __bf16 h[NT], l[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              h[n] = hi[n][i];
              l[n] = lo[n][i];
            }
            store_cols<NT>(sp, at, h);
            store_cols<NT>(sp, at + 2 * (uint32_t)(a.Dk * a.Dv), l);
          }
        }
      }
    }
  };

  if (s.nc > 0) {
    load_rows(0);
    load_scal(0);
    load_tri(0, 0, tf);
    load_tri(0, 1, pf);
    load_kt(0);
    put_state(0);
  }
  for (int c = 0; c < s.nc; ++c) {
    lds_barrier();   // S0 is in LDS
    f32x4 X[NT] = {}, O[NT] = {};
    {
      f32x4 X2[NT] = {}, O2[NT] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 hi = get(Sb[0], ks * NT + n), lo = get(Sb[1], ks * NT + n);
          X[n] = mfma(kf[ks], hi, X[n]);
          O[n] = mfma(qf[ks], hi, O[n]);
          X2[n] = mfma(kf[ks], lo, X2[n]);
          O2[n] = mfma(qf[ks], lo, O2[n]);
        }
      // R = b (V - gam X); rows behind the sequence's end have b = 0 and V = 0
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = vr[i].get(n);
        put_tile(Rb, n, bt * (v - gam * (X[n] + X2[n])));
        O[n] = (O[n] + O2[n]) * (gam * a.scale);
      }
    }
    load_rows(c + 1);
    lds_barrier();   // R is in LDS
    f32x4 U[NT] = {};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (ks <= wave >> 1)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 hi = get(Rb[0], ks * NT + n), lo = get(Rb[1], ks * NT + n);
          U[n] = mfma(tf[ks][0], hi, U[n]);
          U[n] = mfma(tf[ks][1], hi, U[n]);
          U[n] = mfma(tf[ks][0], lo, U[n]);
        }
    load_tri(c + 1, 0, tf);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      put_tile(Eb, n, ge * U[n]);
      put_tile(Ub, n, U[n]);
    }
    const int left = s.len - c * kC;
    const int64_t row0 = (int64_t)s.b * a.T + s.tok0 + (int64_t)c * kC;
    if constexpr (SAVE) {
      const int64_t at = (row0 * a.Hv + s.hv) * a.Dv;
      const Rsrc hp = buffer_at(a.u + at), lp = buffer_at(a.u + (int64_t)a.B * a.T * a.Hv * a.Dv + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * wave + 4 * q + i;
        const uint32_t off = live && t < left ? 2 * (t * (uint32_t)(a.Hv * a.Dv) + col) : kNoRow;
        __bf16 h[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          h[n] = (__bf16)U[n][i];
          l[n] = (__bf16)(U[n][i] - (float)h[n]);
        }
        store_cols<NT>(hp, off, h);
        store_cols<NT>(lp, off, l);
      }
    }
    lds_barrier();   // U is in LDS
    // S' = gam_C S0 + K^T (e^{G_C - G} U)
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int n = 0; n < NT; ++n) S[f][n] *= gc;
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
    load_kt(c + 1);
    load_scal(c + 1);
    // O += P U
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (ks <= wave >> 1)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 hi = get(Ub[0], ks * NT + n), lo = get(Ub[1], ks * NT + n);
          O[n] = mfma(pf[ks][0], hi, O[n]);
          O[n] = mfma(pf[ks][1], hi, O[n]);
          O[n] = mfma(pf[ks][0], lo, O[n]);
        }
    load_tri(c + 1, 1, pf);
    if (c + 1 < s.nc) put_state(c + 1);
    const Rsrc op = buffer_at(a.o + (row0 * a.Hv + s.hv) * a.Dv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 16 * wave + 4 * q + i;
      __bf16 h[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) h[n] = (__bf16)O[n][i];
      store_cols<NT>(op, live && t < left ? 2 * (t * (uint32_t)(a.Hv * a.Dv) + col) : kNoRow, h);
    }
  }
  if (a.hT && live) {
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

template <int KS, int NT>
void launch_scan_as(const Args& a, hipStream_t st) {
  const dim3 grid(scan_blocks(a, 16 * NT));
  if (a.s0) hipLaunchKernelGGL((delta_scan_kernel<KS, NT, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((delta_scan_kernel<KS, NT, false>), grid, dim3(256), 0, st, a);
}

int launch_scan(const Args& a, hipStream_t st) {
  UTTT_DELTA_STEPS(steps_of(a.Dk), KS, switch (scan_tiles(a)) {
    case 1: launch_scan_as<KS, 1>(a, st); break;
    case 2: launch_scan_as<KS, 2>(a, st); break;
    default: launch_scan_as<KS, 4>(a, st); break;
  });
  return check_launch("delta_scan");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int check_args(const Args& a, int B, bool packed, const char* what) {
  UTTT_REQUIRE(B >= 1 && a.T >= 0 && a.nseq >= 1 && a.Hk >= 1 && a.Hv >= 1,
               "%s: bad sizes B=%d T=%d sequences=%d Hk=%d Hv=%d", what, B, a.T, a.nseq, a.Hk, a.Hv);
  UTTT_REQUIRE(a.Hv % a.Hk == 0, "%s: Hv=%d must be a multiple of Hk=%d", what, a.Hv, a.Hk);
  UTTT_REQUIRE(a.Dk >= 8 && a.Dk <= 256 && a.Dk % 8 == 0, "%s: Dk=%d must be a multiple of 8 up to 256",
               what, a.Dk);
  UTTT_REQUIRE(a.Dv >= 8 && a.Dv <= 65536 && a.Dv % 8 == 0,
               "%s: Dv=%d must be a multiple of 8 up to 65536", what, a.Dv);
  UTTT_REQUIRE(packed ? B == 1 : a.nseq == B, "%s: %d sequences in a batch of %d", what, a.nseq, B);
  const int64_t slots = chunk_slots(B, a.T, a.nseq, packed);
  UTTT_REQUIRE(slots >= 0 && slots * a.Hv < (1LL << 31) &&
                   ((int64_t)a.nseq * a.Hv + 8) * ((a.Dv + 63) / 64) < (1LL << 31),
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
  if (const int rc = check_args(a, B, packed, what)) return rc;
  a.nchunks = chunk_slots(B, T, nseq, packed);
  UTTT_REQUIRE(out || T == 0, "%s: null output", what);
  UTTT_REQUIRE(aligned16(out) && aligned16(u_saved) && aligned16(s_saved) && aligned16(workspace),
               "%s: tensors must be 16-byte aligned", what);
  UTTT_REQUIRE((u_saved == nullptr) == (s_saved == nullptr), "%s: save both U and S or neither", what);
  const Workspace w = workspace_of(B, T, nseq, Hk, Hv, Dk, Dv, packed, false);
  UTTT_REQUIRE(w.total == 0 || (workspace && workspace_bytes >= w.total),
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, w.total);
  bind_workspace(a, w, static_cast<uint8_t*>(workspace), packed, false);
  a.h0 = initial_state;
  a.hT = final_state;
  a.o = static_cast<uint16_t*>(out);
  a.u = static_cast<uint16_t*>(u_saved);
  a.s0 = static_cast<uint16_t*>(s_saved);
  const hipStream_t st = as_stream(stream);
  if (packed)
    if (const int rc = launch_table(cu_seqlens, cu_is_int64, nseq, T, a.nchunks,
                                    const_cast<int4*>(a.table), const_cast<int4*>(a.seqs), st))
      return rc;
  if (a.nchunks > 0)
    if (const int rc = launch_prep(a, false, st)) return rc;
  return launch_scan(a, st);
}
