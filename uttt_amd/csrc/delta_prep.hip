// Per-chunk operands of the gated delta rule (the formulas are in delta.h):
// the chunk table of packed sequences, and per chunk and head the decays, T =
// (I + A)^-1, P and the transposed keys, laid out as the matrix instruction's
// operand fragments for the scans that follow.
//
// Bound by memory: K and Q read once; T and P written, 30 KiB a chunk and value
// head (36 in the backward), and K^T (Q^T, K, Q where asked for), 128 bytes a
// feature of a chunk and key head each.  16 x 2048 tokens, 12 heads of 128: 129 us
// forward, 150 backward, 3.9 and 4.2 TB/s.  The backward makes its operands again:
// kept from the forward, transposed, they would hold 430 MB of that layer to save
// a tenth of its step.
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

constexpr int kTableThreads = 1024;
// Sequences up to which the scans start with the longest, so that it does not
// come last and alone: 12 prompts of 1 to 5000 tokens in rising order, 16
// heads, 199 -> 168 us.  The table's kernel ranks each sequence by all others
// (12: 1 us); more than these fill the CUs in any order.
constexpr int kRanked = 256;

// Offsets that descend or leave [0, T] are clamped (a later one counts from
// the highest before it), so that no chunk lies outside the token axis.  The
// slots after the sequences' chunks cover the tokens of no sequence, whose
// outputs are zeros.
__global__ __launch_bounds__(kTableThreads) void delta_table_kernel(const void* cu, int cu64, int nseq,
                                                                    int T, int nchunks,
                                                                    int4* __restrict__ table,
                                                                    int4* __restrict__ seqs) {
  constexpr int kWaves = kTableThreads / 64;
  __shared__ int whi[kWaves], wcnt[kWaves], counts[kRanked];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const auto at = [&](int i) -> int {
    const int64_t x = cu64 ? static_cast<const int64_t*>(cu)[i] : static_cast<const int32_t*>(cu)[i];
    return (int)(x < 0 ? 0 : x > T ? T : x);
  };
  const int first = at(0);
  int carry_hi = first, carry_cnt = 0;   // the same in every thread
  for (int s0 = 0; s0 < nseq; s0 += kTableThreads) {
    const int s = s0 + tid;
    int end = s < nseq ? at(s + 1) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {   // running maximum
      const int x = __shfl_up(end, d);
      if (lane >= d) end = max(end, x);
    }
    if (lane == 63) whi[wave] = end;
    __syncthreads();
    int before = carry_hi;
    for (int w = 0; w < wave; ++w) before = max(before, whi[w]);
    end = max(end, before);
    int start = __shfl_up(end, 1);
    if (lane == 0) start = before;
    const int n = s < nseq ? (end - start + kC - 1) / kC : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {   // running sum
      const int x = __shfl_up(sum, d);
      if (lane >= d) sum += x;
    }
    if (lane == 63) wcnt[wave] = sum;
    __syncthreads();
    int c0 = carry_cnt + sum - n;
    for (int w = 0; w < wave; ++w) c0 += wcnt[w];
    int place = s;
    if (nseq <= kRanked) {
      if (s < nseq) counts[s] = n;
      __syncthreads();
      if (s < nseq) {
        place = 0;
        for (int j = 0; j < nseq; ++j) place += counts[j] > n || (counts[j] == n && j < s);
      }
    }
    if (s < nseq) seqs[place] = make_int4(c0, s, start, end - start);
    // a wave's sequences one after another, 64 chunks at a time
    const int mine = min(64, nseq - (s - lane));
    for (int l = 0; l < mine; ++l) {
      const int ln = __shfl(n, l), lc = __shfl(c0, l), ls = __shfl(start, l), le = __shfl(end, l);
      for (int i = lane; i < ln; i += 64)
        if (lc + i < nchunks)
          table[lc + i] = make_int4(s - lane + l, ls + i * kC, min(kC, le - ls - i * kC), 0);
    }
    for (int w = 0; w < kWaves; ++w) {
      carry_hi = max(carry_hi, whi[w]);
      carry_cnt += wcnt[w];
    }
    __syncthreads();
  }
  const int used = carry_cnt, last = carry_hi;
  const int nfront = (first + kC - 1) / kC, nback = (T - last + kC - 1) / kC;
  for (int i = tid; used + i < nchunks; i += kTableThreads) {
    int4 e = make_int4(-2, 0, 0, 0);
    if (i < nfront) e = make_int4(-1, i * kC, min(kC, first - i * kC), 0);
    else if (i < nfront + nback)
      e = make_int4(-1, last + (i - nfront) * kC, min(kC, T - last - (i - nfront) * kC), 0);
    table[used + i] = e;
  }
}

// e^x of a difference of cumulative log decays held in 64 bits.
__device__ __forceinline__ float exp_diff(double x) { return __expf((float)x); }

// Zeros for the tokens of no sequence.
template <bool BWD>
__device__ void clear_rows(const Args& a, const Chunk& ch, int hk) {
  const int r = a.Hv / a.Hk;
  const uint4 z = make_uint4(0, 0, 0, 0);
  const int per_v = r * a.Dv / 8, per_k = a.Dk / 8;
  for (int i = threadIdx.x; i < ch.n * per_v; i += 256) {
    const int t = i / per_v, x = i - t * per_v;
    const int64_t at = ((int64_t)(ch.t0 + t) * a.Hv + hk * r) * a.Dv + 8 * x;
    *reinterpret_cast<uint4*>((BWD ? a.dv : a.o) + at) = z;
  }
  if constexpr (BWD) {
    for (int i = threadIdx.x; i < ch.n * per_k; i += 256) {
      const int t = i / per_k, x = i - t * per_k;
      const int64_t at = ((int64_t)(ch.t0 + t) * a.Hk + hk) * a.Dk + 8 * x;
      *reinterpret_cast<uint4*>(a.dq + at) = z;
      *reinterpret_cast<uint4*>(a.dk + at) = z;
    }
    for (int i = threadIdx.x; i < ch.n * r; i += 256) {
      const int64_t at = (int64_t)(ch.t0 + i / r) * a.Hv + hk * r + i % r;
      store_any(a.dg, a.g_dtype, at, 0.0f);
      store_any(a.dbeta, a.beta_dtype, at, 0.0f);
    }
  }
}

// A chunk's rows of K or Q (features up to 32 KS, zeros past Dk and the
// chunk's end) into LDS rows of LD elements.
template <int KS, int LD>
__device__ __forceinline__ void stage_rows(const uint16_t* src, int64_t st, int n, int Dk,
                                           uint16_t* lds) {
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int piece = i * 256 + threadIdx.x;
    const int t = piece / (4 * KS), p = piece % (4 * KS);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (t < n && 8 * p < Dk) x = *reinterpret_cast<const uint4*>(src + t * st + 8 * p);
    *reinterpret_cast<uint4*>(lds + t * LD + 8 * p) = x;
  }
}

// The transposed fragments first, first + step, .. of staged rows: 16 features
// by 32 tokens each.
template <int KS, int LD>
__device__ __forceinline__ void write_transposed(const uint16_t* lds, uint8_t* out, int first, int step) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  for (int f = first; f < 4 * KS; f += step) {
    const int feat = 16 * (f >> 1) + r, t0 = 32 * (f & 1) + 8 * q;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = lds[(t0 + 2 * i) * LD + feat] | ((uint32_t)lds[(t0 + 2 * i + 1) * LD + feat] << 16);
    *reinterpret_cast<uint4*>(out + (size_t)f * 1024 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The same of staged rows as they are: 16 tokens by 32 features each.
template <int KS, int LD>
__device__ __forceinline__ void write_rows(const uint16_t* lds, uint8_t* out, int first, int step) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  for (int f = first; f < 4 * KS; f += step)
    *reinterpret_cast<uint4*>(out + (size_t)f * 1024 + lane * 16) =
        *reinterpret_cast<const uint4*>(lds + (16 * (f / KS) + r) * LD + 32 * (f % KS) + 8 * q);
}

constexpr int kLT = kC + 4;   // fp32 row stride of the 64 x 64 matrices

// Fragments first, first + step, .. of a triangular matrix (or its transpose) in
// LDS, each part's behind the part before it.
template <bool TRANS, int PARTS>
__device__ __forceinline__ void write_tri(const float* m, uint8_t* out, int first, int step) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  for (int f = first; f < kTFrags; f += step) {
    const int rt = TRANS ? (f < 4 ? f >> 1 : f - 2) : (f < 2 ? f : 2 + (f - 2) / 2);
    const int ks = TRANS ? (f < 4 ? f & 1 : 1) : (f < 2 ? 0 : f & 1);
    const int row = 16 * rt + r, c0 = 32 * ks + 8 * q;
    f32x4 x, y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = TRANS ? m[(c0 + i) * kLT + row] : m[row * kLT + c0 + i];
      y[i] = TRANS ? m[(c0 + 4 + i) * kLT + row] : m[row * kLT + c0 + 4 + i];
    }
    bf16x8 part[PARTS];
    split8(x, y, part);
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
      *reinterpret_cast<bf16x8*>(out + (k * kTFrags + f) * 1024 + lane * 16) = part[k];
  }
}

// One chunk of one key head, with every value head that shares it.  The
// inverse: 16 x 16 diagonal blocks by forward substitution (a lane per column,
// stable for any keys, where a product of powers of A is not), then pairs of
// blocks joined by T21 = -T22 A21 T11 in fp32 matrix instructions.
template <int KS, bool BWD>
__global__ __launch_bounds__(256, KS <= 4 ? 4 : 2) void delta_prep_kernel(Args a) {
  constexpr int LD = 32 * KS + 8;
  constexpr int kRows = 2 * kC * LD * 2;                 // K and Q, bytes
  constexpr int kMats = 2 * kC * kLT * 4;                // A and P
  __shared__ __attribute__((aligned(16))) uint8_t buf[kRows > kMats ? kRows : kMats];
  __shared__ double Gd[kC];
  __shared__ float bet[kC];
  __shared__ int bad;   // the first row of A that is not finite
  const int c = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk;
  const Chunk ch = chunk_of(a, c);
  if (ch.seq < 0) {
    if (ch.seq == -1) clear_rows<BWD>(a, ch, hk);
    return;
  }
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int group = a.Hv / a.Hk;
  float gv = 0.0f, bv = 0.0f;   // wave 0: the lane's token
  const auto load_gates = [&](int hv) {
    if (lane < ch.n) {
      const int64_t at = ((int64_t)ch.b * a.T + ch.t0 + lane) * a.Hv + hv;
      gv = load_any(a.g, a.g_dtype, at);
      bv = load_any(a.beta, a.beta_dtype, at);
    }
  };
  // Cumulative log decays in 64 bits: differences of far tokens' sums keep
  // fp32's relative order.  A decay below e^-200 is one of zero in fp32 and
  // would only cost the sums their digits.
  const auto put_decays = [&](int hv) {
    const double G = scan64(gv < -200.0f ? -200.0f : gv);
    const double Gc = __shfl(G, 63);
    Gd[lane] = G;
    bet[lane] = bv;
    float* sc = a.scal + ((size_t)c * a.Hv + hv) * kScal;
    sc[lane] = exp_diff(G);
    sc[kC + lane] = exp_diff(Gc - G);
    sc[2 * kC + lane] = bv;
    sc[3 * kC + lane] = (float)G;
    sc[4 * kC + lane] = (float)(G - (double)(float)G);
  };
  if (tid == 0) bad = kC;
  if (wave == 0) load_gates(hk * group);
  uint16_t* Kl = reinterpret_cast<uint16_t*>(buf);
  uint16_t* Ql = Kl + kC * LD;
  stage_rows<KS, LD>(a.k + ch.b * a.k_sb + ch.t0 * a.k_st + hk * a.k_sh, a.k_st, ch.n, a.Dk, Kl);
  stage_rows<KS, LD>(a.q + ch.b * a.q_sb + ch.t0 * a.q_st + hk * a.q_sh, a.q_st, ch.n, a.Dk, Ql);
  __syncthreads();
  f32x4 kk[4] = {}, qk[4] = {};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = 32 * ks + 8 * q;
    const bf16x8 ka = *reinterpret_cast<const bf16x8*>(Kl + (16 * wave + r) * LD + e);
    const bf16x8 qa = *reinterpret_cast<const bf16x8*>(Ql + (16 * wave + r) * LD + e);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      const bf16x8 kb = *reinterpret_cast<const bf16x8*>(Kl + (16 * ct + r) * LD + e);
      kk[ct] = mfma(ka, kb, kk[ct]);
      qk[ct] = mfma(qa, kb, qk[ct]);
    }
  }
  if (wave == 0) {
    put_decays(hk * group);
  } else {
    const size_t frag = ((size_t)c * a.Hk + hk) * (4 * KS) * 1024;
    write_transposed<KS, LD>(Kl, a.kt + frag, wave - 1, 3);
    if constexpr (BWD) write_transposed<KS, LD>(Ql, a.qt + frag, wave - 1, 3);
    if (a.kf) write_rows<KS, LD>(Kl, a.kf + frag, wave - 1, 3);
    if (a.qf) write_rows<KS, LD>(Ql, a.qf + frag, wave - 1, 3);
  }
  __syncthreads();
  float* Am = reinterpret_cast<float*>(buf);
  float* Pm = Am + kC * kLT;
  float* Tm = Pm;   // T takes P's place once P's fragments are written
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    float zero = 0.0f;   // NaN where some value is not finite
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      const int j = 16 * ct + r;
      const double Gj = Gd[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * wave + 4 * q + i;
        const float e = row >= j ? exp_diff(Gd[row] - Gj) : 0.0f;
        const float x = row > j ? bet[row] * e * kk[ct][i] : 0.0f;
        Am[row * kLT + j] = x;
        zero = __builtin_fmaf(x, 0.0f, zero);
        Pm[row * kLT + j] = row >= j ? a.scale * e * qk[ct][i] : 0.0f;
      }
    }
    if (__builtin_expect(zero != 0.0f, 0))
      for (int i = 0; i < 4; ++i)
        for (int ct = 0; ct < 4; ++ct) {
          const int row = 16 * wave + 4 * q + i;
          if (Am[row * kLT + 16 * ct + r] * 0.0f != 0.0f) atomicMin(&bad, row);
        }
    __syncthreads();
    // T's blocks are joined by products whose zeros would make NaN of earlier
    // tokens' rows: from the first row on that is not finite A is left out, and a
    // beta of NaN gives that token's R and so all that comes after it.
    const int first_bad = __builtin_amdgcn_readfirstlane(bad);
    if (__builtin_expect(first_bad < kC, 0)) {
      for (int i = first_bad * kLT + tid; i < kC * kLT; i += 256) Am[i] = 0.0f;
      if (wave == 0 && lane >= first_bad)
        a.scal[((size_t)c * a.Hv + hv) * kScal + 2 * kC + lane] = __builtin_nanf("");
      __syncthreads();
      if (tid == 0) bad = kC;   // for the next head
    }
    uint8_t* tri = a.tri + ((size_t)c * a.Hv + hv) * (BWD ? kTriBwdBytes : kTriBytes);
    // wave 0: column r of diagonal block q, top to bottom; the others: P's fragments
    float t[16];
    if (wave == 0) {
      const float* A0 = Am + 16 * q * kLT + 16 * q;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x = i == r ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) x = __builtin_fmaf(-A0[i * kLT + j], t[j], x);
        t[i] = x;
      }
    } else {
      write_tri<BWD, BWD ? 3 : 2>(Pm, tri + kPFrag * 1024, wave - 1, 3);
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Tm[(16 * q + i) * kLT + 16 * q + r] = t[i];
    } else if (wave == 1) {
      // the zero blocks that a fragment of 32 columns takes in
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Tm[(4 * q + i) * kLT + 16 + r] = 0.0f;
        Tm[(32 + 4 * q + i) * kLT + 48 + r] = 0.0f;
      }
    }
    __syncthreads();
    if (wave < 2) {   // blocks 2w, 2w + 1 joined
      const int b0 = 32 * wave, b1 = b0 + 16;
      f32x4 y = {}, z = {};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        y = mfma_f32(Am[(b1 + r) * kLT + b0 + 4 * s + q], Tm[(b0 + 4 * s + q) * kLT + b0 + r], y);
      // y's rows 4q + s are the contracted axis as they lie
#pragma unroll
      for (int s = 0; s < 4; ++s) z = mfma_f32(Tm[(b1 + r) * kLT + b1 + 4 * q + s], y[s], z);
#pragma unroll
      for (int i = 0; i < 4; ++i) Tm[(b1 + 4 * q + i) * kLT + b0 + r] = -z[i];
    }
    __syncthreads();
    {
      const int ct = wave & 1, rt = wave >> 1;
      f32x4 y[2] = {}, z = {};
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float b = Tm[(4 * s + q) * kLT + 16 * ct + r];
        y[0] = mfma_f32(Am[(32 + r) * kLT + 4 * s + q], b, y[0]);
        y[1] = mfma_f32(Am[(48 + r) * kLT + 4 * s + q], b, y[1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          z = mfma_f32(Tm[(32 + 16 * rt + r) * kLT + 32 + 16 * h + 4 * q + s], y[h][s], z);
#pragma unroll
      for (int i = 0; i < 4; ++i) Tm[(32 + 16 * rt + 4 * q + i) * kLT + 16 * ct + r] = -z[i];
    }
    __syncthreads();
    const bool more = hv + 1 < (hk + 1) * group;
    if (wave == 0 && more) {   // the next head's decays meanwhile
      load_gates(hv + 1);
      put_decays(hv + 1);
    }
    write_tri<BWD, 3>(Tm, tri, more ? (wave == 0 ? kTFrags : wave - 1) : wave, more ? 3 : 4);
    __syncthreads();
  }
}

}  // namespace

int launch_table(const void* cu, int cu64, int nseq, int T, int nchunks, int4* table, int4* seqs,
                 hipStream_t st) {
  hipLaunchKernelGGL(delta_table_kernel, dim3(1), dim3(kTableThreads), 0, st, cu, cu64, nseq, T,
                     nchunks, table, seqs);
  return check_launch("delta_table");
}

int launch_prep(const Args& a, bool transposed, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.nchunks * a.Hk));
  UTTT_DELTA_STEPS(steps_of(a.Dk), KS,
                   if (transposed) hipLaunchKernelGGL((delta_prep_kernel<KS, true>), grid, dim3(256), 0, st, a);
                   else hipLaunchKernelGGL((delta_prep_kernel<KS, false>), grid, dim3(256), 0, st, a));
  return check_launch("delta_prep");
}

}  // namespace delta
}  // namespace uttt
