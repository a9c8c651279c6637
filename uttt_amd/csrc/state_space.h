// Shared pieces of the state space layer's kernels (causal_conv.hip,
// scan_fwd.hip, scan_bwd.hip, scan_step.hip): the sequences of a call and their
// runs of tokens, and scalar loads of any element type.
#pragma once

#include "common.h"

namespace uttt {
namespace ssm {

// nseq sequences: rows of a batch of T tokens each (cu null), or the tokens
// cu[n] .. cu[n + 1] of one row of T.
struct Seqs {
  const void* cu;   // [nseq + 1] or null
  int cu64;
  int B, T, nseq;
  __device__ __forceinline__ int offset(int n) const {   // clamped: never past the token axis
    const int64_t v = cu64 ? static_cast<const int64_t*>(cu)[n] : static_cast<const int32_t*>(cu)[n];
    return (int)(v < 0 ? 0 : v > T ? T : v);
  }
};

// A run: up to `len` tokens of one sequence from a multiple of len on.  Every
// sequence has one run at least (of no tokens, if it has none).
struct Run {
  int seq;       // -1: no run of this number
  int b, tok0;   // batch row and place of the sequence's first token
  int len;       // tokens of the sequence
  int c;         // the run's number in its sequence
  int base;      // the number of the sequence's first run
};

// Runs of R tokens.  Packed sequence n has the numbers from cu[n] / R + n on,
// which holds its ceil(len / R) and always one.
inline int64_t run_count(const Seqs& s, int64_t R) {
  return s.cu ? s.T / R + s.nseq : (int64_t)s.nseq * (s.T > 0 ? (s.T + R - 1) / R : 1);
}
__device__ __forceinline__ int first_run(const Seqs& s, int n, int R) {
  return s.cu ? s.offset(n) / R + n : n * (s.T > 0 ? (s.T + R - 1) / R : 1);
}
__device__ __forceinline__ Run span_of(const Seqs& s, int n, int R) {
  if (!s.cu) return {n, n, 0, s.T, 0, first_run(s, n, R)};
  const int t0 = s.offset(n), t1 = s.offset(n + 1);
  return {n, 0, t0, t1 > t0 ? t1 - t0 : 0, 0, t0 / R + n};
}
__device__ __forceinline__ Run run_of(const Seqs& s, int at, int R) {
  int n;
  if (!s.cu) {
    n = at / (s.T > 0 ? (s.T + R - 1) / R : 1);
  } else {   // the last sequence whose first run is not behind
    int lo = 0, hi = s.nseq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.offset(mid) / R + mid <= at) lo = mid;
      else hi = mid - 1;
    }
    n = lo;
  }
  Run r = span_of(s, n, R);
  r.c = at - r.base;
  if (r.c < 0 || (r.c > 0 && (int64_t)r.c * R >= r.len)) r.seq = -1;
  return r;
}

// Places behind the last run for the tokens of no sequence, which are few where
// buffers are filled: each writes its share in turn.
constexpr int kLooseRuns = 8;
// Token i of the tokens of no sequence of a packed call, -1 past the last one.
__device__ __forceinline__ int loose_token(const Seqs& s, int i) {
  const int head = s.offset(0), tail = s.offset(s.nseq);
  if (i < head) return i;
  const int64_t t = (int64_t)i - head + (tail > head ? tail : head);
  return t < s.T ? (int)t : -1;
}

inline bool seqs_ok(const Seqs& s) {
  return s.B >= 1 && s.T >= 0 && s.nseq >= 1 && (s.cu ? s.B == 1 : s.nseq == s.B);
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == UTTT_F32) return static_cast<const float*>(p)[i];
  const uint16_t h = static_cast<const uint16_t*>(p)[i];
  return dtype == UTTT_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float x) {
  if (dtype == UTTT_F32) static_cast<float*>(p)[i] = x;
  else static_cast<uint16_t*>(p)[i] = dtype == UTTT_BF16 ? f32_to_bf16(x) : f32_to_f16(x);
}

// e^-|x| (to e^-100, below which it is no normal fp32): the hardware's 2^x, an
// ulp off, of x log2 e, whose rounding is made good to the first order.
__device__ __forceinline__ float exp_neg_abs(float x) {
  constexpr float c = 1.44269504088896340736f, c_low = 1.92596303e-8f, ln2 = 0.69314718055994530942f;
  const float v = -fminf(fabsf(x), 100.0f), t = v * c;
  const float low = __builtin_fmaf(v, c_low, __builtin_fmaf(v, c, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, low * ln2, e);
}
// 1 / (1 + e^-x), off by 2 ulp or so.
__device__ __forceinline__ float sigmoid(float x) {
  const float e = exp_neg_abs(x), r = __builtin_amdgcn_rcpf(1.0f + e);
  return x < 0.0f ? e * r : r;
}
// The same where it goes into results of TT.  For 16-bit ones without the
// correction: off by |x| 2^-24 and an ulp or two of it, a third of their 2^-24
// in absolute terms.
template <class TT>
__device__ __forceinline__ float sigmoid_for(float x) {
  if constexpr (sizeof(typename TT::S) == 4) return sigmoid(x);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * x));
}
// ln(1 + e^x) and its slope 1 / (1 + e^-x), with s = 1 + e^-|x| and what its
// rounding left out: ln(1 + e) = ln(s) + (e - (s - 1)) / s to the first order.
__device__ __forceinline__ float softplus(float x, float& slope) {
  const float e = exp_neg_abs(x), s = 1.0f + e, r = __builtin_amdgcn_rcpf(s);
  slope = x < 0.0f ? e * r : r;
  const float l = __builtin_fmaf(__builtin_amdgcn_logf(s), 0.69314718055994530942f, (e - (s - 1.0f)) * r);
  return (x < 0.0f ? 0.0f : x) + l;
}
__device__ __forceinline__ float softplus(float x) {
  float slope;
  return softplus(x, slope);
}

// The rows of a step against a pool's slots.  Rows of one slot follow one
// another in row order: the first one's workgroup takes them all up.
struct Rows {
  const void* idx;   // [B] or null: row b has slot b
  int idx64, B, slots;
  __device__ __forceinline__ int64_t slot_of(int b) const {   // -1: no slot
    const int64_t s = idx == nullptr ? b
                      : idx64        ? static_cast<const int64_t*>(idx)[b]
                                     : static_cast<const int32_t*>(idx)[b];
    return s >= 0 && s < slots ? s : -1;
  }
  // Whether rows before and behind row b have its slot (bits 0 and 1); for whole
  // workgroups.
  template <int THREADS>
  __device__ __forceinline__ int others(int b, int64_t slot) const {
    if (!idx) return 0;
    __shared__ int found[THREADS / kWave];
    int mine = 0;
    for (int j = threadIdx.x; j < B; j += THREADS)
      if (j != b && slot_of(j) == slot) mine |= j < b ? 1 : 2;
    const int wave = (__ballot(mine & 1) ? 1 : 0) | (__ballot(mine & 2) ? 2 : 0);
    if ((threadIdx.x & (kWave - 1)) == 0) found[threadIdx.x / kWave] = wave;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) all |= found[i];
    return all;
  }
  // The next row behind b of its slot, B if there is none; for whole workgroups.
  template <int THREADS>
  __device__ __forceinline__ int next_of(int b, int64_t slot) const {
    __shared__ int next;
    __syncthreads();   // the last answer is read
    if (threadIdx.x == 0) next = B;
    __syncthreads();
    for (int j = b + 1 + threadIdx.x; j < B; j += THREADS)
      if (slot_of(j) == slot) {
        atomicMin(&next, j);
        break;
      }
    __syncthreads();
    return next;
  }
};

// out[e] = the sum of part[i][e] over i < n, for e < M, stored as dtype: in 64
// bits and an order that n alone decides.
struct Sum {
  const float* part;   // null: none
  int64_t M;
  void* out;
  int dtype;
};
int launch_sums(int64_t n, std::initializer_list<Sum> sums, hipStream_t st, const char* what);

}  // namespace ssm
}  // namespace uttt
