// The selective state space scan's geometry (scan_fwd.hip, scan_bwd.hip).  Per
// channel d of group g = d / (D / G), with a state h [N]:
//   dt_t = softplus(raw_t + bias) or raw_t + bias
//   h_t[n] = e^{dt_t A[n]} h_{t-1}[n] + dt_t x_t B_t[g, n]
//   y_t = sum_n C_t[g, n] h_t[n] + Dskip x_t,  out_t = y_t silu(z_t) (y_t without a gate)
// Everything between the loads and the stores is fp32; decays are 2^(dt A log2 e)
// by the hardware's 2^x.
//
// Forward, and in the pass that finds a run's adjoint, a lane has one channel with
// all its states.  In the gradients' pass, whose sums over channels are as many as
// its sums over states, a lane holds four states of CS channels (Geo): LN = ceil(N
// / 4) lanes (a power of two) hold a channel, a workgroup of four waves CB channels
// of one group; its threads turn x, dt, z and the outputs' gradient of 16 tokens
// into what the recurrence takes and put that into LDS, where a channel's lanes read it.
#pragma once

#include <float.h>

#include "state_space.h"

namespace uttt {
namespace ssm {

constexpr int kTile = 16;            // tokens of a tile; a backward's states are kept at their starts
constexpr int kScanThreads = 256;
constexpr int kMaxStates = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct ScanArgs {
  Seqs seqs;
  int D, N, G, Dg;         // Dg = D / G channels share B and C
  int R;                   // tokens of a run, a multiple of kTile
  int nruns, ncb;          // runs; workgroups for a run and group
  const void *x, *dt, *Bm, *Cm, *z;
  int64_t x_sb, x_st, dt_sb, dt_st, z_sb, z_st, B_sb, B_st, B_sg, C_sb, C_st, C_sg;
  int dt_dtype, soft;
  const float *A, *Dskip, *bias, *h0;   // [D, N], [D] or null, [D] or null, [nseq, D, N] or null
  void* out;               // [B, T, D]
  float *hT, *hs;          // [nseq, D, N] or null; [tiles, NP, D] or null
  float *ends, *starts;    // [nruns, NP, D]: of each run on its own; with what came before it
  float* decay;            // [nruns, D] sums of dt over a run
  // backward
  const void* dout;        // [B, T, D]
  int64_t do_sb, do_st;
  const float* dhT;        // or null
  void *dx, *ddt, *dz;     // [B, T, D] in x's, dt's and x's type
  float* dh0;              // or null
  float *part_A, *part_D, *part_bias;   // [rows, D, N], [rows, D], [rows, D] or null; a row a run, or two
  float* part_bc;          // [ncb, B, T, 2, G, N]
};

template <int LN>
struct Geo {
  static constexpr int NP = 4 * LN;               // states with those that only fill up
  static constexpr int CS = LN == 4 || LN == 8 ? 2 : 1;   // channels of a lane
  static constexpr int WC = CS * 64 / LN;         // of a wave
  static constexpr int CB = 4 * WC;               // of a workgroup
  static constexpr int HT = LN == 16 ? kTile : kTile / 2;   // tokens whose states are in registers
  static constexpr int TPP = kScanThreads / CB;   // tokens that the threads cover at a time
  static constexpr int EPT = kTile / TPP;         // elements of a tile per thread
  static constexpr int BPT = (kTile * NP + kScanThreads - 1) / kScanThreads;   // of B or C
};

constexpr int kWanted = 1536;   // workgroups of a split call (scan_runs)
inline int scan_lanes(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
inline int scan_width(int N) {   // Geo<scan_lanes(N)>::CB
  const int ln = scan_lanes(N);
  return (ln == 4 || ln == 8 ? 512 : 256) / ln;
}

// Sum over the LN lanes of a channel, in all of them.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
template <int LN>
__device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (LN > 1) x = dpp_add<0xb1>(x);    // lane ^ 1
  if constexpr (LN > 2) x = dpp_add<0x4e>(x);    // lane ^ 2
  if constexpr (LN > 4) x = dpp_add<0x141>(x);   // 7 - lane % 8
  if constexpr (LN > 8) x = dpp_add<0x140>(x);   // 15 - lane % 16
  asm volatile("" : "+v"(x));   // the last addition stays here, in one instruction with its permutation
  return x;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A log2 e within fp32's finite range: a step of zero then decays nothing for
// an A of -inf too (which a tile's empty tokens rely on).
__device__ __forceinline__ float log2_rate(float A) {
  const float v = A * kLog2e;
  return v < -FLT_MAX ? -FLT_MAX : v > FLT_MAX ? FLT_MAX : v;
}

// A state h, or an adjoint, through a run whose decay is 2^t, and what the run adds to it.  A
// state of zero takes nothing through, also where 2^t is infinite (rates above
// zero, or steps below it), and one that is in range before and behind the run
// arrives where 2^t is not: then h takes it in four equal parts.
__device__ __forceinline__ float through_run(float t, float h, float end) {
  const bool far = !(fabsf(t) <= 126.0f);
  const float f = exp2_hw(far ? 0.25f * t : t);
  float v = h;
  if (far) v = v * f * f * f;
  return h == 0.0f ? end : __builtin_fmaf(f, v, end);
}

// Four states from index n of a row of N.
__device__ __forceinline__ float4 load_states(const float* p, int n, int N) {
  if ((N & 3) == 0) return n < N ? *reinterpret_cast<const float4*>(p + n) : make_float4(0, 0, 0, 0);
  return make_float4(n < N ? p[n] : 0.0f, n + 1 < N ? p[n + 1] : 0.0f, n + 2 < N ? p[n + 2] : 0.0f,
                     n + 3 < N ? p[n + 3] : 0.0f);
}
__device__ __forceinline__ void store_states(float* p, int n, int N, float4 v) {
  if ((N & 3) == 0) {
    if (n < N) *reinterpret_cast<float4*>(p + n) = v;
    return;
  }
  if (n < N) p[n] = v.x;
  if (n + 1 < N) p[n + 1] = v.y;
  if (n + 2 < N) p[n + 2] = v.z;
  if (n + 3 < N) p[n + 3] = v.w;
}
__device__ __forceinline__ void unpack(float4 v, float (&x)[4]) {
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}

// All the states of a channel, zeros behind the last, as the caller's tensors
// hold them (side by side) and as the kernels keep them: NP states of all
// channels, a state of a wave's channels side by side.
template <int NP>
__device__ __forceinline__ void load_row(const float* p, int N, float (&v)[NP]) {
#pragma unroll
  for (int j = 0; j < NP; ++j) v[j] = p[min(j, N - 1)];
#pragma unroll
  for (int j = 0; j < NP; ++j) v[j] = j < N ? v[j] : 0.0f;
}
template <int NP>
__device__ __forceinline__ void store_row(float* p, int N, const float (&v)[NP]) {
#pragma unroll
  for (int j = 0; j < NP; ++j)
    if (j < N) p[j] = v[j];
}
template <int NP>
__device__ __forceinline__ void load_kept(const float* p, int D, uint32_t d, float (&v)[NP]) {
#pragma unroll
  for (int j = 0; j < NP; ++j) v[j] = (p + (int64_t)j * D)[d];
}
template <int NP>
__device__ __forceinline__ void store_kept(float* p, int D, uint32_t d, const float (&v)[NP]) {
#pragma unroll
  for (int j = 0; j < NP; ++j) (p + (int64_t)j * D)[d] = v[j];
}
inline int kept_states(int N) { return 4 * scan_lanes(N); }

// Waves of a SIMD in the kernels with a lane per channel: the loads of tokens
// ahead and other tokens' decays take the registers that are left.
constexpr int fwd_waves(int NP) { return NP <= 16 ? 4 : NP <= 32 ? 3 : 2; }

// B or C of a tile on the way from memory to LDS.
template <class TT, int NP>
struct Rows16 {
  static constexpr int kEach = (kTile * NP + kScanThreads - 1) / kScanThreads;
  typename TT::S v[kEach];
  // the tile's first token, tokens, states; row stride (a tile's offsets fit 32 bits)
  __device__ __forceinline__ void load(const typename TT::S* p, uint32_t step, int n, int N) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t e = threadIdx.x + i * kScanThreads;
      v[i] = p[(uint32_t)min((int)(e / NP), n - 1) * step + (uint32_t)min((int)(e % NP), N - 1)];
    }
  }
  __device__ __forceinline__ void write(float4* to, int n, int N) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = threadIdx.x + i * kScanThreads;
      if (e < kTile * NP) reinterpret_cast<float*>(to)[e] = e / NP < n && e % NP < N ? TT::load(v[i]) : 0.0f;
    }
  }
};

// What a workgroup works on.
struct Place {
  Run run;
  int t0, n;     // its tokens within the sequence
  int g, d0, nc; // group, first channel, channels
  __device__ __forceinline__ bool init(const ScanArgs& a, int CB) {
    const int per = a.G * a.ncb;
    const int at = blockIdx.x / per, blk = blockIdx.x % per;
    g = blk / a.ncb;
    const int c0 = (blk % a.ncb) * CB;
    d0 = g * a.Dg + c0;
    nc = min(CB, a.Dg - c0);
    if (at >= a.nruns) {
      run.seq = -1;
      return false;
    }
    run = run_of(a.seqs, at, a.R);
    t0 = run.c * a.R;
    n = min(a.R, run.len - t0);
    return run.seq >= 0;
  }
};

int scan_check(const ScanArgs& a, int dtype, const char* what);
void scan_runs(ScanArgs& a, int width, int wanted, double chain, double busy, double extra);
bool scan_fits(const ScanArgs& a);

}  // namespace ssm
}  // namespace uttt
