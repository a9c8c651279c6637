// The gated delta rule token by token for gfx950: a few tokens per sequence
// against states [slots, Hv, Dk, Dv] fp32 that are updated in place.
//   p = S^T k, w = S^T q;  u = b (v - e^g p);  o = s (e^g w + (q.k) u);  S = e^g S + k u^T
// Both products of a token come from one pass over the state, so it is read
// once and written once per call whatever the tokens: 8 bytes per element,
// which is what bounds it.  A workgroup holds a block of one head's columns in
// registers, a lane four of them (16 bytes) of every (256 / LC)-th row.  250
// rows of 16 heads of 128 x 128: 91 us, 5.7 TB/s; one row of 4 heads of 192 x
// 192: 5.6 us.
//
// Rows whose slot is that of an earlier row are taken up by that row's
// workgroup, after it and in order, so that a slot named twice is two calls in
// a row and not a race.
#include "delta.h"

namespace uttt {
namespace delta {
namespace {

struct StepArgs {
  const void *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const void *g, *beta;   // [B, T, Hv]
  int g_dtype, beta_dtype;
  int B, T, Hk, Hv, Dk, Dv, slots;
  float scale;
  float* state;
  int64_t s_slot;
  const void* idx;        // [B] or null: row b has slot b
  int idx64;
  void* out;              // [B, T, Hv, Dv]
};

constexpr int kStepThreads = 256;

__device__ __forceinline__ int64_t slot_of(const StepArgs& a, int b) {
  const int64_t s = a.idx == nullptr ? b
                    : a.idx64        ? static_cast<const int64_t*>(a.idx)[b]
                                     : static_cast<const int32_t*>(a.idx)[b];
  return s >= 0 && s < a.slots ? s : -1;
}

// The tokens of row b on the workgroup's columns.  LC lanes of a wave cover 4
// LC columns; RPT rows of the state per lane.
template <class TT, int LC, int RPT>
__device__ __forceinline__ void step_row(const StepArgs& a, int b, int hv, int c4, bool live,
                                         f32x4 (&S)[RPT], float (&kq)[2][256],
                                         f32x4 (&part)[2][kStepThreads / 64][LC]) {
  using E = typename TT::S;
  constexpr int RG = kStepThreads / LC;   // row groups
  const int tid = threadIdx.x, lc = tid % LC, rg = tid / LC, wave = tid >> 6;
  const int hk = hv / (a.Hv / a.Hk);
  for (int t = 0; t < a.T; ++t) {
    const E* kp = static_cast<const E*>(a.k) + b * a.k_sb + t * a.k_st + hk * a.k_sh;
    const E* qp = static_cast<const E*>(a.q) + b * a.q_sb + t * a.q_st + hk * a.q_sh;
    __syncthreads();   // the last token's reads of kq and part are done
    if (tid < a.Dk) {
      kq[0][tid] = TT::load(kp[tid]);
      kq[1][tid] = TT::load(qp[tid]);
    }
    const int64_t at = ((int64_t)b * a.T + t) * a.Hv + hv;
    const float alpha = expf(load_any(a.g, a.g_dtype, at));
    const float beta = load_any(a.beta, a.beta_dtype, at);
    f32x4 v = {};
    if (live) {
      const E* vp = static_cast<const E*>(a.v) + b * a.v_sb + t * a.v_st + hv * a.v_sh + c4;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = TT::load(vp[i]);
    }
    __syncthreads();
    f32x4 p = {}, w = {};
    float qk = 0.0f;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int f = rg + i * RG;
      const float kf = f < a.Dk ? kq[0][f] : 0.0f, qf = f < a.Dk ? kq[1][f] : 0.0f;
      p += S[i] * kf;
      w += S[i] * qf;
      qk = __builtin_fmaf(qf, kf, qk);
    }
    // over the row groups: those of a wave, then the waves' sums
#pragma unroll
    for (int d = LC; d < 64; d <<= 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] += __shfl_xor(p[i], d);
        w[i] += __shfl_xor(w[i], d);
      }
      qk += __shfl_xor(qk, d);
    }
    __shared__ float qks[kStepThreads / 64];
    if ((tid & 63) < LC) {
      part[0][wave][lc] = p;
      part[1][wave][lc] = w;
      if ((tid & 63) == 0) qks[wave] = qk;
    }
    __syncthreads();
    p = part[0][0][lc];
    w = part[1][0][lc];
    qk = qks[0];
#pragma unroll
    for (int x = 1; x < kStepThreads / 64; ++x) {
      p += part[0][x][lc];
      w += part[1][x][lc];
      qk += qks[x];
    }
    const f32x4 u = beta * (v - alpha * p);
    if (live && rg == 0) {
      E* op = static_cast<E*>(a.out) + at * a.Dv + c4;
#pragma unroll
      for (int i = 0; i < 4; ++i) op[i] = TT::store(a.scale * (alpha * w[i] + qk * u[i]));
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int f = rg + i * RG;
      S[i] = S[i] * alpha + u * (f < a.Dk ? kq[0][f] : 0.0f);
    }
  }
}

template <class TT, int LC, int RPT>
__global__ __launch_bounds__(kStepThreads) void delta_step_kernel(StepArgs a) {
  __shared__ float kq[2][256];
  __shared__ f32x4 part[2][kStepThreads / 64][LC];
  __shared__ int next_s;
  constexpr int RG = kStepThreads / LC;
  const int tid = threadIdx.x, lc = tid % LC, rg = tid / LC;
  const int ncb = (a.Dv + 4 * LC - 1) / (4 * LC);
  const int cb = blockIdx.x % ncb, bh = blockIdx.x / ncb;
  int b = bh / a.Hv;
  const int hv = bh % a.Hv;
  const int c4 = cb * 4 * LC + 4 * lc;
  const bool live = c4 < a.Dv;
  const int64_t slot = slot_of(a, b);
  if (slot < 0) {   // a padded row: zeros, no state
    if (live)
      for (int t = rg; t < a.T; t += RG)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          static_cast<typename TT::S*>(a.out)[(((int64_t)b * a.T + t) * a.Hv + hv) * a.Dv + c4 + i] =
              TT::store(0.0f);
    return;
  }
  float* sp = a.state + slot * a.s_slot + ((int64_t)hv * a.Dk) * a.Dv + c4;
  f32x4 S[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int f = rg + i * RG;
    f32x4 x = {};
    if (live && f < a.Dk) x = *reinterpret_cast<const f32x4*>(sp + (int64_t)f * a.Dv);
    S[i] = x;
  }
  if (a.idx) {
    bool before = false;
    for (int j = tid; j < b; j += kStepThreads) before |= slot_of(a, j) == slot;
    if (__syncthreads_or(before)) return;
  }
  for (;;) {
    step_row<TT, LC, RPT>(a, b, hv, c4, live, S, kq, part);
    if (!a.idx) break;
    if (tid == 0) next_s = a.B;
    __syncthreads();
    int mine = a.B;
    for (int j = b + 1 + tid; j < a.B; j += kStepThreads)
      if (slot_of(a, j) == slot) {
        mine = j;
        break;
      }
    if (mine < a.B) atomicMin(&next_s, mine);
    __syncthreads();
    b = next_s;
    if (b >= a.B) break;
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int f = rg + i * RG;
    if (live && f < a.Dk) *reinterpret_cast<f32x4*>(sp + (int64_t)f * a.Dv) = S[i];
  }
}

int64_t step_blocks(const StepArgs& a, int LC) { return (int64_t)a.B * a.Hv * ((a.Dv + 4 * LC - 1) / (4 * LC)); }

template <class TT, int LC, int RPT>
void launch_step_as(const StepArgs& a, hipStream_t st) {
  const int64_t blocks = step_blocks(a, LC);
  hipLaunchKernelGGL((delta_step_kernel<TT, LC, RPT>), dim3((unsigned)blocks), dim3(kStepThreads), 0,
                     st, a);
}

template <class TT>
int launch_step(const StepArgs& a, hipStream_t st) {
  // 16 columns a workgroup, whose rows are only 64 bytes, where 64 columns make
  // less than 64 workgroups: 32 (16 heads of 128 x 128) 4.4 us against 4.8, 16
  // (4 of 256 x 256) 4.8 against 6.0; with 64 of them 5.0 against 4.9 and 6.3
  // against 6.5, with 256 10.0 against 5.9 and 15.0 against 8.8
  const bool narrow = step_blocks(a, 16) < 64;
  if (narrow) {
    if (a.Dk <= 64) launch_step_as<TT, 4, 1>(a, st);
    else if (a.Dk <= 128) launch_step_as<TT, 4, 2>(a, st);
    else launch_step_as<TT, 4, 4>(a, st);
  } else {
    if (a.Dk <= 64) launch_step_as<TT, 16, 4>(a, st);
    else if (a.Dk <= 128) launch_step_as<TT, 16, 8>(a, st);
    else launch_step_as<TT, 16, 16>(a, st);
  }
  return check_launch("delta_step");
}

}  // namespace
}  // namespace delta
}  // namespace uttt

using namespace uttt;
using namespace uttt::delta;

extern "C" int uttt_gated_delta_step(const void* q, const int64_t* q_strides, const void* k,
                                     const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, int dtype, const void* g, int g_dtype,
                                     const void* beta, int beta_dtype, int B, int T, int Hk, int Hv,
                                     int Dk, int Dv, float scale, float* state, int64_t state_stride,
                                     int slots, const void* indices, int indices_int64, void* out,
                                     void* stream) {
  const char* what = "uttt_gated_delta_step";
  UTTT_REQUIRE(B >= 0 && T >= 0 && Hk >= 1 && Hv >= 1 && slots >= 0,
               "%s: bad sizes B=%d T=%d Hk=%d Hv=%d slots=%d", what, B, T, Hk, Hv, slots);
  UTTT_REQUIRE(Hv % Hk == 0, "%s: Hv=%d must be a multiple of Hk=%d", what, Hv, Hk);
  UTTT_REQUIRE(Dk >= 1 && Dk <= 256, "%s: Dk=%d must be at most 256", what, Dk);
  UTTT_REQUIRE(Dv >= 4 && Dv % 4 == 0, "%s: Dv=%d must be a multiple of 4", what, Dv);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(g_dtype) && dtype_bytes(beta_dtype),
               "%s: dtype codes %d, %d, %d", what, dtype, g_dtype, beta_dtype);
  UTTT_REQUIRE(indices || B <= slots, "%s: %d rows without indices, %d slots", what, B, slots);
  // of 256 threads, and a launch has fewer than 2^32
  UTTT_REQUIRE((int64_t)B * Hv * ((Dv + 63) / 64) < (1LL << 24), "%s: too many rows and heads", what);
  if (B == 0 || T == 0) return UTTT_OK;
  UTTT_REQUIRE(q && k && v && g && beta && state && out && q_strides && k_strides && v_strides,
               "%s: null pointer", what);
  UTTT_REQUIRE((reinterpret_cast<uintptr_t>(state) & 15u) == 0 && state_stride % 4 == 0 &&
                   state_stride >= (int64_t)Hv * Dk * Dv,
               "%s: states must be 16-byte aligned, %lld elements apart", what, (long long)state_stride);
  const StepArgs a{q, k, v, q_strides[0], q_strides[1], q_strides[2], k_strides[0], k_strides[1],
                   k_strides[2], v_strides[0], v_strides[1], v_strides[2], g, beta, g_dtype,
                   beta_dtype, B, T, Hk, Hv, Dk, Dv, slots, scale, state, state_stride, indices,
                   indices_int64, out};
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return launch_step<TT>(a, as_stream(stream)));
  return UTTT_OK;
}
