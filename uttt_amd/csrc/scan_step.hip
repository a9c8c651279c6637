// The selective state space scan token by token for gfx950 (formulas: scan.h):
// a few tokens per row against states [slots, D, N] fp32 that are updated in
// place.  The states are read once and written once per call, 8 bytes each,
// which is what bounds it; a lane has four states of one channel (16 bytes).
// 250 rows of 1536 channels of 16 states: 17.6 to 17.9 us, 52 MB at 2.9 to 3.0 TB/s;
// one row: 4.1 us.
#include "rows.h"
#include "scan.h"

namespace uttt {
namespace ssm {
namespace {

struct ScanStepArgs {
  const void *x, *dt, *Bm, *Cm, *z;
  int64_t x_sb, x_st, dt_sb, dt_st, z_sb, z_st, B_sb, B_st, B_sg, C_sb, C_st, C_sg;
  int dt_dtype, soft;
  const float *A, *Dskip, *bias;
  int B, T, D, N, Dg, slots;
  float* state;
  int64_t s_slot;
  const void* idx;
  int idx64;
  void* out;   // [B, T, D]
};

// WHOLE: B and C can be read four elements at a time.
template <class TT, int LN, bool WHOLE>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(ScanStepArgs a) {
  using S = typename TT::S;
  constexpr int CB = kScanThreads / LN;   // channels of a workgroup
  const int ncb = (a.D + CB - 1) / CB;
  const int ln = threadIdx.x % LN, at = (int)(blockIdx.x % ncb) * CB + threadIdx.x / LN;
  Rows rows{a.idx, a.idx64, a.B, a.slots};
  int b = blockIdx.x / ncb;
  const int64_t slot = rows.slot_of(b);
  const bool writes = at < a.D;
  if (slot < 0) {   // a padded row: zeros, no state
    if (ln == 0 && writes)
      for (int t = 0; t < a.T; ++t) static_cast<S*>(a.out)[((int64_t)b * a.T + t) * a.D + at] = TT::store(0.0f);
    return;
  }
  const int d = min(at, a.D - 1), g = d / a.Dg;   // a lane without a channel reads the last one
  float* sp = a.state + slot * a.s_slot + (int64_t)d * a.N;
  float h[4], A2[4];
  unpack(load_states(sp, 4 * ln, a.N), h);
  unpack(load_states(a.A + (int64_t)d * a.N, 4 * ln, a.N), A2);
  const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
  const int others = rows.others<kScanThreads>(b, slot);
  if (others & 1) return;   // an earlier row's workgroup takes this one up
#pragma unroll
  for (int j = 0; j < 4; ++j) A2[j] = log2_rate(A2[j]);
  for (;;) {
    for (int t = 0; t < a.T; ++t) {
      const float x = TT::load((static_cast<const S*>(a.x) + b * a.x_sb + t * a.x_st)[d]);
      const float raw = load_any(a.dt, a.dt_dtype, b * a.dt_sb + t * a.dt_st + d) + bias;
      const float z = a.z ? TT::load((static_cast<const S*>(a.z) + b * a.z_sb + t * a.z_st)[d]) : 0.0f;
      const S* Bp = static_cast<const S*>(a.Bm) + b * a.B_sb + t * a.B_st + g * a.B_sg;
      const S* Cp = static_cast<const S*>(a.Cm) + b * a.C_sb + t * a.C_st + g * a.C_sg;
      float bm[4], cm[4];
      if constexpr (WHOLE) {
        const int n = min(4 * ln, a.N - 4);
        load_piece<TT, 4>(Bp + n, bm);
        load_piece<TT, 4>(Cp + n, cm);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = min(4 * ln + j, a.N - 1);
          bm[j] = TT::load(Bp[n]);
          cm[j] = TT::load(Cp[n]);
        }
      }
      const float dt = a.soft ? softplus(raw) : raw, u = dt * x;
      float y = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = __builtin_fmaf(exp2_hw(dt * A2[j]), h[j], u * bm[j]);
        if (4 * ln + j < a.N) y = __builtin_fmaf(cm[j], h[j], y);
      }
      y = __builtin_fmaf(skip, x, sum_lanes<LN>(y));
      if (a.z) y *= z * sigmoid_for<TT>(z);
      if (ln == 0 && writes) static_cast<S*>(a.out)[((int64_t)b * a.T + t) * a.D + d] = TT::store(y);
    }
    if (!(others & 2)) break;
    b = rows.next_of<kScanThreads>(b, slot);
    if (b >= a.B) break;
  }
  if (writes) store_states(sp, 4 * ln, a.N, make_float4(h[0], h[1], h[2], h[3]));
}

template <class TT, int LN>
void launch_step_as(const ScanStepArgs& a, hipStream_t st) {
  constexpr int CB = kScanThreads / LN, size = 4 * sizeof(typename TT::S);
  // four elements of B and C at a time where they lie so (250 rows of 1536 x 16
  // in bf16: 18 us, with single elements 23)
  const dim3 blocks((unsigned)(a.B * (int64_t)((a.D + CB - 1) / CB)));
  const int64_t steps = a.B_sb | a.B_st | a.B_sg | a.C_sb | a.C_st | a.C_sg | a.N;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.Bm) | reinterpret_cast<uintptr_t>(a.Cm);
  if (steps % 4 == 0 && at % size == 0)
    hipLaunchKernelGGL((scan_step_kernel<TT, LN, true>), blocks, dim3(kScanThreads), 0, st, a);
  else
    hipLaunchKernelGGL((scan_step_kernel<TT, LN, false>), blocks, dim3(kScanThreads), 0, st, a);
}

template <class TT>
int launch_step(const ScanStepArgs& a, hipStream_t st) {
  switch (scan_lanes(a.N)) {
    case 1: launch_step_as<TT, 1>(a, st); break;
    case 2: launch_step_as<TT, 2>(a, st); break;
    case 4: launch_step_as<TT, 4>(a, st); break;
    case 8: launch_step_as<TT, 8>(a, st); break;
    default: launch_step_as<TT, 16>(a, st);
  }
  return check_launch("selective_scan_step");
}

}  // namespace
}  // namespace ssm
}  // namespace uttt

using namespace uttt;
using namespace uttt::ssm;

extern "C" int uttt_selective_scan_step(const void* x, const int64_t* x_strides, int dtype, const void* dt,
                                        const int64_t* dt_strides, int dt_dtype, const float* A, const void* Bm,
                                        const int64_t* B_strides, const void* Cm, const int64_t* C_strides,
                                        const float* skip, const void* gate, const int64_t* gate_strides,
                                        const float* dt_bias, int dt_softplus, int B, int T, int D, int N, int G,
                                        float* state, int64_t state_stride, int slots, const void* indices,
                                        int indices_int64, void* out, void* stream) {
  const char* what = "uttt_selective_scan_step";
  UTTT_REQUIRE(B >= 0 && T >= 0 && slots >= 0, "%s: bad sizes B=%d T=%d slots=%d", what, B, T, slots);
  UTTT_REQUIRE(D >= 1 && G >= 1 && D % G == 0, "%s: D=%d must be a multiple of G=%d", what, D, G);
  UTTT_REQUIRE(N >= 1 && N <= kMaxStates, "%s: N=%d must be at most %d", what, N, kMaxStates);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(dt_dtype), "%s: dtype codes %d, %d", what, dtype, dt_dtype);
  UTTT_REQUIRE(indices || B <= slots, "%s: %d rows without indices, %d slots", what, B, slots);
  const int cb = kScanThreads / scan_lanes(N);
  UTTT_REQUIRE((int64_t)B * ((D + cb - 1) / cb) < (1LL << 24), "%s: too many rows and channels", what);
  if (B == 0 || T == 0) return UTTT_OK;
  UTTT_REQUIRE(x && dt && A && Bm && Cm && out && x_strides && dt_strides && B_strides && C_strides &&
                   (gate_strides || !gate) && (state || slots == 0),
               "%s: null pointer", what);
  UTTT_REQUIRE(state_stride >= (int64_t)D * N, "%s: states %lld elements apart", what, (long long)state_stride);
  UTTT_REQUIRE(N % 4 || (((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(A)) & 15u) == 0 &&
                         state_stride % 4 == 0),
               "%s: A and states must be 16-byte aligned", what);
  ScanStepArgs a{};
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = gate;
  a.x_sb = x_strides[0]; a.x_st = x_strides[1];
  a.dt_sb = dt_strides[0]; a.dt_st = dt_strides[1];
  a.B_sb = B_strides[0]; a.B_st = B_strides[1]; a.B_sg = B_strides[2];
  a.C_sb = C_strides[0]; a.C_st = C_strides[1]; a.C_sg = C_strides[2];
  if (gate) { a.z_sb = gate_strides[0]; a.z_st = gate_strides[1]; }
  a.dt_dtype = dt_dtype; a.soft = dt_softplus;
  a.A = A; a.Dskip = skip; a.bias = dt_bias;
  a.B = B; a.T = T; a.D = D; a.N = N; a.Dg = D / G; a.slots = slots;
  a.state = state; a.s_slot = state_stride; a.idx = indices; a.idx64 = indices_int64; a.out = out;
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return launch_step<TT>(a, as_stream(stream)));
  return UTTT_OK;
}
