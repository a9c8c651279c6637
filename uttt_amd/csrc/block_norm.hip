// The RMS norms around a block for gfx950, with the residual sum, the gate and
// the residual's scale that stand next to them, forward and backward, over rows
// of N elements (rstd = 1 / sqrt(sum(v^2) / N + eps) of the normed row v):
//   after:   y = r + s (x rstd) w silu(z), without what is not given
//     with n = x rstd, f = silu(z), o = s dy:  dr = dy, ds = sum_rows(dy n w f),
//     dz = o n w silu'(z), dw = sum_rows(o n f), m = o w f,
//     dx = rstd (m - n sum(m n) / N)
//   before:  h = r + s x,  y = (h rstd) w
//     with n = h rstd, m = dy w:  dw = sum_rows(dy n),
//     dr = dh + rstd (m - n sum(m n) / N),  dx = s dr, ds = sum_rows(x dr)
// s is `alpha` times a learned [N], or alpha alone.
//
// Bound by memory: every tensor is read or written once.  A row stays in
// registers between its two passes (LPR lanes, NI pieces of V elements each).  Rows
// that no 16 bytes divide (N, strides or addresses off 8 elements, in fp32 too) are
// read by single elements: 32 768 rows of 772 before a block with a scale, both
// directions, 460 us in bf16 and 433 in fp32, of 768 161 and 204.
// The sums over rows for dw and ds stay in registers while a workgroup walks
// over its rows, and are added by a second launch; what a backward needs of a
// row again it reads again from its inputs, so that nothing is rounded twice.
#include "rows.h"
#include "state_space.h"

namespace uttt {
namespace {

using ssm::launch_sums;
using ssm::sigmoid_for;

constexpr int kMaxRow = 8192;

// Row i of a tensor of rows in groups of `heads`: at i / heads * outer + i % heads * inner.
struct Row {
  uint32_t group, head;
  __device__ __forceinline__ Row(int64_t row, int heads)
      : group((uint32_t)row / (uint32_t)heads), head((uint32_t)row - group * (uint32_t)heads) {}
};
struct RowsOf {
  const void* p;
  int64_t outer, inner;
  __device__ __forceinline__ int64_t at(Row r) const { return r.group * outer + r.head * inner; }
};

struct NormArgs {
  RowsOf x, z, r, dy, dh;   // z: after; dh: before; p null where not given
  const void *w, *s;        // [N] or null
  int w_dtype, s_dtype;
  float alpha, eps;
  int r_dtype, y_dtype;     // of r, h, dr and dh; of y and dy
  int64_t rows;
  int heads, N;
  void *y, *h;              // contiguous
  float* rstd;              // [rows] or null
  void *dx, *dz, *dr;       // contiguous; dr: before
  float *part_w, *part_s;   // [workgroups, N] or null
};

template <int LPR, int THREADS>
__device__ __forceinline__ float row_sum(float a, float* red) {
#pragma unroll
  for (int d = (LPR < 64 ? LPR : 64) / 2; d > 0; d >>= 1) a += __shfl_xor(a, d);
  if constexpr (LPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    a = red[0];
#pragma unroll
    for (int i = 1; i < LPR / 64; ++i) a += red[i];
  }
  return a;
}

template <class TT, int V, int LPR, int NI, bool AFTER, bool SCALE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_fwd_kernel(NormArgs a) {
  using S = typename TT::S;
  constexpr int THREADS = LPR > 256 ? LPR : 256, RPB = THREADS / LPR;
  __shared__ float red[16];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  float w[NI][V], s[NI][V];   // for all the rows that the workgroup walks over
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    const int e = (lane + LPR * c) * V;
    if (e < a.N) {
      load_weights<V>(a.w, a.w_dtype, e, 1.0f, w[c]);
      if (SCALE) load_weights<V>(a.s, a.s_dtype, e, 1.0f, s[c]);
#pragma unroll
      for (int i = 0; i < V; ++i) s[c][i] = SCALE ? s[c][i] * a.alpha : a.alpha;
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += (int64_t)gridDim.x * RPB) {
    const bool live = base + slot < a.rows;
    const int64_t row = live ? base + slot : a.rows - 1;
    const Row at(row, a.heads);
    const S* x = static_cast<const S*>(a.x.p) + a.x.at(at);
    const int64_t r0 = a.r.p ? a.r.at(at) : 0, z0 = a.z.p ? a.z.at(at) : 0;
    float v[NI][V], o[NI][V];   // what is normed; the residual
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = 0.0f;
      if (e < a.N) {
        load_piece<TT, V>(x + e, v[c]);
        load_weights<V>(a.r.p, a.r_dtype, r0 + e, 0.0f, o[c]);
        if constexpr (!AFTER)
#pragma unroll
          for (int i = 0; i < V; ++i) v[c][i] = __builtin_fmaf(v[c][i], s[c][i], o[c][i]);
      }
    }
#pragma unroll
    for (int c = 0; c < NI; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) sq = __builtin_fmaf(v[c][i], v[c][i], sq);
    const float rstd = 1.0f / sqrtf(row_sum<LPR, THREADS>(sq, red) / (float)a.N + a.eps);
    if (!live) continue;   // whole rows: no later exchange in this turn
    if (a.rstd && lane == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e >= a.N) continue;
      if constexpr (!AFTER) store_piece_as<V>(a.h, a.r_dtype, row * a.N + e, v[c]);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = v[c][i] * rstd * w[c][i];
      if constexpr (AFTER) {
        if (a.z.p) {
          float z[V];
          load_piece<TT, V>(static_cast<const S*>(a.z.p) + z0 + e, z);
#pragma unroll
          for (int i = 0; i < V; ++i) v[c][i] *= z[i] * sigmoid_for<TT>(z[i]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = __builtin_fmaf(v[c][i], s[c][i], o[c][i]);
      }
      store_piece_as<V>(a.y, a.y_dtype, row * a.N + e, v[c]);
    }
  }
}

template <class TT, int V, int LPR, int NI, bool AFTER, bool SCALE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_bwd_kernel(NormArgs a) {
  using S = typename TT::S;
  constexpr int THREADS = LPR > 256 ? LPR : 256, RPB = THREADS / LPR;
  __shared__ float red[16];
  __shared__ float tot[RPB > 1 ? 2 * LPR * V : 1];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  float w[NI][V], s[NI][V], dw[NI][V], ds[NI][V];
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    const int e = (lane + LPR * c) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) dw[c][i] = ds[c][i] = 0.0f;
    if (e < a.N) {
      load_weights<V>(a.w, a.w_dtype, e, 1.0f, w[c]);
      if (SCALE) load_weights<V>(a.s, a.s_dtype, e, 1.0f, s[c]);
#pragma unroll
      for (int i = 0; i < V; ++i) s[c][i] = SCALE ? s[c][i] * a.alpha : a.alpha;
    }
  }
  const float inv_n = 1.0f / (float)a.N;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += (int64_t)gridDim.x * RPB) {
    const bool live = base + slot < a.rows;
    const int64_t row = live ? base + slot : a.rows - 1;
    const Row at(row, a.heads);
    const S* x = static_cast<const S*>(a.x.p) + a.x.at(at);
    const int64_t g0 = a.dy.p ? a.dy.at(at) : 0;
    const float rstd = a.rstd[row];
    float n[NI][V], m[NI][V];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e >= a.N || !live) continue;
      load_piece<TT, V>(x + e, n[c]);
      load_weights<V>(a.dy.p, a.y_dtype, g0 + e, 0.0f, m[c]);
      if constexpr (AFTER) {
        float z[V], f[V], df[V];
        if (a.z.p) {
          load_piece<TT, V>(static_cast<const S*>(a.z.p) + a.z.at(at) + e, z);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float q = sigmoid_for<TT>(z[i]);
            f[i] = z[i] * q;
            df[i] = q * __builtin_fmaf(z[i], 1.0f - q, 1.0f);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          n[c][i] *= rstd;
          const float o = m[c][i] * s[c][i], nf = n[c][i] * f[i];
          if (SCALE) ds[c][i] = __builtin_fmaf(m[c][i], nf * w[c][i], ds[c][i]);
          dw[c][i] = __builtin_fmaf(o, nf, dw[c][i]);
          if (a.z.p) z[i] = o * n[c][i] * w[c][i] * df[i];
          m[c][i] = o * w[c][i] * f[i];
          sum = __builtin_fmaf(m[c][i], n[c][i], sum);
        }
        if (a.z.p) store_piece<TT, V>(static_cast<S*>(a.dz) + row * a.N + e, z);
      } else {
        float r[V];
        load_weights<V>(a.r.p, a.r_dtype, a.r.at(at) + e, 0.0f, r);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          n[c][i] = __builtin_fmaf(n[c][i], s[c][i], r[i]) * rstd;
          dw[c][i] = __builtin_fmaf(m[c][i], n[c][i], dw[c][i]);
          m[c][i] *= w[c][i];
          sum = __builtin_fmaf(m[c][i], n[c][i], sum);
        }
      }
    }
    sum = row_sum<LPR, THREADS>(sum, red) * inv_n;
    if (!live) continue;   // whole rows: no later exchange in this turn
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e >= a.N) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) m[c][i] = rstd * (m[c][i] - n[c][i] * sum);
      if constexpr (!AFTER) {
        float v[V];
        if (a.dh.p) {
          load_weights<V>(a.dh.p, a.r_dtype, a.dh.at(at) + e, 0.0f, v);
#pragma unroll
          for (int i = 0; i < V; ++i) m[c][i] += v[i];
        }
        store_piece_as<V>(a.dr, a.r_dtype, row * a.N + e, m[c]);
        if (SCALE) {
          load_piece<TT, V>(x + e, v);
#pragma unroll
          for (int i = 0; i < V; ++i) ds[c][i] = __builtin_fmaf(v[i], m[c][i], ds[c][i]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) m[c][i] *= s[c][i];
      }
      store_piece<TT, V>(static_cast<S*>(a.dx) + row * a.N + e, m[c]);
    }
  }
  if (!a.part_w && !a.part_s) return;
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    if constexpr (RPB > 1) {   // the workgroup's rows one after another
      for (int k = 0; k < RPB; ++k) {
        __syncthreads();
        if (slot == k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float* p = tot + (lane * V + i) * 2;
            p[0] = k ? p[0] + dw[c][i] : dw[c][i];
            p[1] = k ? p[1] + ds[c][i] : ds[c][i];
          }
      }
      __syncthreads();
    }
    if (slot == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = (lane + LPR * c) * V + i;
        if (e >= a.N) continue;
        const float tw = RPB > 1 ? tot[(lane * V + i) * 2] : dw[c][i];
        const float ts = RPB > 1 ? tot[(lane * V + i) * 2 + 1] : ds[c][i];
        if (a.part_w) a.part_w[(int64_t)blockIdx.x * a.N + e] = tw;
        if (a.part_s) a.part_s[(int64_t)blockIdx.x * a.N + e] = ts * a.alpha;
      }
  }
}

// Workgroups of the backward, each with 8 rows or more to walk over: 1280, 768 or
// 512, five, three or two a CU (32 768 rows of 768 before a block with a scale,
// three a CU by registers: 1024 of them 128 us, 768 99; 262 144 rows of 192 after a
// block without one: five.  Not every form fits so: with a scale after a block four
// of up to 512 elements stand on a CU, and one of 1024 threads, beyond 4096).  More
// where a thread would add more than 256 rows in a chain of fp32: rounding then
// leaves the same of a sum however many rows there are, and the sum over the
// workgroups is in 64 bits.  A function of the sizes alone, so that sums come out the
// same on every run.
int64_t bwd_blocks(int64_t rows, int N) {
  const int64_t per = N <= 64 ? 32 : 8, n = (rows + per - 1) / per;
  const int64_t once = N <= 64 ? 16 : N <= 256 ? 4 : 1;   // rows of a workgroup at a time, in any form
  const int64_t fill = N <= 512 ? 1280 : N <= 2048 ? 768 : 512, most = (rows + 256 * once - 1) / (256 * once);
  return n < fill ? n : fill > most ? fill : most;
}

template <class TT, int V, int LPR, int NI, bool AFTER, bool SCALE>
void launch_fwd(const NormArgs& a, hipStream_t st) {
  constexpr int THREADS = LPR > 256 ? LPR : 256, RPB = THREADS / LPR;
  int64_t blocks = (a.rows + RPB - 1) / RPB;
  if (blocks > 2048) blocks = 2048;   // 8 workgroups a CU: the weights are read once for many rows
  hipLaunchKernelGGL((norm_fwd_kernel<TT, V, LPR, NI, AFTER, SCALE>), dim3((unsigned)blocks), dim3(THREADS), 0, st, a);
}
template <class TT, int V, int LPR, int NI, bool AFTER, bool SCALE>
void launch_bwd(const NormArgs& a, hipStream_t st) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  hipLaunchKernelGGL((norm_bwd_kernel<TT, V, LPR, NI, AFTER, SCALE>), dim3((unsigned)bwd_blocks(a.rows, a.N)),
                     dim3(THREADS), 0, st, a);
}
template <class TT, int V, int LPR, int NI, bool AFTER, bool SCALE>
void norm_launch(const NormArgs& a, bool bwd, hipStream_t st) {
  if (bwd) launch_bwd<TT, V, LPR, NI, AFTER, SCALE>(a, st);
  else launch_fwd<TT, V, LPR, NI, AFTER, SCALE>(a, st);
}

bool whole_pieces(const NormArgs& a, int size) {
  uintptr_t all = 0;
  for (const RowsOf* t : {&a.x, &a.z, &a.r, &a.dy, &a.dh})
    all |= reinterpret_cast<uintptr_t>(t->p) | (uintptr_t)((t->outer | t->inner) * size);
  for (const void* p : {(const void*)a.w, (const void*)a.s, (const void*)a.y, (const void*)a.h, (const void*)a.dx,
                        (const void*)a.dz, (const void*)a.dr})
    all |= reinterpret_cast<uintptr_t>(p);
  return ((all | (uintptr_t)((int64_t)a.N * size)) & 15u) == 0;
}

template <class TT, bool AFTER, bool SCALE>
int norm_rows(const NormArgs& a, bool bwd, hipStream_t st) {
  constexpr int V = 16 / sizeof(typename TT::S);
  // V elements of another type are 8 bytes or two pieces of 16; with all strides
  // and N multiples of 8 elements each lies right
  if (whole_pieces(a, 2)) {
    const int pieces = (a.N + V - 1) / V;
    // 24 pieces (heads of 192 in 16 bits): forward all of 8 lanes three times and
    // not 24 of 32 (70 us against 98 for 262 144 rows), backward that is more
    // registers than it gains (173 against 142)
    if (pieces <= 8) norm_launch<TT, V, 8, 1, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 16) norm_launch<TT, V, 16, 1, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 24 && !bwd) launch_fwd<TT, V, 8, 3, AFTER, SCALE>(a, st);
    else if (pieces <= 32) norm_launch<TT, V, 32, 1, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 64) norm_launch<TT, V, 64, 1, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 128) norm_launch<TT, V, 64, 2, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 256) norm_launch<TT, V, 256, 1, AFTER, SCALE>(a, bwd, st);
    else if (pieces <= 512) norm_launch<TT, V, 256, 2, AFTER, SCALE>(a, bwd, st);
    else if (V == 8 || pieces <= 1024) norm_launch<TT, V, 1024, 1, AFTER, SCALE>(a, bwd, st);   // 8192 elements at most
    else if constexpr (V == 4) norm_launch<TT, V, 1024, 2, AFTER, SCALE>(a, bwd, st);
  } else {
    if (a.N <= 64) norm_launch<TT, 1, 16, 4, AFTER, SCALE>(a, bwd, st);
    else if (a.N <= 256) norm_launch<TT, 1, 64, 4, AFTER, SCALE>(a, bwd, st);
    else if (a.N <= 1024) norm_launch<TT, 1, 256, 4, AFTER, SCALE>(a, bwd, st);
    else if (a.N <= 2048) norm_launch<TT, 1, 256, 8, AFTER, SCALE>(a, bwd, st);
    else norm_launch<TT, 1, 1024, 8, AFTER, SCALE>(a, bwd, st);
  }
  return check_launch(AFTER ? "norm_after_block" : "norm_before_block");
}

int norm_check(const NormArgs& a, int dtype, const char* what) {
  UTTT_REQUIRE(a.rows >= 0 && a.rows < (1LL << 31) && a.heads >= 1 && a.N >= 1 && a.N <= kMaxRow,
               "%s: bad sizes rows=%lld heads=%d N=%d", what, (long long)a.rows, a.heads, a.N);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(a.r_dtype) && dtype_bytes(a.y_dtype) && dtype_bytes(a.w_dtype) &&
                   dtype_bytes(a.s_dtype),
               "%s: dtype codes %d, %d, %d, %d, %d", what, dtype, a.r_dtype, a.y_dtype, a.w_dtype, a.s_dtype);
  UTTT_REQUIRE(a.rows == 0 || a.x.p, "%s: null pointer", what);
  return UTTT_OK;
}

RowsOf rows_of(const void* p, const int64_t* strides) {
  return p && strides ? RowsOf{p, strides[0], strides[1]} : RowsOf{nullptr, 0, 0};
}

template <bool AFTER>
int norm_run(const NormArgs& a, int dtype, bool bwd, void* workspace, size_t workspace_bytes, void* dweight,
             void* dscale, hipStream_t st, const char* what) {
  if (const int rc = norm_check(a, dtype, what)) return rc;
  if (a.rows == 0) {
    if (dweight)
      if (const int rc = zero_fill_async(dweight, (size_t)a.N * dtype_bytes(a.w_dtype), st, what)) return rc;
    return dscale ? zero_fill_async(dscale, (size_t)a.N * dtype_bytes(a.s_dtype), st, what) : UTTT_OK;
  }
  NormArgs b = a;
  const int64_t blocks = bwd_blocks(a.rows, a.N);
  if (dweight || dscale) {
    const size_t need = (size_t)blocks * 2 * a.N * 4;
    UTTT_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes,
                 need);
    float* p = static_cast<float*>(workspace);
    b.part_w = dweight ? p : nullptr;
    b.part_s = dscale ? p + (size_t)blocks * a.N : nullptr;
  }
  int rc = UTTT_OK;
  switch (dtype) {
    case UTTT_F32: rc = a.s ? norm_rows<F32T, AFTER, true>(b, bwd, st) : norm_rows<F32T, AFTER, false>(b, bwd, st); break;
    case UTTT_BF16: rc = a.s ? norm_rows<BF16T, AFTER, true>(b, bwd, st) : norm_rows<BF16T, AFTER, false>(b, bwd, st); break;
    default: rc = a.s ? norm_rows<F16T, AFTER, true>(b, bwd, st) : norm_rows<F16T, AFTER, false>(b, bwd, st); break;
  }
  if (rc) return rc;
  return launch_sums(blocks, {{b.part_w, a.N, dweight, b.w_dtype}, {b.part_s, a.N, dscale, b.s_dtype}}, st, what);
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_norm_after_fwd(const void* x, const int64_t* x_strides, int dtype, const void* weight, int weight_dtype,
                                   const void* gate, const int64_t* gate_strides, const void* residual,
                                   const int64_t* residual_strides, int out_dtype, const void* scale, int scale_dtype, float alpha,
                                   int64_t rows, int heads, int N, float eps, void* out, float* rstd, void* stream) {
  NormArgs a{};
  a.x = rows_of(x, x_strides); a.z = rows_of(gate, gate_strides); a.r = rows_of(residual, residual_strides);
  a.w = weight; a.s = scale; a.w_dtype = weight_dtype; a.s_dtype = scale_dtype; a.alpha = alpha; a.eps = eps;
  a.r_dtype = a.y_dtype = out_dtype;
  a.rows = rows; a.heads = heads; a.N = N; a.y = out; a.rstd = rstd;
  UTTT_REQUIRE(rows == 0 || out, "uttt_norm_after_fwd: null pointer");
  return norm_run<true>(a, dtype, false, nullptr, 0, nullptr, nullptr, as_stream(stream), "uttt_norm_after_fwd");
}

extern "C" int uttt_norm_before_fwd(const void* x, const int64_t* x_strides, int dtype, const void* residual,
                                    const int64_t* residual_strides, int residual_dtype, const void* weight, int weight_dtype,
                                    const void* scale, int scale_dtype, float alpha, int64_t rows, int heads, int N, float eps,
                                    void* out, void* sum, float* rstd, void* stream) {
  NormArgs a{};
  a.x = rows_of(x, x_strides); a.r = rows_of(residual, residual_strides);
  a.w = weight; a.s = scale; a.w_dtype = weight_dtype; a.s_dtype = scale_dtype; a.alpha = alpha; a.eps = eps;
  a.r_dtype = residual_dtype; a.y_dtype = dtype;
  a.rows = rows; a.heads = heads; a.N = N; a.y = out; a.h = sum; a.rstd = rstd;
  UTTT_REQUIRE(rows == 0 || (out && sum && a.r.p), "uttt_norm_before_fwd: null pointer");
  return norm_run<false>(a, dtype, false, nullptr, 0, nullptr, nullptr, as_stream(stream), "uttt_norm_before_fwd");
}

extern "C" size_t uttt_norm_bwd_workspace_bytes(int64_t rows, int N) {
  return rows <= 0 || N <= 0 ? 0 : (size_t)bwd_blocks(rows, N) * 2 * (size_t)N * 4;
}

extern "C" int uttt_norm_after_bwd(const void* x, const int64_t* x_strides, int dtype, const void* weight, int weight_dtype,
                                   const void* gate, const int64_t* gate_strides, const void* scale, int scale_dtype, float alpha,
                                   int64_t rows, int heads, int N, const float* rstd, const void* dout,
                                   const int64_t* dout_strides, int dout_dtype, void* dx, void* dgate, void* dweight,
                                   void* dscale, void* workspace, size_t workspace_bytes, void* stream) {
  NormArgs a{};
  a.x = rows_of(x, x_strides); a.z = rows_of(gate, gate_strides); a.dy = rows_of(dout, dout_strides);
  a.w = weight; a.s = scale; a.w_dtype = weight_dtype; a.s_dtype = scale_dtype; a.alpha = alpha;
  a.r_dtype = a.y_dtype = dout_dtype;
  a.rows = rows; a.heads = heads; a.N = N; a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.dz = dgate;
  UTTT_REQUIRE(rows == 0 || (rstd && a.dy.p && dx && (dgate || !gate)), "uttt_norm_after_bwd: null pointer");
  return norm_run<true>(a, dtype, true, workspace, workspace_bytes, dweight, dscale, as_stream(stream),
                        "uttt_norm_after_bwd");
}

extern "C" int uttt_norm_before_bwd(const void* x, const int64_t* x_strides, int dtype, const void* residual,
                                    const int64_t* residual_strides, int residual_dtype, const void* weight, int weight_dtype,
                                    const void* scale, int scale_dtype, float alpha, int64_t rows, int heads, int N, const float* rstd,
                                    const void* dout, const int64_t* dout_strides, const void* dsum,
                                    const int64_t* dsum_strides, void* dx, void* dresidual, void* dweight,
                                    void* dscale, void* workspace, size_t workspace_bytes, void* stream) {
  NormArgs a{};
  a.x = rows_of(x, x_strides); a.r = rows_of(residual, residual_strides);
  a.dy = rows_of(dout, dout_strides); a.dh = rows_of(dsum, dsum_strides);
  a.w = weight; a.s = scale; a.w_dtype = weight_dtype; a.s_dtype = scale_dtype; a.alpha = alpha;
  a.r_dtype = residual_dtype; a.y_dtype = dtype;
  a.rows = rows; a.heads = heads; a.N = N; a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.dr = dresidual;
  UTTT_REQUIRE(rows == 0 || (rstd && a.r.p && dx && dresidual), "uttt_norm_before_bwd: null pointer");
  return norm_run<false>(a, dtype, true, workspace, workspace_bytes, dweight, dscale, as_stream(stream),
                         "uttt_norm_before_bwd");
}
