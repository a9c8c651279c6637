// Layer norm over the rows of [rows, N] for gfx950, forward and backward.
//   mean = sum(x) / N, rstd = 1 / sqrt(sum((x - mean)^2) / N + eps)
//   y = (x - mean) rstd w + b
//   with h = (x - mean) rstd and d = dy w:
//   dx = rstd (d - sum(d) / N - h sum(d h) / N),  dw = sum_rows(dy h),  db = sum_rows(dy)
//
// Bound by memory: the forward reads x and writes y, the backward reads x and
// dy and writes dx, each once.  A row stays in registers between its
// reductions (LPR lanes, NI pieces of V elements each), the variance taken
// about the mean.  The backward's workgroups walk over the rows with a fixed
// grid; a lane's columns are the same in every row, so the sums for dw and db
// stay in registers too, and only their totals per workgroup are written, to
// be added in a fixed order by a second launch.  Rows too long for registers
// (over 2048 pieces of 16 bytes, or 8192 elements where no such piece divides
// them) are read again from cache for each pass, their sums in 64 bits.
// 65536 rows of 768 bf16: forward 46 us (4.4 TB/s), backward 65 (4.6) and the
// sum over the workgroups 5.
#include "common.h"

namespace uttt {
namespace {

constexpr int kLnThreads = 256;

struct LnArgs {
  const void* x;
  int64_t x_st;          // elements between rows
  const void *w, *b;     // [N] or null
  int w_dtype, b_dtype;
  int64_t rows;
  int N;
  float eps;
  void* y;               // [rows, N]; the backward's dx
  float* stats;          // [2, rows] mean, rstd; null where nobody keeps them
  const void* dy;        // [rows, N] rows dy_st apart
  int64_t dy_st;
  float* part;           // [workgroups, 2, N]
};

template <class TT, int V>
__device__ __forceinline__ void load_piece(const typename TT::S* p, float (&v)[V]) {
  typename TT::S w[V];
  __builtin_memcpy(w, __builtin_assume_aligned(p, sizeof w > 16 ? 16 : sizeof w), sizeof w);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = TT::load(w[i]);
}
template <class TT, int V>
__device__ __forceinline__ void store_piece(typename TT::S* p, const float (&v)[V]) {
  typename TT::S w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = TT::store(v[i]);
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof w), w, sizeof w);
}
// V weights from element e, `none` where there is no weight tensor.
template <int V>
__device__ __forceinline__ void load_weights(const void* p, int dtype, int e, float none, float (&v)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
  } else if (dtype == UTTT_F32) {
    load_piece<F32T, V>(static_cast<const float*>(p) + e, v);
  } else if (dtype == UTTT_BF16) {
    load_piece<BF16T, V>(static_cast<const uint16_t*>(p) + e, v);
  } else {
    load_piece<F16T, V>(static_cast<const uint16_t*>(p) + e, v);
  }
}
__device__ __forceinline__ float load_w(const void* p, int dtype, int i) {
  if (dtype == UTTT_F32) return static_cast<const float*>(p)[i];
  const uint16_t h = static_cast<const uint16_t*>(p)[i];
  return dtype == UTTT_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}

// Sums of two values over the LPR lanes of a row; red: 8 floats of LDS for
// rows of several waves.
template <int LPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float* red) {
#pragma unroll
  for (int d = (LPR < 64 ? LPR : 64) / 2; d > 0; d >>= 1) {
    a += __shfl_xor(a, d);
    b += __shfl_xor(b, d);
  }
  if constexpr (LPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = a;
      red[2 * wave + 1] = b;
    }
    __syncthreads();
    a = red[0] + red[2] + red[4] + red[6];
    b = red[1] + red[3] + red[5] + red[7];
  }
}

template <class TT, int V, int LPR, int NI>
__global__ __launch_bounds__(kLnThreads) void ln_fwd_kernel(LnArgs a) {
  using S = typename TT::S;
  constexpr int RPB = kLnThreads / LPR;
  __shared__ float red[8];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  float w[NI][V], b[NI][V];   // for all the rows that the workgroup walks over
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    const int e = (lane + LPR * c) * V;
    if (e < a.N) {
      load_weights<V>(a.w, a.w_dtype, e, 1.0f, w[c]);
      load_weights<V>(a.b, a.b_dtype, e, 0.0f, b[c]);
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += (int64_t)gridDim.x * RPB) {
    const bool live = base + slot < a.rows;
    const int64_t row = live ? base + slot : a.rows - 1;
    const S* x = static_cast<const S*>(a.x) + row * a.x_st;
    float v[NI][V];
    float sum = 0.0f, dummy = 0.0f;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e < a.N) load_piece<TT, V>(x + e, v[c]);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < NI; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += v[c][i];
    row_sums<LPR>(sum, dummy, red);
    const float mean = sum / (float)a.N;
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < NI; ++c)
      if ((lane + LPR * c) * V < a.N)
#pragma unroll
        for (int i = 0; i < V; ++i) sq = __builtin_fmaf(v[c][i] - mean, v[c][i] - mean, sq);
    row_sums<LPR>(sq, dummy, red);
    const float rstd = 1.0f / sqrtf(sq / (float)a.N + a.eps);
    if (!live) continue;   // whole rows: no later exchange in this turn
    if (a.stats && lane == 0) {
      a.stats[row] = mean;
      a.stats[a.rows + row] = rstd;
    }
    S* y = static_cast<S*>(a.y) + row * a.N;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e >= a.N) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = __builtin_fmaf((v[c][i] - mean) * rstd, w[c][i], b[c][i]);
      store_piece<TT, V>(y + e, v[c]);
    }
  }
}

template <class TT, int V, int LPR, int NI>
__global__ __launch_bounds__(kLnThreads) void ln_bwd_kernel(LnArgs a) {
  using S = typename TT::S;
  constexpr int RPB = kLnThreads / LPR;
  __shared__ float red[8];
  __shared__ float tot[RPB > 1 ? 2 * LPR * V : 1];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  float w[NI][V], dw[NI][V], db[NI][V];
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    const int e = (lane + LPR * c) * V;
    if (e < a.N) load_weights<V>(a.w, a.w_dtype, e, 1.0f, w[c]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[c][i] = db[c][i] = 0.0f;
  }
  const float inv_n = 1.0f / (float)a.N;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += (int64_t)gridDim.x * RPB) {
    const bool live = base + slot < a.rows;
    const int64_t row = live ? base + slot : a.rows - 1;
    const S* x = static_cast<const S*>(a.x) + row * a.x_st;
    const S* dy = static_cast<const S*>(a.dy) + row * a.dy_st;
    const float mean = a.stats[row], rstd = a.stats[a.rows + row];
    float h[NI][V], g[NI][V];
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e < a.N && live) {
        load_piece<TT, V>(x + e, h[c]);
        load_piece<TT, V>(dy + e, g[c]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[c][i] = (h[c][i] - mean) * rstd;
          dw[c][i] = __builtin_fmaf(g[c][i], h[c][i], dw[c][i]);
          db[c][i] += g[c][i];
          g[c][i] *= w[c][i];
          s0 += g[c][i];
          s1 = __builtin_fmaf(g[c][i], h[c][i], s1);
        }
      }
    }
    row_sums<LPR>(s0, s1, red);
    if (!live) continue;   // whole rows: no later exchange in this turn
    S* dx = static_cast<S*>(a.y) + row * a.N;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int e = (lane + LPR * c) * V;
      if (e >= a.N) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) g[c][i] = rstd * (g[c][i] - inv_n * (s0 + h[c][i] * s1));
      store_piece<TT, V>(dx + e, g[c]);
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.N;
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
            p[1] = k ? p[1] + db[c][i] : db[c][i];
          }
      }
      __syncthreads();
    }
    if (slot == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = (lane + LPR * c) * V + i;
        if (e < a.N) {
          out[e] = RPB > 1 ? tot[(lane * V + i) * 2] : dw[c][i];
          out[a.N + e] = RPB > 1 ? tot[(lane * V + i) * 2 + 1] : db[c][i];
        }
      }
  }
}

// Rows too long for registers: a workgroup per row, the row read again from
// cache for each pass.
template <class TT>
__global__ __launch_bounds__(kLnThreads) void ln_fwd_long_kernel(LnArgs a) {
  using S = typename TT::S;
  __shared__ float red[8];
  const int64_t row = blockIdx.x;
  const S* x = static_cast<const S*>(a.x) + row * a.x_st;
  S* y = static_cast<S*>(a.y) + row * a.N;
  float dummy = 0.0f;
  double lsum = 0.0, lsq = 0.0;
  for (int e = threadIdx.x; e < a.N; e += kLnThreads) lsum += TT::load(x[e]);
  float sum = (float)lsum;
  row_sums<kLnThreads>(sum, dummy, red);
  const float mean = sum / (float)a.N;
  for (int e = threadIdx.x; e < a.N; e += kLnThreads) {
    const float d = TT::load(x[e]) - mean;
    lsq += (double)d * d;
  }
  float sq = (float)lsq;
  row_sums<kLnThreads>(sq, dummy, red);
  const float rstd = 1.0f / sqrtf(sq / (float)a.N + a.eps);
  if (a.stats && threadIdx.x == 0) {
    a.stats[row] = mean;
    a.stats[a.rows + row] = rstd;
  }
  for (int e = threadIdx.x; e < a.N; e += kLnThreads) {
    float h = (TT::load(x[e]) - mean) * rstd;
    if (a.w) h *= load_w(a.w, a.w_dtype, e);
    if (a.b) h += load_w(a.b, a.b_dtype, e);
    y[e] = TT::store(h);
  }
}

template <class TT>
__global__ __launch_bounds__(kLnThreads) void ln_bwd_long_kernel(LnArgs a) {
  using S = typename TT::S;
  __shared__ float red[8];
  const int64_t row = blockIdx.x;
  const S* x = static_cast<const S*>(a.x) + row * a.x_st;
  const S* dy = static_cast<const S*>(a.dy) + row * a.dy_st;
  S* dx = static_cast<S*>(a.y) + row * a.N;
  const float mean = a.stats[row], rstd = a.stats[a.rows + row], inv_n = 1.0f / (float)a.N;
  double l0 = 0.0, l1 = 0.0;
  for (int e = threadIdx.x; e < a.N; e += kLnThreads) {
    const float g = TT::load(dy[e]) * (a.w ? load_w(a.w, a.w_dtype, e) : 1.0f);
    l0 += g;
    l1 += (double)g * ((TT::load(x[e]) - mean) * rstd);
  }
  float s0 = (float)l0, s1 = (float)l1;
  row_sums<kLnThreads>(s0, s1, red);
  for (int e = threadIdx.x; e < a.N; e += kLnThreads) {
    const float g = TT::load(dy[e]) * (a.w ? load_w(a.w, a.w_dtype, e) : 1.0f);
    dx[e] = TT::store(rstd * (g - inv_n * (s0 + (TT::load(x[e]) - mean) * rstd * s1)));
  }
}

// dw and db of long rows: a workgroup sums a run of rows for 256 columns.
template <class TT>
__global__ __launch_bounds__(kLnThreads) void ln_cols_kernel(LnArgs a, int64_t run) {
  using S = typename TT::S;
  const int64_t e = (int64_t)blockIdx.x * kLnThreads + threadIdx.x, r0 = blockIdx.y * run;
  if (e >= a.N) return;
  double dw = 0.0, db = 0.0;
  for (int64_t r = r0; r < r0 + run && r < a.rows; ++r) {
    const float g = TT::load(static_cast<const S*>(a.dy)[r * a.dy_st + e]);
    const float h = (TT::load(static_cast<const S*>(a.x)[r * a.x_st + e]) - a.stats[r]) * a.stats[a.rows + r];
    dw += (double)g * h;
    db += g;
  }
  float* out = a.part + (int64_t)blockIdx.y * 2 * a.N;
  out[e] = (float)dw;
  out[a.N + e] = (float)db;
}

// The workgroups' totals added: 16 columns by 64 slices of the workgroups, in
// a fixed order.  Past kSumBlocks * 16 columns (of dw and db together) a
// workgroup has several such runs: a launch has fewer than 2^32 threads.
constexpr int kSumSlices = 64, kSumBlocks = 1 << 20;
__global__ __launch_bounds__(16 * kSumSlices) void ln_sum_kernel(const float* __restrict__ part, int n, int N,
                                                                 void* dw, int w_dtype, void* db, int b_dtype) {
  __shared__ float red[kSumSlices][17];
  const int c = threadIdx.x & 15, s = threadIdx.x >> 4;
  for (int64_t base = (int64_t)blockIdx.x * 16; base < 2 * (int64_t)N; base += (int64_t)kSumBlocks * 16) {
    const int64_t e = base + c;   // over dw then db
    float sum = 0.0f;
    if (e < 2 * (int64_t)N)
#pragma unroll 8
      for (int i = s; i < n; i += kSumSlices) sum += part[(int64_t)i * 2 * N + e];
    __syncthreads();   // the run before is read
    red[s][c] = sum;
    __syncthreads();
#pragma unroll
    for (int d = kSumSlices / 2; d > 0; d >>= 1) {
      if (s < d) red[s][c] += red[s + d][c];
      __syncthreads();
    }
    if (s != 0 || e >= 2 * (int64_t)N) continue;
    sum = red[0][c];
    const bool second = e >= N;
    void* out = second ? db : dw;
    const int dt = second ? b_dtype : w_dtype;
    const int64_t at = second ? e - N : e;
    if (!out) continue;
    if (dt == UTTT_F32) static_cast<float*>(out)[at] = sum;
    else static_cast<uint16_t*>(out)[at] = dt == UTTT_BF16 ? f32_to_bf16(sum) : f32_to_f16(sum);
  }
}

constexpr int kLnPieces = 2048, kLnOddMost = 8192;   // longest rows held in registers

bool whole_pieces(const LnArgs& a, int size) {
  return ((int64_t)a.N * size) % 16 == 0 && (a.x_st * size) % 16 == 0 && (a.dy_st * size) % 16 == 0 &&
         ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
           reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.w) |
           reinterpret_cast<uintptr_t>(a.b)) & 15u) == 0;
}

// Workgroups of the backward: each writes 8 bytes per column, so that it has
// 4 rows or more to walk over (4099 rows of 1537 fp32: 256 workgroups 55 us,
// 1024 23 us).  A function of the sizes alone, so that its sums come out the
// same on every run (the rows of a workgroup are added in an order that also goes
// by whether 16-byte pieces fit).
int64_t bwd_blocks(int64_t rows, int N) {
  const int64_t per = N <= 64 ? 16 : 4;
  const int64_t n = (rows + per - 1) / per;
  return n < 1024 ? n : 1024;
}

template <class TT, int V, int LPR, int NI>
void ln_launch(const LnArgs& a, bool bwd, hipStream_t st) {
  constexpr int RPB = kLnThreads / LPR;
  int64_t blocks = (a.rows + RPB - 1) / RPB;
  if (blocks > 2048) blocks = 2048;   // 8 workgroups a CU: the weights are read once for many rows
  if (bwd)
    hipLaunchKernelGGL((ln_bwd_kernel<TT, V, LPR, NI>), dim3((unsigned)bwd_blocks(a.rows, a.N)),
                       dim3(kLnThreads), 0, st, a);
  else
    hipLaunchKernelGGL((ln_fwd_kernel<TT, V, LPR, NI>), dim3((unsigned)blocks), dim3(kLnThreads), 0, st, a);
}

template <class TT>
int ln_rows(const LnArgs& a, bool bwd, hipStream_t st) {
  constexpr int V = 16 / sizeof(typename TT::S);
  if (whole_pieces(a, sizeof(typename TT::S)) && a.N / V <= kLnPieces) {
    const int pieces = a.N / V;
    if (pieces <= 16) ln_launch<TT, V, 16, 1>(a, bwd, st);
    else if (pieces <= 64) ln_launch<TT, V, 64, 1>(a, bwd, st);
    else if (pieces <= 128) ln_launch<TT, V, 64, 2>(a, bwd, st);
    else if (pieces <= 256) ln_launch<TT, V, 64, 4>(a, bwd, st);
    else if (pieces <= 512) ln_launch<TT, V, 256, 2>(a, bwd, st);
    else if (pieces <= 1024) ln_launch<TT, V, 256, 4>(a, bwd, st);
    else ln_launch<TT, V, 256, 8>(a, bwd, st);
  } else if (a.N <= kLnOddMost) {
    if (a.N <= 64) ln_launch<TT, 1, 16, 4>(a, bwd, st);
    else if (a.N <= 256) ln_launch<TT, 1, 64, 4>(a, bwd, st);
    else if (a.N <= 1024) ln_launch<TT, 1, 64, 16>(a, bwd, st);
    else if (a.N <= 2048) ln_launch<TT, 1, 256, 8>(a, bwd, st);
    else ln_launch<TT, 1, 256, 32>(a, bwd, st);
  } else if (!bwd) {
    hipLaunchKernelGGL((ln_fwd_long_kernel<TT>), dim3((unsigned)a.rows), dim3(kLnThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((ln_bwd_long_kernel<TT>), dim3((unsigned)a.rows), dim3(kLnThreads), 0, st, a);
    if (a.part) {
      const int64_t blocks = bwd_blocks(a.rows, a.N), run = (a.rows + blocks - 1) / blocks;
      hipLaunchKernelGGL((ln_cols_kernel<TT>),
                         dim3((unsigned)((a.N + kLnThreads - 1) / kLnThreads), (unsigned)blocks),
                         dim3(kLnThreads), 0, st, a, run);
    }
  }
  return check_launch("layer_norm");
}

int ln_check(const LnArgs& a, int dtype, const char* what) {
  UTTT_REQUIRE(a.rows >= 0 && a.rows < (1LL << 31) && a.N >= 1 && a.N <= (1 << 27), "%s: bad sizes rows=%lld N=%d",
               what, (long long)a.rows, a.N);
  UTTT_REQUIRE(dtype_bytes(dtype) && dtype_bytes(a.w_dtype) && dtype_bytes(a.b_dtype),
               "%s: dtype codes %d, %d, %d", what, dtype, a.w_dtype, a.b_dtype);
  UTTT_REQUIRE(a.rows == 0 || (a.x && a.y), "%s: null pointer", what);
  UTTT_REQUIRE(a.x_st >= 0 && a.dy_st >= 0, "%s: negative row stride", what);
  return UTTT_OK;
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_layer_norm_fwd(const void* x, int dtype, int64_t x_stride, int64_t rows, int N,
                                   const void* weight, int weight_dtype, const void* bias,
                                   int bias_dtype, float eps, void* out, float* stats, void* stream) {
  LnArgs a{};
  a.x = x; a.x_st = x_stride; a.dy_st = 0;
  a.w = weight; a.w_dtype = weight_dtype; a.b = bias; a.b_dtype = bias_dtype;
  a.rows = rows; a.N = N; a.eps = eps; a.y = out; a.stats = stats;
  if (const int rc = ln_check(a, dtype, "uttt_layer_norm_fwd")) return rc;
  if (rows == 0) return UTTT_OK;
  UTTT_DTYPE_SWITCH_LR(dtype, TT, return ln_rows<TT>(a, false, as_stream(stream)));
  return UTTT_OK;
}

extern "C" size_t uttt_layer_norm_bwd_workspace_bytes(int64_t rows, int N) {
  return rows <= 0 || N <= 0 ? 0 : (size_t)bwd_blocks(rows, N) * 2 * (size_t)N * 4;
}

extern "C" int uttt_layer_norm_bwd(const void* x, int dtype, int64_t x_stride, const void* dy,
                                   int64_t dy_stride, int64_t rows, int N, const void* weight,
                                   int weight_dtype, const float* stats, void* dx, void* dweight,
                                   void* dbias, int bias_dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const char* what = "uttt_layer_norm_bwd";
  LnArgs a{};
  a.x = x; a.x_st = x_stride; a.dy = dy; a.dy_st = dy_stride;
  a.w = weight; a.w_dtype = weight_dtype; a.b_dtype = bias_dtype;
  a.rows = rows; a.N = N; a.y = dx; a.stats = const_cast<float*>(stats);
  if (const int rc = ln_check(a, dtype, what)) return rc;
  const hipStream_t st = as_stream(stream);
  const bool sums = dweight || dbias;
  if (rows == 0) {
    if (dweight)
      if (const int rc = zero_fill_async(dweight, (size_t)N * dtype_bytes(weight_dtype), st, what)) return rc;
    return dbias ? zero_fill_async(dbias, (size_t)N * dtype_bytes(bias_dtype), st, what) : UTTT_OK;
  }
  UTTT_REQUIRE(dy && stats, "%s: null pointer", what);
  const size_t need = uttt_layer_norm_bwd_workspace_bytes(rows, N);
  UTTT_REQUIRE(!sums || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, %zu needed", what,
               workspace_bytes, need);
  a.part = sums ? static_cast<float*>(workspace) : nullptr;
  int rc = UTTT_OK;
  switch (dtype) {
    case UTTT_F32: rc = ln_rows<F32T>(a, true, st); break;
    case UTTT_BF16: rc = ln_rows<BF16T>(a, true, st); break;
    default: rc = ln_rows<F16T>(a, true, st); break;
  }
  if (rc || !sums) return rc;
  const int64_t runs = (2 * (int64_t)N + 15) / 16;
  hipLaunchKernelGGL(ln_sum_kernel, dim3((unsigned)(runs < kSumBlocks ? runs : kSumBlocks)), dim3(16 * kSumSlices), 0, st,
                     a.part, (int)bwd_blocks(rows, N), N, dweight, weight_dtype, dbias, bias_dtype);
  return check_launch("layer_norm_sum");
}
