// Shared pieces of the gated delta rule's chunked kernels (delta_fwd.hip,
// delta_bwd.hip): the call's geometry, the chunk table of packed sequences,
// operand fragments and the split of fp32 values into bf16 parts.
//
// The rule, per value head, with a state S [Dk, Dv]:
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,  u_t = b_t (v_t - e^{g_t} S_{t-1}^T k_t),
//   o_t = s S_t^T q_t
// Over a chunk of C = 64 tokens that starts from S0, with G = cumsum(g),
// gam = e^G, E_ij = e^{G_i - G_j}:
//   A_ij = b_i E_ij k_i.k_j (j < i),  T = (I + A)^-1,  P_ij = s E_ij q_i.k_j (j <= i)
//   R = b (V - gam K S0),  U = T R
//   O = s gam Q S0 + P U
//   S' = gam_C S0 + (e^{G_C - G} K)^T U
// and for gradients dO and dS' of a chunk's outputs
//   dU = P^T dO + e^{G_C - G} K dS',  dR = T^T dU,  dV = b dR
//   dS0 = gam_C dS' + (s gam Q)^T dO - (b gam K)^T dR
//
// Precision.  The state and its gradient are fp32 and stay exact to fp32's
// order: a product with one of them, with U, T, R, P, e^{G_C - G} U or their
// gradients takes that fp32 operand as the sum of three bf16 values (x1 = bf16(x),
// x2 = bf16(x - x1), x3 = bf16(x - x1 - x2), all of its 24 bits) and adds the
// products that are not below 2^-24 in fp32; q, k, v and do are bf16 as given.
// Where only 16-bit results come of it the first two parts go in, at most 2^-16
// left out where the result's rounding is 2^-8 or 2^-11: S0, U and P for the
// outputs; D, M and X of the gradients, and there U, S0, dR and dS' where g and
// beta are both 16-bit types.  What a backward keeps or exchanges (U, S0, dR, dS')
// is stored in fp32.  With two parts throughout states came out 4e-6 off the
// 64-bit recurrence and dg and dbeta 5e-6, with three 1.3e-7 and 3e-7, as the same
// sums in plain fp32.  Decays are e^x by the hardware's 2^x, off by |x| 2^-24 and
// an ulp or two, of differences of sums held in 64 bits.
//
// Fragments.  v_mfma_f32_16x16x32_bf16 takes from lane (r = lane % 16, q =
// lane / 16) eight consecutive values 8q..8q+7 of the contracted axis for row
// (column) r, and gives it rows 4q..4q+3 of column r.
#pragma once

#include "common.h"

namespace uttt {
namespace delta {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;           // tokens of a chunk
constexpr int kTFrags = 6;       // nonzero 16 x 32 fragments of a triangular 64 x 64 operand
constexpr int kPFrag = 3 * kTFrags;                  // P's first fragment, behind T's three parts
constexpr int kTriBytes = (kPFrag + 2 * kTFrags) * 1024;      // P in two parts
constexpr int kTriBwdBytes = (kPFrag + 3 * kTFrags) * 1024;   // P^T in three
constexpr int kScal = 5 * kC;    // gam, e^{G_C - G}, beta and G in two parts, per token

struct Args {
  const uint16_t *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const void *g, *beta;          // [B, T, Hv]
  int g_dtype, beta_dtype;
  int B, T, Hk, Hv, Dk, Dv, nseq, nchunks;   // nchunks: slots of the chunk table
  int cps;                       // chunks per sequence where there is no table
  float scale;
  const int4* table;             // [nchunks] sequence, first token, tokens; packed sequences only
  const int4* seqs;              // [nseq] first chunk, sequence, first token, tokens
  uint8_t* tri;                  // [nchunks, Hv] kTriBytes, in the backward kTriBwdBytes
  float* scal;                   // [nchunks, Hv, kScal]
  uint8_t* kt;                   // [nchunks, Hk, 4 KS] KiB: K^T fragments
  uint8_t* qt;                   // the same of Q (backward)
  uint8_t *kf, *qf;              // [nchunks, Hk, 4 KS] KiB: K and Q fragments, or null: rows are read
  const float* h0;               // [nseq, Hv, Dk, Dv] or null
  uint16_t* o;                   // [B, T, Hv, Dv]
  float* hT;                     // final states or null
  float* u;                      // [B, T, Hv, Dv], or null
  float* s0;                     // [nchunks, Hv, Dk, Dv], or null
  // backward
  const uint16_t* dout;          // [B, T, Hv, Dv]
  int64_t do_sb, do_st, do_sh;
  const float* dhT;              // or null
  float* dh0;                    // or null
  float* ds;                     // [nchunks, Hv, Dk, Dv] dS'
  float* dr;                     // [B, T, Hv, Dv]
  uint16_t *dq, *dk;             // [B, T, Hk, Dk]
  uint16_t* dv;                  // [B, T, Hv, Dv]
  void *dg, *dbeta;              // [B, T, Hv] in their inputs' types
};

struct Chunk {
  int seq;        // -1: tokens of no sequence, -2: nothing
  int b, t0, n;   // batch row, first token, tokens
};

__device__ __forceinline__ Chunk chunk_of(const Args& a, int c) {
  if (a.table == nullptr) {
    const int seq = c / a.cps, t0 = (c - seq * a.cps) * kC;
    return {seq, seq, t0, min(kC, a.T - t0)};
  }
  const int4 e = a.table[c];
  return {e.x, 0, e.y, e.z};
}

// Index of fragment (16-row tile, 32-column step) of a lower triangular
// operand, its row tiles 0, 1 having step 0 alone; of an upper one (its
// transpose) tiles 2, 3 have step 1 alone.
__device__ __forceinline__ constexpr int lower_frag(int rt, int ks) {
  return rt < 2 ? rt : 2 + 2 * (rt - 2) + ks;
}
__device__ __forceinline__ constexpr int upper_frag(int rt, int ks) {
  return rt < 2 ? 2 * rt + ks : 2 + rt;
}

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// The first PARTS bf16 parts of a, b.
template <int PARTS>
__device__ __forceinline__ void split8(f32x4 a, f32x4 b, bf16x8 (&out)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[k][i] = (__bf16)a[i];
      out[k][4 + i] = (__bf16)b[i];
      a[i] -= (float)out[k][i];
      b[i] -= (float)out[k][4 + i];
    }
}

// Raw buffers: a lane whose offset has bit 31 (past any record count) reads
// zeros and writes nothing, without a branch.  The bit is set by arithmetic:
// of two offsets chosen between by a condition the compiler makes two branches
// with a load in each.
typedef __amdgpu_buffer_rsrc_t Rsrc;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t kNoRow = 0x80000000u;
__device__ __forceinline__ Rsrc buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, 0x7fffffff, 0x00020000);
}
__device__ __forceinline__ uint32_t miss_from(int i, int n) {   // kNoRow where i >= n
  return (uint32_t)(n - 1 - i) & kNoRow;
}
__device__ __forceinline__ bf16x8 load_frag(Rsrc r, uint32_t off, uint32_t uniform = 0) {
  return __builtin_bit_cast(bf16x8, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(r, off, uniform, 0));
}
__device__ __forceinline__ f32x4 load_f4(Rsrc r, uint32_t off, uint32_t uniform = 0) {
  return __builtin_bit_cast(f32x4, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(r, off, uniform, 0));
}
__device__ __forceinline__ float load_f1(Rsrc r, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}

// NT adjacent bf16 columns of one row, held as raw words.
template <int NT>
struct Cols {
  uint32_t w[NT / 2];
  __device__ __forceinline__ void load(Rsrc r, uint32_t off) {
    if constexpr (NT == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else {
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
      w[0] = x[0];
      w[1] = x[1];
    }
  }
  __device__ __forceinline__ float get(int c) const {
    return __uint_as_float(c & 1 ? w[c / 2] & 0xffff0000u : w[c / 2] << 16);
  }
  __device__ __forceinline__ uint32_t half(int c) const { return c & 1 ? w[c / 2] >> 16 : w[c / 2] & 0xffffu; }
};

template <>
struct Cols<1> {
  uint16_t w;   // widened where it is used, not where it is loaded
  __device__ __forceinline__ void load(Rsrc r, uint32_t off) {
    w = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  }
  __device__ __forceinline__ float get(int) const { return bf16_to_f32(w); }
  __device__ __forceinline__ uint32_t half(int) const { return w; }
};

// Every load that is under way done.  Before a pipelined loop: the compiler's
// wait counts at the loop's head allow for both ways into it, and loads in
// another order in front of it made each turn wait for its own last loads.
__device__ __forceinline__ void settle() { __builtin_amdgcn_s_waitcnt(0); }

// Four fp32 rows of one column as bf16 parts, two rows a word.
struct Parts {
  u32x2 hi, lo;
};
__device__ __forceinline__ Parts parts_of(f32x4 x) {
  Parts p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    p.hi[i] = h;
    p.lo[i] = pack_bf16x2(x[2 * i] - __uint_as_float(h << 16), x[2 * i + 1] - __uint_as_float(h & 0xffff0000u));
  }
  return p;
}
// The same as three parts.
struct Parts3 {
  u32x2 p[3];
};
__device__ __forceinline__ Parts3 parts3_of(f32x4 x) {
  Parts3 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      r.p[k][i] = pack_bf16x2(a, b);
      a -= __uint_as_float(r.p[k][i] << 16);
      b -= __uint_as_float(r.p[k][i] & 0xffff0000u);
    }
  }
  return r;
}
__device__ __forceinline__ u32x2 round_of(f32x4 x) {
  u32x2 p;
  p[0] = pack_bf16x2(x[0], x[1]);
  p[1] = pack_bf16x2(x[2], x[3]);
  return p;
}
// Row i of NT columns' words to memory as adjacent bf16.
template <int NT>
__device__ __forceinline__ void store_row(Rsrc r, uint32_t off, const u32x2 (&x)[NT], int i) {
  const auto pair = [&](int n) -> uint32_t {
    const uint32_t a = x[n][i >> 1], b = x[n + 1][i >> 1];
    return i & 1 ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
  };
  if constexpr (NT == 1)
    __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(i & 1 ? x[0][i >> 1] >> 16 : x[0][i >> 1]), r, off, 0, 0);
  else if constexpr (NT == 2)
    __builtin_amdgcn_raw_buffer_store_b32(pair(0), r, off, 0, 0);
  else {
    const u32x2 w = {pair(0), pair(2)};
    __builtin_amdgcn_raw_buffer_store_b64(w, r, off, 0, 0);
  }
}
// Row i of NT columns to memory as adjacent fp32.
template <int NT>
__device__ __forceinline__ void store_row(Rsrc r, uint32_t off, const f32x4 (&x)[NT], int i) {
  if constexpr (NT == 1)
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[0][i]), r, off, 0, 0);
  else if constexpr (NT == 2)
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x[0][i]), __float_as_uint(x[1][i])}, r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(x[0][i]), __float_as_uint(x[1][i]),
                                                 __float_as_uint(x[2][i]), __float_as_uint(x[3][i])}, r, off, 0, 0);
}

// Sum over the 16 lanes of equal lane / 16, in all of them: four additions
// with a lane permutation each, where a shuffle goes through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// Inclusive sums over the 64 lanes in 64 bits: within rows of 16, then the
// totals of the rows before.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add64(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, true);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double scan64(double x) {
  x = dpp_add64<0x111, 0xf>(x);
  x = dpp_add64<0x112, 0xf>(x);
  x = dpp_add64<0x114, 0xf>(x);
  x = dpp_add64<0x118, 0xf>(x);
  x = dpp_add64<0x142, 0xa>(x);   // lane 15 of rows 0 and 2 to rows 1 and 3
  return dpp_add64<0x143, 0xc>(x);   // lane 31 to rows 2 and 3
}
__device__ __forceinline__ float sum16(float x) {
  x = dpp_add<0xb1>(x);    // lane ^ 1
  x = dpp_add<0x4e>(x);    // lane ^ 2
  x = dpp_add<0x141>(x);   // 7 - lane % 8: the other four of eight
  return dpp_add<0x140>(x);   // 15 - lane % 16
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

// The part of a call that a scan's workgroup walks over: one sequence, one
// value head, `width` columns.  Column blocks of one head are eight workgroups
// apart: on one XCD, whose L2 the head's fragments then pass once.
struct Scan {
  int head, seq, hv, hk, b, c0, nc, tok0, len, col0;
  __device__ __forceinline__ bool init(const Args& a, int width) {
    const int ncb = (a.Dv + width - 1) / width;
    const int grp = blockIdx.x / (8 * ncb), in = blockIdx.x % (8 * ncb);
    const int at = grp * 8 + (in & 7);
    if (at >= a.nseq * a.Hv) return false;
    col0 = (in >> 3) * width;
    seq = at / a.Hv;
    hv = at % a.Hv;
    hk = hv / (a.Hv / a.Hk);
    b = a.table ? 0 : seq;
    if (a.table) {
      const int4 s = a.seqs[seq];
      c0 = s.x; seq = s.y; tok0 = s.z; len = s.w;
      nc = (len + kC - 1) / kC;
    } else {
      c0 = seq * a.cps; nc = a.cps; tok0 = 0; len = a.T;
    }
    head = seq * a.Hv + hv;
    return true;
  }
};
inline int64_t scan_blocks(const Args& a, int width) {
  return ((int64_t)a.nseq * a.Hv + 7) / 8 * 8 * ((a.Dv + width - 1) / width);
}
// 16-column tiles of a scan's workgroup.  Wide ones do more work a CU, narrow
// ones end a long sequence sooner.  What is estimated: rounds of workgroups
// over the 256 CUs, a chunk of them as 2.0, 2.8 and 4.3 us for 1, 2 and 4 tiles
// (what a busy card takes at 128 features; 4.0 for 4 tiles in the backward and
// where what it reads is stored, which is most of the time then), and of packed
// sequences, whose
// lengths the host does not know, the work over the CUs and a longest sequence
// of three times the mean.  Measured, forward scans, us for 1, 2, 4 tiles:
//   4096 tokens, 4 heads of 192                         96, 163, 358
//   8192 tokens, 16 heads of 128                       177, 249, 532
//   4 x 4096 tokens, 16 heads of 128                   258, 178, 297
//   16 x 2048 tokens, 12 heads of 128                  387, 284, 333
//   16 x 4096 tokens, 16 heads of 64 x 128             711, 589, 530
//   12 prompts of 1 to 5000 tokens, 16 heads of 128    256, 195, 346
//   8 packed sequences of 1024, 4 heads of 192          60,  52, 102
// and with what a backward reads, then the backward's
//   8 x 1024 tokens, 4 heads of 192                     78,  61, 106    95,  70
//   16 x 2048 tokens, 12 heads of 128                  569, 398, 380   556, 385, 392
//   16 x 2048 tokens, 16 heads of 64                   280, 194, 154   291, 204, 182
//   32 x 2048 tokens, 4 heads of 96                    280, 223, 171   297, 289, 221
//   16 x 2048 tokens, 4 heads of 256                   527, 412        534, 397
// The packed rows are one where the guess of the longest sequence is near and one
// where it is three times too long and takes the narrower scan.
// The three parts of 64 columns fit in LDS up to 192 features, the backward's up
// to 128.
constexpr int scan_widest(int KS, bool backward) { return KS <= (backward ? 4 : 6) ? 4 : 2; }
inline int scan_tiles(int64_t T, int nseq, int Hv, int Dk, int Dv, bool packed, bool backward, bool stored) {
  const int tiles[3] = {1, 2, 4}, tenths[3] = {20, 28, stored ? 40 : 43};
  const int widths = scan_widest((Dk + 31) / 32, backward) == 4 ? 3 : 2;
  const int64_t total = T / kC + nseq, mean = (total + nseq - 1) / nseq, cps = (T + kC - 1) / kC;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int i = 0; i < widths; ++i) {
    const int64_t blocks = (Dv + 16 * tiles[i] - 1) / (16 * tiles[i]);
    int64_t cost;
    if (packed) {
      const int64_t longest = 3 * mean < total ? 3 * mean : total, work = total * Hv * blocks / 256;
      cost = (longest > work ? longest : work) * tenths[i];
    } else {
      cost = ((int64_t)nseq * Hv * blocks + 255) / 256 * cps * tenths[i];
    }
    if (cost < least) {
      least = cost;
      best = tiles[i];
    }
  }
  return best;
}
inline int scan_tiles(const Args& a, bool backward) {
  return scan_tiles(a.T, a.nseq, a.Hv, a.Dk, a.Dv, a.table != nullptr, backward, a.s0 != nullptr);
}

// Features up to which a kernel instance goes, in steps of 32: the next of 2,
// 3, 4, 6, 8 (K, Q past Dk are zeros in LDS).
inline int steps_of(int Dk) {
  const int ks = (Dk + 31) / 32;
  return ks <= 2 ? 2 : ks <= 4 ? ks : ks <= 6 ? 6 : 8;
}

#define UTTT_DELTA_STEPS(ks, KS, ...)                       \
  switch (ks) {                                             \
    case 2: { constexpr int KS = 2; __VA_ARGS__; } break;   \
    case 3: { constexpr int KS = 3; __VA_ARGS__; } break;   \
    case 4: { constexpr int KS = 4; __VA_ARGS__; } break;   \
    case 6: { constexpr int KS = 6; __VA_ARGS__; } break;   \
    default: { constexpr int KS = 8; __VA_ARGS__; } break;  \
  }

// delta_prep.hip: the chunk table of packed sequences (cu [nseq + 1], clamped
// to ascending offsets within T) and the per-chunk operands.  `transposed`:
// T^T, P^T and Q^T for the backward, else T and P.
int launch_table(const void* cu, int cu64, int nseq, int T, int nchunks, int4* table, int4* seqs,
                 hipStream_t st);
int launch_prep(const Args& a, bool transposed, hipStream_t st);

// The parts of a call's workspace, in order.
struct Workspace {
  size_t table, seqs, scal, kt, tri, kf, qf, qt, ds, dr, total;
};
inline int chunk_slots(int64_t B, int64_t T, int nseq, bool packed) {
  const int64_t n = packed ? T / kC + nseq + 2 : B * ((T + kC - 1) / kC);
  return n > 0x7fffffff ? -1 : (int)n;
}
inline Workspace workspace_of(int64_t B, int64_t T, int nseq, int Hk, int Hv, int Dk, int Dv,
                              bool packed, bool backward) {
  Workspace w{};
  const size_t n = (size_t)chunk_slots(B, T, nseq, packed);
  const size_t frags = n * Hk * 4 * steps_of(Dk) * 1024;
  size_t at = 0;
  const auto take = [&at](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  w.table = take(packed ? n * 16 : 0);
  w.seqs = take(packed ? (size_t)nseq * 16 : 0);
  w.scal = take(n * Hv * kScal * 4);
  w.kt = take(frags);
  w.tri = take(n * Hv * (backward ? kTriBwdBytes : kTriBytes));
  // Where 16 columns a workgroup are taken, each of them loads all of K and Q:
  // then from a copy in fragment order, 1 KiB a load, and not 64 bytes of each
  // of 16 rows (a chunk of 192 features 2.1 -> 1.5 us; with more columns a
  // workgroup the copy costs more than it saves).
  const bool copies = scan_tiles(T, nseq, Hv, Dk, Dv, packed, backward, backward) == 1;
  w.kf = take(copies ? frags : 0);
  w.qf = take(copies && !backward ? frags : 0);
  if (!copies) w.kf = w.qf = SIZE_MAX;
  if (backward) w.qf = SIZE_MAX;
  w.qt = take(backward ? frags : 0);
  w.ds = take(backward ? n * Hv * Dk * Dv * 4 : 0);
  w.dr = take(backward ? (size_t)B * T * Hv * Dv * 4 : 0);
  w.total = at;
  return w;
}
// Fills the fields of `a` that point into the workspace.
inline void bind_workspace(Args& a, const Workspace& w, uint8_t* ws, bool packed, bool backward) {
  a.table = packed ? reinterpret_cast<const int4*>(ws + w.table) : nullptr;
  a.seqs = packed ? reinterpret_cast<const int4*>(ws + w.seqs) : nullptr;
  a.scal = reinterpret_cast<float*>(ws + w.scal);
  a.kt = ws + w.kt;
  a.tri = ws + w.tri;
  a.kf = w.kf == SIZE_MAX ? nullptr : ws + w.kf;
  a.qf = w.qf == SIZE_MAX ? nullptr : ws + w.qf;
  if (backward) {
    a.qt = ws + w.qt;
    a.ds = reinterpret_cast<float*>(ws + w.ds);
    a.dr = reinterpret_cast<float*>(ws + w.dr);
  }
}

// delta_fwd.hip: the argument checks of both directions.
int check_args(const Args& a, int B, bool packed, bool backward, const char* what);

}  // namespace delta
}  // namespace uttt
