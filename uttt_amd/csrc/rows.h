// Pieces of V adjacent elements of a row, widened to fp32 and rounded back: the
// row norms' loads and stores (layer_norm.hip, block_norm.hip).
#pragma once

#include "common.h"

namespace uttt {

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
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof w > 16 ? 16 : sizeof w), w, sizeof w);
}
// V elements from e of a tensor of any type, `none` where there is no tensor.
template <int V>
__device__ __forceinline__ void load_weights(const void* p, int dtype, int64_t e, float none, float (&v)[V]) {
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
template <int V>
__device__ __forceinline__ void store_piece_as(void* p, int dtype, int64_t e, const float (&v)[V]) {
  if (dtype == UTTT_F32) store_piece<F32T, V>(static_cast<float*>(p) + e, v);
  else if (dtype == UTTT_BF16) store_piece<BF16T, V>(static_cast<uint16_t*>(p) + e, v);
  else store_piece<F16T, V>(static_cast<uint16_t*>(p) + e, v);
}

}  // namespace uttt
