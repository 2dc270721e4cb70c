// Rows of logits read 16 bytes a thread at a time: the loads that the log-probability kernels (qws_logprobs.hip) and the losses'
// (qws_loss.hip) share.
#pragma once
#include "qws_lse.h"

#include <type_traits>

namespace qws {

template <typename T>
constexpr int lp_e() { return 16 / (int)sizeof(T); }  // elements of a vector
template <typename T>
using lp_bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

template <typename T>
__device__ __forceinline__ float lp_one(const T* p) {
  if constexpr (sizeof(T) == 4)
    return lse_clean(*gmem((const float*)p));
  else
    return lse_clean(__uint_as_float((uint32_t)*gmem((const uint16_t*)p) << 16));
}
template <typename T>
__device__ __forceinline__ void lp_unpack(vu4 r, float* x) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __uint_as_float(r[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[2 * j] = __uint_as_float(r[j] << 16);
      x[2 * j + 1] = __uint_as_float(r[j] & 0xFFFF0000u);
    }
  }
}
// the vector at position v of `base` (16-byte aligned), of which [lead, end) exist: the rest reads -inf
template <typename T>
__device__ __forceinline__ vu4 lp_load_edge(const T* base, int v, int lead, int end) {
  constexpr int E = lp_e<T>();
  vu4 r;
  if (v >= lead && v + E <= end) {
    r = *gmem((const vu4*)(base + v));
  } else {
    uint32_t y[E];
#pragma unroll
    for (int j = 0; j < E; j++) y[j] = *gmem((const lp_bits<T>*)base + min(max(v + j, lead), end - 1));
#pragma unroll
    for (int j = 0; j < E; j++)
      if (v + j < lead || v + j >= end) y[j] = 0xFF800000u >> (sizeof(T) == 4 ? 0 : 16);
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = sizeof(T) == 4 ? y[j] : y[j * (E / 4)] | y[(j * (E / 4) + 1) % E] << 16;
  }
  return r;
}

// The largest of a vector; a NaN shows in the sums, not here
template <int E>
__device__ __forceinline__ float lp_max(const float* x) {
  float m = lse_max3(x[0], x[1], x[2]);
#pragma unroll
  for (int j = 3; j + 1 < E; j += 2) m = lse_max3(m, x[j], x[j + 1]);
  return lse_max3(m, x[E - 1], x[E - 1]);
}

}  // namespace qws
