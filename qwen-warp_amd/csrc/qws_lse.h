// Running log-sum-exp of a row of logits with its entropy: the statistics that the log-probability kernels
// (qws_logprobs.hip) and the scoring head (qws_fp8.hip) keep per lane, join over lanes, waves and workgroups, and finish.
//
// With c = log2(e) / T and d_i = c (x_i - m), m the largest x so far:
//   s = sum 2^d_i,   t = sum 2^d_i d_i    (fp32)
// A larger maximum m' (delta = c (m' - m)) turns them into 2^-delta s and 2^-delta (t - delta s): one pass, any order.
// Then
//   log p_i = (x_i - m) / T - ln s,   H = ln s - ln 2 * t / s.
// With m the largest x both terms of H are >= 0 (s >= 1, t <= 0; either may be off by a rounding): nothing cancels.  m may be
// any value near it instead: with one that lies up to 8 units of d below (k_lp_scan's, so that it rarely moves) the terms cancel
// by at most 8 ln 2 = 5.5, an error of a few 5.5 * 2^-24 in H.
// The general form takes differences to m before the scaling, so rows at the type's lowest value and rows mixing it with
// -inf are exact; NaN counts as -inf (the sampling stage's rule), +inf as the largest finite value (so tokens at +inf share
// the row); d is held above -D_MIN, where 2^d is 0 in fp32: no infinity meets a 0 in t.
#pragma once
#include "qws_device.h"

namespace qws {

constexpr float LSE_DMIN = 150.0f;
constexpr float LN2 = 0.69314718055994531f;
constexpr float F32_MAX = 3.402823466e+38f;

struct Lse {
  float m, s, t;
};

__device__ __forceinline__ float lse_exp2(float d) { return __builtin_amdgcn_exp2f(d); }
// NaN -> -inf (the median of three with a quiet NaN is the smaller of the others; with a signalling one it is not, so x is
// quieted first), +inf -> the largest finite value.  The -inf comes from a register that the compiler does not see through: it
// would fold the median into min(x, F32_MAX), whose answer for NaN is F32_MAX.
__device__ __forceinline__ float lse_clean(float x) {
  float lowest;
  asm("s_mov_b32 %0, 0xff800000" : "=s"(lowest));
  return __builtin_amdgcn_fmed3f(__builtin_canonicalizef(x), lowest, F32_MAX);
}
__device__ __forceinline__ float lse_temp(float T) { return T > 0.0f ? T : 1.0f; }  // 0 (a greedy row), negative, NaN: as T = 1
__device__ __forceinline__ float lse_scale(float T) { return fminf((float)LOG2E / lse_temp(T), 0.5f * F32_MAX); }
// (x - m) / 2: the difference of the largest and the lowest value is past fp32, its half is not
__device__ __forceinline__ float lse_half(float x, float m) { return fmaf(0.5f, x, -0.5f * m); }
__device__ __forceinline__ float lse_d(float x, float m, float c) { return fmaxf(lse_half(x, m) * (2.0f * c), -LSE_DMIN); }  // NaN (-inf - -inf): -D_MIN

// The largest of three; a NaN does not show in it.  One instruction, where fmaxf on values that may be signalling NaNs also
// has to quiet them.
__device__ __forceinline__ float lse_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Sums of moderate values (below LSE_MOST in magnitude, c as well) relative to M = fl(c m) take one multiply-add for d; what
// rounding M took, r = c m - M, is given back at the end.  m itself has d = r, so M stays below LSE_NEAR, where |r| <= 1/2: at
// 2^31 r passes 64, and from 2^32 on a lane's 2^r is 0 or infinite (at temperature 1e-9, or beside a mask's -1e11).
constexpr float LSE_MOST = 0x1p60f, LSE_NEAR = 0x1p24f;
__device__ __forceinline__ Lse lse_exact(float m, float M, float s, float t, float c) {
  const float r = fmaf(c, m, -M), e = lse_exp2(-r);
  return {m, s * e, e * fmaf(-r, s, t)};
}

__device__ __forceinline__ Lse lse_join(Lse a, Lse b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = lse_d(a.m, m, c), db = lse_d(b.m, m, c), ea = lse_exp2(da), eb = lse_exp2(db);
  return {m, fmaf(ea, a.s, eb * b.s), fmaf(ea, fmaf(da, a.s, a.t), eb * fmaf(db, b.s, b.t))};
}
// the wave's values joined, in every lane
__device__ __forceinline__ Lse lse_join_wave(Lse v, float c) {
  const float m = wave_max_f(v.m), d = lse_d(v.m, m, c), e = lse_exp2(d);
  return {m, wave_sum<float>(e * v.s), wave_sum<float>(e * fmaf(d, v.s, v.t))};
}
__device__ inline Lse lse_join_lanes(Lse v, float c, int from, int to) {  // butterfly over lane bits `from` .. `to` (powers of two)
  for (int i = from; i <= to; i <<= 1) v = lse_join(v, {__shfl_xor(v.m, i), __shfl_xor(v.s, i), __shfl_xor(v.t, i)}, c);
  return v;
}
__device__ __forceinline__ float lse_log(Lse v) { return logf(v.s); }
// log p of a (clean) logit; -inf for a masked one and in a row without a candidate.  Neither it nor the entropy leaves its range
// where the sums are off by a rounding (a sure token's s = 1 - 2^-24); a NaN would pass.
__device__ __forceinline__ float lse_logprob(Lse v, float x, float T) {
  const float p = x == -INFINITY ? -INFINITY : 2.0f * (lse_half(x, v.m) / lse_temp(T)) - lse_log(v);
  return p > 0.0f ? 0.0f : p;
}
__device__ __forceinline__ float lse_entropy(Lse v) {
  const float h = v.m == -INFINITY ? 0.0f : lse_log(v) - LN2 * (v.t / v.s);
  return h < 0.0f ? 0.0f : h;
}

}  // namespace qws
