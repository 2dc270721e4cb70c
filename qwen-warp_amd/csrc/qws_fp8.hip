// qws 8-bit head: logits of T hidden states from a head kept in 8 bits, and the scoring of given tokens by the same
// product without the logits in memory (the definitions: include/qws.h qws_fp8_*).
//
// Numbers.  A block of 128 consecutive values of a row (a weight row or a hidden state) is held as e4m3 values q and one
// exponent e, x ~ q 2^e, with e the least whole number such that max|x| <= 448 * 2^e: the scaling itself is exact.
//
// Why the products run on the bf16 matrix instruction.  The 8-bit ones (16x16x32 and 16x16x128, with and without scales)
// align a group's products to the largest and cut what lies about 2^-13 below it: measured over 128 products of normal
// data 1.4e-5 of the result's norm, and ten times that with a few large columns.  e4m3 values times a power of two are
// exact in bf16, whose instruction sums exact products in fp32 (measured 7e-8).  v_cvt_scalef32_pk_bf16_fp8 turns two
// values and their block's scale into bf16 at the rate of any vector instruction, so the scales cost nothing more.
//
// Layout.  16 rows x 64 values are a fragment of 1 KB: lane l's 16 bytes are row l % 16, values 16 (l / 16) .. + 15, the
// operands of two 16x16x32 products.  (Which 32 of the values share a product does not matter, as long as both operands
// take the same.)  Every load of a wave is 1 KB of consecutive bytes, in memory and in LDS.  The fragments of a group of 16
// rows lie along K; the exponents (biased by 127) of four consecutive blocks are the bytes of one word per row.  Rows and
// values beyond N, T and K are 0.
#include "qws_lse.h"

#include <type_traits>

namespace qws {

typedef __bf16 f8_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 f8_b8 __attribute__((ext_vector_type(8)));

constexpr int F8_KB = 128;       // values of a block
constexpr int F8_FRAG = 1024;    // bytes of a fragment; two along K are a block
constexpr int F8_ROWS = 256;     // packed rows are a multiple of this
constexpr int F8_NMAX = 1 << 24, F8_KMAX = 1 << 20;

__host__ __device__ inline int f8_up(int n, int m) { return (n + m - 1) / m * m; }
struct F8Layout {
  int rows, kb, kb4;      // padded rows, blocks, words of exponents per row
  size_t scales, total;   // byte offsets
};
__host__ __device__ inline F8Layout f8_layout(int rows, int K) {
  F8Layout l;
  l.rows = f8_up(rows, F8_ROWS);
  l.kb = f8_up(K, F8_KB) / F8_KB;
  l.kb4 = (l.kb + 3) / 4;
  l.scales = (size_t)l.rows * l.kb * F8_KB;
  l.total = (l.scales + (size_t)l.rows * l.kb4 * 4 + 255) & ~(size_t)255;
  return l;
}

// One wave per block of 16 rows: lane l takes row l % 16, values 16 (l / 16) .. + 15 of both fragments.  A value that is not
// finite becomes NaN, the one such value that e4m3 has.
template <typename T>
__global__ void __launch_bounds__(256) k_f8_pack(const T* x, long long stride, int rows, int K, F8Layout l, char* out) {
  const int lane = lane_id(), kb = blockIdx.y * 4 + wave_id(), group = blockIdx.x;
  if (kb >= l.kb4 * 4) return;
  const int r = group * 16 + (lane & 15), k0 = kb * F8_KB + (lane >> 4) * 16;
  float v[32];
  const T* row = x + (long long)min(r, rows - 1) * stride;
  if (r < rows && k0 + 80 <= K && ((uintptr_t)(row + k0) & 15) == 0) {
    constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 32 / E; i++) {
      const vu4 w = *gmem((const vu4*)(row + k0 + (i / (16 / E)) * 64) + i % (16 / E));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (sizeof(T) == 4) {
          v[4 * i + j] = __uint_as_float(w[j]);
        } else {
          v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++) {  // loads inside the row, without branches
      const int k = k0 + (j >> 4) * 64 + (j & 15);
      float f;
      if constexpr (sizeof(T) == 4)
        f = *gmem((const float*)row + min(k, K - 1));
      else
        f = __uint_as_float((uint32_t)*gmem((const uint16_t*)row + min(k, K - 1)) << 16);
      v[j] = r < rows && k < K ? f : 0.0f;
    }
  }
  uint32_t most = 0;  // the largest magnitude, as bits
#pragma unroll
  for (int j = 0; j < 32; j++) most = max(most, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  most = max(most, (uint32_t)__shfl_xor((int)most, 16));
  most = max(most, (uint32_t)__shfl_xor((int)most, 32));
  // 448 = 1.75 * 2^8: biased exponent of the block, one more where the fraction is above .75; at least 0 (2^-127)
  const int e = max((int)(most >> 23) - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0), 0);
  if ((lane >> 4) == 0) *((uint8_t*)(out + l.scales) + (((size_t)group * l.kb4 + kb / 4) * 16 + lane) * 4 + (kb & 3)) = (uint8_t)(kb < l.kb ? e : 0);
  if (kb >= l.kb) return;
  const float up = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e)
  uint32_t q[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = fabsf(v[4 * j + i]) <= F32_MAX ? v[4 * j + i] * up : NAN;
    q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), true);
  }
  vu4* d = (vu4*)(out + ((size_t)group * l.kb + kb) * 2 * F8_FRAG);
  d[lane] = (vu4){q[0], q[1], q[2], q[3]};
  d[64 + lane] = (vu4){q[4], q[5], q[6], q[7]};
}

struct F8Args {
  const char* w;   // packed weights
  const char* x;   // packed hidden states
  F8Layout lw, lx;
  int N, T;
  void* out;       // logits: fp32 or bf16 [T][out_stride], or null
  long long out_stride;
  const int* tok;  // scoring
  const float* temp;
  float4* part;    // [T][parts] m, s, t
  float* given;    // [T] the given tokens' logits
  int parts;
};

// bf16 operand of product h (0, 1) of a fragment's 16 bytes, times the block's scale
template <int H>
__device__ __forceinline__ f8_b8 f8_wide(vu4 r, float scale) {
  union {
    f8_b2 p[4];
    f8_b8 v;
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[2 * H], scale, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[2 * H], scale, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[2 * H + 1], scale, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[2 * H + 1], scale, true);
  return u.v;
}
__device__ __forceinline__ vf4 f8_mfma(f8_b8 a, f8_b8 b, vf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// the scale of block k from its word of four exponents
__device__ __forceinline__ float f8_scale(uint32_t word, int k) { return __uint_as_float(((word >> (8 * (k & 3))) & 255u) << 23); }

// bits of x rounded to bf16, nearest even; NaN stays NaN
__device__ __forceinline__ uint32_t f8_bf16(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
// Four consecutive logits of one hidden state
template <typename O>
__device__ __forceinline__ void f8_put(O* out, long long stride, int t, int n, int T, int N, vf4 v, bool wide) {
  if (t >= T || n >= N) return;
  O* p = out + (long long)t * stride + n;
  if (wide && n + 4 <= N) {
    if constexpr (sizeof(O) == 4)
      *(vf4*)p = v;
    else
      *(uint2*)p = make_uint2(f8_bf16(v[0]) | f8_bf16(v[1]) << 16, f8_bf16(v[2]) | f8_bf16(v[3]) << 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (n + i < N) {
      if constexpr (sizeof(O) == 4)
        p[i] = v[i];
      else
        p[i] = (O)f8_bf16(v[i]);
    }
}

// A wave's logits of hidden state `t` (one of the lane's 16-lane column) at rows n0 + 16 i + 4 (lane / 16) + r, joined over the
// column's four lanes; the given token's logit goes to a.given.
template <int F>
__device__ __forceinline__ Lse f8_stats(const F8Args& a, const vf4* y, int t, int n0) {
  const int tok = t < a.T ? a.tok[t] : -1;
  const float c = lse_scale(a.temp && t < a.T ? a.temp[t] : 1.0f);
  const int nq = n0 + 4 * (lane_id() >> 4);
  Lse v = {-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < F; i++)
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (nq + 16 * i + r < a.N) v.m = fmaxf(v.m, lse_clean(y[i][r]));
#pragma unroll
  for (int i = 0; i < F; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int n = nq + 16 * i + r;
      const float x = n < a.N ? lse_clean(y[i][r]) : -INFINITY;
      const float d = lse_d(x, v.m, c), e = lse_exp2(d);
      v.s += e;
      v.t = fmaf(e, d, v.t);
      if (n == tok) a.given[t] = x;
    }
  return lse_join_lanes(v, c, 16, 32);
}
__device__ __forceinline__ void f8_put_part(const F8Args& a, int t, int part, Lse v) { a.part[(size_t)t * a.parts + part] = make_float4(v.m, v.s, v.t, 0.0f); }
template <typename O>
__device__ __forceinline__ bool f8_can_be_wide(const F8Args& a) {
  return (a.out_stride & 3) == 0 && ((uintptr_t)a.out & (4 * sizeof(O) - 1)) == 0;
}
template <typename O>
using f8_out = std::conditional_t<std::is_void_v<O>, float, O>;

// Few hidden states (T <= 16 TF): the weights' bytes bound it.  A workgroup takes G groups of 16 weight rows, its 4 waves a
// quarter of K each, straight from memory into registers, one block ahead; their sums meet in LDS.
template <typename O, int G, int TF>
__global__ void __launch_bounds__(256) k_f8_few(F8Args a) {
  __shared__ vf4 s_acc[4][G * TF][64];
  __shared__ Lse s_lse[G][16 * TF];
  const int lane = lane_id(), wave = wave_id(), g0 = blockIdx.x * G;
  const int kb = a.lw.kb, kb4 = a.lw.kb4, per = (kb + 3) / 4, lo = wave * per, hi = min(lo + per, kb);
  const char* pw = a.w + (size_t)g0 * kb * (2 * F8_FRAG) + 16 * lane;
  const char* px = a.x + 16 * lane;
  const uint32_t* qw = (const uint32_t*)(a.w + a.lw.scales) + (size_t)g0 * kb4 * 16 + (lane & 15);
  const uint32_t* qx = (const uint32_t*)(a.x + a.lx.scales) + (lane & 15);
  vf4 acc[G][TF] = {};
  vu4 w[G][2], x[TF][2];
  uint32_t ew[G], ex[TF];
  auto load = [&](int k) {
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int h = 0; h < 2; h++) w[g][h] = *gmem((const vu4*)(pw + ((size_t)g * kb + k) * (2 * F8_FRAG) + h * F8_FRAG));
#pragma unroll
    for (int j = 0; j < TF; j++)
#pragma unroll
      for (int h = 0; h < 2; h++) x[j][h] = *gmem((const vu4*)(px + ((size_t)j * kb + k) * (2 * F8_FRAG) + h * F8_FRAG));
#pragma unroll
    for (int g = 0; g < G; g++) ew[g] = *gmem(qw + ((size_t)g * kb4 + k / 4) * 16);
#pragma unroll
    for (int j = 0; j < TF; j++) ex[j] = *gmem(qx + ((size_t)j * kb4 + k / 4) * 16);
  };
  if (lo < hi) load(lo);
  for (int k = lo; k < hi; k++) {
    vu4 cw[G][2], cx[TF][2];
    float sw[G], sx[TF];
#pragma unroll
    for (int g = 0; g < G; g++) {
      cw[g][0] = w[g][0];
      cw[g][1] = w[g][1];
      sw[g] = f8_scale(ew[g], k);
    }
#pragma unroll
    for (int j = 0; j < TF; j++) {
      cx[j][0] = x[j][0];
      cx[j][1] = x[j][1];
      sx[j] = f8_scale(ex[j], k);
    }
    load(min(k + 1, hi - 1));
#pragma unroll
    for (int h = 0; h < 2; h++) {
      f8_b8 b0[TF], b1[TF];
#pragma unroll
      for (int j = 0; j < TF; j++) {
        b0[j] = f8_wide<0>(cx[j][h], sx[j]);
        b1[j] = f8_wide<1>(cx[j][h], sx[j]);
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        const f8_b8 a0 = f8_wide<0>(cw[g][h], sw[g]), a1 = f8_wide<1>(cw[g][h], sw[g]);
#pragma unroll
        for (int j = 0; j < TF; j++) acc[g][j] = f8_mfma(a1, b1[j], f8_mfma(a0, b0[j], acc[g][j]));
      }
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int j = 0; j < TF; j++) s_acc[wave][g * TF + j][lane] = acc[g][j];
  bar();
  const bool wide = f8_can_be_wide<f8_out<O>>(a);
  for (int i = wave; i < G * TF; i += 4) {
    const int g = i / TF, t = 16 * (i % TF) + (lane & 15), n0 = 16 * (g0 + g);
    const vf4 y = (s_acc[0][i][lane] + s_acc[1][i][lane]) + (s_acc[2][i][lane] + s_acc[3][i][lane]);
    if constexpr (std::is_void_v<O>) {
      const Lse v = f8_stats<1>(a, &y, t, n0);
      if (lane < 16) s_lse[g][t] = v;
    } else {
      f8_put<O>((O*)a.out, a.out_stride, t, n0 + 4 * (lane >> 4), a.T, a.N, y, wide);
    }
  }
  if constexpr (std::is_void_v<O>) {
    bar();
    const int t = threadIdx.x;
    if (t < 16 * TF && t < a.T) {
      Lse v = s_lse[0][t];
      const float c = lse_scale(a.temp ? a.temp[t] : 1.0f);
#pragma unroll
      for (int g = 1; g < G; g++) v = lse_join(v, s_lse[g][t], c);
      f8_put_part(a, t, blockIdx.x, v);
    }
  }
}

// Tiles of BN weight rows x BT hidden states, WN x WT waves.  A block of 128 along K is a stage: in registers while the one
// before is computed, then in one of two LDS buffers.
template <typename O, int BN, int BT, int WN, int WT>
__global__ void __launch_bounds__(64 * WN * WT, 2) k_f8_tile(F8Args a, int tiles_n, int tiles_t) {
  constexpr int NT = 64 * WN * WT, GN = BN / 16, GT = BT / 16, FN = GN / WN, FT = GT / WT, GB = 2 * F8_FRAG;
  constexpr int LN = GN * GB / (16 * NT), LT = GT * GB / (16 * NT), STEP = 16 * NT / GB;  // loads of a thread; groups of one load
  static_assert(LN * 16 * NT == GN * GB && LT * 16 * NT == GT * GB && STEP * GB == 16 * NT, "whole loads");
  static_assert(BN + BT <= NT, "a thread per row for the scales");
  __shared__ vu4 s_buf[2][(GN + GT) * GB / 16];
  __shared__ uint32_t s_sc[2][BN + BT];
  __shared__ Lse s_lse[std::is_void_v<O> ? WN : 1][std::is_void_v<O> ? BT : 1];
  // XCD x (workgroups x, x + 8, ..) takes the tiles of weight rows x, x + 8, .., all of their hidden states in a row: the
  // weights of a tile come into one L2 once
  const int seq = blockIdx.x >> 3, tn = (seq / tiles_t) * 8 + (blockIdx.x & 7), tt = seq % tiles_t;
  if (tn >= tiles_n) return;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), wn = wave / WT, wt = wave % WT;
  const int n0 = tn * BN, t0 = tt * BT, kb = a.lw.kb, kb4 = a.lw.kb4;
  const size_t run = (size_t)kb * GB;  // bytes of a group
  const char* pw = a.w + (size_t)(n0 / 16) * run + (size_t)(tid * 16 / GB) * run + tid * 16 % GB;
  const char* px = a.x + (size_t)(t0 / 16) * run + (size_t)(tid * 16 / GB) * run + tid * 16 % GB;
  const int row = tid < BN ? n0 + tid : t0 + tid - BN;
  const uint32_t* ps = (const uint32_t*)(tid < BN ? a.w + a.lw.scales : a.x + a.lx.scales) + (size_t)(row / 16) * kb4 * 16 + row % 16;
  const bool has_scale = tid < BN + BT;
  vu4 r[LN + LT];
  auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < LN; i++) r[i] = *gmem((const vu4*)(pw + i * STEP * run + (size_t)k * GB));
#pragma unroll
    for (int i = 0; i < LT; i++) r[LN + i] = *gmem((const vu4*)(px + i * STEP * run + (size_t)k * GB));
  };
  auto store = [&](int b) {
#pragma unroll
    for (int i = 0; i < LN + LT; i++) s_buf[b][i * NT + tid] = r[i];
  };
  uint32_t word = 0;
  if (has_scale) s_sc[0][tid] = *gmem(ps);
  load(0);
  store(0);
  load(min(1, kb - 1));
  bar();
  vf4 acc[FN][FT] = {};
  for (int k = 0; k < kb; k++) {
    if (k + 1 < kb) store((k + 1) & 1);
    if ((k & 3) == 0 && has_scale) word = *gmem(ps + (size_t)min(k / 4 + 1, kb4 - 1) * 16);
    if ((k & 3) == 3 && has_scale) s_sc[(k / 4 + 1) & 1][tid] = word;
    load(min(k + 2, kb - 1));
    const uint32_t* sc = s_sc[(k / 4) & 1];
    const vu4* buf = s_buf[k & 1] + lane;
    float sw[FN], sx[FT];
#pragma unroll
    for (int i = 0; i < FN; i++) sw[i] = f8_scale(sc[(wn * FN + i) * 16 + (lane & 15)], k);
#pragma unroll
    for (int j = 0; j < FT; j++) sx[j] = f8_scale(sc[BN + (wt * FT + j) * 16 + (lane & 15)], k);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      f8_b8 b0[FT], b1[FT];
#pragma unroll
      for (int j = 0; j < FT; j++) {
        const vu4 x = buf[(GN + wt * FT + j) * (GB / 16) + h * 64];
        b0[j] = f8_wide<0>(x, sx[j]);
        b1[j] = f8_wide<1>(x, sx[j]);
      }
#pragma unroll
      for (int i = 0; i < FN; i++) {
        const vu4 w = buf[(wn * FN + i) * (GB / 16) + h * 64];
        const f8_b8 a0 = f8_wide<0>(w, sw[i]), a1 = f8_wide<1>(w, sw[i]);
#pragma unroll
        for (int j = 0; j < FT; j++) acc[i][j] = f8_mfma(a0, b0[j], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FT; j++) acc[i][j] = f8_mfma(a1, b1[j], acc[i][j]);
      }
    }
    bar();
  }
  const bool wide = f8_can_be_wide<f8_out<O>>(a);
#pragma unroll
  for (int j = 0; j < FT; j++) {
    const int tl = (wt * FT + j) * 16 + (lane & 15), n = n0 + wn * FN * 16;
    vf4 y[FN];
#pragma unroll
    for (int i = 0; i < FN; i++) y[i] = acc[i][j];
    if constexpr (std::is_void_v<O>) {
      const Lse v = f8_stats<FN>(a, y, t0 + tl, n);
      if (lane < 16) s_lse[wn][tl] = v;
    } else {
#pragma unroll
      for (int i = 0; i < FN; i++) f8_put<O>((O*)a.out, a.out_stride, t0 + tl, n + 16 * i + 4 * (lane >> 4), a.T, a.N, y[i], wide);
    }
  }
  if constexpr (std::is_void_v<O>) {
    bar();
    const int t = t0 + tid;
    if (tid < BT && t < a.T) {
      Lse v = s_lse[0][tid];
      const float c = lse_scale(a.temp ? a.temp[t] : 1.0f);
#pragma unroll
      for (int i = 1; i < WN; i++) v = lse_join(v, s_lse[i][tid], c);
      f8_put_part(a, t, tn, v);
    }
  }
}
// One wave per hidden state: its parts joined
__global__ void __launch_bounds__(256) k_f8_score(F8Args a, float* out_lp, float* out_h) {
  const int lane = lane_id(), t = blockIdx.x * 4 + wave_id();
  if (t >= a.T) return;
  const float temp = a.temp ? a.temp[t] : 1.0f, c = lse_scale(temp);
  Lse v = {-INFINITY, 0.0f, 0.0f};
  for (int i = lane; i < a.parts; i += 64) {
    const float4 q = a.part[(size_t)t * a.parts + i];
    v = lse_join(v, {q.x, q.y, q.z}, c);
  }
  v = lse_join_lanes(v, c, 1, 32);
  if (lane) return;
  const int tok = a.tok[t];
  out_lp[t] = tok >= 0 && tok < a.N ? lse_logprob(v, a.given[t], temp) : 0.0f;
  if (out_h) out_h[t] = lse_entropy(v);
}

template <typename T>
int f8_pack(const void* x, long long stride, int rows, int K, char* out, hipStream_t st) {
  const F8Layout l = f8_layout(rows, K);
  hipLaunchKernelGGL((k_f8_pack<T>), dim3(l.rows / 16, l.kb4), dim3(256), 0, st, (const T*)x, stride, rows, K, l, out);
  return (int)hipGetLastError();
}

// What runs T hidden states against N weight rows: row groups of a workgroup of k_f8_few (0: k_f8_tile), the tile, and the
// parts that scoring joins per hidden state.
struct F8Plan {
  int groups, frags, bt, parts;
};
constexpr int F8_BN = 256;
inline F8Plan f8_plan(int T, int N) {
  F8Plan p = {};
  if (T <= 64) {
    p.frags = T <= 16 ? 1 : T <= 32 ? 2 : 4;
    // one group to a workgroup where the card would not be full of four
    p.groups = f8_up(N, 64) / 64 < 512 ? 1 : p.frags == 4 ? 2 : 4;
    p.parts = f8_up(N, 16 * p.groups) / (16 * p.groups);
  } else {
    p.bt = T <= 128 ? 128 : 256;
    p.parts = f8_up(N, F8_BN) / F8_BN;
  }
  return p;
}
struct F8Ws {
  size_t part, given, total;
};
inline F8Ws f8_ws(int T, int N, int K, bool score) {
  F8Ws w;
  w.part = f8_layout(T, K).total;
  w.given = w.part + (score ? (size_t)T * f8_plan(T, N).parts * sizeof(float4) : 0);
  w.total = (w.given + (score ? (size_t)T * 4 : 0) + 255) & ~(size_t)255;
  return w;
}
inline bool f8_shape(int T, int N, int K) { return T >= 1 && N >= 1 && K >= 1; }
inline bool f8_fits(int T, int N, int K) { return N <= F8_NMAX && K <= F8_KMAX && T <= (1 << 22); }
inline bool f8_aligned(const void* p) { return p && ((uintptr_t)p & 255) == 0; }

}  // namespace qws

extern "C" size_t qws_fp8_pack_bytes(int N, int K) { return qws::f8_shape(1, N, K) && qws::f8_fits(1, N, K) ? qws::f8_layout(N, K).total : 0; }

extern "C" int qws_fp8_pack(const void* w, int dtype, int N, int K, long long row_stride, void* packed, void* stream) {
  using namespace qws;
  if (!f8_shape(1, N, K) || (dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) || !w || row_stride < 0 || !f8_aligned(packed)) return QWS_ERR_INVALID;
  if ((uintptr_t)w & (dtype == QWS_DTYPE_F32 ? 3 : 1)) return QWS_ERR_INVALID;
  if (!f8_fits(1, N, K)) return QWS_ERR_NOT_SUPPORTED;
  return dtype == QWS_DTYPE_F32 ? f8_pack<float>(w, row_stride, N, K, (char*)packed, (hipStream_t)stream)
                                : f8_pack<uint16_t>(w, row_stride, N, K, (char*)packed, (hipStream_t)stream);
}

extern "C" size_t qws_fp8_head_ws_bytes(int T, int N, int K) {
  return qws::f8_shape(T, N, K) && qws::f8_fits(T, N, K) ? qws::f8_ws(T, N, K, false).total : 0;
}

extern "C" size_t qws_fp8_score_ws_bytes(int T, int N, int K) {
  return qws::f8_shape(T, N, K) && qws::f8_fits(T, N, K) ? qws::f8_ws(T, N, K, true).total : 0;
}

namespace qws {
// the checks that both products share; QWS_OK with T = 0: nothing to do
static int f8_check(const void* packed, int N, int K, const void* x, long long x_stride, int T, const void* ws) {
  if (!f8_shape(1, N, K) || T < 0 || x_stride < 0 || !f8_aligned(packed)) return QWS_ERR_INVALID;
  if (!f8_fits(T, N, K)) return QWS_ERR_NOT_SUPPORTED;
  if (T && (!x || ((uintptr_t)x & 1) || !f8_aligned(ws))) return QWS_ERR_INVALID;
  return QWS_OK;
}
static F8Args f8_args(const void* packed, int N, int K, int T, const void* ws) {
  F8Args a = {};
  a.w = (const char*)packed;
  a.x = (const char*)ws;
  a.lw = f8_layout(N, K);
  a.lx = f8_layout(T, K);
  a.N = N;
  a.T = T;
  return a;
}
template <typename O, int G, int TF>
static void f8_few(const F8Args& a, hipStream_t st) {
  hipLaunchKernelGGL((k_f8_few<O, G, TF>), dim3((a.N + 16 * G - 1) / (16 * G)), dim3(256), 0, st, a);
}
template <typename O, int BT, int WN, int WT>
static void f8_tile(const F8Args& a, hipStream_t st) {
  const int tn = (a.N + F8_BN - 1) / F8_BN, tt = (a.T + BT - 1) / BT;
  hipLaunchKernelGGL((k_f8_tile<O, F8_BN, BT, WN, WT>), dim3((tn + 7) / 8 * 8 * tt), dim3(64 * WN * WT), 0, st, a, tn, tt);
}
template <typename O>
static int f8_product(F8Args a, hipStream_t st) {
  const F8Plan p = f8_plan(a.T, a.N);
  a.parts = p.parts;
  if (p.groups == 0)
    p.bt == 128 ? f8_tile<O, 128, 4, 2>(a, st) : f8_tile<O, 256, 2, 4>(a, st);
  else if (p.frags == 1)
    p.groups == 1 ? f8_few<O, 1, 1>(a, st) : f8_few<O, 4, 1>(a, st);
  else if (p.frags == 2)
    p.groups == 1 ? f8_few<O, 1, 2>(a, st) : f8_few<O, 4, 2>(a, st);
  else
    p.groups == 1 ? f8_few<O, 1, 4>(a, st) : f8_few<O, 2, 4>(a, st);
  return (int)hipGetLastError();
}
}  // namespace qws

extern "C" int qws_fp8_head(const void* packed, int N, int K, const void* x, long long x_stride, int T, void* out, int out_dtype, long long out_stride, void* ws,
                            size_t ws_bytes, void* stream) {
  using namespace qws;
  const int c = f8_check(packed, N, K, x, x_stride, T, ws);
  if (c != QWS_OK) return c;
  if (out_dtype != QWS_DTYPE_F32 && out_dtype != QWS_DTYPE_BF16) return QWS_ERR_INVALID;
  if (T == 0) return QWS_OK;
  if (!out || ((uintptr_t)out & (out_dtype == QWS_DTYPE_F32 ? 3 : 1)) || (T > 1 && out_stride < N) || ws_bytes < f8_ws(T, N, K, false).total) return QWS_ERR_INVALID;
  const int e = f8_pack<uint16_t>(x, x_stride, T, K, (char*)ws, (hipStream_t)stream);
  if (e) return e;
  F8Args a = f8_args(packed, N, K, T, ws);
  a.out = out;
  a.out_stride = out_stride;
  return out_dtype == QWS_DTYPE_F32 ? f8_product<float>(a, (hipStream_t)stream) : f8_product<uint16_t>(a, (hipStream_t)stream);
}

extern "C" int qws_fp8_score(const void* packed, int N, int K, const void* x, long long x_stride, int T, const int* tokens, const float* temperature,
                             float* out_logprobs, float* out_entropy, void* ws, size_t ws_bytes, void* stream) {
  using namespace qws;
  const int c = f8_check(packed, N, K, x, x_stride, T, ws);
  if (c != QWS_OK || T == 0) return c;
  const F8Ws w = f8_ws(T, N, K, true);
  if (!tokens || !out_logprobs || ws_bytes < w.total) return QWS_ERR_INVALID;
  int e = f8_pack<uint16_t>(x, x_stride, T, K, (char*)ws, (hipStream_t)stream);
  if (e) return e;
  F8Args a = f8_args(packed, N, K, T, ws);
  a.tok = tokens;
  a.temp = temperature;
  a.part = (float4*)((char*)ws + w.part);
  a.given = (float*)((char*)ws + w.given);
  a.parts = f8_plan(T, N).parts;
  e = f8_product<void>(a, (hipStream_t)stream);
  if (e) return e;
  hipLaunchKernelGGL(k_f8_score, dim3((T + 3) / 4), dim3(256), 0, (hipStream_t)stream, a, out_logprobs, out_entropy);
  return (int)hipGetLastError();
}
