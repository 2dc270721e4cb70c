// qws 8-bit head: logits of T hidden states from a head kept in 8 bits, and the scoring of given tokens by the same
// product without the logits in memory (the definitions: include/qws.h qws_fp8_*).
//
// Numbers.  A block of 128 consecutive values of a row (a weight row or a hidden state) is held as e4m3 values q and one
// exponent e, x ~ q 2^e, with e the least whole number such that max|x| <= 448 * 2^e: the scaling itself is exact.
//
// Why the products run on the bf16 matrix instruction.  The 8-bit ones (16x16x32 and 16x16x128, with and without scales)
// align a group's products to the largest and cut what lies about 2^-13 below it: measured over 128 products of normal
// data 1.4e-5 of the result's norm, and ten times that with a few large columns.  e4m3 values times a power of two are
// exact in bf16 (down to its least, 2^-133), whose instruction sums exact products in fp32 (measured 7e-8).
// v_cvt_scalef32_pk_bf16_fp8 turns two values and their block's scale into bf16 at the rate of any vector instruction, so the
// scales cost nothing more.
//
// Layout.  16 rows x 64 values are a fragment of 1 KB: lane l's 16 bytes are row l % 16, values 16 (l / 16) .. + 15, the
// operands of two 16x16x32 products.  (Which 32 of the values share a product does not matter, as long as both operands
// take the same.)  Every load of a wave is 1 KB of consecutive bytes, in memory and in LDS.  A tile's fragments (256 weight
// rows; the hidden states of a workgroup) lie together for each 64 values of K, so that a workgroup copies runs of several
// KB.  The exponents (biased by 127) of four consecutive blocks are the bytes of one word per row, a tile's words together.
// Rows and values beyond N, T and K are 0.
#include "qws_lds.h"
#include "qws_lse.h"

#include <type_traits>
#include <utility>

namespace qws {

typedef __bf16 f8_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 f8_b8 __attribute__((ext_vector_type(8)));

constexpr int F8_KB = 128;       // values of a block
constexpr int F8_FRAG = 1024;    // bytes of a fragment; two along K are a block
constexpr int F8_ROWS = 256;     // weight rows of a tile
constexpr int F8_CUS = 256;
constexpr int F8_NMAX = 1 << 24, F8_KMAX = 1 << 20;

__host__ __device__ inline int f8_up(int n, int m) { return (n + m - 1) / m * m; }
struct F8Layout {
  int rows, kb, kb4;      // padded rows, blocks, words of exponents per row
  int groups;             // groups of 16 rows of a tile
  size_t scales, total;   // byte offsets
};
// rows: in whole tiles; bytes: of a value
__host__ __device__ inline F8Layout f8_layout(int rows, int K, int groups, int bytes) {
  F8Layout l;
  l.groups = groups;
  l.rows = f8_up(rows, 16 * groups);
  l.kb = f8_up(K, F8_KB) / F8_KB;
  l.kb4 = (l.kb + 3) / 4;
  l.scales = (size_t)l.rows * l.kb * F8_KB * bytes;
  l.total = (l.scales + (bytes == 1 ? (size_t)l.rows * l.kb4 * 4 : 0) + 255) & ~(size_t)255;
  return l;
}
__host__ __device__ inline F8Layout f8_weights(int N, int K) { return f8_layout(N, K, F8_ROWS / 16, 1); }

// bf16 operand of product h (0, 1) of a fragment's 16 bytes, times the block's scale.  Of the scale the instruction reads the
// exponent bits alone: none set (0.0f as a number, biased exponent 0) is 2^-127, as any others are theirs.
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

// The biased exponent of a block whose largest magnitude is `most` (as bits): 448 = 1.75 * 2^8, so the value's own less 8, one
// more where its fraction is above .75; at least 0 (2^-127)
__device__ __forceinline__ int f8_exponent(uint32_t most) { return max((int)(most >> 23) - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0), 0); }
// four values over the block's scale, rounded to e4m3; one that is not finite becomes NaN, the only such value it has
__device__ __forceinline__ uint32_t f8_four(const float* v, int e) {
  const float up = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e)
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; i++) f[i] = fabsf(v[i]) <= F32_MAX ? v[i] * up : NAN;
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), true);
}

// One wave per block of 16 rows: lane l takes row l % 16, values 16 (l / 16) .. + 15 of both fragments, so that a block's
// largest value is two steps over lanes away and a fragment leaves as 1 KB.  Bound by memory (248,320 x 5,120 bf16 weights, 2.54
// GB read and 1.28 GB written: 780 us, 4.9 TB/s, the rate of a large copy); a few hidden states are one launch's latency
// (4.7 us).
//   WIDE: the values as bf16 instead (exact), as k_f8_tile takes hidden states: product h of fragment c is 1 KB of its own.
template <typename T, bool WIDE>
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
  const int e = f8_exponent(most);
  if (WIDE && kb >= l.kb) return;
  uint32_t q[8];
#pragma unroll
  for (int j = 0; j < 8; j++) q[j] = f8_four(v + 4 * j, e);
  const size_t place = ((size_t)(group / l.groups) * l.kb + kb) * 2 * l.groups + group % l.groups;  // fragment 0 of the block; fragment 1: + l.groups
  if constexpr (WIDE) {
    const float scale = __uint_as_float((uint32_t)e << 23);
    vu4* d = (vu4*)(out + place * 2 * F8_FRAG);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const vu4 w = {q[4 * c], q[4 * c + 1], q[4 * c + 2], q[4 * c + 3]};
      d[c * l.groups * 128 + lane] = __builtin_bit_cast(vu4, f8_wide<0>(w, scale));
      d[c * l.groups * 128 + 64 + lane] = __builtin_bit_cast(vu4, f8_wide<1>(w, scale));
    }
  } else {
    if ((lane >> 4) == 0) {
      const size_t word = ((size_t)(group / l.groups) * l.kb4 + kb / 4) * l.groups * 16 + group % l.groups * 16 + lane;
      *((uint8_t*)(out + l.scales) + word * 4 + (kb & 3)) = (uint8_t)(kb < l.kb ? e : 0);
    }
    if (kb >= l.kb) return;
    vu4* d = (vu4*)(out + place * F8_FRAG);
    d[lane] = (vu4){q[0], q[1], q[2], q[3]};
    d[l.groups * 64 + lane] = (vu4){q[4], q[5], q[6], q[7]};
  }
}

struct F8Args {
  const char* w;   // packed weights
  const char* x;   // packed hidden states, or the hidden states themselves
  F8Layout lw, lx;
  int N, T, K;
  long long x_stride;  // hidden states as they came: elements
  void* out;       // logits: fp32 or bf16 [T][out_stride], or null
  long long out_stride;
  const int* tok;  // scoring
  const float* temp;
  float4* part;    // [T][parts] m, s, t
  float* given;    // [T] the given tokens' logits
  int parts;
};

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

// Logits y of hidden state `t` at rows n0 + 16 i + 4 (lane / 16) + r, joined over the four lanes that hold t; the logit of its
// given token `tok` goes to a.given.  c: the temperature's scale.
template <int F>
__device__ __forceinline__ Lse f8_stats(const F8Args& a, const vf4* y, int t, int n0, int tok, float c) {
  const int nq = n0 + 4 * (lane_id() >> 4);
  if (__any(tok >= n0 && tok < n0 + 16 * F)) {
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (nq + 16 * i + r == tok) a.given[t] = lse_clean(y[i][r]);
  }
  Lse v;
  float m = lse_max3(y[0][0], y[0][1], y[0][2]);
#pragma unroll
  for (int i = 0; i < F; i++) m = i == 0 ? lse_max3(m, y[0][3], y[0][3]) : lse_max3(lse_max3(m, y[i][0], y[i][1]), y[i][2], y[i][3]);
  const float M = c * m;
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int i = 0; i < F; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const float d = fmaf(y[i][r], c, -M), e = lse_exp2(d);
      s += e;
      q = fmaf(e, d, q);
    }
  if (n0 + 16 * F <= a.N && __all(fabsf(M) < LSE_NEAR && c <= LSE_MOST && fabsf(q) < INFINITY)) {
    v = lse_exact(m, M, s, q, c);
  } else {  // rows behind the last, NaN or extreme logits, small temperatures
    v = {-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (nq + 16 * i + r < a.N) v.m = fmaxf(v.m, lse_clean(y[i][r]));
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float d = lse_d(nq + 16 * i + r < a.N ? lse_clean(y[i][r]) : -INFINITY, v.m, c), e = lse_exp2(d);
        v.s += e;
        v.t = fmaf(e, d, v.t);
      }
  }
  return lse_join_lanes(v, c, 16, 32);
}
__device__ __forceinline__ int f8_token(const F8Args& a, int t) { return t < a.T ? a.tok[t] : -1; }
__device__ __forceinline__ float f8_temp_scale(const F8Args& a, int t) { return lse_scale(a.temp && t < a.T ? a.temp[t] : 1.0f); }
__device__ __forceinline__ void f8_put_part(const F8Args& a, int t, int part, Lse v) { a.part[(size_t)t * a.parts + part] = make_float4(v.m, v.s, v.t, 0.0f); }
template <typename O>
__device__ __forceinline__ bool f8_can_be_wide(const F8Args& a) {
  return (a.out_stride & 3) == 0 && ((uintptr_t)a.out & (4 * sizeof(O) - 1)) == 0;
}
template <typename O>
using f8_out = std::conditional_t<std::is_void_v<O>, float, O>;

// Few hidden states (T <= 16 TF): the weights' bytes bound it.  A workgroup takes G groups of 16 weight rows, its 4 waves a
// quarter of K each, straight from memory into registers, one block ahead; their sums meet in LDS.  Every weight is used by one
// wave, so LDS would only add a step; K is split because that leaves 3,880 workgroups of 64 rows at N = 248,320 and still
// enough at N = 8,191.  One hidden state at K = 5,120, N = 248,320: 214 us, 6.0 TB/s of weights; eight: 225, 5.7 TB/s.
// From nine on large heads are k_f8_tile's, whose weights each workgroup widens once for 32 columns (f8_plan).
//   RAW (TF = 1): the hidden states as they came, 16-byte aligned vectors of 8; each workgroup rounds them into LDS itself,
//   under its first loads of weights, which for a few KB takes less than a launch of k_f8_pack.
template <int G, int TF>
constexpr int f8_sums() { return 4 * G * TF * 64 * (int)sizeof(vf4); }
__host__ __device__ inline int f8_raw_row(int kb) { return kb * F8_KB + 16; }  // bytes of a row in LDS: rows start in other banks
__host__ __device__ inline int f8_raw_bytes(int T, int kb) { return T * (f8_raw_row(kb) + kb * 4); }
template <typename O, int G, int TF, bool RAW>
__global__ void __launch_bounds__(256, RAW ? 4 : 1) k_f8_few(F8Args a) {
  extern __shared__ __attribute__((aligned(16))) char s_mem[];  // the rounded hidden states, then the sums
  vf4(*s_acc)[G * TF][64] = (vf4(*)[G * TF][64])s_mem;
  __shared__ Lse s_lse[std::is_void_v<O> ? G : 1][16 * TF];
  const int lane = lane_id(), wave = wave_id(), g0 = blockIdx.x * G;
  const int kb = a.lw.kb, kb4 = a.lw.kb4, per = (kb + 3) / 4, lo = wave * per, hi = min(lo + per, kb);
  constexpr int WG = F8_ROWS / 16;  // groups of a tile; G divides it
  const char* pw = a.w + ((size_t)(g0 / WG) * kb * 2 * WG + g0 % WG) * F8_FRAG + 16 * lane;
  const char* px = a.x + 16 * lane;
  const uint32_t* qw = (const uint32_t*)(a.w + a.lw.scales) + ((size_t)(g0 / WG) * kb4 * WG + g0 % WG) * 16 + (lane & 15);
  const uint32_t* qx = (const uint32_t*)(a.x + a.lx.scales) + (lane & 15);
  const int rs = f8_raw_row(kb), mine = min(lane & 15, a.T - 1);  // RAW: a lane without a row reads the last one, as zeros
  const char* rx = s_mem + mine * rs + 16 * (lane >> 4);
  float* rscale = (float*)(s_mem + a.T * rs);
  vf4 acc[G][TF] = {};
  vu4 w[G][2], x[TF][2];
  uint32_t ew[G], ex[TF];
  auto load_w = [&](int k) {
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int h = 0; h < 2; h++) w[g][h] = *gmem((const vu4*)(pw + ((size_t)(2 * k + h) * WG + g) * F8_FRAG));
#pragma unroll
    for (int g = 0; g < G; g++) ew[g] = *gmem(qw + ((size_t)(k / 4) * WG + g) * 16);
  };
  auto load_x = [&](int k) {
    if constexpr (RAW) {
      const bool row = (lane & 15) < a.T;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        x[0][h] = *(const vu4*)(rx + k * F8_KB + h * 64);
        if (!row) x[0][h] = (vu4){0, 0, 0, 0};
      }
      ex[0] = __float_as_uint(rscale[mine * kb + k]);
    } else {
#pragma unroll
      for (int j = 0; j < TF; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) x[j][h] = *gmem((const vu4*)(px + ((size_t)(2 * k + h) * TF + j) * F8_FRAG));
#pragma unroll
      for (int j = 0; j < TF; j++) ex[j] = *gmem(qx + ((size_t)(k / 4) * TF + j) * 16);
    }
  };
  auto load = [&](int k) {
    load_w(k);
    load_x(k);
  };
  if constexpr (RAW) {
    if (lo < hi) load_w(lo);
    // 16 lanes take a block, 8 values each
    for (int u = threadIdx.x; u < a.T * kb * 16; u += 256) {
      const int row = u / (kb * 16), k0 = u % (kb * 16) * 8;
      vu4 r = {};
      if (k0 < a.K) r = *gmem((const vu4*)((const uint16_t*)a.x + (long long)row * a.x_stride + k0));
      float v[8];
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        v[i] = __uint_as_float(i & 1 ? r[i / 2] & 0xFFFF0000u : r[i / 2] << 16);
        most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
      }
      most = max8(most);
      most = max(most, dpp_perm<0x140>(most));  // row_mirror: the other eight lanes
      const int e = f8_exponent(most);
      *(uint2*)(s_mem + row * rs + k0) = make_uint2(f8_four(v, e), f8_four(v + 4, e));
      if ((lane & 15) == 0) rscale[row * kb + k0 / F8_KB] = __uint_as_float((uint32_t)e << 23);
    }
    bar();
    if (lo < hi) load_x(lo);
  } else {
    if (lo < hi) load(lo);
  }
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
      sx[j] = RAW ? __uint_as_float(ex[j]) : f8_scale(ex[j], k);
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
  if constexpr (RAW) bar();  // the sums take the hidden states' place
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
      const Lse v = f8_stats<1>(a, &y, t, n0, f8_token(a, t), f8_temp_scale(a, t));
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
      const float c = f8_temp_scale(a, t);
#pragma unroll
      for (int g = 1; g < G; g++) v = lse_join(v, s_lse[g][t], c);
      f8_put_part(a, t, blockIdx.x, v);
    }
  }
}

// Many hidden states: the products bound it, below some 200 the weights' bytes.  A tile is WN x WT = 4 waves of 16 FN weight
// rows x 16 FT hidden states: 2 x 2, one wave to a SIMD, so that each has the registers for up to 128 x 128 sums and an operand
// read from LDS serves eight products; for up to 64 hidden states 4 x 1, so that only one wave widens a weight (widening and
// LDS reads, not products, fill its time), and two workgroups to a CU.  A stage is 64 values along K, WN FN KB of weights and
// 2 WT FT KB of hidden states (already bf16: k_f8_pack; in 8 bits each wave would widen them again: 3,687 us against 3,600),
// copied by the memory system straight into one of three LDS buffers, three stages ahead.  A stage has two halves of 32 values:
// the first half's products run while the second half's hidden states are read, then everybody meets (a wave first waits for
// its own copies of the next stage; the newest stage's stay in flight), and the second half's products run while the next
// stage's operands are read.  A half has a step for each fragment of weights: its FT products, and beside them the next
// fragment's widening to bf16, a few reads and one copy (into the buffer that the last meeting freed: over the second half and
// the next first one), little enough for the time of as many products.  A workgroup takes every 256th (512th) tile; the first
// stages of its next one are copied while it finishes the last.
//   2,048 states scored at K = 5,120, N = 248,320: 3,610 us, 1,443 TFLOP/s; without the copies 3,120, the products alone 2,330:
//   the card's power bounds them all (nothing but these products, on such values, makes 2,200 TFLOP/s, and with 32x32x16
//   products 1,910).  300 states' bf16 logits: 652 us, 1,170 TFLOP/s (20 of 320 columns are padding, and the last of 8
//   rounds of tiles is 0.6 of one).  16 states' fp32 logits: 227 us, 5.7 TB/s with them; 64: 263, 5.1 TB/s.
template <int FN, int FT, int WT>
struct F8Buf {
  vu4 w[4 / WT * FN * 64];
  vu4 x[WT * FT * 128];
  uint32_t e[256];  // exponents of the tile's weight rows
};
template <typename O, int FN, int FT, int WT>
__global__ void __launch_bounds__(256, 1) k_f8_tile(F8Args a, int tiles_n, int tiles_t) {
  constexpr int WN = 4 / WT, GN = WN * FN, BN = 16 * GN, BT = 16 * WT * FT, XW = WT * FT / 2;
  static_assert(GN % 4 == 0 && XW * 2 == WT * FT, "a stage's weights and hidden states in KB, split over the waves");
  constexpr int SUB = F8_ROWS / BN;  // workgroups' tiles of a tile as it is packed
  constexpr int NEW = GN / 4 + XW + 1;  // copies of a wave per stage: KB of weights, of hidden states, 64 exponents
  constexpr int CP = (NEW + 2 * FN - 1) / (2 * FN);  // copies of a step
  using Buf = F8Buf<FN, FT, WT>;
  __shared__ Buf b0, b1, b2;
  __shared__ Lse s_lse[std::is_void_v<O> ? WN : 1][std::is_void_v<O> ? BT : 1];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), wn = wave / WT, wt = wave % WT;
  const int kb4 = a.lw.kb4, stages = 2 * a.lw.kb;
  const uint32_t o16 = 16 * lane, o4 = 4 * lane;
  const char *pw, *px, *pe;  // the wave's copies of the tile
  // XCD x (workgroups x, x + 8, ..) takes the tiles of weight rows x, x + 8, .., all of their hidden states in a row: the
  // weights of a tile come into one L2 once
  auto row_tile = [&](int id) { return (id >> 3) / tiles_t * 8 + (id & 7); };
  auto point = [&](int id) {
    const int tn = row_tile(id), tt = (id >> 3) % tiles_t;
    pw = a.w + ((size_t)(tn / SUB) * stages * GN * SUB + tn % SUB * GN + GN / 4 * wave) * F8_FRAG;
    px = a.x + ((size_t)tt * stages * 2 * WT * FT + XW * wave) * 1024;
    pe = a.w + a.lw.scales + (size_t)(tn / SUB) * kb4 * 4 * F8_ROWS + (tn % SUB * BN + 64 * wave % BN) * 4;  // where BN is 128, twice
  };
  auto copy = [&](int k, Buf& b, auto D) {  // copy D of stage k
    constexpr int d = decltype(D)::value, xd = d - GN / 4;
    k = min(k, stages - 1);  // past the end: the last stage again, into a buffer that is not read any more
    if constexpr (d < GN / 4)
      lds_copy<d * 1024>(pw + (size_t)k * (F8_ROWS / 16 * F8_FRAG), o16, b.w + GN / 4 * wave * 64);
    else if constexpr (d < NEW - 1)
      lds_copy<xd % 4 * 1024>(px + (size_t)k * (2 * WT * FT * 1024) + xd / 4 * 4096, o16, b.x + (XW * wave + xd / 4 * 4) * 64);
    else if constexpr (d == NEW - 1)
      lds_copy_words(pe + (size_t)(k / 8) * (4 * F8_ROWS), o4, b.e + 64 * wave);
  };
  auto each = [&](auto f) {  // f(0) .. f(FN - 1), as constants
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>()), ...); }(std::make_integer_sequence<int, FN>());
  };
  // step i of the first FN steps of a stage's copies, and of the others
  auto copy_first = [&](int k, Buf& b, auto I) {
    copy(k, b, std::integral_constant<int, decltype(I)::value * CP>());
    if constexpr (CP > 1) copy(k, b, std::integral_constant<int, decltype(I)::value * CP + 1>());
  };
  auto copy_others = [&](int k, Buf& b, auto I) { copy_first(k, b, std::integral_constant<int, decltype(I)::value + FN>()); };
  auto copy_all = [&](int k, Buf& b) {
    each([&](auto I) { copy_first(k, b, I); });
    each([&](auto I) { copy_others(k, b, I); });
  };
  vu4 w[FN];
  uint32_t word[FN];
  f8_b8 x0[FT], x1[FT], q;
  vf4 acc[FN][FT];
  auto read_x = [&](const Buf& b, int h, int j) { return __builtin_bit_cast(f8_b8, b.x[((wt * FT + j) * 2 + h) * 64 + lane]); };
  auto read_w = [&](const Buf& b, int i) {
    w[i] = b.w[(wn * FN + i) * 64 + lane];
    word[i] = b.e[16 * (wn * FN + i) + (lane & 15)];
  };
  // stage k in b; `next` holds the next one, `last` the one before (free; the copies of stage k + 2 go on into it)
  auto stage = [&](int k, Buf& b, const Buf& next, Buf& last) {
    const int kb = k >> 1, kn = (k + 1) >> 1;
    each([&](auto I) {
      constexpr int i = decltype(I)::value;
#pragma unroll
      for (int j = 0; j < FT; j++)
        if (j / 2 == i) x1[j] = read_x(b, 1, j);
      const f8_b8 qn = i + 1 < FN ? f8_wide<0>(w[(i + 1) % FN], f8_scale(word[(i + 1) % FN], kb)) : f8_wide<1>(w[0], f8_scale(word[0], kb));
#pragma unroll
      for (int j = 0; j < FT; j++) acc[i][j] = f8_mfma(q, x0[j], acc[i][j]);
      copy_others(k + 2, last, I);
      q = qn;
      __builtin_amdgcn_sched_barrier(0);
    });
    lds_meet<NEW>();
    each([&](auto I) {
      constexpr int i = decltype(I)::value;
      f8_b8 qn;
      if (i + 1 < FN) qn = f8_wide<1>(w[(i + 1) % FN], f8_scale(word[(i + 1) % FN], kb));
#pragma unroll
      for (int j = 0; j < FT; j++)
        if (j / 2 == i) x0[j] = read_x(next, 0, j);
      read_w(next, i);
      if (i + 1 == FN) qn = f8_wide<0>(w[0], f8_scale(word[0], kn));
#pragma unroll
      for (int j = 0; j < FT; j++) acc[i][j] = f8_mfma(q, x1[j], acc[i][j]);
      copy_first(k + 3, b, I);
      q = qn;
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  const int total = (tiles_n + 7) / 8 * 8 * tiles_t;
  int id = blockIdx.x;
  while (id < total && row_tile(id) >= tiles_n) id += gridDim.x;
  if (id >= total) return;
  point(id);
  copy_all(0, b0);
  copy_all(1, b1);
  for (;;) {
    const int tn = row_tile(id), n0 = tn * BN, t0 = (id >> 3) % tiles_t * BT;
    each([&](auto I) { copy_first(2, b2, I); });  // the others follow in the first half
    lds_meet<NEW + (FN * CP < NEW ? FN * CP : NEW)>();
#pragma unroll
    for (int i = 0; i < FN; i++) read_w(b0, i);
#pragma unroll
    for (int j = 0; j < FT; j++) x0[j] = read_x(b0, 0, j);
    q = f8_wide<0>(w[0], f8_scale(word[0], 0));
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
      for (int j = 0; j < FT; j++) acc[i][j] = (vf4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < stages; k += 3) {
      stage(k, b0, b1, b2);
      if (k + 1 < stages) stage(k + 1, b1, b2, b0);
      if (k + 2 < stages) stage(k + 2, b2, b0, b1);
    }
    lds_meet<0>();  // the copies past the end
    do id += gridDim.x;
    while (id < total && row_tile(id) >= tiles_n);
    if (id < total) {
      point(id);
      copy_all(0, b0);
      copy_all(1, b1);
    }
    if constexpr (std::is_void_v<O>) {
      int tok[FT];
      float c[FT];
#pragma unroll
      for (int j = 0; j < FT; j++) {
        const int t = t0 + (wt * FT + j) * 16 + (lane & 15);
        tok[j] = f8_token(a, t);
        c[j] = f8_temp_scale(a, t);
      }
#pragma unroll
      for (int j = 0; j < FT; j++) {
        const int tl = (wt * FT + j) * 16 + (lane & 15);
        vf4 y[FN];
#pragma unroll
        for (int i = 0; i < FN; i++) y[i] = acc[i][j];
        const Lse v = f8_stats<FN>(a, y, t0 + tl, n0 + wn * FN * 16, tok[j], c[j]);
        if (lane < 16) s_lse[wn][tl] = v;
      }
      bar();
      const int t = t0 + tid;
      if (tid < BT && t < a.T) {  // BT <= 256 threads
        Lse v = s_lse[0][tid];
#pragma unroll
        for (int i = 1; i < WN; i++) v = lse_join(v, s_lse[i][tid], f8_temp_scale(a, t));
        f8_put_part(a, t, tn, v);
      }
      bar();  // before the next tile's statistics
    } else {
      const bool wide = f8_can_be_wide<O>(a);
#pragma unroll
      for (int j = 0; j < FT; j++)
#pragma unroll
        for (int i = 0; i < FN; i++)
          f8_put<O>((O*)a.out, a.out_stride, t0 + (wt * FT + j) * 16 + (lane & 15), n0 + (wn * FN + i) * 16 + 4 * (lane >> 4), a.T, a.N, acc[i][j], wide);
    }
    if (id >= total) return;
  }
}

// One workgroup per hidden state: its parts joined, up to 3,880 of them at the full head, four loads of a thread at once
// (by one wave a state's call took 247 us, 228 so; 2,048 states at 970 parts, 32 MB: 8.2 us)
__global__ void __launch_bounds__(256) k_f8_score(F8Args a, float* out_lp, float* out_h) {
  __shared__ Lse s_lse[4];
  const int lane = lane_id(), wave = wave_id(), t = blockIdx.x;
  const float temp = a.temp ? a.temp[t] : 1.0f, c = lse_scale(temp);
  const int tok = a.tok[t];
  const bool ok = tok >= 0 && tok < a.N;
  const float given = ok ? a.given[t] : 0.0f;
  const float4* part = a.part + (size_t)t * a.parts;
  Lse v = {-INFINITY, 0.0f, 0.0f};
  constexpr int U = 4;  // parts of a thread loaded together
  for (int i = threadIdx.x; i < a.parts; i += 256 * U) {
    float4 q[U];
#pragma unroll
    for (int u = 0; u < U; u++) q[u] = part[min(i + 256 * u, a.parts - 1)];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + 256 * u < a.parts) v = lse_join(v, {q[u].x, q[u].y, q[u].z}, c);
  }
  v = lse_join_wave(v, c);
  if (lane == 0) s_lse[wave] = v;
  bar();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < 4; w++) v = lse_join(v, s_lse[w], c);
  out_lp[t] = ok ? lse_logprob(v, given, temp) : 0.0f;
  if (out_h) out_h[t] = lse_entropy(v);
}

template <typename T, bool WIDE>
int f8_pack(const void* x, long long stride, int rows, int K, F8Layout l, char* out, hipStream_t st) {
  hipLaunchKernelGGL((k_f8_pack<T, WIDE>), dim3(l.rows / 16, l.kb4), dim3(256), 0, st, (const T*)x, stride, rows, K, l, out);
  return (int)hipGetLastError();
}

// What runs T hidden states against N weight rows: k_f8_few with `groups` row groups to a workgroup and `frags` fragments of
// hidden states, or (groups = 0) k_f8_tile with waves of fn x frags fragments, wt of them along the hidden states; the parts
// that scoring joins per hidden state.
// Measured, us, k_f8_few / tiles of 256 x 32: 9 states' logits at K = 5,120, N = 248,320 231 / 229, 16 246 / 236, 32 267 / 245; 12
// states at K = 1,280, N = 24,000 18 / 23, at 40,000 23 / 24, at 50,000 27 / 26 (32: 21 / 23, 26 / 24, 29 / 26): from more
// tiles than half the CUs on.  Tiles of 256 x 64 / of 2 x 2 waves: 64 states 274 / 290, 96 361 / 304; at N = 24,000 26 / 25.
// Without that many tiles k_f8_few / 2 x 2 waves: 64 states at N = 8,191, K = 1,000 19 / 24, at N = 32,001, K = 1,280 30 / 27.
struct F8Plan {
  int groups, frags, fn, wt, parts;
  int rows() const { return 64 / wt * fn; }  // of a tile
  int cols() const { return 16 * wt * frags; }
};
inline F8Plan f8_plan(int T, int N) {
  F8Plan p = {};
  const bool many = N > 256 * F8_CUS / 2;
  if (T <= 8 || (T <= 32 && !many) || (T <= 64 && N < 128 * F8_CUS / 2)) {
    p.frags = T <= 16 ? 1 : T <= 32 ? 2 : 4;
    p.groups = p.frags == 4 ? 2 : 4;
    p.parts = f8_up(N, 16 * p.groups) / (16 * p.groups);
    return p;
  }
  if (T <= 64 && many) {
    p.fn = 4;
    p.wt = 1;
    p.frags = T <= 32 ? 2 : 4;
    p.parts = f8_up(N, p.rows()) / p.rows();
    return p;
  }
  p.wt = 2;
  // The least rounds of workgroups times a tile's time: its products, per fragment of weights their widening, and a constant
  // (512 states: tiles of 256 x 256 965 us, 128 x 256 1,080, 256 x 128 1,063; 300: 256 x 160 654, 256 x 128 796; 77 states
  // at N = 32,001, K = 1,280: 128 x 96 27, 256 x 96 33).
  long long best = 0;
  for (int fn = 8; fn >= 4; fn -= 4)
    for (int frags = 8; frags >= 3; frags--) {
      const long long tiles = (long long)(f8_up(N, 32 * fn) / (32 * fn)) * (f8_up(T, 32 * frags) / (32 * frags));
      const long long cost = (tiles + F8_CUS - 1) / F8_CUS * (fn * (4 * frags + 3) + 38);
      if (p.fn == 0 || cost < best) {
        best = cost;
        p.fn = fn;
        p.frags = frags;
      }
    }
  p.parts = f8_up(N, p.rows()) / p.rows();
  return p;
}
// Whether each workgroup of k_f8_few rounds the hidden states itself: up to 20,480 values (us with / without, K = 5,120:
// one state at N = 248,320 222 / 226, at N = 64,000 59 / 62, four 65 / 66, five 66.2 / 65.8; sixteen 552 / 241).
constexpr int F8_RAW = 20480;
inline bool f8_raw(const F8Plan& p, int T, int K, const void* x, long long stride) {
  return p.groups && p.frags == 1 && K % 8 == 0 && ((uintptr_t)x & 15) == 0 && (T == 1 || stride % 8 == 0) && T * f8_up(K, F8_KB) <= F8_RAW;
}
// the packed hidden states: a workgroup's are a tile, 8-bit or (k_f8_tile) bf16
inline F8Layout f8_states(int T, int N, int K) {
  const F8Plan p = f8_plan(T, N);
  return p.groups ? f8_layout(T, K, p.frags, 1) : f8_layout(T, K, p.wt * p.frags, 2);
}
struct F8Ws {
  size_t part, given, total;
};
inline F8Ws f8_ws(int T, int N, int K, bool score) {
  F8Ws w;
  w.part = f8_states(T, N, K).total;
  w.given = w.part + (score ? (size_t)T * f8_plan(T, N).parts * sizeof(float4) : 0);
  w.total = (w.given + (score ? (size_t)T * 4 : 0) + 255) & ~(size_t)255;
  return w;
}
inline bool f8_shape(int T, int N, int K) { return T >= 1 && N >= 1 && K >= 1; }
inline bool f8_fits(int T, int N, int K) { return N <= F8_NMAX && K <= F8_KMAX && T <= (1 << 22); }
inline bool f8_aligned(const void* p) { return p && ((uintptr_t)p & 255) == 0; }

}  // namespace qws

extern "C" size_t qws_fp8_pack_bytes(int N, int K) { return qws::f8_shape(1, N, K) && qws::f8_fits(1, N, K) ? qws::f8_weights(N, K).total : 0; }

extern "C" int qws_fp8_pack(const void* w, int dtype, int N, int K, long long row_stride, void* packed, void* stream) {
  using namespace qws;
  if (!f8_shape(1, N, K) || (dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) || !w || row_stride < 0 || !f8_aligned(packed)) return QWS_ERR_INVALID;
  if ((uintptr_t)w & (dtype == QWS_DTYPE_F32 ? 3 : 1)) return QWS_ERR_INVALID;
  if (!f8_fits(1, N, K)) return QWS_ERR_NOT_SUPPORTED;
  const F8Layout l = f8_weights(N, K);
  return dtype == QWS_DTYPE_F32 ? f8_pack<float, false>(w, row_stride, N, K, l, (char*)packed, (hipStream_t)stream)
                                : f8_pack<uint16_t, false>(w, row_stride, N, K, l, (char*)packed, (hipStream_t)stream);
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
  a.lw = f8_weights(N, K);
  a.lx = f8_states(T, N, K);
  a.N = N;
  a.T = T;
  a.K = K;
  return a;
}
template <typename O, int G, int TF, bool RAW>
static void f8_few(const F8Args& a, hipStream_t st) {
  const int raw = RAW ? f8_raw_bytes(a.T, a.lw.kb) : 0, sums = f8_sums<G, TF>();
  hipLaunchKernelGGL((k_f8_few<O, G, TF, RAW>), dim3((a.N + 16 * G - 1) / (16 * G)), dim3(256), raw > sums ? raw : sums, st, a);
}
template <typename O, int FN, int FT, int WT>
static void f8_tile(const F8Args& a, hipStream_t st) {
  constexpr int BN = 64 / WT * FN, BT = 16 * WT * FT, wgs = WT == 1 ? 2 * F8_CUS : F8_CUS;
  const int tn = f8_up(a.N, BN) / BN, tt = f8_up(a.T, BT) / BT;
  const long long total = (long long)((tn + 7) / 8 * 8) * tt;
  hipLaunchKernelGGL((k_f8_tile<O, FN, FT, WT>), dim3(total < wgs ? (int)total : wgs), dim3(256), 0, st, a, tn, tt);
}
template <typename O, int FN>
static void f8_tiles(const F8Args& a, int frags, hipStream_t st) {
  switch (frags) {
    case 3: return f8_tile<O, FN, 3, 2>(a, st);
    case 4: return f8_tile<O, FN, 4, 2>(a, st);
    case 5: return f8_tile<O, FN, 5, 2>(a, st);
    case 6: return f8_tile<O, FN, 6, 2>(a, st);
    case 7: return f8_tile<O, FN, 7, 2>(a, st);
    default: return f8_tile<O, FN, 8, 2>(a, st);
  }
}
// packs the hidden states and runs the product
template <typename O>
static int f8_product(F8Args a, int K, const void* x, long long x_stride, char* ws, hipStream_t st) {
  const F8Plan p = f8_plan(a.T, a.N);
  a.parts = p.parts;
  if (p.groups == 0 && (long long)(p.parts + 7) * (f8_up(a.T, p.cols()) / p.cols()) > 0x7FFF0000) return QWS_ERR_NOT_SUPPORTED;
  if (f8_raw(p, a.T, K, x, x_stride)) {
    a.x = (const char*)x;
    a.x_stride = x_stride;
    f8_few<O, 4, 1, true>(a, st);
    return (int)hipGetLastError();
  }
  const int e = p.groups ? f8_pack<uint16_t, false>(x, x_stride, a.T, K, a.lx, ws, st) : f8_pack<uint16_t, true>(x, x_stride, a.T, K, a.lx, ws, st);
  if (e) return e;
  if (p.groups == 0 && p.wt == 1)
    p.frags == 2 ? f8_tile<O, 4, 2, 1>(a, st) : f8_tile<O, 4, 4, 1>(a, st);
  else if (p.groups == 0)
    p.fn == 8 ? f8_tiles<O, 8>(a, p.frags, st) : f8_tiles<O, 4>(a, p.frags, st);
  else if (p.frags == 1)
    f8_few<O, 4, 1, false>(a, st);
  else if (p.frags == 2)
    f8_few<O, 4, 2, false>(a, st);
  else
    f8_few<O, 2, 4, false>(a, st);
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
  F8Args a = f8_args(packed, N, K, T, ws);
  a.out = out;
  a.out_stride = out_stride;
  return out_dtype == QWS_DTYPE_F32 ? f8_product<float>(a, K, x, x_stride, (char*)ws, (hipStream_t)stream)
                                    : f8_product<uint16_t>(a, K, x, x_stride, (char*)ws, (hipStream_t)stream);
}

extern "C" int qws_fp8_score(const void* packed, int N, int K, const void* x, long long x_stride, int T, const int* tokens, const float* temperature,
                             float* out_logprobs, float* out_entropy, void* ws, size_t ws_bytes, void* stream) {
  using namespace qws;
  const int c = f8_check(packed, N, K, x, x_stride, T, ws);
  if (c != QWS_OK || T == 0) return c;
  const F8Ws w = f8_ws(T, N, K, true);
  if (!tokens || !out_logprobs || ws_bytes < w.total) return QWS_ERR_INVALID;
  F8Args a = f8_args(packed, N, K, T, ws);
  a.tok = tokens;
  a.temp = temperature;
  a.part = (float4*)((char*)ws + w.part);
  a.given = (float*)((char*)ws + w.given);
  a.parts = f8_plan(T, N).parts;
  const int e = f8_product<void>(a, K, x, x_stride, (char*)ws, (hipStream_t)stream);
  if (e) return e;
  hipLaunchKernelGGL(k_f8_score, dim3(T), dim3(256), 0, (hipStream_t)stream, a, out_logprobs, out_entropy);
  return (int)hipGetLastError();
}
