// qws 4-bit head: logits of T hidden states from a head kept in 4 bits with a scale and a zero point for each group of 32, 64 or
// 128 weights along K (the definitions: include/qws.h qws_int4_*).
//
// Products.  y = sum over groups of s (sum_k q x - z sum_k x), q and z in 0 .. 15.  The codes enter the bf16 matrix instruction
// as 16 + q, which is exact in bf16 and takes an and-or for two of them, and for three of four pairs a shift: a code's four bits are the top of the
// fraction of a number in [16, 32).  The hidden states enter as they are, so a group's products are exact and summed in fp32; the
// 16 is taken off with the zero point, (16 + z) sum_k x, whose sum of hidden states is a product with ones, once for
// all of a wave's weights.  Then the scale is applied in fp32: nothing is rounded to fewer bits.  The offset makes a group's sum
// some five times as large as what is left of it, so its error is a few 2^-24 of the group's terms.
//
// Layout.  16 weight rows x 128 values are a fragment of 1 KB: lane l's 16 bytes are row l % 16, word j values 32 j + 8 (l / 16)
// .. + 7, the second operand of the 16x16x32 product j; a word's pairs lie so that one mask takes a pair, turned by a multiple of four,
// into the halves of a register where the fractions' top bits are (i4_word).  Four fragments (64 rows) lie together for each 128 values of K, 4 KB that one
// wave reads at once.  A scale is a word: fp32 (from bf16 or fp16: the low 13 bits are 0) with 16 + z in its low byte; the 64 words of a
// tile's rows lie together for each group.  Values beyond K are 0, rows beyond N not used.
#include "qws_lds.h"
#include "qws_lse.h"

#include <type_traits>

namespace qws {

typedef __bf16 i4_b8 __attribute__((ext_vector_type(8)));

constexpr int I4_KB = 128;     // values of a fragment's row
constexpr int I4_ROWS = 64;    // weight rows that lie together
constexpr int I4_NMAX = 1 << 24, I4_KMAX = 1 << 20, I4_TMAX = 1 << 22;

__host__ __device__ inline int i4_up(int n, int m) { return (n + m - 1) / m * m; }
struct I4Layout {
  int tiles, kb, kg;     // tiles of 64 rows, blocks of 128 values, groups of a row
  size_t scales, total;  // byte offsets
};
__host__ __device__ inline I4Layout i4_layout(int N, int K, int group) {
  I4Layout l;
  l.tiles = i4_up(N, I4_ROWS) / I4_ROWS;
  l.kb = i4_up(K, I4_KB) / I4_KB;
  l.kg = l.kb * (I4_KB / group);
  l.scales = (size_t)l.tiles * l.kb * (I4_ROWS * I4_KB / 2);
  l.total = l.scales + (size_t)l.tiles * l.kg * I4_ROWS * 4;
  return l;
}

// ------------------------------------------------------------------------------------------------ packing
struct I4Pack {
  const void* w;  // weights, or codes
  long long stride;
  const uint16_t* scales;  // given codes: bf16 or fp16 bits, a row's groups together
  long long scale_stride;
  int half;  // fp16
  const uint8_t* zeros;  // or null: 8
  long long zero_stride;
  int N, K;
  I4Layout l;
  char* out;
};
__device__ __forceinline__ uint32_t i4_nearest_bf16(float x) {  // a finite x >= 0 as the bits of a bf16 value, ties to even
  const uint32_t u = __float_as_uint(x);
  return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// Eight codes as a word: pair p = codes 2 p and 2 p + 1 at bits 3 .. 6 and 19 .. 22 of the word turned right by 4 p
__device__ __forceinline__ uint32_t i4_word(const uint32_t (&code)[8]) {
  uint32_t f[4];
#pragma unroll
  for (int p = 0; p < 4; p++) f[p] = code[2 * p] << 3 | code[2 * p + 1] << 19;
  return f[0] | f[1] << 4 | f[2] << 8 | (f[3] >> 4 | f[3] << 28);
}
// Elements k0 .. k0 + 7 of a row as bits, those from K on as 0
template <typename T>
__device__ __forceinline__ void i4_load(const T* row, int k0, int K, uint32_t (&v)[8]) {
  if (k0 + 8 <= K && ((uintptr_t)(row + k0) & (sizeof(T) == 1 ? 7 : 15)) == 0) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const vu4 w = *gmem((const vu4*)(row + k0) + h);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * h + e] = w[e];
      }
    } else if constexpr (sizeof(T) == 2) {
      const vu4 w = *gmem((const vu4*)(row + k0));
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = w[e / 2] >> (16 * (e & 1)) & 0xFFFFu;
    } else {
      const uint64_t w = *gmem((const uint64_t*)(row + k0));
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = (uint32_t)(w >> (8 * e)) & 0xFFu;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++) {  // loads inside the row, without branches
    uint32_t u;
    if constexpr (sizeof(T) == 4)
      u = *gmem((const uint32_t*)row + min(k0 + e, K - 1));
    else if constexpr (sizeof(T) == 2)
      u = *gmem((const uint16_t*)row + min(k0 + e, K - 1));
    else
      u = *gmem((const uint8_t*)row + min(k0 + e, K - 1));
    v[e] = k0 + e < K ? u : 0;
  }
}

// One wave per fragment.  T: float, uint16_t (bf16) or uint8_t (codes).  A group of a row's values lies in one to four words of
// each of four lanes.  Bound by memory.
template <typename T, int GROUP>
__global__ void __launch_bounds__(256) k_i4_pack(I4Pack a) {
  constexpr int J = GROUP / 32;  // words of a group
  const int lane = lane_id(), quad = lane >> 4, kb = blockIdx.y * 4 + wave_id();
  if (kb >= a.l.kb) return;
  const int r = blockIdx.x * 16 + (lane & 15), at = min(r, a.N - 1);
  const T* row = (const T*)a.w + (long long)at * a.stride;
  const int tile = r / I4_ROWS, in_tile = r % I4_ROWS;
  uint32_t* words = (uint32_t*)(a.out + a.l.scales) + (size_t)tile * a.l.kg * I4_ROWS + in_tile;
  uint32_t q[4];
#pragma unroll
  for (int g = 0; g < 4 / J; g++) {
    const int kg = kb * (4 / J) + g;
    uint32_t word = 16;
    if constexpr (sizeof(T) == 1) {
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int k0 = kb * I4_KB + 32 * (g * J + j) + 8 * quad;
        uint32_t code[8];
        i4_load(row, k0, a.K, code);
#pragma unroll
        for (int e = 0; e < 8; e++) code[e] &= 15u;
        q[g * J + j] = i4_word(code);
      }
      if (r < a.N && kg * GROUP < a.K) {
        const uint32_t s = *gmem(a.scales + (long long)at * a.scale_stride + kg);
        const uint32_t z = a.zeros ? *gmem(a.zeros + (long long)at * a.zero_stride + kg) & 15u : 8u;
        const uint32_t f = a.half ? __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)s)) : s << 16;
        word = ((f & 0x7FFFFFFFu) < 0x7F800000u ? f : 0x7FC00000u) | (16 + z);
      }
    } else {
      float v[J][8], lo = 0.0f, hi = 0.0f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < J; j++) {
        uint32_t bits[8];
        i4_load(row, kb * I4_KB + 32 * (g * J + j) + 8 * quad, a.K, bits);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float f = __uint_as_float(sizeof(T) == 4 ? bits[e] : bits[e] << 16);
          bad = bad || !(fabsf(f) <= F32_MAX);
          v[j][e] = f;
          lo = fminf(lo, f);
          hi = fmaxf(hi, f);
        }
      }
#pragma unroll
      for (int i = 16; i <= 32; i <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, i));
        hi = fmaxf(hi, __shfl_xor(hi, i));
        bad = __shfl_xor((int)bad, i) || bad;
      }
      const float range = (hi - lo) * (1.0f / 15.0f);
      bad = bad || !(range <= F32_MAX);
      const uint32_t s = bad ? 0 : i4_nearest_bf16(range);
      bad = bad || s >= 0x7F80u;
      const float d = s && !bad ? __uint_as_float(s << 16) : 1.0f;
      const float z = fminf(fmaxf(rintf(-lo / d), 0.0f), 15.0f);
#pragma unroll
      for (int j = 0; j < J; j++) {
        uint32_t code[8];
#pragma unroll
        for (int e = 0; e < 8; e++) code[e] = bad ? 0u : (uint32_t)fminf(fmaxf(rintf(v[j][e] / d) + z, 0.0f), 15.0f);
        q[g * J + j] = i4_word(code);
      }
      if (bad)
        word = 0x7FC00000u | 16;  // a value that is not finite, or a range past fp32: NaN
      else
        word = s << 16 | (16 + (uint32_t)z);
    }
    if (quad == 0) words[(size_t)kg * I4_ROWS] = word;
  }
  vu4* d = (vu4*)(a.out + ((size_t)tile * a.l.kb + kb) * (I4_ROWS * I4_KB / 2)) + (in_tile >> 4) * 64;
  d[lane] = (vu4){q[0], q[1], q[2], q[3]};
}

// Hidden states as rows of kb * 128 values, the last ones 0, for those whose rows a lane cannot read 16 bytes at a time
__global__ void __launch_bounds__(256) k_i4_states(const uint16_t* x, long long stride, int K, int width, uint16_t* out) {
  const uint16_t* row = x + (long long)blockIdx.x * stride;
  uint16_t* to = out + (size_t)blockIdx.x * width;
  for (int k = blockIdx.y * 256 + threadIdx.x; k < width; k += gridDim.y * 256) to[k] = k < K ? *gmem(row + k) : (uint16_t)0;
}

// ------------------------------------------------------------------------------------------------ products
struct I4Args {
  const char* w;
  I4Layout l;
  const uint16_t* x;
  long long x_stride;
  int N, T, K;
  int tiles_t;
  void* out;
  long long out_stride;
};

// The pairs of a word's eight codes as 16 + q in bf16: an and-or each, and a shift for all but the first.  The instruction takes one
// scalar operand, so one of the two constants is a register that the compiler does not see through (it would take two instructions).
struct I4Wide {
  uint32_t mask, base;
  __device__ __forceinline__ I4Wide() {
    asm("s_mov_b32 %0, 0x00780078" : "=s"(mask));
    asm("v_mov_b32 %0, 0x41804180" : "=v"(base));
  }
  __device__ __forceinline__ i4_b8 operator()(uint32_t w) const {
    const vu4 u = {(w & mask) | base, (w >> 4 & mask) | base, (w >> 8 & mask) | base, (__builtin_amdgcn_alignbit(w, w, 28) & mask) | base};
    return __builtin_bit_cast(i4_b8, u);
  }
};
__device__ __forceinline__ vf4 i4_mfma(i4_b8 a, i4_b8 b, vf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ uint32_t i4_bf16(float x) {  // nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// PAST: around the caches, which k_i4_tile's weights and hidden states need more (32 states at N = 248,320 150 -> 139 us; k_i4_few, whose
// stores are few, 106 -> 107)
template <bool PAST, typename O>
__device__ __forceinline__ void i4_put(O* p, float y) {
  O v;
  if constexpr (sizeof(O) == 4)
    v = y;
  else
    v = (O)i4_bf16(y);
  if constexpr (PAST)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

// A workgroup takes 64 weight rows and 16 TF hidden states, its NW waves a part of K each; their sums meet in LDS.
template <typename O, int GROUP, int TF, int NW>
__global__ void __launch_bounds__(64 * NW, TF > 2 ? 2 : 4) k_i4_few(I4Args a) {
  constexpr int G = I4_ROWS / 16, C = I4_KB / GROUP, J = GROUP / 32;  // fragments, groups of a block, products of a group
  __shared__ vf4 s_acc[NW][G * TF][64];
  const int lane = lane_id(), wave = wave_id(), quad = lane >> 4;
  // XCD x (workgroups x, x + 8, ..) takes the tiles of weight rows x, x + 8, .., all of their hidden states in a row
  const int tile = (blockIdx.x >> 3) / a.tiles_t * 8 + (blockIdx.x & 7), t0 = (blockIdx.x >> 3) % a.tiles_t * 16 * TF;
  if (tile >= a.l.tiles) return;
  const int kb = a.l.kb, per = (kb + NW - 1) / NW, lo = wave * per, hi = min(lo + per, kb);
  const char* pw = a.w + (size_t)tile * kb * (I4_ROWS * I4_KB / 2) + 16 * lane;
  const uint32_t* ps = (const uint32_t*)(a.w + a.l.scales) + (size_t)tile * a.l.kg * I4_ROWS + (lane & 15);
  const uint16_t* px[TF];
#pragma unroll
  for (int j = 0; j < TF; j++) px[j] = a.x + (long long)min(t0 + 16 * j + (lane & 15), a.T - 1) * a.x_stride + 8 * quad;
  const vu4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const i4_b8 ones = __builtin_bit_cast(i4_b8, one);
  vf4 acc[G][TF] = {};
  vu4 w[G];
  uint32_t sw[G][C];
  const I4Wide wide;
  auto load = [&](int k) {
#pragma unroll
    for (int g = 0; g < G; g++) w[g] = __builtin_nontemporal_load((const QWS_G vu4*)(pw + ((size_t)k * G + g) * 1024));
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int g = 0; g < G; g++) sw[g][c] = *gmem(ps + ((size_t)k * C + c) * I4_ROWS + 16 * g);
  };
  if (lo < hi) load(lo);
  for (int k = lo; k < hi; k++) {
    vu4 cw[G], x[TF][4];
    uint32_t cs[G][C];
#pragma unroll
    for (int j = 0; j < TF; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int at = k * I4_KB + 32 * i;
        if (at + 8 * quad < a.K)
          x[j][i] = *gmem((const vu4*)(px[j] + at));
        else
          x[j][i] = (vu4){0, 0, 0, 0};
      }
#pragma unroll
    for (int g = 0; g < G; g++) {
      cw[g] = w[g];
#pragma unroll
      for (int c = 0; c < C; c++) cs[g][c] = sw[g][c];
    }
    load(min(k + 1, hi - 1));
#pragma unroll
    for (int c = 0; c < C; c++) {
      vf4 sum[TF] = {};
#pragma unroll
      for (int i = 0; i < J; i++)
#pragma unroll
        for (int j = 0; j < TF; j++) sum[j] = i4_mfma(__builtin_bit_cast(i4_b8, x[j][c * J + i]), ones, sum[j]);
#pragma unroll
      for (int g = 0; g < G; g++) {
        vf4 d[TF] = {};
#pragma unroll
        for (int i = 0; i < J; i++) {
          const i4_b8 b = wide(cw[g][c * J + i]);
#pragma unroll
          for (int j = 0; j < TF; j++) d[j] = i4_mfma(__builtin_bit_cast(i4_b8, x[j][c * J + i]), b, d[j]);
        }
        const float z = (float)(cs[g][c] & 255u), s = __uint_as_float(cs[g][c] & 0xFFFFFF00u);
#pragma unroll
        for (int j = 0; j < TF; j++)
#pragma unroll
          for (int r = 0; r < 4; r++) acc[g][j][r] = fmaf(s, fmaf(-z, sum[j][r], d[j][r]), acc[g][j][r]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int j = 0; j < TF; j++) s_acc[wave][g * TF + j][lane] = acc[g][j];
  bar();
  const int n = tile * I4_ROWS + lane;  // a store is 64 consecutive rows of one hidden state
  for (int t = wave; t < 16 * TF && t0 + t < a.T; t += NW) {
    const int i = (lane >> 4) * TF + (t >> 4), l = (t >> 2 & 3) * 16 + (lane & 15), r = t & 3;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w += 4) y += (s_acc[w][i][l][r] + s_acc[w + 1][i][l][r]) + (s_acc[w + 2][i][l][r] + s_acc[w + 3][i][l][r]);
    if (n < a.N) i4_put<false>((O*)a.out + (long long)(t0 + t) * a.out_stride + n, y);
  }
}

// Hidden states as k_i4_tile takes them: for each 16 TF of them and each block of 128 values, an even number of blocks, 4 TF fragments
// of 1 KB (the first operand of product i of the states 16 j .. is fragment 4 j + i), then, in 1 KB, the groups' sums: word c * 16 TF
// + t.  Values beyond K and T are 0.  One wave per 16 states and block.
constexpr int i4_record(int tf) { return (4 * tf + 1) * 1024; }
template <int GROUP>
__global__ void __launch_bounds__(256) k_i4_states_tile(const uint16_t* x, long long stride, int T, int K, int kb_count, int tf, char* out) {
  constexpr int J = GROUP / 32;
  const int lane = lane_id(), quad = lane >> 4, kb = blockIdx.y * 4 + wave_id(), frag = blockIdx.x;  // 16 states
  if (kb >= kb_count) return;
  const int t = frag * 16 + (lane & 15);
  const uint16_t* row = x + (long long)min(t, T - 1) * stride;
  char* rec = out + ((size_t)(frag / tf) * kb_count + kb) * i4_record(tf);
  const int j = frag % tf;
#pragma unroll
  for (int c = 0; c < 4 / J; c++) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < J; i++) {
      const int k0 = kb * I4_KB + 32 * (c * J + i) + 8 * quad;
      uint32_t v[8];
      i4_load(row, k0, K, v);
      if (t >= T) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) sum += __uint_as_float(v[e] << 16);
      ((vu4*)(rec + (4 * j + c * J + i) * 1024))[lane] = (vu4){v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (quad == 0) ((float*)(rec + 4 * tf * 1024))[c * 16 * tf + 16 * j + lane] = sum;
  }
}

// More hidden states: a workgroup takes 256 weight rows and 16 TF hidden states, a wave 64 of the rows over all of K.  Hidden states and
// their sums are copied into LDS by the memory system two blocks ahead (three buffers), the weights go straight into registers, two
// blocks ahead as well: one block ahead left too few bytes in flight (36 states at K = 5,120, N = 248,320 172 us, 163 so; 155 with the later steps).  What bounds it:
// up to 48 states mostly the bytes (36 states 155 us: 4.6 TB/s of weights and logits); from there on the products and the vector
// instructions beside them, which take turns on this card: a 16x16x32 product and four others take 25 cycles of a SIMD, alone 17 and 11.
// So the instructions are what counts: seven for eight codes (eight, 64 states 191 us, 188 so), two for each scaled sum.
template <typename O, int GROUP, int TF>
__global__ void __launch_bounds__(256, 2) k_i4_tile(I4Args a) {
  constexpr int G = I4_ROWS / 16, C = I4_KB / GROUP, J = GROUP / 32, REC = i4_record(TF);
  __shared__ __attribute__((aligned(16))) char s_x[3 * REC];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), quad = lane >> 4;
  const int tiles = (a.l.tiles + 3) / 4;
  const int big = (blockIdx.x >> 3) / a.tiles_t * 8 + (blockIdx.x & 7), tt = (blockIdx.x >> 3) % a.tiles_t, t0 = tt * 16 * TF;
  if (big >= tiles) return;
  const int tile = min(big * 4 + wave, a.l.tiles - 1), kb = a.l.kb, kx = i4_up(kb, 2);  // a wave past the last rows computes them again and stores nothing
  const char* pw = a.w + (size_t)tile * kb * (I4_ROWS * I4_KB / 2) + 16 * lane;
  const uint32_t* ps = (const uint32_t*)(a.w + a.l.scales) + (size_t)tile * a.l.kg * I4_ROWS + (lane & 15);
  const char* px = (const char*)a.x + (size_t)tt * kx * REC;
  struct W {
    vu4 w[G];
    uint32_t s[G][C];
  } even, odd;
  vf4 acc[G][TF] = {}, d[2][TF], sum[TF];
  const I4Wide wide;
  auto load_w = [&](W& v, int k, int g) { v.w[g] = *gmem((const vu4*)(pw + ((size_t)min(k, kb - 1) * G + g) * 1024)); };
  auto load_s = [&](W& v, int k, int g) {
#pragma unroll
    for (int c = 0; c < C; c++) v.s[g][c] = *gmem(ps + ((size_t)min(k, kb - 1) * C + c) * I4_ROWS + 16 * g);
  };
  auto copy_x = [&](int k, char* to) {  // a quarter of the record, and of its sums
    const char* rec = px + (size_t)min(k, kx - 1) * REC;
    const char* mine = rec + wave * (TF * 1024);
    lds_copy<0>(mine, 16 * lane, to + wave * (TF * 1024));
    if constexpr (TF > 1) lds_copy<1024>(mine, 16 * lane, to + wave * (TF * 1024));
    if constexpr (TF > 2) lds_copy<2 * 1024>(mine, 16 * lane, to + wave * (TF * 1024));
    if constexpr (TF > 3) lds_copy<3 * 1024>(mine, 16 * lane, to + wave * (TF * 1024));
    lds_copy_words(rec + TF * 4096 + wave * 256, 4 * lane, to + TF * 4096 + wave * 256);
  };
  // what is left of fragment g's group c when its products are done
  auto finish = [&](const W& v, int g, int c, int j) {
    const float z = (float)(v.s[g][c] & 255u), s = __uint_as_float(v.s[g][c] & 0xFFFFFF00u);
#pragma unroll
    for (int r = 0; r < 4; r++) acc[g][j][r] = fmaf(s, fmaf(-z, sum[j][r], d[g & 1][j][r]), acc[g][j][r]);
  };
  i4_b8 x[TF][J];
  auto read_x = [&](const char* from, int c, int i) {
#pragma unroll
    for (int j = 0; j < TF; j++) x[j][i] = __builtin_bit_cast(i4_b8, ((const vu4*)(from + (4 * j + c * J + i) * 1024))[lane]);
  };
  auto read_sum = [&](const char* from, int c) {
#pragma unroll
    for (int j = 0; j < TF; j++) sum[j] = *(const vf4*)((const float*)(from + TF * 4096) + c * 16 * TF + 16 * j + 4 * quad);
  };
  char *x0 = s_x, *x1 = s_x + REC, *x2 = s_x + 2 * REC;  // of blocks k, k + 1 and k + 2
  copy_x(0, x0);
  copy_x(1, x1);
#pragma unroll
  for (int g = 0; g < G; g++) {
    load_w(even, 0, g);
    load_s(even, 0, g);
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    load_w(odd, 1, g);
    load_s(odd, 1, g);
  }
  lds_meet<2 * G * (1 + C)>();
#pragma unroll
  for (int i = 0; i < J; i++) read_x(x0, 0, i);
  read_sum(x0, 0);
  i4_b8 b = wide(even.w[0][0]);
  // Block k, whose first hidden states are in registers.  The states of block k + 2 are copied into LDS meanwhile, and its weights
  // replace this block's.
  auto block = [&](int k, W& now, const W& then) __attribute__((always_inline)) {
    copy_x(k + 2, x2);
#pragma unroll
    for (int c = 0; c < C; c++) {
      const char* from = c + 1 < C ? x0 : x1;  // where the next group's states lie
      // A step is one product of a fragment for all the hidden states: beside it the next product's weights are widened, the last
      // fragment's sums scaled and, after the group's last use of them, hidden states replaced: about as many other instructions
      // as fit into the products' time.
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < J; i++) {
          const bool last = i == J - 1, end = last && g == G - 1;
          const i4_b8 next = wide(!last ? now.w[g][c * J + i + 1] : !end ? now.w[g + 1 < G ? g + 1 : 0][c * J] : c + 1 < C ? now.w[0][(c + 1) % C * J] : then.w[0][0]);
#pragma unroll
          for (int j = 0; j < TF; j++) {
            const vf4 none = {0.0f, 0.0f, 0.0f, 0.0f};
            d[g & 1][j] = i4_mfma(x[j][i], b, i ? d[g & 1][j] : none);
          }
          if (g == G - 1) read_x(from, (c + 1) % C, i);
          if (g > 0) {
#pragma unroll
            for (int j = 0; j < TF; j++)
              if (j * J / TF == i) finish(now, g - 1, c, j);
          }
          b = next;
          if (last && c == C - 1) {
            load_w(now, k + 2, g);
            if (g > 0) load_s(now, k + 2, g - 1);
          }
#pragma unroll
          for (int j = 0; j < TF; j++) {  // a product, then the instructions of its time
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (8 + 8 * TF / J + TF - 1) / TF, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int j = 0; j < TF; j++) finish(now, G - 1, c, j);
      read_sum(from, (c + 1) % C);
    }
    load_s(now, k + 2, G - 1);
    lds_meet<G * (1 + C)>();  // all but this block's loads of weights
    char* t = x0;
    x0 = x1;
    x1 = x2;
    x2 = t;
  };
  for (int k = 0; k < kx; k += 2) {
    block(k, even, odd);
    block(k + 1, odd, even);
  }
  if (big * 4 + wave >= a.l.tiles) return;
  // A lane holds four hidden states of 16 weight rows each; a transposition of the four fragments against the four quarters of the
  // wave gives each lane one of 64 consecutive rows, so that a store is 256 bytes in a row.
  const int n = tile * I4_ROWS + lane;
#pragma unroll
  for (int j = 0; j < TF; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      uint32_t v[4];
#pragma unroll
      for (int g = 0; g < G; g++) v[g] = __float_as_uint(acc[g][j][r]);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const auto q = __builtin_amdgcn_permlane32_swap(v[h], v[h + 2], false, false);
        v[h] = q[0];
        v[h + 2] = q[1];
      }
#pragma unroll
      for (int h = 0; h < 4; h += 2) {
        const auto q = __builtin_amdgcn_permlane16_swap(v[h], v[h + 1], false, false);
        v[h] = q[0];
        v[h + 1] = q[1];
      }
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int t = t0 + 16 * j + 4 * q + r;
        if (t < a.T && n < a.N) i4_put<true>((O*)a.out + (long long)t * a.out_stride + n, __uint_as_float(v[q]));
      }
    }
}

inline bool i4_group(int group) { return group == 32 || group == 64 || group == 128; }
inline bool i4_shape(int T, int N, int K, int group) { return T >= 1 && N >= 1 && K >= 1 && i4_group(group); }
inline bool i4_fits(int T, int N, int K) { return N <= I4_NMAX && K <= I4_KMAX && T <= I4_TMAX; }
inline bool i4_aligned(const void* p) { return p && ((uintptr_t)p & 255) == 0; }
// Up to so many workgroups of k_i4_few each has eight waves, an eighth of K each, instead of four (K = 5,120, us, four / eight: N = 8,191, 1
// state 14.6 / 9.4; N = 16,384 15.4 / 10.9; N = 24,000 17.0 / 15.5; N = 64,000 30.6 / 30.1; 30 states at N = 16,384, 512 workgroups, 18.4 / 19.7).
constexpr int I4_SPARSE = 384;
// What runs T hidden states against N weight rows: k_i4_tile or k_i4_few, with 16 tf of them to a workgroup: the least estimated time.  A
// kernel's workgroups take `least` us for 40 blocks of K where each CU has one, and `each` for every one of them where it has several,
// between the mean and the largest number of them
// (k_i4_few's for 16 states: with eight waves); k_i4_tile's states are packed by a launch of 3 us.  Measured, us, k_i4_few / k_i4_tile:
// K = 5,120, N = 248,320: 1 state 107 / 118, 8 states 125 / 126, 12 139 / 129, 16 153 / 132, 36 272 / 163, 64 346 / 197, 200 1,260 / 620; N =
// 64,000: 8 states 33 / 34, 16 40 / 35, 64 95 / 59; N = 32,001: 12 states 19 / 30, 40 44 / 38, 64 51 / 39; N = 16,384: 64 states 30 / 36.
struct I4Plan {
  bool tile;
  int tf;
};
inline I4Plan i4_plan(int T, int N, int K) {
  if (T <= 8) return {false, 1};
  struct Cost {
    double least, each;
  };
  constexpr Cost few[3] = {{11, 10}, {22, 12.5}, {28, 24}}, tile[4] = {{26, 31}, {32, 33}, {37, 37}, {43, 47}};
  const double blocks = i4_up(K, I4_KB) / I4_KB / 40.0;
  auto time = [&](Cost c, int rows, int states) {
    const double wgs = (double)(i4_up(N, rows) / rows) * (i4_up(T, states) / states) / 256, each = c.each * (wgs + ceil(wgs)) / 2;
    return blocks * (each > c.least ? each : c.least);
  };
  I4Plan p = {false, 1};
  double best = time(few[0], I4_ROWS, 16);
  for (int tf = 2; tf <= 4; tf += tf) {
    const double t = time(few[tf / 2], I4_ROWS, 16 * tf);
    if (t < best) {
      best = t;
      p.tf = tf;
    }
  }
  for (int tf = 1; tf <= 4; tf++) {
    const double t = 3 + time(tile[tf - 1], 4 * I4_ROWS, 16 * tf);
    if (t < best) {
      best = t;
      p = {true, tf};
    }
  }
  return p;
}
inline size_t i4_ws(int T, int N, int K) {
  const I4Plan p = i4_plan(T, N, K);
  const int kb = i4_up(K, I4_KB) / I4_KB;
  return p.tile ? (size_t)(i4_up(T, 16 * p.tf) / (16 * p.tf)) * i4_up(kb, 2) * i4_record(p.tf) : ((size_t)T * kb * I4_KB * 2 + 255) & ~(size_t)255;
}
// whether a lane can read hidden states 16 bytes at a time as they came
inline bool i4_direct(const void* x, long long stride, int T, int K) { return K % 8 == 0 && ((uintptr_t)x & 15) == 0 && (T == 1 || stride % 8 == 0); }

template <typename T>
static int i4_pack(const I4Pack& a, int group, hipStream_t st) {
  const dim3 grid(a.l.tiles * (I4_ROWS / 16), (a.l.kb + 3) / 4);
  switch (group) {
    case 32: hipLaunchKernelGGL((k_i4_pack<T, 32>), grid, dim3(256), 0, st, a); break;
    case 64: hipLaunchKernelGGL((k_i4_pack<T, 64>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((k_i4_pack<T, 128>), grid, dim3(256), 0, st, a); break;
  }
  return (int)hipGetLastError();
}

template <typename O, int GROUP>
static int i4_run(I4Args a, char* ws, hipStream_t st) {
  const I4Plan p = i4_plan(a.T, a.N, a.K);
  const int tf = p.tf;
  a.tiles_t = i4_up(a.T, 16 * tf) / (16 * tf);
  const long long wgs = (long long)i4_up(p.tile ? (a.l.tiles + 3) / 4 : a.l.tiles, 8) * a.tiles_t;
  if (wgs > 0xFFFFFF) return QWS_ERR_NOT_SUPPORTED;  // below 2^32 threads
  const dim3 grid((unsigned)wgs), nt(256);
  if (p.tile) {
    hipLaunchKernelGGL((k_i4_states_tile<GROUP>), dim3(a.tiles_t * tf, (a.l.kb + 4) / 4), nt, 0, st, a.x, a.x_stride, a.T, a.K, i4_up(a.l.kb, 2), tf, ws);
    a.x = (const uint16_t*)ws;
    switch (tf) {
      case 1: hipLaunchKernelGGL((k_i4_tile<O, GROUP, 1>), grid, nt, 0, st, a); break;
      case 2: hipLaunchKernelGGL((k_i4_tile<O, GROUP, 2>), grid, nt, 0, st, a); break;
      case 3: hipLaunchKernelGGL((k_i4_tile<O, GROUP, 3>), grid, nt, 0, st, a); break;
      default: hipLaunchKernelGGL((k_i4_tile<O, GROUP, 4>), grid, nt, 0, st, a); break;
    }
    return (int)hipGetLastError();
  }
  if (!i4_direct(a.x, a.x_stride, a.T, a.K)) {
    const int width = a.l.kb * I4_KB;
    hipLaunchKernelGGL(k_i4_states, dim3(a.T, (width + 1023) / 1024), nt, 0, st, a.x, a.x_stride, a.K, width, (uint16_t*)ws);
    a.x = (const uint16_t*)ws;
    a.x_stride = width;
    a.K = width;
  }
  switch (tf) {
    case 1:
      if (wgs <= I4_SPARSE)
        hipLaunchKernelGGL((k_i4_few<O, GROUP, 1, 8>), grid, dim3(512), 0, st, a);
      else
        hipLaunchKernelGGL((k_i4_few<O, GROUP, 1, 4>), grid, nt, 0, st, a);
      break;
    case 2: hipLaunchKernelGGL((k_i4_few<O, GROUP, 2, 4>), grid, nt, 0, st, a); break;
    default: hipLaunchKernelGGL((k_i4_few<O, GROUP, 4, 4>), grid, nt, 0, st, a); break;
  }
  return (int)hipGetLastError();
}
template <typename O>
static int i4_product(const I4Args& a, int group, char* ws, hipStream_t st) {
  return group == 32 ? i4_run<O, 32>(a, ws, st) : group == 64 ? i4_run<O, 64>(a, ws, st) : i4_run<O, 128>(a, ws, st);
}

}  // namespace qws

extern "C" size_t qws_int4_pack_bytes(int N, int K, int group) {
  return qws::i4_shape(1, N, K, group) && qws::i4_fits(1, N, K) ? qws::i4_layout(N, K, group).total : 0;
}

extern "C" int qws_int4_pack(const void* w, int dtype, int N, int K, long long row_stride, int group, void* packed, void* stream) {
  using namespace qws;
  if (!i4_shape(1, N, K, group) || (dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) || !w || row_stride < 0 || !i4_aligned(packed)) return QWS_ERR_INVALID;
  if ((uintptr_t)w & (dtype == QWS_DTYPE_F32 ? 3 : 1)) return QWS_ERR_INVALID;
  if (!i4_fits(1, N, K)) return QWS_ERR_NOT_SUPPORTED;
  I4Pack a = {};
  a.w = w;
  a.stride = row_stride;
  a.N = N;
  a.K = K;
  a.l = i4_layout(N, K, group);
  a.out = (char*)packed;
  return dtype == QWS_DTYPE_F32 ? i4_pack<float>(a, group, (hipStream_t)stream) : i4_pack<uint16_t>(a, group, (hipStream_t)stream);
}

extern "C" int qws_int4_pack_codes(const unsigned char* codes, long long code_stride, const void* scales, int scales_fp16, long long scale_stride,
                                   const unsigned char* zeros, long long zero_stride, int N, int K, int group, void* packed, void* stream) {
  using namespace qws;
  if (!i4_shape(1, N, K, group) || !codes || !scales || ((uintptr_t)scales & 1) || code_stride < 0 || scale_stride < 0 || zero_stride < 0 || !i4_aligned(packed))
    return QWS_ERR_INVALID;
  if (!i4_fits(1, N, K)) return QWS_ERR_NOT_SUPPORTED;
  I4Pack a = {};
  a.w = codes;
  a.stride = code_stride;
  a.scales = (const uint16_t*)scales;
  a.scale_stride = scale_stride;
  a.half = scales_fp16 != 0;
  a.zeros = zeros;
  a.zero_stride = zero_stride;
  a.N = N;
  a.K = K;
  a.l = i4_layout(N, K, group);
  a.out = (char*)packed;
  return i4_pack<uint8_t>(a, group, (hipStream_t)stream);
}

extern "C" size_t qws_int4_head_ws_bytes(int T, int N, int K, int group) {
  return qws::i4_shape(T, N, K, group) && qws::i4_fits(T, N, K) ? qws::i4_ws(T, N, K) : 0;
}

extern "C" int qws_int4_head(const void* packed, int N, int K, int group, const void* x, long long x_stride, int T, void* out, int out_dtype,
                             long long out_stride, void* ws, size_t ws_bytes, void* stream) {
  using namespace qws;
  if (!i4_shape(1, N, K, group) || T < 0 || x_stride < 0 || !i4_aligned(packed) || (out_dtype != QWS_DTYPE_F32 && out_dtype != QWS_DTYPE_BF16)) return QWS_ERR_INVALID;
  if (!i4_fits(T, N, K)) return QWS_ERR_NOT_SUPPORTED;
  if (T == 0) return QWS_OK;
  if (!x || ((uintptr_t)x & 1) || !out || ((uintptr_t)out & (out_dtype == QWS_DTYPE_F32 ? 3 : 1)) || (T > 1 && out_stride < N)) return QWS_ERR_INVALID;
  if (!i4_aligned(ws) || ws_bytes < i4_ws(T, N, K)) return QWS_ERR_INVALID;
  I4Args a = {};
  a.w = (const char*)packed;
  a.l = i4_layout(N, K, group);
  a.x = (const uint16_t*)x;
  a.x_stride = x_stride;
  a.N = N;
  a.T = T;
  a.K = K;
  a.out = out;
  a.out_stride = out_stride;
  hipStream_t st = (hipStream_t)stream;
  return out_dtype == QWS_DTYPE_F32 ? i4_product<float>(a, group, (char*)ws, st) : i4_product<uint16_t>(a, group, (char*)ws, st);
}
