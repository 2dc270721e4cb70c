// qws losses over given tokens with their gradient at the logits: the clipped policy loss with a KL term and the preference loss of
// paired log ratios (the definitions: include/qws.h qws_policy_loss, qws_preference_loss; the running sums: qws_lse.h).
//
// Both depend on the logits through log p of each row's token, so their gradient is
//   dL/dx_j = (dL/dlog p) ([j = token] - p_j) / T,
// one number a row beside what the softmax needs.  A row's maximum m and sum s come from one pass over its logits, the loss and
// dL/dlog p from a few numbers a row (in 64 bits: they are differences of log probabilities), the gradient from a second pass.
//
// The policy loss's slope depends on its row alone, so one workgroup does a row from the first pass to the second and keeps what
// fits of it in between (k_ls_policy): the logits are read once, the gradient written once.  The preference loss's depends on every
// row of a pair, so between its passes lies a launch and, past the caches, the logits are read twice.
//
//   k_ls_policy      a workgroup per row: the policy loss with its gradient.  Bound by the bytes: 2,048 bf16 rows of 248,320 391 us, 5.2
//                    TB/s of 2.03 GB, which is what was read and written (a large copy makes 4.97); 512 fp32 rows 210 us, 1.26 GB with
//                    what a row's workgroup cannot keep, read twice; a few short rows by one row's latency, 13 us for 32,001 logits.
//   k_ls_scan        R x G workgroups: each lane's running maximum and sum.  Bound by the bytes of the rows with a token: 240 of 256
//                    fp32 rows 44 us, 5.4 TB/s; 1,125 of 1,200 bf16 rows 99 us, 5.6 TB/s.
//   k_ls_policy_rows a wave per row: joins the row's parts, log p, the row's term and slope (5.4 us up to 512 rows: latency)
//   k_ls_rows        the same for the preference loss: log p and the row's sequence (5-6 us)
//   k_ls_pairs       a wave per pair: the sequences' sums, the pair's term, the two slopes
//   k_ls_sum         the loss: the sum of the terms (4-5 us); k_ls_few, k_ls_policy_few: pairs and a few rows in the same launch (5-10 us)
//   k_ls_grad        R x G workgroups: the gradient's rows.  Bound by the bytes: 1,200 bf16 rows 193 us, 6.0 TB/s; where it finds the
//                    gradient written 4.5 us.
#include "qws_logits.h"

namespace qws {

constexpr int LS_NT = 256;
constexpr int LS_NW = LS_NT / 64;
constexpr int LS_U = 4;          // vectors of a thread loaded together
constexpr int LS_VMAX = 1 << 24, LS_RMAX = 1 << 24;
constexpr int LS_ONE = 1024;     // threads of the kernels that run as one workgroup
constexpr double LS_FAR = 80.0;  // log ratios above count as this: e^80 stays in fp32

// what the gradient needs of a row
struct LsRow {
  float c, m, M, inv;  // 2^(c x - M) inv = p (mode 1), 2^(c (x - m)) inv = p (mode 2)
  float per_t;         // 1 / T
  int tok, slot;       // slot: which slope
  int mode;            // 0: no gradient
};
struct LsHead {
  float scale;  // of every slope
};

struct LsArgs {
  const void* x;
  long long stride, block_stride;
  int block;  // rows at one stride
  const int* tok;
  const float* temp;
  int R, V;
  int G, per;  // workgroups of a row, stripes of each
  // the state
  LsHead* head;
  LsRow* rows;
  float* slope;   // policy: [R]; preference: [2 P]
  double* lp;     // [R]
  double* term;   // policy: [R]; preference: [P]
  float2* part;   // [R][G] maximum, sum
  // policy
  const float *old_lp, *adv, *ref, *weights;
  float clip_low, clip_high, kl;
  float *out_loss, *out_lp, *out_ratio, *out_kl;
  // preference
  const int* starts;
  int P;
  float beta, margin, smoothing;
  int average;
  float *out_sums, *out_margins;
  // gradient
  void* grad;
  long long grad_stride;
  const float* upstream;  // the gradient's factor, or null: grad_scale
  float grad_scale;
};

template <typename T>
__device__ __forceinline__ const T* ls_row(const LsArgs& a, int r) {
  const int b = r / a.block;
  return (const T*)a.x + (long long)b * a.block_stride + (long long)(r - b * a.block) * a.stride;
}
__device__ __forceinline__ int ls_token(const LsArgs& a, int r) {  // -1: none
  const int t = a.tok[r];
  return t >= 0 && t < a.V ? t : -1;
}

// ------------------------------------------------------------------------------------------------ a row's maximum and sum
struct LsSum {
  float m, s;
};
__device__ __forceinline__ LsSum ls_join(LsSum a, LsSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, fmaf(lse_exp2(lse_d(a.m, m, c)), a.s, lse_exp2(lse_d(b.m, m, c)) * b.s)};
}
__device__ __forceinline__ LsSum ls_join_wave(LsSum v, float c) {
  const float m = wave_max_f(v.m);
  return {m, wave_sum<float>(lse_exp2(lse_d(v.m, m, c)) * v.s)};
}

// A lane's sum over moderate logits relative to a reference M = fl(c m) that lies within LS_SLACK of the largest, so that it rarely
// moves: a multiply-add, an exponential and an addition per logit.  -inf adds 0; blocks with NaN, +inf or a new maximum of
// extreme size go to the general form.
constexpr float LS_SLACK = 8.0f;  // in log2 units
struct LsFast {
  float m, M, limit, s;
};
template <int U, int E>
__device__ __forceinline__ bool ls_fast(LsFast& f, const float (&x)[U][E], float best, float c) {
  if (__any(best > f.limit)) {
    if (__any(best > f.limit && !(fabsf(c * best) < LSE_NEAR))) return false;
    if (best > f.limit) {
      const float M = c * best;
      f = {best, M, best + LS_SLACK / c, f.s * lse_exp2(f.M - M)};
    }
  }
  float s = f.s;
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < E; j++) s += lse_exp2(fmaf(x[u][j], c, -f.M));
  if (__any(!(s < INFINITY))) return false;
  f.s = s;
  return true;
}
template <int U, int E>
__device__ __forceinline__ void ls_slow(LsSum& v, const float (&x)[U][E], float best, float c) {
  const float m = fmaxf(v.m, best);
  v = {m, v.s * lse_exp2(lse_d(v.m, m, c))};
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < E; j++) v.s += lse_exp2(lse_d(lse_clean(x[u][j]), m, c));
}

template <typename T>
constexpr int ls_stripe(int nt = LS_NT) { return nt * lp_e<T>(); }

// The maximum and sum of stripes s_begin .. s_end of a row by NT threads; lane's own
template <typename T, int U, int NT>
__device__ __forceinline__ LsSum ls_scan_part(const T* p, int V, int s_begin, int s_end, float c) {
  constexpr int E = lp_e<T>(), SE = ls_stripe<T>(NT);
  const int tid = threadIdx.x, lead = (int)((uintptr_t)p / sizeof(T)) & (E - 1), end = lead + V;
  const T* base = p - lead;
  s_end = min(s_end, (end + SE - 1) / SE);
  vu4 r[U];
  auto load = [&](int s) {
    const int first = s * SE;
    if (first >= lead && first + U * SE <= end && s + U <= s_end) {
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = *gmem((const vu4*)(base + first + u * SE + tid * E));
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = lp_load_edge(base, first + u * SE + tid * E, s + u < s_end ? lead : end, end);
    }
  };
  if (s_begin < s_end) load(s_begin);
  LsSum v = {-INFINITY, 0.0f};
  LsFast f = {-INFINITY, -1e30f, -INFINITY, 0.0f};
  for (int s = s_begin; s < s_end; s += U) {
    float x[U][E], best = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
      lp_unpack<T>(r[u], x[u]);
      best = fmaxf(best, lp_max<E>(x[u]));
    }
    if (!ls_fast(f, x, best, c)) ls_slow(v, x, fminf(best, F32_MAX), c);
    if (s + U < s_end) load(s + U);
  }
  if (f.m != -INFINITY) {
    const Lse q = lse_exact(f.m, f.M, f.s, 0.0f, c);
    v = ls_join(v, {q.m, q.s}, c);
  }
  return v;
}
// joined over the workgroup, in thread 0
template <int NT>
__device__ __forceinline__ LsSum ls_join_group(LsSum v, float c, LsSum* s_sum) {
  v = ls_join_wave(v, c);
  if (lane_id() == 0) s_sum[wave_id()] = v;
  bar();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < NT / 64; w++) v = ls_join(v, s_sum[w], c);
  }
  return v;
}

template <typename T, int U>
__global__ void __launch_bounds__(LS_NT, 5) k_ls_scan(LsArgs a) {
  __shared__ LsSum s_sum[LS_NW];
  const int row = blockIdx.x / a.G, ch = blockIdx.x % a.G;
  if (ls_token(a, row) < 0) return;  // no one reads its parts
  const float c = lse_scale(a.temp ? a.temp[row] : 1.0f);
  LsSum v = ls_scan_part<T, U, LS_NT>(ls_row<T>(a, row), a.V, ch * a.per, ch * a.per + a.per, c);
  v = ls_join_group<LS_NT>(v, c, s_sum);
  if (threadIdx.x == 0) a.part[(size_t)row * a.G + ch] = make_float2(v.m, v.s);
}

// A row's parts joined by a wave
__device__ __forceinline__ LsSum ls_parts(const LsArgs& a, int row, float c) {
  LsSum v = {-INFINITY, 0.0f};
  for (int i = lane_id(); i < a.G; i += 64) {
    const float2 q = a.part[(size_t)row * a.G + i];
    v = ls_join(v, {q.x, q.y}, c);
  }
  return ls_join_wave(v, c);
}

// Log p of a row's token from the row's maximum and sum, in 64 bits (-inf: masked), and what the gradient needs
template <typename T>
__device__ __forceinline__ double ls_finish(const LsArgs& a, int row, int tok, int slot, LsSum v, float c, float temp) {
  const float x = lp_one(ls_row<T>(a, row) + tok);
  LsRow q = {c, v.m, c * v.m, 0.0f, 1.0f / lse_temp(temp), tok, slot, 0};
  if (x == -INFINITY) {
    a.rows[row] = q;
    return -INFINITY;
  }
  if (fabsf(q.M) < LSE_NEAR && fabsf(v.m) < LSE_MOST && c <= LSE_MOST) {
    q.mode = 1;
    q.inv = lse_exp2(-fmaf(c, v.m, -q.M)) / v.s;
  } else {
    q.mode = 2;
    q.inv = 1.0f / v.s;
  }
  a.rows[row] = q;
  const double p = ((double)x - (double)v.m) / (double)lse_temp(temp) - log((double)v.s);
  return p > 0.0 ? 0.0 : p;
}

// ------------------------------------------------------------------------------------------------ the policy loss's rows
// One lane: the term and the slope of a row, its three results.
template <typename T>
__device__ __forceinline__ double ls_policy(const LsArgs& a, int row, int tok, LsSum v, float c, float temp) {
  double lp = 0.0, term = 0.0, ratio = 1.0, kl = 0.0, slope = 0.0;
  if (tok >= 0) {
    lp = ls_finish<T>(a, row, tok, row, v, c, temp);
    if (lp > -INFINITY) {
      const double adv = a.adv[row], w = a.weights ? a.weights[row] : 1.0;
      double d = lp - a.old_lp[row];
      ratio = exp(d > LS_FAR ? LS_FAR : d);
      const double low = 1.0 - a.clip_low, high = 1.0 + a.clip_high;
      const double straight = ratio * adv, clipped = (ratio < low ? low : ratio > high ? high : ratio) * adv;
      term = straight <= clipped ? -straight : -clipped;
      if (!(straight > clipped)) slope = -straight;  // NaN stays
      if (a.ref) {
        d = a.ref[row] - lp;
        d = d > LS_FAR ? LS_FAR : d;
        const double e = expm1(d);
        kl = e - d;
        term += a.kl * kl;
        slope -= a.kl * e;
      }
      term *= w;
      slope *= w;
    }
  } else {
    a.rows[row] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, -1, row, 0};
  }
  a.slope[row] = (float)slope;
  if (a.out_lp) a.out_lp[row] = (float)lp;
  if (a.out_ratio) a.out_ratio[row] = (float)ratio;
  if (a.out_kl) a.out_kl[row] = (float)kl;
  return term;
}
// One wave: a row's parts joined, its term (lane 0's); k counts the rows with a token
template <typename T>
__device__ __forceinline__ double ls_policy_row(const LsArgs& a, int row, int& k) {
  const int tok = ls_token(a, row);
  const float temp = a.temp ? a.temp[row] : 1.0f, c = lse_scale(temp);
  const LsSum v = tok < 0 ? LsSum{-INFINITY, 0.0f} : ls_parts(a, row, c);
  k += tok >= 0;
  return lane_id() == 0 ? ls_policy<T>(a, row, tok, v, c, temp) : 0.0;
}
template <typename T>
__global__ void __launch_bounds__(LS_NT) k_ls_policy_rows(LsArgs a) {
  const int row = blockIdx.x * LS_NW + wave_id();
  if (row >= a.R) return;
  int k = 0;
  const double term = ls_policy_row<T>(a, row, k);
  if (lane_id() == 0) a.term[row] = term;
}

// ------------------------------------------------------------------------------------------------ the preference loss's rows and pairs
__device__ __forceinline__ int ls_start(const LsArgs& a, int i) { return min(max(a.starts[i], 0), a.R); }
// the last i in [0, 2 P] with starts[i] <= row, or -1
__device__ __forceinline__ int ls_sequence(const LsArgs& a, int row) {
  int lo = -1, hi = a.P ? 2 * a.P + 1 : 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (a.starts[mid] <= row ? lo : hi) = mid;
  }
  return lo;
}
// one wave
template <typename T>
__device__ __forceinline__ void ls_preference_row(const LsArgs& a, int row) {
  const int tok = ls_token(a, row), seq = ls_sequence(a, row);
  const float temp = a.temp ? a.temp[row] : 1.0f, c = lse_scale(temp);
  const LsSum v = tok < 0 ? LsSum{-INFINITY, 0.0f} : ls_parts(a, row, c);
  if (lane_id()) return;
  double lp = NAN;  // no token
  if (tok >= 0)
    lp = ls_finish<T>(a, row, tok, seq, v, c, temp);
  if (tok < 0 || seq < 0 || seq >= 2 * a.P) a.rows[row] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, -1, 0, 0};
  a.lp[row] = lp;
  if (a.out_lp) a.out_lp[row] = tok >= 0 ? (float)lp : 0.0f;
}
template <typename T>
__global__ void __launch_bounds__(LS_NT) k_ls_rows(LsArgs a) {
  const int row = blockIdx.x * LS_NW + wave_id();
  if (row < a.R) ls_preference_row<T>(a, row);
}

// One wave: pair i's term; the slopes and results of its sequences
__device__ __forceinline__ double ls_pair(const LsArgs& a, int i) {
  double sum[2];
  int count[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int from = ls_start(a, 2 * i + h), to = ls_start(a, 2 * i + h + 1);
    double s = 0.0;
    int n = 0;
    constexpr int U = 8;  // loaded together
    for (int r = from + lane_id(); r < to; r += 64 * U) {
      double p[U];
#pragma unroll
      for (int u = 0; u < U; u++) p[u] = a.lp[min(r + 64 * u, a.R - 1)];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (r + 64 * u < to) {
          if (p[u] > -INFINITY) s += p[u];
          if (p[u] == p[u]) n++;
        }
    }
    sum[h] = wave_sum<double>(s);
    count[h] = a.average ? max(wave_sum<int>(n), 1) : 1;
    sum[h] /= count[h];
  }
  double d = sum[0] - sum[1];
  if (a.ref) d = (sum[0] - a.ref[2 * i]) - (sum[1] - a.ref[2 * i + 1]);
  const double u = a.beta * d - a.margin, w = a.weights ? a.weights[i] : 1.0, eps = a.smoothing;
  const double e = exp(-fabs(u)), sig = u >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);  // sigmoid(-u); NaN stays
  const double term = w * ((u < 0.0 ? -u : u == u ? 0.0 : u) + log1p(e) + (eps != 0.0 ? eps * u : 0.0)), slope = a.beta * w * (eps - sig);
  if (lane_id() == 0) {
    a.slope[2 * i] = (float)(slope / count[0]);
    a.slope[2 * i + 1] = (float)(-slope / count[1]);
    if (a.out_sums) {
      a.out_sums[2 * i] = (float)sum[0];
      a.out_sums[2 * i + 1] = (float)sum[1];
    }
    if (a.out_margins) a.out_margins[i] = (float)u;
  }
  return term;
}
__global__ void __launch_bounds__(LS_NT) k_ls_pairs(LsArgs a) {
  const int i = blockIdx.x * LS_NW + wave_id();
  if (i >= a.P) return;
  const double term = ls_pair(a, i);
  if (lane_id() == 0) a.term[i] = term;
}

// The loss from the threads' sums of terms and counts, in a fixed order.  Without weights it is their mean: over the rows with a
// token, or the pairs.
__device__ __forceinline__ void ls_total(const LsArgs& a, double s, int k, int pairs) {
  __shared__ double s_sum[LS_ONE / 64];
  __shared__ int s_count[LS_ONE / 64];
  s = wave_sum<double>(s);
  k = wave_sum<int>(k);
  if (lane_id() == 0) {
    s_sum[wave_id()] = s;
    s_count[wave_id()] = k;
  }
  bar();
  if (threadIdx.x) return;
  for (int w = 1; w < LS_ONE / 64; w++) {
    s += s_sum[w];
    k += s_count[w];
  }
  if (pairs) k = pairs;
  const double scale = a.weights || k == 0 ? 1.0 : 1.0 / k;
  a.head->scale = (float)scale;
  *a.out_loss = (float)(s * scale);
}
// One workgroup: the loss of n terms
template <bool POLICY>
__global__ void __launch_bounds__(LS_ONE) k_ls_sum(LsArgs a, int n) {
  constexpr int U = 8;  // loaded together
  double s = 0.0;
  int k = 0;
  for (int i = threadIdx.x; i < n; i += LS_ONE * U) {
    double v[U];
    int t[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = min(i + LS_ONE * u, n - 1);
      v[u] = a.term[at];
      t[u] = POLICY ? ls_token(a, at) : 0;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + LS_ONE * u < n) {
        s += v[u];
        if (POLICY) k += t[u] >= 0;
      }
  }
  ls_total(a, s, k, POLICY ? 0 : n);
}
// One workgroup for a few pairs (and, with ROWS, a few rows): rows, pairs and the loss without launches between them, 3 us of the
// host's time each.  Rows go to the waves in turn, which the card pays for from some number on: the policy loss of 16 rows of 248,320
// without gradient 14.2 us in a graph in one launch behind the scan, 14.4 in two, of 40 rows 16.0 and 12.4, of 64 24.3 and 14.6.  The
// preference loss of 16, 32, 48 and 64 rows of 248,320 takes 12.2, 16.8, 18.0 and 21.9 us in a graph in one launch, 12.6, 15.1, 14.1 and
// 16.1 in two, but called one by one, where the host's time counts, 20.4, 19.9, 20.1 and 22.9 against 22.4, 22.4, 22.7 and 23.2; of 96 rows
// of 32,001 25.3 against 22.6.
constexpr int LS_FEW = 64, LS_FEW_ROWS = 48, LS_FEW_POLICY = 16;  // pairs; rows of the preference loss; rows of the policy loss, whose exponentials in 64 bits take longer
template <typename T, bool ROWS>
__global__ void __launch_bounds__(LS_ONE) k_ls_few(LsArgs a) {
  if constexpr (ROWS) {
    for (int row = wave_id(); row < a.R; row += LS_ONE / 64) ls_preference_row<T>(a, row);
    __syncthreads();  // the rows' log probabilities are other waves' in memory
  }
  double s = 0.0;
  for (int i = wave_id(); i < a.P; i += LS_ONE / 64) {
    const double term = ls_pair(a, i);
    if (lane_id() == 0) s += term;
  }
  ls_total(a, s, 0, a.P);
}

// The same for a few rows of the policy loss
template <typename T>
__global__ void __launch_bounds__(LS_ONE) k_ls_policy_few(LsArgs a) {
  double s = 0.0;
  int k = 0;
  for (int row = wave_id(); row < a.R; row += LS_ONE / 64) {
    const double term = ls_policy_row<T>(a, row, k);
    if (lane_id() == 0) s += term;
  }
  ls_total(a, s, lane_id() ? 0 : k, 0);
}

// ------------------------------------------------------------------------------------------------ the gradient's rows
typedef vu4 ls_any __attribute__((aligned(2)));  // 16 bytes at any element: the hardware takes them
// the vector at place v of `base`, at any element, of which [lead, end) exist: the rest reads -inf
template <typename T>
__device__ __forceinline__ vu4 lp_load_any(const T* base, int v, int lead, int end) {
  if (v >= lead && v + lp_e<T>() <= end) return *(const QWS_G ls_any*)(base + v);
  return lp_load_edge(base, v, lead, end);
}
template <typename T, int E>
__device__ __forceinline__ vu4 ls_pack(const float* y) {
  vu4 r;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (sizeof(T) == 4) {
      r[j] = __float_as_uint(y[j]);
    } else {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      const b2 h = {(__bf16)y[2 * j], (__bf16)y[2 * j + 1]};
      r[j] = __builtin_bit_cast(uint32_t, h);
    }
  }
  return r;
}
// E elements of the gradient at place j0 of a row: k p_j, and at the token's the slope as well
template <int E>
__device__ __forceinline__ void ls_slopes(const LsRow& q, const float* x, float* y, float k, float at_token, int tok, int j0) {
  if (q.mode == 1) {
#pragma unroll
    for (int j = 0; j < E; j++) y[j] = k * lse_exp2(fmaxf(fmaf(x[j], q.c, -q.M), -LSE_DMIN));  // NaN: 0
  } else {
#pragma unroll
    for (int j = 0; j < E; j++) y[j] = k * lse_exp2(lse_d(lse_clean(x[j]), q.m, q.c));
  }
  if ((unsigned)(tok - j0) < (unsigned)E) {
#pragma unroll
    for (int j = 0; j < E; j++)
      if (j0 + j == tok) y[j] += at_token;
  }
}

// the vector at place j0, of which [lead, end) exist
template <typename T>
__device__ __forceinline__ void ls_grad_edge(const LsRow& q, const T* base, T* to, int lead, int end, int j0, int tok, float k, float slope) {
  constexpr int E = lp_e<T>();
  const bool zero = slope == 0.0f;
  if (j0 >= lead && j0 + E <= end) {
    float x[E], y[E];
    vu4 w = {0, 0, 0, 0};
    if (!zero) {
      const vu4 r = *(const QWS_G ls_any*)(base + j0);
      lp_unpack<T>(r, x);
      ls_slopes<E>(q, x, y, k, slope, tok, j0);
      w = ls_pack<T, E>(y);
    }
    __builtin_nontemporal_store(w, (vu4*)(to + j0));
    return;
  }
  for (int j = max(j0, lead); j < min(j0 + E, end); j++) {
    float x, y = 0.0f;
    if constexpr (sizeof(T) == 4)
      x = *gmem((const float*)base + j);
    else
      x = __uint_as_float((uint32_t)*gmem((const uint16_t*)base + j) << 16);
    if (!zero) ls_slopes<1>(q, &x, &y, k, slope, tok, j);
    if constexpr (sizeof(T) == 4)
      *((float*)to + j) = y;
    else
      *((__bf16*)to + j) = (__bf16)y;
  }
}
// Stripes s_begin .. s_end of a row's gradient.  Its stores go around the caches, which then keep logits for their second reading (512 fp32
// rows of 248,320 in k_ls_policy 259 -> 217 us, 2,048 bf16 rows 412 -> 389; 1,200 bf16 rows by k_ls_scan and k_ls_grad 356 -> 317, and 304
// with its loads, the logits' last, marked so as well).
template <typename T, int U, int NT>
__device__ __forceinline__ void ls_grad_part(const LsRow& q, const T* x_row, T* out, int V, int s_begin, int s_end, float slope) {
  constexpr int E = lp_e<T>(), SE = ls_stripe<T>(NT);
  // aligned to the gradient's vectors; the logits' loads are at any element
  const int tid = threadIdx.x, lead = (int)((uintptr_t)out / sizeof(T)) & (E - 1), end = lead + V;
  const T* base = x_row - lead;
  T* to = out - lead;
  s_end = min(s_end, (end + SE - 1) / SE);
  const float k = -slope * q.inv;
  const bool zero = slope == 0.0f;
  const int tok = q.tok + lead;
  for (int s = s_begin; s < s_end; s += U) {
    const int first = s * SE;
    if (first >= lead && first + U * SE <= end && s + U <= s_end) {
      vu4 r[U];
      if (!zero) {
#pragma unroll
        for (int u = 0; u < U; u++) r[u] = __builtin_nontemporal_load((const QWS_G ls_any*)(base + first + u * SE + tid * E));
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j0 = first + u * SE + tid * E;
        float x[E], y[E];
        vu4 w = {0, 0, 0, 0};
        if (!zero) {
          lp_unpack<T>(r[u], x);
          ls_slopes<E>(q, x, y, k, slope, tok, j0);
          w = ls_pack<T, E>(y);
        }
        __builtin_nontemporal_store(w, (vu4*)(to + j0));
      }
    } else {
      for (int u = 0; u < U && s + u < s_end; u++) ls_grad_edge<T>(q, base, to, lead, end, first + u * SE + tid * E, tok, k, slope);
    }
  }
}
// A row's slope at its logits.  Held where it passes fp32: no infinity meets a p of 0; NaN stays, and so does what an upstream
// gradient that is not finite makes of it, which a loss scaler looks for.  A slope of 0 is one at every temperature, where 1 / T is
// past fp32 (T below 2^-128) as well.
__device__ __forceinline__ float ls_slope(float slope, float scale, float per_t) {
  slope *= scale;
  if (slope == 0.0f) return 0.0f;
  slope *= per_t;
  return fabsf(slope) > 0.25f * F32_MAX && fabsf(scale) <= F32_MAX ? copysignf(0.25f * F32_MAX, slope) : slope;
}

// written != 0: the gradient is there, for an upstream of that value.  Rows from the last on: the logits that k_ls_scan read last may still be in the
// memory's cache.
template <typename T, int U>
__global__ void __launch_bounds__(LS_NT) k_ls_grad(LsArgs a, float written) {
  const float upstream = a.upstream ? *a.upstream : a.grad_scale;
  if (written != 0.0f && upstream == written) return;
  const float scale = a.head->scale * upstream;
  for (unsigned i = blockIdx.x; i < (unsigned)a.R * a.G; i += gridDim.x) {
    const int row = a.R - 1 - (int)(i / a.G), ch = i % a.G;
    const LsRow q = a.rows[row];
    const float slope = q.mode ? ls_slope(a.slope[q.slot], scale, q.per_t) : 0.0f;
    ls_grad_part<T, U, LS_NT>(q, ls_row<T>(a, row), (T*)a.grad + (long long)row * a.grad_stride, a.V, ch * a.per, ch * a.per + a.per, slope);
  }
}

// ------------------------------------------------------------------------------------------------ the policy loss, a row at a time
// A workgroup per row: its maximum and sum, its term and slope, its gradient.  Of the row's stripes that lie inside it, NL stay in
// LDS and NV in registers between the two passes; the others are read again, the last ones first.
template <typename T, int NT, int NV, int NL>
__global__ void __launch_bounds__(NT) k_ls_policy(LsArgs a) {
  constexpr int E = lp_e<T>(), SE = ls_stripe<T>(NT), U = E == 8 ? 2 : 4;
  static_assert(NV % U == 0 && NL % U == 0 && NV >= 2 * U, "blocks");
  extern __shared__ __attribute__((aligned(16))) char s_mem[];
  vu4* held = (vu4*)s_mem + threadIdx.x;  // [NL][NT]: a thread's own
  __shared__ LsSum s_sum[NT / 64];
  __shared__ LsRow s_row;
  __shared__ float s_slope;
  const int tid = threadIdx.x, row = blockIdx.x, tok = ls_token(a, row);
  const float temp = a.temp ? a.temp[row] : 1.0f, c = lse_scale(temp);
  T* out = (T*)a.grad + (long long)row * a.grad_stride;
  const int lead = (int)((uintptr_t)out / sizeof(T)) & (E - 1), end = lead + a.V;
  const T* base = ls_row<T>(a, row) - lead;
  T* to = out - lead;
  const int stripes = (end + SE - 1) / SE, s0 = lead ? 1 : 0, full = max(end / SE - s0, 0) / U * U;  // whole stripes from s0 on, in blocks
  const int in_lds = min(full, NL), in_regs = min(full - in_lds, NV), s1 = s0 + in_lds, s2 = s1 + in_regs;
  vu4 r[NV];
  LsSum v = {-INFINITY, 0.0f};
  LsFast f = {-INFINITY, -1e30f, -INFINITY, 0.0f};
  auto vec = [&](int s) { return *(const QWS_G ls_any*)(base + s * SE + tid * E); };
  auto add = [&](const vu4* w) {
    float x[U][E], best = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
      lp_unpack<T>(w[u], x[u]);
      best = fmaxf(best, lp_max<E>(x[u]));
    }
    if (!ls_fast(f, x, best, c)) ls_slow(v, x, fminf(best, F32_MAX), c);
  };
  if (tok >= 0) {
    if constexpr (NL > 0) {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (in_lds) r[u] = vec(s0 + u);
#pragma unroll
      for (int i = 0; i < NL; i += U)
        if (i < in_lds) {
          vu4* now = r + i / U % 2 * U;
          vu4* next = r + (i / U + 1) % 2 * U;
          if (i + U < in_lds) {
#pragma unroll
            for (int u = 0; u < U; u++) next[u] = vec(s0 + i + U + u);
          }
          add(now);
#pragma unroll
          for (int u = 0; u < U; u++) held[(i + u) * NT] = now[u];
        }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (i < in_regs) r[i] = vec(s1 + i);
#pragma unroll
    for (int i = 0; i < NV; i += U)
      if (i < in_regs) add(r + i);
    // the rest: whole blocks, then what is left of the row's ends
    vu4 w[U];
    int s = s2;
    for (; s < s0 + full; s += U) {
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = vec(s + u);
      add(w);
    }
    for (; s < stripes + s0; s += U) {  // stripe 0, where it is not whole, at the end
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int at = s + u < stripes ? s + u : 0;
        w[u] = lp_load_any(base, at * SE + tid * E, s + u < stripes + s0 ? lead : end, end);
      }
      add(w);
    }
    if (f.m != -INFINITY) {
      const Lse q = lse_exact(f.m, f.M, f.s, 0.0f, c);
      v = ls_join(v, {q.m, q.s}, c);
    }
  }
  v = ls_join_group<NT>(v, c, s_sum);
  if (tid == 0) {
    a.term[row] = ls_policy<T>(a, row, tok, v, c, temp);
    const LsRow q = a.rows[row];  // this thread's own
    s_row = q;
    s_slope = q.mode ? ls_slope(a.slope[row], (a.weights ? 1.0f : a.head->scale) * a.grad_scale, q.per_t) : 0.0f;
  }
  bar();
  const LsRow q = s_row;
  const float slope = s_slope, k = -slope * q.inv;
  const bool zero = slope == 0.0f;
  const int at_tok = q.tok + lead;
  auto put = [&](int s, vu4 w) {
    const int j0 = s * SE + tid * E;
    float x[E], y[E];
    lp_unpack<T>(w, x);
    ls_slopes<E>(q, x, y, k, slope, at_tok, j0);
    __builtin_nontemporal_store(ls_pack<T, E>(y), (vu4*)(to + j0));
  };
  if (zero) {
    for (int s = 0; s < stripes; s++) ls_grad_edge<T>(q, base, to, lead, end, s * SE + tid * E, at_tok, k, slope);
    return;
  }
  for (int s = stripes + s0 - 1; s >= s0 + full; s--) ls_grad_edge<T>(q, base, to, lead, end, (s < stripes ? s : 0) * SE + tid * E, at_tok, k, slope);
  for (int s = s0 + full - U; s >= s2; s -= U) {
    vu4 w[U];
#pragma unroll
    for (int u = 0; u < U; u++) w[u] = vec(s + u);
#pragma unroll
    for (int u = 0; u < U; u++) put(s + u, w[u]);
  }
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (i < in_regs) put(s1 + i, r[i]);
  if constexpr (NL > 0) {
#pragma unroll 2
    for (int i = 0; i < NL; i++)
      if (i < in_lds) put(s0 + i, held[i * NT]);
  }
}
// One workgroup: without weights, the scale of the slopes is known before them: 1 over the rows with a token
__global__ void __launch_bounds__(LS_ONE) k_ls_count(LsArgs a) {
  __shared__ int s_count[LS_ONE / 64];
  constexpr int U = 8;  // loaded together
  int k = 0;
  for (int i = threadIdx.x; i < a.R; i += LS_ONE * U) {
    int t[U];
#pragma unroll
    for (int u = 0; u < U; u++) t[u] = ls_token(a, min(i + LS_ONE * u, a.R - 1));
#pragma unroll
    for (int u = 0; u < U; u++) k += i + LS_ONE * u < a.R && t[u] >= 0;
  }
  k = wave_sum<int>(k);
  if (lane_id() == 0) s_count[wave_id()] = k;
  bar();
  if (threadIdx.x) return;
  for (int w = 1; w < LS_ONE / 64; w++) k += s_count[w];
  a.head->scale = k ? (float)(1.0 / k) : 1.0f;
}

// ------------------------------------------------------------------------------------------------ the host's side
struct LsPlan {
  int G, per;
};
// Stripes (4 KB) of a workgroup: one while they are few, then as many as leave about 4,096 workgroups, whole blocks of LS_U.
template <typename T>
inline LsPlan ls_plan(int R, int V) {
  const long long stripes = (V + lp_e<T>() - 1 + ls_stripe<T>() - 1) / ls_stripe<T>(), all = stripes * R;
  long long per = all <= 2048 ? 1 : (all + 4095) / 4096;
  if (per > 1) per = (per + LS_U - 1) / LS_U * LS_U;
  if (per > stripes) per = stripes;
  return {(int)((stripes + per - 1) / per), (int)per};
}
inline LsPlan ls_plan_of(int dtype, int R, int V) { return dtype == QWS_DTYPE_F32 ? ls_plan<float>(R, V) : ls_plan<uint16_t>(R, V); }

struct LsState {
  size_t rows, slope, lp, term, part, total;
};
// slopes and terms: R and R, or 2 P and P
inline LsState ls_state(int dtype, int R, int V, long long slopes, long long terms) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  LsState s;
  s.rows = 256;
  s.slope = s.rows + up((size_t)R * sizeof(LsRow));
  s.lp = s.slope + up((size_t)slopes * 4);
  s.term = s.lp + up((size_t)R * 8);
  s.part = s.term + up((size_t)terms * 8);
  s.total = s.part + up((size_t)R * ls_plan_of(dtype, R, V).G * sizeof(float2));
  return s;
}
static bool ls_rows_ok(const qws_loss_rows& r) {
  const uintptr_t mask = r.dtype == QWS_DTYPE_F32 ? 3 : 1;
  return (r.dtype == QWS_DTYPE_F32 || r.dtype == QWS_DTYPE_BF16) && r.R >= 0 && r.V >= 1 && r.block >= 0 && r.row_stride >= 0 && r.block_stride >= 0 &&
         (r.R == 0 || (r.logits && !((uintptr_t)r.logits & mask) && r.tokens));
}
static bool ls_fits(int R, int V) { return R < LS_RMAX && V <= LS_VMAX; }
static bool ls_grad_ok(const qws_loss_rows& r, const void* grad, long long stride) {
  return !((uintptr_t)grad & (r.dtype == QWS_DTYPE_F32 ? 3 : 1)) && (r.R <= 1 || stride >= r.V);
}
static LsArgs ls_args(const qws_loss_rows& r, char* state, const LsState& l) {
  LsArgs a = {};
  a.x = r.logits;
  a.stride = r.row_stride;
  a.block = r.block > 0 ? r.block : r.R > 0 ? r.R : 1;
  a.block_stride = r.block_stride;
  a.tok = r.tokens;
  a.temp = r.temperature;
  a.R = r.R;
  a.V = r.V;
  const LsPlan p = ls_plan_of(r.dtype, r.R, r.V);
  a.G = p.G;
  a.per = p.per;
  a.head = (LsHead*)state;
  a.rows = (LsRow*)(state + l.rows);
  a.slope = (float*)(state + l.slope);
  a.lp = (double*)(state + l.lp);
  a.term = (double*)(state + l.term);
  a.part = (float2*)(state + l.part);
  return a;
}
template <typename T>
static void ls_scan(const LsArgs& a, hipStream_t st) {
  if (a.per == 1)
    hipLaunchKernelGGL((k_ls_scan<T, 1>), dim3((unsigned)a.R * a.G), dim3(LS_NT), 0, st, a);
  else
    hipLaunchKernelGGL((k_ls_scan<T, LS_U>), dim3((unsigned)a.R * a.G), dim3(LS_NT), 0, st, a);
}
template <typename T>
static void ls_grad_of(const LsArgs& a, float written, hipStream_t st) {
  unsigned wgs = (unsigned)a.R * a.G;
  if (written != 0.0f && wgs > 4096) wgs = 4096;  // most often they find it written
  if (a.per == 1)
    hipLaunchKernelGGL((k_ls_grad<T, 1>), dim3(wgs), dim3(LS_NT), 0, st, a, written);
  else
    hipLaunchKernelGGL((k_ls_grad<T, LS_U>), dim3(wgs), dim3(LS_NT), 0, st, a, written);
}
static void ls_grad(const LsArgs& a, int dtype, float written, hipStream_t st) {
  dtype == QWS_DTYPE_F32 ? ls_grad_of<float>(a, written, st) : ls_grad_of<uint16_t>(a, written, st);
}
// Whether a policy loss with its gradient takes a workgroup per row (k_ls_policy): from 128 rows on, or where the row's workgroup holds
// all of it (up to 12,288 vectors).  Measured, us a call, k_ls_policy / the launches of ls_policy_run and k_ls_grad: 248,320 bf16 logits, 16 rows
// 35 / 26, 64 rows 37 / 28, 100 rows 38 / 36, 128 rows 38 / 42, 150 rows 39 / 45, 256 rows 58 / 68, 2,048 rows 396 / 528; fp32, 64 rows 43 / 40,
// 100 rows 55 / 57, 128 rows 64 / 68, 192 rows 91 / 97, 512 rows 215 / 250; 32,001 bf16 logits, 64 rows 26 / 27, 1,024 rows 36 / 48.
constexpr int LS_HELD = 512 * 24;
static int ls_vectors(int dtype, int V) { return V / (dtype == QWS_DTYPE_F32 ? 4 : 8); }
static bool ls_one_pass(int dtype, int R, int V) { return R >= 128 || ls_vectors(dtype, V) <= LS_HELD; }
template <typename T, int NT, int NV, int NL>
static void ls_policy_rows(const LsArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((k_ls_policy<T, NT, NV, NL>), dim3(a.R), dim3(NT), NL * NT * 16, st, a);
}
// The least workgroup that holds a row: 2,048 bf16 rows, us with 256 x 16 / 512 x 24 / 1,024 x 24 vectors: of 16,000 logits 33 / 42 / 64,
// of 32,001 65 / 72 / 95, of 40,000 82 / 81 / 101, of 100,000 221 / 181 / 188, of 130,000 308 / 239 / 244, of 200,000 439 / 376 / 347.  Where
// there are at most two rows to a CU the larger one is quicker from some 2,000 vectors on (in a graph): 32,001 bf16 logits, 24 rows 16.9 /
// 14.4, 400 rows 21.4 / 19.0; 16,000 (2,000 vectors: the border), 100 rows 12.8 / 12.0, 400 rows 15.1 / 14.7; 12,000, 100 rows 11.9 /
// 11.8; 8,000, 4 and 100 rows 10.9 / 11.0.
template <typename T>
static void ls_policy_one_pass(const LsArgs& a, hipStream_t st) {
  const int n = a.V / lp_e<T>();
  if (n <= 2048 || (n <= 4096 && a.R > 512))
    ls_policy_rows<T, 256, 16, 0>(a, st);
  else if (n <= LS_HELD)
    ls_policy_rows<T, 512, 16, 8>(a, st);
  else
    ls_policy_rows<T, 1024, 16, 8>(a, st);
}
template <typename T>
static void ls_policy_run(const LsArgs& a, hipStream_t st) {
  if (a.R) ls_scan<T>(a, st);
  if (a.R <= LS_FEW_POLICY) {
    hipLaunchKernelGGL((k_ls_policy_few<T>), dim3(1), dim3(LS_ONE), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((k_ls_policy_rows<T>), dim3((a.R + LS_NW - 1) / LS_NW), dim3(LS_NT), 0, st, a);
  hipLaunchKernelGGL((k_ls_sum<true>), dim3(1), dim3(LS_ONE), 0, st, a, a.R);
}
template <typename T>
static void ls_preference_run(const LsArgs& a, hipStream_t st) {
  if (a.R) ls_scan<T>(a, st);
  if (a.P <= LS_FEW && a.R <= LS_FEW_ROWS) {
    hipLaunchKernelGGL((k_ls_few<T, true>), dim3(1), dim3(LS_ONE), 0, st, a);
    return;
  }
  if (a.R) hipLaunchKernelGGL((k_ls_rows<T>), dim3((a.R + LS_NW - 1) / LS_NW), dim3(LS_NT), 0, st, a);
  if (a.P <= LS_FEW) {
    hipLaunchKernelGGL((k_ls_few<T, false>), dim3(1), dim3(LS_ONE), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(k_ls_pairs, dim3((a.P + LS_NW - 1) / LS_NW), dim3(LS_NT), 0, st, a);
  hipLaunchKernelGGL((k_ls_sum<false>), dim3(1), dim3(LS_ONE), 0, st, a, a.P);
}
static bool ls_aligned(const void* p) { return p && ((uintptr_t)p & 255) == 0; }
static bool ls_launches(const LsArgs& a) { return (long long)a.R * a.G <= 0xFFFFFF; }  // below 2^32 threads
static bool ls_number(float x) { return x == x && x >= -F32_MAX && x <= F32_MAX; }

}  // namespace qws

extern "C" size_t qws_policy_state_bytes(int dtype, int R, int V) {
  using namespace qws;
  if ((dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) || R < 0 || V < 1 || !ls_fits(R, V)) return 0;
  return ls_state(dtype, R, V, R, R).total;
}
extern "C" size_t qws_preference_state_bytes(int dtype, int R, int V, int P) {
  using namespace qws;
  if ((dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) || R < 0 || V < 1 || P < 0 || !ls_fits(R, V) || P >= LS_RMAX / 2) return 0;
  return ls_state(dtype, R, V, 2ll * P, P).total;
}

extern "C" int qws_policy_loss(const qws_policy_batch* b, void* state, size_t state_bytes, void* grad, long long grad_stride, float grad_scale, void* stream) {
  using namespace qws;
  if (!ls_number(grad_scale)) return QWS_ERR_INVALID;
  if (!b || !ls_rows_ok(b->rows) || !b->out_loss || !ls_aligned(state)) return QWS_ERR_INVALID;
  if (!(b->clip_low >= 0.0f && b->clip_low <= 1.0f) || !(b->clip_high >= 0.0f) || !ls_number(b->clip_high) || !ls_number(b->kl)) return QWS_ERR_INVALID;
  const int R = b->rows.R, V = b->rows.V;
  if (!ls_fits(R, V)) return QWS_ERR_NOT_SUPPORTED;
  if (R && (!b->old_logprobs || !b->advantages || (grad && !ls_grad_ok(b->rows, grad, grad_stride)))) return QWS_ERR_INVALID;
  const LsState l = ls_state(b->rows.dtype, R, V, R, R);
  if (state_bytes < l.total) return QWS_ERR_INVALID;
  LsArgs a = ls_args(b->rows, (char*)state, l);
  if (!ls_launches(a)) return QWS_ERR_NOT_SUPPORTED;
  a.old_lp = b->old_logprobs;
  a.adv = b->advantages;
  a.ref = b->ref_logprobs;
  a.weights = b->weights;
  a.clip_low = b->clip_low;
  a.clip_high = b->clip_high;
  a.kl = b->kl;
  a.out_loss = b->out_loss;
  a.out_lp = b->out_logprobs;
  a.out_ratio = b->out_ratio;
  a.out_kl = b->out_kl;
  a.grad_scale = grad_scale;
  hipStream_t st = (hipStream_t)stream;
  if (R && grad && ls_one_pass(b->rows.dtype, R, V)) {
    a.grad = grad;
    a.grad_stride = grad_stride;
    if (!a.weights) hipLaunchKernelGGL(k_ls_count, dim3(1), dim3(LS_ONE), 0, st, a);
    b->rows.dtype == QWS_DTYPE_F32 ? ls_policy_one_pass<float>(a, st) : ls_policy_one_pass<uint16_t>(a, st);
    hipLaunchKernelGGL((k_ls_sum<true>), dim3(1), dim3(LS_ONE), 0, st, a, R);
    return (int)hipGetLastError();
  }
  b->rows.dtype == QWS_DTYPE_F32 ? ls_policy_run<float>(a, st) : ls_policy_run<uint16_t>(a, st);
  if (R && grad) {
    a.grad = grad;
    a.grad_stride = grad_stride;
    ls_grad(a, b->rows.dtype, 0, st);
  }
  return (int)hipGetLastError();
}

extern "C" int qws_preference_loss(const qws_preference_batch* b, void* state, size_t state_bytes, void* grad, long long grad_stride, float grad_scale, void* stream) {
  using namespace qws;
  if (!ls_number(grad_scale)) return QWS_ERR_INVALID;
  if (!b || !ls_rows_ok(b->rows) || !b->out_loss || !ls_aligned(state) || b->P < 0 || (b->P && !b->starts)) return QWS_ERR_INVALID;
  if (!ls_number(b->beta) || !ls_number(b->margin) || !(b->smoothing >= 0.0f && b->smoothing <= 1.0f)) return QWS_ERR_INVALID;
  const int R = b->rows.R, V = b->rows.V, P = b->P;
  if (!ls_fits(R, V) || P >= LS_RMAX / 2) return QWS_ERR_NOT_SUPPORTED;
  if (R && grad && !ls_grad_ok(b->rows, grad, grad_stride)) return QWS_ERR_INVALID;
  const LsState l = ls_state(b->rows.dtype, R, V, 2ll * P, P);
  if (state_bytes < l.total) return QWS_ERR_INVALID;
  LsArgs a = ls_args(b->rows, (char*)state, l);
  if (!ls_launches(a)) return QWS_ERR_NOT_SUPPORTED;
  a.starts = b->starts;
  a.P = P;
  a.ref = b->ref;
  a.weights = b->weights;
  a.beta = b->beta;
  a.margin = b->margin;
  a.smoothing = b->smoothing;
  a.average = b->average;
  a.out_loss = b->out_loss;
  a.out_lp = b->out_token_logprobs;
  a.out_sums = b->out_logprobs;
  a.out_margins = b->out_margins;
  a.grad_scale = grad_scale;
  hipStream_t st = (hipStream_t)stream;
  b->rows.dtype == QWS_DTYPE_F32 ? ls_preference_run<float>(a, st) : ls_preference_run<uint16_t>(a, st);
  if (R && grad) {
    a.grad = grad;
    a.grad_stride = grad_stride;
    ls_grad(a, b->rows.dtype, 0, st);
  }
  return (int)hipGetLastError();
}

extern "C" int qws_policy_one_pass(int dtype, int R, int V) { return R > 0 && V > 0 && qws::ls_one_pass(dtype, R, V); }

extern "C" int qws_loss_grad(const qws_loss_rows* r, const void* state, const float* upstream, void* grad, long long grad_stride, float written, void* stream) {
  using namespace qws;
  if (!ls_number(written) || !r || !ls_rows_ok(*r) || !ls_aligned(state) || (r->R && (!grad || !ls_grad_ok(*r, grad, grad_stride)))) return QWS_ERR_INVALID;
  if (!ls_fits(r->R, r->V)) return QWS_ERR_NOT_SUPPORTED;
  if (r->R == 0) return QWS_OK;
  LsArgs a = ls_args(*r, (char*)state, ls_state(r->dtype, r->R, r->V, 0, 0));  // the places of the rows and slopes do not depend on the loss
  if (!ls_launches(a)) return QWS_ERR_NOT_SUPPORTED;
  a.upstream = upstream;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.grad_scale = 1.0f;
  ls_grad(a, r->dtype, upstream ? written : 0.0f, (hipStream_t)stream);
  return (int)hipGetLastError();
}
