// qws log probabilities of given tokens, their ranks, the row's entropy and its best alternatives, over rows of logits
// (the definition: include/qws.h qws_logprobs; the running sums: qws_lse.h).
//
//   k_lp_scan   R x G workgroups of 256: one pass over the logits.  Each lane keeps the running maximum and sums of its
//               elements; each given token's rank is counted by ballots; and the maximum of every 64 consecutive logits
//               (a group) goes to the workspace.
//   k_lp_row    R workgroups of 256: joins the row's parts, writes log probabilities, ranks and entropy, and takes the
//               alternatives in two selections: the n groups with the best maxima (ties: the first), then the n best of
//               those groups' logits.  That is exact: a logit outside those groups has n better ones, the maxima of the n
//               groups (each larger, or equal and of a lower index, since groups are consecutive runs of tokens).  So the
//               pass over the logits does nothing more for 64 alternatives than for none, whatever their order in memory.
#include "qws_lse.h"

namespace qws {

constexpr int LP_NT = 256;      // threads
constexpr int LP_NW = LP_NT / 64;
constexpr int LP_GRP = 64;      // consecutive logits of a group
constexpr int LP_NMAX = 64;     // alternatives and given tokens of a row at most
constexpr int LP_U = 4;         // 16-byte vectors of a thread in flight together
constexpr int LP_VMAX = 1 << 19;
constexpr int LP_WGS = 2048;    // workgroups that fill the card: 8 of 256 threads on each of 256 CUs

template <typename T>
constexpr int lp_e() { return 16 / (int)sizeof(T); }  // elements of a vector
template <typename T>
constexpr int lp_stripe() { return LP_NT * lp_e<T>(); }  // elements that a workgroup's threads load at once

struct LpArgs {
  const void* x;
  long long stride;
  const int* tok;
  const float* temp;
  int V, M, top;
  int G, per;      // workgroups of a row, stripes of each
  int groups;      // groups of a row in `gmax`
  float4* part;    // [R][G] m, s, t
  int* cnt;        // [R][G][M] logits before the given token
  float* gmax;     // [R][groups]
  float* out_lp;
  int* out_rank;
  float* out_h;
  int* out_ids;
  float* out_top;
};

template <typename T>
__device__ __forceinline__ float lp_one(const T* p) {
  if constexpr (sizeof(T) == 4)
    return lse_clean(*gmem((const float*)p));
  else
    return lse_clean(__uint_as_float((uint32_t)*gmem((const uint16_t*)p) << 16));
}
// the vector at virtual position v (elements [lead, end) of `base` exist; base is 16-byte aligned)
template <typename T>
__device__ __forceinline__ void lp_unpack(vu4 r, float* x) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = lse_clean(__uint_as_float(r[j]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[2 * j] = lse_clean(__uint_as_float(r[j] << 16));
      x[2 * j + 1] = lse_clean(__uint_as_float(r[j] & 0xFFFF0000u));
    }
  }
}
template <typename T>
__device__ inline void lp_load_edge(const T* base, int v, int lead, int end, float* x) {
#pragma unroll
  for (int j = 0; j < lp_e<T>(); j++) x[j] = v + j >= lead && v + j < end ? lp_one(base + v + j) : -INFINITY;
}

// RANK: 0 no given tokens' ranks, 1 one token per row (held in registers), 2 several (in LDS)
template <typename T, int RANK, bool TOP>
__global__ void __launch_bounds__(LP_NT, 8) k_lp_scan(LpArgs a) {
  constexpr int E = lp_e<T>(), SE = lp_stripe<T>();
  __shared__ float s_xt[LP_NMAX];
  __shared__ int s_tv[LP_NMAX], s_cnt[LP_NMAX];
  __shared__ Lse s_lse[LP_NW];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int row = blockIdx.x / a.G, ch = blockIdx.x % a.G;
  const T* p = (const T*)a.x + (long long)row * a.stride;
  const int lead = (int)((uintptr_t)p / sizeof(T)) & (E - 1), end = lead + a.V;
  const T* base = p - lead;
  const float c = lse_scale(a.temp ? a.temp[row] : 1.0f);
  const int nstripes = (end + SE - 1) / SE, s_end = min((ch + 1) * a.per, nstripes);
  float xt = 0.0f;
  int tv = -1, cnt = 0;  // virtual position of the token (-1: skipped), logits before it
  if constexpr (RANK == 1) {
    const int t = a.tok[row];
    if (t >= 0 && t < a.V) {
      tv = t + lead;
      xt = lp_one(p + t);
    }
  }
  if constexpr (RANK == 2) {
    if (tid < a.M) {
      const int t = a.tok[(long long)row * a.M + tid];
      const bool ok = t >= 0 && t < a.V;
      s_tv[tid] = ok ? t + lead : -1;
      s_xt[tid] = ok ? lp_one(p + t) : 0.0f;
      s_cnt[tid] = 0;
    }
    bar();
  }
  Lse v = {-INFINITY, 0.0f, 0.0f};
  for (int s = ch * a.per; s < s_end; s += LP_U) {
    float x[LP_U][E];
    const int first = s * SE;
    if (first >= lead && first + LP_U * SE <= end && s + LP_U <= s_end) {
      vu4 r[LP_U];
#pragma unroll
      for (int u = 0; u < LP_U; u++) r[u] = *gmem((const vu4*)(base + first + u * SE + tid * E));
#pragma unroll
      for (int u = 0; u < LP_U; u++) lp_unpack<T>(r[u], x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < LP_U; u++) lp_load_edge(base, first + u * SE + tid * E, lead, s + u < s_end ? end : 0, x[u]);
    }
    float best = -INFINITY;
#pragma unroll
    for (int u = 0; u < LP_U; u++) {
      float m = x[u][0];
#pragma unroll
      for (int j = 1; j < E; j++) m = fmaxf(m, x[u][j]);
      best = fmaxf(best, m);
      if constexpr (TOP) {
        constexpr int L = LP_GRP / E;  // lanes of a group: 8 or 16
        m = fmaxf(m, dpp_perm<0xB1>(m));
        m = fmaxf(m, dpp_perm<0x4E>(m));
        m = fmaxf(m, dpp_perm<0x141>(m));
        if constexpr (L == 16) m = fmaxf(m, dpp_perm<0x140>(m));
        if ((lane & (L - 1)) == 0 && s + u < s_end) a.gmax[(long long)row * a.groups + (first + u * SE + tid * E) / LP_GRP] = m;
      }
    }
    {  // the new maximum, then the elements
      const float m = fmaxf(v.m, best), d = lse_d(v.m, m, c), e = lse_exp2(d);
      v = {m, v.s * e, e * fmaf(d, v.s, v.t)};
    }
#pragma unroll
    for (int u = 0; u < LP_U; u++)
#pragma unroll
      for (int j = 0; j < E; j++) {
        const float d = lse_d(x[u][j], v.m, c), e = lse_exp2(d);
        v.s += e;
        v.t = fmaf(e, d, v.t);
      }
    if constexpr (RANK != 0) {
      const int n = RANK == 1 ? 1 : a.M;
      for (int k = 0; k < n; k++) {
        const float xk = RANK == 1 ? xt : s_xt[k];
        const int tk = RANK == 1 ? tv : s_tv[k];
        int add = 0;
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
          // this wave's elements: [lo, lo + 64 E); a stripe of the next workgroup lies behind every token
          const int lo = s + u < s_end ? first + u * SE + wave * 64 * E : 0x7FFFFFFF - 64 * E;
          if (lo + 64 * E <= tk) {
#pragma unroll
            for (int j = 0; j < E; j++) add += __popcll(__ballot(x[u][j] >= xk));
          } else if (lo > tk) {
#pragma unroll
            for (int j = 0; j < E; j++) add += __popcll(__ballot(x[u][j] > xk));
          } else {
#pragma unroll
            for (int j = 0; j < E; j++) add += __popcll(__ballot(x[u][j] > xk || (x[u][j] == xk && lo + lane * E + j < tk)));
          }
        }
        if constexpr (RANK == 1)
          cnt += add;
        else if (lane == 0)
          atomicAdd(&s_cnt[k], add);
      }
    }
  }
  v = lse_join_lanes(v, c, 1, 32);
  if constexpr (RANK == 1) {
    if (tid == 0) s_cnt[0] = 0;
    bar();
    if (lane == 0) atomicAdd(&s_cnt[0], cnt);
  }
  if (lane == 0) s_lse[wave] = v;
  bar();
  const long long o = (long long)row * a.G + ch;
  if (tid == 0) {
    for (int w = 1; w < LP_NW; w++) v = lse_join(v, s_lse[w], c);
    a.part[o] = make_float4(v.m, v.s, v.t, 0.0f);
  }
  if constexpr (RANK != 0)
    if (tid < (RANK == 1 ? 1 : a.M)) a.cnt[o * a.M + tid] = s_cnt[tid];
}

struct LpSel {
  uint64_t col[LP_NW][64], best[64], thr;
  int rank[64], n;
  int win[LP_NMAX];
};
// A lower bound of the block's n-th largest key (n <= 64; keys distinct, 0 = none): the n-th largest of the 64 lanes' best
// keys, each over the lane of every wave.  0 when fewer lanes have a key.  Clears s.n; ends with a barrier.
__device__ inline uint64_t lp_threshold(uint64_t mine, int n, LpSel& s) {
  const int lane = lane_id(), wave = wave_id();
  bar();
  s.col[wave][lane] = mine;
  if (wave == 0) s.rank[lane] = 0;
  if (threadIdx.x == 0) s.thr = 0, s.n = 0;
  bar();
#pragma unroll
  for (int w = 0; w < LP_NW; w++) mine = max(mine, s.col[w][lane]);
  if (wave == 0) s.best[lane] = mine;
  bar();
  int above = 0;
#pragma unroll
  for (int j = 0; j < 64 / LP_NW; j++) above += s.best[wave * (64 / LP_NW) + j] > mine;
  atomicAdd(&s.rank[lane], above);
  bar();
  if (wave == 0 && mine && s.rank[lane] == n - 1) s.thr = mine;
  bar();
  return s.thr;
}
__device__ __forceinline__ void lp_take(uint64_t k, uint64_t thr, LpSel& s, uint64_t* list) {
  if (k && k >= thr) list[atomicAdd(&s.n, 1)] = k;
}
// calls put(rank, key) for every key of the list that is among its n best
template <typename F>
__device__ __forceinline__ void lp_ranked(const LpSel& s, const uint64_t* list, int n, F put) {
  const int c = s.n;
  for (int i = threadIdx.x; i < c; i += LP_NT) {
    const uint64_t k = list[i];
    int r = 0;
    for (int j = 0; j < c; j++) r += list[j] > k;
    if (r < n) put(r, k);
  }
}

template <typename T>
__global__ void __launch_bounds__(LP_NT) k_lp_row(LpArgs a) {
  constexpr int E = lp_e<T>();
  extern __shared__ uint64_t list[];  // as many keys as a selection can keep: max(groups, 64 top)
  __shared__ LpSel s;
  __shared__ Lse s_lse[LP_NW];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), row = blockIdx.x;
  const T* p = (const T*)a.x + (long long)row * a.stride;
  const int lead = (int)((uintptr_t)p / sizeof(T)) & (E - 1), end = lead + a.V;
  const float temp = a.temp ? a.temp[row] : 1.0f, c = lse_scale(temp);
  Lse v = {-INFINITY, 0.0f, 0.0f};
  for (int g = tid; g < a.G; g += LP_NT) {
    const float4 q = a.part[(long long)row * a.G + g];
    v = lse_join(v, {q.x, q.y, q.z}, c);
  }
  v = lse_join_lanes(v, c, 1, 32);
  if (lane == 0) s_lse[wave] = v;
  bar();
  v = s_lse[0];
#pragma unroll
  for (int w = 1; w < LP_NW; w++) v = lse_join(v, s_lse[w], c);
  if (tid == 0 && a.out_h) a.out_h[row] = lse_entropy(v);
  for (int m = wave; m < a.M; m += LP_NW) {
    const long long o = (long long)row * a.M + m;
    const int t = a.tok[o];
    const bool ok = t >= 0 && t < a.V;
    const float x = ok ? lp_one(p + t) : 0.0f;
    if (a.out_lp && lane == 0) a.out_lp[o] = ok ? lse_logprob(v, x, temp) : 0.0f;
    if (a.out_rank) {
      int n = 0;
      for (int g = lane; g < a.G; g += 64) n += a.cnt[((long long)row * a.G + g) * a.M + m];
      n = wave_sum<int>(n);
      if (x == -INFINITY) n -= lead;  // the places before the row were counted as -inf of lower indices
      if (lane == 0) a.out_rank[o] = ok ? n : -1;
    }
  }
  if (a.top == 0) return;
  const float* gm = a.gmax + (long long)row * a.groups;
  uint64_t best = 0;
  for (int g = tid; g < a.groups; g += LP_NT) {
    const float x = gm[g];
    if (x > -INFINITY) best = max(best, comp(okey(x), (uint32_t)g));
  }
  uint64_t thr = lp_threshold(best, a.top, s);
  for (int g = tid; g < a.groups; g += LP_NT) {
    const float x = gm[g];
    if (x > -INFINITY) lp_take(comp(okey(x), (uint32_t)g), thr, s, list);
  }
  bar();
  lp_ranked(s, list, a.top, [&](int r, uint64_t k) { s.win[r] = (int)comp_idx(k); });
  const int nw = min(s.n, a.top);
  bar();
  uint64_t key[LP_NMAX / LP_NW];
  best = 0;
#pragma unroll
  for (int i = 0; i < LP_NMAX / LP_NW; i++) {
    const int k = i * LP_NW + wave;
    key[i] = 0;
    if (k < nw) {
      const int e = s.win[k] * LP_GRP + lane;
      if (e >= lead && e < end) {
        const float x = lp_one(p + (e - lead));
        if (x > -INFINITY) key[i] = comp(okey(x), (uint32_t)(e - lead));
      }
    }
    best = max(best, key[i]);
  }
  thr = lp_threshold(best, a.top, s);
#pragma unroll
  for (int i = 0; i < LP_NMAX / LP_NW; i++) lp_take(key[i], thr, s, list);
  bar();
  int* ids = a.out_ids + (long long)row * a.top;
  float* lps = a.out_top + (long long)row * a.top;
  lp_ranked(s, list, a.top, [&](int r, uint64_t k) {
    ids[r] = (int)comp_idx(k);
    lps[r] = lse_logprob(v, okey_val(comp_key(k)), temp);
  });
  for (int r = s.n + tid; r < a.top; r += LP_NT) {
    ids[r] = -1;
    lps[r] = -INFINITY;
  }
}

struct LpPlan {
  int G, per, groups;
  size_t part, cnt, gmax, total;  // byte offsets
};
// Workgroups of a row: all of its stripes' while the card is not full, else as many as fill it (more would add parts to
// join and no bandwidth).
template <typename T>
LpPlan lp_plan(int R, int V, int M, int top) {
  LpPlan q;
  const int stripes = (V + lp_e<T>() - 1 + lp_stripe<T>() - 1) / lp_stripe<T>();
  const long long all = (long long)R * stripes;
  q.per = (int)((all + LP_WGS - 1) / LP_WGS);
  if (q.per > stripes) q.per = stripes;
  if (q.per > LP_U) q.per = (q.per + LP_U - 1) / LP_U * LP_U;
  q.G = (stripes + q.per - 1) / q.per;
  q.groups = top ? stripes * (lp_stripe<T>() / LP_GRP) : 0;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  q.part = 0;
  q.cnt = up((size_t)R * q.G * sizeof(float4));
  q.gmax = q.cnt + up((size_t)R * q.G * M * sizeof(int));
  q.total = q.gmax + up((size_t)R * q.groups * sizeof(float));
  return q;
}

template <typename T, int RANK>
void lp_launch_scan(const LpArgs& a, int R, hipStream_t st) {
  if (a.top)
    hipLaunchKernelGGL((k_lp_scan<T, RANK, true>), dim3((unsigned)R * a.G), dim3(LP_NT), 0, st, a);
  else
    hipLaunchKernelGGL((k_lp_scan<T, RANK, false>), dim3((unsigned)R * a.G), dim3(LP_NT), 0, st, a);
}
template <typename T>
int lp_launch(LpArgs a, int R, char* ws, size_t ws_bytes, hipStream_t st) {
  const LpPlan q = lp_plan<T>(R, a.V, a.M, a.top);
  if (ws_bytes < q.total || (uint64_t)R * q.G > 0x7FFFFFFFull) return ws_bytes < q.total ? QWS_ERR_INVALID : QWS_ERR_NOT_SUPPORTED;
  a.G = q.G;
  a.per = q.per;
  a.groups = q.groups;
  a.part = (float4*)(ws + q.part);
  a.cnt = (int*)(ws + q.cnt);
  a.gmax = (float*)(ws + q.gmax);
  if (!a.M || !a.out_rank)
    lp_launch_scan<T, 0>(a, R, st);
  else if (a.M == 1)
    lp_launch_scan<T, 1>(a, R, st);
  else
    lp_launch_scan<T, 2>(a, R, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const size_t lds = a.top ? sizeof(uint64_t) * (size_t)(q.groups > LP_GRP * a.top ? q.groups : LP_GRP * a.top) : 0;
  hipLaunchKernelGGL((k_lp_row<T>), dim3(R), dim3(LP_NT), lds, st, a);
  return (int)hipGetLastError();
}

}  // namespace qws

extern "C" size_t qws_logprobs_ws_bytes(int dtype, int R, int V, int M, int top) {
  using namespace qws;
  if (R < 1 || V < 1 || V > LP_VMAX || M < 0 || M > LP_NMAX || top < 0 || top > LP_NMAX) return 0;
  if (dtype == QWS_DTYPE_F32) return lp_plan<float>(R, V, M, top).total;
  return dtype == QWS_DTYPE_BF16 ? lp_plan<uint16_t>(R, V, M, top).total : 0;
}

extern "C" int qws_logprobs(const qws_logprobs_batch* b, void* ws, size_t ws_bytes, void* stream) {
  using namespace qws;
  if (!b || b->R < 0 || b->V < 1 || b->M < 0 || b->top < 0 || (b->dtype != QWS_DTYPE_F32 && b->dtype != QWS_DTYPE_BF16)) return QWS_ERR_INVALID;
  if (b->V > LP_VMAX || b->M > LP_NMAX || b->top > LP_NMAX) return QWS_ERR_NOT_SUPPORTED;
  if (b->R == 0) return QWS_OK;
  const size_t size = b->dtype == QWS_DTYPE_F32 ? 4 : 2;
  if (!b->logits || ((uintptr_t)b->logits & (size - 1)) || !ws || ((uintptr_t)ws & 255) || b->row_stride < 0) return QWS_ERR_INVALID;
  if ((b->M && (!b->tokens || !b->out_logprobs)) || (!b->M && (b->out_logprobs || b->out_ranks)) || (b->top && (!b->out_top_ids || !b->out_top_logprobs)))
    return QWS_ERR_INVALID;
  LpArgs a = {};
  a.x = b->logits;
  a.stride = b->row_stride;
  a.tok = b->tokens;
  a.temp = b->temperature;
  a.V = b->V;
  a.M = b->M;
  a.top = b->top;
  a.out_lp = b->out_logprobs;
  a.out_rank = b->out_ranks;
  a.out_h = b->out_entropy;
  a.out_ids = b->out_top_ids;
  a.out_top = b->out_top_logprobs;
  return b->dtype == QWS_DTYPE_F32 ? lp_launch<float>(a, b->R, (char*)ws, ws_bytes, (hipStream_t)stream)
                                   : lp_launch<uint16_t>(a, b->R, (char*)ws, ws_bytes, (hipStream_t)stream);
}
