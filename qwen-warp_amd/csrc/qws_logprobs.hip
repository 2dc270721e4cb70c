// qws log probabilities of given tokens, their ranks, the row's entropy and its best alternatives, over rows of logits
// (the definition: include/qws.h qws_logprobs; the running sums: qws_lse.h).
//
//   k_lp_scan   R x G workgroups of 256: one pass over the logits.  Each lane keeps the running maximum and sums of its
//               elements; each given token's rank is counted by ballots; and the maximum of every 64 consecutive logits
//               (a group) goes to the workspace.  Bound by the logits' bytes in fp32 (256 rows of 248,320: 41 us, 6.1
//               TB/s), in bf16 by the vector instructions, five and a half a logit, beside them (2,048 rows: 201-209 us, 5
//               TB/s), and for few rows by one load's and one launch's latency (1 bf16 row 3.9 us, 36 fp32 rows 9.2).  With
//               several tokens by the ranks, a comparison and two scalar instructions for each logit and token (128 rows x
//               16 tokens: fp32 56 us, bf16 50, where one token a row takes 21 and 13 by the bytes at 6 TB/s).
//   k_lp_row    R workgroups of 256: joins the row's parts, writes log probabilities, ranks and entropy, and takes the
//               alternatives in two selections: the n groups with the best maxima (ties: the first), then the n best of
//               those groups' logits.  That is exact: a logit outside those groups has n better ones, the maxima of the n
//               groups (each larger, or equal and of a lower index, since groups are consecutive runs of tokens).  So the
//               pass over the logits does nothing more for 64 alternatives than for none, whatever their order in memory.
//               Bound by latency: a chain of five loads and some twenty barriers (6.4-9.2 us up to 256 rows; 2,048
//               rows, all on the card at once, 16); for alternatives near 64 by the ranking of the keys that the value
//               bounds leave (64 of one row: 48 us, of 256 rows 62).
// The join is a launch of its own: a row's last workgroup finishing it in k_lp_scan has to make every workgroup's results
// visible to other dies' caches first (256 fp32 rows 125 us with stores through the cache, 518 with a release each, against
// 53; only a single row gained, 21.8 -> 17.9).
#include "qws_lse.h"

#include <type_traits>

namespace qws {

constexpr int LP_NT = 256;      // threads
constexpr int LP_NW = LP_NT / 64;
constexpr int LP_GRP = 64;      // consecutive logits of a group
constexpr int LP_NMAX = 64;     // alternatives and given tokens of a row at most
constexpr int LP_VMAX = 1 << 19;
constexpr int LP_CUS = 256;
constexpr int LP_WGS = (int)((1ll << 32) / LP_NT - 1);  // workgroups of a launch at most: below 2^32 threads
constexpr int LP_U = 4;         // vectors of a thread loaded together, where it has more than one

template <typename T>
constexpr int lp_e() { return 16 / (int)sizeof(T); }  // elements of a vector
template <typename T>
constexpr int lp_waves(int u) { return u * lp_e<T>() > 16 ? 5 : 8; }  // waves of a SIMD that the block's registers allow
template <typename T>
constexpr int lp_stripe() { return LP_NT * lp_e<T>(); }  // elements that a workgroup's threads load at once

template <typename T>
using lp_bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

// the next larger value
__device__ __forceinline__ float lp_above(float x) {
  const int b = __float_as_int(x + 0.0f);
  return __int_as_float(b >= 0 ? b + 1 : b - 1);
}

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

// The largest of a vector; a NaN shows in the sums (lp_fast), not here
template <int E>
__device__ __forceinline__ float lp_max(const float* x) {
  float m = lse_max3(x[0], x[1], x[2]);
#pragma unroll
  for (int j = 3; j + 1 < E; j += 2) m = lse_max3(m, x[j], x[j + 1]);
  return lse_max3(m, x[E - 1], x[E - 1]);
}

// The largest of each group's lanes (8 or 16), in every lane: one instruction a step, where fmaxf of a moved value takes four.
// A lane's value is written at least two instructions before another lane's step reads it (the hardware does not wait).
template <int U, int E>
__device__ __forceinline__ void lp_group_max(float (&m)[U]) {
#define QWS_DPP(n, ctrl) "v_max_f32_dpp %" #n ", %" #n ", %" #n " " ctrl " row_mask:0xf bank_mask:0xf\n\t"
#define QWS_STEP(ctrl)                                                                                                                \
  if constexpr (U == 4)                                                                                                               \
    asm("s_nop 1\n\t" QWS_DPP(0, ctrl) QWS_DPP(1, ctrl) QWS_DPP(2, ctrl) QWS_DPP(3, ctrl) : "+v"(m[0]), "+v"(m[U / 4]), "+v"(m[U / 2]), "+v"(m[U - 1])); \
  else                                                                                                                                \
    asm("s_nop 1\n\t" QWS_DPP(0, ctrl) : "+v"(m[0]))
  static_assert(U == 1 || U == 4, "vectors of a block");
  QWS_STEP("quad_perm:[1,0,3,2]");
  QWS_STEP("quad_perm:[2,3,0,1]");
  QWS_STEP("row_half_mirror");
  if constexpr (E == 4) { QWS_STEP("row_mirror"); }
#undef QWS_STEP
#undef QWS_DPP
}

// A lane's sums over blocks of logits of moderate size (below LSE_MOST in magnitude at their largest, no -inf, no NaN),
// relative to any reference M = fl(c m) within LP_SLACK of the largest, so that M rarely moves: a multiply-add, an
// exponential and two sums per logit.  Blocks with anything else, and those that would move M to LSE_NEAR or past it, go to Lse's
// general form (lp_slow).  A lane that has seen nothing but a mask's finite value may go on to -2^31 (-1e9 at temperatures from
// 0.7 on): |r| <= 64 there, and only a row with nothing above -2^23, where fp32 logits are whole numbers, has its entropy's terms
// cancel by as much (such masks, 256 bf16 rows of 248,320: 47.5 us with lp_slow, 42.5 so).
constexpr float LP_SLACK = 8.0f;    // in log2 units: d <= 8, so the entropy's two terms cancel by 8 units at most
constexpr float LP_MASKED = -0x1p23f, LP_FAR = -0x1p31f;
struct LpFast {
  float m, M, limit, s, t;
};
template <int U, int E>
__device__ __forceinline__ bool lp_fast(LpFast& f, const float (&x)[U][E], float best, float c) {
  if (__any(best > f.limit)) {
    if (__any(best > f.limit && !(fabsf(c * best) < LSE_NEAR || (best < LP_MASKED && c * best > LP_FAR)))) return false;
    if (best > f.limit) {
      const float M = c * best, d = f.M - M, e = lse_exp2(d);
      f = {best, M, best + LP_SLACK / c, f.s * e, e * fmaf(d, f.s, f.t)};
    }
  }
  float s = f.s, t = f.t;
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < E; j++) {
      const float d = fmaf(x[u][j], c, -f.M), e = lse_exp2(d);
      s += e;
      t = fmaf(e, d, t);
    }
  if (__any(!(fabsf(t) < INFINITY))) return false;  // -inf or NaN among them
  f.s = s;
  f.t = t;
  return true;
}
__device__ __forceinline__ Lse lp_fast_end(const LpFast& f, float c) {
  if (f.m == -INFINITY) return {-INFINITY, 0.0f, 0.0f};
  return lse_exact(f.m, f.M, f.s, f.t, c);
}
template <int U, int E>
__device__ __forceinline__ void lp_slow(Lse& v, const float (&x)[U][E], float best, float c) {
  const float m = fmaxf(v.m, best), d = lse_d(v.m, m, c), e = lse_exp2(d);
  v = {m, v.s * e, e * fmaf(d, v.s, v.t)};
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < E; j++) {
      const float dj = lse_d(x[u][j], m, c), ej = lse_exp2(dj);
      v.s += ej;
      v.t = fmaf(ej, dj, v.t);
    }
}

// The selections of a row's workgroup.  A key is a value's order and its place (comp): larger = earlier.
struct LpSel {
  uint64_t col[LP_NW][64], best[64], thr;
  int rank[64], n;
  int win[64];
};
// The n-th largest (n <= 64) of the 64 lanes' best values (order keys, 0 = none), each over the lane of every wave; 0 when
// fewer lanes have one: a lower bound of the workgroup's n-th largest value.  Clears s.n; every wave gets it without a second
// barrier, by bisection over the key's bits: all 16 of a bf16 value, 20 of an fp32 one (the few more that lie within 2^-11 of the
// bound cost less than twelve more steps: 2,048 bf16 rows of 32,001 56.5 us a call with 32 steps, 52.9 so; 36 fp32 rows 22.5,
// 21.2; leaving at exactly n lanes took longer, 63).
template <typename T>
__device__ __forceinline__ uint32_t lp_bound(uint32_t mine, int n, LpSel& s) {
  uint32_t* col = (uint32_t*)s.col;
  bar();
  col[threadIdx.x] = mine;
  if (threadIdx.x == 0) s.n = 0;
  bar();
#pragma unroll
  for (int w = 0; w < LP_NW; w++) mine = max(mine, col[64 * w + lane_id()]);
  uint32_t t = 0;
#pragma unroll
  for (uint32_t bit = 0x80000000u; bit >= (sizeof(T) == 4 ? 0x1000u : 0x10000u); bit >>= 1)
    if (__popcll(__ballot(mine >= (t | bit))) >= n) t |= bit;
  return t;
}
// The same over whole keys (distinct, 0 = none): no more of them than lp_list are at or above it, however many values tie.
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
// calls put(rank, key) for every key of the list that is among its n best (after a barrier behind the list's last write)
template <typename F>
__device__ __forceinline__ void lp_ranked(LpSel& s, const uint64_t* list, int n, F put) {
  const int c = s.n, lane = lane_id(), wave = wave_id();
  if (c <= 64) {  // each wave compares the lanes' keys with a quarter of the list
    if (wave == 0) s.rank[lane] = 0;
    bar();
    const uint64_t k = lane < c ? list[lane] : 0;
    const int q = (c + LP_NW - 1) / LP_NW, hi = min((wave + 1) * q, c);
    int r = 0;
#pragma unroll 4
    for (int j = wave * q; j < hi; j++) r += list[j] > k;
    atomicAdd(&s.rank[lane], r);
    bar();
    if (wave == 0 && lane < c && s.rank[lane] < n) put(s.rank[lane], k);
    return;
  }
  for (int i = threadIdx.x; i < c; i += LP_NT) {
    const uint64_t k = list[i];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < c; j++) r += list[j] > k;
    if (r < n) put(r, k);
  }
}
// Keys that a selection of the n best can list: those of the n lanes whose best are the n largest; a lane has one of every 64
// groups, then one of each of up to 64 groups looked through.
inline size_t lp_list(int groups, int n) {
  const int a = n * ((groups + 63) / 64), b = n * 64;
  return (size_t)(a > b ? a : b);
}
__device__ __forceinline__ uint32_t lp_value(float x) { return x > -INFINITY ? okey(x) : 0; }

// RANK: 0 no given tokens' ranks, 1 one token per row (held in registers), 2 several (a lane each).  U vectors of a thread make a
// block: loaded together, one step of the running maximum.
template <typename T, int RANK, bool TOP, int U>
__global__ void __launch_bounds__(LP_NT, lp_waves<T>(U)) k_lp_scan(LpArgs a) {
  constexpr int E = lp_e<T>(), SE = lp_stripe<T>();
  __shared__ int s_cnt[LP_NMAX];
  __shared__ Lse s_lse[LP_NW];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int row = blockIdx.x / a.G, ch = blockIdx.x % a.G;
  const T* p = (const T*)a.x + (long long)row * a.stride;
  const int lead = (int)((uintptr_t)p / sizeof(T)) & (E - 1), end = lead + a.V;
  const T* base = p - lead;
  const float c = lse_scale(a.temp ? a.temp[row] : 1.0f);
  const int nstripes = (end + SE - 1) / SE, s_begin = ch * a.per, s_end = min(s_begin + a.per, nstripes);
  vu4 r[U];
  auto load = [&](int s) {
    const int first = s * SE;
    if (first >= lead && first + U * SE <= end && s + U <= s_end) {
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = __builtin_nontemporal_load((const QWS_G vu4*)(base + first + u * SE + tid * E));  // read once
    } else {  // past the row's end, or into the next workgroup's stripes: nothing
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = lp_load_edge(base, first + u * SE + tid * E, s + u < s_end ? lead : end, end);
    }
  };
  load(s_begin);  // before the given tokens' two loads in a row (36 fp32 rows 23.2 us a call, 22.7 so)
  float xt = 0.0f;  // the given token's logit; with several, lane m's is token m's
  int tv = -1, cnt = 0;  // its place (-1: skipped), logits before it
  bool moderate = c <= LSE_MOST;  // no given token's logit is extreme
  if constexpr (RANK == 1) {
    const int t = a.tok[row];
    if (t >= 0 && t < a.V) {
      tv = t + lead;
      xt = lp_one(p + t);
      moderate = moderate && fabsf(xt) < LSE_MOST;
    }
  }
  if constexpr (RANK == 2) {
    const int t = lane < a.M ? a.tok[(long long)row * a.M + lane] : -1;
    if (t >= 0 && t < a.V) {
      tv = t + lead;
      xt = lp_one(p + t);
    }
    moderate = moderate && __all(fabsf(xt) < LSE_MOST);
  }
  Lse v = {-INFINITY, 0.0f, 0.0f};
  LpFast f = {-INFINITY, -1e30f, -INFINITY, 0.0f, 0.0f};
  char* gmax = (char*)(a.gmax + (long long)row * a.groups);
  for (int s = s_begin; s < s_end; s += U) {
    const int first = s * SE;
    float top[U];
    float x[U][E], best = -INFINITY, least = INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
      lp_unpack<T>(r[u], x[u]);
      top[u] = lp_max<E>(x[u]);
      best = fmaxf(best, top[u]);
      least = fminf(least, top[u]);
    }
    if (!(moderate && __all(best < LSE_MOST && least > -LSE_MOST)) || !lp_fast(f, x, best, c)) {
      bool unclean = best == INFINITY;  // or a NaN: else the values and their largest are right as they are
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < E; j += 2) unclean = unclean || __builtin_isunordered(x[u][j], x[u][j + 1]);
      if (__any(unclean)) {
        best = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
          top[u] = -INFINITY;
#pragma unroll
          for (int j = 0; j < E; j++) {
            x[u][j] = lse_clean(x[u][j]);
            top[u] = fmaxf(top[u], x[u][j]);
          }
          best = fmaxf(best, top[u]);
        }
      }
      lp_slow(v, x, best, c);
    }
    if constexpr (TOP) {
      lp_group_max<U, E>(top);
#pragma unroll
      for (int u = 0; u < U; u++)  // byte offsets in 32 bits: one address register for all
        if ((lane & (LP_GRP / E - 1)) == 0 && s + u < s_end) *(float*)(gmax + (unsigned)((first + u * SE + tid * E) / LP_GRP * 4)) = top[u];
    }
    // Before a token: the logits at or above its own in places before it, the larger ones behind it.  A wave's 64 E places lie
    // on one side of almost every token: one comparison a logit.
    if constexpr (RANK == 1) {
      if (__any(best >= xt)) {  // else a likely token: nothing here is before it
#pragma unroll
        for (int u = 0; u < U; u++) {
          // this wave's elements: [lo, lo + 64 E); a stripe of the next workgroup lies behind every token
          const int lo = s + u < s_end ? first + u * SE + wave * 64 * E : 0x7FFFFFFF - 64 * E;
          if (lo + 64 * E <= tv) {
#pragma unroll
            for (int j = 0; j < E; j++) cnt += __popcll(__ballot(x[u][j] >= xt));
          } else if (lo > tv) {
#pragma unroll
            for (int j = 0; j < E; j++) cnt += __popcll(__ballot(x[u][j] > xt));
          } else {
#pragma unroll
            for (int j = 0; j < E; j++) cnt += __popcll(__ballot(x[u][j] > xt || (x[u][j] == xt && lo + lane * E + j < tv)));
          }
        }
      }
    }
    if constexpr (RANK == 2) {  // without branches, a bound for each side; a token that is among them has its equals added
      float bound[U];
      int lo[U];
      bool among = false;
#pragma unroll
      for (int u = 0; u < U; u++) {
        lo[u] = s + u < s_end ? first + u * SE + wave * 64 * E : 0x7FFFFFFF - 64 * E;
        bound[u] = lo[u] + 64 * E <= tv ? xt : lp_above(xt);
        among = among || (tv >= lo[u] && tv < lo[u] + 64 * E);
      }
      uint64_t left = __ballot(among);
#pragma unroll 2
      for (int k = 0; k < a.M; k++) {
        int n = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
          const float b = readlane<float>(bound[u], k);
#pragma unroll
          for (int j = 0; j < E; j++) n += __popcll(__ballot(x[u][j] >= b));
        }
        cnt += lane == k ? n : 0;
      }
      for (; left; left &= left - 1) {
        const int k = __ffsll((long long)left) - 1, tk = readlane<int>(tv, k);
        const float xk = readlane<float>(xt, k);
        int n = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
          if (tk >= lo[u] && tk < lo[u] + 64 * E)
#pragma unroll
            for (int j = 0; j < E; j++) n += __popcll(__ballot(x[u][j] == xk && lo[u] + lane * E + j < tk));
        cnt += lane == k ? n : 0;
      }
    }
    if constexpr (U != 1)
      if (s + U < s_end) load(s + U);  // here, not before the sums: a second block in registers costs waves (bf16 219 -> 273 us)
  }
  v = lse_join_wave(lse_join(v, lp_fast_end(f, c), c), c);
  if constexpr (RANK != 0) {
    const int n = RANK == 1 ? 1 : a.M;
    if (tid < n) s_cnt[tid] = 0;
    bar();
    if (lane < n) atomicAdd(&s_cnt[lane], cnt);
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

// A row's second stage: joins its parts, writes the given tokens' results and the entropy, and selects the
// alternatives.  Both selections first take the values at or above lp_bound, which are few where values differ: up to 64
// groups are all looked through, whether among the n best or not, and up to 64 logits are ranked.  Where more are (ties, or
// n near 64), keys with their places decide.
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_NT) k_lp_row(LpArgs a) {
  __shared__ LpSel s;
  __shared__ Lse s_lse[LP_NW];
  __shared__ int s_cnt[LP_NMAX];
  extern __shared__ uint64_t list[];  // lp_list(groups, top) keys
  constexpr int E = lp_e<T>(), KPT = 16;  // groups of a thread that are held in registers: all, up to V = 262,144
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), row = blockIdx.x;
  const T* p = (const T*)a.x + (long long)row * a.stride;
  const int lead = (int)((uintptr_t)p / sizeof(T)) & (E - 1), end = lead + a.V;
  const int ng = (end + LP_GRP - 1) / LP_GRP;
  const float* gm = a.gmax + (long long)row * a.groups;
  float gv[TOP ? KPT : 1];
  auto load_groups = [&](int g0) {
#pragma unroll
    for (int i = 0; i < KPT; i++) {
      const int g = g0 + i * LP_NT + tid;
      const float x = *gmem(gm + min(g, ng - 1));
      gv[i] = g < ng ? x : -INFINITY;
    }
  };
  if constexpr (TOP) load_groups(0);
  const float temp = a.temp ? a.temp[row] : 1.0f, c = lse_scale(temp);
  // thread m has given token m; the parts of its count are spread over all threads
  bool ok = false;
  float xt = 0.0f;
  if (tid < a.M) {
    const int t = a.tok[(long long)row * a.M + tid];
    ok = t >= 0 && t < a.V;
    if (ok) xt = lp_one(p + t);
    s_cnt[tid] = 0;
  }
  int cnt = 0;
  if (a.M && a.out_rank) {
    const int parts = LP_NT / a.M;
    if (tid < parts * a.M)
      for (int g = tid / a.M; g < a.G; g += parts) cnt += a.cnt[((long long)row * a.G + g) * a.M + tid % a.M];
  }
  Lse v = {-INFINITY, 0.0f, 0.0f};
  for (int g = tid; g < a.G; g += LP_NT) {
    const float4 q = a.part[(long long)row * a.G + g];
    v = lse_join(v, {q.x, q.y, q.z}, c);
  }
  v = lse_join_wave(v, c);
  if (lane == 0) s_lse[wave] = v;
  bar();
  if (cnt) atomicAdd(&s_cnt[tid % a.M], cnt);
  v = s_lse[0];
#pragma unroll
  for (int w = 1; w < LP_NW; w++) v = lse_join(v, s_lse[w], c);
  bar();
  if (tid == 0 && a.out_h) a.out_h[row] = lse_entropy(v);
  if (tid < a.M) {
    const long long o = (long long)row * a.M + tid;
    if (ok) {
      const int places = xt == -INFINITY ? lead : 0;  // before the row: they were counted as -inf of lower indices
      a.out_lp[o] = lse_logprob(v, xt, temp);
      if (a.out_rank) a.out_rank[o] = s_cnt[tid] - places;
    } else {
      a.out_lp[o] = 0.0f;
      if (a.out_rank) a.out_rank[o] = -1;
    }
  }
  if constexpr (TOP) {
    const int n = a.top;
    const bool held = ng <= KPT * LP_NT;
    auto chunks = [&](auto f) {  // f(first group) with gv loaded, over the row
      for (int g0 = 0; g0 < ng; g0 += KPT * LP_NT) {
        if (!held) load_groups(g0);
        f(g0);
      }
    };
    float best = -INFINITY;
    chunks([&](int) {
#pragma unroll
      for (int i = 0; i < KPT; i += 2) best = lse_max3(best, gv[i], gv[i + 1]);
    });
    const uint32_t bound = max(lp_bound<T>(lp_value(best), n, s), KEY_NEGINF + 1);
    const float least = okey_val(bound);
    chunks([&](int g0) {
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < KPT; i++) mine |= gv[i] >= least ? 1u << i : 0u;
      if (mine) {
        int at = atomicAdd(&s.n, __popc(mine));
        for (; mine; mine &= mine - 1, at++)
          if (at < 64) s.win[at] = g0 + (__ffs(mine) - 1) * LP_NT + tid;
      }
    });
    bar();
    int nw = s.n;
    if (nw > 64) {
      auto key = [&](int g0, int i) { return gv[i] > -INFINITY ? comp(okey(gv[i]), (uint32_t)(g0 + i * LP_NT + tid)) : 0; };
      uint64_t top = 0;
      chunks([&](int g0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) top = max(top, key(g0, i));
      });
      const uint64_t thr = lp_threshold(top, n, s);
      chunks([&](int g0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) lp_take(key(g0, i), thr, s, list);
      });
      bar();
      lp_ranked(s, list, n, [&](int r, uint64_t k) { s.win[r] = (int)comp_idx(k); });
      nw = min(s.n, n);
      bar();
    }
    // the groups' logits: lane l takes place l of every fourth group
    constexpr int PER = 64 / LP_NW;
    const int mine = s.win[min(lane * LP_NW + wave, 63)];  // this wave's groups, by lanes
    auto place = [&](int i) { return __builtin_amdgcn_readlane(mine, i) * LP_GRP + lane - lead; };
    float x[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
      x[i] = -INFINITY;
      if (i * LP_NW + wave < nw) x[i] = lp_one(p + min(max(place(i), 0), a.V - 1));
    }
    best = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      if (i * LP_NW + wave < nw && (place(i) < 0 || place(i) >= a.V)) x[i] = -INFINITY;
      best = fmaxf(best, x[i]);
    }
    const float low = okey_val(max(lp_bound<T>(lp_value(best), n, s), KEY_NEGINF + 1));
    {
      uint32_t took = 0;
#pragma unroll
      for (int i = 0; i < PER; i++) took |= x[i] >= low ? 1u << i : 0u;
      if (took) {
        int at = atomicAdd(&s.n, __popc(took));
        for (; took; took &= took - 1, at++)
          if (at < 64) {
            const int e = s.win[(__ffs(took) - 1) * LP_NW + wave] * LP_GRP + lane - lead;
            list[at] = comp(okey(lp_one(p + e)), (uint32_t)e);
          }
      }
    }
    bar();
    if (s.n > 64) {
      auto key = [&](int i) { return x[i] > -INFINITY ? comp(okey(x[i]), (uint32_t)place(i)) : 0; };
      uint64_t top = 0;
#pragma unroll
      for (int i = 0; i < PER; i++) top = max(top, key(i));
      const uint64_t thr = lp_threshold(top, n, s);
#pragma unroll
      for (int i = 0; i < PER; i++) lp_take(key(i), thr, s, list);
      bar();
    }
    int* ids = a.out_ids + (long long)row * n;
    float* lps = a.out_top + (long long)row * n;
    lp_ranked(s, list, n, [&](int r, uint64_t k) {
      ids[r] = (int)comp_idx(k);
      lps[r] = lse_logprob(v, okey_val(comp_key(k)), temp);
    });
    for (int r = s.n + tid; r < n; r += LP_NT) {
      ids[r] = -1;
      lps[r] = -INFINITY;
    }
  }
}

struct LpPlan {
  int G, per, groups;
  size_t part, cnt, gmax, total;  // byte offsets
  bool fits(int R) const { return (long long)R * G <= LP_WGS; }
};
// Stripes of a workgroup: one while the card holds them all at once; then four (a block), eight, and as many as leave eight
// rounds of workgroups, so that the last round is a small part (2,048 bf16 rows of 248,320: 257 us with one round of whole
// rows, 229 with eight; 256 fp32 rows: 60 and 57; 36 rows, one stripe each: 35, eight: 25).
template <typename T>
LpPlan lp_plan(int R, int V, int M, int top) {
  LpPlan q;
  const int stripes = (V + lp_e<T>() - 1 + lp_stripe<T>() - 1) / lp_stripe<T>();
  const long long all = (long long)R * stripes, fill = LP_CUS * lp_waves<T>(LP_U);  // fill: workgroups of four waves held at once
  const long long rounds = (all + 8 * fill - 1) / (8 * fill), few = (stripes + LP_U - 1) / LP_U * LP_U;
  const long long per = all <= fill || stripes == 1 ? 1 : all <= 4 * fill ? LP_U : rounds <= 2 * LP_U ? 2 * LP_U : (rounds + LP_U - 1) / LP_U * LP_U;
  q.per = (int)(per > few ? few : per);
  q.G = (stripes + q.per - 1) / q.per;
  q.groups = top ? stripes * (lp_stripe<T>() / LP_GRP) : 0;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  q.part = 0;
  q.cnt = up((size_t)R * q.G * sizeof(float4));
  q.gmax = q.cnt + up((size_t)R * q.G * M * sizeof(int));
  q.total = q.gmax + up((size_t)R * q.groups * sizeof(float));
  return q;
}

template <typename T, int RANK, bool TOP>
void lp_launch_scan(const LpArgs& a, int R, hipStream_t st) {
  if (a.per == 1)
    hipLaunchKernelGGL((k_lp_scan<T, RANK, TOP, 1>), dim3((unsigned)R * a.G), dim3(LP_NT), 0, st, a);
  else
    hipLaunchKernelGGL((k_lp_scan<T, RANK, TOP, LP_U>), dim3((unsigned)R * a.G), dim3(LP_NT), 0, st, a);
}
template <typename T, bool TOP>
void lp_launch_scan(const LpArgs& a, int R, hipStream_t st) {
  if (!a.M || !a.out_rank)
    lp_launch_scan<T, 0, TOP>(a, R, st);
  else if (a.M == 1)
    lp_launch_scan<T, 1, TOP>(a, R, st);
  else
    lp_launch_scan<T, 2, TOP>(a, R, st);
}
template <typename T>
int lp_launch(LpArgs a, int R, char* ws, size_t ws_bytes, hipStream_t st) {
  const LpPlan q = lp_plan<T>(R, a.V, a.M, a.top);
  if (!q.fits(R)) return QWS_ERR_NOT_SUPPORTED;
  if (ws_bytes < q.total) return QWS_ERR_INVALID;
  a.G = q.G;
  a.per = q.per;
  a.groups = q.groups;
  a.part = (float4*)(ws + q.part);
  a.cnt = (int*)(ws + q.cnt);
  a.gmax = (float*)(ws + q.gmax);
  const size_t lds = a.top ? sizeof(uint64_t) * lp_list(q.groups, a.top) : 0;
  if (a.top)
    lp_launch_scan<T, true>(a, R, st);
  else
    lp_launch_scan<T, false>(a, R, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (a.top)
    hipLaunchKernelGGL((k_lp_row<T, true>), dim3(R), dim3(LP_NT), lds, st, a);
  else
    hipLaunchKernelGGL((k_lp_row<T, false>), dim3(R), dim3(LP_NT), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace qws

static_assert(sizeof(qws_logprobs_batch) == 96 && offsetof(qws_logprobs_batch, tokens) == 32 && offsetof(qws_logprobs_batch, out_top_logprobs) == 88,
              "qws_logprobs_batch layout (the ctypes binding's)");

extern "C" size_t qws_logprobs_ws_bytes(int dtype, int R, int V, int M, int top) {
  using namespace qws;
  if (R < 1 || V < 1 || V > LP_VMAX || M < 0 || M > LP_NMAX || top < 0 || top > LP_NMAX) return 0;
  if (dtype != QWS_DTYPE_F32 && dtype != QWS_DTYPE_BF16) return 0;
  const LpPlan q = dtype == QWS_DTYPE_F32 ? lp_plan<float>(R, V, M, top) : lp_plan<uint16_t>(R, V, M, top);
  return q.fits(R) ? q.total : 0;
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
