// Routing of tokens to experts: from a row of router logits to the chosen
// experts and their weights, the step before moe_align / moe_gemm, and its
// gradient.
//
//   s = softmax(x) or sigmoid(x)           (over the E experts of a row)
//   c = s + bias                           (bias steers the choice only)
//   keep the topk_groups groups with the largest sum of their group_top best c
//   choose the topk largest c of them, largest first, ties to the lowest index
//   w = scale * s[chosen]                  (renorm: divided by the sum of the chosen s)
//
// An expert whose logit is -inf or NaN, or whose c is, cannot be chosen; a
// place that no expert is left for gets id -1 and weight 0.
//
// The choice is the one of Float64. Without a bias the experts of a row rank as
// their logits do, which needs no arithmetic. With a bias, and between groups, c
// is computed in 32 bits first; where two values that decide the order are
// closer than those 32 bits tell apart, the candidates, or where groups are in
// doubt the whole row, are ranked again in 64 bits (where those cannot tell them
// apart either, as sigmoids of 40 and 50, it is a tie). How often that happens
// is up to the inputs: for 8 of 256 experts by sigmoid, one row in 2000 for f32
// logits of deviation 1.5 under a bias of deviation 0.1; under a zero bias a third
// of the rows for the same logits in bf16, half of them for f32 logits of
// deviation 5, and every row for deviation 8, whose sigmoids saturate.
//
// A row belongs to LANES lanes of a warp, NV neighbouring experts to a lane, so
// that a tie goes to the first lane and the first register. Each choice is one
// maximum over the lanes and a rescan of the winner's NV registers. Rows of up
// to 64 experts take 8 lanes (four rows per warp).
//
// Bound by instruction issue (IPC 2.7), not by HBM: 65536 x 256 f32 takes 40
// us without a bias and 61 with bias and groups (840 instructions a row) against
// 10 at the copy rate; 16384 rows 12 and 17 to 18. The 64-bit ranking shows: 16384 x
// 256 with 4 of 8 groups and a zero bias takes 17 us for logits of deviation 1.5
// (24 in bf16), 26 for 5, 55 for 8; by softmax 21, 26 and 46, and 42 for 0.05.
#include "ctb_common.cuh"

#include <algorithm>

namespace ctb {
namespace {

constexpr int ROUTE_THREADS = 128;
constexpr int ROUTE_MAX_EXPERTS = 256;
constexpr int ROUTE_MAX_TOPK = 32;
constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A run of up to 16 bytes of T.
template <int BYTES> struct Raw;
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };

// NV neighbouring values of a row, as vectors of at most 16 bytes where VEC.
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void load_run(const T* p, int i0, int E, float pad,
                                         float (&v)[NV]) {
  if (VEC) {
    constexpr int W = NV * (int)sizeof(T) < 16 ? NV : 16 / (int)sizeof(T);
    using R = typename Raw<W * (int)sizeof(T)>::type;
#pragma unroll
    for (int c = 0; c < NV; c += W) {
      if (i0 < E) {  // E is a multiple of NV on this path
        union {
          R raw;
          T e[W];
        } u;
        u.raw = *reinterpret_cast<const R*>(p + i0 + c);
#pragma unroll
        for (int i = 0; i < W; ++i) v[c + i] = to_float(u.e[i]);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[c + i] = pad;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = i0 + i < E ? to_float(p[i0 + i]) : pad;
  }
}
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void store_run(T* p, int i0, int E, const float (&v)[NV]) {
  if (VEC) {
    constexpr int W = NV * (int)sizeof(T) < 16 ? NV : 16 / (int)sizeof(T);
    using R = typename Raw<W * (int)sizeof(T)>::type;
    if (i0 < E) {
#pragma unroll
      for (int c = 0; c < NV; c += W) {
        union {
          R raw;
          T e[W];
        } u;
#pragma unroll
        for (int i = 0; i < W; ++i) store_as(&u.e[i], v[c + i]);
        *reinterpret_cast<R*>(p + i0 + c) = u.raw;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i0 + i < E) store_as(&p[i0 + i], v[i]);
  }
}

// ---- reductions over the LANES lanes of a row ------------------------------------
template <int LANES>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
template <int LANES, typename S>
__device__ __forceinline__ S row_sum(S v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// ---- order-preserving keys ----------------------------------------------------------
// Adding +0 first makes -0 and +0 the same key. The key of -inf, and 0, stand
// for "not available" (is_live); NaN has no key.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ (uint32_t)((int32_t)u >> 31 | 0x80000000);
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kNone32 = 0x007fffffu;              // key_of(-inf)
constexpr uint64_t kNone64 = 0x000fffffffffffffull;
__device__ __forceinline__ bool is_live(uint32_t k) { return k > kNone32; }
__device__ __forceinline__ bool is_live(uint64_t k) { return k > kNone64; }
template <typename S> struct KeyOf;
template <> struct KeyOf<float> { using type = uint32_t; };
template <> struct KeyOf<double> { using type = uint64_t; };

template <int LANES>
__device__ __forceinline__ uint32_t row_max_key(uint32_t v) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(FULL, v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(FULL, v, o));
    return v;
  }
}
template <int LANES>
__device__ __forceinline__ uint64_t row_max_key(uint64_t v) {
  if constexpr (LANES == 32) {  // the high words' maximum, then the low words' among those
    const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      const uint64_t w = __shfl_xor_sync(FULL, v, o);
      v = w > v ? w : v;
    }
    return v;
  }
}

struct RouteArgs {
  const float* bias;
  float* weights;
  int32_t* ids;
  int T, E, topk;
  int64_t ldx;
  int sigmoid, groups, topk_groups, group_top, renorm;
  int group_size;   // experts per group
  int group_lanes;  // lanes per group where that is a power of two of whole lanes, else 0
  float pair_error; // of the scores of two experts of a row together
  bool bias_runs;   // the bias is made of whole runs of NV floats, 16-byte aligned
  float scale;
};

// The fast exponential and reciprocal: 2 and 1 ulp, results below the normal
// range become 0.
__device__ __forceinline__ float ex2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Whether two choice values hi >= lo are too close for 32 bits to order them.
// 2^(d log2 e) carries at most 2.4e-7 (ex2.approx) + 2e-7 |d| (the roundings of
// d, of log2 e and of their product) relative error. Of a sigmoid that is s (1 -
// s) times as much, at most 7e-8, and its sum and reciprocal add 1.8e-7: 2.5e-7
// each, 6e-7 the two of a pair, 1.2e-6 the four of two groups. Of a softmax the
// row's sum (its terms' errors weighted, 8 levels of additions) adds at most
// 2e-6, reciprocal and product 2.4e-7; a row's scores add up to at most 1, so two
// or four of them err by at most 4e-6 together. Each addition (of a bias, of a
// group's two) adds 2^-24 of its result: 1e-7 of the magnitudes of a pair, 3e-7
// of the largest group's. Without a bias the error is relative, |ln hi| standing
// for |d|; sums so small that 32 bits lose them are never certain.
__device__ __forceinline__ bool too_close(float hi, float lo, float error) {
  return !(hi - lo > error);
}
__device__ __forceinline__ bool too_close_unbiased(float hi, float lo) {
  return !(hi > 1e-30f && hi - lo > 2.f * hi * (4e-6f + 2.5e-7f * fabsf(__logf(hi))));
}

// Whether the order between the kept groups (`in`) and the others is too close
// for 32 bits; each lane holds a group's score and the magnitude of its terms.
__device__ __forceinline__ bool groups_close(const RouteArgs& a, bool counts, bool in, float score,
                                             float magnitude) {
  const uint32_t k = key_of(score);
  const float lo = value_of(__reduce_min_sync(FULL, counts && in ? k : 0xffffffffu));
  const float hi = value_of(__reduce_max_sync(FULL, counts && !in ? k : kNone32));
  const float mag = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(magnitude)));
  // A group without an expert (-inf) is not in doubt.
  return hi > -INFINITY &&
         (a.bias ? too_close(lo, hi, (a.sigmoid ? 1.2e-6f : 4e-6f) + 3e-7f * mag)
                 : too_close_unbiased(lo, hi));
}

// Keys of the experts outside the best topk_groups groups become 0 (c is -inf
// where an expert is not available); returns whether the choice between groups
// was too close for 32 bits. LANES == 32.
template <typename S, int NV>
__device__ __forceinline__ bool keep_groups(const RouteArgs& a, const S (&c)[NV],
                                            typename KeyOf<S>::type (&key)[NV], S* row) {
  const int lane = threadIdx.x & 31, size = a.group_size;
  const S none = -INFINITY;
  S best = none, second = none;
  if (a.group_lanes > 0) {
    // A power of two of whole lanes per group: the two best of a lane's
    // registers, then of neighbours, so that every lane of a group knows its
    // score. Its rank among the groups is counted by the group's lanes together.
    const int span = a.group_lanes, part = lane & (span - 1), first = lane - part;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      second = max(second, min(best, c[v]));
      best = max(best, c[v]);
    }
    for (int o = 1; o < span; o <<= 1) {
      const S b = __shfl_xor_sync(FULL, best, o), s = __shfl_xor_sync(FULL, second, o);
      second = max(max(second, s), min(best, b));
      best = max(best, b);
    }
    const S score = a.group_top > 1 && second > none ? best + second : best;
    const bool counts = first < a.groups * span;  // lanes past the last expert have no group
    int rank = 0;
    for (int i = 0; i < a.groups; i += span) {
      const int from = (i + part) * span;  // a lane of group i + part
      const S o = __shfl_sync(FULL, score, min(from, 31));
      rank += i + part < a.groups && (o > score || (o == score && from < first));
    }
    for (int o = 1; o < span; o <<= 1) rank += __shfl_xor_sync(FULL, rank, o);
    const bool in = rank < a.topk_groups;
    if (!in) {
#pragma unroll
      for (int v = 0; v < NV; ++v) key[v] = 0;
    }
    if (sizeof(S) != 4) return false;
    const float magnitude = !counts || !(best > none) ? 0.f
                            : fabsf((float)best) + (second > none ? fabsf((float)second) : 0.f);
    return groups_close(a, counts, in, (float)score, magnitude);
  }
  // Through shared memory, a lane per group; one word in 32 is skipped so that
  // lanes that start a multiple of 32 apart use different banks.
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = lane * NV + v;
    if (i < a.E) row[i + (i >> 5)] = c[v];
  }
  __syncwarp();
  if (lane < a.groups)
    for (int i = lane * size; i < (lane + 1) * size; ++i) {
      const S x = row[i + (i >> 5)];
      second = max(second, min(best, x));
      best = max(best, x);
    }
  __syncwarp();
  const S score = a.group_top > 1 && second > none ? best + second : best;
  int rank = 0;
  for (int g = 0; g < a.groups; ++g) {
    const S o = __shfl_sync(FULL, score, g);
    rank += o > score || (o == score && g < lane);
  }
  const bool counts = lane < a.groups, in = counts && rank < a.topk_groups;
  const unsigned kept = __ballot_sync(FULL, in);
  int g = lane * NV / size, at = lane * NV - g * size;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (lane * NV + v < a.E && !(kept >> g & 1u)) key[v] = 0;
    if (++at == size) {
      at = 0;
      ++g;
    }
  }
  if (sizeof(S) != 4) return false;
  const float magnitude = !counts || !(best > none) ? 0.f
                          : fabsf((float)best) + (second > none ? fabsf((float)second) : 0.f);
  return groups_close(a, counts, in, (float)score, magnitude);
}

// The chosen experts of a row, largest first, and their keys; one place more
// than topk where neighbours are to be checked.
struct Chosen {
  int id[ROUTE_MAX_TOPK + 1];
  uint32_t key[ROUTE_MAX_TOPK + 1];  // of the 32-bit choice
  int candidates;                    // how many the choice was made from; -1: all experts
};

// Fills row->id[0..rounds), -1 where no expert is left, and row->key for 32-bit keys.
//
// A whole warp's row with 32-bit keys: the rounds-th largest of the lanes' best
// is a bound that at least `rounds` experts reach and few others do (12 of 256
// for the best 8 of random scores); those candidates move to one lane each, and
// a lane's rank among them is its place. 160 instructions for 8 of 256, against
// 450 for choosing one after the other, which is left for rows with more than
// 32 candidates, for narrower rows and for 64 bits. `slack` lowers the bound so
// that whatever 64 bits could choose instead is a candidate too. There a lane knows its two
// best, so that it looks through its registers again only when it has been
// chosen from twice.
template <typename K, int LANES, int NV>
__device__ __forceinline__ void choose(K (&key)[NV], Chosen* row, uint64_t* cand, int rounds,
                                       float slack) {
  const int lane = threadIdx.x & 31, sub = lane % LANES, base = lane - sub;
  if constexpr (LANES == 32 && sizeof(K) == 4) {
    uint32_t t = key[0], bound = 0;
#pragma unroll
    for (int v = 1; v < NV; ++v) t = max(t, key[v]);
#pragma unroll 4
    for (int j = 0; j < rounds; ++j) {
      bound = __reduce_max_sync(FULL, t);
      if (t == bound) t = 0;
    }
    bound = max(bound, kNone32 + 1);
    if (slack > 0.f && bound > kNone32 + 1) {
      const float b = value_of(bound);
      if (b < INFINITY) bound = max(key_of(b - (slack + 2e-7f * fabsf(b))), kNone32 + 1);
    }
    int total = 0, at[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const unsigned b = __ballot_sync(FULL, key[v] >= bound);
      at[v] = total + __popc(b & ((1u << lane) - 1u));
      total += __popc(b);
    }
    if (total <= 32) {
      cand[lane] = 0;
      __syncwarp();
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (key[v] >= bound) cand[at[v]] = (uint64_t)key[v] << 32 | (uint32_t)~(lane * NV + v);
      __syncwarp();
      const uint64_t mine = cand[lane];
      int place = 0;
      for (int i = 0; i < total; i += 4) {  // zeros after the last are never above
        const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(cand + i);
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(cand + i + 2);
        place += (p.x > mine) + (p.y > mine) + (q.x > mine) + (q.y > mine);
      }
      if (lane >= total) place = lane;  // places that no expert is left for
      if (place < rounds) {
        row->id[place] = mine ? (int)~(uint32_t)mine : -1;
        row->key[place] = (uint32_t)(mine >> 32);
      }
      if (lane == 0) {
        if (rounds > 32) row->key[32] = 0;
        row->candidates = total;
      }
      __syncwarp();
      return;
    }
    if (lane == 0) row->candidates = -1;
  }
  K k1 = 0, k2 = 0;
  int v1 = 0, v2 = 0;
  bool two = true;  // (k2, v2) is the second best still
  auto scan = [&] {
    k1 = k2 = 0;
    v1 = v2 = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const K k = key[v];
      if (k > k1) {
        k2 = k1;
        v2 = v1;
        k1 = k;
        v1 = v;
      } else if (k > k2) {
        k2 = k;
        v2 = v;
      }
    }
  };
  scan();
  unsigned taken = 0;
  for (int j = 0; j < rounds; ++j) {
    const K m = row_max_key<LANES>(k1);
    const unsigned who = __ballot_sync(FULL, k1 == m) >> base;
    const int win = __ffs(LANES == 32 ? who : who & ((1u << (LANES & 31)) - 1u)) - 1;
    if (sub == win) {
      row->id[j] = is_live(m) ? sub * NV + v1 : -1;
      if (sizeof(K) == 4) row->key[j] = is_live(m) ? (uint32_t)m : 0u;
      taken |= 1u << v1;
      if (two) {
        k1 = k2;
        v1 = v2;
        two = false;
      } else {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          if (taken >> v & 1u) key[v] = 0;
        scan();
        two = true;
      }
    }
  }
  __syncwarp();
}

// Whether two neighbours in the order (the first one left out included) are
// too close.
template <int LANES>
__device__ __forceinline__ bool neighbours_close(const RouteArgs& a, const Chosen* row) {
  bool close = false;
  for (int j = threadIdx.x % LANES; j < a.topk; j += LANES) {
    const uint32_t hi = row->key[j], lo = row->key[j + 1];
    if (lo) {
      const float x = value_of(hi), y = value_of(lo);
      close |= too_close(x, y, a.pair_error + 1e-7f * (fabsf(x) + fabsf(y)));
    }
  }
  return close;
}

// The same row ranked in 64 bits. The loops with an exponential stay rolled: the
// code is rarely run, so its length (instruction misses) is most of its time.
template <typename T, int LANES, int NV, bool GROUPED>
__device__ __noinline__ void choose_exact(const RouteArgs& a, const T* x, int i0,
                                          bool in_range, Chosen* sel, double* row) {
  double c[NV];
  uint64_t key[NV];
  double top = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    c[v] = in_range && i0 + v < a.E ? (double)to_float(x[i0 + v]) : -INFINITY;
    if (isnan(c[v])) c[v] = -INFINITY;
    top = max(top, c[v]);
  }
  double total = 1.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(FULL, top, o));
    if (top == -INFINITY) top = 0.0;
    total = 0.0;
#pragma unroll 1
    for (int v = 0; v < NV; ++v) total += exp(c[v] - top);
    total = row_sum<LANES>(total);
  }
#pragma unroll 1
  for (int v = 0; v < NV; ++v) {
    const double xv = c[v];
    const double e = exp(a.sigmoid ? -xv : xv - top);
    const double s = (a.sigmoid ? 1.0 : e) / (a.sigmoid ? 1.0 + e : total);
    c[v] = a.bias && i0 + v < a.E ? s + (double)a.bias[i0 + v] : s;
    if (!(xv > -INFINITY && c[v] > -INFINITY)) c[v] = -INFINITY;
    key[v] = key_of(a.bias || !(c[v] > -INFINITY) ? c[v] : xv);
  }
  if (GROUPED) keep_groups<double, NV>(a, c, key, row);
  choose<uint64_t, LANES, NV>(key, sel, nullptr, a.topk, 0.f);
}

// The candidates of a whole warp's row ranked again in 64 bits, one to a lane.
template <typename T, int NV>
__device__ __noinline__ void rank_exact(const RouteArgs& a, const T* x, int i0, float top,
                                        Chosen* sel, uint64_t* cand) {
  const int lane = threadIdx.x & 31, total = sel->candidates;
  const int id = lane < total ? (int)~(uint32_t)cand[lane] : 0;
  double sum = 1.0;
  if (!a.sigmoid) {
    sum = 0.0;
#pragma unroll 1
    for (int v = 0; v < NV; ++v) {
      const double xv = i0 + v < a.E ? (double)to_float(x[i0 + v]) : -INFINITY;
      sum += isnan(xv) ? 0.0 : exp(xv - (double)top);
    }
    sum = row_sum<32>(sum);
  }
  const double xv = (double)to_float(x[id]);
  const double e = exp(a.sigmoid ? -xv : xv - (double)top);
  const double s = (a.sigmoid ? 1.0 : e) / (a.sigmoid ? 1.0 + e : sum);
  const uint64_t mine = key_of(s + (double)a.bias[id]);
  __syncwarp();
  cand[lane] = mine;
  __syncwarp();
  int place = 0;
  for (int i = 0; i < total; ++i) {
    const int other = __shfl_sync(FULL, id, i);
    place += cand[i] > mine || (cand[i] == mine && other < id);
  }
  if (lane < total && place < a.topk) sel->id[place] = id;
  __syncwarp();
}

template <typename T, int LANES, int NV, bool VEC, bool GROUPED>
__global__ void __launch_bounds__(ROUTE_THREADS) moe_route_kernel(const T* x,
                                                                  const RouteArgs a) {
  constexpr int ROWS = ROUTE_THREADS / LANES;
  constexpr int SLOTS = ROUTE_MAX_TOPK / LANES;  // places of a row per lane
  __shared__ Chosen sel_all[ROWS];
  __shared__ __align__(16) uint64_t cand[LANES == 32 ? ROUTE_THREADS / 32 : 1][LANES == 32 ? 32 : 1];
  __shared__ double scratch[GROUPED ? ROUTE_THREADS / 32 : 1]
                           [GROUPED ? ROUTE_MAX_EXPERTS + ROUTE_MAX_EXPERTS / 32 : 1];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, sub = lane % LANES, r = threadIdx.x / LANES;
  const int64_t t = (int64_t)blockIdx.x * ROWS + r;
  const bool in_range = t < a.T;
  const T* xr = x + (in_range ? t : 0) * a.ldx;
  Chosen* sel = &sel_all[r];
  const int i0 = sub * NV;

  float xv[NV];
  load_run<T, NV, VEC>(xr, i0, in_range ? a.E : 0, -INFINITY, xv);
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    xv[v] = fmaxf(xv[v], -INFINITY);  // NaN becomes -inf
    top = fmaxf(top, xv[v]);
  }
  // Softmax over the row, where the choice or the weights need it.
  float total = 1.f;
  const bool scores = a.bias != nullptr || GROUPED;
  if (!a.sigmoid && (scores || !a.renorm)) {
    top = row_max<LANES>(top);
    if (top == -INFINITY) top = 0.f;
    total = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) total += ex2_fast(kLog2e * (xv[v] - top));
    total = row_sum<LANES>(total);
  }
  const float scale_of = rcp_fast(total);
  float c[NV], bias[NV];
  uint32_t key[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) bias[v] = 0.f;
  if (a.bias) {
    if (a.bias_runs) load_run<float, NV, true>(a.bias, i0, a.E, 0.f, bias);
    else load_run<float, NV, false>(a.bias, i0, a.E, 0.f, bias);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    c[v] = xv[v];
    if (scores) {
      const float s = a.sigmoid ? rcp_fast(1.f + ex2_fast(-kLog2e * xv[v]))
                                : ex2_fast(kLog2e * (xv[v] - top)) * scale_of;
      c[v] = fmaxf(s + bias[v], -INFINITY);
      if (xv[v] == -INFINITY) c[v] = -INFINITY;
    }
    key[v] = key_of(a.bias ? c[v] : xv[v]);
  }
  bool close = false;
  double* row = scratch[GROUPED ? threadIdx.x / 32 : 0];
  if (GROUPED) close = keep_groups<float, NV>(a, c, key, reinterpret_cast<float*>(row));
  const bool check = a.bias != nullptr;
  choose<uint32_t, LANES, NV>(key, sel, cand[LANES == 32 ? threadIdx.x / 32 : 0],
                              a.topk + (check ? 1 : 0), check ? a.pair_error : 0.f);
  const bool order = check && neighbours_close<LANES>(a, sel);
  if (LANES == 32) {
    if (in_range && (__any_sync(FULL, close) || __any_sync(FULL, order))) {
      // Only the order of the candidates is in doubt, unless it is the groups'.
      if (__any_sync(FULL, close) || sel->candidates < 0)
        choose_exact<T, LANES, NV, GROUPED>(a, xr, i0, in_range, sel, row);
      else
        rank_exact<T, NV>(a, xr, i0, top, sel, cand[LANES == 32 ? threadIdx.x / 32 : 0]);
    }
  } else if (__any_sync(FULL, order && in_range)) {
    choose_exact<T, LANES, NV, GROUPED>(a, xr, i0, in_range, sel, row);
  }

  // Weights: place j belongs to lane j % LANES of its row.
  float xs[SLOTS], w[SLOTS];
  int id[SLOTS];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = sub + i * LANES;
    id[i] = in_range && j < a.topk ? sel->id[j] : -1;
    xs[i] = id[i] >= 0 ? to_float(xr[id[i]]) : -INFINITY;
    m = fmaxf(m, xs[i]);
  }
  // exp by ex2.approx: |x - shift| <= 24 gives 24 * 1.2e-7 relative error, 2e-7 at
  // the differences of 1 to 2 that matter most.
  if (a.renorm) {
    // The common factor exp(-m) (sigmoid: exp(-min(m, 0))) leaves the shares as
    // they are and keeps them exact where all scores of a row underflow.
    m = row_max<LANES>(m);
    const float shift = a.sigmoid ? fminf(m, 0.f) : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      w[i] = 0.f;
      if (id[i] >= 0) {
        w[i] = a.sigmoid && xs[i] > 0.f ? 1.f : ex2_fast(kLog2e * (xs[i] - shift));
        if (a.sigmoid) w[i] *= rcp_fast(1.f + ex2_fast(-kLog2e * fabsf(xs[i])));
      }
      sum += w[i];
    }
    sum = row_sum<LANES>(sum);
    const float share = rcp_fast(sum);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) w[i] = id[i] >= 0 ? w[i] * share : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      w[i] = id[i] < 0 ? 0.f
             : a.sigmoid ? rcp_fast(1.f + ex2_fast(-kLog2e * xs[i]))
                         : ex2_fast(kLog2e * (xs[i] - top)) * scale_of;
  }
  if (in_range) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int j = sub + i * LANES;
      if (j < a.topk) {
        a.weights[t * a.topk + j] = w[i] * a.scale;
        a.ids[t * a.topk + j] = id[i];
      }
    }
  }
}

// -----------------------------------------------------------------------------
// Gradient of the weights with respect to the logits (the choice itself and the
// bias have none). With g = scale * dw, s the scores and p = s / sum(chosen s):
//   softmax         dx = s * (g - sum(g s))              over the whole row
//   softmax, renorm dx = p * (g - sum(g p))              chosen experts only
//   sigmoid         dx = g s (1 - s)                     chosen experts only
//   sigmoid, renorm dx = p (1 - s) * (g - sum(g p))      chosen experts only
// One pass: the row (plain softmax) or the chosen logits are read, the whole
// row of dx is written once. 65536 x 256 f32 plain softmax, 8 chosen: 39 us, 20 at
// the copy rate, beside which a lane compares its 8 registers with each of the 8
// places and takes 8 expf; 16384 x 64: 4.8 us with its launch.
// -----------------------------------------------------------------------------
struct RouteBwdArgs {
  const float* dweights;
  const int32_t* ids;
  int T, E, topk;
  int64_t ldx, lddx;
  int sigmoid, renorm;
  float scale;
};

template <typename T, int LANES, int NV, bool VEC>
__global__ void __launch_bounds__(ROUTE_THREADS)
    moe_route_bwd_kernel(const T* x, T* dx, const RouteBwdArgs a) {
  constexpr int ROWS = ROUTE_THREADS / LANES;
  constexpr int SLOTS = ROUTE_MAX_TOPK / LANES;
  __shared__ int2 slot_all[ROWS][ROUTE_MAX_TOPK];  // (expert, gradient bits) of each place
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, sub = lane % LANES, r = threadIdx.x / LANES;
  const int64_t t = (int64_t)blockIdx.x * ROWS + r;
  const bool in_range = t < a.T;
  const T* xr = x + (in_range ? t : 0) * a.ldx;
  int2* slot = slot_all[r];
  const int i0 = sub * NV;

  const bool whole = !a.sigmoid && !a.renorm;
  float xv[NV], top = -INFINITY, total = 1.f;
  if (whole) {
    load_run<T, NV, VEC>(xr, i0, in_range ? a.E : 0, -INFINITY, xv);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (isnan(xv[v])) xv[v] = -INFINITY;
      top = fmaxf(top, xv[v]);
    }
    top = row_max<LANES>(top);
    if (top == -INFINITY) top = 0.f;
    total = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xv[v] = expf(xv[v] - top);
      total += xv[v];
    }
    total = row_sum<LANES>(total);
    if (!(total > 0.f)) total = 1.f;
  }
  float xs[SLOTS], g[SLOTS], p[SLOTS];
  int id[SLOTS];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = sub + i * LANES;
    id[i] = in_range && j < a.topk ? a.ids[t * a.topk + j] : -1;
    if (id[i] >= a.E) id[i] = -1;
    xs[i] = id[i] >= 0 ? to_float(xr[id[i]]) : -INFINITY;
    if (isnan(xs[i])) xs[i] = -INFINITY;
    if (xs[i] == -INFINITY) id[i] = -1;  // no share, no gradient
    g[i] = id[i] >= 0 ? a.dweights[t * a.topk + j] * a.scale : 0.f;
    m = fmaxf(m, xs[i]);
  }
  if (a.renorm) {
    m = row_max<LANES>(m);
    const float shift = a.sigmoid ? fminf(m, 0.f) : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      p[i] = 0.f;
      if (id[i] >= 0) {
        p[i] = a.sigmoid && xs[i] > 0.f ? 1.f : expf(xs[i] - shift);
        if (a.sigmoid) p[i] /= 1.f + expf(-fabsf(xs[i]));
      }
      sum += p[i];
    }
    sum = row_sum<LANES>(sum);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      p[i] *= inv;
      dot += g[i] * p[i];
    }
    dot = row_sum<LANES>(dot);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      g[i] = p[i] * (g[i] - dot);
      if (a.sigmoid) g[i] /= 1.f + expf(xs[i]);
    }
  } else if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const float e = expf(-fabsf(xs[i]));  // s (1 - s) = e / (1 + e)^2, either sign of x
      if (id[i] >= 0) g[i] *= e / ((1.f + e) * (1.f + e));
    }
  } else {
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (id[i] >= 0) g[i] *= expf(xs[i] - top) / total;
      dot += g[i];
    }
    dot = row_sum<LANES>(dot);
#pragma unroll
    for (int v = 0; v < NV; ++v) xv[v] *= -dot / total;
  }
  if (!whole) {
#pragma unroll
    for (int v = 0; v < NV; ++v) xv[v] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = sub + i * LANES;
    if (j < a.topk) slot[j] = make_int2(id[i], __float_as_int(g[i]));
  }
  __syncwarp();
  for (int j = 0; j < a.topk; ++j) {
    const int2 s = slot[j];
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (s.x == i0 + v) xv[v] += __int_as_float(s.y);
  }
  if (in_range) store_run<T, NV, VEC>(dx + t * a.lddx, i0, a.E, xv);
}

// ---- host ----------------------------------------------------------------------
// Whether rows of T can move as NV-wide vectors of at most 16 bytes.
template <typename T>
bool runs_ok(const void* p, int64_t ld, int E, int NV) {
  const int64_t bytes = std::min<int64_t>(16, NV * (int64_t)sizeof(T));
  return E % NV == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0 &&
         (ld * (int64_t)sizeof(T)) % bytes == 0;
}

template <typename T, int LANES, int NV, bool GROUPED>
int route_launch(const T* x, const RouteArgs& given, cudaStream_t st) {
  RouteArgs a = given;
  const int rows = ROUTE_THREADS / LANES;
  const unsigned grid = (unsigned)(((int64_t)a.T + rows - 1) / rows);
  a.group_size = a.E / a.groups;
  const int span = a.group_size / NV;
  a.group_lanes = a.group_size % NV == 0 && (span & (span - 1)) == 0 ? span : 0;
  a.bias_runs = a.E % NV == 0 && aligned16(a.bias);
  a.pair_error = a.sigmoid ? 6e-7f : 4e-6f;
  auto k = runs_ok<T>(x, a.ldx, a.E, NV) ? moe_route_kernel<T, LANES, NV, true, GROUPED>
                                         : moe_route_kernel<T, LANES, NV, false, GROUPED>;
  return launch_overlapped("moe_route_kernel", k, dim3(grid), ROUTE_THREADS, 0, 0, st, x, a);
}
template <typename T>
int route_dispatch(const T* x, const RouteArgs& a, cudaStream_t st) {
  if (a.topk_groups < a.groups) {  // a group per lane: always a whole warp per row
    if (a.E <= 32) return route_launch<T, 32, 1, true>(x, a, st);
    if (a.E <= 64) return route_launch<T, 32, 2, true>(x, a, st);
    if (a.E <= 128) return route_launch<T, 32, 4, true>(x, a, st);
    return route_launch<T, 32, 8, true>(x, a, st);
  }
  if (a.E <= 8) return route_launch<T, 8, 1, false>(x, a, st);
  if (a.E <= 16) return route_launch<T, 8, 2, false>(x, a, st);
  if (a.E <= 32) return route_launch<T, 8, 4, false>(x, a, st);
  if (a.E <= 64) return route_launch<T, 8, 8, false>(x, a, st);
  if (a.E <= 128) return route_launch<T, 16, 8, false>(x, a, st);
  return route_launch<T, 32, 8, false>(x, a, st);
}

template <typename T, int LANES, int NV>
int route_bwd_launch(const T* x, T* dx, const RouteBwdArgs& a, cudaStream_t st) {
  const int rows = ROUTE_THREADS / LANES;
  const unsigned grid = (unsigned)(((int64_t)a.T + rows - 1) / rows);
  auto k = runs_ok<T>(x, a.ldx, a.E, NV) && runs_ok<T>(dx, a.lddx, a.E, NV)
               ? moe_route_bwd_kernel<T, LANES, NV, true>
               : moe_route_bwd_kernel<T, LANES, NV, false>;
  return launch_overlapped("moe_route_bwd_kernel", k, dim3(grid), ROUTE_THREADS, 0, 0, st, x, dx,
                           a);
}
template <typename T>
int route_bwd_dispatch(const T* x, T* dx, const RouteBwdArgs& a, cudaStream_t st) {
  if (a.E <= 8) return route_bwd_launch<T, 8, 1>(x, dx, a, st);
  if (a.E <= 16) return route_bwd_launch<T, 8, 2>(x, dx, a, st);
  if (a.E <= 32) return route_bwd_launch<T, 8, 4>(x, dx, a, st);
  if (a.E <= 64) return route_bwd_launch<T, 8, 8>(x, dx, a, st);
  if (a.E <= 128) return route_bwd_launch<T, 16, 8>(x, dx, a, st);
  return route_bwd_launch<T, 32, 8>(x, dx, a, st);
}

// What both directions check; `k` names the entry point.
int route_check(const char* k, int dtype, int T, int E, int topk, int64_t ldx, int score) {
  const std::string n(k);
  if (dtype != CTB_F16 && dtype != CTB_BF16 && dtype != CTB_F32)
    return set_error(CTB_ERR_DTYPE, n + ": logits must be Float16, BFloat16 or Float32");
  if (T < 0) return set_error(CTB_ERR_SHAPE, n + ": negative number of rows");
  if (E < 1 || E > ROUTE_MAX_EXPERTS) return set_error(CTB_ERR_SHAPE, n + ": 1 to 256 experts");
  if (topk < 1 || topk > ROUTE_MAX_TOPK || topk > E)
    return set_error(CTB_ERR_SHAPE, n + ": topk must be 1 to min(experts, 32)");
  if (ldx < E) return set_error(CTB_ERR_LAYOUT, n + ": row stride smaller than the row");
  if (score != CTB_SCORE_SOFTMAX && score != CTB_SCORE_SIGMOID)
    return set_error(CTB_ERR_ARG, n + ": unknown score");
  return CTB_OK;
}

}  // namespace
}  // namespace ctb

using namespace ctb;

extern "C" int ctb_moe_route(int32_t dtype, const void* logits, const float* bias, float* weights,
                             int32_t* ids, int32_t T, int32_t E, int32_t topk, int64_t ldx,
                             int32_t score, int32_t groups, int32_t topk_groups,
                             int32_t group_top, int32_t renorm, float scale, void* stream) {
  clear_error();
  if (int rc = route_check("moe_route", dtype, T, E, topk, ldx, score)) return rc;
  if (groups < 1 || groups > 32 || E % groups != 0)
    return set_error(CTB_ERR_SHAPE, "moe_route: 1 to 32 groups that divide the experts");
  if (topk_groups < 1 || topk_groups > groups)
    return set_error(CTB_ERR_SHAPE, "moe_route: topk_groups must be 1 to groups");
  if (group_top != 1 && group_top != 2)
    return set_error(CTB_ERR_ARG, "moe_route: group_top must be 1 or 2");
  if (topk > topk_groups * (E / groups))
    return set_error(CTB_ERR_SHAPE, "moe_route: topk exceeds the experts of topk_groups groups");
  if (T == 0) return CTB_OK;
  if (!logits || !weights || !ids) return set_error(CTB_ERR_ARG, "moe_route: NULL pointer");
  const int size = dtype == CTB_F32 ? 4 : 2;
  const Lines x = lines_of(logits, T, E, ldx, size), b = bytes_of(bias, 4ll * E),
              w = bytes_of(weights, 4ll * T * topk), i = bytes_of(ids, 4ll * T * topk);
  if (!apart(w, {x, b, i}) || !apart(i, {x, b}))
    return set_error(CTB_ERR_ARG, "moe_route: weights and ids must be memory of their own");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  RouteArgs a = {};
  a.bias = bias;
  a.weights = weights;
  a.ids = ids;
  a.T = T;
  a.E = E;
  a.topk = topk;
  a.ldx = ldx;
  a.sigmoid = score == CTB_SCORE_SIGMOID;
  a.groups = groups;
  a.topk_groups = topk_groups;
  a.group_top = group_top;
  a.renorm = renorm != 0;
  a.scale = scale;
  auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CTB_F16: return route_dispatch((const __half*)logits, a, st);
    case CTB_BF16: return route_dispatch((const __nv_bfloat16*)logits, a, st);
    default: return route_dispatch((const float*)logits, a, st);
  }
}

extern "C" int ctb_moe_route_bwd(int32_t dtype, const float* dweights, const void* logits,
                                 const int32_t* ids, void* dlogits, int32_t T, int32_t E,
                                 int32_t topk, int64_t ldx, int64_t lddx, int32_t score,
                                 int32_t renorm, float scale, void* stream) {
  clear_error();
  if (int rc = route_check("moe_route_bwd", dtype, T, E, topk, ldx, score)) return rc;
  if (lddx < E)
    return set_error(CTB_ERR_LAYOUT, "moe_route_bwd: row stride smaller than the row");
  if (T == 0) return CTB_OK;
  if (!dweights || !logits || !ids || !dlogits)
    return set_error(CTB_ERR_ARG, "moe_route_bwd: NULL pointer");
  const int size = dtype == CTB_F32 ? 4 : 2;
  const Lines x = lines_of(logits, T, E, ldx, size), dx = lines_of(dlogits, T, E, lddx, size);
  if (!apart(dx, {bytes_of(dweights, 4ll * T * topk), bytes_of(ids, 4ll * T * topk)}) ||
      !(same_place(dx, x) || apart(dx, {x})))
    return set_error(CTB_ERR_ARG, "moe_route_bwd: dlogits must be memory of its own (or the logits, "
                                  "with the same row stride)");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  RouteBwdArgs a;
  a.dweights = dweights;
  a.ids = ids;
  a.T = T;
  a.E = E;
  a.topk = topk;
  a.ldx = ldx;
  a.lddx = lddx;
  a.sigmoid = score == CTB_SCORE_SIGMOID;
  a.renorm = renorm != 0;
  a.scale = scale;
  auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CTB_F16:
      return route_bwd_dispatch((const __half*)logits, (__half*)dlogits, a, st);
    case CTB_BF16:
      return route_bwd_dispatch((const __nv_bfloat16*)logits, (__nv_bfloat16*)dlogits, a, st);
    default: return route_bwd_dispatch((const float*)logits, (float*)dlogits, a, st);
  }
}
