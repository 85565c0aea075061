// The experts' rows back to one row per token, the step after the experts'
// products, and its gradient:
//   out[t] = residual[t] + sum_j w[t, j] * y[t * topk + j]
//   dy[t * topk + j] = w[t, j] * dout[t],  dw[t, j] = <dout[t], y[t * topk + j]>
// A slot that no expert took (its id is outside [0, E)) is skipped: its row of
// y was never written and is not read.
//
// Both are bound by HBM: every row of y is moved once. Forward: one thread per
// 16 bytes of a token's row (per element where rows are no 16-byte runs: 4096
// tokens x 2 x 4095 take 93 us, x 4096 21), whose loads, up to 8 slots' and the
// residual's, are all in flight before the first is used; with more slots their
// ids and rows are loaded in turn. Sums in Float32, rounded once. Gradient:
// one warp per slot, the slots of a token in neighbouring warps, so dout comes
// from HBM once and from L1 for the other slots; the warp's lanes keep the dot
// product's partial sums and join them with shuffles (fixed order). 16384 tokens
// x 2 x 4096 f16 with residual: 79 to 82 us, the copy rate (6.6 TB/s); gradients of
// 4099 x 8 x 2048 bf16: 48 to 49 us, 5.9 TB/s (97 where N is 2047).
#include "ctb_common.cuh"

#include <algorithm>

namespace ctb {
namespace {

constexpr int COMBINE_THREADS = 256;

__device__ __forceinline__ float2 pair_to_float(uint32_t v, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float2 pair_to_float(uint32_t v, const __nv_bfloat16*) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ uint32_t pair_from_float(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_from_float(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float one_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float one_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void one_from_float(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void one_from_float(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// W neighbouring elements: 8 (one 16-byte access) or 1.
template <typename T, int W> struct Run;
template <typename T> struct Run<T, 8> {
  uint4 raw;
  __device__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  // Rows that are read once: not kept in L1, first to leave L2.
  __device__ void load_once(const T* p) {
    asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                 : "l"(p));
  }
  __device__ void get(float (&f)[8]) const {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = pair_to_float(u[i], (const T*)nullptr);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ void put(T* p, const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = pair_from_float(f[2 * i], f[2 * i + 1], (const T*)nullptr);
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <typename T> struct Run<T, 1> {
  T v;
  __device__ void zero() { one_from_float(&v, 0.f); }
  __device__ void load(const T* p) { v = *p; }
  __device__ void load_once(const T* p) { v = *p; }
  __device__ void get(float (&f)[1]) const { f[0] = one_to_float(v); }
  static __device__ void put(T* p, const float (&f)[1]) { one_from_float(p, f[0]); }
};

template <typename T>
struct CombineArgs {
  const T* y;
  const float* weights;
  const int32_t* ids;
  const T* residual;
  T* out;
  int64_t items;  // T * runs
  int runs;       // runs of W elements per row
  int topk, E;
  int64_t ldy, ldr, ldo;
};

// TOPK > 0: that many slots, all loads in flight; 0: any number, in turn.
template <typename T, int W, int TOPK>
__global__ void __launch_bounds__(COMBINE_THREADS) moe_combine_kernel(const CombineArgs<T> a) {
  let_next_start();
  wait_for_previous();
  const int64_t i = (int64_t)blockIdx.x * COMBINE_THREADS + threadIdx.x;
  if (i >= a.items) return;
  const int64_t t = a.items >> 31 ? i / a.runs : (int64_t)((uint32_t)i / (uint32_t)a.runs);
  const int c = (int)(i - t * a.runs) * W;
  const int topk = TOPK ? TOPK : a.topk;
  const int64_t s0 = t * topk;
  float acc[W];
  Run<T, W> res;
  if (a.residual) res.load(a.residual + t * a.ldr + c);
  if (TOPK) {
    Run<T, W> v[TOPK ? TOPK : 1];
    float w[TOPK ? TOPK : 1];
#pragma unroll
    for (int j = 0; j < TOPK; ++j) {
      const int id = a.ids ? a.ids[s0 + j] : 0;
      const bool used = id >= 0 && id < a.E;
      if (used) v[j].load_once(a.y + (s0 + j) * a.ldy + c);
      else v[j].zero();
      w[j] = !used ? 0.f : a.weights ? a.weights[s0 + j] : 1.f;
    }
    if (a.residual) res.get(acc);
    else
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.f;
#pragma unroll
    for (int j = 0; j < TOPK; ++j) {
      float f[W];
      v[j].get(f);
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = fmaf(w[j], f[e], acc[e]);
    }
  } else {
    if (a.residual) res.get(acc);
    else
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int j = 0; j < topk; ++j) {
      const int id = a.ids ? a.ids[s0 + j] : 0;
      if (id < 0 || id >= a.E) continue;
      Run<T, W> v;
      v.load_once(a.y + (s0 + j) * a.ldy + c);
      const float w = a.weights ? a.weights[s0 + j] : 1.f;
      float f[W];
      v.get(f);
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = fmaf(w, f[e], acc[e]);
    }
  }
  Run<T, W>::put(a.out + t * a.ldo + c, acc);
}

template <typename T>
struct CombineBwdArgs {
  const T* dout;
  const T* y;
  const float* weights;
  const int32_t* ids;
  T* dy;
  float* dweights;
  int64_t slots;
  int topk, N, E;
  int64_t lddo, ldy, lddy;
};

template <typename T, int W>
__global__ void __launch_bounds__(COMBINE_THREADS)
    moe_combine_bwd_kernel(const CombineBwdArgs<T> a) {
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31;
  const int64_t s = (int64_t)blockIdx.x * (COMBINE_THREADS / 32) + threadIdx.x / 32;
  if (s >= a.slots) return;
  const int id = a.ids ? a.ids[s] : 0;
  const bool used = id >= 0 && id < a.E;
  const float w = !used ? 0.f : a.weights ? a.weights[s] : 1.f;
  const T* d = a.dout + s / a.topk * a.lddo;
  const T* y = a.y + (a.weights ? s * a.ldy : 0);
  T* dy = a.dy + s * a.lddy;
  // Unsigned columns: the step past the end of the longest row (2^31 - 1) does not wrap.
  const uint32_t N = (uint32_t)a.N, first = (uint32_t)lane * W;
  float dot = 0.f;
  if (!used) {
    float z[W];
#pragma unroll
    for (int e = 0; e < W; ++e) z[e] = 0.f;
    for (uint32_t c = first; c < N; c += 32 * W) Run<T, W>::put(dy + c, z);
  } else {
    // FLIGHT runs of both rows are asked for before the first is used (the
    // stores between them could alias, so the compiler would not).
    constexpr int FLIGHT = 4;
    for (uint32_t c0 = first; c0 < N; c0 += FLIGHT * 32 * W) {
      Run<T, W> rd[FLIGHT], ry[FLIGHT];
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        const uint32_t c = c0 + j * 32 * W;
        if (c < N) {
          rd[j].load(d + c);
          if (a.weights) ry[j].load_once(y + c);
        }
      }
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        const uint32_t c = c0 + j * 32 * W;
        if (c < N) {
          float fd[W], fy[W];
          rd[j].get(fd);
          if (a.weights) {
            ry[j].get(fy);
#pragma unroll
            for (int e = 0; e < W; ++e) {
              dot = fmaf(fd[e], fy[e], dot);
              fd[e] *= w;
            }
          }
          Run<T, W>::put(dy + c, fd);
        }
      }
    }
  }
  if (a.weights) {
    dot = warp_sum(dot);
    if (lane == 0) a.dweights[s] = dot;
  }
}

// Whether rows from `p`, `ld` elements apart, are made of whole 16-byte runs.
template <typename T>
bool rows16(const T* p, int64_t ld) {
  return aligned16(p) && ld % 8 == 0;
}

template <typename T, int W>
int combine_launch(const CombineArgs<T>& a, cudaStream_t st) {
  const int64_t grid = (a.items + COMBINE_THREADS - 1) / COMBINE_THREADS;
  if (grid > 0x7fffffff) return set_error(CTB_ERR_SHAPE, "moe_combine: too many elements");
  // Up to 8 slots by straight code, any other number in a loop: 4096 tokens of 4096
  // columns 26 us against 36 for 3 slots, 53 against 70 for 8.
  auto k = moe_combine_kernel<T, W, 0>;
  switch (a.topk) {
    case 1: k = moe_combine_kernel<T, W, 1>; break;
    case 2: k = moe_combine_kernel<T, W, 2>; break;
    case 3: k = moe_combine_kernel<T, W, 3>; break;
    case 4: k = moe_combine_kernel<T, W, 4>; break;
    case 5: k = moe_combine_kernel<T, W, 5>; break;
    case 6: k = moe_combine_kernel<T, W, 6>; break;
    case 7: k = moe_combine_kernel<T, W, 7>; break;
    case 8: k = moe_combine_kernel<T, W, 8>; break;
    default: break;
  }
  return launch_overlapped("moe_combine_kernel", k, dim3((unsigned)grid), COMBINE_THREADS, 0, 0, st,
                           a);
}

template <typename T>
int combine_dispatch(CombineArgs<T> a, int T_, int N, cudaStream_t st) {
  const bool vec = N % 8 == 0 && rows16(a.y, a.ldy) && rows16(a.out, a.ldo) &&
                   (!a.residual || rows16(a.residual, a.ldr));
  a.runs = vec ? N / 8 : N;
  a.items = (int64_t)T_ * a.runs;
  return vec ? combine_launch<T, 8>(a, st) : combine_launch<T, 1>(a, st);
}

template <typename T>
int combine_bwd_dispatch(const CombineBwdArgs<T>& a, cudaStream_t st) {
  const int per = COMBINE_THREADS / 32;
  const int64_t grid = (a.slots + per - 1) / per;
  if (grid > 0x7fffffff) return set_error(CTB_ERR_SHAPE, "moe_combine_bwd: too many slots");
  const bool vec = a.N % 8 == 0 && rows16(a.dout, a.lddo) && rows16(a.dy, a.lddy) &&
                   (!a.weights || rows16(a.y, a.ldy));
  return launch_overlapped("moe_combine_bwd_kernel",
                           vec ? moe_combine_bwd_kernel<T, 8> : moe_combine_bwd_kernel<T, 1>,
                           dim3((unsigned)grid), COMBINE_THREADS, 0, 0, st, a);
}

int combine_check(const std::string& n, int dtype, int T, int topk, int N, int E, bool ids) {
  if (dtype != CTB_F16 && dtype != CTB_BF16)
    return set_error(CTB_ERR_DTYPE, n + ": rows must be Float16 or BFloat16");
  if (T < 0 || N < 0) return set_error(CTB_ERR_SHAPE, n + ": negative size");
  if (topk < 1 || (int64_t)T * topk > 0x7fffffff)
    return set_error(CTB_ERR_SHAPE, n + ": topk must be positive and T * topk fit 32 bits");
  if (ids && E < 1) return set_error(CTB_ERR_SHAPE, n + ": ids need the number of experts");
  return CTB_OK;
}

}  // namespace
}  // namespace ctb

using namespace ctb;

extern "C" int ctb_moe_combine(int32_t dtype, const void* y, const float* weights,
                               const int32_t* ids, const void* residual, void* out, int32_t T,
                               int32_t topk, int32_t N, int32_t E, int64_t ldy, int64_t ldr,
                               int64_t ldo, void* stream) {
  clear_error();
  if (int rc = combine_check("moe_combine", dtype, T, topk, N, E, ids != nullptr)) return rc;
  if (ldy < N || ldo < N || (residual && ldr < N))
    return set_error(CTB_ERR_LAYOUT, "moe_combine: row stride smaller than the row");
  if (T == 0 || N == 0) return CTB_OK;
  if (!y || !out) return set_error(CTB_ERR_ARG, "moe_combine: NULL pointer");
  const Lines o = lines_of(out, T, N, ldo, 2), r = lines_of(residual, T, N, ldr, 2),
              ys = lines_of(y, (int64_t)T * topk, N, ldy, 2);
  if (!apart(o, {bytes_of(weights, 4ll * T * topk), bytes_of(ids, 4ll * T * topk)}) ||
      !(same_place(o, r) || apart(o, {r})) || !((topk == 1 && same_place(o, ys)) || apart(o, {ys})))
    return set_error(CTB_ERR_ARG, "moe_combine: out must be memory of its own (or the residual, or y "
                                  "where topk is 1, with the same row stride)");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto* tag) {
    using E_ = std::remove_pointer_t<decltype(tag)>;
    CombineArgs<E_> a;
    a.y = static_cast<const E_*>(y);
    a.weights = weights;
    a.ids = ids;
    a.residual = static_cast<const E_*>(residual);
    a.out = static_cast<E_*>(out);
    a.topk = topk;
    a.E = ids ? E : 1;
    a.ldy = ldy;
    a.ldr = ldr;
    a.ldo = ldo;
    return combine_dispatch<E_>(a, T, N, st);
  };
  return dtype == CTB_F16 ? go((__half*)nullptr) : go((__nv_bfloat16*)nullptr);
}

extern "C" int ctb_moe_combine_bwd(int32_t dtype, const void* dout, const void* y,
                                   const float* weights, const int32_t* ids, void* dy,
                                   float* dweights, int32_t T, int32_t topk, int32_t N, int32_t E,
                                   int64_t lddo, int64_t ldy, int64_t lddy, void* stream) {
  clear_error();
  if (int rc = combine_check("moe_combine_bwd", dtype, T, topk, N, E, ids != nullptr)) return rc;
  if (lddo < N || lddy < N || (weights && ldy < N))
    return set_error(CTB_ERR_LAYOUT, "moe_combine_bwd: row stride smaller than the row");
  if (T == 0) return CTB_OK;
  if ((N > 0 && (!dout || !dy)) || (weights && (!dweights || (N > 0 && !y))))
    return set_error(CTB_ERR_ARG, "moe_combine_bwd: NULL pointer");
  const int64_t slots = (int64_t)T * topk;
  const Lines d = lines_of(dout, T, N, lddo, 2), ys = lines_of(weights ? y : nullptr, slots, N, ldy, 2),
              dys = lines_of(dy, slots, N, lddy, 2), w = bytes_of(weights, 4 * slots),
              i = bytes_of(ids, 4 * slots), dw = bytes_of(weights ? dweights : nullptr, 4 * slots);
  if (!apart(dys, {w, i, dw}) || !(same_place(dys, ys) || apart(dys, {ys})) ||
      !((topk == 1 && same_place(dys, d)) || apart(dys, {d})) || !apart(dw, {d, ys, i}) ||
      !(same_place(dw, w) || apart(dw, {w})))
    return set_error(CTB_ERR_ARG, "moe_combine_bwd: dy and dweights must be memory of their own (dy "
                                  "may be y, or dout where topk is 1, with the same row stride; "
                                  "dweights may be the weights)");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto* tag) {
    using E_ = std::remove_pointer_t<decltype(tag)>;
    CombineBwdArgs<E_> a;
    a.dout = static_cast<const E_*>(dout);
    a.y = static_cast<const E_*>(y);
    a.weights = weights;
    a.ids = ids;
    a.dy = static_cast<E_*>(dy);
    a.dweights = dweights;
    a.slots = (int64_t)T * topk;
    a.topk = topk;
    a.N = N;
    a.E = ids ? E : 1;
    a.lddo = lddo;
    a.ldy = ldy;
    a.lddy = lddy;
    return combine_bwd_dispatch<E_>(a, st);
  };
  return dtype == CTB_F16 ? go((__half*)nullptr) : go((__nv_bfloat16*)nullptr);
}
