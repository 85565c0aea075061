// What the kernels of the dense layer (dense.cu, dense_sm100.cu) share: the
// problem they are given, the activations, and 16-bit element access.
#pragma once

#include "ctb_common.cuh"

namespace ctb {
namespace dense {

// One matrix product of the layer or of its gradients, in row-major terms:
//   D[r, c] = act(sum_k P(r, k) * Q(c, k) + bias[c]) + R[r, c],  r < rows, c < cols
// An operand is "k-major" when k is its contiguous dimension (element (r, k) at
// r * ld + k) and "row-major-k" (mn) when its row or column index is (k * ld + r).
// All matrices are 16-bit (F16 or BF16, the same for all); sums are Float32.
struct Product {
  const void* P;
  const void* Q;
  int64_t ldp, ldq;
  bool p_mn, q_mn;
  void* D;
  int64_t ldd;
  int rows, cols, depth;
  // epilogue
  const void* bias;  // cols elements, or NULL
  bool bias_f32;     // Float32, else the operands' type
  int act;
  const void* R;     // residual, added after the activation, or NULL
  int64_t ldr;
  void* Z;           // receives the value before the activation, or NULL
  int64_t ldz;
};

// ---- 16-bit elements --------------------------------------------------------------
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float2 unpack2(uint32_t v, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float2 unpack2(uint32_t v, const __nv_bfloat16*) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2(w[i], (const T*)nullptr);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1], (const T*)nullptr), pack2(f[2], f[3], (const T*)nullptr),
                    pack2(f[4], f[5], (const T*)nullptr), pack2(f[6], f[7], (const T*)nullptr));
}

// ---- activations --------------------------------------------------------------------
// Evaluated on pairs: the packed f32x2 instructions take one issue slot for two
// elements, and an epilogue's slots are what an activation costs (its power too).
// ex2.approx.ftz and rcp.approx.ftz are documented to 2 ulp and 1 ulp; results
// below the normal range become 0. That shows in BFloat16 only, in values of
// 1e-36 and below: silu(-88), -5e-37 exactly, is 0 here.
using f2 = uint64_t;
__device__ __forceinline__ f2 mk2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(f2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2 all2(float a) { return mk2(a, a); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
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
__device__ __forceinline__ f2 ex2_2(f2 v) {
  float a, b;
  un2(v, a, b);
  return mk2(ex2_fast(a), ex2_fast(b));
}
__device__ __forceinline__ f2 rcp_2(f2 v) {
  float a, b;
  un2(v, a, b);
  return mk2(rcp_fast(a), rcp_fast(b));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;  // 1 / sqrt(2 pi)
constexpr float kGeluScale = 1.5957691216057308f;    // 2 sqrt(2 / pi)
constexpr float kGeluCube = 0.044715f;

// 1 / (1 + 2^v). 2^v = inf gives 0.
__device__ __forceinline__ f2 logistic_ex2(f2 v) {
  return rcp_2(add2(ex2_2(v), all2(1.f)));
}

// The upper tail of the normal distribution, Q(a) = 0.5 erfc(a / sqrt(2)), a >= 0,
// and exp(-a^2 / 2) on the way: with t = 1 / (1 + 0.273 a), Q(a) exp(a^2 / 2) / t
// is smooth in t over (0, 1]; this is its polynomial of degree 6 with the least
// largest relative error (1.8e-6, by reweighted least squares on 4400 points
// of [0, 40]). In 32 bits z * Phi(z) is within 4e-7 of the exact value for |z| <
// 12. A call of erfcf instead makes a 4096 x 4096 x 1024 bf16 layer take 60 us,
// against 33 us, and 29 without an activation.
__device__ __forceinline__ f2 normal_tail(f2 a, f2* density) {
  const f2 e = ex2_2(mul2(mul2(a, a), all2(-0.5f * kLog2e)));
  const f2 t = rcp_2(fma2(a, all2(0.273f), all2(1.f)));
  f2 p = fma2(all2(-0.05735107883810997f), t, all2(0.14058725535869598f));
  p = fma2(p, t, all2(-0.006268841680139303f));
  p = fma2(p, t, all2(0.10854672640562057f));
  p = fma2(p, t, all2(0.09625127166509628f));
  p = fma2(p, t, all2(0.10933801531791687f));
  p = fma2(p, t, all2(0.10889600962400436f));
  *density = e;
  return mul2(mul2(p, t), e);
}

// |z|, at most 30, where Q has long been 0 (an infinity would make 0 * inf of
// it); NaN stays NaN.
__device__ __forceinline__ float tail_arg(float z) {
  const float a = fabsf(z);
  return a > 30.f ? 30.f : a;
}

// Both elements of a pair through the activation.
template <int ACT>
__device__ __forceinline__ void activate2(float& a, float& b) {
  if (ACT == CTB_ACT_RELU) {
    a = a < 0.f ? 0.f : a;
    b = b < 0.f ? 0.f : b;
  } else if (ACT == CTB_ACT_SILU) {
    const f2 z = mk2(a, b);
    un2(mul2(z, logistic_ex2(mul2(z, all2(-kLog2e)))), a, b);
  } else if (ACT == CTB_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| Q(|z|)
    const float ta = tail_arg(a), tb = tail_arg(b);
    f2 e;
    const f2 q = normal_tail(mk2(ta, tb), &e);
    un2(fma2(mk2(-ta, -tb), q, mk2(fmaxf(a, 0.f), fmaxf(b, 0.f))), a, b);
  } else if (ACT == CTB_ACT_GELU_TANH) {  // 0.5 (1 + tanh(u)) is the logistic function of 2 u
    const f2 z = mk2(a, b);
    const f2 u = mul2(z, fma2(mul2(z, z), all2(-kLog2e * kGeluScale * kGeluCube),
                              all2(-kLog2e * kGeluScale)));
    un2(mul2(z, logistic_ex2(u)), a, b);
  }
}
// Both elements of a pair replaced by the activation's slope there.
template <int ACT>
__device__ __forceinline__ void slope2(float& a, float& b) {
  if (ACT == CTB_ACT_RELU) {
    a = a > 0.f ? 1.f : 0.f;
    b = b > 0.f ? 1.f : 0.f;
  } else if (ACT == CTB_ACT_SILU) {  // s (1 + z (1 - s))
    const f2 z = mk2(a, b);
    const f2 s = logistic_ex2(mul2(z, all2(-kLog2e)));
    un2(mul2(s, fma2(z, fma2(s, all2(-1.f), all2(1.f)), all2(1.f))), a, b);
  } else if (ACT == CTB_ACT_GELU) {  // Phi(z) + z phi(z)
    const float ta = tail_arg(a), tb = tail_arg(b);
    f2 e;
    const f2 q = normal_tail(mk2(ta, tb), &e);
    const f2 d = mul2(mul2(mk2(copysignf(ta, a), copysignf(tb, b)), all2(kInvSqrt2Pi)), e);
    float qa, qb;
    un2(q, qa, qb);
    un2(add2(d, mk2(a > 0.f ? 1.f - qa : qa, b > 0.f ? 1.f - qb : qb)), a, b);
  } else if (ACT == CTB_ACT_GELU_TANH) {  // s + z s (1 - s) * du/dz
    const f2 z = mk2(a, b), zz = mul2(z, z);
    const f2 s = logistic_ex2(mul2(z, fma2(zz, all2(-kLog2e * kGeluScale * kGeluCube),
                                           all2(-kLog2e * kGeluScale))));
    const f2 w = mul2(mul2(z, s), fma2(s, all2(-1.f), all2(1.f)));
    float ua, ub;  // du/dz, kept finite where z^2 is not: w has long been 0 there
    un2(fma2(zz, all2(3.f * kGeluCube * kGeluScale), all2(kGeluScale)), ua, ub);
    un2(fma2(w, mk2(fminf(ua, 3e38f), fminf(ub, 3e38f)), s), a, b);
  } else {
    a = b = 1.f;
  }
}
// Chosen at run time, one element: for code that nothing waits on.
__device__ __forceinline__ float activate_any(float z, int act) {
  float unused = 0.f;
  switch (act) {
    case CTB_ACT_RELU: activate2<CTB_ACT_RELU>(z, unused); break;
    case CTB_ACT_GELU: activate2<CTB_ACT_GELU>(z, unused); break;
    case CTB_ACT_GELU_TANH: activate2<CTB_ACT_GELU_TANH>(z, unused); break;
    case CTB_ACT_SILU: activate2<CTB_ACT_SILU>(z, unused); break;
    default: break;
  }
  return z;
}

}  // namespace dense
}  // namespace ctb
