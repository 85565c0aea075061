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
// The logistic function by the fast exponential: relative error under 1e-6 for
// |v| < 16, far below the half step of the 16-bit result (2^-9 and 2^-12).
__device__ __forceinline__ float logistic(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

constexpr float kSqrtHalf = 0.70710678118654752f;        // 1 / sqrt(2)
constexpr float kInvSqrt2Pi = 0.39894228040143268f;      // 1 / sqrt(2 pi)
constexpr float kGeluScale = 1.5957691216057308f;        // 2 sqrt(2 / pi)
constexpr float kGeluCube = 0.044715f;

// 0.5 (1 + tanh(u)) is the logistic function of 2 u.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == CTB_ACT_RELU) return z < 0.f ? 0.f : z;
  if (ACT == CTB_ACT_SILU) return z * logistic(z);
  if (ACT == CTB_ACT_GELU) return 0.5f * z * erfcf(-kSqrtHalf * z);
  if (ACT == CTB_ACT_GELU_TANH) return z * logistic(kGeluScale * z * fmaf(kGeluCube * z, z, 1.f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float activate_slope(float z) {
  if (ACT == CTB_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == CTB_ACT_SILU) {
    const float s = logistic(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == CTB_ACT_GELU)
    return fmaf(z * kInvSqrt2Pi, __expf(-0.5f * z * z), 0.5f * erfcf(-kSqrtHalf * z));
  if (ACT == CTB_ACT_GELU_TANH) {
    const float s = logistic(kGeluScale * z * fmaf(kGeluCube * z, z, 1.f));
    return fmaf(z * s * (1.f - s), kGeluScale * fmaf(3.f * kGeluCube * z, z, 1.f), s);
  }
  return 1.f;
}
// Chosen at run time, for code that the product does not wait on.
__device__ __forceinline__ float activate_any(float z, int act) {
  switch (act) {
    case CTB_ACT_RELU: return activate<CTB_ACT_RELU>(z);
    case CTB_ACT_GELU: return activate<CTB_ACT_GELU>(z);
    case CTB_ACT_GELU_TANH: return activate<CTB_ACT_GELU_TANH>(z);
    case CTB_ACT_SILU: return activate<CTB_ACT_SILU>(z);
    default: return z;
  }
}

}  // namespace dense
}  // namespace ctb
