// Shared helpers for the sm_100a kernels of libcutile_b200.so: status
// plumbing, the device error word, vector loads/stores and CTA reductions.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include <initializer_list>
#include <string>

#include "../../include/cutile_b200.h"

namespace ctb {

// ---- host-side status -------------------------------------------------------
// Records `msg` as this thread's last error and returns `code`.
int set_error(int code, const std::string& msg);
void clear_error();
// Maps a CUDA error to CTB_ERR_CUDA with `what` as context.
int cuda_fail(cudaError_t e, const char* what);

#define CTB_CUDA_CHECK(call)                                   \
  do {                                                         \
    cudaError_t _e = (call);                                   \
    if (_e != cudaSuccess) return ::ctb::cuda_fail(_e, #call); \
  } while (0)

// After a kernel launch: report a launch-configuration error.
inline int launch_status(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  return CTB_OK;
}

// ---- operands that may not share memory ------------------------------------------
// `rows` lines of `len` bytes, `pitch` bytes apart. Nothing where p is NULL.
struct Lines {
  const void* p;
  int64_t rows, len, pitch;
  uintptr_t begin, end;  // all bytes from the first line's to the last's; both 0 for nothing
};
// A matrix of elements of `size` bytes whose lines are `ld` elements apart.
inline Lines lines_of(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t size) {
  Lines l = {p, rows, cols * size, rows > 1 ? ld * size : cols * size, 0, 0};
  if (!p || rows <= 0 || cols <= 0) return l;
  l.begin = reinterpret_cast<uintptr_t>(p);
  uintptr_t bytes;
  if (__builtin_mul_overflow((uintptr_t)(rows - 1), (uintptr_t)l.pitch, &bytes) ||
      __builtin_add_overflow(bytes, l.begin + (uintptr_t)l.len, &l.end))
    l.end = UINTPTR_MAX;
  return l;
}
inline Lines bytes_of(const void* p, int64_t bytes) { return lines_of(p, 1, bytes, bytes, 1); }
// Whether lines whose bytes from first to last meet share any.
bool lines_meet(const Lines& a, const Lines& b);
// Whether any byte belongs to both. Lines that lie between one another's (columns
// of one wider buffer, every other row of it) do not overlap.
inline bool overlap(const Lines& a, const Lines& b) {
  return a.begin < b.end && b.begin < a.end && lines_meet(a, b);
}
inline bool apart(const Lines& a, std::initializer_list<Lines> others) {
  for (const Lines& o : others)
    if (overlap(a, o)) return false;
  return true;
}
// The same lines at the same place: what an output that may be an input is held to.
inline bool same_place(const Lines& a, const Lines& b) {
  return a.p == b.p && a.rows == b.rows && a.len == b.len && a.pitch == b.pitch;
}

struct DeviceProps {
  int sm_count = 0;
  int max_smem_optin = 0;
  int cc_major = 0, cc_minor = 0;
};
// Properties of the current device (cached per device; ctb_init fills them).
int current_props(DeviceProps* out);

// Unique ID (never reused within a process) of the current device's primary
// context. Per-device set-up (kernel attributes, symbol addresses) is
// remembered with this ID, so after a cudaDeviceReset it is done again.
int current_context_id(unsigned long long* id);

// ---- device error word ------------------------------------------------------
// Set by a kernel whose bounded wait gave up; read by ctb_check_device.
// Bits: 1 = GEMM, 2 = FMHA, 4 = LayerNorm backward, 8 = MoE pipeline wait,
// 32 = the wait self-test (ctb_selftest_wait_timeout), 64 = the dense layer.
// The library is built without relocatable device code, so every translation
// unit owns its copy; a unit whose kernels flag errors exposes a reader
// (take_device_error) that ctb_check_device polls.
static __device__ unsigned int g_device_error = 0;

// Reads and clears this translation unit's error word on the current device.
static inline int take_device_error(unsigned int* out) {
  unsigned int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(out, g_device_error, sizeof(*out));
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
  return e == cudaSuccess ? 0 : (int)e;
}

__device__ __forceinline__ void flag_device_error(unsigned int bit) {
  atomicOr(&g_device_error, bit);
}

// ---- programmatic dependent launch ---------------------------------------------
// A kernel launched with launch_overlapped may start while its predecessor on
// the stream still runs, once every CTA of that one has called
// let_next_start() (or ended); it touches global memory only after
// wait_for_previous(), which returns when the predecessor has completed and its
// writes are visible. That hides a launch's latency and a kernel's set-up behind
// the predecessor's tail. A kernel that allocates tensor memory lets the next
// start only after the allocation: CTAs of the next one hold theirs while they
// wait. What a predecessor may have written is read with ordinary loads, not
// through the read-only path (no const __restrict__ parameters), whose data must
// not change while the kernel runs.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <typename... P, typename... A>
inline int launch_overlapped(const char* what, void (*kernel)(P...), dim3 grid, int threads,
                             int smem, int cluster, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_fail(e, what);
  }
  return CTB_OK;
}

// ---- vector memory helpers --------------------------------------------------
// Streaming loads: data is read once, do not allocate in L1.
__device__ __forceinline__ float4 ld_stream_f4(const float* p) {
  float4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}
// Evict-first stores for outputs that are not re-read by this kernel.
__device__ __forceinline__ void st_stream_f4(float* p, float4 v) {
  asm volatile("st.global.cs.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// CTA-wide reduction for NWARPS warps; `red` is NWARPS floats of shared memory.
// Every thread returns the total. Contains two __syncthreads.
template <int NWARPS, bool IS_MAX>
__device__ __forceinline__ float block_reduce(float v, float* red) {
  v = IS_MAX ? warp_max(v) : warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (NWARPS == 1) return v;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float t = lane < NWARPS ? red[lane] : (IS_MAX ? -INFINITY : 0.f);
  t = IS_MAX ? warp_max(t) : warp_sum(t);
  __syncthreads();  // `red` may be reused by the caller's next reduction
  return t;
}

// -----------------------------------------------------------------------------
// Register-resident row staging shared by softmax and layernorm: a CTA of
// THREADS threads holds one row of up to THREADS*NV*4 floats, NV float4 per
// thread, element index (k*THREADS + t)*4 + e. Padding slots get `pad`.
// -----------------------------------------------------------------------------
template <int THREADS, int NV, bool VEC>
__device__ __forceinline__ void load_row(const float* __restrict__ p, int len, float pad,
                                         float (&v)[NV * 4]) {
  const int t = threadIdx.x;
  if (VEC) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int idx = (k * THREADS + t) * 4;
      if (idx < len) {  // len % 4 == 0 on this path
        float4 q = ld_stream_f4(p + idx);
        v[4 * k + 0] = q.x;
        v[4 * k + 1] = q.y;
        v[4 * k + 2] = q.z;
        v[4 * k + 3] = q.w;
      } else {
        v[4 * k + 0] = v[4 * k + 1] = v[4 * k + 2] = v[4 * k + 3] = pad;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int idx = (k * THREADS + t) * 4 + e;
        v[4 * k + e] = idx < len ? p[idx] : pad;
      }
  }
}

template <int THREADS, int NV, bool VEC>
__device__ __forceinline__ void store_row(float* __restrict__ p, int len,
                                          const float (&v)[NV * 4]) {
  const int t = threadIdx.x;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int idx0 = (k * THREADS + t) * 4;
    if (VEC) {
      if (idx0 < len)
        st_stream_f4(p + idx0, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (idx0 + e < len) p[idx0 + e] = v[4 * k + e];
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace ctb
