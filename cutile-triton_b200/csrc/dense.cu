// The dense layer: a matrix product with bias, activation and residual in its
// epilogue, and its gradients (ctb_dense_fwd, ctb_dense_bwd).
//
//   Z = A B .+ b,  C = act.(Z) .+ R               (Julia, column-major)
//   dZ = dC .* act'(Z),  db = sum(dZ; dims = 2),  dA = dZ B',  dB = A' dZ
//
// dZ is rounded to the operands' 16 bits: it is an operand of two tensor-core
// products. db is summed from the unrounded values, in Float32.
#include "dense.cuh"

#include <algorithm>

namespace ctb {
namespace dense {

// dense_sm100.cu
template <typename T>
int product_sm100(const Product& p, int sms, cudaStream_t st);

namespace {

// ---- a product over nothing: act(bias) + R ---------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) product_empty_kernel(const Product p) {
  let_next_start();
  wait_for_previous();
  const int64_t total = (int64_t)p.rows * p.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / p.cols;
    const int c = (int)(i - r * p.cols);
    float z = 0.f;
    if (p.bias)
      z = p.bias_f32 ? static_cast<const float*>(p.bias)[c] : to_f32(static_cast<const T*>(p.bias)[c]);
    if (p.Z) from_f32(static_cast<T*>(p.Z) + r * p.ldz + c, z);
    float v = activate_any(z, p.act);
    if (p.R) v += to_f32(static_cast<const T*>(p.R)[r * p.ldr + c]);
    from_f32(static_cast<T*>(p.D) + r * p.ldd + c, v);
  }
}

// ---- operands that TMA cannot address ----------------------------------------------------
int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
// Copies have lines of whole 128-byte rows: lines that TMA can address but that
// start inside a 128-byte line load more slowly (768 x 1000 x 1000, where nothing is
// copied, 12.5 us; 768 x 1024 x 1024 7.4).
int64_t pitch(int64_t n) { return (n + 63) / 64 * 64; }

// A matrix of `lines` lines of `len` contiguous elements is addressable where
// it starts on a 16-byte boundary and its lines do.
bool tma_lines(const void* p, int64_t ld, int64_t lines) {
  return aligned16(p) && (ld % 8 == 0 || lines <= 1);
}
int64_t packed_bytes(int64_t lines, int64_t len) { return round256(2 * lines * pitch(len)); }

// Copies lines of 16-bit elements to lines pitch(len) apart; one thread per 16
// bytes of the result. Both operands of a product in one launch (the grid's y).
// One row by 4097 x 8193: 40 us, of which the copy of the weight (134 MB moved, 20 us
// at the copy rate) is 27; 13 us where the weight's lines are aligned.
struct Pack {
  const uint16_t* src;
  uint4* dst;
  int64_t lines, ld;
  int len;
  int64_t dst_runs;  // 16-byte runs from line to line of the result
};
__global__ void __launch_bounds__(256) pack_kernel(const Pack first, const Pack second) {
  let_next_start();
  wait_for_previous();
  const Pack& k = blockIdx.y ? second : first;
  const int runs = (int)(((int64_t)k.len + 7) / 8);  // a length may be 2^31 - 1
  const int64_t total = k.lines * runs;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t l = i / runs;
    const int c = (int)(i - l * runs) * 8;
    const uint16_t* p = k.src + l * k.ld + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = c + 2 * j < k.len ? p[2 * j] : 0;
      const uint32_t hi = c + 2 * j + 1 < k.len ? p[2 * j + 1] : 0;
      w[j] = lo | hi << 16;
    }
    k.dst[l * k.dst_runs + c / 8] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// An operand of `lines` lines of `len` elements, and its replacement by a copy
// in the workspace where TMA cannot address it.
struct Operand {
  const void** p;
  int64_t* ld;
  int64_t lines, len;
};
int pack_operands(Operand a, Operand b, uint8_t* ws, int sms, cudaStream_t st) {
  Pack k[2] = {};
  int n = 0;
  int64_t most = 0;
  for (const Operand& o : {a, b}) {
    if (o.lines == 0 || o.len == 0 || tma_lines(*o.p, *o.ld, o.lines)) continue;
    k[n++] = {static_cast<const uint16_t*>(*o.p), reinterpret_cast<uint4*>(ws), o.lines, *o.ld,
              (int)o.len, pitch(o.len) / 8};
    most = std::max(most, o.lines * ((o.len + 7) / 8));
    *o.p = ws;
    *o.ld = pitch(o.len);
    ws += packed_bytes(o.lines, o.len);
  }
  if (n == 0) return CTB_OK;
  const int64_t grid = std::min<int64_t>((most + 255) / 256, 16ll * sms);
  return launch_overlapped("pack_kernel", pack_kernel, dim3((unsigned)grid, n), 256, 0, 0, st, k[0],
                           k[1]);
}

template <typename T>
int product(const Product& p, int sms, cudaStream_t st) {
  if (p.depth > 0) return product_sm100<T>(p, sms, st);
  const int64_t grid = std::min<int64_t>(((int64_t)p.rows * p.cols + 255) / 256, 16ll * sms);
  return launch_overlapped("product_empty_kernel", product_empty_kernel<T>, dim3((unsigned)grid),
                           256, 0, 0, st, p);
}

// ---- dZ = dC .* act'(Z) and its column sums ---------------------------------------------
// One pass over dC and Z, bound by HBM. A warp takes 32 runs of W neighbouring
// columns (16 bytes a lane where the rows allow it), a CTA eight rows at a time
// of one strip, two of them in flight per warp; a lane keeps its columns' sums.
// The strip's rows are split into spans so that every SM has several CTAs'
// worth; spans are summed afterwards in order, so the result does not depend on
// the schedule. Bias gradient of 4096 x 16384 (268 MB read, no dZ written, 41 us
// at the copy rate): 45 us with relu, 53 silu, 58 gelu_tanh, 67 gelu (18
// instructions an element; 2 rows in flight at 4 CTAs an SM measured better than
// 1, and than 4 rows at 2 or 3 CTAs: 68-72 us).
constexpr int SLOPE_THREADS = 256, SLOPE_WARPS = SLOPE_THREADS / 32, SLOPE_FLIGHT = 2;
constexpr int SLOPE_CTAS = 16 * 148;

template <typename T, int W> struct Columns;
template <typename T> struct Columns<T, 8> {
  uint4 raw;
  __device__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ void get(float (&f)[8]) const { unpack8<T>(raw, f); }
  static __device__ void put(T* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = pack8<T>(f);
  }
};
template <typename T> struct Columns<T, 1> {
  T v;
  __device__ void load(const T* p) { v = *p; }
  __device__ void get(float (&f)[1]) const { f[0] = to_f32(v); }
  static __device__ void put(T* p, const float (&f)[1]) { from_f32(p, f[0]); }
};

template <typename T, int W, int ACT>
__global__ void __launch_bounds__(SLOPE_THREADS, 4)
    slope_kernel(const T* dC, const T* Z, T* dZ,
                 float* partial, int N, int M, int64_t lddc, int64_t ldz,
                 int64_t lddz, int span) {
  let_next_start();
  wait_for_previous();
  __shared__ float red[SLOPE_WARPS][32 * W];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c = (int)(blockIdx.x * 32 + lane) * W;
  const int64_t n0 = (int64_t)blockIdx.y * span, n1 = min((int64_t)N, n0 + span);
  float sum[W];
#pragma unroll
  for (int i = 0; i < W; ++i) sum[i] = 0.f;
  if (c < M) {
    for (int64_t n = n0 + warp; n < n1; n += SLOPE_WARPS * SLOPE_FLIGHT) {
      Columns<T, W> d[SLOPE_FLIGHT], z[SLOPE_FLIGHT];
#pragma unroll
      for (int j = 0; j < SLOPE_FLIGHT; ++j) {
        const int64_t r = n + j * SLOPE_WARPS;
        if (r < n1) {
          d[j].load(dC + r * lddc + c);
          if (ACT != CTB_ACT_NONE) z[j].load(Z + r * ldz + c);
        }
      }
#pragma unroll
      for (int j = 0; j < SLOPE_FLIGHT; ++j) {
        const int64_t r = n + j * SLOPE_WARPS;
        if (r < n1) {
          float f[W], s[W];
          d[j].get(f);
          if (ACT != CTB_ACT_NONE) {
            z[j].get(s);
            if (W == 1) {
              float unused = 0.f;
              slope2<ACT>(s[0], unused);
            } else {
#pragma unroll
              for (int i = 0; i + 1 < W; i += 2) slope2<ACT>(s[i], s[i + 1]);
            }
#pragma unroll
            for (int i = 0; i < W; ++i) f[i] *= s[i];
          }
#pragma unroll
          for (int i = 0; i < W; ++i) sum[i] += f[i];
          if (dZ) Columns<T, W>::put(dZ + r * lddz + c, f);
        }
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int i = 0; i < W; ++i) red[warp][lane * W + i] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * W; i += SLOPE_THREADS) {
    const int col = (int)blockIdx.x * 32 * W + i;
    float t = red[0][i];
#pragma unroll
    for (int w = 1; w < SLOPE_WARPS; ++w) t += red[w][i];
    if (col < M) partial[(int64_t)blockIdx.y * M + col] = t;
  }
}

// Sums the spans: 32 columns a CTA, eight threads a column, joined in order.
__global__ void __launch_bounds__(256)
    fold_kernel(const float* partial, float* out, int M, int spans) {
  let_next_start();
  wait_for_previous();
  __shared__ float red[8][32];
  const int cl = threadIdx.x % 32, g = threadIdx.x / 32, c = blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < M)
#pragma unroll 8
    for (int i = g; i < spans; i += 8) s += partial[(int64_t)i * M + c];
  red[g][cl] = s;
  __syncthreads();
  if (g == 0 && c < M) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][cl];
    out[c] = s;
  }
}

// Spans of the rows: 32 rows at least, at most what gives SLOPE_CTAS CTAs.
int spans_of(int N, int M) {
  const int64_t strips = std::max<int64_t>(1, ((int64_t)M + 255) / 256);
  return (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)N + 31) / 32, SLOPE_CTAS / strips));
}

template <typename T, int W>
int slope_launch(const T* dC, const T* Z, T* dZ, float* sums, int N, int M, int64_t lddc,
                 int64_t ldz, int64_t lddz, int act, int spans, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)M + 32 * W - 1) / (32 * W)), spans);
  auto k = slope_kernel<T, W, CTB_ACT_NONE>;
  switch (act) {
    case CTB_ACT_RELU: k = slope_kernel<T, W, CTB_ACT_RELU>; break;
    case CTB_ACT_GELU: k = slope_kernel<T, W, CTB_ACT_GELU>; break;
    case CTB_ACT_GELU_TANH: k = slope_kernel<T, W, CTB_ACT_GELU_TANH>; break;
    case CTB_ACT_SILU: k = slope_kernel<T, W, CTB_ACT_SILU>; break;
    default: break;
  }
  return launch_overlapped("slope_kernel", k, grid, SLOPE_THREADS, 0, 0, st, dC, Z, dZ, sums, N, M,
                           lddc, ldz, lddz, (int)(((int64_t)N + spans - 1) / spans));
}

// dZ goes to the workspace where it is not dC itself: with an activation, or
// where TMA cannot address dC.
bool dz_apart(const void* dC, int64_t lddc, int N, int act) {
  return act != CTB_ACT_NONE || !tma_lines(dC, lddc, N);
}

template <typename T>
int dense_bwd(const T* dC, const T* A, const T* B, const T* Z, T* dA, T* dB, float* dbias, int M,
              int N, int K, int64_t lddc, int64_t lda, int64_t ldb, int64_t ldz, int64_t ldda,
              int64_t lddb, int act, uint8_t* ws, int sms, cudaStream_t st) {
  const void* dZ = dC;
  int64_t lddz = lddc;
  const bool products = (dA || dB) && K > 0;
  const bool apart = products && dz_apart(dC, lddc, N, act);
  if ((apart || dbias) && M > 0) {
    const int spans = spans_of(N, M);
    float* sums = dbias;
    if (dbias && spans > 1) sums = reinterpret_cast<float*>(ws);
    if (dbias) ws += round256(4ll * spans * M);
    T* dz = nullptr;
    if (apart) {
      dz = reinterpret_cast<T*>(ws);
      ws += packed_bytes(N, M);
      dZ = dz;
      lddz = pitch(M);
    }
    const bool runs = M % 8 == 0 && tma_lines(dC, lddc, N) &&
                      (act == CTB_ACT_NONE || tma_lines(Z, ldz, N));
    int rc = runs ? slope_launch<T, 8>(dC, Z, dz, sums, N, M, lddc, ldz, lddz, act, spans, st)
                  : slope_launch<T, 1>(dC, Z, dz, sums, N, M, lddc, ldz, lddz, act, spans, st);
    if (rc) return rc;
    if (dbias && spans > 1) {
      rc = launch_overlapped("fold_kernel", fold_kernel, dim3((unsigned)(((int64_t)M + 31) / 32)), 256, 0, 0,
                             st, sums,
                             dbias, M, spans);
      if (rc) return rc;
    }
  }
  const void *qA = A, *qB = B;
  if (int rc = pack_operands({&qA, &lda, dB ? K : 0, M}, {&qB, &ldb, dA ? N : 0, K}, ws, sms, st))
    return rc;
  if (dB && N > 0 && K > 0) {
    Product p = {};
    p.P = dZ;
    p.ldp = lddz;
    p.Q = qA;
    p.ldq = lda;
    p.D = dB;
    p.ldd = lddb;
    p.rows = N;
    p.cols = K;
    p.depth = M;
    if (int rc = product<T>(p, sms, st)) return rc;
  }
  if (dA && M > 0 && K > 0) {
    Product p = {};
    p.P = qB;
    p.ldp = ldb;
    p.p_mn = true;
    p.Q = dZ;
    p.ldq = lddz;
    p.q_mn = true;
    p.D = dA;
    p.ldd = ldda;
    p.rows = K;
    p.cols = M;
    p.depth = N;
    if (int rc = product<T>(p, sms, st)) return rc;
  }
  return CTB_OK;
}

int dense_check(const char* k, int dtype, int M, int N, int K, int act) {
  const std::string n(k);
  if (dtype != CTB_F16 && dtype != CTB_BF16)
    return set_error(CTB_ERR_DTYPE, n + ": matrices must be Float16 or BFloat16");
  if (M < 0 || N < 0 || K < 0) return set_error(CTB_ERR_SHAPE, n + ": negative size");
  if (act < CTB_ACT_NONE || act > CTB_ACT_SILU)
    return set_error(CTB_ERR_ARG, n + ": unknown activation");
  return CTB_OK;
}

}  // namespace
}  // namespace dense
}  // namespace ctb

using namespace ctb;

extern "C" int64_t ctb_dense_fwd_workspace_bytes(const void* A, const void* B, int32_t M, int32_t N,
                                                 int32_t K, int64_t lda, int64_t ldb) {
  using namespace dense;
  if (M < 0 || N < 0 || K < 0) return -1;
  return (tma_lines(A, lda, K) ? 0 : packed_bytes(K, M)) +
         (tma_lines(B, ldb, N) ? 0 : packed_bytes(N, K));
}

extern "C" int64_t ctb_dense_bwd_workspace_bytes(const void* dC, const void* A, const void* B,
                                                 int32_t M, int32_t N, int32_t K, int64_t lddc,
                                                 int64_t lda, int64_t ldb, int32_t act,
                                                 int32_t need_dbias) {
  using namespace dense;
  if (M < 0 || N < 0 || K < 0) return -1;
  return (need_dbias ? round256(4ll * spans_of(N, M) * M) : 0) +
         (dz_apart(dC, lddc, N, act) ? packed_bytes(N, M) : 0) +
         (tma_lines(A, lda, K) ? 0 : packed_bytes(K, M)) +
         (tma_lines(B, ldb, N) ? 0 : packed_bytes(N, K));
}

extern "C" int ctb_dense_fwd(int32_t dtype, const void* A, const void* B, const void* bias,
                             int32_t bias_dtype, const void* R, void* Z, void* C, int32_t M,
                             int32_t N, int32_t K, int64_t lda, int64_t ldb, int64_t ldr,
                             int64_t ldz, int64_t ldc, int32_t act, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = dense::dense_check("dense", dtype, M, N, K, act)) return rc;
  if (bias && bias_dtype != dtype && bias_dtype != CTB_F32)
    return set_error(CTB_ERR_DTYPE, "dense: the bias must be Float32 or of the matrices' type");
  if (lda < M || ldb < K || ldc < M || (R && ldr < M) || (Z && ldz < M))
    return set_error(CTB_ERR_LAYOUT, "dense: leading dimension smaller than the column length");
  if (M == 0 || N == 0) return CTB_OK;
  if (!C || (K > 0 && (!A || !B))) return set_error(CTB_ERR_ARG, "dense: NULL pointer");
  const int64_t need = ctb_dense_fwd_workspace_bytes(A, B, M, N, K, lda, ldb);
  const Lines a = lines_of(A, K, M, lda, 2), b = lines_of(B, N, K, ldb, 2),
              bi = bytes_of(bias, (bias_dtype == CTB_F32 ? 4ll : 2ll) * M),
              r = lines_of(R, N, M, ldr, 2), z = lines_of(Z, N, M, ldz, 2),
              c = lines_of(C, N, M, ldc, 2), w = bytes_of(workspace, need);
  if (!apart(c, {a, b, bi, z, w}) || !(same_place(c, r) || apart(c, {r})) ||
      !apart(z, {a, b, bi, r, w}) || !apart(w, {a, b, bi, r}))
    return set_error(CTB_ERR_ARG, "dense: C, Z and the workspace must be memory of their own (C may "
                                  "be R, with the same leading dimension)");
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(CTB_ERR_ARG, "dense: the workspace needs " + std::to_string(need) +
                                      " bytes, 16-byte aligned");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  dense::Product p = {};
  p.P = B;
  p.ldp = ldb;
  p.Q = A;
  p.ldq = lda;
  p.q_mn = true;
  p.D = C;
  p.ldd = ldc;
  p.rows = N;
  p.cols = M;
  p.depth = K;
  p.bias = bias;
  p.bias_f32 = bias_dtype == CTB_F32;
  p.act = act;
  p.R = R;
  p.ldr = ldr;
  p.Z = Z;
  p.ldz = ldz;
  auto st = static_cast<cudaStream_t>(stream);
  auto* ws = static_cast<uint8_t*>(workspace);
  if (int rc = dense::pack_operands({&p.P, &p.ldp, N, K}, {&p.Q, &p.ldq, K, M}, ws, pr.sm_count, st))
    return rc;
  return dtype == CTB_F16 ? dense::product<__half>(p, pr.sm_count, st)
                          : dense::product<__nv_bfloat16>(p, pr.sm_count, st);
}

extern "C" int ctb_dense_bwd(int32_t dtype, const void* dC, const void* A, const void* B,
                             const void* Z, void* dA, void* dB, float* dbias, int32_t M, int32_t N,
                             int32_t K, int64_t lddc, int64_t lda, int64_t ldb, int64_t ldz,
                             int64_t ldda, int64_t lddb, int32_t act, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = dense::dense_check("dense_bwd", dtype, M, N, K, act)) return rc;
  const bool slope = act != CTB_ACT_NONE;
  if (lddc < M || (dB && lda < M) || (dA && ldb < K) || (slope && ldz < M) || (dA && ldda < M) ||
      (dB && lddb < K))
    return set_error(CTB_ERR_LAYOUT, "dense_bwd: leading dimension smaller than the column length");
  const bool some = M > 0 && N > 0;
  if ((some && (!dC || (slope && !Z))) || (some && K > 0 && ((dB && !A) || (dA && !B))))
    return set_error(CTB_ERR_ARG, "dense_bwd: NULL pointer");
  const int64_t need = ctb_dense_bwd_workspace_bytes(dC, A, B, M, N, K, lddc, lda, ldb, act,
                                                     dbias != nullptr);
  // Operands that are read: Z where there is an activation, A for dB, B for dA.
  const Lines c = lines_of(dC, N, M, lddc, 2), z = lines_of(slope ? Z : nullptr, N, M, ldz, 2),
              a = lines_of(dB ? A : nullptr, K, M, lda, 2),
              b = lines_of(dA ? B : nullptr, N, K, ldb, 2), oa = lines_of(dA, K, M, ldda, 2),
              ob = lines_of(dB, N, K, lddb, 2), obi = bytes_of(dbias, 4ll * M),
              w = bytes_of(workspace, need);
  if (!apart(oa, {c, z, a, b, ob, obi, w}) || !apart(ob, {c, z, a, b, obi, w}) ||
      !apart(obi, {c, z, a, b, w}) || !apart(w, {c, z, a, b}))
    return set_error(CTB_ERR_ARG,
                     "dense_bwd: gradients and the workspace must be memory of their own");
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(CTB_ERR_ARG, "dense_bwd: the workspace needs " + std::to_string(need) +
                                      " bytes, 16-byte aligned");
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  auto* ws = static_cast<uint8_t*>(workspace);
  if (dtype == CTB_F16)
    return dense::dense_bwd<__half>((const __half*)dC, (const __half*)A, (const __half*)B,
                                    (const __half*)Z, (__half*)dA, (__half*)dB, dbias, M, N, K,
                                    lddc, lda, ldb, ldz, ldda, lddb, act, ws, pr.sm_count, st);
  using bf = __nv_bfloat16;
  return dense::dense_bwd<bf>((const bf*)dC, (const bf*)A, (const bf*)B, (const bf*)Z, (bf*)dA,
                              (bf*)dB, dbias, M, N, K, lddc, lda, ldb, ldz, ldda, lddb, act, ws,
                              pr.sm_count, st);
}
