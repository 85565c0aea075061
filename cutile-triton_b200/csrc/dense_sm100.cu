// Matrix products of the dense layer (dense.cuh: Product) on the 5th-generation
// tensor cores.
//
// product_split_kernel: one 128 (columns of D) x BN (rows of D) tile per cluster
// of S CTAs, each CTA summing its own run of 64-deep k-blocks. The columns are
// the tensor cores' M side, so that a few tokens cost a tile of 16 rows and
// not of 128: the weight is then streamed once at memory speed, split over k so
// that every SM has its share. Each CTA keeps its partial tile in its own
// shared memory (Float32); the CTAs of a cluster then read one another's
// partials over distributed shared memory and add them in rank order, each
// finishing (bias, activation, residual, rounding) its share of the tile. No
// workspace, no atomics, the same result every time.
#include "dense.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <mutex>

namespace ctb {
namespace dense {

constexpr unsigned ERR_BIT = 64u;
constexpr int BK = 64;  // k-block: one 128-byte swizzled row of 16-bit elements

// ---- epilogue of 8 neighbouring columns of one row ---------------------------------
struct Epilogue {
  const void* bias;
  const void* R;
  void* Z;
  void* D;
  int64_t ldr, ldz, ldd;
  int rows, cols;
  int act;
  bool bias_f32;
  bool vec;  // D (and Z, R) rows are whole 16-byte runs
};

template <typename T, int ACT>
__device__ __forceinline__ void activate8(float (&z)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = activate<ACT>(z[i]);
}
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t r, int c, float (&z)[8]) {
  const int n = min(8, e.cols - c);
  if (e.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n)
        z[i] += e.bias_f32 ? static_cast<const float*>(e.bias)[c + i]
                           : to_f32(static_cast<const T*>(e.bias)[c + i]);
  }
  const bool whole = e.vec && n == 8;
  if (e.Z) {
    T* zp = static_cast<T*>(e.Z) + r * e.ldz + c;
    if (whole) {
      *reinterpret_cast<uint4*>(zp) = pack8<T>(z);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) from_f32(zp + i, z[i]);
    }
  }
  switch (e.act) {
    case CTB_ACT_RELU: activate8<T, CTB_ACT_RELU>(z); break;
    case CTB_ACT_GELU: activate8<T, CTB_ACT_GELU>(z); break;
    case CTB_ACT_GELU_TANH: activate8<T, CTB_ACT_GELU_TANH>(z); break;
    case CTB_ACT_SILU: activate8<T, CTB_ACT_SILU>(z); break;
    default: break;
  }
  if (e.R) {
    const T* rp = static_cast<const T*>(e.R) + r * e.ldr + c;
    if (whole) {
      float f[8];
      unpack8<T>(*reinterpret_cast<const uint4*>(rp), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += f[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) z[i] += to_f32(rp[i]);
    }
  }
  T* dp = static_cast<T*>(e.D) + r * e.ldd + c;
  if (whole) {
    *reinterpret_cast<uint4*>(dp) = pack8<T>(z);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) from_f32(dp + i, z[i]);
  }
}

template <typename T> struct Format;
template <> struct Format<__half> {
  static constexpr uint32_t idesc = 0;
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
};
template <> struct Format<__nv_bfloat16> {
  static constexpr uint32_t idesc = (1u << 7) | (1u << 10);  // A and B are BF16
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
};

// ---- split kernel --------------------------------------------------------------------
constexpr int SP_COLS = 128;
constexpr int SP_THREADS = 128;
constexpr int SP_Q_BYTES = SP_COLS * BK * 2;
// Stages for about 96 KB, so that two CTAs share an SM: one's epilogue runs
// under the other's loads.
__host__ __device__ constexpr int sp_stages(int BN) { return BN <= 32 ? 5 : BN == 64 ? 4 : 3; }
__host__ __device__ constexpr int sp_stage_bytes(int BN) { return SP_Q_BYTES + BN * BK * 2; }
constexpr int sp_smem(int BN) { return sp_stages(BN) * sp_stage_bytes(BN) + 1024 + 256; }

struct SplitArgs {
  Epilogue e;
  int num_kb;  // k-blocks of the whole product
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// A producer that gave up waits (for at most a second each) until the loads it
// has issued have landed, so that none outlives the CTA.
__device__ __noinline__ void drain_loads(uint64_t* full, int64_t issued, int stages) {
  const int64_t from = issued > stages ? issued - stages : 0;
  for (int64_t i = from; i < issued; ++i) {
    const uint64_t t0 = sm100::global_ns();
    while (!sm100::mbar_try_wait_sleep(&full[i % stages], (uint32_t)((i / stages) & 1), 20000u) &&
           sm100::global_ns() - t0 < 1000000000ull) {
    }
  }
}

template <typename T, bool Q_MN, bool P_MN, int BN>
__global__ void __launch_bounds__(SP_THREADS, 2)
    product_split_kernel(const __grid_constant__ CUtensorMap tmQ,
                         const __grid_constant__ CUtensorMap tmP, const SplitArgs a) {
  using namespace sm100;
  static_assert(!P_MN || BN >= 64, "a row-major-k box is 64 rows wide");
  constexpr int STAGES = sp_stages(BN);
  constexpr int STAGE_BYTES = sp_stage_bytes(BN);
  constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* partial = reinterpret_cast<float*>(smem);  // [BN][128], once the stages are consumed
  static_assert(BN * SP_COLS * 4 <= STAGES * STAGE_BYTES, "the partial tile reuses the stages");
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t S = cluster_nctarank(), rank = cluster_ctarank();
  const int c0 = (int)(blockIdx.x / S) * SP_COLS;
  const int64_t r0 = (int64_t)blockIdx.y * BN;
  const int kb0 = (int)((int64_t)a.num_kb * rank / S);
  const int kb1 = (int)((int64_t)a.num_kb * (rank + 1) / S);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmP);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, kb = kb0;
      uint32_t phase = 0;
      for (; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, ERR_BIT)) break;
        uint8_t* sq = smem + stage * STAGE_BYTES;
        uint8_t* sp = sq + SP_Q_BYTES;
        mbar_arrive_expect_tx(&full[stage], STAGE_BYTES);
        if (Q_MN) {
          tma_load_2d(sq, &tmQ, &full[stage], c0, kb * BK);
          tma_load_2d(sq + 64 * BK * 2, &tmQ, &full[stage], c0 + 64, kb * BK);
        } else {
          tma_load_2d(sq, &tmQ, &full[stage], kb * BK, c0);
        }
        if (P_MN) {
#pragma unroll
          for (int i = 0; i < BN / 64; ++i)
            tma_load_2d(sp + i * 64 * BK * 2, &tmP, &full[stage], (int)r0 + 64 * i, kb * BK);
        } else {
          tma_load_2d(sp, &tmP, &full[stage], kb * BK, (int)r0);
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (kb < kb1) drain_loads(full, kb - kb0, STAGES);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_f16_f32(SP_COLS, BN, Q_MN, P_MN) | Format<T>::idesc;
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], phase, abort_flag, ERR_BIT)))
        break;
      tc_fence_after();
      const uint32_t sq = smem_u32(smem + stage * STAGE_BYTES);
      // Row-major-k operand: LBO = 8 KB between 64-row boxes, SBO = 1 KB between
      // groups of 8 k; 16 k = 2 KB. K-major operand: SBO = 1 KB between groups
      // of 8 rows; 16 k = 32 bytes inside the swizzled row.
      const uint64_t qd = smem_desc_sw128(sq, Q_MN ? 8192 : 16, 1024);
      const uint64_t pd = smem_desc_sw128(sq + SP_Q_BYTES, P_MN ? 8192 : 16, 1024);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k)
        mma_f16_ss_elect(tmem, qd + (uint64_t)((Q_MN ? 2048 : 32) * k >> 4),
                         pd + (uint64_t)((P_MN ? 2048 : 32) * k >> 4), idesc,
                         kb > kb0 || k > 0);
      mma_commit_elect(&empty[stage]);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    mma_commit_elect(done);
  }
  // All roles meet at the finished accumulator. It exists on the way out of a
  // wait that gave up too; the host is told by the error word.
  mbar_wait_bounded(done, 0, abort_flag, ERR_BIT);
  __syncwarp();
  tc_fence_after();
  const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
  if (BN >= 32) {
#pragma unroll 1
    for (int r = 0; r < BN; r += 32) {
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + lane_base + r, v);
      tmem_ld_wait_regs(v);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        partial[(r + j) * SP_COLS + threadIdx.x] = __uint_as_float(v[j]);
    }
  } else {
    uint32_t v[16];
    tmem_ld_32x32b_x16(tmem + lane_base, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) partial[j * SP_COLS + threadIdx.x] = __uint_as_float(v[j]);
  }
  tc_fence_before();
  if (S > 1) cluster_sync_all();
  else __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }

  const uint32_t mine = smem_u32(partial);
  const int live_rows = (int)min((int64_t)BN, a.e.rows - r0);
  for (int i = (int)rank * SP_THREADS + threadIdx.x; i < live_rows * (SP_COLS / 8);
       i += (int)S * SP_THREADS) {
    const int r = i / (SP_COLS / 8), c = i % (SP_COLS / 8) * 8;
    if (c0 + c >= a.e.cols) continue;
    float z[8] = {};
    for (uint32_t s = 0; s < S; ++s) {
      const uint32_t from = mapa_shared(mine, s) + (uint32_t)(r * SP_COLS + c) * 4;
      const float4 lo = ld_cluster_f4(from), hi = ld_cluster_f4(from + 16);
      z[0] += lo.x;
      z[1] += lo.y;
      z[2] += lo.z;
      z[3] += lo.w;
      z[4] += hi.x;
      z[5] += hi.y;
      z[6] += hi.z;
      z[7] += hi.w;
    }
    finish8<T>(a.e, r0 + r, c0 + c, z);
  }
  if (S > 1) cluster_sync_all();  // no CTA leaves while a peer may read its partials
}

// ---- host ------------------------------------------------------------------------------
static unsigned long long g_dense_ctx[64];  // context ID the set-up was done in
static std::mutex g_dense_mu;

template <typename T, bool Q_MN, bool P_MN, int BN>
int split_attr() {
  CTB_CUDA_CHECK(cudaFuncSetAttribute(product_split_kernel<T, Q_MN, P_MN, BN>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, sp_smem(BN)));
  return CTB_OK;
}
template <typename T>
int split_attrs() {
  int rc = CTB_OK;
  if (!rc) rc = split_attr<T, true, false, 16>();
  if (!rc) rc = split_attr<T, true, false, 32>();
  if (!rc) rc = split_attr<T, true, false, 64>();
  if (!rc) rc = split_attr<T, true, false, 128>();
  if (!rc) rc = split_attr<T, false, false, 16>();
  if (!rc) rc = split_attr<T, false, false, 32>();
  if (!rc) rc = split_attr<T, false, false, 64>();
  if (!rc) rc = split_attr<T, false, false, 128>();
  if (!rc) rc = split_attr<T, true, true, 64>();
  if (!rc) rc = split_attr<T, true, true, 128>();
  return rc;
}

int device_setup() {
  int dev = 0;
  CTB_CUDA_CHECK(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(g_dense_mu);
  unsigned long long ctx = 0;
  if (int rc = current_context_id(&ctx)) return rc;
  if (dev < 64 && g_dense_ctx[dev] == ctx) return CTB_OK;
  if (int rc = split_attrs<__half>()) return rc;
  if (int rc = split_attrs<__nv_bfloat16>()) return rc;
  if (dev < 64) g_dense_ctx[dev] = ctx;
  return CTB_OK;
}

// An operand of `extent` rows and `depth` k as boxes of 64 k x box_rows rows
// (k-major) or 64 rows x 64 k.
template <typename T>
int operand_map(CUtensorMap* m, const void* base, int64_t ld, bool mn, int extent, int depth,
                int box_rows) {
  const uint64_t dims[2] = {(uint64_t)(mn ? extent : depth), (uint64_t)(mn ? depth : extent)};
  const uint64_t strides[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {64, (uint32_t)(mn ? 64 : box_rows)};
  return encode_tmap(m, Format<T>::map, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

static bool rows16(const void* p, int64_t ld, int rows) {
  return aligned16(p) && (ld % 8 == 0 || rows <= 1);
}

template <typename T, bool Q_MN, bool P_MN, int BN>
int split_launch(const Product& p, const Epilogue& e, int sms, cudaStream_t st) {
  CUtensorMap tmQ, tmP;
  if (int rc = operand_map<T>(&tmQ, p.Q, p.ldq, Q_MN, p.cols, p.depth, SP_COLS)) return rc;
  if (int rc = operand_map<T>(&tmP, p.P, p.ldp, P_MN, p.rows, p.depth, BN)) return rc;
  SplitArgs a;
  a.e = e;
  a.num_kb = (p.depth + BK - 1) / BK;
  const int64_t tiles_c = (p.cols + SP_COLS - 1) / SP_COLS, tiles_r = ((int64_t)p.rows + BN - 1) / BN;
  if (tiles_r > 65535) return set_error(CTB_ERR_SHAPE, "dense: too many rows");
  // As many CTAs per tile as fill two per SM once, with 2 k-blocks each at least.
  int S = (int)std::max<int64_t>(1, std::min<int64_t>(8, 2ll * sms / (tiles_c * tiles_r)));
  S = std::max(1, std::min(S, a.num_kb / 2));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(tiles_c * S), (unsigned)tiles_r, 1);
  cfg.blockDim = dim3(SP_THREADS, 1, 1);
  cfg.dynamicSmemBytes = sp_smem(BN);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, product_split_kernel<T, Q_MN, P_MN, BN>, tmQ, tmP, a));
  return launch_status("product_split_kernel");
}

// The product on the tensor cores. Operands start on 16-byte boundaries, their
// leading dimensions are multiples of 8 (or they have one line only); depth > 0.
template <typename T>
int product_sm100(const Product& p0, cudaStream_t st) {
  DeviceProps pr;
  if (int rc = current_props(&pr)) return rc;
  if (int rc = device_setup()) return rc;
  Product p = p0;
  // The distance between lines does not matter where there is one: any that TMA takes.
  if ((p.p_mn ? p.depth : p.rows) == 1) p.ldp = ((p.p_mn ? p.rows : p.depth) + 7) / 8 * 8;
  if ((p.q_mn ? p.depth : p.cols) == 1) p.ldq = ((p.q_mn ? p.cols : p.depth) + 7) / 8 * 8;
  Epilogue e;
  e.bias = p.bias;
  e.R = p.R;
  e.Z = p.Z;
  e.D = p.D;
  e.ldr = p.ldr;
  e.ldz = p.ldz;
  e.ldd = p.ldd;
  e.rows = p.rows;
  e.cols = p.cols;
  e.act = p.act;
  e.bias_f32 = p.bias_f32;
  e.vec = rows16(p.D, p.ldd, p.rows) && (!p.Z || rows16(p.Z, p.ldz, p.rows)) &&
          (!p.R || rows16(p.R, p.ldr, p.rows));
  const int sms = pr.sm_count;
  if (p.p_mn) {
    if (p.rows <= 64) return split_launch<T, true, true, 64>(p, e, sms, st);
    return split_launch<T, true, true, 128>(p, e, sms, st);
  }
  if (p.q_mn) {
    if (p.rows <= 16) return split_launch<T, true, false, 16>(p, e, sms, st);
    if (p.rows <= 32) return split_launch<T, true, false, 32>(p, e, sms, st);
    if (p.rows <= 64) return split_launch<T, true, false, 64>(p, e, sms, st);
    return split_launch<T, true, false, 128>(p, e, sms, st);
  }
  if (p.rows <= 16) return split_launch<T, false, false, 16>(p, e, sms, st);
  if (p.rows <= 32) return split_launch<T, false, false, 32>(p, e, sms, st);
  if (p.rows <= 64) return split_launch<T, false, false, 64>(p, e, sms, st);
  return split_launch<T, false, false, 128>(p, e, sms, st);
}
template int product_sm100<__half>(const Product&, cudaStream_t);
template int product_sm100<__nv_bfloat16>(const Product&, cudaStream_t);

}  // namespace dense

int dense_take_device_error(unsigned int* out) { return take_device_error(out); }
}  // namespace ctb
