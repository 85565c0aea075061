// Matrix products of the dense layer (dense.cuh: Product) on the 5th-generation
// tensor cores.
//
// product_split_kernel: one 128 (columns of D) x BN (rows of D) tile per cluster
// of S CTAs, each CTA summing its own run of 64-deep k-blocks. The columns are
// the tensor cores' M side, so that a few tokens cost a tile of 16 rows and
// not of 128: the weight is then streamed once at memory speed, split over k so
// that every SM has its share. Each CTA keeps its partial tile in its own
// shared memory (Float32); the CTAs of a cluster then read one another's
// partials over distributed shared memory (tiles of up to 32 rows: send them to
// the row's owner) and add them in rank order, each finishing (bias, activation,
// residual, rounding) its share of the tile. No workspace, no atomics, the same
// result every time. Bound by HBM from some tens of MB of weight up (37 x 14336 x
// 4096 bf16: 23 us, 5.2 TB/s), below that by set-up, first load and the joining
// of the sums (1 x 4096 x 4096 f16: 8.0 us, 4.2 TB/s; 64 x 1024 x 1024: 4.2 us).
//
// product_pair_kernel: 256 x 256 tiles over two SMs (tcgen05 cta_group::2),
// persistent, for products with tiles enough to fill the GPU. Here the rows of D
// are the tensor cores' M side: a thread of the epilogue then holds neighbouring
// columns of one row, which move through swizzled shared memory as 16-byte
// pieces and in and out of it by TMA, and the bias is the same for all lanes.
// Bound by the tensor pipe, in long runs by the power cap: 8192 x 14336 x 4096 bf16
// with bias, gelu and Z 726 to 756 us back to back (1325 to 1272 TFLOP/s, from one
// GPU to another), 673 without an epilogue (1430); 4096 x 4096 x 1024 bf16 29 us, 33
// with gelu, 41 with bias, gelu and Z.
#include "dense.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <mutex>

namespace ctb {
namespace dense {

constexpr unsigned ERR_BIT = 64u;
constexpr int BK = 64;  // k-block: one 128-byte swizzled row of 16-bit elements

// ---- epilogue -------------------------------------------------------------------------
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
  for (int i = 0; i < 8; i += 2) activate2<ACT>(z[i], z[i + 1]);
}
// 8 neighbouring columns of one row, of matrices whose rows are 16-byte runs; the
// last run of a row may be short.
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t r, int c, float (&z)[8],
                                        const float (&bias)[8]) {
  const int n = min(8, e.cols - c);
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] += bias[i];
  const bool whole = n == 8;
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

// One element, its bias added, and its residual.
template <typename T>
__device__ __forceinline__ void finish1(const Epilogue& e, int64_t r, int c, float z,
                                        float residual) {
  if (e.Z) from_f32(static_cast<T*>(e.Z) + r * e.ldz + c, z);
  from_f32(static_cast<T*>(e.D) + r * e.ldd + c, activate_any(z, e.act) + residual);
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
__host__ __device__ constexpr int sp_stages(int BN) { return BN == 16 ? 5 : BN <= 64 ? 4 : 3; }
__host__ __device__ constexpr int sp_stage_bytes(int BN) { return SP_Q_BYTES + BN * BK * 2; }
// Tiles of up to 32 rows: room for the partial sums that the cluster's CTAs send (at
// most BN + 7 rows, when BN rows are split over up to 8 owners).
__host__ __device__ constexpr int sp_inbox_bytes(int BN) {
  return BN <= 32 ? (BN + 7) * SP_COLS * 4 : 0;
}
constexpr int sp_smem(int BN) {
  return sp_stages(BN) * sp_stage_bytes(BN) + sp_inbox_bytes(BN) + 1024 + 256;
}

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
__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&v)[32]) {
  sm100::tmem_ld_32x32b_x32(addr, v);
}
__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&v)[16]) {
  sm100::tmem_ld_32x32b_x16(addr, v);
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
  float* inbox = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);  // [S][owned rows][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + sp_inbox_bytes(BN));
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint64_t* received = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t S = cluster_nctarank(), rank = cluster_ctarank();
  const int c0 = (int)(blockIdx.x / S) * SP_COLS;
  const int64_t r0 = (int64_t)blockIdx.y * BN;
  const int kb0 = (int)((int64_t)a.num_kb * rank / S);
  const int kb1 = (int)((int64_t)a.num_kb * (rank + 1) / S);
  const int live_rows = (int)min((int64_t)BN, a.e.rows - r0);
  // Tiles of up to 32 rows (a few tokens) are finished by owners: CTA r of the cluster
  // owns `each` rows from r * each on, and the others send it their partial sums
  // of those, counted on its barrier. That is one way over distributed shared
  // memory instead of a barrier, a read and a closing barrier (1 x 4096 x 4096:
  // 0.25 + 0.6 us instead of 0.85 + 0.25 + 0.8).
  const bool send = BN <= 32 && S > 1;
  const int each = (live_rows + (int)S - 1) / (int)S;
  const int owned = max(0, min(each, live_rows - (int)rank * each));

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmP);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(received, 1);
    *abort_flag = 0;
    fence_mbar_init();
    if (send && owned > 0)
      mbar_arrive_expect_tx(received, S * (uint32_t)owned * SP_COLS * 4);
  }
  if (warp == 2) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (send) cluster_arrive();  // this CTA's inbox is ready
  let_next_start();
  wait_for_previous();

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
  // A thread's columns are the same for all its rows: 8 neighbours of one of 16
  // runs, or (rows that are no 16-byte runs) lane, lane + 32, ...
  const int c = a.e.vec ? (int)(threadIdx.x % (SP_COLS / 8)) * 8 : lane;
  const int step = a.e.vec ? 1 : 32;
  float bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t at = (int64_t)c0 + c + i * step;
    bias[i] = !a.e.bias || at >= a.e.cols || (!a.e.vec && i >= SP_COLS / 32) ? 0.f
              : a.e.bias_f32 ? static_cast<const float*>(a.e.bias)[at]
                             : to_f32(static_cast<const T*>(a.e.bias)[at]);
  }
  // All roles meet at the finished accumulator. It exists on the way out of a
  // wait that gave up too; the host is told by the error word.
  mbar_wait_bounded(done, 0, abort_flag, ERR_BIT);
  __syncwarp();
  tc_fence_after();
  const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
  if (send) cluster_wait();  // every CTA's inbox is ready
  uint32_t owner = 0;
  int k = 0;  // the next row is row k of the owner's
  constexpr int AT_ONCE = BN < 32 ? BN : 32;
#pragma unroll 1
  for (int r = 0; r < BN; r += AT_ONCE) {
    uint32_t v[AT_ONCE];
    tmem_ld_rows(tmem + lane_base + r, v);
    tmem_ld_wait_regs(v);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (!send) {
        partial[(r + j) * SP_COLS + threadIdx.x] = __uint_as_float(v[j]);
      } else if (r + j < live_rows) {
        const int row = (int)rank * min(each, live_rows - (int)owner * each) + k;
        st_async_cluster(mapa_shared(smem_u32(inbox + row * SP_COLS + threadIdx.x), owner), v[j],
                         mapa_shared(smem_u32(received), owner));
        if (++k == each) {
          k = 0;
          ++owner;
        }
      }
    }
  }
  tc_fence_before();
  if (S > 1 && !send) cluster_sync_all();
  else __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  // Every CTA sends, also one whose pipeline gave up (after 4 s without progress).
  if (send && owned > 0) wait_received(received, abort_flag, ERR_BIT, 12000000000ull);

  const uint32_t mine = smem_u32(partial);
  const int first_row = send ? (int)rank * each : 0, end_row = send ? first_row + owned : live_rows;
  const int shares = send ? 1 : (int)S, share = send ? 0 : (int)rank;  // of the rows of a tile
  if (!a.e.vec) {
    // A warp per row, so that the 2-byte accesses of a row stay together, four
    // rows' residuals asked for at a time.
    constexpr int WARPS = SP_THREADS / 32, FLIGHT = 4, EACH = SP_COLS / 32;
    for (int rb = first_row + share * WARPS + warp; rb < end_row; rb += shares * WARPS * FLIGHT) {
      T res[FLIGHT][EACH];
      if (a.e.R) {
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j)
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            const int r = rb + j * shares * WARPS, col = c0 + i * 32 + lane;
            if (r < end_row && col < a.e.cols)
              res[j][i] = static_cast<const T*>(a.e.R)[(r0 + r) * a.e.ldr + col];
          }
      }
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        const int r = rb + j * shares * WARPS;
        if (r >= end_row) break;
        float z[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) z[i] = 0.f;
        for (uint32_t s = 0; s < S; ++s) {
          const int at = r * SP_COLS + lane;
          const float* sent = inbox + ((int)s * owned + r - first_row) * SP_COLS + lane;
          const uint32_t from = mapa_shared(mine, s) + (uint32_t)at * 4;
#pragma unroll
          for (int i = 0; i < EACH; ++i)
            z[i] += send ? sent[i * 32]
                    : s == rank ? partial[at + i * 32] : ld_cluster_f1(from + i * 128);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int col = c0 + i * 32 + lane;
          if (col < a.e.cols)
            finish1<T>(a.e, r0 + r, col, z[i] + bias[i], a.e.R ? to_f32(res[j][i]) : 0.f);
        }
      }
    }
  }
  for (int r = first_row + (share * SP_THREADS + (int)threadIdx.x) / (SP_COLS / 8);
       a.e.vec && r < end_row && c0 + c < a.e.cols; r += shares * (SP_THREADS / (SP_COLS / 8))) {
    float z[8] = {};
    for (uint32_t s = 0; s < S; ++s) {
      float4 lo, hi;
      if (send || s == rank) {
        const float4* from = reinterpret_cast<const float4*>(
            send ? inbox + ((int)s * owned + r - first_row) * SP_COLS + c
                 : partial + r * SP_COLS + c);
        lo = from[0];
        hi = from[1];
      } else {
        const uint32_t from = mapa_shared(mine, s) + (uint32_t)(r * SP_COLS + c) * 4;
        lo = ld_cluster_f4(from);
        hi = ld_cluster_f4(from + 16);
      }
      z[0] += lo.x;
      z[1] += lo.y;
      z[2] += lo.z;
      z[3] += lo.w;
      z[4] += hi.x;
      z[5] += hi.y;
      z[6] += hi.z;
      z[7] += hi.w;
    }
    finish8<T>(a.e, r0 + r, c0 + c, z, bias);
  }
  if (S > 1 && !send) cluster_sync_all();  // no CTA leaves while a peer may read its partials
}

// ---- pair kernel -----------------------------------------------------------------------
// Warps: 0 TMA producer, 1 TMEM owner and MMA issuer (even CTA), 2..9 epilogue:
// two per quarter of the TMEM lanes, 128 columns each, so that an activation of
// 40 instructions an element still hides under a main loop of 1024 k.
// Each CTA loads its own 128 rows of P and 128 columns of Q (32 KB a k-block, 5
// stages); two 256-column accumulators let a tile's epilogue run under the next
// tile's main loop. Barriers as in gemm_sm100.cu: full[] and tmem_empty[] in the
// even CTA, empty[] and tmem_full[] in both.
constexpr int PR_THREADS = 320;
constexpr int PR_STAGES = 5;
constexpr int PR_OP_BYTES = 128 * BK * 2;
constexpr int PR_STAGE_BYTES = 2 * PR_OP_BYTES;
constexpr int PR_WARPS = 8;                   // epilogue warps
constexpr int PR_BOX = 32 * 32 * 2;           // 32 rows x 32 columns, 64-byte swizzle
constexpr int PR_BOXES = 4;                   // per warp: 2 for stores, 2 for the residual
constexpr int PR_SMEM = PR_STAGES * PR_STAGE_BYTES + PR_WARPS * PR_BOXES * PR_BOX +
                        PR_WARPS * 32 * 4 + 1024 + 512;
constexpr int PR_GROUP = 16;  // row tiles per group of the tile order (8: as fast; 4, 32: 5 to 13% slower)

struct PairArgs {
  Epilogue e;
  int num_kb, tiles_r, tiles_c;
  int64_t num_tiles;
  bool d_tma, z_tma, r_tma;
};

__device__ __forceinline__ void pair_tile(const PairArgs& p, int64_t t, int& tr, int& tc) {
  const int64_t span = (int64_t)PR_GROUP * p.tiles_c;
  const int64_t g = t / span;
  const int first = (int)g * PR_GROUP;
  const int size = min(p.tiles_r - first, PR_GROUP);
  const int rest = (int)(t - g * span);
  tr = first + rest % size;
  tc = rest / size;
}

// Byte offset of 16-byte piece `piece` (0..3) of row `row` in a 64-byte-swizzled box.
__device__ __forceinline__ int box_at(int row, int piece) {
  return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}

template <typename T, int ACT>
__device__ __forceinline__ void activate32(uint32_t (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float x = __uint_as_float(v[j]), y = __uint_as_float(v[j + 1]);
    activate2<ACT>(x, y);
    v[j] = __float_as_uint(x);
    v[j + 1] = __float_as_uint(y);
  }
}

template <typename T, bool P_MN, bool Q_MN>
__global__ void __launch_bounds__(PR_THREADS, 1)
    product_pair_kernel(const __grid_constant__ CUtensorMap tmP,
                        const __grid_constant__ CUtensorMap tmQ,
                        const __grid_constant__ CUtensorMap tmD,
                        const __grid_constant__ CUtensorMap tmZ,
                        const __grid_constant__ CUtensorMap tmR, const PairArgs a) {
  using namespace sm100;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* boxes = smem + PR_STAGES * PR_STAGE_BYTES;
  float* bias_all = reinterpret_cast<float*>(boxes + PR_WARPS * PR_BOXES * PR_BOX);
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_all + PR_WARPS * 32);
  uint64_t* empty = full + PR_STAGES;
  uint64_t* tmem_full = empty + PR_STAGES;  // [2]
  uint64_t* tmem_empty = tmem_full + 2;     // [2]
  uint64_t* r_full = tmem_empty + 2;        // [PR_WARPS][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(r_full + 2 * PR_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int64_t pair = blockIdx.x / 2, num_pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < PR_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], 2 * PR_WARPS * 32);
    }
    for (int i = 0; i < 2 * PR_WARPS; ++i) mbar_init(&r_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmP);
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  cluster_sync_all();  // barriers initialised in both CTAs before any cross-CTA use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  let_next_start();
  wait_for_previous();
  const uint32_t full_leader = mapa_shared(smem_u32(&full[0]), 0);

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      bool ok = true;
      for (int64_t t = pair; ok && t < a.num_tiles && !*abort_flag; t += num_pairs) {
        int tr, tc;
        pair_tile(a, t, tr, tc);
        const int r0 = tr * 256 + (int)rank * 128, c0 = tc * 256 + (int)rank * 128;
        for (int kb = 0; kb < a.num_kb; ++kb) {
          if (!(ok = mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, ERR_BIT))) break;
          uint8_t* sp = smem + stage * PR_STAGE_BYTES;
          uint8_t* sq = sp + PR_OP_BYTES;
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * PR_STAGE_BYTES);
          const uint32_t bar = full_leader + stage * 8;
          if (P_MN) {
            tma_load_2d_pair(sp, &tmP, bar, r0, kb * BK);
            tma_load_2d_pair(sp + PR_OP_BYTES / 2, &tmP, bar, r0 + 64, kb * BK);
          } else {
            tma_load_2d_pair(sp, &tmP, bar, kb * BK, r0);
          }
          if (Q_MN) {
            tma_load_2d_pair(sq, &tmQ, bar, c0, kb * BK);
            tma_load_2d_pair(sq + PR_OP_BYTES / 2, &tmQ, bar, c0 + 64, kb * BK);
          } else {
            tma_load_2d_pair(sq, &tmQ, bar, kb * BK, c0);
          }
          ++issued;
          if (++stage == PR_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // The even CTA's barriers count both CTAs' loads; the other stays until
      // the cluster barrier below.
      if (*abort_flag && leader) drain_loads(full, issued, PR_STAGES);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA only) ----------------
    if (leader) {
      constexpr uint32_t idesc = idesc_f16_f32(256, 256, P_MN, Q_MN) | Format<T>::idesc;
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int64_t t = pair; ok && t < a.num_tiles; t += num_pairs, ++it) {
        const int buf = it & 1;
        const uint32_t acc_phase = (it >> 1) & 1;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&tmem_empty[buf], acc_phase ^ 1,
                                                             abort_flag, ERR_BIT))))
          break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * 256;
        for (int kb = 0; kb < a.num_kb; ++kb) {
          if (!(ok = __all_sync(0xffffffffu,
                                mbar_wait_bounded(&full[stage], phase, abort_flag, ERR_BIT))))
            break;
          tc_fence_after();
          const uint32_t sp = smem_u32(smem + stage * PR_STAGE_BYTES);
          const uint64_t pd = smem_desc_sw128(sp, P_MN ? 8192 : 16, 1024);
          const uint64_t qd = smem_desc_sw128(sp + PR_OP_BYTES, Q_MN ? 8192 : 16, 1024);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_f16_ss_pair_elect(d_tmem, pd + (uint64_t)((P_MN ? 2048 : 32) * k >> 4),
                                  qd + (uint64_t)((Q_MN ? 2048 : 32) * k >> 4), idesc,
                                  (kb | k) != 0);
          mma_commit_pair_both_elect(&empty[stage]);
          if (++stage == PR_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair_both_elect(&tmem_full[buf]);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int q = warp & 3, half = (warp - 2) >> 2, w = warp - 2;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    uint8_t* box = boxes + w * PR_BOXES * PR_BOX;
    float* bias_s = bias_all + w * 32;
    uint64_t* rbar = r_full + 2 * w;
    const uint32_t tmem_empty_leader = mapa_shared(smem_u32(&tmem_empty[0]), 0);
    const Epilogue& e = a.e;
    int sbuf = 0;
    bool by_bulk = false;  // the last box was stored by TMA
    uint32_t r_issued = 0, r_used = 0;  // residual boxes asked for and read
    int it = 0;

    // Rows r0.. and columns c.. of this warp's chunk `i` (32 columns) of tile t.
    auto fetch_residual = [&](int r0, int c) {
      if (lane == 0) {
        uint64_t* bar = &rbar[r_issued & 1];
        mbar_arrive_expect_tx(bar, PR_BOX);
        tma_load_2d(box + (2 + (r_issued & 1)) * PR_BOX, &tmR, bar, c, r0);
      }
      ++r_issued;
    };
    auto put = [&](const uint32_t (&v)[32], const CUtensorMap* map, void* base, int64_t ld,
                   bool tma, int r0, int c) {
      uint8_t* b = box + sbuf * PR_BOX;
      // A TMA store ends a row at a 16-byte boundary (measured: columns of a row's
      // last run that are past the matrix are written too), so the last chunk of
      // rows that end elsewhere is stored by the warp.
      tma = tma && (e.cols % 8 == 0 || e.cols - c >= 32);
      // This box's previous store has read it: the last bulk store but one where
      // the box between went by TMA, else possibly the last.
      if (lane == 0) {
        if (by_bulk) bulk_wait_read<1>();
        else bulk_wait_read<0>();
      }
      by_bulk = tma;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[8 * j + i]);
        *reinterpret_cast<uint4*>(b + box_at(lane, j)) = pack8<T>(f);
      }
      if (tma) {
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(map, b, c, r0);
          bulk_commit();
        }
      } else {
        __syncwarp();
        T* out = static_cast<T*>(base) + (int64_t)r0 * ld + c + lane;
        if (c + lane < e.cols)
          for (int r = 0; r < 32 && r0 + r < e.rows; ++r)
            out[r * ld] = *reinterpret_cast<const T*>(b + box_at(r, lane >> 3) + (lane & 7) * 2);
        __syncwarp();
      }
      sbuf ^= 1;
    };

    for (int64_t t = pair; t < a.num_tiles && !*abort_flag; t += num_pairs, ++it) {
      const int buf = it & 1;
      const uint32_t acc_phase = (it >> 1) & 1;
      int tr, tc;
      pair_tile(a, t, tr, tc);
      const int r0 = tr * 256 + (int)rank * 128 + q * 32;
      const int c0 = tc * 256 + half * 128;
      // Chunks of this tile that hold any of D (a prefix of the four).
      const int chunks =
          r0 < e.rows && c0 < e.cols ? (int)min(4u, ((uint32_t)(e.cols - c0) + 31) / 32) : 0;
      const bool by_tma = e.R && a.r_tma;
      if (by_tma)
        for (int i = 0; i < min(2, chunks); ++i) fetch_residual(r0, c0 + 32 * i);
      if (!__all_sync(0xffffffffu,
                      mbar_wait_bounded(&tmem_full[buf], acc_phase, abort_flag, ERR_BIT)))
        break;
      tc_fence_after();
      const uint32_t tcol = tmem_base + buf * 256 + half * 128 + lane_base;
      bool ok = true;
      auto finish = [&](uint32_t (&v)[32], int i) {
        if (i >= chunks) return;
        const int c = c0 + 32 * i;
        if (e.bias) {
          bias_s[lane] = c + lane >= e.cols ? 0.f
                         : e.bias_f32 ? static_cast<const float*>(e.bias)[c + lane]
                                      : to_f32(static_cast<const T*>(e.bias)[c + lane]);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 b = reinterpret_cast<const float4*>(bias_s)[j];
            v[4 * j + 0] = __float_as_uint(__uint_as_float(v[4 * j + 0]) + b.x);
            v[4 * j + 1] = __float_as_uint(__uint_as_float(v[4 * j + 1]) + b.y);
            v[4 * j + 2] = __float_as_uint(__uint_as_float(v[4 * j + 2]) + b.z);
            v[4 * j + 3] = __float_as_uint(__uint_as_float(v[4 * j + 3]) + b.w);
          }
          __syncwarp();
        }
        if (e.Z) put(v, &tmZ, e.Z, e.ldz, a.z_tma, r0, c);
        switch (e.act) {
          case CTB_ACT_RELU: activate32<T, CTB_ACT_RELU>(v); break;
          case CTB_ACT_GELU: activate32<T, CTB_ACT_GELU>(v); break;
          case CTB_ACT_GELU_TANH: activate32<T, CTB_ACT_GELU_TANH>(v); break;
          case CTB_ACT_SILU: activate32<T, CTB_ACT_SILU>(v); break;
          default: break;
        }
        if (e.R) {
          uint8_t* b = box + (2 + (by_tma ? r_used & 1 : 0)) * PR_BOX;
          if (by_tma) {
            ok &= (bool)__all_sync(0xffffffffu,
                                   mbar_wait_bounded(&rbar[r_used & 1], (r_used >> 1) & 1,
                                                     abort_flag, ERR_BIT));
            ++r_used;
          } else {
            const T* in = static_cast<const T*>(e.R) + (int64_t)r0 * e.ldr + c + lane;
            if (c + lane < e.cols)
              for (int r = 0; r < 32 && r0 + r < e.rows; ++r)
                *reinterpret_cast<T*>(b + box_at(r, lane >> 3) + (lane & 7) * 2) = in[r * e.ldr];
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float f[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(b + box_at(lane, j)), f);
#pragma unroll
            for (int i2 = 0; i2 < 8; ++i2)
              v[8 * j + i2] = __float_as_uint(__uint_as_float(v[8 * j + i2]) + f[i2]);
          }
          __syncwarp();
          if (by_tma && i + 2 < chunks) fetch_residual(r0, c + 64);
        }
        put(v, &tmD, e.D, e.ldd, a.d_tma, r0, c);
      };
      uint32_t ra[32], rb[32];
      tmem_ld_32x32b_x32(tcol, ra);
#pragma unroll 1
      for (int i = 0; i < 4; i += 2) {
        tmem_ld_wait_regs(ra);
        tmem_ld_32x32b_x32(tcol + 32 * (i + 1), rb);
        finish(ra, i);
        tmem_ld_wait_regs(rb);
        if (i + 2 < 4) {
          tmem_ld_32x32b_x32(tcol + 32 * (i + 2), ra);
        } else {
          // The accumulator is in registers: the next tile but one may have it.
          tc_fence_before();
          if (leader) mbar_arrive(&tmem_empty[buf]);
          else mbar_arrive_cluster(tmem_empty_leader + buf * 8);
        }
        finish(rb, i + 1);
      }
      if (!ok) break;
    }
    if (lane == 0) {
      for (; r_used < r_issued; ++r_used) {  // only after a wait that gave up
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait_sleep(&rbar[r_used & 1], (r_used >> 1) & 1, 20000u) &&
               global_ns() - t0 < 1000000000ull) {
        }
      }
      bulk_wait<0>();  // staged boxes must outlive their stores
    }
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its peer may still touch its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---- host ------------------------------------------------------------------------------
static unsigned long long g_dense_ctx[64];  // context ID the set-up was done in
static int g_dense_pairs[64];               // CTA pairs that are resident at once
static std::mutex g_dense_mu;

template <typename T, bool P_MN, bool Q_MN>
int pair_attr() {
  CTB_CUDA_CHECK(cudaFuncSetAttribute(product_pair_kernel<T, P_MN, Q_MN>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, PR_SMEM));
  return CTB_OK;
}
template <typename T>
int pair_attrs() {
  int rc = pair_attr<T, false, true>();
  if (!rc) rc = pair_attr<T, false, false>();
  if (!rc) rc = pair_attr<T, true, true>();
  return rc;
}
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

// Kernel attributes of the current device, once per context; `pairs` receives the
// CTA pairs that are resident at once.
int device_setup(int* pairs_out) {
  int dev = 0;
  CTB_CUDA_CHECK(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(g_dense_mu);
  unsigned long long ctx = 0;
  if (int rc = current_context_id(&ctx)) return rc;
  *pairs_out = dev < 64 ? g_dense_pairs[dev] : 0;
  if (dev < 64 && g_dense_ctx[dev] == ctx) return CTB_OK;
  if (int rc = split_attrs<__half>()) return rc;
  if (int rc = split_attrs<__nv_bfloat16>()) return rc;
  if (int rc = pair_attrs<__half>()) return rc;
  if (int rc = pair_attrs<__nv_bfloat16>()) return rc;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(PR_THREADS);
  cfg.dynamicSmemBytes = PR_SMEM;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int pairs = 0;
  CTB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&pairs, product_pair_kernel<__half, false, true>, &cfg));
  if (dev < 64) {
    g_dense_pairs[dev] = pairs;
    g_dense_ctx[dev] = ctx;
  }
  *pairs_out = pairs;
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

// ---- which kernel, tile and split ------------------------------------------------------
// A model of the two kernels' times in microseconds. Its numbers make the choice
// by it the fastest one measured as nearly as possible over 1658 runs of forward
// products with nothing in their epilogue (150 of f16, 1 to 6000 rows, 256 to 14336
// columns, 300 to 14336 k, each with every tile and split): it takes 1.2% longer
// than the best, 20% at worst. They are a fit and no rates of the chip (9.66 TB/s,
// say, is above what HBM gives). On 48 other products in bf16 (1 to 4096 rows, 256
// to 4096 columns, 8 to 8192 k) its choice took longer than the best by, on average
// and at worst: forward 4% and 12%, with gelu and Z 7% and 29% (513 x 4096 x 2048 on
// the pair kernel, whose epilogue no longer hides there), dB 4% and 12%, dA 1% and
// 3%. Splits of 5 and 7 are left out: on these they beat the rest once, by 1.5%. A split
// CTA takes its k-blocks at 79 GB/s, alone or beside another on its SM; 256 CTAs
// in clusters are sure to be resident at once, 296 single ones; more row tiles
// read the weight again from L2. A pair takes 0.3 us a k-block and 3.1 us a tile.
struct Plan {
  int BN, S;  // BN = 0: the pair kernel
};

static double split_us(const Product& p, int BN, int S, int sms, double out_bytes) {
  const double tiles_r = (double)(((int64_t)p.rows + BN - 1) / BN);
  const double ctas = (double)(((int64_t)p.cols + SP_COLS - 1) / SP_COLS) * tiles_r * S;
  const int kb = (int)(((int64_t)p.depth + BK - 1) / BK), per = (kb + S - 1) / S;
  const double waves = std::ceil(ctas / (2 * sms));
  const double both = ctas > sms ? 2 : 1;
  const double load = waves * per * sp_stage_bytes(BN) / 79e3;
  const double moved = std::pow(tiles_r, 0.486) * 2.0 * p.cols * p.depth + 2.0 * p.rows * p.depth +
                       out_bytes;
  return 2.33 + std::max(load, moved / 9.66e6) + waves * both * BN * 0.032 + (S > 1 ? 0.22 : 0) +
         0.21 * S;
}
static double pair_us(const Product& p, int pairs) {
  const double tiles = (double)(((int64_t)p.rows + 255) / 256 * (((int64_t)p.cols + 255) / 256));
  const int kb = (int)(((int64_t)p.depth + BK - 1) / BK);
  return 3.7 + std::ceil(tiles / pairs) * (3.06 + 0.297 * kb);
}

// CTB_DENSE_PAIR=0 never takes the pair kernel, =1 whenever a pair can be resident.
static int pair_mode() {
  static const int mode = [] {
    const char* v = getenv("CTB_DENSE_PAIR");
    return v ? (v[0] == '1' ? 1 : 0) : -1;
  }();
  return mode;
}

// Tile rows (256: the pair kernel) and split that the self-tests ask for, rows << 8
// | split; 0: none asked for.
static std::atomic<int> g_asked{0};

static Plan choose_plan(const Product& p, int sms, int pairs) {
  const double out_bytes = (1 + (p.Z ? 1 : 0) + (p.R ? 1 : 0)) * 2.0 * p.rows * p.cols;
  Plan best = {0, 1};
  if (const int asked = g_asked.load(std::memory_order_relaxed)) {
    const int BN = asked >> 8, kb = (int)(((int64_t)p.depth + BK - 1) / BK);
    if (BN == 256 && pairs > 0) return best;
    // A tile of row-major-k rows is 64 wide at least; each CTA has two k-blocks at least.
    return {std::max(p.p_mn ? 64 : 16, std::min(BN, 128)),
            std::max(1, std::min(asked & 255, kb / 2))};
  }
  double us = pairs > 0 ? pair_us(p, pairs) : 1e30;
  const int mode = pair_mode();
  if (mode == 1 && pairs > 0) return best;
  if (mode == 0) us = 1e30;
  const int64_t tiles_c = ((int64_t)p.cols + SP_COLS - 1) / SP_COLS;
  const int kb = (int)(((int64_t)p.depth + BK - 1) / BK);
  for (int BN = p.p_mn ? 64 : 16; BN <= 128; BN *= 2) {
    const int64_t tiles_r = ((int64_t)p.rows + BN - 1) / BN;
    if (tiles_r > 65535 && !(BN == 128 && us >= 1e30)) continue;  // the grid's y
    for (int S = 1; S <= 8; ++S) {
      if (S > 1 && (S > kb / 2 || tiles_c * tiles_r * S > 256)) break;
      if (S == 5 || S == 7) continue;
      const double t = split_us(p, BN, S, sms, out_bytes);
      if (t < us) {
        us = t;
        best = {BN, S};
      }
    }
    if (BN >= p.rows) break;  // a wider tile has no more rows
  }
  return best;
}

template <typename T, bool Q_MN, bool P_MN, int BN>
int split_launch(const Product& p, const Epilogue& e, int S, cudaStream_t st) {
  CUtensorMap tmQ, tmP;
  if (int rc = operand_map<T>(&tmQ, p.Q, p.ldq, Q_MN, p.cols, p.depth, SP_COLS)) return rc;
  if (int rc = operand_map<T>(&tmP, p.P, p.ldp, P_MN, p.rows, p.depth, BN)) return rc;
  SplitArgs a;
  a.e = e;
  a.num_kb = (int)(((int64_t)p.depth + BK - 1) / BK);
  const int64_t tiles_c = ((int64_t)p.cols + SP_COLS - 1) / SP_COLS, tiles_r = ((int64_t)p.rows + BN - 1) / BN;
  if (tiles_r > 65535) return set_error(CTB_ERR_SHAPE, "dense: too many rows");
  return launch_overlapped("product_split_kernel", product_split_kernel<T, Q_MN, P_MN, BN>,
                           dim3((unsigned)(tiles_c * S), (unsigned)tiles_r), SP_THREADS,
                           sp_smem(BN), S, st, tmQ, tmP, a);
}

// A 16-bit matrix as boxes of 32 rows x 32 columns for the epilogue; a matrix
// that is not there, or that TMA cannot address, gets an empty map.
template <typename T>
int box_map(CUtensorMap* m, const void* base, int64_t ld, int rows, int cols, bool usable) {
  if (!usable) {
    std::memset(m, 0, sizeof(*m));
    return CTB_OK;
  }
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)(rows > 1 ? ld : ((int64_t)cols + 7) / 8 * 8) * 2};
  const uint32_t box[2] = {32, 32};
  return encode_tmap(m, Format<T>::map, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <typename T, bool P_MN, bool Q_MN>
int pair_launch(const Product& p, const Epilogue& e, int pairs, cudaStream_t st) {
  CUtensorMap tmP, tmQ, tmD, tmZ, tmR;
  PairArgs a;
  a.e = e;
  a.d_tma = rows16(p.D, p.ldd, p.rows);
  a.z_tma = p.Z && rows16(p.Z, p.ldz, p.rows);
  a.r_tma = p.R && rows16(p.R, p.ldr, p.rows);
  if (int rc = operand_map<T>(&tmP, p.P, p.ldp, P_MN, p.rows, p.depth, 128)) return rc;
  if (int rc = operand_map<T>(&tmQ, p.Q, p.ldq, Q_MN, p.cols, p.depth, 128)) return rc;
  if (int rc = box_map<T>(&tmD, p.D, p.ldd, p.rows, p.cols, a.d_tma)) return rc;
  if (int rc = box_map<T>(&tmZ, p.Z, p.ldz, p.rows, p.cols, a.z_tma)) return rc;
  if (int rc = box_map<T>(&tmR, p.R, p.ldr, p.rows, p.cols, a.r_tma)) return rc;
  a.num_kb = (int)(((int64_t)p.depth + BK - 1) / BK);
  a.tiles_r = (int)(((int64_t)p.rows + 255) / 256);
  a.tiles_c = (int)(((int64_t)p.cols + 255) / 256);
  a.num_tiles = (int64_t)a.tiles_r * a.tiles_c;
  return launch_overlapped("product_pair_kernel", product_pair_kernel<T, P_MN, Q_MN>,
                           dim3((unsigned)(2 * std::min<int64_t>(a.num_tiles, pairs))), PR_THREADS,
                           PR_SMEM, 2, st, tmP, tmQ, tmD, tmZ, tmR, a);
}

// The product on the tensor cores. Operands start on 16-byte boundaries, their
// leading dimensions are multiples of 8 (or they have one line only); depth > 0.
template <typename T>
int product_sm100(const Product& p0, int sms, cudaStream_t st) {
  int pairs = 0;
  if (int rc = device_setup(&pairs)) return rc;
  Product p = p0;
  // The distance between lines does not matter where there is one: any that TMA takes.
  if ((p.p_mn ? p.depth : p.rows) == 1) p.ldp = ((int64_t)(p.p_mn ? p.rows : p.depth) + 7) / 8 * 8;
  if ((p.q_mn ? p.depth : p.cols) == 1) p.ldq = ((int64_t)(p.q_mn ? p.cols : p.depth) + 7) / 8 * 8;
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
  const Plan plan = choose_plan(p, sms, pairs);
  if (plan.BN == 0) {
    if (p.p_mn) return pair_launch<T, true, true>(p, e, pairs, st);
    if (p.q_mn) return pair_launch<T, false, true>(p, e, pairs, st);
    return pair_launch<T, false, false>(p, e, pairs, st);
  }
  if (p.p_mn) {
    if (plan.BN == 64) return split_launch<T, true, true, 64>(p, e, plan.S, st);
    return split_launch<T, true, true, 128>(p, e, plan.S, st);
  }
  if (p.q_mn) {
    if (plan.BN == 16) return split_launch<T, true, false, 16>(p, e, plan.S, st);
    if (plan.BN == 32) return split_launch<T, true, false, 32>(p, e, plan.S, st);
    if (plan.BN == 64) return split_launch<T, true, false, 64>(p, e, plan.S, st);
    return split_launch<T, true, false, 128>(p, e, plan.S, st);
  }
  if (plan.BN == 16) return split_launch<T, false, false, 16>(p, e, plan.S, st);
  if (plan.BN == 32) return split_launch<T, false, false, 32>(p, e, plan.S, st);
  if (plan.BN == 64) return split_launch<T, false, false, 64>(p, e, plan.S, st);
  return split_launch<T, false, false, 128>(p, e, plan.S, st);
}
template int product_sm100<__half>(const Product&, int, cudaStream_t);
template int product_sm100<__nv_bfloat16>(const Product&, int, cudaStream_t);

}  // namespace dense

int dense_take_device_error(unsigned int* out) { return take_device_error(out); }
}  // namespace ctb

extern "C" int ctb_selftest_dense_plan(int32_t rows, int32_t split) {
  using namespace ctb;
  clear_error();
  if (rows != 0 && rows != 16 && rows != 32 && rows != 64 && rows != 128 && rows != 256)
    return set_error(CTB_ERR_ARG, "ctb_selftest_dense_plan: rows must be 0, 16, 32, 64, 128 or 256");
  if (rows != 0 && (split < 1 || split > 8))
    return set_error(CTB_ERR_ARG, "ctb_selftest_dense_plan: split must be 1 to 8");
  dense::g_asked = rows ? rows << 8 | split : 0;
  return CTB_OK;
}
