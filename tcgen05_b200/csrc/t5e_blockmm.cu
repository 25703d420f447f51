// t5e_blockmm.cu -- the matrix product of block-scaled E2M1 rows on the
// tensor cores: tcgen05.mma kind::mxf4 (UE8M0, blocks of 32) and
// kind::mxf4nvf4 (UE4M3 or UE8M0, blocks of 16), F32 accumulators in tensor
// memory.
#include <cuda.h>
#include <cuda_runtime.h>

#include "t5e.h"
#include "t5e_blocks.cuh"
#include "t5e_dispatch.h"

namespace t5e {
namespace blockmm {

using blocks::from_f32;
using blocks::pack2;
using blocks::to_f32;

constexpr int kStageK = 256;      // elements of K per pipeline stage: 128 bytes, one swizzle atom wide
constexpr int kInstrK = 64;       // elements of K per tcgen05.mma
constexpr int kRowBytes = 128;    // bytes of a row in a stage
// Bounded waits: a wait polls at most this often (each poll itself suspends
// for up to some microseconds), then the tile is given up.
constexpr uint32_t kWaitPolls = 1u << 22;

__device__ int g_expired;  // 1 once a wait ran out on this device

struct Params {
  CUtensorMap p_map, q_map;      // the operand with 128 rows a tile, the other one
  const uint8_t* p_scales;
  const uint8_t* q_scales;
  const float* multiplier_a;
  const float* multiplier_b;
  const void* c;
  void* d;
  int64_t c_p_stride, c_q_stride;  // elements
  int64_t d_stride;                // elements, along the axis that is not contiguous
  uint32_t p_rows, q_rows;
  uint32_t k, stages, groups;      // elements, pipeline stages, groups of four scales per row
  uint32_t idesc;
  float alpha;
  int32_t c_type, d_type;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- barriers --------------------------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count));
}

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2;\n\t"
               "selp.b32 %0, 1, 0, P1;\n\t}\n"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}

// Waits for the phase; gives up after kWaitPolls polls or once another thread
// of the block gave up (*failed).
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
  for (uint32_t poll = 0; poll < kWaitPolls; ++poll) {
    if (barrier_try(bar, parity)) return true;
    if (*failed) return false;
  }
  *failed = 1;
  return false;
}

// ---- copies -----------------------------------------------------------------

__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
               "[%4];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

__device__ __forceinline__ void load_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// ---- tensor memory and products -----------------------------------------------

// Shared-memory descriptor of K-major rows of 128 bytes with the 128-byte
// swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}

// Descriptor of a 512-byte tile of scales: 32 lines of 16 bytes, groups of 8
// lines 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

// 512 bytes of scales to four columns, the same in each 32-lane quarter.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(scale_desc(smem)) : "memory");
}

template <int BLOCK>
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t dp, uint64_t dq, uint32_t idesc, uint32_t tsp, uint32_t tsq,
                                    uint32_t accumulate) {
  if constexpr (BLOCK == 32) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n"
                 :: "r"(tmem_d), "l"(dp), "l"(dq), "r"(idesc), "r"(accumulate), "r"(tsp), "r"(tsq));
  } else {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n"
                 :: "r"(tmem_d), "l"(dp), "l"(dq), "r"(idesc), "r"(accumulate), "r"(tsp), "r"(tsq));
  }
}

__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 accumulator columns of this thread's lane.
__device__ __forceinline__ void load_acc16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
               "%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- results ---------------------------------------------------------------------

__device__ __forceinline__ float read_real(const void* p, int64_t i, int32_t type) {
  if (type == T5E_REAL_F32) return static_cast<const float*>(p)[i];
  if (type == T5E_REAL_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void write_real(void* p, int64_t i, int32_t type, float v) {
  if (type == T5E_REAL_F32) static_cast<float*>(p)[i] = v;
  else if (type == T5E_REAL_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f32<T5E_REAL_BF16>(v);
  else static_cast<__half*>(p)[i] = from_f32<T5E_REAL_F16>(v);
}

// N neighbouring results of row p of the tile grid, columns q .. q + count - 1:
// scales them, adds C and stores them.  SWAP: D is contiguous along p (lanes
// store neighbouring elements), otherwise along q (a lane stores vectors where
// the row is aligned).
template <bool SWAP, int N>
__device__ __forceinline__ void store_results(const Params& P, float alpha, uint32_t p, uint32_t q, int count,
                                              float (&v)[N]) {
  if (p >= P.p_rows) return;
  if (q + count > P.q_rows) count = q >= P.q_rows ? 0 : (int)(P.q_rows - q);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float add = 0.f;
    if (P.c != nullptr && i < count)
      add = read_real(P.c, (int64_t)p * P.c_p_stride + (int64_t)(q + i) * P.c_q_stride, P.c_type);
    v[i] = P.c != nullptr ? __fmaf_rn(v[i], alpha, add) : v[i] * alpha;
  }
  if constexpr (SWAP) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) write_real(P.d, (int64_t)(q + i) * P.d_stride + p, P.d_type, v[i]);
  } else {
    const int64_t at = (int64_t)p * P.d_stride + q;
    if (P.d_type == T5E_REAL_F32) {
      float* dst = static_cast<float*>(P.d) + at;
      if (N % 4 == 0 && count == N && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
          reinterpret_cast<float4*>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        return;
      }
    } else {
      uint16_t* dst = static_cast<uint16_t*>(P.d) + at;
      if (N % 8 == 0 && count == N && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          w[i] = P.d_type == T5E_REAL_BF16 ? pack2<T5E_REAL_BF16>(v[2 * i], v[2 * i + 1])
                                           : pack2<T5E_REAL_F16>(v[2 * i], v[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < N / 8; ++i)
          reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) write_real(P.d, at + i, P.d_type, v[i]);
  }
}

// ---- one tile per block ------------------------------------------------------------
//
// A block of 128 threads computes a tile of 128 rows of one operand (P) by BN
// rows of the other (Q).  One thread keeps `kStages` stages of 256 K in flight
// with TMA, one issues the products; then all four warps take the
// accumulators from tensor memory.  A cluster of `split` blocks shares one
// tile, each with its part of K; the partial sums meet in shared memory and
// each block finishes BN / split columns, adding the parts in rank order.
template <int BN, int BLOCK>
struct TileShape {
  static constexpr int kGroups = kStageK / (4 * BLOCK);  // 512-byte scale tiles per stage
  static constexpr int kScaleBytes = kGroups * 512;
  static constexpr int kPBytes = 128 * kRowBytes, kQBytes = BN * kRowBytes;
  static constexpr int kStageBytes = kPBytes + kQBytes + 2 * kScaleBytes;
  static constexpr int kStages = 110 * 1024 / kStageBytes;  // two blocks on an SM
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kScaleCol = BN < 32 ? 32 : BN;  // tensor memory column of the scales
  static constexpr int kTmemCols = BN > 64 ? 256 : 128;
  static_assert(kStages * kStageBytes >= 128 * BN * 4, "the partial sums reuse the stages");
  static_assert(kScaleCol + 2 * 2 * kGroups * 4 <= kTmemCols, "accumulators and two stages of scales");
};

template <int BN, int BLOCK, bool SWAP>
__global__ void __launch_bounds__(128) tile_kernel(const __grid_constant__ Params P, uint32_t split) {
  using S = TileShape<BN, BLOCK>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], finished;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  uint8_t* stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&tmem_slot)), "r"(S::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (t == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      barrier_init(smem_u32(&full[i]), 1);
      barrier_init(smem_u32(&empty[i]), 1);
    }
    barrier_init(smem_u32(&finished), 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(&P.p_map));
    asm volatile("prefetch.tensormap [%0];" :: "l"(&P.q_map));
  }
  fence_before();
  __syncthreads();
  fence_after();
  blocks::let_next_grid_start();
  blocks::wait_for_previous_grid();
  const uint32_t tmem = tmem_slot;
  const uint32_t rank = blockIdx.x % split;
  const uint32_t tile = blockIdx.x / split, p_tiles = (P.p_rows + 127u) >> 7;
  const uint32_t p0 = tile % p_tiles * 128u, q0 = tile / p_tiles * (uint32_t)BN;
  const uint32_t first = (uint32_t)((uint64_t)P.stages * rank / split);
  const uint32_t last = (uint32_t)((uint64_t)P.stages * (rank + 1) / split);
  if (warp == 0 && lane == 0) {
    const uint8_t* ps = P.p_scales + (uint64_t)(p0 >> 7) * P.groups * 512u;
    const uint8_t* qs = P.q_scales + (uint64_t)(q0 >> 7) * P.groups * 512u;
    uint32_t issued = 0;
    bool ok = true;
    for (uint32_t st = first; st < last; ++st, ++issued) {
      const uint32_t slot = issued % S::kStages, round = issued / S::kStages;
      ok = barrier_wait(smem_u32(&empty[slot]), (round & 1u) ^ 1u, &failed);
      if (!ok) break;
      const uint32_t base = smem_u32(stages) + slot * S::kStageBytes, bar = smem_u32(&full[slot]);
      const uint32_t g0 = st * S::kGroups;
      const uint32_t gn = P.groups - g0 < (uint32_t)S::kGroups ? P.groups - g0 : (uint32_t)S::kGroups;
      barrier_expect(bar, S::kPBytes + S::kQBytes + 2u * gn * 512u);
      load_tile(base, &P.p_map, (int32_t)(st * kRowBytes), (int32_t)p0, bar);
      load_tile(base + S::kPBytes, &P.q_map, (int32_t)(st * kRowBytes), (int32_t)q0, bar);
      load_bytes(base + S::kPBytes + S::kQBytes, ps + (uint64_t)g0 * 512u, gn * 512u, bar);
      load_bytes(base + S::kPBytes + S::kQBytes + S::kScaleBytes, qs + (uint64_t)g0 * 512u, gn * 512u, bar);
    }
    if (!ok) {  // given up: no copy may still be in flight when the block ends
      for (uint32_t i = issued > (uint32_t)S::kStages ? issued - S::kStages : 0u; i < issued; ++i)
        for (uint32_t poll = 0; poll < kWaitPolls && !barrier_try(smem_u32(&full[i % S::kStages]), (i / S::kStages) & 1u);
             ++poll) {
        }
    }
  } else if (warp == 1 && lane == 0) {
    bool ok = true;
    uint32_t used = 0;
    for (uint32_t st = first; st < last; ++st, ++used) {
      const uint32_t slot = used % S::kStages;
      ok = barrier_wait(smem_u32(&full[slot]), (used / S::kStages) & 1u, &failed);
      if (!ok) break;
      fence_after();
      const uint32_t base = smem_u32(stages) + slot * S::kStageBytes;
      const uint32_t left = P.k - st * kStageK;
      const uint32_t steps = left >= (uint32_t)kStageK ? kStageK / kInstrK : (left + kInstrK - 1) / kInstrK;
      const uint32_t tsp = tmem + S::kScaleCol + (used & 1u) * (2 * S::kGroups * 4), tsq = tsp + S::kGroups * 4;
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
        if (g * (BLOCK / 16) < (int)steps) {
          copy_scales(tsp + g * 4, base + S::kPBytes + S::kQBytes + g * 512);
          copy_scales(tsq + g * 4, base + S::kPBytes + S::kQBytes + S::kScaleBytes + g * 512);
        }
      }
      const uint64_t dp = operand_desc(base), dq = operand_desc(base + S::kPBytes);
#pragma unroll
      for (int j = 0; j < kStageK / kInstrK; ++j) {
        if (j < (int)steps) {
          // a column of scales holds four bytes per row: one product's with
          // blocks of 16, two products' with blocks of 32 (bytes 0-1, 2-3)
          const int col = BLOCK == 16 ? j * 4 : j / 2 * 4;
          const uint32_t id = BLOCK == 16 ? 0u : (uint32_t)(j & 1) * 2u;
          mma<BLOCK>(tmem, dp + j * 2, dq + j * 2, P.idesc | (id << 4) | (id << 29), tsp + col, tsq + col,
                     used != 0u || j != 0);
        }
      }
      commit(smem_u32(&empty[slot]));
    }
    commit(smem_u32(&finished));  // after a wait that ran out too: the products issued before it complete
  }
  __syncwarp();
  bool arrived = false;
  for (uint32_t poll = 0; poll < kWaitPolls && !arrived; ++poll) arrived = barrier_try(smem_u32(&finished), 0);
  fence_after();
  const bool bad = __syncthreads_or(!arrived || *static_cast<volatile int*>(&failed));
  if (bad && t == 0) atomicExch(&g_expired, 1);
  const float nan = __uint_as_float(0x7FC00000u);
  const float alpha = P.alpha * (P.multiplier_a != nullptr ? 1.f / *P.multiplier_a : 1.f) *
                      (P.multiplier_b != nullptr ? 1.f / *P.multiplier_b : 1.f);
  const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
  if (split == 1u) {
#pragma unroll 1
    for (int q = 0; q < BN; q += 16) {
      if (q0 + q >= P.q_rows) break;
      float v[16];
      load_acc16(lanes + q, v);
      if (bad) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = nan;
      }
      store_results<SWAP, 16>(P, alpha, p0 + t, q0 + q, 16, v);
    }
  } else {
    float* part = reinterpret_cast<float*>(stages);
#pragma unroll 1
    for (int q = 0; q < BN; q += 16) {
      float v[16];
      load_acc16(lanes + q, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(q + i) * 128 + t] = bad ? nan : v[i];
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int width = BN / (int)split, w0 = width * (int)rank;
#pragma unroll 1
    for (int q = w0; q < w0 + width; q += 8) {
      if (q0 + q >= P.q_rows) break;
      const int count = width < 8 ? width : 8;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      for (uint32_t r = 0; r < split; ++r) {
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(part + q * 128 + t)), "r"(r));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < count) {
            float x;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(there + i * 512) : "memory");
            v[i] += x;
          }
        }
      }
      store_results<SWAP, 8>(P, alpha, p0 + t, q0 + q, count, v);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  if (warp == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(S::kTmemCols));
  }
}

// ---- host side ----------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor map encoder, looked up once.
EncodeTiled encoder() {
  static std::atomic<EncodeTiled> found{nullptr};
  EncodeTiled f = found.load(std::memory_order_acquire);
  if (f) return f;
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q);
  if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) {
    set_cuda_error("cuTensorMapEncodeTiled lookup", e != cudaSuccess ? e : cudaErrorNotSupported);
    return nullptr;
  }
  f = reinterpret_cast<EncodeTiled>(p);
  found.store(f, std::memory_order_release);
  return f;
}

// Map of a matrix of codes as bytes, boxes of 128 bytes by `box_rows` rows;
// what lies outside reads as zero codes.
int encode(CUtensorMap* map, const t5e_blocks& b, uint32_t box_rows) {
  const EncodeTiled f = encoder();
  if (!f) return T5E_ERR_CUDA;
  const cuuint64_t dims[2] = {(cuuint64_t)((b.k + 1) / 2), (cuuint64_t)b.rows};
  const cuuint64_t strides[1] = {(cuuint64_t)b.stride};
  const cuuint32_t box[2] = {(cuuint32_t)kRowBytes, box_rows}, unit[2] = {1, 1};
  const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, b.data, dims, strides, box, unit,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_cuda_error("cuTensorMapEncodeTiled", cudaErrorInvalidValue);
    return T5E_ERR_CUDA;
  }
  return T5E_OK;
}

// Instruction descriptor: E2M1 x E2M1, M = 128, `n` columns.
uint32_t instruction(const t5e_blocks& b, uint32_t n, uint32_t m = 128) {
  return (1u << 7) | (1u << 10) | ((n / 8u) << 17) | ((b.scale_format == T5E_SCALE_UE8M0 ? 1u : 0u) << 23) |
         ((m / 128u) << 27);
}

template <int BN, int BLOCK, bool SWAP>
int launch_tile(Params& P, const t5e_blocks& p, const t5e_blocks& q, uint32_t split, cudaStream_t stream) {
  using S = TileShape<BN, BLOCK>;
  int rc = encode(&P.p_map, p, 128);
  if (rc == T5E_OK) rc = encode(&P.q_map, q, BN);
  if (rc == T5E_OK) rc = raise_smem_limit<tile_kernel<BN, BLOCK, SWAP>>(S::kSmem, "block product attribute");
  if (rc != T5E_OK) return rc;
  P.idesc = instruction(p, BN);
  cudaLaunchConfig_t cfg = {};
  const uint64_t grid = ((p.rows + 127) / 128) * ((q.rows + BN - 1) / BN) * split;
  if (grid > 0x7FFFFFFFull) return T5E_ERR_INVALID;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {split, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tile_kernel<BN, BLOCK, SWAP>, P, split);
  if (e != cudaSuccess) {
    set_cuda_error("block product launch", e);
    return T5E_ERR_CUDA;
  }
  return kernel_status("block product launch");
}

template <int BLOCK>
int launch_form(Params& P, const t5e_blocks& p, const t5e_blocks& q, bool swap, uint32_t split, cudaStream_t stream) {
  if (q.rows <= 16)
    return swap ? launch_tile<16, BLOCK, true>(P, p, q, split, stream) : launch_tile<16, BLOCK, false>(P, p, q, split, stream);
  if (q.rows <= 32)
    return swap ? launch_tile<32, BLOCK, true>(P, p, q, split, stream) : launch_tile<32, BLOCK, false>(P, p, q, split, stream);
  if (q.rows <= 64)
    return swap ? launch_tile<64, BLOCK, true>(P, p, q, split, stream) : launch_tile<64, BLOCK, false>(P, p, q, split, stream);
  return swap ? launch_tile<128, BLOCK, true>(P, p, q, split, stream) : launch_tile<128, BLOCK, false>(P, p, q, split, stream);
}

uint64_t tiles_of(uint64_t p_rows, uint64_t q_rows) { return ((p_rows + 127) / 128) * ((q_rows + 127) / 128); }

}  // namespace blockmm
}  // namespace t5e

extern "C" {

int t5e_block_scaled_mm(const t5e_block_mm* mm, void* stream) {
  using namespace t5e;
  using namespace t5e::blockmm;
  if (!mm || !blocks_ok(mm->a) || !blocks_ok(mm->b)) return T5E_ERR_INVALID;
  const t5e_blocks &a = *mm->a, &b = *mm->b;
  auto real = [](int32_t t) { return t == T5E_REAL_F32 || t == T5E_REAL_BF16 || t == T5E_REAL_F16; };
  if (a.k != b.k || a.scale_format != b.scale_format || a.scale_block != b.scale_block || !real(mm->d_type) ||
      (mm->c && !real(mm->c_type)))
    return T5E_ERR_INVALID;
  if (mm->split != 0 && mm->split != 1 && mm->split != 2 && mm->split != 4 && mm->split != 8) return T5E_ERR_INVALID;
  if (a.rows == 0 || b.rows == 0) return T5E_OK;
  const int bytes = mm->d_type == T5E_REAL_F32 ? 4 : 2;
  if (!mm->d || (reinterpret_cast<uintptr_t>(mm->d) & (bytes - 1)) ||
      (a.rows > 1 && mm->d_stride < (int64_t)b.rows))
    return T5E_ERR_INVALID;
  if (mm->c && (reinterpret_cast<uintptr_t>(mm->c) & (mm->c_type == T5E_REAL_F32 ? 3 : 1))) return T5E_ERR_INVALID;
  // the operand with fewer rows takes the narrow side of the tile
  const bool swap = a.rows < b.rows && a.rows <= 128;
  const t5e_blocks &p = swap ? b : a, &q = swap ? a : b;
  Params P = {};
  P.p_scales = static_cast<const uint8_t*>(p.scales);
  P.q_scales = static_cast<const uint8_t*>(q.scales);
  P.multiplier_a = mm->multiplier_a;
  P.multiplier_b = mm->multiplier_b;
  P.c = mm->c;
  P.d = mm->d;
  P.c_p_stride = swap ? mm->c_col_stride : mm->c_row_stride;
  P.c_q_stride = swap ? mm->c_row_stride : mm->c_col_stride;
  P.d_stride = mm->d_stride;
  P.p_rows = (uint32_t)p.rows;
  P.q_rows = (uint32_t)q.rows;
  P.k = (uint32_t)a.k;
  P.stages = (uint32_t)((a.k + kStageK - 1) / kStageK);
  P.groups = scale_groups(a);
  P.alpha = mm->alpha;
  P.c_type = mm->c_type;
  P.d_type = mm->d_type;
  uint32_t split = (uint32_t)mm->split;
  if (split == 0) {
    split = 1;
    const uint64_t tiles = tiles_of(p.rows, q.rows);
    while (split < 8 && tiles * split * 2 <= (uint64_t)sm_count() && P.stages >= split * 4) split *= 2;
  }
  if (split > P.stages) return T5E_ERR_INVALID;  // every part has work
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a.scale_block == 32 ? launch_form<32>(P, p, q, swap, split, s) : launch_form<16>(P, p, q, swap, split, s);
}

int t5e_block_scaled_mm_expired(int32_t* expired) {
  using namespace t5e;
  if (!expired) return T5E_ERR_INVALID;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(expired, blockmm::g_expired, sizeof(int));
  if (e != cudaSuccess) {
    set_cuda_error("t5e_block_scaled_mm_expired", e);
    return T5E_ERR_CUDA;
  }
  return T5E_OK;
}

}  // extern "C"
