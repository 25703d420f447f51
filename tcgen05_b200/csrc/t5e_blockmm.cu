// t5e_blockmm.cu -- the matrix product of block-scaled E2M1 rows on the
// tensor cores: tcgen05.mma kind::mxf4 (UE8M0, blocks of 32) and
// kind::mxf4nvf4 (UE4M3 or UE8M0, blocks of 16), F32 accumulators in tensor
// memory.
#include <cuda.h>
#include <cuda_runtime.h>

#include "t5e.h"
#include "t5e_blocks.cuh"
#include "t5e_blocktiles.h"
#include "t5e_dispatch.h"

namespace t5e {
namespace blockmm {

using blocks::from_f32;
using blocks::pack2;
using blocks::to_f32;

constexpr int kStageK = 256;      // elements of K per pipeline stage: 128 bytes, one swizzle atom wide
constexpr int kInstrK = 64;       // elements of K per tcgen05.mma
constexpr int kRowBytes = 128;    // bytes of a row in a stage
// Bounded waits: after this long (4 s) the tile is given up.
constexpr uint64_t kWaitNs = 4000000000ull;

__device__ int g_expired;  // 1 once a wait ran out on this device

struct Params {
  const float* multiplier_a;
  const float* multiplier_b;
  const void* c;
  void* d;
  int64_t c_p_stride, c_q_stride;  // elements
  int64_t d_stride;                // elements, along the axis that is not contiguous
  uint32_t p_rows, q_rows;         // P: the operand with 128 rows a tile, Q: the other one
  uint32_t k, stages;              // elements, pipeline stages
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

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Waits for the phase; gives up after kWaitNs, or once another thread of the
// block gave up (*failed; NULL: do not look).
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
  if (barrier_try(bar, parity)) return true;
  const uint64_t start = now_ns();
  do {
    if (barrier_try(bar, parity)) return true;
    if (failed != nullptr && *failed) return false;
  } while (now_ns() - start < kWaitNs);
  if (failed != nullptr) *failed = 1;
  return false;
}

// One thread of a converged warp.  elect.sync (rather than lane == 0) and a
// broadcast warp index let the compiler see that what follows is uniform,
// which the operands of tcgen05 and TMA instructions have to be.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, P;\n\t}\n" : "=r"(p));
  return p != 0u;
}
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The address of a variable of this block in block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void arrive_in(uint32_t bar_in_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(bar_in_cluster) : "memory");
}

// ---- copies -----------------------------------------------------------------
//
// In a pair the barrier may be the other block's (cta_group::2).

template <bool PAIR>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
                 "[%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
                 "[%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Into L2 only.
__device__ __forceinline__ void fetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" :: "l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void fetch_3d(const CUtensorMap* map, int32_t x, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];"
               :: "l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                                        uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
                 "[%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
                 "[%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
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

// 512 bytes of scales to four columns, the same in each 32-lane quarter (in a
// pair each block's bytes to its own tensor memory).
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(scale_desc(smem)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(scale_desc(smem)) : "memory");
}

#define T5E_BLOCK_MMA(group, form)                                                                       \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                         \
               "tcgen05.mma.cta_group::" group ".kind::" form " [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" \
               :: "r"(tmem_d), "l"(dp), "l"(dq), "r"(idesc), "r"(accumulate), "r"(tsp), "r"(tsq))

template <bool PAIR, int BLOCK>
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t dp, uint64_t dq, uint32_t idesc, uint32_t tsp, uint32_t tsq,
                                    uint32_t accumulate) {
  if constexpr (PAIR && BLOCK == 32) T5E_BLOCK_MMA("2", "mxf4.block_scale.block32");
  else if constexpr (PAIR) T5E_BLOCK_MMA("2", "mxf4nvf4.block_scale.block16");
  else if constexpr (BLOCK == 32) T5E_BLOCK_MMA("1", "mxf4.block_scale.block32");
  else T5E_BLOCK_MMA("1", "mxf4nvf4.block_scale.block16");
}

#undef T5E_BLOCK_MMA

// Arrives on this block's barrier when what this thread issued so far is
// complete; commit_all arrives on it in both blocks of a pair.
template <bool PAIR>
__device__ __forceinline__ void commit_here(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void commit_all(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(bar), "h"((uint16_t)3) : "memory");
  else
    commit_here<false>(bar);
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

__device__ __forceinline__ void load_acc32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
               "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr) : "memory");
}
__device__ __forceinline__ void acc_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

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

// The value of an element of C from its bits.
template <int BYTES>
__device__ __forceinline__ float c_value(const Params& P, uint32_t bits) {
  if constexpr (BYTES == 4) return __uint_as_float(bits);
  return P.c_type == T5E_REAL_BF16 ? __uint_as_float(bits << 16)
                                   : __half2float(__ushort_as_half((unsigned short)bits));
}

// N neighbouring finished results of row p, columns q .. q + N - 1: vectors where
// the row is aligned.
template <int N>
__device__ __forceinline__ void store_plain(const Params& P, uint32_t p, uint32_t q, float (&v)[N], int count = N) {
  if (p >= P.p_rows) return;
  if (q + count > P.q_rows) count = q >= P.q_rows ? 0 : (int)(P.q_rows - q);
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

// What sums are multiplied by, alpha * (1 / ma) * (1 / mb): one F32 number,
// except where that product, or its first step, leaves the normal F32 range
// although the results need not (both tensors near 2^76: the product is infinite
// and turned rows of zeros into NaN; near 2^-65: it is zero, and so were results
// of 2^-118).  There the factor keeps its digits in `alpha`, at the end of the F32
// range, and sums are first multiplied by the powers of two `by` and `by2`, which
// is exact wherever the result is not beyond F32 anyway.
struct Factor {
  float alpha, by, by2;  // by = 1: alpha alone
};

__host__ __device__ __forceinline__ bool is_normal(float v) {
  const float size = v < 0.f ? -v : v;
  return size >= 0x1p-126f && size <= 0x1.fffffep127f;
}

__device__ __forceinline__ Factor factor_of(float alpha, float ma, float mb) {
  const float ra = 1.f / ma, rb = 1.f / mb, first = alpha * ra, joint = first * rb;
  Factor f = {joint, 1.f, 1.f};
  if (is_normal(first) && is_normal(joint)) return f;
  const double whole = (double)alpha * ra * rb;  // three F32 numbers: within F64's range
  const int e = (int)((__double_as_longlong(whole) >> 52) & 0x7FF) - 1023;
  if (whole == 0. || e == 1024) {
    f.alpha = (float)whole;
    return f;
  }
  const int s = e < -126 ? e + 126 : e > 126 ? e - 126 : 0, part = s < -126 ? -126 : s > 127 ? 127 : s;
  const int rest = s - part < -126 ? -126 : s - part > 127 ? 127 : s - part;  // beyond: zero or infinite without it
  f.alpha = (float)(whole * __longlong_as_double((long long)(1023 - s) << 52));
  f.by = __uint_as_float((uint32_t)(part + 127) << 23);
  f.by2 = __uint_as_float((uint32_t)(rest + 127) << 23);
  return f;
}

__device__ __forceinline__ float multiplier_at(const float* p) { return p != nullptr ? *p : 1.f; }

template <int N>
__device__ __forceinline__ void rescale(const Factor& f, float* v) {
  if (f.by == 1.f) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = v[i] * f.by * f.by2;
}

// N neighbouring results of row p of the tile grid, columns q .. q + count - 1:
// scales them, adds C and stores them.  SWAP: D is contiguous along p (lanes
// store neighbouring elements), otherwise along q (a lane stores vectors).
template <bool SWAP, int N>
__device__ __forceinline__ void store_results(const Params& P, const Factor& f, uint32_t p, uint32_t q, int count,
                                              float (&v)[N]) {
  if (p >= P.p_rows) return;
  rescale<N>(f, v);
  if (q + count > P.q_rows) count = q >= P.q_rows ? 0 : (int)(P.q_rows - q);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float add = 0.f;
    if (P.c != nullptr && i < count)
      add = read_real(P.c, (int64_t)p * P.c_p_stride + (int64_t)(q + i) * P.c_q_stride, P.c_type);
    v[i] = P.c != nullptr ? __fmaf_rn(v[i], f.alpha, add) : v[i] * f.alpha;
  }
  if constexpr (SWAP) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) write_real(P.d, (int64_t)(q + i) * P.d_stride + p, P.d_type, v[i]);
  } else {
    store_plain<N>(P, p, q, v, count);
  }
}

// A warp's 32 x 32 results by way of shared memory (a 32 x 33 buffer of its
// own): lane r brings row p + r, columns q .. q + 31; the stores, and the loads
// of C, then run along the rows, 32 neighbouring elements at a time, whatever
// the alignment.  ADD: bytes of an element of C, 0 for none.
template <int TYPE, int ADD>
__device__ __forceinline__ void turned_rows(const Params& P, float alpha, uint32_t p, uint32_t col, int rows,
                                            const float* column) {
  using T = typename blocks::Real<TYPE>::type;
  T* dst = static_cast<T*>(P.d) + (int64_t)p * P.d_stride + col;
  // C of all rows is on its way before the first is used
  uint32_t add[ADD ? 32 : 1];
  if constexpr (ADD > 0) {
    const char* from = static_cast<const char*>(P.c) + ((int64_t)p * P.c_p_stride + (int64_t)col * P.c_q_stride) * ADD;
#pragma unroll
    for (int r = 0; r < 32; ++r, from += P.c_p_stride * ADD)
      add[r] = r >= rows ? 0u : ADD == 4 ? *reinterpret_cast<const uint32_t*>(from)
                                         : (uint32_t)*reinterpret_cast<const uint16_t*>(from);
  }
#pragma unroll
  for (int r = 0; r < 32; r += 8) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = column[(r + j) * 33];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (ADD > 0) x[j] = __fmaf_rn(x[j], alpha, c_value<ADD>(P, add[r + j]));
      else x[j] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j, dst += P.d_stride)
      if (r + j < rows) *dst = from_f32<TYPE>(x[j]);
  }
}

template <int TYPE>
__device__ __forceinline__ void turned_type(const Params& P, float alpha, uint32_t p, uint32_t col, int rows,
                                            const float* column) {
  if (P.c == nullptr) turned_rows<TYPE, 0>(P, alpha, p, col, rows, column);
  else if (P.c_type == T5E_REAL_F32) turned_rows<TYPE, 4>(P, alpha, p, col, rows, column);
  else turned_rows<TYPE, 2>(P, alpha, p, col, rows, column);
}

__device__ __forceinline__ void store_turned(const Params& P, float alpha, uint32_t p, uint32_t q, const float* v,
                                             float* buffer) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) buffer[lane * 33 + j] = v[j];
  __syncwarp();
  const uint32_t col = q + lane;
  if (col >= P.q_rows || p >= P.p_rows) return;
  const int rows = P.p_rows - p < 32u ? (int)(P.p_rows - p) : 32;
  if (P.d_type == T5E_REAL_F32) turned_type<T5E_REAL_F32>(P, alpha, p, col, rows, buffer + lane);
  else if (P.d_type == T5E_REAL_BF16) turned_type<T5E_REAL_BF16>(P, alpha, p, col, rows, buffer + lane);
  else turned_type<T5E_REAL_F16>(P, alpha, p, col, rows, buffer + lane);
}

// v = v * alpha + C for 64 columns of row p, C's rows being contiguous and on
// 16-byte boundaries (or one row for all).
template <int BYTES>
__device__ __forceinline__ void add_row(const Params& P, float alpha, uint32_t p, uint32_t q, float* v) {
  constexpr int kPer = 16 / BYTES;
  const char* row = static_cast<const char*>(P.c) + ((int64_t)p * P.c_p_stride + q) * BYTES;
  const bool there = p < P.p_rows;
  uint4 w[64 / kPer];
#pragma unroll
  for (int j = 0; j < 64 / kPer; ++j) {
    w[j] = make_uint4(0u, 0u, 0u, 0u);
    if (there && q + (j + 1) * kPer <= P.q_rows) {
      w[j] = *(reinterpret_cast<const uint4*>(row) + j);
    } else if (there && q + j * kPer < P.q_rows) {
      uint32_t words[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (q + j * kPer + i < P.q_rows) {
          if constexpr (BYTES == 4) words[i] = reinterpret_cast<const uint32_t*>(row)[j * kPer + i];
          else words[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[j * kPer + i] << (16 * (i & 1));
        }
      }
      w[j] = make_uint4(words[0], words[1], words[2], words[3]);
    }
  }
#pragma unroll
  for (int j = 0; j < 64 / kPer; ++j) {
    const uint32_t words[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t raw = BYTES == 4 ? words[i] : (words[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
      v[j * kPer + i] = __fmaf_rn(v[j * kPer + i], alpha, c_value<BYTES>(P, raw));
    }
  }
}

// A warp's 32 rows by 64 finished results through a box of 32 rows of 128 bytes
// that TMA writes (two boxes, one after the other, for F32): whole lines, and
// swizzled as the map says, so that the lanes' 16-byte stores meet no bank twice.
__device__ __forceinline__ void store_box(const Params& P, const CUtensorMap* map, uint32_t p, uint32_t q, const float* v,
                                          uint8_t* box) {
  const int lane = threadIdx.x & 31;
  const bool wide = P.d_type == T5E_REAL_F32;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half == 1 && !wide) break;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // what was in the box has been read
    __syncwarp();
    uint8_t* row = box + lane * 128;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint4 w;
      if (wide) {
        const float* x = v + half * 32 + 4 * j;
        w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      } else {
        const float* x = v + 8 * j;
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          h[i] = P.d_type == T5E_REAL_BF16 ? pack2<T5E_REAL_BF16>(x[2 * i], x[2 * i + 1])
                                           : pack2<T5E_REAL_F16>(x[2 * i], x[2 * i + 1]);
        w = make_uint4(h[0], h[1], h[2], h[3]);
      }
      *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) * 16)) = w;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      const uint32_t col = q + half * 32;
      if (col < P.q_rows && p < P.p_rows)
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                     :: "l"(map), "r"((int32_t)col), "r"((int32_t)p), "r"(smem_u32(box)) : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
}

// ---- the pipeline both kernels share ----------------------------------------------
//
// Four roles, one thread each, and two rings of shared-memory stages of 256 K:
//
//   operands   TMA loads the codes of P and Q into the operand ring
//   scales     TMA loads the scale tiles into the scale ring
//   spread     tcgen05.cp copies a unit's scales (128 K) from the scale ring
//              to one of four unit buffers in tensor memory
//   products   waits for a stage's codes and a unit's scales and issues the
//              unit's two tcgen05.mma
//
// The scales have a ring and a thread of their own because a tcgen05.cp of 512
// bytes takes about 32 cycles, and issued by the products' thread it runs
// between them: a 256 x 256 pair stage (512 cycles of products) spent 384 more
// on its 12 copies.  From another thread the copies run beside the products, and
// ahead of the codes, so that a stage of codes is held no longer than its load
// and its products take.
//
// 8192^3 in blocks of 16 takes 202 to 206 us (5.3 to 5.4 PFLOP/s).  Repeating
// each product 8 times puts the products alone at 140 at the clock that the
// power limit leaves.  Of an earlier state that took 219: without the products
// 179, without the scales' loads and copies 174, without both 130.  Results:
// 8192 x 4096 x 4096, then 58.7 us, took 52.9 without storing them.
//
// In a pair (PAIR) both blocks load their own parts, and the first block
// spreads and issues for both; its barriers count the bytes of both, and its
// commits arrive in both.
// STAGES and SCALE_STAGES are the most that the barriers provide for; a launch
// says how many it has room for (Depth).
template <bool PAIR_, int BN_, int BLOCK_, int STAGES_, int SCALE_STAGES_, int TMEM_>
struct Pipe {
  static constexpr bool PAIR = PAIR_;
  static constexpr int BN = BN_, BLOCK = BLOCK_, STAGES = STAGES_, SCALE_STAGES = SCALE_STAGES_;
  static constexpr int kTmem = TMEM_;                            // columns allocated
  static constexpr int kGroups = kStageK / (4 * BLOCK);          // 512-byte scale tiles of a stage per 128 rows
  static constexpr int kUnitGroups = kGroups / 2;
  static constexpr int kQTiles = (BN + 127) / 128;               // scale tiles of Q's rows
  static constexpr int kQRows = PAIR ? BN / 2 : BN;              // rows of Q a block loads
  static constexpr int kPBytes = 128 * kRowBytes, kQBytes = kQRows * kRowBytes;
  static constexpr int kStageBytes = kPBytes + kQBytes;
  static constexpr int kScaleBytes = kGroups * 512 * (1 + kQTiles);
  static constexpr int kUnitCols = kUnitGroups * 4 * (1 + kQTiles);
  static constexpr int kUnits = 4;
  static constexpr int kScaleCol = kTmem - kUnits * kUnitCols;   // first column of the unit buffers
  static constexpr int kBlocks = PAIR ? 2 : 1;
};

template <typename S>
struct Barriers {
  uint64_t full[S::STAGES], empty[S::STAGES];
  uint64_t scale_full[S::SCALE_STAGES], scale_empty[S::SCALE_STAGES];
  uint64_t unit_full[S::kUnits], unit_empty[S::kUnits];
};

struct Maps {
  CUtensorMap p, q, ps, qs;
};

template <typename S>
__device__ __forceinline__ void init_barriers(Barriers<S>& b) {
  for (int i = 0; i < S::STAGES; ++i) {
    barrier_init(smem_u32(&b.full[i]), 1);
    barrier_init(smem_u32(&b.empty[i]), 1);
  }
  for (int i = 0; i < S::SCALE_STAGES; ++i) {
    barrier_init(smem_u32(&b.scale_full[i]), 1);
    barrier_init(smem_u32(&b.scale_empty[i]), 1);
  }
  for (int i = 0; i < S::kUnits; ++i) {
    barrier_init(smem_u32(&b.unit_full[i]), 1);
    barrier_init(smem_u32(&b.unit_empty[i]), 1);
  }
}

__device__ __forceinline__ void prefetch_maps(const Maps& m) {
  asm volatile("prefetch.tensormap [%0];" :: "l"(&m.p));
  asm volatile("prefetch.tensormap [%0];" :: "l"(&m.q));
  asm volatile("prefetch.tensormap [%0];" :: "l"(&m.ps));
  asm volatile("prefetch.tensormap [%0];" :: "l"(&m.qs));
}

struct Depth {
  uint32_t stages, scale_stages;
};

// A role's place in a ring: the slot, the parity of the round, uses so far.
struct Use {
  uint32_t slot = 0, parity = 0, count = 0;
  __device__ __forceinline__ void next(uint32_t size) {
    ++count;
    if (++slot == size) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// Waits until the slot has been released by its use before (at once the first
// time round); until it has been filled.
__device__ __forceinline__ bool wait_slot(uint64_t* empty, const Use& u, int* failed) {
  return barrier_wait(smem_u32(empty + u.slot), u.parity ^ 1u, failed);
}
__device__ __forceinline__ bool wait_use(uint64_t* full, const Use& u, int* failed) {
  return barrier_wait(smem_u32(full + u.slot), u.parity, failed);
}

// Announces `bytes` per block and returns the barrier that the copies arrive
// on: the first block's in a pair.
template <typename S>
__device__ __forceinline__ uint32_t announce(uint64_t* full, uint32_t rank, uint32_t bytes) {
  const uint32_t bar = smem_u32(full);
  if (!S::PAIR || rank == 0) barrier_expect(bar, S::kBlocks * bytes);
  return S::PAIR ? in_block(bar, 0) : bar;
}

// Stages first .. last - 1 of a tile.
template <typename S>
__device__ __forceinline__ bool load_operands(const Maps& m, Barriers<S>& b, uint8_t* ring, const Depth& depth, uint32_t rank,
                                              uint32_t first, uint32_t last, int32_t p0, int32_t q0, Use& u, int* failed) {
  for (uint32_t st = first; st < last; ++st, u.next(depth.stages)) {
    if (!wait_slot(b.empty, u, failed)) return false;
    const uint32_t at = smem_u32(ring) + u.slot * S::kStageBytes;
    const uint32_t bar = announce<S>(&b.full[u.slot], rank, S::kStageBytes);
    load_2d<S::PAIR>(at, &m.p, (int32_t)(st * kRowBytes), p0, bar);
    load_2d<S::PAIR>(at + S::kPBytes, &m.q, (int32_t)(st * kRowBytes), q0, bar);
  }
  return true;
}

template <typename S>
__device__ __forceinline__ bool load_scales(const Maps& m, Barriers<S>& b, uint8_t* ring, const Depth& depth, uint32_t rank,
                                            uint32_t first, uint32_t last, int32_t p_tile, int32_t q_tile, Use& u,
                                            int* failed) {
  for (uint32_t st = first; st < last; ++st, u.next(depth.scale_stages)) {
    if (!wait_slot(b.scale_empty, u, failed)) return false;
    const uint32_t at = smem_u32(ring) + u.slot * S::kScaleBytes;
    const uint32_t bar = announce<S>(&b.scale_full[u.slot], rank, S::kScaleBytes);
    load_3d<S::PAIR>(at, &m.ps, 0, (int32_t)(st * S::kGroups), p_tile, bar);
    load_3d<S::PAIR>(at + S::kGroups * 512, &m.qs, 0, (int32_t)(st * S::kGroups), q_tile, bar);
  }
  return true;
}

// Products of K = 64 in a stage.
__device__ __forceinline__ uint32_t steps_in(uint32_t k, uint32_t st) {
  const uint32_t left = (k - st * kStageK + kInstrK - 1) / kInstrK;
  return left < (uint32_t)(kStageK / kInstrK) ? left : kStageK / kInstrK;
}

template <typename S>
__device__ __forceinline__ bool spread_scales(Barriers<S>& b, uint8_t* ring, const Depth& depth, uint32_t tmem, uint32_t k,
                                              uint32_t first, uint32_t last, Use& u, Use& unit, int* failed) {
  for (uint32_t st = first; st < last; ++st, u.next(depth.scale_stages)) {
    if (!wait_use(b.scale_full, u, failed)) return false;
    const uint32_t at = smem_u32(ring) + u.slot * S::kScaleBytes;
    const uint32_t steps = steps_in(k, st);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 2 >= (int)steps) break;
      if (!wait_slot(b.unit_empty, unit, failed)) return false;
      fence_after();
      const uint32_t to = tmem + S::kScaleCol + unit.slot * S::kUnitCols;
#pragma unroll
      for (int g = 0; g < S::kUnitGroups; ++g) {
        const int from = half * S::kUnitGroups + g;
        copy_scales<S::PAIR>(to + g * 4, at + from * 512);
        // Q's scales of one group side by side: 4 columns per 128 rows
#pragma unroll
        for (int h = 0; h < S::kQTiles; ++h)
          copy_scales<S::PAIR>(to + (S::kUnitGroups + g * S::kQTiles + h) * 4, at + (S::kGroups * (1 + h) + from) * 512);
      }
      commit_here<S::PAIR>(smem_u32(&b.unit_full[unit.slot]));
      unit.next(S::kUnits);
    }
    commit_all<S::PAIR>(smem_u32(&b.scale_empty[u.slot]));
  }
  return true;
}

template <typename S>
__device__ __forceinline__ bool issue_products(Barriers<S>& b, uint8_t* ring, const Depth& depth, uint32_t acc, uint32_t tmem,
                                               uint32_t k, uint32_t idesc, uint32_t first, uint32_t last, Use& u, Use& unit,
                                               int* failed) {
  for (uint32_t st = first; st < last; ++st, u.next(depth.stages)) {
    if (!wait_use(b.full, u, failed)) return false;
    const uint32_t at = smem_u32(ring) + u.slot * S::kStageBytes;
    const uint64_t dp = operand_desc(at), dq = operand_desc(at + S::kPBytes);
    const uint32_t steps = steps_in(k, st);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 2 >= (int)steps) break;
      if (!wait_use(b.unit_full, unit, failed)) return false;
      fence_after();
      const uint32_t tsp = tmem + S::kScaleCol + unit.slot * S::kUnitCols, tsq = tsp + S::kUnitGroups * 4;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (half * 2 + j < (int)steps) {
          // a column of scales holds four bytes per row: one product's with
          // blocks of 16, two products' (bytes 0-1, 2-3) with blocks of 32
          const int g = S::BLOCK == 16 ? j : 0;
          const uint32_t id = S::BLOCK == 16 ? 0u : (uint32_t)j * 2u;
          mma<S::PAIR, S::BLOCK>(acc, dp + (half * 2 + j) * 2, dq + (half * 2 + j) * 2, idesc | (id << 4) | (id << 29),
                                 tsp + g * 4, tsq + g * S::kQTiles * 4, st != first || half + j != 0);
        }
      }
      commit_here<S::PAIR>(smem_u32(&b.unit_empty[unit.slot]));
      unit.next(S::kUnits);
    }
    commit_all<S::PAIR>(smem_u32(&b.empty[u.slot]));
  }
  return true;
}

// Waits until the last uses of a ring have been released: no copy into it is in
// flight then.
__device__ __forceinline__ bool drain_ring(uint64_t* empty, const Use& u, uint32_t size) {
  bool ok = true;
  for (uint32_t i = u.count > size ? u.count - size : 0u; i < u.count; ++i)
    ok &= barrier_wait(smem_u32(empty + i % size), (i / size) & 1u, nullptr);
  return ok;
}

// ---- one tile per block ------------------------------------------------------------
//
// A block of 128 threads computes a tile of 128 rows of one operand (P) by BN
// rows of the other (Q): its warps are the four roles first, and all take the
// accumulators from tensor memory afterwards.  A cluster of `split` blocks
// shares one tile, each with its part of K; the partial sums meet in shared
// memory and each block finishes BN / split columns, adding the parts in rank
// order.
//
// FACTORS: whether there are multipliers, or an alpha that is not a normal number;
// without them the code of factor_of stays out (48 x 14336 x 4096: 12.84 us, with
// it 13.20).  Multipliers are on their way while the pipeline runs (the same
// with two of them: 13.70, read behind it 14.05).
//
// Depth of the rings: half of the shared memory where two blocks share an SM,
// all of it where there are no more blocks than SMs; a row of tiles that streams
// a weight matrix past a few rows is bound by the bytes in flight.
template <int BN, int BLOCK>
struct TileShape {
  static constexpr int kScaleBytes = kStageK / (4 * BLOCK) * 512 * 2, kStageBytes = (128 + BN) * kRowBytes;
  static constexpr int kHalf = 110 * 1024, kWhole = 222 * 1024;
  static constexpr uint32_t kScaleStages = 3, kDeepScaleStages = 8;
  static constexpr uint32_t kStages = (kHalf - kScaleStages * kScaleBytes) / kStageBytes;
  static constexpr uint32_t kDeepStages = (kWhole - kDeepScaleStages * kScaleBytes) / kStageBytes;
  using Pipe = blockmm::Pipe<false, BN, BLOCK, kDeepStages, kDeepScaleStages, BN <= 64 ? 128 : 256>;
  static constexpr int kSmem = kHalf + 1024, kDeepSmem = kWhole + 1024;
  static_assert(Pipe::kStageBytes == kStageBytes && Pipe::kScaleBytes == kScaleBytes, "sizes");
  static_assert(kStages * kStageBytes >= 128 * BN * 4, "the partial sums reuse the stages");
  static_assert(Pipe::kScaleCol >= BN, "accumulators and scales share tensor memory");
};

struct TileParams {
  Maps maps;
  Params r;
  Depth depth;
};

// Adds the parts of N columns of a row, in rank order, and stores the results.
// `here` is the address of the row's first column in this block's part.
template <bool SWAP, int N>
__device__ __forceinline__ void join_parts(const Params& P, const Factor& f, uint32_t split, uint32_t here, uint32_t p,
                                           uint32_t q) {
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (uint32_t r = 0; r < split; r += 2) {  // two blocks' parts in flight
    float x[2][N];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t there = in_block(here, r + s);
      if constexpr (N == 2) {
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x[s][0]), "=f"(x[s][1]) : "r"(there) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(x[s][i]), "=f"(x[s][i + 1]), "=f"(x[s][i + 2]), "=f"(x[s][i + 3]) : "r"(there + i / 4 * 2048)
                       : "memory");
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (v[i] + x[0][i]) + x[1][i];
  }
  store_results<SWAP, N>(P, f, p, q, N, v);
}

template <int BN, int BLOCK, bool SWAP, bool FACTORS>
__global__ void __launch_bounds__(128) tile_kernel(const __grid_constant__ TileParams T, uint32_t split) {
  using S = typename TileShape<BN, BLOCK>::Pipe;
  const Params& P = T.r;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers<S> bars;
  __shared__ uint64_t finished;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int t = threadIdx.x, warp = warp_index();
  uint8_t* stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* scale_stages = stages + T.depth.stages * S::kStageBytes;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&tmem_slot)), "n"(S::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (t == 0) {
    init_barriers(bars);
    barrier_init(smem_u32(&finished), 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_maps(T.maps);
  }
  const uint32_t rank = blockIdx.x % split;
  const uint32_t tile = blockIdx.x / split, p_tiles = (P.p_rows + 127u) >> 7;
  const uint32_t p0 = tile % p_tiles * 128u, q0 = tile / p_tiles * (uint32_t)BN;
  const uint32_t first = (uint32_t)((uint64_t)P.stages * rank / split);
  const uint32_t last = (uint32_t)((uint64_t)P.stages * (rank + 1) / split);
  if (SWAP && warp == 3 && elected()) {
    // The first stages of the many-row operand (the weights) into L2 while the
    // kernel before (the rounding of the few rows) still runs: L2 sees that
    // kernel's writes, so this may come before the wait for it.  One token
    // rounded and multiplied, 8192 x 8192: 13.0 -> 12.5 us; 8 or 32 stages gain
    // no more.
    for (uint32_t st = first; st < last && st < first + 4; ++st) {
      fetch_2d(&T.maps.p, (int32_t)(st * kRowBytes), (int32_t)p0);
      fetch_3d(&T.maps.ps, 0, (int32_t)(st * S::kGroups), (int32_t)(p0 >> 7));
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  blocks::let_next_grid_start();
  blocks::wait_for_previous_grid();
  // under way while the pipeline runs
  const float ma = FACTORS ? multiplier_at(P.multiplier_a) : 1.f, mb = FACTORS ? multiplier_at(P.multiplier_b) : 1.f;
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  if (elected()) {
    Use u, unit;
    if (warp == 0) {
      ok = load_operands<S>(T.maps, bars, stages, T.depth, 0, first, last, (int32_t)p0, (int32_t)q0, u, &failed);
      ok &= drain_ring(bars.empty, u, T.depth.stages);
    } else if (warp == 1) {
      ok = issue_products<S>(bars, stages, T.depth, tmem, tmem, P.k, P.idesc, first, last, u, unit, &failed);
      commit_here<false>(smem_u32(&finished));  // after a wait that ran out too: what was issued completes
    } else if (warp == 2) {
      ok = load_scales<S>(T.maps, bars, scale_stages, T.depth, 0, first, last, (int32_t)(p0 >> 7), (int32_t)(q0 >> 7), u,
                          &failed);
      ok &= drain_ring(bars.scale_empty, u, T.depth.scale_stages);
    } else {
      ok = spread_scales<S>(bars, scale_stages, T.depth, tmem, P.k, first, last, u, unit, &failed);
    }
  }
  __syncwarp();
  ok &= barrier_wait(smem_u32(&finished), 0, nullptr);
  fence_after();
  const bool bad = __syncthreads_or(!ok);
  if (bad && t == 0) atomicExch(&g_expired, 1);
  const float nan = __uint_as_float(0x7FC00000u);
  const Factor f = FACTORS ? factor_of(P.alpha, ma, mb) : Factor{P.alpha, 1.f, 1.f};
  const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
  if (split == 1u && !SWAP && BN >= 32) {
    // the stages are free: 32 x 33 floats of them for each warp
    float* buffer = reinterpret_cast<float*>(stages) + warp * (32 * 33);
#pragma unroll 1
    for (int q = 0; q < BN; q += 32) {
      if (q0 + q >= P.q_rows) break;
      float v[32];
      load_acc32(lanes + q, v);
      acc_loaded();
      if (bad) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = nan;
      }
      rescale<32>(f, v);
      store_turned(P, f.alpha, p0 + warp * 32u, q0 + q, v, buffer);
    }
  } else if (split == 1u) {
#pragma unroll 1
    for (int q = 0; q < BN; q += 16) {
      if (q0 + q >= P.q_rows) break;
      float v[16];
      load_acc16(lanes + q, v);
      if (bad) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = nan;
      }
      store_results<SWAP, 16>(P, f, p0 + t, q0 + q, 16, v);
    }
  } else {
    // four columns of a row side by side, so that both sides move 16 bytes a lane
    float4* part = reinterpret_cast<float4*>(stages);
#pragma unroll 1
    for (int q = 0; q < BN; q += 16) {
      float v[16];
      load_acc16(lanes + q, v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[(q / 4 + i) * 128 + t] = bad ? make_float4(nan, nan, nan, nan)
                                          : make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    cluster_sync();
    const int width = BN / (int)split, w0 = width * (int)rank;
    if (width >= 8) {
#pragma unroll 1
      for (int q = w0; q < w0 + width; q += 8) {
        if (q0 + q >= P.q_rows) break;
        join_parts<SWAP, 8>(P, f, split, smem_u32(part + q / 4 * 128 + t), p0 + t, q0 + q);
      }
    } else if (width == 4) {
      join_parts<SWAP, 4>(P, f, split, smem_u32(part + w0 / 4 * 128 + t), p0 + t, q0 + w0);
    } else {
      join_parts<SWAP, 2>(P, f, split, smem_u32(part + w0 / 4 * 128 + t) + w0 % 4 * 4, p0 + t, q0 + w0);
    }
    cluster_sync();
  }
  fence_before();
  __syncthreads();
  if (warp == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "n"(S::kTmem));
  }
}

// ---- large products: pairs of blocks -------------------------------------------------
//
// A cluster of two blocks on one SM pair computes tiles of 256 rows (of A) by BN
// rows (of B) with cta_group::2 instructions that the first block issues: each
// block holds its 128 rows of A and half of B's rows, so B crosses shared
// memory once for both, and accumulates its 128 x BN part in its own tensor
// memory.  The blocks are persistent (tile = cluster, cluster + clusters, ...)
// and specialised: four warps are the pipeline's roles, eight take results out,
// so that the results of a tile leave while the next one is computed.
//
// Tensor memory (512 columns): two accumulators of BN columns and the unit
// buffers of the scales.  For BN = 256 the accumulators share columns: the
// results' warps take those out first and then let the next tile start.
template <int BN, int BLOCK>
struct PairShape {
  static constexpr int kScaleStages = 4;
  static constexpr int kScaleBytes = kStageK / (4 * BLOCK) * 512 * (1 + BN / 128);
  static constexpr int kBoxBytes = 5120;  // a results warp's shared memory: its box, or the 32 x 33 buffer
  static constexpr int kStages =
      (226 * 1024 - 1024 - 8 * kBoxBytes - kScaleStages * kScaleBytes) / (128 * kRowBytes + BN / 2 * kRowBytes);
  using Pipe = blockmm::Pipe<true, BN, BLOCK, kStages, kScaleStages, 512>;
  static constexpr int kSmem = kStages * Pipe::kStageBytes + kScaleStages * Pipe::kScaleBytes + 8 * kBoxBytes + 1024;
  static constexpr int kSecond = 128;           // column of the second accumulator
  static constexpr int kShared = BN - kSecond;  // columns both use: 0 or 128
  static_assert((BN == 128 || BN == 256) && kSecond + BN <= Pipe::kScaleCol, "tensor memory");
};

struct PairParams {
  Maps maps;
  CUtensorMap d_map;
  Params r;
  uint32_t p_tiles, q_tiles;
  int32_t boxed;  // results leave through d_map: rows of D, and of C, on 16-byte boundaries
};

constexpr int kPairThreads = 384;  // warps 0-3 the roles, 4-11 the results: two warps for each 32 rows

template <int BN, int BLOCK>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1) pair_kernel(const __grid_constant__ PairParams P) {
  using L = PairShape<BN, BLOCK>;
  using S = typename L::Pipe;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers<S> bars;
  __shared__ uint64_t acc_full[2], acc_free[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int t = threadIdx.x, warp = warp_index(), lane = t & 31;
  const uint32_t rank = cluster_rank();
  uint8_t* boxes = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* stages = boxes + 8 * L::kBoxBytes;
  uint8_t* scale_stages = stages + S::STAGES * S::kStageBytes;
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&tmem_slot)), "n"(S::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (t == 0) {
    init_barriers(bars);
    for (int i = 0; i < 2; ++i) {
      barrier_init(smem_u32(&acc_full[i]), 1);
      barrier_init(smem_u32(&acc_free[i]), 16);  // eight warps of each block
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_maps(P.maps);
  }
  fence_before();
  cluster_sync();
  fence_after();
  blocks::let_next_grid_start();
  blocks::wait_for_previous_grid();
  const uint32_t tmem = tmem_slot;
  const uint32_t clusters = gridDim.x / 2, tiles = P.p_tiles * P.q_tiles, stage_count = P.r.stages;
  bool ok = true;
  if (warp < 4) {
    if ((rank == 0 || warp == 0 || warp == 2) && elected()) {
      constexpr Depth depth = {S::STAGES, S::SCALE_STAGES};
      Use u, unit;
      uint32_t count = 0;
      for (uint32_t tile = blockIdx.x / 2; ok && tile < tiles; tile += clusters, ++count) {
        const uint32_t pt = tile % P.p_tiles, qt = tile / P.p_tiles;
        const int32_t p0 = (int32_t)(pt * 256u + rank * 128u), q0 = (int32_t)(qt * BN + rank * (BN / 2));
        if (warp == 0) {
          ok = load_operands<S>(P.maps, bars, stages, depth, rank, 0, stage_count, p0, q0, u, &failed);
        } else if (warp == 2) {
          ok = load_scales<S>(P.maps, bars, scale_stages, depth, rank, 0, stage_count, p0 >> 7, (int32_t)(qt * S::kQTiles),
                              u, &failed);
        } else if (warp == 3) {
          ok = spread_scales<S>(bars, scale_stages, depth, tmem, P.r.k, 0, stage_count, u, unit, &failed);
        } else {
          // the columns shared with the tile before are free (and all of the
          // one before that, whose results were taken out first), or without
          // shared columns those of the tile before the last
          const uint32_t back = L::kShared ? 1u : 2u;
          if (count >= back) {
            const uint32_t before = count - back;
            ok = barrier_wait(smem_u32(&acc_free[before & 1u]), (before >> 1) & 1u, &failed);
            if (!ok) break;
            fence_after();
          }
          ok = issue_products<S>(bars, stages, depth, tmem + (count & 1u) * L::kSecond, tmem, P.r.k, P.r.idesc, 0,
                                 stage_count, u, unit, &failed);
          if (ok) commit_all<true>(smem_u32(&acc_full[count & 1u]));  // if not, the results' waits run out too
        }
      }
      if (warp == 0) ok &= drain_ring(bars.empty, u, S::STAGES);
      if (warp == 2) ok &= drain_ring(bars.scale_empty, u, S::SCALE_STAGES);
    }
  } else {
    const int quarter = warp & 3;  // the lanes of tensor memory that this warp may read
    const Factor f = factor_of(P.r.alpha, multiplier_at(P.r.multiplier_a), multiplier_at(P.r.multiplier_b));
    const int side = warp >= 8;     // of the two warps of these lanes: every other chunk
    uint8_t* box = boxes + (quarter * 2 + side) * L::kBoxBytes;
    uint32_t count = 0, tile = blockIdx.x / 2;
    for (; ok && tile < tiles; tile += clusters, ++count) {
      const uint32_t pt = tile % P.p_tiles, qt = tile / P.p_tiles;
      const uint32_t p = pt * 256u + rank * 128u + quarter * 32u, q0 = qt * BN;
      ok = barrier_wait(smem_u32(&acc_full[count & 1u]), (count >> 1) & 1u, &failed);
      ok = __all_sync(0xFFFFFFFFu, ok);
      fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (count & 1u) * L::kSecond;
      const uint32_t free_bar = in_block(smem_u32(&acc_free[count & 1u]), 0);
      // 64 columns at a time.  The shared ones (the last of the first accumulator,
      // the first of the second) go first, and let the next tile start before
      // anything is done with them
      auto take = [&](int chunk, bool release) {
        float v[64];
        load_acc32(acc + chunk * 64, v);
        load_acc32(acc + chunk * 64 + 32, v + 32);
        acc_loaded();
        if (release) {
          fence_before();
          __syncwarp();
          if (lane == 0) arrive_in(free_bar);
        }
        if (!ok) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = __uint_as_float(0x7FC00000u);
        }
        rescale<64>(f, v);
        const uint32_t q = q0 + chunk * 64;
        if (P.boxed) {
          if (P.r.c == nullptr) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] *= f.alpha;
          } else if (P.r.c_type == T5E_REAL_F32) {
            add_row<4>(P.r, f.alpha, p + lane, q, v);
          } else {
            add_row<2>(P.r, f.alpha, p + lane, q, v);
          }
          store_box(P.r, &P.d_map, p, q, v, box);
        } else {
          store_turned(P.r, f.alpha, p, q, v, reinterpret_cast<float*>(box));
          store_turned(P.r, f.alpha, p, q + 32, v + 32, reinterpret_cast<float*>(box));
        }
      };
      if constexpr (L::kShared > 0) {
        const int shared = (count & 1u) == 0u ? 2 : 0;
        take(shared + side, true);
        take(2 - shared + side, false);
      } else {
        take(side, true);
      }
    }
    // a wait ran out: the tiles behind that one become NaN as well.  No waits, and
    // no accumulators released: the other block's may be good and not yet taken
    spoil_tiles<BN>(tile, tiles, clusters, P.p_tiles, rank * 128u + quarter * 32u, side * 64u, lane, P.r.p_rows, P.r.q_rows,
                    [&](uint32_t row, uint32_t col) {
                      write_real(P.r.d, (int64_t)row * P.r.d_stride + col, P.r.d_type, __uint_as_float(0x7FC00000u));
                    });
    if (P.boxed && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  fence_before();
  const bool bad = __syncthreads_or(!ok);
  if (t == 0 && bad) atomicExch(&g_expired, 1);
  cluster_sync();
  if (warp == 4) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "n"(S::kTmem));
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

// Map of scale tiles as 32-bit words: 128 words, the groups, the tiles of rows;
// boxes of one pipeline stage's groups by `tiles` tiles.
int encode_scales(CUtensorMap* map, const t5e_blocks& b, uint32_t box_groups, uint32_t box_tiles) {
  const EncodeTiled f = encoder();
  if (!f) return T5E_ERR_CUDA;
  const cuuint64_t groups = scale_groups(b), tiles = (b.rows + 127) / 128;
  const cuuint64_t dims[3] = {128, groups, tiles}, strides[2] = {512, groups * 512};
  const cuuint32_t box[3] = {128, box_groups, box_tiles}, unit[3] = {1, 1, 1};
  const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, b.scales, dims, strides, box, unit,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_cuda_error("cuTensorMapEncodeTiled", cudaErrorInvalidValue);
    return T5E_ERR_CUDA;
  }
  return T5E_OK;
}

// Map of the results, boxes of 128 bytes by 32 rows; *boxed = 0 where the rows
// do not lie on 16-byte boundaries.
int encode_results(CUtensorMap* map, const Params& P, int32_t* boxed) {
  const int bytes = P.d_type == T5E_REAL_F32 ? 4 : 2;
  *boxed = 0;
  if ((reinterpret_cast<uintptr_t>(P.d) & 15u) || (P.d_stride * bytes) % 16 || P.d_stride * bytes >= (1ll << 40)) return T5E_OK;
  const EncodeTiled f = encoder();
  if (!f) return T5E_ERR_CUDA;
  const cuuint64_t dims[2] = {P.q_rows, P.p_rows}, strides[1] = {(cuuint64_t)(P.d_stride * bytes)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), 32}, unit[2] = {1, 1};
  const CUtensorMapDataType type = P.d_type == T5E_REAL_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : P.d_type == T5E_REAL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = f(map, type, 2, P.d, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_cuda_error("cuTensorMapEncodeTiled", cudaErrorInvalidValue);
    return T5E_ERR_CUDA;
  }
  *boxed = 1;
  return T5E_OK;
}

template <typename S>
int encode_maps(Maps* m, const t5e_blocks& p, const t5e_blocks& q) {
  int rc = encode(&m->p, p, 128);
  if (rc == T5E_OK) rc = encode(&m->q, q, S::kQRows);
  if (rc == T5E_OK) rc = encode_scales(&m->ps, p, S::kGroups, 1);
  if (rc == T5E_OK) rc = encode_scales(&m->qs, q, S::kGroups, S::kQTiles);
  return rc;
}

// Instruction descriptor: E2M1 x E2M1, M = 128, `n` columns.
uint32_t instruction(const t5e_blocks& b, uint32_t n, uint32_t m = 128) {
  return (1u << 7) | (1u << 10) | ((n / 8u) << 17) | ((b.scale_format == T5E_SCALE_UE8M0 ? 1u : 0u) << 23) |
         ((m / 128u) << 27);
}

int blocks_launched(cudaError_t e) {
  if (e != cudaSuccess) {
    set_cuda_error("block product launch", e);
    return T5E_ERR_CUDA;
  }
  return kernel_status("block product launch");
}

// Blocks of clusters of `split` that the device runs at once with one block an SM
// (clusters stay within a group of SMs: 148, 148, 132 and 120 blocks on a B200),
// looked up once per device.
uint64_t blocks_at_once(uint32_t split) {
  static std::atomic<int> known[64][4];
  const int which = split == 1u ? 0 : split == 2u ? 1 : split == 4u ? 2 : 3;
  int dev = 0;
  const bool cached = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
  int n = cached ? known[dev][which].load(std::memory_order_relaxed) : 0;
  if (n > 0) return (uint64_t)n;
  using S = TileShape<128, 16>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = S::kDeepSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {split, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (raise_smem_limit<tile_kernel<128, 16, false, true>>(S::kDeepSmem, "block product attribute") != T5E_OK ||
      cudaOccupancyMaxActiveClusters(&n, tile_kernel<128, 16, false, true>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();  // an estimate only: the launch reports what is wrong
    return (uint64_t)sm_count();
  }
  n *= (int)split;
  if (cached) known[dev][which].store(n, std::memory_order_relaxed);
  return (uint64_t)n;
}

template <int BN, int BLOCK, bool SWAP>
int launch_tile(const Params& params, const t5e_blocks& p, const t5e_blocks& q, uint32_t split, cudaStream_t stream) {
  using S = TileShape<BN, BLOCK>;
  TileParams P;
  P.r = params;
  int rc = encode_maps<typename S::Pipe>(&P.maps, p, q);
  // no multipliers and an ordinary alpha need none of factor_of's code
  const bool plain = params.multiplier_a == nullptr && params.multiplier_b == nullptr && is_normal(params.alpha);
  const auto kernel = plain ? tile_kernel<BN, BLOCK, SWAP, false> : tile_kernel<BN, BLOCK, SWAP, true>;
  if (rc == T5E_OK)
    rc = plain ? raise_smem_limit<tile_kernel<BN, BLOCK, SWAP, false>>(S::kDeepSmem, "block product attribute")
               : raise_smem_limit<tile_kernel<BN, BLOCK, SWAP, true>>(S::kDeepSmem, "block product attribute");
  if (rc != T5E_OK) return rc;
  P.r.idesc = instruction(p, BN);
  cudaLaunchConfig_t cfg = {};
  const uint64_t grid = ((p.rows + 127) / 128) * ((q.rows + BN - 1) / BN) * split;
  if (grid > 0x7FFFFFFFull) return T5E_ERR_INVALID;
  const bool deep = grid <= blocks_at_once(split);
  P.depth = deep ? Depth{S::kDeepStages, S::kDeepScaleStages} : Depth{S::kStages, S::kScaleStages};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = deep ? S::kDeepSmem : S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {split, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return blocks_launched(cudaLaunchKernelEx(&cfg, kernel, P, split));
}

template <int BLOCK>
int launch_form(const Params& P, const t5e_blocks& p, const t5e_blocks& q, bool swap, uint32_t split, cudaStream_t stream) {
  if (q.rows <= 16)
    return swap ? launch_tile<16, BLOCK, true>(P, p, q, split, stream) : launch_tile<16, BLOCK, false>(P, p, q, split, stream);
  if (q.rows <= 32)
    return swap ? launch_tile<32, BLOCK, true>(P, p, q, split, stream) : launch_tile<32, BLOCK, false>(P, p, q, split, stream);
  if (q.rows <= 64)
    return swap ? launch_tile<64, BLOCK, true>(P, p, q, split, stream) : launch_tile<64, BLOCK, false>(P, p, q, split, stream);
  return swap ? launch_tile<128, BLOCK, true>(P, p, q, split, stream) : launch_tile<128, BLOCK, false>(P, p, q, split, stream);
}

template <int BN, int BLOCK>
int launch_pair(const Params& params, const t5e_blocks& a, const t5e_blocks& b, cudaStream_t stream) {
  using S = PairShape<BN, BLOCK>;
  PairParams P;
  P.r = params;
  int rc = encode_maps<typename S::Pipe>(&P.maps, a, b);
  if (rc == T5E_OK) rc = raise_smem_limit<pair_kernel<BN, BLOCK>>(S::kSmem, "block product attribute");
  if (rc != T5E_OK) return rc;
  P.boxed = 0;
  const int c_bytes = params.c_type == T5E_REAL_F32 ? 4 : 2;
  if (params.c == nullptr || (params.c_q_stride == 1 && (params.c_p_stride * c_bytes) % 16 == 0 &&
                              (reinterpret_cast<uintptr_t>(params.c) & 15u) == 0)) {
    rc = encode_results(&P.d_map, params, &P.boxed);
    if (rc != T5E_OK) return rc;
  }
  if (!P.boxed) P.d_map = P.maps.p;  // not read
  P.r.idesc = instruction(a, BN, 256);
  P.p_tiles = (uint32_t)((a.rows + 255) / 256);
  P.q_tiles = (uint32_t)((b.rows + BN - 1) / BN);
  const uint64_t tiles = (uint64_t)P.p_tiles * P.q_tiles, room = (uint64_t)sm_count() / 2;
  if (tiles > 0x7FFFFFFFull) return T5E_ERR_INVALID;
  return blocks_launched(launch_dependent(pair_kernel<BN, BLOCK>, dim3((unsigned)(2 * (tiles < room ? tiles : room))),
                                          kPairThreads, S::kSmem, stream, P));
}

uint32_t choose_form(uint64_t p_rows, uint64_t q_rows, uint32_t stages, bool swap) {
  const uint64_t pairs = (uint64_t)sm_count() / 2;
  auto tiles = [&](uint64_t rows, uint64_t cols) { return ((p_rows + rows - 1) / rows) * ((q_rows + cols - 1) / cols); };
  // Parts of K: as many as run at once, with two stages or more each; where Q is
  // one tile, two blocks an SM (1 x 8192 x 8192 in 4 parts 10.9 us, in 2 parts
  // 12.1; 100 x 8192 x 8192 16.0 and 18.7; but 512 x 512 x 8192 in 8 parts 11.3,
  // in 4 parts 10.0).  Counting blocks is not best everywhere: the two parts it
  // picks take 13.5 us for 48 x 14336 x 4096, whole 13.2, and for 48 x 18944 x
  // 4096 (UE4M3) 16.3 and 15.0
  const uint64_t share = q_rows <= 128 ? 2 : 1;
  uint32_t split = 1;
  while (split < 8 && stages >= split * 4 && tiles(128, 128) * split * 2 <= share * blocks_at_once(split * 2)) split *= 2;
  if (swap || q_rows <= 64 || split >= 4) return split;
  // Whole K in pairs: waves of tiles over the pairs (the main loop alone: neither
  // K nor the results' phase, the longer one at few stages, is counted), a
  // 256-wide tile taking 1.6
  // times a 128-wide one (1536 x 1536 x 8192: 16.7 us in 36 tiles of 256, 15.8
  // in 72 of 128; 8192 x 4096 x 4096: 59 us in 7 waves, 81 in 14)
  const uint64_t wide = (tiles(256, 256) + pairs - 1) / pairs * 16, narrow = (tiles(256, 128) + pairs - 1) / pairs * 10;
  return wide < narrow ? 256 : 128;
}

}  // namespace blockmm
}  // namespace t5e

extern "C" {

int t5e_block_scaled_mm(const t5e_block_mm* mm, void* stream) {
  using namespace t5e;
  using namespace t5e::blockmm;
  if (!mm || !blocks_ok(&mm->a) || !blocks_ok(&mm->b)) return T5E_ERR_INVALID;
  const t5e_blocks &a = mm->a, &b = mm->b;
  auto real = [](int32_t t) { return t == T5E_REAL_F32 || t == T5E_REAL_BF16 || t == T5E_REAL_F16; };
  if (a.k != b.k || a.scale_format != b.scale_format || a.scale_block != b.scale_block || !real(mm->d_type) ||
      (mm->c && !real(mm->c_type)))
    return T5E_ERR_INVALID;
  const int32_t form = mm->form;
  if (form != 0 && form != 1 && form != 2 && form != 4 && form != 8 && form != 128 && form != 256) return T5E_ERR_INVALID;
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
  P.alpha = mm->alpha;
  P.c_type = mm->c_type;
  P.d_type = mm->d_type;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t chosen = form != 0 ? (uint32_t)form : choose_form(p.rows, q.rows, P.stages, swap);
  if (chosen >= 128) {
    if (swap) return T5E_ERR_INVALID;  // few rows: a tile of 256 would be empty
    if (chosen == 256)
      return a.scale_block == 32 ? launch_pair<256, 32>(P, p, q, s) : launch_pair<256, 16>(P, p, q, s);
    return a.scale_block == 32 ? launch_pair<128, 32>(P, p, q, s) : launch_pair<128, 16>(P, p, q, s);
  }
  if (chosen > P.stages) return T5E_ERR_INVALID;  // every part has work
  return a.scale_block == 32 ? launch_form<32>(P, p, q, swap, chosen, s) : launch_form<16>(P, p, q, swap, chosen, s);
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
