// t5e_blocks.cu -- real tensors to block-scaled E2M1 rows and back.
//
// All of it is bound by memory: a BF16 element is 2 bytes in and 0.56 out
// (0.53 with 32-element blocks), about 14 thread instructions at the rate HBM
// delivers it.
#include <cuda_runtime.h>

#include "t5e.h"
#include "t5e_blocks.cuh"
#include "t5e_dispatch.h"

namespace t5e {
namespace blocks {

constexpr int kThreads = 256;

// ---- the largest magnitude -------------------------------------------------
//
// Magnitudes are compared as integers: the bits of |x| order like |x|, and a
// NaN sorts above infinity, so it is not lost as it would be in fmaxf.

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < blockDim.x / 32 ? shared[threadIdx.x] : 0u;
  if (threadIdx.x < 32) {
    v = __reduce_max_sync(0xFFFFFFFFu, v);
    if (threadIdx.x == 0) shared[0] = v;
  }
  __syncthreads();
  return shared[0];
}

template <int TYPE>
__device__ __forceinline__ uint32_t word_max(uint32_t w) {
  if constexpr (TYPE == T5E_REAL_F32) {
    return w & 0x7FFFFFFFu;
  } else {  // the two halves' magnitudes, both kept as 16-bit bit patterns
    return w & 0x7FFF7FFFu;
  }
}

// F32 bits of a 16-bit type's magnitude bits.
template <int TYPE>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t h) {
  if constexpr (TYPE == T5E_REAL_F32) return h;
  else if constexpr (TYPE == T5E_REAL_BF16) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

template <int TYPE>
__device__ __forceinline__ uint32_t join_max(uint32_t a, uint32_t b) {
  if constexpr (TYPE == T5E_REAL_F32) return max(a, b);
  else return __vmaxu2(a, b);
}

template <int TYPE>
__device__ __forceinline__ uint32_t final_max(uint32_t v) {
  if constexpr (TYPE == T5E_REAL_F32) return v;
  else return magnitude_bits<TYPE>(max(v & 0xFFFFu, v >> 16));
}

template <int TYPE>
__device__ __forceinline__ uint32_t element_bits(const void* x, uint64_t i) {
  if constexpr (TYPE == T5E_REAL_F32) return static_cast<const uint32_t*>(x)[i] & 0x7FFFFFFFu;
  else return static_cast<const uint16_t*>(x)[i] & 0x7FFFu;
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kThreads) partials_kernel(const void* __restrict__ x, uint64_t rows, uint64_t cols,
                                                            int64_t stride, uint32_t* __restrict__ partials) {
  __shared__ uint32_t shared[kThreads / 32];
  let_next_grid_start();
  wait_for_previous_grid();
  constexpr int kPer = 16 / Real<TYPE>::kBytes;
  uint32_t best = 0u;
  // a contiguous tensor comes as one row, which all blocks share; otherwise
  // each block takes whole rows
  const bool one = rows == 1;
  const uint64_t first = one ? (uint64_t)blockIdx.x * kThreads + threadIdx.x : threadIdx.x;
  const uint64_t step = one ? (uint64_t)gridDim.x * kThreads : kThreads;
  for (uint64_t r = one ? 0 : blockIdx.x; r < rows; r += one ? 1 : gridDim.x) {
    const char* row = static_cast<const char*>(x) + (int64_t)r * stride * Real<TYPE>::kBytes;
    uint64_t done = 0;
    if constexpr (VEC) {
      const uint64_t vecs = cols / kPer;
      const uint4* p = reinterpret_cast<const uint4*>(row);
      uint64_t i = first;
      for (; i + 3 * step < vecs; i += 4 * step) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __ldg(p + i + j * step);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          best = join_max<TYPE>(best, join_max<TYPE>(join_max<TYPE>(word_max<TYPE>(v[j].x), word_max<TYPE>(v[j].y)),
                                                     join_max<TYPE>(word_max<TYPE>(v[j].z), word_max<TYPE>(v[j].w))));
      }
      for (; i < vecs; i += step) {
        const uint4 v = __ldg(p + i);
        best = join_max<TYPE>(best, join_max<TYPE>(join_max<TYPE>(word_max<TYPE>(v.x), word_max<TYPE>(v.y)),
                                                   join_max<TYPE>(word_max<TYPE>(v.z), word_max<TYPE>(v.w))));
      }
      done = vecs * kPer;
    }
    for (uint64_t i = done + first; i < cols; i += step) best = join_max<TYPE>(best, element_bits<TYPE>(row, i));
  }
  const uint32_t m = block_max(final_max<TYPE>(best), shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

__global__ void __launch_bounds__(kThreads) multiplier_kernel(const uint32_t* __restrict__ partials, int count,
                                                              float* __restrict__ multiplier) {
  __shared__ uint32_t shared[kThreads / 32];
  let_next_grid_start();
  wait_for_previous_grid();
  uint32_t best = 0u;
  for (int i = threadIdx.x; i < count; i += kThreads) best = max(best, partials[i]);
  best = block_max(best, shared);
  if (threadIdx.x == 0) *multiplier = multiplier_of(best);
}

// The multiplier a quantising block works with: none, given, or taken from the
// partial maxima (every block joins them for itself, which saves a launch;
// block 0 stores the result).
__device__ __forceinline__ float load_multiplier(float* multiplier, const uint32_t* partials, int count,
                                                 uint32_t* shared) {
  if (partials != nullptr) {
    uint32_t best = 0u;
    for (int i = threadIdx.x; i < count; i += blockDim.x) best = max(best, __ldg(partials + i));
    const float m = multiplier_of(block_max(best, shared));
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *multiplier = m;
    return m;
  }
  return multiplier != nullptr ? *multiplier : 1.f;
}

// ---- blocks along the rows ---------------------------------------------------
//
// A thread takes 16 consecutive elements: one block, or half of a 32-element
// one whose other half its neighbour lane holds.  Per row the chunks run up
// to a whole group of four scales, so that four (eight) neighbouring lanes
// always hold one group and one of them stores its four scale bytes as a word.
template <int TYPE, bool E8M0, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const void* __restrict__ x, uint32_t rows, uint64_t row0,
                                                                 uint32_t k, int64_t stride, bool ceil,
                                                                 float* multiplier, const uint32_t* partials, int count,
                                                                 uint8_t* __restrict__ data, int64_t data_stride,
                                                                 uint8_t* __restrict__ scales, uint32_t groups) {
  __shared__ uint32_t shared[kThreads / 32];
  let_next_grid_start();
  wait_for_previous_grid();
  const float m = load_multiplier(multiplier, partials, count, shared);
  constexpr uint32_t kLanes = BLOCK / 4;               // lanes of one group of four scales
  const uint32_t chunks = groups * kLanes;             // 16-element chunks per row
  const uint32_t stored = ((k + 31u) / 32u) * 2u;      // chunks with codes in `data`
  const uint32_t total = rows * chunks;
  const int lane = threadIdx.x & 31;
  for (uint32_t base = blockIdx.x * kThreads + (threadIdx.x & ~31u); base < total; base += gridDim.x * kThreads) {
    const uint32_t item = base + lane;
    const bool in = item < total;
    const uint32_t row = in ? item / chunks : 0u, chunk = in ? item - row * chunks : 0u;
    const uint32_t e0 = chunk * 16u;
    float v[16];
    uint32_t top = 0u;
    const char* src = static_cast<const char*>(x) + ((int64_t)(row0 + row) * stride + e0) * Real<TYPE>::kBytes;
    if (VEC && in && e0 + 16u <= k) {
      constexpr int kVecs = Real<TYPE>::kBytes;  // 16-byte vectors of 16 elements
      uint4 w[kVecs];
#pragma unroll
      for (int j = 0; j < kVecs; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(src) + j);
      const uint32_t* words = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
      for (int j = 0; j < kVecs * 4; ++j) {
        top = join_max<TYPE>(top, word_max<TYPE>(words[j]));
        if constexpr (TYPE == T5E_REAL_F32) v[j] = __uint_as_float(words[j]);
        else unpack2<TYPE>(words[j], v[2 * j], v[2 * j + 1]);
      }
      top = final_max<TYPE>(top);
    } else {
      using T = typename Real<TYPE>::type;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        v[j] = in && e0 + j < k ? to_f32(reinterpret_cast<const T*>(src)[j]) : 0.f;
        top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
    }
    if constexpr (BLOCK == 32) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    float step, inv;
    // rounding to F32 is monotonic: the largest product is the product of the largest
    uint32_t word = block_scale<E8M0>(__uint_as_float(top) * m, ceil, step, inv);
    const bool finite = word != (E8M0 ? 0xFFu : 0x7Fu);
    if (e0 / BLOCK * BLOCK >= k) word = 0u;  // a scale behind the last block
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = divide<E8M0>(v[j] * m, step, inv);
    uint2 codes = make_uint2(e2m1x8(v), e2m1x8(v + 8));
    if (!finite) codes = make_uint2(0u, 0u);
    if (in && chunk < stored)
      *reinterpret_cast<uint2*>(data + (int64_t)(row0 + row) * data_stride + chunk * 8u) = codes;
    // four scale bytes to one word
    if constexpr (BLOCK == 16) {
      word <<= 8 * (lane & 3);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
    } else {
      word <<= 8 * ((lane >> 1) & 3);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
    }
    if (in && lane % kLanes == 0)
      *reinterpret_cast<uint32_t*>(scales + scale_offset(row0 + row, e0 / BLOCK, groups)) = word;
  }
}

// ---- blocks along the columns -------------------------------------------------
//
// Element i of output row c is x[i][c].  A warp takes 32 rows by 64 columns: a
// lane holds two neighbouring columns of all 32 rows in registers (two
// 16-element blocks or one of 32), so the maxima need no exchange and every
// load is one line of a row.  Eight warps stack to 256 rows; the codes are
// turned through shared memory so that each output row gets 128 consecutive
// bytes.
constexpr int kColTileC = 64, kColTileR = 256, kColPitch = kColTileR / 2 + 16;

template <int TYPE, bool E8M0, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_cols_kernel(const void* __restrict__ x, uint64_t rows, uint64_t cols,
                                                                 int64_t stride, bool ceil, float* multiplier,
                                                                 const uint32_t* partials, int count,
                                                                 uint8_t* __restrict__ data, int64_t data_stride,
                                                                 uint8_t* __restrict__ scales, uint32_t groups) {
  __shared__ uint32_t shared[kThreads / 32];
  __shared__ __align__(16) uint8_t codes[kColTileC * kColPitch];
  __shared__ __align__(16) uint8_t steps[kColTileC * (kColTileR / 16)];
  let_next_grid_start();
  wait_for_previous_grid();
  const float m = load_multiplier(multiplier, partials, count, shared);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kSteps = kColTileR / BLOCK;  // scales of a tile per column
  const uint64_t c0 = (uint64_t)blockIdx.x * kColTileC;
  const uint64_t padded = (rows + 31) / 32 * 32;
  for (uint64_t r0 = (uint64_t)blockIdx.y * kColTileR; r0 < padded; r0 += (uint64_t)gridDim.y * kColTileR) {
    const uint64_t r = r0 + warp * 32, c = c0 + lane * 2;
    using T = typename Real<TYPE>::type;
    const T* src = static_cast<const T*>(x) + (int64_t)r * stride + (int64_t)c;
    float v[2][32];
    if (VEC && r + 32 <= rows && c + 2 <= cols) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if constexpr (TYPE == T5E_REAL_F32) {
          const float2 f = __ldg(reinterpret_cast<const float2*>(src + i * stride));
          v[0][i] = f.x;
          v[1][i] = f.y;
        } else {
          unpack2<TYPE>(__ldg(reinterpret_cast<const uint32_t*>(src + i * stride)), v[0][i], v[1][i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[0][i] = r + i < rows && c < cols ? to_f32(src[i * stride]) : 0.f;
        v[1][i] = r + i < rows && c + 1 < cols ? to_f32(src[i * stride + 1]) : 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t out[4];
#pragma unroll
      for (int b = 0; b < 32 / BLOCK; ++b) {
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < BLOCK; ++i) top = max(top, __float_as_uint(v[h][b * BLOCK + i]) & 0x7FFFFFFFu);
        float step, inv;
        uint32_t word = block_scale<E8M0>(__uint_as_float(top) * m, ceil, step, inv);
        const bool finite = word != (E8M0 ? 0xFFu : 0x7Fu);
        if (r + b * BLOCK >= rows) word = 0u;
#pragma unroll
        for (int i = 0; i < BLOCK; ++i) v[h][b * BLOCK + i] = divide<E8M0>(v[h][b * BLOCK + i] * m, step, inv);
#pragma unroll
        for (int i = 0; i < BLOCK / 8; ++i)
          out[b * (BLOCK / 8) + i] = finite ? e2m1x8(&v[h][b * BLOCK + 8 * i]) : 0u;
        steps[(lane * 2 + h) * (kColTileR / 16) + warp * (32 / BLOCK) + b] = (uint8_t)word;
      }
      *reinterpret_cast<uint4*>(codes + (lane * 2 + h) * kColPitch + warp * 16) =
          make_uint4(out[0], out[1], out[2], out[3]);
    }
    __syncthreads();
    // 64 output rows of 8 vectors of 16 bytes
#pragma unroll
    for (int i = threadIdx.x; i < kColTileC * (kColTileR / 32); i += kThreads) {
      const int col = i / (kColTileR / 32), part = i % (kColTileR / 32);
      if (c0 + col < cols && r0 + part * 32 < padded)
        *reinterpret_cast<uint4*>(data + (int64_t)(c0 + col) * data_stride + (int64_t)(r0 / 2) + part * 16) =
            *reinterpret_cast<const uint4*>(codes + col * kColPitch + part * 16);
    }
    // one word of four scales per column and group
    for (int i = threadIdx.x; i < kColTileC * (kSteps / 4); i += kThreads) {
      const int col = i % kColTileC, g = i / kColTileC;
      const uint32_t group = (uint32_t)(r0 / (4 * BLOCK)) + g;
      if (c0 + col < cols && group < groups)
        *reinterpret_cast<uint32_t*>(scales + scale_offset(c0 + col, group * 4, groups)) =
            *reinterpret_cast<const uint32_t*>(steps + col * (kColTileR / 16) + g * 4);
    }
    __syncthreads();
  }
}

// ---- back to real values -------------------------------------------------------

template <int TYPE, bool E8M0, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ data, int64_t data_stride,
                                                              const uint8_t* __restrict__ scales, uint32_t groups,
                                                              uint32_t rows, uint64_t row0, uint32_t k,
                                                              const float* multiplier, void* __restrict__ out,
                                                              int64_t out_stride) {
  let_next_grid_start();
  wait_for_previous_grid();
  const float back = multiplier != nullptr ? 1.f / *multiplier : 1.f;
  const uint32_t chunks = (k + 15u) / 16u;
  const uint32_t total = rows * chunks;
  using T = typename Real<TYPE>::type;
  for (uint32_t item = blockIdx.x * kThreads + threadIdx.x; item < total; item += gridDim.x * kThreads) {
    const uint32_t row = item / chunks, chunk = item - row * chunks, e0 = chunk * 16u;
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(data + (int64_t)(row0 + row) * data_stride + chunk * 8u));
    const float s = scale_value<E8M0>(__ldg(scales + scale_offset(row0 + row, e0 / BLOCK, groups)));
    float v[16];
    from_e2m1x8(w.x, v);
    from_e2m1x8(w.y, v + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = v[j] * s * back;
    T* dst = static_cast<T*>(out) + (int64_t)(row0 + row) * out_stride + e0;
    if (VEC && e0 + 16u <= k) {
      if constexpr (TYPE == T5E_REAL_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          reinterpret_cast<float4*>(dst)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          reinterpret_cast<uint4*>(dst)[j] =
              make_uint4(pack2<TYPE>(v[8 * j], v[8 * j + 1]), pack2<TYPE>(v[8 * j + 2], v[8 * j + 3]),
                         pack2<TYPE>(v[8 * j + 4], v[8 * j + 5]), pack2<TYPE>(v[8 * j + 6], v[8 * j + 7]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (e0 + j < k) dst[j] = from_f32<TYPE>(v[j]);
    }
  }
}

// ---- host side -------------------------------------------------------------------

int type_bytes(int32_t type) { return type == T5E_REAL_F32 ? 4 : 2; }

bool type_ok(int32_t type) { return type == T5E_REAL_F32 || type == T5E_REAL_BF16 || type == T5E_REAL_F16; }

int launched(cudaError_t err, const char* what) {
  if (err != cudaSuccess) {
    set_cuda_error(what, err);
    return T5E_ERR_CUDA;
  }
  return kernel_status(what);
}

// Calls f with compile-time (type, UE8M0, block, vector) for a run-time choice.
template <typename F>
int with_form(int32_t type, const t5e_blocks& b, bool vec, F f) {
  auto by_vec = [&](auto t, auto e8, auto blk) {
    return vec ? f(t, e8, blk, std::true_type{}) : f(t, e8, blk, std::false_type{});
  };
  auto by_scale = [&](auto t) {
    if (b.scale_format == T5E_SCALE_UE4M3) return by_vec(t, std::false_type{}, std::integral_constant<int, 16>{});
    if (b.scale_block == 16) return by_vec(t, std::true_type{}, std::integral_constant<int, 16>{});
    return by_vec(t, std::true_type{}, std::integral_constant<int, 32>{});
  };
  if (type == T5E_REAL_F32) return by_scale(std::integral_constant<int, T5E_REAL_F32>{});
  if (type == T5E_REAL_BF16) return by_scale(std::integral_constant<int, T5E_REAL_BF16>{});
  return by_scale(std::integral_constant<int, T5E_REAL_F16>{});
}

unsigned grid_of(uint64_t blocks, unsigned per_sm) {
  const uint64_t cap = (uint64_t)sm_count() * per_sm;
  return (unsigned)(blocks < cap ? (blocks ? blocks : 1) : cap);
}

// Rows of one launch: the kernels count chunks of a launch in 32 bits.
uint64_t rows_per_launch(uint64_t chunks) { return chunks ? (uint64_t(1) << 30) / chunks : 1; }

int quantize_rows(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride, bool ceil, float* multiplier,
                  const uint32_t* partials, int count, const t5e_blocks& out, cudaStream_t stream) {
  const uint32_t groups = scale_groups(out);
  const uint64_t chunks = (uint64_t)groups * (out.scale_block / 4);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (rows == 1 || (stride * type_bytes(type)) % 16 == 0);
  const uint64_t per = rows_per_launch(chunks);
  for (uint64_t row0 = 0; row0 < rows; row0 += per) {
    const uint32_t n = (uint32_t)(rows - row0 < per ? rows - row0 : per);
    const unsigned grid = grid_of(((uint64_t)n * chunks + kThreads - 1) / kThreads, 8);
    const int rc = with_form(type, out, vec, [&](auto t, auto e8, auto blk, auto v) {
      return launched(launch_dependent(quantize_rows_kernel<decltype(t)::value, decltype(e8)::value, decltype(blk)::value,
                                                            decltype(v)::value>,
                                       grid, kThreads, 0, stream, x, n, row0, (uint32_t)cols, stride, ceil, multiplier,
                                       partials, count, static_cast<uint8_t*>(out.data), out.stride,
                                       static_cast<uint8_t*>(out.scales), groups),
                      "quantize_rows_kernel launch");
    });
    if (rc != T5E_OK) return rc;
  }
  return T5E_OK;
}

int quantize_cols(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride, bool ceil, float* multiplier,
                  const uint32_t* partials, int count, const t5e_blocks& out, cudaStream_t stream) {
  const int bytes = type_bytes(type);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & (2 * bytes - 1)) == 0 && (rows == 1 || stride % 2 == 0);
  const uint64_t tiles = (rows + kColTileR - 1) / kColTileR;
  dim3 grid((unsigned)((cols + kColTileC - 1) / kColTileC), (unsigned)(tiles < 65535 ? tiles : 65535));
  return with_form(type, out, vec, [&](auto t, auto e8, auto blk, auto v) {
    return launched(launch_dependent(quantize_cols_kernel<decltype(t)::value, decltype(e8)::value, decltype(blk)::value,
                                                          decltype(v)::value>,
                                     grid, kThreads, 0, stream, x, rows, cols, stride, ceil, multiplier, partials, count,
                                     static_cast<uint8_t*>(out.data), out.stride, static_cast<uint8_t*>(out.scales),
                                     scale_groups(out)),
                    "quantize_cols_kernel launch");
  });
}

bool matrix_ok(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride) {
  if (rows == 0 || cols == 0) return true;
  return x && (reinterpret_cast<uintptr_t>(x) & (type_bytes(type) - 1)) == 0 && (rows == 1 || stride >= (int64_t)cols);
}

int partial_maxima(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride, uint32_t* partials,
                   int32_t count, cudaStream_t stream) {
  if (rows == 0 || cols == 0) rows = cols = 0;
  if (rows > 1 && stride == (int64_t)cols) {
    cols *= rows;
    rows = 1;
  }
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (rows <= 1 || (stride * type_bytes(type)) % 16 == 0);
  auto go = [&](auto t, auto v) {
    return launched(launch_dependent(partials_kernel<decltype(t)::value, decltype(v)::value>, dim3((unsigned)count),
                                     kThreads, 0, stream, x, rows, cols, stride, partials),
                    "partials_kernel launch");
  };
  auto by_vec = [&](auto t) { return vec ? go(t, std::true_type{}) : go(t, std::false_type{}); };
  if (type == T5E_REAL_F32) return by_vec(std::integral_constant<int, T5E_REAL_F32>{});
  if (type == T5E_REAL_BF16) return by_vec(std::integral_constant<int, T5E_REAL_BF16>{});
  return by_vec(std::integral_constant<int, T5E_REAL_F16>{});
}

}  // namespace blocks

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  const bool cached = dev >= 0 && dev < 64;
  int sms = cached ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return 148;
  if (cached) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

uint32_t scale_groups(const t5e_blocks& b) {
  const uint64_t per = 4ull * (uint64_t)b.scale_block;
  return (uint32_t)(((uint64_t)b.k + per - 1) / per);
}

bool blocks_ok(const t5e_blocks* b) {
  if (!b || b->k < 1 || b->k > T5E_MAX_BLOCK_K || b->rows > T5E_MAX_BLOCK_ROWS) return false;
  const bool form = (b->scale_format == T5E_SCALE_UE4M3 && b->scale_block == 16) ||
                    (b->scale_format == T5E_SCALE_UE8M0 && (b->scale_block == 16 || b->scale_block == 32));
  if (!form || b->stride % 16 || b->stride < (b->k + 31) / 32 * 16) return false;
  if (b->rows == 0) return true;
  return b->data && b->scales && (reinterpret_cast<uintptr_t>(b->data) & 15u) == 0 &&
         (reinterpret_cast<uintptr_t>(b->scales) & 15u) == 0;
}

}  // namespace t5e

extern "C" {

int t5e_block_multiplier(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride, uint32_t* partials,
                         int32_t count, float* multiplier, void* stream) {
  using namespace t5e;
  using namespace t5e::blocks;
  if (!type_ok(type) || !partials || !multiplier || count < 1 || count > T5E_MAX_PARTIALS ||
      !matrix_ok(type, x, rows, cols, stride))
    return T5E_ERR_INVALID;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = partial_maxima(type, x, rows, cols, stride, partials, count, s);
  if (rc != T5E_OK) return rc;
  return launched(launch_dependent(multiplier_kernel, dim3(1), kThreads, 0, s, partials, count, multiplier),
                  "multiplier_kernel launch");
}

int t5e_quantize_blocks(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride, int32_t rounding,
                        float* multiplier, uint32_t* partials, int32_t count, const t5e_blocks* by_rows,
                        const t5e_blocks* by_cols, void* stream) {
  using namespace t5e;
  using namespace t5e::blocks;
  if (!type_ok(type) || (!by_rows && !by_cols)) return T5E_ERR_INVALID;
  if (partials && (!multiplier || count < 1 || count > T5E_MAX_PARTIALS)) return T5E_ERR_INVALID;
  if (by_rows && (!blocks_ok(by_rows) || by_rows->rows != rows || (uint64_t)by_rows->k != cols)) return T5E_ERR_INVALID;
  if (by_cols && (!blocks_ok(by_cols) || by_cols->rows != cols || (uint64_t)by_cols->k != rows)) return T5E_ERR_INVALID;
  if (by_rows && by_cols &&
      (by_rows->scale_format != by_cols->scale_format || by_rows->scale_block != by_cols->scale_block))
    return T5E_ERR_INVALID;
  const int32_t format = (by_rows ? by_rows : by_cols)->scale_format;
  if (format == T5E_SCALE_UE4M3 ? rounding != T5E_SCALE_ROUND_NEAREST
                                : rounding != T5E_SCALE_ROUND_FLOOR && rounding != T5E_SCALE_ROUND_CEIL)
    return T5E_ERR_INVALID;
  if (!matrix_ok(type, x, rows, cols, stride)) return T5E_ERR_INVALID;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool ceil = rounding == T5E_SCALE_ROUND_CEIL;
  if (rows == 0 || cols == 0)
    return partials ? t5e_block_multiplier(type, x, rows, cols, stride, partials, count, multiplier, stream) : T5E_OK;
  if (partials) {
    const int rc = partial_maxima(type, x, rows, cols, stride, partials, count, s);
    if (rc != T5E_OK) return rc;
  }
  if (by_rows) {
    const int rc = quantize_rows(type, x, rows, cols, stride, ceil, multiplier, partials, count, *by_rows, s);
    if (rc != T5E_OK) return rc;
  }
  if (by_cols) return quantize_cols(type, x, rows, cols, stride, ceil, multiplier, partials, count, *by_cols, s);
  return T5E_OK;
}

int t5e_dequantize_blocks(const t5e_blocks* b, const float* multiplier, int32_t type, void* out, int64_t out_stride,
                          void* stream) {
  using namespace t5e;
  using namespace t5e::blocks;
  if (!blocks_ok(b) || !type_ok(type)) return T5E_ERR_INVALID;
  if (b->rows == 0) return T5E_OK;
  if (!out || (reinterpret_cast<uintptr_t>(out) & (type_bytes(type) - 1)) || (b->rows > 1 && out_stride < b->k))
    return T5E_ERR_INVALID;
  const uint32_t groups = scale_groups(*b);
  const uint64_t chunks = ((uint64_t)b->k + 15) / 16;
  const bool vec = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 &&
                   (b->rows == 1 || (out_stride * type_bytes(type)) % 16 == 0);
  const uint64_t per = rows_per_launch(chunks);
  for (uint64_t row0 = 0; row0 < b->rows; row0 += per) {
    const uint32_t n = (uint32_t)(b->rows - row0 < per ? b->rows - row0 : per);
    const unsigned grid = grid_of(((uint64_t)n * chunks + kThreads - 1) / kThreads, 8);
    const int rc = with_form(type, *b, vec, [&](auto t, auto e8, auto blk, auto v) {
      return launched(launch_dependent(dequantize_kernel<decltype(t)::value, decltype(e8)::value, decltype(blk)::value,
                                                         decltype(v)::value>,
                                       dim3(grid), kThreads, 0, static_cast<cudaStream_t>(stream),
                                       static_cast<const uint8_t*>(b->data), b->stride,
                                       static_cast<const uint8_t*>(b->scales), groups, n, row0, (uint32_t)b->k,
                                       multiplier, out, out_stride),
                      "dequantize_kernel launch");
    });
    if (rc != T5E_OK) return rc;
  }
  return T5E_OK;
}

}  // extern "C"
