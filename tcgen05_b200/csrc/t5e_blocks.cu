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

// F32 bits of a 16-bit type's magnitude bits.
template <int TYPE>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t h) {
  if constexpr (TYPE == T5E_REAL_F32) return h;
  else if constexpr (TYPE == T5E_REAL_BF16) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

// The larger magnitude: of F32 bits as integers (a NaN sorts above infinity);
// of two 16-bit values at once with the instruction that takes magnitudes and
// keeps a NaN.  The sign bits of the latter mean nothing.
template <int TYPE>
__device__ __forceinline__ uint32_t join_max(uint32_t best, uint32_t word) {
  if constexpr (TYPE == T5E_REAL_F32) {
    return max(best, word & 0x7FFFFFFFu);
  } else {
    uint32_t r;
    if constexpr (TYPE == T5E_REAL_BF16)
      asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(best), "r"(word));
    else
      asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(best), "r"(word));
    return r;
  }
}

// F32 bits of the largest of the two halves (or of the one F32).
template <int TYPE>
__device__ __forceinline__ uint32_t final_max(uint32_t v) {
  if constexpr (TYPE == T5E_REAL_F32) return v;
  else return magnitude_bits<TYPE>(max(v & 0x7FFFu, (v >> 16) & 0x7FFFu));
}

template <int TYPE>
__device__ __forceinline__ uint32_t element_bits(const void* x, uint64_t i) {
  if constexpr (TYPE == T5E_REAL_F32) return static_cast<const uint32_t*>(x)[i] & 0x7FFFFFFFu;
  else return static_cast<const uint16_t*>(x)[i] & 0x7FFFu;
}

// One tensor of a launch: what to read, what to write.  Launches take two, and
// blocks of the grid from `first_block` on work on the second.  Without holes: 128
// bytes (at 144 a launch took 0.4 us more of the host).
struct Job {
  const void* x;
  uint64_t rows, cols;
  int64_t stride;
  float* multiplier;
  float* kept;         // NULL, or where the multiplier is stored as well
  uint32_t* partials;  // NULL: the multiplier is given
  int32_t count;
  uint32_t first_block;
  uint8_t* row_data;   // NULL: no blocks along the rows
  int64_t row_stride;
  uint8_t* row_scales;
  uint8_t* col_data;   // NULL: no blocks along the columns
  int64_t col_stride;
  uint8_t* col_scales;
  uint32_t row_groups, col_groups;
  bool vec;            // rows start on 16-byte boundaries
  bool wide;           // on 32-byte boundaries
  bool words;          // on 4-byte boundaries
};
static_assert(sizeof(Job) == 128, "no holes");
struct Jobs {
  Job job[2];
};

__device__ __forceinline__ const Job& job_of(const Jobs& jobs) {
  return jobs.job[blockIdx.x >= jobs.job[1].first_block ? 1 : 0];
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) partials_kernel(const __grid_constant__ Jobs jobs) {
  __shared__ uint32_t shared[kThreads / 32];
  const Job& J = job_of(jobs);
  let_next_grid_start();
  wait_for_previous_grid();
  constexpr int kPer = 16 / Real<TYPE>::kBytes;
  uint32_t best = 0u;
  // a contiguous tensor comes as one row, which all blocks share; otherwise
  // each block takes whole rows
  const bool one = J.rows == 1;
  const uint32_t block = blockIdx.x - J.first_block;
  const uint64_t first = one ? (uint64_t)block * kThreads + threadIdx.x : threadIdx.x;
  const uint64_t step = one ? (uint64_t)J.count * kThreads : kThreads;
  for (uint64_t r = one ? 0 : block; r < J.rows; r += one ? 1 : J.count) {
    const char* row = static_cast<const char*>(J.x) + (int64_t)r * J.stride * Real<TYPE>::kBytes;
    uint64_t done = 0;
    if (J.vec) {
      const uint64_t vecs = J.cols / kPer;
      const uint4* p = reinterpret_cast<const uint4*>(row);
      uint64_t i = first;
      for (; i + 3 * step < vecs; i += 4 * step) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load16(p + i + j * step);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          best = join_max<TYPE>(join_max<TYPE>(join_max<TYPE>(join_max<TYPE>(best, v[j].x), v[j].y), v[j].z), v[j].w);
      }
      for (; i < vecs; i += step) {
        const uint4 v = load16(p + i);
        best = join_max<TYPE>(join_max<TYPE>(join_max<TYPE>(join_max<TYPE>(best, v.x), v.y), v.z), v.w);
      }
      done = vecs * kPer;
    }
    for (uint64_t i = done + first; i < J.cols; i += step) best = join_max<TYPE>(best, element_bits<TYPE>(row, i));
  }
  const uint32_t m = block_max(final_max<TYPE>(best), shared);
  if (threadIdx.x == 0) J.partials[block] = m;
}

__global__ void __launch_bounds__(kThreads) multiplier_kernel(const uint32_t* partials, int count,
                                                              float* multiplier) {
  __shared__ uint32_t shared[kThreads / 32];
  let_next_grid_start();
  wait_for_previous_grid();
  uint32_t best = 0u;
  for (int i = threadIdx.x; i < count; i += kThreads) best = max(best, partials[i]);
  best = block_max(best, shared);
  if (threadIdx.x == 0) *multiplier = multiplier_of(best);
}

// The multiplier a quantising block works with: none, given, or taken from the
// partial maxima (every block joins them for itself, which saves a launch; the
// job's first block stores the result, and what is to be kept).
__device__ __forceinline__ float load_multiplier(const Job& J, uint32_t* shared) {
  const bool first = blockIdx.x == J.first_block && threadIdx.x == 0;
  float m;
  if (J.partials != nullptr) {
    uint32_t best = 0u;
    for (int i = threadIdx.x; i < J.count; i += kThreads) best = max(best, J.partials[i]);
    m = multiplier_of(block_max(best, shared));
    if (first) *J.multiplier = m;
  } else {
    m = J.multiplier != nullptr ? *J.multiplier : 1.f;
  }
  if (first && J.kept != nullptr) *J.kept = m;
  return m;
}

// n / d for n < 2^31: mul = floor(2^(31 + shift) / d) + 1 with 2^(shift-1) < d <=
// 2^shift (d > 1).
struct Divider {
  uint32_t d, mul, shift;
};
__device__ __forceinline__ uint32_t divided(uint32_t n, const Divider& v) {
  return v.d == 1u ? n : __umulhi(n, v.mul) >> (v.shift - 1);
}

// ---- blocks along the rows ---------------------------------------------------
//
// A thread takes 32 consecutive elements: two blocks of 16 or one of 32, so
// that no maximum needs an exchange, and what a chunk costs besides its
// elements (places, scales) is paid half as often as with 16 (11 thread
// instructions per element there, which bound the kernel: 8192 x 8192 BF16 to
// UE4M3 blocks 37 us).  Per row the chunks run up to a whole group of four
// scales: two (four) neighbouring lanes hold one group, and one of them stores
// its four scale bytes as a word.  The next elements are loaded before the
// present ones are worked on.  Where rows do not start on 16-byte boundaries
// (VEC false) a lane loads the aligned vectors around its elements and shifts
// them into place (2051 x 4101 F16: 26 us by elements).
constexpr int kChunk = 32;

template <int TYPE, bool VEC>
struct Chunk {
  static constexpr int kVecs = 2 * Real<TYPE>::kBytes + (VEC ? 0 : 1);
  uint32_t row, e0;  // e0 beyond k: nothing
  uint32_t shift;    // bytes between the first vector and the elements
  uint4 w[kVecs];
};

// N words that start `shift` bytes (0..15) into `in`.
template <int N, bool HALVES>
__device__ __forceinline__ void shift_words(const uint32_t* in, uint32_t shift, uint32_t* out) {
  uint32_t t[N + 2], u[N + 1];
#pragma unroll
  for (int i = 0; i < N + 2; ++i) t[i] = shift & 8u ? in[i + 2 < N + 4 ? i + 2 : i] : in[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) u[i] = shift & 4u ? t[i + 1] : t[i];
  const uint32_t select = HALVES && (shift & 2u) ? 0x5432u : 0x3210u;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = HALVES ? __byte_perm(u[i], u[i + 1], select) : u[i];
}

// Whether [p, p + bytes) lies within the tensor's first and last element.
template <int TYPE>
__device__ __forceinline__ bool within(const Job& J, const void* p, uint32_t bytes) {
  const char* first = static_cast<const char*>(J.x);
  const char* behind = first + ((int64_t)(J.rows - 1) * J.stride + (int64_t)J.cols) * Real<TYPE>::kBytes;
  return static_cast<const char*>(p) >= first && static_cast<const char*>(p) + bytes <= behind;
}

// Places of a thread's chunks, a launch's threads apart from one to the next.
struct Walk {
  uint32_t row, chunk;
  __device__ __forceinline__ void start(uint32_t item, const Divider& chunks) {
    row = divided(item, chunks);
    chunk = item - row * chunks.d;
  }
  __device__ __forceinline__ void advance(uint32_t rows_on, uint32_t chunks_on, uint32_t per_row) {
    row += rows_on;
    chunk += chunks_on;
    if (chunk >= per_row) {
      chunk -= per_row;
      ++row;
    }
  }
};

template <int TYPE, bool VEC>
__device__ __forceinline__ void load_chunk(const Job& J, uint64_t row0, const Walk& at, uint32_t rows,
                                           Chunk<TYPE, VEC>& c) {
  using T = typename Real<TYPE>::type;
  constexpr int kVecs = Chunk<TYPE, VEC>::kVecs, kPer = 16 / Real<TYPE>::kBytes;
  const uint32_t k = (uint32_t)J.cols;
  // after a pass for the largest value the last rows are the likeliest in L2
  c.row = J.partials != nullptr ? rows - 1u - at.row : at.row;
  c.e0 = at.row < rows ? at.chunk * kChunk : 0x7FFFFFFFu;
  c.shift = 0u;
  const T* src = static_cast<const T*>(J.x) + ((int64_t)(row0 + c.row) * J.stride + c.e0);
  if (c.e0 + kChunk <= k) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < kVecs; j += 2) load32(reinterpret_cast<const uint4*>(src) + j, J.wide, c.w[j], c.w[j + 1]);
      return;
    } else {
      const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15u;
      const uint4* first = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) - shift);
      if (within<TYPE>(J, first, kVecs * 16)) {
        c.shift = shift;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) c.w[j] = load16(first + j);
        return;
      }
    }
  }
  // the end of a row, the tensor's ends, or nothing: what exists, then zeros
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    uint32_t words[4] = {0u, 0u, 0u, 0u};
    if (c.e0 + j * kPer < k && j * kPer < kChunk) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (c.e0 + j * kPer + i < k) {
          if constexpr (TYPE == T5E_REAL_F32)
            words[i] = reinterpret_cast<const uint32_t*>(src)[j * kPer + i];
          else
            words[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[j * kPer + i] << (16 * (i & 1));
        }
      }
    }
    c.w[j] = make_uint4(words[0], words[1], words[2], words[3]);
  }
}

template <int TYPE, bool E8M0, int BLOCK, int HOW, bool VEC>
__device__ __forceinline__ void round_rows(const Job& J, uint32_t rows, uint64_t row0, const Divider& chunks, bool ceil,
                                           float m, const float* inverses) {
  constexpr int kWords = kChunk * Real<TYPE>::kBytes / 4, kBlocks = kChunk / BLOCK;
  const uint32_t k = (uint32_t)J.cols;
  const uint32_t total = rows * chunks.d, step = gridDim.x * kThreads;
  const uint32_t rows_on = divided(step, chunks), chunks_on = step - rows_on * chunks.d;
  const int lane = threadIdx.x & 31;
  uint8_t* scales = J.row_scales + scale_offset(row0, 0, J.row_groups);  // row0 is a multiple of 128
  uint32_t base = blockIdx.x * kThreads + (threadIdx.x & ~31u);
  Walk at;
  at.start(base + lane, chunks);
  Chunk<TYPE, VEC> c;
  if (base < total) load_chunk<TYPE, VEC>(J, row0, at, rows, c);
  for (; base < total; base += step) {
    const uint32_t row = c.row, e0 = c.e0;
    uint32_t words[kWords];
    {
      uint32_t raw[4 * Chunk<TYPE, VEC>::kVecs];
#pragma unroll
      for (int j = 0; j < Chunk<TYPE, VEC>::kVecs; ++j) {
        raw[4 * j] = c.w[j].x;
        raw[4 * j + 1] = c.w[j].y;
        raw[4 * j + 2] = c.w[j].z;
        raw[4 * j + 3] = c.w[j].w;
      }
      if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) words[j] = raw[j];
      } else {
        shift_words<kWords, TYPE != T5E_REAL_F32>(raw, c.shift, words);
      }
    }
    at.advance(rows_on, chunks_on, chunks.d);
    if (base + step < total) load_chunk<TYPE, VEC>(J, row0, at, rows, c);
    uint32_t out[4], bytes = 0u;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      constexpr int kIn = kWords / kBlocks;
      const uint32_t* mine = words + b * kIn;
      uint32_t top = 0u;
#pragma unroll
      for (int j = 0; j < kIn; ++j) top = join_max<TYPE>(top, mine[j]);
      float step_value, inv;
      uint32_t word = block_scale<E8M0, HOW>(__uint_as_float(final_max<TYPE>(top)), m, ceil, inverses, step_value, inv);
      const bool finite = word != (E8M0 ? 0xFFu : 0x7Fu);
      if (e0 + b * BLOCK >= k) word = 0u;  // a scale behind the last block
      bytes |= word << (8 * b);
#pragma unroll
      for (int h = 0; h < BLOCK / 8; ++h) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8 * Real<TYPE>::kBytes / 4; ++j) {
          const uint32_t w = mine[h * 8 * Real<TYPE>::kBytes / 4 + j];
          if constexpr (TYPE == T5E_REAL_F32) v[j] = __uint_as_float(w);
          else unpack2<TYPE>(w, v[2 * j], v[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = divide<E8M0, HOW>(v[j], m, step_value, inv);
        out[b * (BLOCK / 8) + h] = finite ? e2m1x8(v) : 0u;
      }
    }
    if (e0 < k) {  // chunks are the rows' groups of 32 codes
      *reinterpret_cast<uint4*>(J.row_data + (int64_t)(row0 + row) * J.row_stride + e0 / 2u) =
          make_uint4(out[0], out[1], out[2], out[3]);
    }
    // four scale bytes to one word
    if constexpr (BLOCK == 16) {
      bytes <<= 16 * (lane & 1);
      bytes |= __shfl_xor_sync(0xFFFFFFFFu, bytes, 1);
    } else {
      bytes <<= 8 * (lane & 3);
      bytes |= __shfl_xor_sync(0xFFFFFFFFu, bytes, 1);
      bytes |= __shfl_xor_sync(0xFFFFFFFFu, bytes, 2);
    }
    if (lane % (BLOCK / 8) == 0 && row < rows)
      *reinterpret_cast<uint32_t*>(scales + ((row >> 7) * J.row_groups + e0 / (4 * BLOCK)) * 512u + (row & 31u) * 16u +
                                   ((row >> 5) & 3u) * 4u) = bytes;
  }
}

template <int TYPE, bool E8M0, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ Jobs jobs, uint32_t rows,
                                                                 uint64_t row0, Divider chunks, bool ceil) {
  __shared__ uint32_t shared[kThreads / 32];
  __shared__ float inverses[128];
  const Job& J = jobs.job[0];
  let_next_grid_start();
  wait_for_previous_grid();
  const float m = load_multiplier(J, shared);
  if (is_narrow<TYPE, E8M0>(m)) {
    if constexpr (!E8M0) {
      fill_inverses(inverses, m);
      __syncthreads();
    }
    round_rows<TYPE, E8M0, BLOCK, kNarrow, VEC>(J, rows, row0, chunks, ceil, m, inverses);
  } else {
    round_rows<TYPE, E8M0, BLOCK, kExact, VEC>(J, rows, row0, chunks, ceil, m, inverses);
  }
}

// ---- blocks along the columns, or along both axes in one read -----------------------
//
// A block of 256 threads takes a tile of 128 x 128 elements into shared memory.
// Along the rows a thread rounds 16 neighbouring elements, four times; along
// the columns it rounds two neighbouring columns of 32 rows (two 16-element
// blocks or one of 32), so that neither maximum needs an exchange beyond a
// neighbour lane.  Codes and scale bytes of the columns are put in order in
// shared memory: each output row gets 64 consecutive bytes, and the scale
// tiles of 128 rows leave whole.
constexpr int kTile = 128, kColPitch = kTile / 2 + 16;

template <int TYPE>
struct TileBytes {
  static constexpr int kPitch = kTile * Real<TYPE>::kBytes + 16;
  static constexpr int kInput = kTile * kPitch;
  static constexpr int kCodes = kTile * kColPitch;
  static constexpr int kSteps = kTile * (kTile / 16);  // scale bytes of one axis, in the tiles' order
  static constexpr int kAll = kInput + kCodes + 2 * kSteps;
};

// Where scale b (of 8 or 4 per row of the tile) of row r belongs in the tile's
// own scale tiles.
__device__ __forceinline__ int step_at(int r, int b) { return (b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3); }

template <int TYPE, bool E8M0, int BLOCK, int HOW>
__device__ __forceinline__ void round_tile(const Job& J, uint8_t* smem, uint64_t r0, uint64_t c0, bool ceil, float m,
                                           const float* inverses) {
  using B = TileBytes<TYPE>;
  uint8_t* input = smem;
  uint8_t* codes = smem + B::kInput;
  uint8_t* row_steps = codes + B::kCodes;
  uint8_t* col_steps = row_steps + B::kSteps;
  constexpr int kNan = E8M0 ? 0xFF : 0x7F;
  const int t = threadIdx.x;
  if (J.row_data != nullptr) {
    const uint64_t padded = (J.cols + 31) / 32 * 32;
#pragma unroll
    for (int i = 0; i < kTile * (kTile / 16) / kThreads; ++i) {
      const int item = i * kThreads + t, r = item >> 3, chunk = item & 7;
      const uint4* src = reinterpret_cast<const uint4*>(input + r * B::kPitch + chunk * 16 * Real<TYPE>::kBytes);
      uint32_t words[4 * Real<TYPE>::kBytes];
#pragma unroll
      for (int j = 0; j < Real<TYPE>::kBytes; ++j) reinterpret_cast<uint4*>(words)[j] = src[j];
      float v[16];
      uint32_t top = 0u;
#pragma unroll
      for (int j = 0; j < 4 * Real<TYPE>::kBytes; ++j) {
        top = join_max<TYPE>(top, words[j]);
        if constexpr (TYPE == T5E_REAL_F32) v[j] = __uint_as_float(words[j]);
        else unpack2<TYPE>(words[j], v[2 * j], v[2 * j + 1]);
      }
      top = final_max<TYPE>(top);
      if constexpr (BLOCK == 32) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      float step, inv;
      uint32_t word = block_scale<E8M0, HOW>(__uint_as_float(top), m, ceil, inverses, step, inv);
      const bool finite = word != (uint32_t)kNan;
      if (c0 + chunk * 16 / BLOCK * BLOCK >= J.cols) word = 0u;
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = divide<E8M0, HOW>(v[j], m, step, inv);
      const uint2 out = finite ? make_uint2(e2m1x8(v), e2m1x8(v + 8)) : make_uint2(0u, 0u);
      if (r0 + r < J.rows && c0 + chunk * 16 < padded)
        *reinterpret_cast<uint2*>(J.row_data + (int64_t)(r0 + r) * J.row_stride + (int64_t)(c0 / 2) + chunk * 8) = out;
      if (BLOCK == 16 || (chunk & 1) == 0) row_steps[step_at(r, chunk * 16 / BLOCK)] = (uint8_t)word;
    }
  }
  if (J.col_data != nullptr) {
    const int pair = t & 63, part = t >> 6;  // columns 2 pair, 2 pair + 1; rows 32 part ..
    float v[2][32];
    uint32_t top[2][32 / BLOCK];
#pragma unroll
    for (int b = 0; b < 32 / BLOCK; ++b) top[0][b] = top[1][b] = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint8_t* src = input + (part * 32 + i) * B::kPitch + pair * 2 * Real<TYPE>::kBytes;
      if constexpr (TYPE == T5E_REAL_F32) {
        const float2 f = *reinterpret_cast<const float2*>(src);
        v[0][i] = f.x;
        v[1][i] = f.y;
        top[0][i / BLOCK] = max(top[0][i / BLOCK], __float_as_uint(f.x) & 0x7FFFFFFFu);
        top[1][i / BLOCK] = max(top[1][i / BLOCK], __float_as_uint(f.y) & 0x7FFFFFFFu);
      } else {  // both columns' maxima in one word
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src);
        top[0][i / BLOCK] = join_max<TYPE>(top[0][i / BLOCK], w);
        unpack2<TYPE>(w, v[0][i], v[1][i]);
      }
    }
#pragma unroll
    for (int b = 0; b < 32 / BLOCK; ++b) {
      if constexpr (TYPE != T5E_REAL_F32) {
        const uint32_t both = top[0][b];
        top[0][b] = magnitude_bits<TYPE>(both & 0x7FFFu);
        top[1][b] = magnitude_bits<TYPE>((both >> 16) & 0x7FFFu);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t out[4];
#pragma unroll
      for (int b = 0; b < 32 / BLOCK; ++b) {
        float step, inv;
        uint32_t word = block_scale<E8M0, HOW>(__uint_as_float(top[h][b]), m, ceil, inverses, step, inv);
        const bool finite = word != (uint32_t)kNan;
        if (r0 + part * 32 + b * BLOCK >= J.rows) word = 0u;
#pragma unroll
        for (int i = 0; i < BLOCK; ++i) v[h][b * BLOCK + i] = divide<E8M0, HOW>(v[h][b * BLOCK + i], m, step, inv);
#pragma unroll
        for (int i = 0; i < BLOCK / 8; ++i)
          out[b * (BLOCK / 8) + i] = finite ? e2m1x8(&v[h][b * BLOCK + 8 * i]) : 0u;
        col_steps[step_at(pair * 2 + h, part * (32 / BLOCK) + b)] = (uint8_t)word;
      }
      *reinterpret_cast<uint4*>(codes + (pair * 2 + h) * kColPitch + part * 16) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  __syncthreads();
  constexpr int kGroups = kTile / (4 * BLOCK);  // scale tiles of the tile per axis
  if (J.row_data != nullptr && t < kGroups * 32) {
    // a line of 16 bytes: rows r, r + 32, r + 64, r + 96 of the tile; lines of
    // rows that do not exist belong to the padding of the last scale tile
    const uint32_t group = (uint32_t)(c0 / (4 * BLOCK)) + t / 32;
    if (group < J.row_groups)
      *reinterpret_cast<uint4*>(J.row_scales + ((r0 >> 7) * J.row_groups + group) * 512u + (t & 31) * 16) =
          *reinterpret_cast<const uint4*>(row_steps + t * 16);
  }
  if (J.col_data != nullptr) {
    const uint64_t padded = (J.rows + 31) / 32 * 32;
#pragma unroll
    for (int i = 0; i < kTile * 4 / kThreads; ++i) {
      const int item = i * kThreads + t, col = item >> 2, part = item & 3;
      if (c0 + col < J.cols && r0 + part * 32 < padded)
        *reinterpret_cast<uint4*>(J.col_data + (int64_t)(c0 + col) * J.col_stride + (int64_t)(r0 / 2) + part * 16) =
            *reinterpret_cast<const uint4*>(codes + col * kColPitch + part * 16);
    }
    if (t >= kThreads - kGroups * 32) {
      const int i = t - (kThreads - kGroups * 32);
      const uint32_t group = (uint32_t)(r0 / (4 * BLOCK)) + i / 32;
      if (group < J.col_groups)
        *reinterpret_cast<uint4*>(J.col_scales + ((c0 >> 7) * J.col_groups + group) * 512u + (i & 31) * 16) =
            *reinterpret_cast<const uint4*>(col_steps + i * 16);
    }
  }
}

template <int TYPE, bool E8M0, int BLOCK>
__global__ void __launch_bounds__(kThreads, TYPE == T5E_REAL_BF16 ? 4 : TYPE == T5E_REAL_F16 ? 3 : 2) quantize_tiles_kernel(const __grid_constant__ Jobs jobs, bool ceil) {
  using B = TileBytes<TYPE>;
  using T = typename Real<TYPE>::type;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t shared[kThreads / 32];
  __shared__ float inverses[128];
  const Job& J = job_of(jobs);
  let_next_grid_start();
  wait_for_previous_grid();
  const uint64_t across = (J.cols + kTile - 1) / kTile;
  uint64_t tile = blockIdx.x - J.first_block;
  // after a pass for the largest value the last rows are the likeliest in L2
  if (J.partials != nullptr) tile = across * ((J.rows + kTile - 1) / kTile) - 1 - tile;
  const uint64_t r0 = tile / across * kTile, c0 = tile % across * kTile;
  const T* src = static_cast<const T*>(J.x) + (int64_t)r0 * J.stride + (int64_t)c0;
  const bool whole = r0 + kTile <= J.rows && c0 + kTile <= J.cols;
  if (J.vec && whole) {
    constexpr int kPer = 16 / Real<TYPE>::kBytes, kVecs = kTile / kPer, kRows = kThreads / kVecs;
    const int r = threadIdx.x / kVecs, v = threadIdx.x % kVecs;
    const T* from = src + (int64_t)r * J.stride + v * kPer;
    uint32_t to = (uint32_t)__cvta_generic_to_shared(smem + r * B::kPitch + v * 16);
#pragma unroll
    for (int i = 0; i < kTile / kRows; ++i, from += kRows * J.stride, to += kRows * B::kPitch)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(from) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else if (J.vec) {
    constexpr int kPer = 16 / Real<TYPE>::kBytes, kVecs = kTile / kPer;  // elements of a vector, vectors of a row
#pragma unroll 2
    for (int i = 0; i < kTile * kVecs / kThreads; ++i) {
      const int item = i * kThreads + threadIdx.x, r = item / kVecs, v = item % kVecs;
      // bytes of the vector that exist; the others become zeros
      const int64_t have = r0 + r < J.rows ? (int64_t)(J.cols - c0) - v * kPer : 0;
      const uint32_t bytes = have >= kPer ? 16u : (have > 0 ? (uint32_t)have * Real<TYPE>::kBytes : 0u);
      const T* from = bytes ? src + (int64_t)r * J.stride + v * kPer : static_cast<const T*>(J.x);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                   :: "r"((uint32_t)__cvta_generic_to_shared(smem + r * B::kPitch + v * 16)), "l"(from), "r"(bytes) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else if (J.words) {  // rows on 4-byte boundaries: words, all in flight at once
    constexpr int kPer = 4 / Real<TYPE>::kBytes, kWords = kTile / kPer;
#pragma unroll 4
    for (int i = 0; i < kTile * kWords / kThreads; ++i) {
      const int item = i * kThreads + threadIdx.x, r = item / kWords, v = item % kWords;
      const int64_t have = r0 + r < J.rows ? (int64_t)(J.cols - c0) - v * kPer : 0;
      const uint32_t bytes = have >= kPer ? 4u : (have > 0 ? (uint32_t)have * Real<TYPE>::kBytes : 0u);
      const T* from = bytes ? src + (int64_t)r * J.stride + v * kPer : static_cast<const T*>(J.x);
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                   :: "r"((uint32_t)__cvta_generic_to_shared(smem + r * B::kPitch + v * 4)), "l"(from), "r"(bytes) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else if (TYPE != T5E_REAL_F32 && whole && r0 + c0 > 0 && (r0 + kTile < J.rows || c0 + kTile + 8 <= J.cols)) {
    // the aligned vectors around the tile's rows, which lie within the tensor:
    // shifted into place, a lane taking the one behind its own from its
    // neighbour (1501 x 1999 F16: 15.5 us by elements)
    constexpr int kVecs = kTile / 8, kRows = kThreads / kVecs, kBatch = 4;
    const int v = threadIdx.x % kVecs;
    const char* row = reinterpret_cast<const char*>(src + (int64_t)(threadIdx.x / kVecs) * J.stride);
    uint8_t* to = smem + threadIdx.x / kVecs * B::kPitch + v * 16;
#pragma unroll 1
    for (int i = 0; i < kTile / kRows; i += kBatch) {
      uint4 a[kBatch], b[kBatch];
      uint32_t shift[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j, row += (int64_t)kRows * J.stride * Real<TYPE>::kBytes) {
        shift[j] = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
        const uint4* p = reinterpret_cast<const uint4*>(row - shift[j]) + v;
        a[j] = load16(p);
        b[j] = make_uint4(0u, 0u, 0u, 0u);
        if (v == kVecs - 1) b[j] = load16(p + 1);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j, to += kRows * B::kPitch) {
        uint4 n;
        n.x = __shfl_down_sync(0xFFFFFFFFu, a[j].x, 1);
        n.y = __shfl_down_sync(0xFFFFFFFFu, a[j].y, 1);
        n.z = __shfl_down_sync(0xFFFFFFFFu, a[j].z, 1);
        n.w = __shfl_down_sync(0xFFFFFFFFu, a[j].w, 1);
        if (v == kVecs - 1) n = b[j];
        const uint32_t in[8] = {a[j].x, a[j].y, a[j].z, a[j].w, n.x, n.y, n.z, n.w};
        uint32_t out[4];
        shift_words<4, true>(in, shift[j], out);
        *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
  } else {
#pragma unroll 16
    for (int i = 0; i < kTile * kTile / kThreads; ++i) {
      const int item = i * kThreads + threadIdx.x, r = item / kTile, c = item % kTile;
      reinterpret_cast<T*>(smem + r * B::kPitch)[c] =
          r0 + r < J.rows && c0 + c < J.cols ? src[(int64_t)r * J.stride + c] : from_f32<TYPE>(0.f);
    }
  }
  const float m = load_multiplier(J, shared);
  if constexpr (!E8M0) fill_inverses(inverses, m);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (is_narrow<TYPE, E8M0>(m)) round_tile<TYPE, E8M0, BLOCK, kNarrow>(J, smem, r0, c0, ceil, m, inverses);
  else round_tile<TYPE, E8M0, BLOCK, kExact>(J, smem, r0, c0, ceil, m, inverses);
}

// ---- back to real values -------------------------------------------------------

// A thread takes 32 codes of two places of the launch at a time, all loaded
// before the first is worked on.  Rows of `out` on 16-byte boundaries take
// vectors; others pass through shared memory, so that the lanes' stores are
// neighbours.  FOLD: 1 / m is a power of two near 1, so its product with the
// scale is exact and one product per element is enough.
template <int TYPE, bool E8M0, int BLOCK, bool VEC, bool FOLD>
__device__ __forceinline__ void open_rows(const uint8_t* data, int64_t data_stride,
                                          const uint8_t* scales, uint32_t groups, uint32_t rows, uint64_t row0,
                                          uint32_t k, const Divider& chunks, float back, void* out,
                                          int64_t out_stride, bool wide, float* turn) {
  constexpr int kAtOnce = 2, kBlocks = kChunk / BLOCK;
  const uint32_t total = rows * chunks.d, step = gridDim.x * kThreads;
  const uint32_t rows_on = divided(step, chunks), chunks_on = step - rows_on * chunks.d;
  const int lane = threadIdx.x & 31;
  using T = typename Real<TYPE>::type;
  scales += scale_offset(row0, 0, groups);  // row0 is a multiple of 128
  uint32_t base = blockIdx.x * kThreads + (threadIdx.x & ~31u);
  Walk walk;
  walk.start(base + lane, chunks);
  for (; base < total; base += kAtOnce * step) {
    uint32_t row[kAtOnce], e0[kAtOnce], bytes[kAtOnce];
    uint4 w[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const bool in = walk.row < rows;
      row[i] = walk.row;
      e0[i] = in ? walk.chunk * kChunk : 0x7FFFFFFFu;  // nothing to store
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      bytes[i] = 0u;
      if (in) {
        w[i] = load16(data + (int64_t)(row0 + row[i]) * data_stride + e0[i] / 2u);
        const uint32_t b = e0[i] / BLOCK;
        const uint8_t* at = scales + ((row[i] >> 7) * groups + (b >> 2)) * 512u + (row[i] & 31u) * 16u +
                            ((row[i] >> 5) & 3u) * 4u + (b & 3u);
        if constexpr (BLOCK == 16) bytes[i] = *reinterpret_cast<const uint16_t*>(at);
        else bytes[i] = *at;
      }
      walk.advance(rows_on, chunks_on, chunks.d);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (base + i * step >= total) break;
      float v[32];
      from_e2m1x8(w[i].x, v);
      from_e2m1x8(w[i].y, v + 8);
      from_e2m1x8(w[i].z, v + 16);
      from_e2m1x8(w[i].w, v + 24);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const float s = scale_value<E8M0>((bytes[i] >> (8 * b)) & 0xFFu);
        if constexpr (FOLD) {
          const float f = s * back;
#pragma unroll
          for (int j = 0; j < BLOCK; ++j) v[b * BLOCK + j] *= f;
        } else if constexpr (E8M0) {
          // a code times a scale of 2^126 or more may be beyond F32 where the
          // value is not: what the scale has above 2^64 comes last (a product
          // up to there is at least 2^-65 in front of it, so nothing is lost)
          const bool far = s > 0x1p64f;
          const float f = far ? 0x1p64f : s, rest = far ? s * 0x1p-64f : 1.f;
#pragma unroll
          for (int j = 0; j < BLOCK; ++j) v[b * BLOCK + j] = v[b * BLOCK + j] * f * back * rest;
        } else {
#pragma unroll
          for (int j = 0; j < BLOCK; ++j) v[b * BLOCK + j] = v[b * BLOCK + j] * s * back;
        }
      }
      const int64_t at = (int64_t)(row0 + row[i]) * out_stride + e0[i];
      if constexpr (VEC) {
        T* dst = static_cast<T*>(out) + at;
        if (e0[i] + kChunk <= k) {
          uint4 o[2 * Real<TYPE>::kBytes];
          uint32_t* words = reinterpret_cast<uint32_t*>(o);
#pragma unroll
          for (int j = 0; j < 8 * Real<TYPE>::kBytes; ++j) {
            if constexpr (TYPE == T5E_REAL_F32) words[j] = __float_as_uint(v[j]);
            else words[j] = pack2<TYPE>(v[2 * j], v[2 * j + 1]);
          }
#pragma unroll
          for (int j = 0; j < 2 * Real<TYPE>::kBytes; j += 2)
            store32(reinterpret_cast<uint4*>(dst) + j, wide, o[j], o[j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            if (e0[i] + j < k) dst[j] = from_f32<TYPE>(v[j]);
        }
      } else {
        constexpr int kPitch = 36;  // floats of a lane: vectors of a warp meet no bank twice
        float* mine = turn + threadIdx.x * kPitch;
        const float* warp = turn + (threadIdx.x & ~31) * kPitch;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          reinterpret_cast<float4*>(mine)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {  // lane j's 32 elements
          const int64_t place = __shfl_sync(0xFFFFFFFFu, at, j) + lane;
          if (__shfl_sync(0xFFFFFFFFu, e0[i], j) + lane < k) static_cast<T*>(out)[place] = from_f32<TYPE>(warp[j * kPitch + lane]);
        }
      }
    }
  }
}

template <int TYPE, bool E8M0, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* data, int64_t data_stride,
                                                              const uint8_t* scales, uint32_t groups,
                                                              uint32_t rows, uint64_t row0, uint32_t k, Divider chunks,
                                                              const float* multiplier, void* out,
                                                              int64_t out_stride, bool wide) {
  __shared__ __align__(16) float turn[VEC ? 4 : kThreads * 36];
  let_next_grid_start();
  wait_for_previous_grid();
  const float back = multiplier != nullptr ? 1.f / *multiplier : 1.f;
  if (is_narrow<T5E_REAL_BF16, E8M0>(back))
    open_rows<TYPE, E8M0, BLOCK, VEC, true>(data, data_stride, scales, groups, rows, row0, k, chunks, back, out, out_stride,
                                            wide, turn);
  else
    open_rows<TYPE, E8M0, BLOCK, VEC, false>(data, data_stride, scales, groups, rows, row0, k, chunks, back, out,
                                             out_stride, wide, turn);
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

// Calls f with compile-time (type, UE8M0, block) for a run-time choice.
template <typename F>
int with_form(int32_t type, int32_t scale_format, int32_t scale_block, F f) {
  auto by_scale = [&](auto t) {
    if (scale_format == T5E_SCALE_UE4M3) return f(t, std::false_type{}, std::integral_constant<int, 16>{});
    if (scale_block == 16) return f(t, std::true_type{}, std::integral_constant<int, 16>{});
    return f(t, std::true_type{}, std::integral_constant<int, 32>{});
  };
  if (type == T5E_REAL_F32) return by_scale(std::integral_constant<int, T5E_REAL_F32>{});
  if (type == T5E_REAL_BF16) return by_scale(std::integral_constant<int, T5E_REAL_BF16>{});
  return by_scale(std::integral_constant<int, T5E_REAL_F16>{});
}

unsigned grid_of(uint64_t blocks, unsigned per_sm) {
  const uint64_t cap = (uint64_t)sm_count() * per_sm;
  return (unsigned)(blocks < cap ? (blocks ? blocks : 1) : cap);
}

// Rows of one launch: the kernels count chunks and scale bytes of a launch in 32
// bits.  T5E_MAX_BLOCK_K leaves at least 128 rows.
uint64_t rows_per_launch(uint64_t chunks) { return (uint64_t(1) << 30) / chunks; }

bool rows_aligned(int32_t type, const void* x, uint64_t rows, int64_t stride, unsigned bytes = 16) {
  return reinterpret_cast<uintptr_t>(x) % bytes == 0 && (rows <= 1 || (stride * type_bytes(type)) % bytes == 0);
}

Divider divider(uint32_t d) {
  uint32_t shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {d, d == 1u ? 0u : (uint32_t)((1ull << (31 + shift)) / d + 1), shift};
}

constexpr uint32_t kNever = 0xFFFFFFFFu;

int quantize_rows(int32_t type, const Jobs& jobs, const t5e_blocks& out, bool ceil, cudaStream_t stream) {
  const Job& J = jobs.job[0];
  const Divider chunks = divider(J.row_groups * (uint32_t)(out.scale_block / 8));
  const uint64_t per = rows_per_launch(chunks.d) / 128 * 128;
  for (uint64_t row0 = 0; row0 < J.rows; row0 += per) {
    const uint32_t n = (uint32_t)(J.rows - row0 < per ? J.rows - row0 : per);
    const unsigned grid = grid_of(((uint64_t)n * chunks.d + kThreads - 1) / kThreads, 6);
    const int rc = with_form(type, out.scale_format, out.scale_block, [&](auto t, auto e8, auto blk) {
      auto go = [&](auto v) {
        return launched(launch_dependent(quantize_rows_kernel<decltype(t)::value, decltype(e8)::value,
                                                              decltype(blk)::value, decltype(v)::value>,
                                         dim3(grid), kThreads, 0, stream, jobs, n, row0, chunks, ceil),
                        "quantize_rows_kernel launch");
      };
      return J.vec ? go(std::true_type{}) : go(std::false_type{});
    });
    if (rc != T5E_OK) return rc;
  }
  return T5E_OK;
}

int quantize_tiles(int32_t type, Jobs& jobs, int n, int32_t scale_format, int32_t scale_block, bool ceil,
                   cudaStream_t stream) {
  uint64_t blocks = 0;
  for (int i = 0; i < 2; ++i) {
    jobs.job[i].first_block = i < n ? (uint32_t)blocks : kNever;
    if (i < n)
      blocks += ((jobs.job[i].rows + kTile - 1) / kTile) * ((jobs.job[i].cols + kTile - 1) / kTile);
    if (blocks > 0x7FFFFFFFull) return T5E_ERR_INVALID;
  }
  return with_form(type, scale_format, scale_block, [&](auto t, auto e8, auto blk) {
    constexpr auto kernel = quantize_tiles_kernel<decltype(t)::value, decltype(e8)::value, decltype(blk)::value>;
    constexpr int smem = TileBytes<decltype(t)::value>::kAll;
    const int rc = raise_smem_limit<kernel>(smem, "quantize_tiles_kernel attribute");
    if (rc != T5E_OK) return rc;
    return launched(launch_dependent(kernel, dim3((unsigned)blocks), kThreads, smem, stream, jobs, ceil),
                    "quantize_tiles_kernel launch");
  });
}

bool matrix_ok(int32_t type, const void* x, uint64_t rows, uint64_t cols, int64_t stride) {
  if (rows == 0 || cols == 0) return true;
  return x && (reinterpret_cast<uintptr_t>(x) & (type_bytes(type) - 1)) == 0 && (rows == 1 || stride >= (int64_t)cols);
}

// The partial maxima of the jobs that want them.
int partial_maxima(int32_t type, const Jobs& jobs, int n, cudaStream_t stream) {
  Jobs work = {};
  int wanted = 0;
  uint32_t blocks = 0;
  for (int i = 0; i < n; ++i) {
    if (jobs.job[i].partials == nullptr) continue;
    Job& J = work.job[wanted++];
    J = jobs.job[i];
    J.first_block = blocks;
    blocks += (uint32_t)J.count;
    if (J.rows == 0 || J.cols == 0) J.rows = J.cols = 0;
    if (J.rows > 1 && J.stride == (int64_t)J.cols) {
      J.cols *= J.rows;
      J.rows = 1;
    }
    J.vec = rows_aligned(type, J.x, J.rows, J.stride);
  }
  if (wanted == 0) return T5E_OK;
  if (wanted == 1) work.job[1].first_block = kNever;
  auto go = [&](auto t) {
    return launched(launch_dependent(partials_kernel<decltype(t)::value>, dim3(blocks), kThreads, 0, stream, work),
                    "partials_kernel launch");
  };
  if (type == T5E_REAL_F32) return go(std::integral_constant<int, T5E_REAL_F32>{});
  if (type == T5E_REAL_BF16) return go(std::integral_constant<int, T5E_REAL_BF16>{});
  return go(std::integral_constant<int, T5E_REAL_F16>{});
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
  Jobs jobs = {};
  Job& J = jobs.job[0];
  J.x = x;
  J.rows = rows;
  J.cols = cols;
  J.stride = stride;
  J.partials = partials;
  J.count = count;
  J.vec = rows_aligned(type, x, rows, stride);
  const int rc = partial_maxima(type, jobs, 1, s);
  if (rc != T5E_OK) return rc;
  return launched(launch_dependent(multiplier_kernel, dim3(1), kThreads, 0, s, partials, count, multiplier),
                  "multiplier_kernel launch");
}

int t5e_quantize_blocks(const t5e_quantize* q, int32_t n, void* stream) {
  using namespace t5e;
  using namespace t5e::blocks;
  if (!q || n < 1 || n > 2) return T5E_ERR_INVALID;
  Jobs jobs = {};
  const t5e_blocks* form = nullptr;
  bool cols = false, empty = true;
  for (int i = 0; i < n; ++i) {
    const t5e_quantize& Q = q[i];
    const bool by_rows = Q.by_rows.data != nullptr, by_cols = Q.by_cols.data != nullptr;
    if (!type_ok(Q.type) || Q.type != q[0].type || Q.rounding != q[0].rounding || Q.reserved != 0) return T5E_ERR_INVALID;
    if (Q.partials && (!Q.multiplier || Q.count < 1 || Q.count > T5E_MAX_PARTIALS)) return T5E_ERR_INVALID;
    if (!matrix_ok(Q.type, Q.x, Q.rows, Q.cols, Q.stride)) return T5E_ERR_INVALID;
    if (!by_rows && !by_cols) {
      if (Q.rows && Q.cols) return T5E_ERR_INVALID;
      continue;  // no element: nothing to write
    }
    for (const t5e_blocks* b : {by_rows ? &Q.by_rows : nullptr, by_cols ? &Q.by_cols : nullptr}) {
      if (!b) continue;
      if (!form) form = b;
      const bool mine = b == &Q.by_rows;
      if (!blocks_ok(b) || b->rows != (mine ? Q.rows : Q.cols) || (uint64_t)b->k != (mine ? Q.cols : Q.rows) ||
          b->scale_format != form->scale_format || b->scale_block != form->scale_block)
        return T5E_ERR_INVALID;
    }
    if (Q.rows == 0 || Q.cols == 0) continue;
    empty = false;
    cols |= by_cols;
    Job& J = jobs.job[i];
    J.x = Q.x;
    J.rows = Q.rows;
    J.cols = Q.cols;
    J.stride = Q.stride;
    J.multiplier = Q.multiplier;
    J.kept = Q.kept;
    J.partials = Q.partials;
    J.count = Q.count;
    J.vec = rows_aligned(Q.type, Q.x, Q.rows, Q.stride);
    J.wide = rows_aligned(Q.type, Q.x, Q.rows, Q.stride, 32);
    J.words = rows_aligned(Q.type, Q.x, Q.rows, Q.stride, 4);
    if (by_rows) {
      J.row_data = static_cast<uint8_t*>(Q.by_rows.data);
      J.row_stride = Q.by_rows.stride;
      J.row_scales = static_cast<uint8_t*>(Q.by_rows.scales);
      J.row_groups = scale_groups(Q.by_rows);
    }
    if (by_cols) {
      J.col_data = static_cast<uint8_t*>(Q.by_cols.data);
      J.col_stride = Q.by_cols.stride;
      J.col_scales = static_cast<uint8_t*>(Q.by_cols.scales);
      J.col_groups = scale_groups(Q.by_cols);
    }
  }
  if (form) {
    const bool nearest = q[0].rounding == T5E_SCALE_ROUND_NEAREST;
    const bool power = q[0].rounding == T5E_SCALE_ROUND_FLOOR || q[0].rounding == T5E_SCALE_ROUND_CEIL;
    if (form->scale_format == T5E_SCALE_UE4M3 ? !nearest : !power) return T5E_ERR_INVALID;
  }
  if (empty) return T5E_OK;
  if (n == 2 && (jobs.job[0].x == nullptr || jobs.job[1].x == nullptr)) {  // one of the two is empty
    if (jobs.job[0].x == nullptr) jobs.job[0] = jobs.job[1];
    n = 1;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool ceil = q[0].rounding == T5E_SCALE_ROUND_CEIL;
  int rc = partial_maxima(q[0].type, jobs, n, s);
  if (rc != T5E_OK) return rc;
  // one tensor's rows alone need no tile in shared memory
  if (n == 1 && !cols) return quantize_rows(q[0].type, jobs, *form, ceil, s);
  return quantize_tiles(q[0].type, jobs, n, form->scale_format, form->scale_block, ceil, s);
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
  const Divider chunks = divider((uint32_t)(((uint64_t)b->k + kChunk - 1) / kChunk));
  const bool vec = rows_aligned(type, out, b->rows, out_stride), wide = rows_aligned(type, out, b->rows, out_stride, 32);
  const uint64_t per = rows_per_launch(chunks.d) / 128 * 128;
  for (uint64_t row0 = 0; row0 < b->rows; row0 += per) {
    const uint32_t n = (uint32_t)(b->rows - row0 < per ? b->rows - row0 : per);
    const unsigned grid = grid_of(((uint64_t)n * chunks.d + kThreads - 1) / kThreads, 8);
    const int rc = with_form(type, b->scale_format, b->scale_block, [&](auto t, auto e8, auto blk) {
      auto go = [&](auto v) {
        return launched(launch_dependent(dequantize_kernel<decltype(t)::value, decltype(e8)::value, decltype(blk)::value,
                                                           decltype(v)::value>,
                                         dim3(grid), kThreads, 0, static_cast<cudaStream_t>(stream),
                                         static_cast<const uint8_t*>(b->data), b->stride,
                                         static_cast<const uint8_t*>(b->scales), groups, n, row0, (uint32_t)b->k, chunks,
                                         multiplier, out, out_stride, wide),
                        "dequantize_kernel launch");
      };
      return vec ? go(std::true_type{}) : go(std::false_type{});
    });
    if (rc != T5E_OK) return rc;
  }
  return T5E_OK;
}

}  // extern "C"
