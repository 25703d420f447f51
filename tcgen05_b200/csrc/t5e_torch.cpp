// t5e_torch.cpp -- the PyTorch side of the block-scaled calls: checks, allocation
// and the autograd node, over the C ABI of include/t5e.h.
//
// These calls are microseconds long on the device, so what the host does for
// one counts: from Python, with ctypes, rounding one token and multiplying it
// took 18 us of host time for 13 us of device time, and a small linear layer's
// training step 130 us, most of it in the backward pass's Python.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

#include "t5e.h"

namespace {

using at::Tensor;
using c10::optional;

void check(int rc, const char* what) {
  if (rc == T5E_OK) return;
  TORCH_CHECK(rc != T5E_ERR_CUDA, what, ": CUDA error: ", t5e_last_error());
  TORCH_CHECK_VALUE(false, what, ": invalid arguments (code ", rc, ")");
}

int32_t real_type(at::ScalarType t) {
  return t == at::kFloat ? T5E_REAL_F32 : t == at::kBFloat16 ? T5E_REAL_BF16 : t == at::kHalf ? T5E_REAL_F16 : -1;
}

// Refuses a tensor whose elements are no longer all there: its storage can be
// freed under it, and kernels would read or write where it was.
void check_stored(const Tensor& t, const char* name) {
  if (t.numel() == 0) return;
  int64_t last = t.storage_offset();
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  TORCH_CHECK_VALUE((int64_t)t.storage().nbytes() >= (last + 1) * (int64_t)t.itemsize(), "the memory of ", name,
                    " was freed");
}

void check_real(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(real_type(x.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.is_cuda() && x.layout() == at::kStrided, name,
                    " must be a dense tensor on a CUDA device (there is no CPU fallback)");
  check_stored(x, name);
}

// Forward-mode derivatives are not computed: an input's would be lost, an
// output's would no longer fit its value.
void check_no_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), name, " must not carry a forward-mode tangent");
}

void* stream_of(const c10::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

int64_t row_stride(int64_t k) { return (k + 31) / 32 * 16; }

int64_t scale_bytes(int64_t rows, int64_t k, int64_t block) {
  return (rows + 127) / 128 * ((k + 4 * block - 1) / (4 * block)) * 512;
}

// Rows of E2M1 codes with their scales: a t5e_blocks and what keeps its memory.
struct Rows {
  t5e_blocks b{};
  Tensor buffer;        // the rows, then the scale tiles; or undefined, and
  Tensor data, scales;  // two tensors of a caller's
  Tensor multiplier;    // undefined: 1
  const float* factor = nullptr;  // where the multiplier lies
  c10::Device device{c10::kCPU};

  // Refuses rows whose memory is no longer where the calls take it: a storage can
  // be freed, grown or exchanged under a tensor that somebody still holds.
  void check_there(const char* name) const {
    const auto holds = [](const Tensor& t, const void* p, int64_t bytes) {
      return bytes == 0 || (t.const_data_ptr() == p &&
                            (int64_t)t.storage().nbytes() >= t.storage_offset() * (int64_t)t.itemsize() + bytes);
    };
    const int64_t codes = (int64_t)b.rows * b.stride, steps = scale_bytes((int64_t)b.rows, b.k, b.scale_block);
    const bool there = buffer.defined() ? holds(buffer, b.data, codes + steps)
                                        : holds(data, b.data, codes) && holds(scales, b.scales, steps);
    TORCH_CHECK_VALUE(there && (!multiplier.defined() || holds(multiplier, factor, 4)), "the memory of ", name,
                      " was freed or moved since they were made");
  }
  Tensor get_data() const {
    check_there("the rows");
    if (data.defined()) return data;
    return buffer.narrow(0, 0, (int64_t)b.rows * b.stride).view({(int64_t)b.rows, b.stride});
  }
  Tensor get_scales() const {
    check_there("the rows");
    if (scales.defined()) return scales;
    const int64_t at = (int64_t)b.rows * b.stride;
    return buffer.narrow(0, at, buffer.size(0) - at)
        .view({((int64_t)b.rows + 127) / 128, (b.k + 4 * b.scale_block - 1) / (4 * b.scale_block), 512});
  }
  void keep_multiplier(const Tensor& m) {
    multiplier = m;
    factor = m.defined() ? m.const_data_ptr<float>() : nullptr;
  }
};

t5e_blocks blocks_at(char* at, int64_t rows, int64_t k, int32_t fmt, int32_t block) {
  t5e_blocks b{};
  b.stride = row_stride(k);
  b.data = at;
  b.scales = at + rows * b.stride;
  b.rows = (uint64_t)rows;
  b.k = k;
  b.scale_format = fmt;
  b.scale_block = block;
  return b;
}

int64_t blocks_size(int64_t rows, int64_t k, int64_t block) { return rows * row_stride(k) + scale_bytes(rows, k, block); }

Tensor bytes_on(const c10::Device& device, int64_t n) { return at::empty({n}, at::TensorOptions(device).dtype(at::kByte)); }

Rows new_rows(const c10::Device& device, int64_t rows, int64_t k, int32_t fmt, int32_t block, const Tensor& multiplier) {
  Rows r;
  r.buffer = bytes_on(device, blocks_size(rows, k, block));
  r.b = blocks_at(static_cast<char*>(r.buffer.data_ptr()), rows, k, fmt, block);
  r.keep_multiplier(multiplier);
  r.device = device;
  return r;
}

Rows given_rows(const Tensor& data, const Tensor& scales, int64_t k, int32_t fmt, int32_t block,
                const optional<Tensor>& multiplier) {
  TORCH_CHECK_VALUE(k >= 1 && k <= T5E_MAX_BLOCK_K, "K=", k, " outside 1..", (int64_t)T5E_MAX_BLOCK_K);
  TORCH_CHECK_VALUE(data.dim() == 2 && data.scalar_type() == at::kByte && (data.size(0) == 0 || data.is_contiguous()),
                    "data must be a contiguous [rows, stride] uint8 tensor");
  const int64_t rows = data.size(0), stride = data.size(1);
  TORCH_CHECK_VALUE((uint64_t)rows <= T5E_MAX_BLOCK_ROWS, "more than ", (uint64_t)T5E_MAX_BLOCK_ROWS, " rows");
  TORCH_CHECK_VALUE(stride % 16 == 0 && stride >= row_stride(k), "row stride ", stride, " is not a multiple of 16 of at least ",
                    row_stride(k));
  const int64_t tiles = (rows + 127) / 128, groups = (k + 4 * block - 1) / (4 * block);
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kByte && scales.dim() == 3 && scales.size(0) == tiles &&
                        scales.size(1) == groups && scales.size(2) == 512 && scales.is_contiguous(),
                    "scales must be a contiguous [", tiles, ", ", groups, ", 512] uint8 tensor (tile_scales)");
  TORCH_CHECK_VALUE(scales.device() == data.device(), "data and scales are on different devices");
  if (multiplier)
    TORCH_CHECK_VALUE(multiplier->scalar_type() == at::kFloat && multiplier->numel() == 1 &&
                          multiplier->device() == data.device(),
                      "multiplier must be a one-element float32 tensor on the data's device");
  const auto at = reinterpret_cast<uintptr_t>(data.data_ptr()), scales_at = reinterpret_cast<uintptr_t>(scales.data_ptr());
  TORCH_CHECK_VALUE(at % 16 == 0 && scales_at % 16 == 0, "data and scales must start on 16-byte boundaries");
  Rows r;
  r.data = data;
  r.scales = scales;
  if (multiplier) r.keep_multiplier(multiplier->resolve_neg());
  r.device = data.device();
  r.b.data = data.data_ptr();
  r.b.stride = stride;
  r.b.scales = scales.data_ptr();
  r.b.rows = (uint64_t)rows;
  r.b.k = k;
  r.b.scale_format = fmt;
  r.b.scale_block = block;
  return r;
}

// x as rows of its last dimension with unit column stride, or `turned`, the
// matrix whose columns those rows are (no copy of a transposed matrix); other
// layouts are copied.
struct Matrix {
  Tensor x;
  int64_t rows, cols, stride;
  bool turned;
};

Matrix matrix_of(Tensor x) {
  if (x.is_neg()) x = x.resolve_neg();
  if (x.dim() != 2) x = x.reshape({-1, x.size(-1)});
  const int64_t rows = x.size(0), cols = x.size(1), down = x.stride(0), across = x.stride(1);
  if ((across == 1 || cols == 1) && (rows == 1 || down >= cols)) return {x, rows, cols, down, false};
  if (down == 1 && across >= rows) return {x, cols, rows, across, true};
  x = x.contiguous();
  return {x, rows, cols, cols, false};
}

// Blocks that look for the largest of n elements: 8192 elements each, up to four
// per multiprocessor.
int32_t partial_count(int64_t n) {
  const int64_t c = (n + 8191) / 8192;
  return (int32_t)(c < 1 ? 1 : c > 592 ? 592 : c);
}

t5e_quantize job_of(const Matrix& m, int32_t rounding, float* multiplier, uint32_t* partials, int32_t count,
                    const t5e_blocks* rows, const t5e_blocks* cols, float* kept = nullptr) {
  if (m.turned) std::swap(rows, cols);
  t5e_quantize q{};
  q.x = m.x.const_data_ptr();
  q.rows = (uint64_t)m.rows;
  q.cols = (uint64_t)m.cols;
  q.stride = m.stride;
  q.type = real_type(m.x.scalar_type());
  q.rounding = rounding;
  q.multiplier = multiplier;
  q.partials = partials;
  q.count = count;
  if (rows) q.by_rows = *rows;
  if (cols) q.by_cols = *cols;
  q.kept = kept;
  return q;
}

Tensor multiplier_of(const Tensor& x0) {
  check_real(x0, "x");
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor x = x0.dim() == 0 ? x0.reshape({1}) : x0;
  if (x.numel() == 0) return at::ones({1}, x.options().dtype(at::kFloat));
  const c10::cuda::CUDAGuard guard(x.device());
  const Matrix m = matrix_of(x);
  const int32_t count = partial_count(x.numel());
  const Tensor work = at::empty({1 + count}, x.options().dtype(at::kFloat));
  float* at = work.mutable_data_ptr<float>();
  check(t5e_block_multiplier(real_type(x.scalar_type()), m.x.const_data_ptr(), (uint64_t)m.rows, (uint64_t)m.cols, m.stride,
                             reinterpret_cast<uint32_t*>(at + 1), count, at, stream_of(x.device())),
        "t5e_block_multiplier");
  return work.narrow(0, 0, 1);
}

enum { kByRows = 1, kByCols = 2 };

// The rows and the columns of x that `axes` asks for (the other stays empty).
// The blocks keep the value that `given` has now, not the caller's tensor: a
// program may update it in place, and what was rounded before stands as it was.
// The rounding kernel copies it (a copy of its own would be another launch).
std::pair<Rows, Rows> quantize(const Tensor& x, int axes, int32_t fmt, int32_t block, int32_t rounding,
                               const optional<Tensor>& given, bool automatic) {
  check_real(x, "x");
  at::AutoDispatchBelowADInplaceOrView below;
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "x must have at least one dimension and a non-empty last one");
  const int64_t k = x.size(-1), r = x.numel() / k;
  const bool by_rows = axes & kByRows, by_cols = axes & kByCols;
  TORCH_CHECK_VALUE(!(by_rows && k > T5E_MAX_BLOCK_K) && !(by_cols && r > T5E_MAX_BLOCK_K) &&
                        (uint64_t)std::max(r, k) <= T5E_MAX_BLOCK_ROWS,
                    "x is larger than ", (int64_t)T5E_MAX_BLOCK_K, " elements along a block axis or ",
                    (uint64_t)T5E_MAX_BLOCK_ROWS, " rows");
  TORCH_CHECK_VALUE(!(by_cols && r == 0), "blocks along an empty axis");
  const c10::Device device = x.device();
  const c10::cuda::CUDAGuard guard(device);
  Tensor source, multiplier;  // `source`: the given one
  uint32_t* partials = nullptr;
  int32_t count = 0;
  if (given) {
    TORCH_CHECK_VALUE(given->scalar_type() == at::kFloat && given->numel() == 1 && given->device() == device,
                      "multiplier must be a one-element float32 tensor on x's device");
    check_stored(*given, "multiplier");
    source = given->resolve_neg();
    multiplier = r > 0 ? at::empty({1}, x.options().dtype(at::kFloat)) : source.reshape({1}).clone();
  } else if (automatic && r > 0) {
    count = partial_count(r * k);
    const Tensor work = at::empty({1 + count}, x.options().dtype(at::kFloat));
    partials = reinterpret_cast<uint32_t*>(work.mutable_data_ptr<float>() + 1);
    multiplier = work.narrow(0, 0, 1);
  }
  std::pair<Rows, Rows> out;
  if (by_rows) out.first = new_rows(device, r, k, fmt, block, multiplier);
  if (by_cols) out.second = new_rows(device, k, r, fmt, block, multiplier);
  if (r > 0) {
    const Matrix m = matrix_of(x);
    float* const at = multiplier.defined() ? multiplier.mutable_data_ptr<float>() : nullptr;
    const t5e_quantize q = job_of(m, rounding, given ? const_cast<float*>(source.const_data_ptr<float>()) : at, partials, count,
                                  by_rows ? &out.first.b : nullptr, by_cols ? &out.second.b : nullptr, given ? at : nullptr);
    check(t5e_quantize_blocks(&q, 1, stream_of(device)), "t5e_quantize_blocks");
  }
  return out;
}

py::object py_quantize(const Tensor& x, int axes, int32_t fmt, int32_t block, int32_t rounding,
                       const optional<Tensor>& given, bool automatic) {
  std::pair<Rows, Rows> q = quantize(x, axes, fmt, block, rounding, given, automatic);
  if (axes == (kByRows | kByCols)) return py::make_tuple(std::move(q.first), std::move(q.second));
  return py::cast(axes == kByRows ? std::move(q.first) : std::move(q.second));
}

// [first, behind the last) byte of a tensor's elements.
std::pair<uintptr_t, uintptr_t> span_of(const Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const auto at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {at, at + (uintptr_t)(last + 1) * t.element_size()};
}

// The result: `out` checked, or a new tensor.
Tensor result(const optional<Tensor>& out, int64_t rows, int64_t cols, at::ScalarType dtype, const c10::Device& device) {
  if (!out) return at::empty({rows, cols}, at::TensorOptions(device).dtype(dtype));
  TORCH_CHECK_VALUE(out->dim() == 2 && out->size(0) == rows && out->size(1) == cols && out->scalar_type() == dtype &&
                        out->device() == device,
                    "out must be a [", rows, ", ", cols, "] ", dtype, " tensor on ", device);
  TORCH_CHECK_VALUE(out->numel() == 0 || ((cols == 1 || out->stride(1) == 1) && (rows == 1 || out->stride(0) >= cols)),
                    "out must have unit column stride and rows that do not overlap");
  TORCH_CHECK_VALUE(!(out->requires_grad() && at::GradMode::is_enabled()), "out must not require a gradient");
  check_no_tangent(*out, "out");
  check_stored(*out, "out");
  TORCH_CHECK_VALUE(!out->is_neg(), "out must not be a negated view");
  return *out;
}

// Refuses an `out` that shares memory with the blocks it is computed from, or
// with their multiplier, which every block of a kernel reads for itself.
void check_apart(const Tensor& out, const Rows& r, const char* name) {
  if (out.numel() == 0) return;
  const auto d = span_of(out);
  const auto overlaps = [&](const void* p, int64_t n) {
    const auto at = reinterpret_cast<uintptr_t>(p);
    return at < d.second && d.first < at + (uintptr_t)n;
  };
  TORCH_CHECK_VALUE(!overlaps(r.b.data, (int64_t)r.b.rows * r.b.stride) &&
                        !overlaps(r.b.scales, scale_bytes((int64_t)r.b.rows, r.b.k, r.b.scale_block)) &&
                        !(r.factor != nullptr && overlaps(r.factor, sizeof(float))),
                    "out overlaps ", name);
}

// Tells autograd, as PyTorch's own `out` arguments do, that `out` is written: a
// graph that saved it refuses its backward pass.  Refuses an inference tensor
// outside inference mode.  Called last before the launch, so that a refused call
// leaves no trace.
void note_written(const Tensor& out) { out.unsafeGetTensorImpl()->bump_version(); }

void check_on_device(const Rows& r, const char* name) {
  TORCH_CHECK_VALUE(r.device.is_cuda(), name, " must be on a CUDA device (there is no CPU fallback)");
}

Tensor dequantize(const Rows& r, at::ScalarType dtype, const optional<Tensor>& given) {
  r.check_there("blocks");
  check_on_device(r, "blocks");
  TORCH_CHECK_VALUE(real_type(dtype) >= 0, "dtype must be float32, bfloat16 or float16, not ", dtype);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(r.device);
  Tensor out = result(given, (int64_t)r.b.rows, r.b.k, dtype, r.device);
  if (given) {
    check_apart(out, r, "blocks");
    note_written(out);
  }
  check(t5e_dequantize_blocks(&r.b, r.factor, real_type(dtype), out.mutable_data_ptr(),
                              r.b.rows > 1 ? out.stride(0) : r.b.k, stream_of(r.device)),
        "t5e_dequantize_blocks");
  return out;
}

void launch_product(const t5e_blocks& a, const t5e_blocks& b, const float* ma, const float* mb, float alpha, int32_t form,
                    const Tensor* c, Tensor& out, const c10::Device& device) {
  t5e_block_mm mm{};
  mm.a = a;
  mm.b = b;
  mm.multiplier_a = ma;
  mm.multiplier_b = mb;
  mm.alpha = alpha;
  mm.form = form;
  if (c) {
    mm.c = c->const_data_ptr();
    mm.c_type = real_type(c->scalar_type());
    mm.c_row_stride = c->stride(0);
    mm.c_col_stride = c->stride(1);
  }
  mm.d = out.mutable_data_ptr();
  mm.d_type = real_type(out.scalar_type());
  mm.d_stride = a.rows > 1 ? out.stride(0) : (int64_t)b.rows;
  check(t5e_block_scaled_mm(&mm, stream_of(device)), "t5e_block_scaled_mm");
}

Tensor mm(const Rows& a, const Rows& b, const optional<Tensor>& addend, double alpha, at::ScalarType dtype,
          const optional<Tensor>& given, int32_t form) {
  a.check_there("a");
  b.check_there("b");
  check_on_device(a, "a");
  check_on_device(b, "b");
  TORCH_CHECK_VALUE(a.b.scale_format == b.b.scale_format && a.b.scale_block == b.b.scale_block,
                    "a and b have different forms of scales");
  TORCH_CHECK_VALUE(a.b.k == b.b.k, "a has K=", a.b.k, " but b has K=", b.b.k);
  TORCH_CHECK_VALUE(a.device == b.device, "a and b are on different devices");
  TORCH_CHECK_VALUE(real_type(dtype) >= 0, "dtype must be float32, bfloat16 or float16, not ", dtype);
  TORCH_CHECK_VALUE(!std::isfinite(alpha) || std::isfinite((float)alpha), "alpha=", alpha, " is not a float32");
  const int64_t m = (int64_t)a.b.rows, n = (int64_t)b.b.rows;
  Tensor c;
  if (addend) {
    check_real(*addend, "c");
    TORCH_CHECK_VALUE(addend->device() == a.device, "c is on another device");
    TORCH_CHECK_VALUE(!(addend->requires_grad() && at::GradMode::is_enabled()),
                      "block_scaled_mm gives c no gradient; detach it or use block_scaled_linear");
    check_no_tangent(*addend, "c");
    TORCH_CHECK_VALUE(addend->dim() <= 2, "c must broadcast to [", m, ", ", n, "]");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  if (addend) {
    const int64_t rows = addend->dim() == 2 ? addend->size(0) : 1, cols = addend->dim() > 0 ? addend->size(-1) : 1;
    TORCH_CHECK_VALUE((rows == 1 || rows == m) && (cols == 1 || cols == n), "c of shape ", addend->sizes(),
                      " does not broadcast to [", m, ", ", n, "]");
    c = (addend->is_neg() ? addend->resolve_neg() : *addend).expand({m, n});
  }
  const c10::cuda::CUDAGuard guard(a.device);
  Tensor out = result(given, m, n, dtype, a.device);
  if (given) {
    check_apart(out, a, "a");
    check_apart(out, b, "b");
    if (c.defined() && out.numel() > 0) {
      const auto cs = span_of(c), ds = span_of(out);
      const bool same = cs.first == ds.first && c.scalar_type() == out.scalar_type() &&
                        (m == 1 || c.stride(0) == out.stride(0)) && (n == 1 || c.stride(1) == out.stride(1));
      TORCH_CHECK_VALUE(!(cs.first < ds.second && ds.first < cs.second) || same, "c overlaps out without being out");
    }
    note_written(out);
  }
  launch_product(a.b, b.b, a.factor, b.factor, (float)alpha, form, c.defined() ? &c : nullptr, out,
                 a.device);
  return out;
}

// ---- the linear layer ------------------------------------------------------------

// Gradients that were computed from raw memory: differentiating them again is
// refused (they would be constants to autograd, although dx depends on w and dw
// on x).  `tie` is any tensor that requires a gradient, so that the node exists
// whether the incoming gradient requires one or not.
struct Once : torch::autograd::Function<Once> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, Tensor grad, const Tensor&) {
    return {grad};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "block_scaled_linear is differentiable once");
  }
};

// Parts of one allocation: sizes are added up first.
struct Space {
  int64_t size = 0;
  int64_t take(int64_t n) {
    const int64_t at = size;
    size = (at + n + 255) / 256 * 256;
    return at;
  }
};

// The three products of block_scaled_linear.  The calls are those of
// quantize_blocks and block_scaled_mm, x and w rounded in the same launches and
// everything a pass needs in one allocation.
struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, int64_t fmt, int64_t block,
                        int64_t rounding, bool need_x, bool need_w) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = w.size(0), k = w.size(1), tokens = x.numel() / k;
    const bool automatic = fmt == T5E_SCALE_UE4M3;
    auto& saved = ctx->saved_data;
    saved["shape"] = x.sizes().vec();
    saved["sizes"] = std::vector<int64_t>{n, k, tokens, fmt, block, rounding};
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n;
    if (tokens == 0) return at::empty(shape, x.options());
    const c10::Device device = x.device();
    const c10::cuda::CUDAGuard guard(device);
    // Blocks run along the contraction: K here, the tokens and N in the
    // gradients, so what a gradient needs is rounded along the other axis.  Kept
    // for the backward pass: the multipliers, then the columns.
    Space kept, passing;
    kept.take(8);
    const int64_t xt = need_w ? kept.take(blocks_size(k, tokens, block)) : -1;
    const int64_t wt = need_x ? kept.take(blocks_size(k, n, block)) : -1;
    const int64_t xr = passing.take(blocks_size(tokens, k, block)), wr = passing.take(blocks_size(n, k, block));
    const int32_t x_count = automatic ? partial_count(tokens * k) : 0, w_count = automatic ? partial_count(n * k) : 0;
    const int64_t partials = passing.take(4 * (x_count + w_count));
    const Tensor keep = bytes_on(device, kept.size), work = bytes_on(device, passing.size);
    char *base = static_cast<char*>(keep.data_ptr()), *there = static_cast<char*>(work.data_ptr());
    const auto at = [&](char* p, int64_t off, int64_t rows, int64_t length) {
      return blocks_at(p + off, rows, length, (int32_t)fmt, (int32_t)block);
    };
    const t5e_blocks xb = at(there, xr, tokens, k), wb = at(there, wr, n, k);
    t5e_blocks xc{}, wc{};
    if (need_w) xc = at(base, xt, k, tokens);
    if (need_x) wc = at(base, wt, k, n);
    float* m = automatic ? reinterpret_cast<float*>(base) : nullptr;
    uint32_t* p = automatic ? reinterpret_cast<uint32_t*>(there + partials) : nullptr;
    const Matrix xm = matrix_of(x), wm = matrix_of(w);
    const t5e_quantize jobs[2] = {
        job_of(xm, (int32_t)rounding, m, p, x_count, &xb, need_w ? &xc : nullptr),
        job_of(wm, (int32_t)rounding, automatic ? m + 1 : nullptr, automatic ? p + x_count : nullptr, w_count, &wb,
               need_x ? &wc : nullptr)};
    check(t5e_quantize_blocks(jobs, 2, stream_of(device)), "t5e_quantize_blocks");
    Tensor y = at::empty({tokens, n}, x.options());
    launch_product(xb, wb, m, automatic ? m + 1 : nullptr, 1.f, 0, nullptr, y, device);
    ctx->save_for_backward({keep});
    saved["parts"] = std::vector<int64_t>{xt, wt, kept.size};
    return x.dim() == 2 ? y : y.view(shape);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const Tensor g = grads[0];
    Tensor dx, dw;
    if (g.defined()) {
      {
        at::AutoDispatchBelowADInplaceOrView below;
        gradients(ctx, g, dx, dw);
      }
      // grad mode is on here only under create_graph=True
      if (at::GradMode::is_enabled()) {
        Tensor tie = at::empty({0});
        tie.set_requires_grad(true);
        if (dx.defined()) dx = Once::apply(dx, tie)[0];
        if (dw.defined()) dw = Once::apply(dw, tie)[0];
      }
    }
    return {dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }

  static void gradients(torch::autograd::AutogradContext* ctx, const Tensor& g, Tensor& dx, Tensor& dw) {
    auto& saved = ctx->saved_data;
    const std::vector<int64_t> shape = saved["shape"].toIntVector(), sizes = saved["sizes"].toIntVector();
    const int64_t n = sizes[0], k = sizes[1], tokens = sizes[2], fmt = sizes[3], block = sizes[4], rounding = sizes[5];
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    if (tokens == 0) {
      if (need_x) dx = at::zeros(shape, g.options());
      if (need_w) dw = at::zeros({n, k}, g.options());
      return;
    }
    if (!need_x && !need_w) return;
    const bool automatic = fmt == T5E_SCALE_UE4M3;
    const std::vector<int64_t> parts = saved["parts"].toIntVector();
    const Tensor keep = ctx->get_saved_variables()[0];
    const c10::Device device = g.device();
    // hooks on saved tensors may have put another one in its place
    TORCH_CHECK_VALUE(keep.device() == device && keep.scalar_type() == at::kByte && keep.dim() == 1 &&
                          keep.size(0) == parts[2] && keep.is_contiguous() &&
                          reinterpret_cast<uintptr_t>(keep.const_data_ptr()) % 16 == 0,
                      "what block_scaled_linear saved came back on another device or in another form");
    const c10::cuda::CUDAGuard guard(device);
    Space space;
    const int64_t gr = need_x ? space.take(blocks_size(tokens, n, block)) : -1;
    const int64_t gt = need_w ? space.take(blocks_size(n, tokens, block)) : -1;
    const int32_t count = automatic ? partial_count(tokens * n) : 0;
    const int64_t small = space.take(4 * (1 + count));
    const Tensor work = bytes_on(device, space.size);
    char *base = static_cast<char*>(keep.data_ptr()), *there = static_cast<char*>(work.data_ptr());
    const auto at = [&](char* p, int64_t off, int64_t rows, int64_t length) {
      return blocks_at(p + off, rows, length, (int32_t)fmt, (int32_t)block);
    };
    t5e_blocks grb{}, gtb{};
    if (need_x) grb = at(there, gr, tokens, n);
    if (need_w) gtb = at(there, gt, n, tokens);
    const float* m = automatic ? reinterpret_cast<const float*>(base) : nullptr;
    float* mg = automatic ? reinterpret_cast<float*>(there + small) : nullptr;
    const Matrix gm = matrix_of(g);
    const t5e_quantize job = job_of(gm, (int32_t)rounding, mg, automatic ? reinterpret_cast<uint32_t*>(mg + 1) : nullptr, count,
                                    need_x ? &grb : nullptr, need_w ? &gtb : nullptr);
    check(t5e_quantize_blocks(&job, 1, stream_of(device)), "t5e_quantize_blocks");
    if (need_x) {
      dx = at::empty({tokens, k}, g.options());
      launch_product(grb, at(base, parts[1], k, n), mg, automatic ? m + 1 : nullptr, 1.f, 0, nullptr, dx, device);
      if (shape.size() != 2) dx = dx.view(shape);
    }
    if (need_w) {
      dw = at::empty({n, k}, g.options());
      launch_product(gtb, at(base, parts[0], k, tokens), mg, m, 1.f, 0, nullptr, dw, device);
    }
  }
};

Tensor linear(const Tensor& x, const Tensor& w, int64_t fmt, int64_t block, int64_t rounding) {
  check_real(x, "x");
  check_real(w, "w");
  check_no_tangent(x, "x");
  check_no_tangent(w, "w");
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), "x [..., K] and w [N, K] do not fit: ", x.sizes(),
                    ", ", w.sizes());
  TORCH_CHECK_VALUE(w.numel() > 0, "w must not be empty");
  TORCH_CHECK_VALUE(x.scalar_type() == w.scalar_type() && x.device() == w.device(), "x and w must have one type and device");
  const int64_t most = std::max({w.size(0), w.size(1), x.numel() / w.size(1)});
  TORCH_CHECK_VALUE(most <= T5E_MAX_BLOCK_K, "a size of x or w is larger than ", (int64_t)T5E_MAX_BLOCK_K);
  const bool grad = at::GradMode::is_enabled();
  return Linear::apply(x, w, fmt, block, rounding, grad && x.requires_grad(), grad && w.requires_grad());
}

}  // namespace

PYBIND11_MODULE(t5e_torch, m) {
  py::class_<Rows>(m, "Rows")
      .def(py::init(&given_rows))
      .def_property_readonly("rows", [](const Rows& r) { return r.b.rows; })
      .def_property_readonly("k", [](const Rows& r) { return r.b.k; })
      .def_property_readonly("block", [](const Rows& r) { return r.b.scale_block; })
      .def_property_readonly("data", &Rows::get_data)
      .def_property_readonly("scales", &Rows::get_scales)
      .def_property_readonly("device", [](const Rows& r) { return r.device; })
      .def_property_readonly("multiplier", [](const Rows& r) -> optional<Tensor> {
        return r.multiplier.defined() ? optional<Tensor>(r.multiplier) : optional<Tensor>();
      });
  m.def("quantize", &py_quantize);
  m.def("multiplier", &multiplier_of);
  m.def("dequantize", &dequantize);
  m.def("mm", &mm);
  m.def("linear", &linear);
  m.attr("abi_version") = (int)T5E_ABI_VERSION;
  m.attr("built_for") = T5E_BUILT_FOR;  // what the build command looks for in the file
}
