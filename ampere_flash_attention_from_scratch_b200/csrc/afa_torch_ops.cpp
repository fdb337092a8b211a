// afa_torch_ops.cpp -- the operators around a 4-bit key/value cache in the
// `afa_flash_attention_kernels` torch extension (none has a counterpart in the
// reference):
//     q, k   = rotary(q, k, positions, inv_freq, sections=None, interleaved=False,
//                     inverse=False, q_out=None, k_out=None)
//     cache  = cache4_empty(n_pages, n_kv_heads, page_size, head_dim, device)
//     None   = cache4_write(k, v, cache, page_table, kv_lens, new_lens=None)
//     k, v   = cache4_read(cache, page_table, kv_lens, n, dtype, new_lens=None, k_out=None, v_out=None)
//     O, lse = forward_cache4(q, cache, page_table, kv_lens, o=None, causal=False,
//                             softmax_scale=None, return_lse=False, new_lens=None)
// Checks and errors are those of forward_ext: RuntimeError before the launch for
// what the host can see, and for a bad page or length, which only the kernel
// sees, by the next call on the device or check_status().  Nothing here
// synchronises; what a call needs besides its outputs comes from torch's
// allocator on the call's stream, so calls and captured graphs never share it.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/extension.h>

#include <atomic>
#include <optional>
#include <tuple>
#include <vector>

#include "afa_sm100_ops.h"
#include "afa_torch_common.h"

namespace {

using afa_torch::dtype_code;
using afa_torch::raise_earlier_abort;
using afa_torch::status_word;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The compute capability of a device never changes: looked up once for each.
void check_arch(int dev) {
  static std::atomic<int> known[64];  // 10 * major + minor, 0: not looked up
  const bool kept = dev >= 0 && dev < 64;
  int cc = kept ? known[dev].load(std::memory_order_relaxed) : 0;
  if (cc == 0) {
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cc = 10 * major + minor;
    if (kept) known[dev].store(cc, std::memory_order_relaxed);
  }
  TORCH_CHECK(cc == 100, "Flash Attention (sm_100a build) requires SM_100 (current: SM_", cc / 10, ".", cc % 10, ")");
}

void check_positive(const at::Tensor& t, const char* name) {
  for (int d = 0; d < 4; ++d)
    TORCH_CHECK(t.size(d) > 0 && t.size(d) <= INT32_MAX, name, ": every dimension must be positive and fit 32 bits");
}

void fill_strides(int64_t (&s)[3], const at::Tensor& t) {
  for (int d = 0; d < 3; ++d) s[d] = t.stride(d);
}

// A new contiguous tensor on `dev`, past the dispatcher (0.3 us of host time less; a call takes 6 to 10).
at::Tensor fresh_tensor(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(shape, type, dev, std::nullopt));
}

// A tensor of the caller's has been written: autograd notices if it had saved
// it.  (Tensors made in inference mode have no version, and are never saved.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether forward-mode differentiation follows t.
bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

// Tensors of an operator without a gradient: what autograd would follow is refused, since its graph would end there.
void check_constant(const at::Tensor& t, const char* name, const char* op) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()) && !has_tangent(t), op, " is not differentiable: ", name,
              " must not require a gradient or have a tangent (detach it, or call under torch.no_grad())");
}

// `out` if given (checked against `like`), else a new contiguous tensor.
at::Tensor output_like(const std::optional<at::Tensor>& out, const at::Tensor& like, const char* name) {
  if (!out.has_value() || !out->defined()) return fresh_tensor(like.sizes(), like.scalar_type(), like.device());
  const at::Tensor& o = out.value();
  TORCH_CHECK(o.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(o.dim() == 4 && o.stride(3) == 1, name,
              " must be 4-D [batch, seq, heads, head_dim] with a contiguous head_dim");
  TORCH_CHECK(o.dtype() == like.dtype(), name, ": Output tensor must have the same dtype as inputs");
  TORCH_CHECK(o.sizes() == like.sizes(), name, ": output and input tensors must have the same shape");
  TORCH_CHECK(o.device() == like.device(), name, ": Output tensor must be on the same device");
  return o;
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------
struct RotaryPlan {
  std::vector<int64_t> sections;
  bool interleaved;
  bool inverse;
};

void check_rotary(const at::Tensor& x, const char* name, const at::Tensor& positions, const at::Tensor& inv_freq) {
  TORCH_CHECK(x.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 4 && x.stride(3) == 1, name,
              " must be 4-D [batch, seq, heads, head_dim] with a contiguous head_dim");
  TORCH_CHECK(dtype_code(x) > 0, "Only fp16 and bf16 are supported");
  check_positive(x, name);
  TORCH_CHECK(positions.device() == x.device() && inv_freq.device() == x.device(),
              "Input tensors must be on the same device");
  TORCH_CHECK(positions.dim() == 3 && positions.size(1) == x.size(0) && positions.size(2) == x.size(1),
              "positions must be [axes, batch, seq] for ", name);
}

// Launches on the current stream; k (and k_out) may be undefined.
void rotary_launch(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_out, const at::Tensor& k_out,
                   const at::Tensor& positions, const at::Tensor& inv_freq, const RotaryPlan& plan) {
  AfaRotaryArgs a{};
  a.q = q.data_ptr();
  a.q_out = q_out.data_ptr();
  fill_strides(a.q_strides, q);
  fill_strides(a.q_out_strides, q_out);
  if (k.defined()) {
    a.k = k.data_ptr();
    a.k_out = k_out.data_ptr();
    fill_strides(a.k_strides, k);
    fill_strides(a.k_out_strides, k_out);
    a.n_k_heads = static_cast<int32_t>(k.size(2));
  }
  a.positions = positions.data_ptr();
  fill_strides(a.pos_strides, positions);
  a.pos_type = positions.scalar_type() == at::kLong  ? AFA_POS_INT64
               : positions.scalar_type() == at::kInt ? AFA_POS_INT32
                                                     : AFA_POS_FP32;
  a.inv_freq = inv_freq.data_ptr<float>();
  a.n_axes = static_cast<int32_t>(plan.sections.size());
  for (size_t i = 0; i < plan.sections.size(); ++i) a.sections[i] = static_cast<int32_t>(plan.sections[i]);
  a.batch = static_cast<int32_t>(q.size(0));
  a.seq_len = static_cast<int32_t>(q.size(1));
  a.n_heads = static_cast<int32_t>(q.size(2));
  a.head_dim = static_cast<int32_t>(q.size(3));
  a.rot_dim = static_cast<int32_t>(2 * inv_freq.size(0));
  a.dtype = dtype_code(q);
  a.interleaved = plan.interleaved ? 1 : 0;
  a.inverse = plan.inverse ? 1 : 0;
  const int rc = afa_rotary_sm100(&a, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == AFA_OK, "afa_rotary_sm100 failed: ", afa_strerror(rc));
}

variable_list rotary_new(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                         const at::Tensor& inv_freq, const RotaryPlan& plan) {
  c10::cuda::CUDAGuard guard{q.device()};
  at::Tensor q_out = fresh_tensor(q.sizes(), q.scalar_type(), q.device());
  at::Tensor k_out = k.defined() ? fresh_tensor(k.sizes(), k.scalar_type(), k.device()) : at::Tensor();
  rotary_launch(q, k, q_out, k_out, positions, inv_freq, plan);
  return {q_out, k_out};
}

// A gradient as the kernel takes it: autograd may hand over expanded or
// otherwise strided tensors.
at::Tensor as_rows(const at::Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) == 1 || t.stride(d) % 8 == 0);
  return ok ? t : t.contiguous();
}

variable_list rotary_any(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                         const at::Tensor& inv_freq, const RotaryPlan& plan);

// The gradient of a rotation is the rotation back, differentiable again.
struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const std::optional<at::Tensor>& k,
                               const at::Tensor& positions, const at::Tensor& inv_freq,
                               const std::vector<int64_t>& sections, bool interleaved, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    variable_list out = rotary_new(q, k.has_value() ? *k : at::Tensor(), positions, inv_freq,
                                   RotaryPlan{sections, interleaved, inverse});
    if (!k.has_value()) out.pop_back();
    // an output follows its own input only
    variable_list constant;
    if (!q.requires_grad()) constant.push_back(out[0]);
    if (k.has_value() && !k->requires_grad()) constant.push_back(out[1]);
    if (!constant.empty()) ctx->mark_non_differentiable(constant);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const RotaryPlan back{ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(),
                          !ctx->saved_data["inverse"].toBool()};
    at::Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : at::Tensor();
    if (dq.defined()) dq = as_rows(dq);
    if (dk.defined()) dk = as_rows(dk);
    if (dq.defined()) {
      const variable_list out = rotary_any(dq, dk, saved[0], saved[1], back);
      dq = out[0];
      dk = out[1];
    } else if (dk.defined()) {
      dk = rotary_any(dk, at::Tensor(), saved[0], saved[1], back)[0];
    }
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Forward mode: a rotation is linear, so an output's tangent is its input's tangent turned alike.
variable_list rotary_dual(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                          const at::Tensor& inv_freq, const RotaryPlan& plan) {
  at::Tensor x[2], dx[2];
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = i == 0 ? q : k;
    if (!t.defined()) continue;
    std::tie(x[i], dx[i]) = at::_unpack_dual(t, 0);
    if (dx[i].defined()) dx[i] = dx[i]._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : as_rows(dx[i]);
  }
  variable_list out = rotary_any(x[0], x[1], positions, inv_freq, plan);
  at::Tensor d[2];
  if (dx[0].defined()) {
    const variable_list turned = rotary_any(dx[0], dx[1], positions, inv_freq, plan);
    d[0] = turned[0];
    d[1] = turned[1];
  } else {
    d[1] = rotary_any(dx[1], at::Tensor(), positions, inv_freq, plan)[0];
  }
  for (int i = 0; i < 2; ++i)
    if (d[i].defined()) out[i] = at::_make_dual(out[i], d[i], 0);
  return out;
}

variable_list rotary_any(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                         const at::Tensor& inv_freq, const RotaryPlan& plan) {
  if (has_tangent(q) || has_tangent(k)) return rotary_dual(q, k, positions, inv_freq, plan);
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
    const std::optional<at::Tensor> second = k.defined() ? std::optional<at::Tensor>(k) : std::nullopt;
    variable_list out =
        RotaryFunction::apply(q, second, positions, inv_freq, plan.sections, plan.interleaved, plan.inverse);
    if (!k.defined()) out.emplace_back();
    return out;
  }
  return rotary_new(q, k, positions, inv_freq, plan);
}

std::tuple<at::Tensor, std::optional<at::Tensor>> rotary(const at::Tensor& q, const std::optional<at::Tensor>& k_,
                                                         const at::Tensor& positions, const at::Tensor& inv_freq,
                                                         const std::optional<std::vector<int64_t>>& sections_,
                                                         bool interleaved, bool inverse,
                                                         const std::optional<at::Tensor>& q_out_,
                                                         const std::optional<at::Tensor>& k_out_) {
  const at::Tensor k = k_.has_value() ? k_.value() : at::Tensor();
  check_rotary(q, "q", positions, inv_freq);
  if (k.defined()) {
    check_rotary(k, "k", positions, inv_freq);
    TORCH_CHECK(k.dtype() == q.dtype(), "Input tensors must have the same data type");
    TORCH_CHECK(k.device() == q.device(), "Input tensors must be on the same device");
    TORCH_CHECK(k.size(3) == q.size(3), "query and key head_dim differ");
  }
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt ||
                  positions.scalar_type() == at::kFloat,
              "positions must be int32, int64 or float32");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous(),
              "inv_freq must be a contiguous 1-D float32 tensor");
  const int64_t axes = positions.size(0), pairs = inv_freq.size(0), d = q.size(3);
  TORCH_CHECK(q.size(2) + (k.defined() ? k.size(2) : 0) <= AFA_ROTARY_MAX_HEADS, "at most ", AFA_ROTARY_MAX_HEADS,
              " query and key heads together");
  TORCH_CHECK(axes >= 1 && axes <= AFA_ROTARY_MAX_AXES, "positions must have 1 to ", AFA_ROTARY_MAX_AXES, " axes");
  TORCH_CHECK(d % 16 == 0 && d <= 512, "head_dim must be a multiple of 16 and at most 512 (got ", d, ")");
  TORCH_CHECK(pairs > 0 && pairs % 8 == 0 && 2 * pairs <= d,
              "inv_freq must hold a multiple of 8 pairs, at most head_dim / 2 (got ", pairs, ")");
  RotaryPlan plan{{}, interleaved, inverse};
  if (sections_.has_value())
    plan.sections = sections_.value();
  else
    plan.sections = {pairs};
  TORCH_CHECK(static_cast<int64_t>(plan.sections.size()) == axes, "sections must have one entry for each of the ", axes,
              " axes of positions");
  int64_t sum = 0;
  for (const int64_t s : plan.sections) {
    TORCH_CHECK(s >= 0 && s <= pairs, "sections must not be negative and must add up to the pairs of inv_freq");
    sum += s;
  }
  TORCH_CHECK(sum == pairs, "sections must add up to the ", pairs, " pairs of inv_freq (got ", sum, ")");
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK((!grad || (!positions.requires_grad() && !inv_freq.requires_grad())) && !has_tangent(positions) &&
                  !has_tangent(inv_freq),
              "positions and inv_freq are not differentiable");
  const bool out_given = (q_out_.has_value() && q_out_->defined()) || (k_out_.has_value() && k_out_->defined());
  TORCH_CHECK(k.defined() || !k_out_.has_value() || !k_out_->defined(), "k_out without k");

  c10::cuda::CUDAGuard guard{q.device()};
  check_arch(q.device().index());
  raise_earlier_abort(q.device().index());
  variable_list out;
  if (out_given) {
    TORCH_CHECK((!grad || !(q.requires_grad() || (k.defined() && k.requires_grad()))) && !has_tangent(q) && !has_tangent(k),
                "q_out and k_out cannot be given for inputs that require a gradient or have a tangent");
    const at::Tensor q_out = output_like(q_out_, q, "q_out");
    const at::Tensor k_out = k.defined() ? output_like(k_out_, k, "k_out") : at::Tensor();
    TORCH_CHECK((!grad || !(q_out.requires_grad() || (k_out.defined() && k_out.requires_grad()))) &&
                    !has_tangent(q_out) && !has_tangent(k_out),
                "q_out and k_out must not require a gradient or have a tangent");
    rotary_launch(q, k, q_out, k_out, positions, inv_freq, plan);
    written(q_out);
    if (k_out.defined()) written(k_out);
    out = {q_out, k_out};
  } else {
    out = rotary_any(q, k, positions, inv_freq, plan);
  }
  std::optional<at::Tensor> second;
  if (k.defined()) second = out[1];
  return std::make_tuple(out[0], second);
}

// ---------------------------------------------------------------------------
// The 4-bit cache
// ---------------------------------------------------------------------------
void check_ints(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == dev, "Input tensors must be on the same device");
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
}

int row_head_dim(int64_t bytes) {
  for (const int d : {64, 128})
    if (afa_cache4_row_bytes(d) == bytes) return d;
  return 0;
}

// Checks a cache and its sequences and fills the C structure; dtype: AFA_DTYPE_*.
AfaCache4 cache_args(const at::Tensor& cache, const at::Tensor& page_table, const at::Tensor& kv_lens,
                     const std::optional<at::Tensor>& new_lens, int64_t batch, int dtype) {
  AFA_CHECK_CUDA(cache);
  TORCH_CHECK(cache.dim() == 5 && cache.scalar_type() == at::kByte && cache.size(2) == 2 && row_head_dim(cache.size(4)) != 0,
              "cache must be uint8 [pages, kv_heads, 2, page_size, row] with rows of ", afa_cache4_row_bytes(64),
              " bytes (head_dim 64) or ", afa_cache4_row_bytes(128), " bytes (head_dim 128)");
  const int64_t page_size = cache.size(3), row = cache.size(4), heads = cache.size(1);
  TORCH_CHECK(cache.size(0) > 0 && cache.size(0) <= INT32_MAX && heads > 0 && heads <= INT32_MAX,
              "cache: every dimension must be positive and fit 32 bits");
  TORCH_CHECK(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
              "page_size must be 16, 32, 64, 128 or 256 (got ", page_size, ")");
  TORCH_CHECK(cache.stride(4) == 1 && cache.stride(3) == row && cache.stride(2) == page_size * row &&
                  (heads == 1 || cache.stride(1) == 2 * page_size * row),
              "cache must be dense within a page");
  const at::Device dev = cache.device();
  check_ints(page_table, "page_table", dev);
  TORCH_CHECK(page_table.dim() == 2 && page_table.size(0) == batch && page_table.size(1) > 0 &&
                  page_table.size(1) <= INT32_MAX && (page_table.size(1) == 1 || page_table.stride(1) == 1),
              "page_table must be [batch, pages] with contiguous rows");
  check_ints(kv_lens, "kv_lens", dev);
  TORCH_CHECK(kv_lens.dim() == 1 && kv_lens.size(0) == batch && kv_lens.is_contiguous(),
              "kv_lens must be a contiguous [batch] tensor");
  AfaCache4 c{};
  if (new_lens.has_value() && new_lens->defined()) {
    check_ints(*new_lens, "new_lens", dev);
    TORCH_CHECK(new_lens->dim() == 1 && new_lens->size(0) == batch && new_lens->is_contiguous(),
                "new_lens must be a contiguous [batch] tensor");
    c.new_lens = new_lens->data_ptr<int32_t>();
  }
  c.cache = cache.data_ptr();
  c.page_stride = cache.stride(0);
  c.page_table = page_table.data_ptr<int32_t>();
  c.table_stride = page_table.stride(0);
  c.kv_lens = kv_lens.data_ptr<int32_t>();
  c.status = status_word(dev.index()).device;
  c.n_pages = static_cast<int32_t>(cache.size(0));
  c.page_size = static_cast<int32_t>(page_size);
  c.max_pages = static_cast<int32_t>(page_table.size(1));
  c.batch = static_cast<int32_t>(batch);
  c.n_kv_heads = static_cast<int32_t>(heads);
  c.head_dim = row_head_dim(row);
  c.dtype = dtype;
  return c;
}

at::Tensor cache4_empty(int64_t n_pages, int64_t n_kv_heads, int64_t page_size, int64_t head_dim,
                        const std::optional<at::Device>& device) {
  const int32_t row = head_dim > 0 && head_dim <= INT32_MAX ? afa_cache4_row_bytes(static_cast<int32_t>(head_dim)) : -1;
  TORCH_CHECK(row > 0, "no sm_100a kernel for head_dim ", head_dim, " (64 and 128 are compiled)");
  TORCH_CHECK(n_pages > 0 && n_kv_heads > 0, "n_pages and n_kv_heads must be positive");
  TORCH_CHECK(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
              "page_size must be 16, 32, 64, 128 or 256 (got ", page_size, ")");
  return at::empty({n_pages, n_kv_heads, 2, page_size, row},
                   at::TensorOptions().dtype(at::kByte).device(device.has_value() ? *device : at::Device(at::kCUDA)));
}

void cache4_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cache, const at::Tensor& page_table,
                  const at::Tensor& kv_lens, const std::optional<at::Tensor>& new_lens) {
  AFA_CHECK_CUDA(k);
  AFA_CHECK_CUDA(v);
  AFA_CHECK_LAST_DIM(k);
  AFA_CHECK_LAST_DIM(v);
  AFA_CHECK_CUDA(cache);
  c10::cuda::CUDAGuard guard{k.device()};
  const int dev = k.device().index();
  check_arch(dev);
  raise_earlier_abort(dev);
  TORCH_CHECK(dtype_code(k) > 0, "Only fp16 and bf16 are supported");
  TORCH_CHECK(v.dtype() == k.dtype(), "Input tensors must have the same data type");
  TORCH_CHECK(v.device() == k.device() && cache.device() == k.device(), "Input tensors must be on the same device");
  TORCH_CHECK(k.sizes() == v.sizes(), "key and value tensors must have the same shape");
  check_positive(k, "k");
  check_constant(k, "k", "cache4_write");
  check_constant(v, "v", "cache4_write");
  const AfaCache4 c = cache_args(cache, page_table, kv_lens, new_lens, k.size(0), dtype_code(k));
  TORCH_CHECK(k.size(2) == c.n_kv_heads && k.size(3) == c.head_dim, "k and v [batch, seq, ", k.size(2), ", ", k.size(3),
              "] do not match the cache's ", c.n_kv_heads, " heads of head_dim ", c.head_dim);
  int64_t ks[3], vs[3];
  fill_strides(ks, k);
  fill_strides(vs, v);
  const int rc = afa_cache4_write_sm100(&c, k.data_ptr(), v.data_ptr(), ks, vs, static_cast<int32_t>(k.size(1)),
                                        at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == AFA_OK, "afa_cache4_write_sm100 failed: ", afa_strerror(rc));
  written(cache);
}

std::tuple<at::Tensor, at::Tensor> cache4_read(const at::Tensor& cache, const at::Tensor& page_table,
                                               const at::Tensor& kv_lens, int64_t n, at::ScalarType dtype,
                                               const std::optional<at::Tensor>& new_lens,
                                               const std::optional<at::Tensor>& k_out,
                                               const std::optional<at::Tensor>& v_out) {
  AFA_CHECK_CUDA(cache);
  c10::cuda::CUDAGuard guard{cache.device()};
  const int dev = cache.device().index();
  check_arch(dev);
  raise_earlier_abort(dev);
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "Only fp16 and bf16 are supported");
  TORCH_CHECK(n > 0 && n <= INT32_MAX, "n must be positive and fit 32 bits");
  TORCH_CHECK(page_table.dim() == 2 && page_table.size(0) > 0 && page_table.size(0) <= INT32_MAX,
              "page_table must be [batch, pages] with contiguous rows");
  const int64_t batch = page_table.size(0);
  const AfaCache4 c = cache_args(cache, page_table, kv_lens, new_lens, batch,
                                 dtype == at::kHalf ? AFA_DTYPE_FP16 : AFA_DTYPE_BF16);
  auto make = [&](const std::optional<at::Tensor>& out, const char* name) {
    const std::vector<int64_t> shape = {batch, n, c.n_kv_heads, c.head_dim};
    if (!out.has_value() || !out->defined()) return fresh_tensor(shape, dtype, cache.device());
    const at::Tensor& o = *out;
    TORCH_CHECK(o.device() == cache.device() && o.scalar_type() == dtype && o.dim() == 4 && o.sizes() == at::IntArrayRef(shape) &&
                    o.stride(3) == 1,
                name, " must be [batch, n, kv_heads, head_dim] of the given dtype on the cache's device, with a contiguous head_dim");
    check_constant(o, name, "cache4_read");
    return o;
  };
  const at::Tensor k = make(k_out, "k_out"), v = make(v_out, "v_out");
  int64_t ks[3], vs[3];
  fill_strides(ks, k);
  fill_strides(vs, v);
  const int rc = afa_cache4_read_sm100(&c, k.data_ptr(), v.data_ptr(), ks, vs, static_cast<int32_t>(n),
                                       at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == AFA_OK, "afa_cache4_read_sm100 failed: ", afa_strerror(rc));
  written(k);
  written(v);
  return std::make_tuple(k, v);
}

std::tuple<at::Tensor, std::optional<at::Tensor>> forward_cache4(
    const at::Tensor& q, const at::Tensor& cache, const at::Tensor& page_table, const at::Tensor& kv_lens,
    const std::optional<at::Tensor>& o_, bool causal, std::optional<double> softmax_scale, bool return_lse,
    const std::optional<at::Tensor>& new_lens) {
  AFA_CHECK_CUDA(q);
  AFA_CHECK_LAST_DIM(q);
  AFA_CHECK_CUDA(cache);
  c10::cuda::CUDAGuard guard{q.device()};
  const int dev = q.device().index();
  check_arch(dev);
  raise_earlier_abort(dev);
  TORCH_CHECK(dtype_code(q) > 0, "Only fp16 and bf16 are supported");
  TORCH_CHECK(cache.device() == q.device(), "Input tensors must be on the same device");
  check_positive(q, "q");
  check_constant(q, "q", "forward_cache4");
  const AfaCache4 c = cache_args(cache, page_table, kv_lens, new_lens, q.size(0), dtype_code(q));
  TORCH_CHECK(q.size(3) == c.head_dim, "query head_dim (", q.size(3), ") and the cache's (", c.head_dim, ") differ");
  TORCH_CHECK(q.size(2) % c.n_kv_heads == 0, "the number of query heads (", q.size(2),
              ") must be a multiple of the number of key/value heads (", c.n_kv_heads, ")");
  double scale = 0.0;
  if (softmax_scale.has_value()) {
    scale = softmax_scale.value();
    TORCH_CHECK(scale > 0.0, "softmax_scale must be positive");
    TORCH_CHECK(static_cast<float>(scale) > 0.0f && scale < 1e38, "softmax_scale ", scale, " is not one of fp32's range");
  }
  const at::Tensor o = output_like(o_, q, "o");
  check_constant(o, "o", "forward_cache4");
  const int32_t n = static_cast<int32_t>(q.size(1)), heads = static_cast<int32_t>(q.size(2));
  std::optional<at::Tensor> lse;
  if (return_lse)
    lse = fresh_tensor({q.size(0), q.size(2), q.size(1)}, at::kFloat, q.device());
  const int64_t bytes = afa_cache4_fwd_workspace(&c, n, heads);
  TORCH_CHECK(bytes >= 0, "afa_cache4_fwd_workspace failed: ", afa_strerror(static_cast<int>(-bytes)));
  const at::Tensor ws = fresh_tensor({bytes}, at::kByte, q.device());
  AfaCache4FwdArgs a{};
  a.q = q.data_ptr();
  a.o = o.data_ptr();
  fill_strides(a.q_strides, q);
  fill_strides(a.o_strides, o);
  a.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
  a.workspace = ws.data_ptr();
  a.workspace_bytes = bytes;
  a.seq_len = n;
  a.n_heads = heads;
  a.causal = causal ? 1 : 0;
  a.scale = static_cast<float>(scale);
  const int rc = afa_cache4_fwd_sm100(&c, &a, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == AFA_OK, "afa_cache4_fwd_sm100 failed: ", afa_strerror(rc));
  written(o);
  return std::make_tuple(o, lse);
}

}  // namespace

namespace afa_torch {

void bind_ops(pybind11::module_& m) {
  m.def("rotary", &rotary, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"),
        py::arg("sections") = py::none(), py::arg("interleaved") = false, py::arg("inverse") = false,
        py::arg("q_out") = py::none(), py::arg("k_out") = py::none(),
        "Rotary positions with several axes: q [batch, seq, heads, d] and k (or None) turned by positions "
        "[axes, batch, seq] * inv_freq [pairs], sections[a] pairs for axis a; differentiable in q and k");
  m.def("cache4_empty", &cache4_empty, py::arg("n_pages"), py::arg("n_kv_heads"), py::arg("page_size"),
        py::arg("head_dim"), py::arg("device") = py::none(),
        "An uninitialised 4-bit cache: uint8 [n_pages, n_kv_heads, 2, page_size, row]");
  m.def("cache4_write", &cache4_write, py::arg("k"), py::arg("v"), py::arg("cache"), py::arg("page_table"),
        py::arg("kv_lens"), py::arg("new_lens") = py::none(),
        "Quantises k, v [batch, seq, kv_heads, d] to 4 bits into the last new_lens[b] (default: seq) of each "
        "sequence's kv_lens[b] tokens");
  m.def("cache4_read", &cache4_read, py::arg("cache"), py::arg("page_table"), py::arg("kv_lens"), py::arg("n"),
        py::arg("dtype"), py::arg("new_lens") = py::none(), py::arg("k_out") = py::none(), py::arg("v_out") = py::none(),
        "k, v [batch, n, kv_heads, d] of the last new_lens[b] (default: n) of each sequence's kv_lens[b] tokens; "
        "rows behind them are zero");
  m.def("forward_cache4", &forward_cache4, py::arg("q"), py::arg("cache"), py::arg("page_table"), py::arg("kv_lens"),
        py::arg("o") = py::none(), py::arg("causal") = false, py::arg("softmax_scale") = py::none(),
        py::arg("return_lse") = false, py::arg("new_lens") = py::none(),
        "Attention forward of q [batch, seq, heads, d] over a paged 4-bit cache; returns (O, lse or None)");
}

}  // namespace afa_torch
