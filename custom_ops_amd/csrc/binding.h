// binding.h — what the operators' implementations for PyTorch-ROCm share: fresh tensors,
// the checks of arguments, overlap of caches, and the refusal of derivatives.
#ifndef MI355_BINDING_H
#define MI355_BINDING_H

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <torch/library.h>

#include <dlfcn.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <tuple>

namespace mi355ops {
namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;

// A fresh tensor on x's GPU, straight from the caching allocator (the dispatcher's
// at::empty costs another 0.5 us, six times for the layout)
Tensor fresh(const Tensor& x, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, x.device(), std::nullopt);
}

void* stream_of(const Tensor& x) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
}

void finish(int rc, const char* err) { TORCH_CHECK(rc == 0, err); }

void check_gpu(const Tensor& x, const Tensor& like, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(x.device() == like.device(), "all tensors must be on the same device (", name, " is not on q's)");
}

void check_half(const Tensor& q) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be float16 or bfloat16");
}

// A tensor of rows that move as 16-byte chunks: innermost stride 1, the others
// multiples of 8 elements (where their size asks for them) and not negative.
void check_rows(const Tensor& x, const Tensor& q, const char* name, int64_t dim) {
  check_gpu(x, q, name);
  TORCH_CHECK(x.scalar_type() == q.scalar_type(), name, " dtype must match q");
  TORCH_CHECK(x.dim() == dim, name, " must be ", dim, "D");
  TORCH_CHECK(x.size(-1) <= 1 || x.stride(-1) == 1, name, " must have an innermost stride of 1");
  for (int64_t i = 0; i + 1 < dim; ++i)
    TORCH_CHECK(x.size(i) <= 1 || (x.stride(i) % 8 == 0), name, " must have strides that are multiples of 8 elements");
  TORCH_CHECK(x.numel() == 0 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

// The stride of a dimension as the kernels take it: of a single row, which is never
// stepped over, any multiple of 8 will do.
int64_t step(const Tensor& x, int64_t i) { return x.size(i) <= 1 ? 0 : x.stride(i); }

void check_ints(const Tensor& x, const Tensor& q, const char* name, at::ScalarType type, int64_t n) {
  check_gpu(x, q, name);
  TORCH_CHECK(x.scalar_type() == type, name, " must be ", type);
  TORCH_CHECK(x.dim() == 1 && x.size(0) == n, name, " must have ", n, " elements");
  TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
}

const float* slopes_of(const Maybe& s, const Tensor& q, int64_t heads) {
  if (!s.has_value()) return nullptr;
  check_gpu(*s, q, "slopes");
  TORCH_CHECK(s->scalar_type() == at::kFloat, "slopes must be float32");
  TORCH_CHECK(s->dim() == 1 && s->size(0) == heads && s->is_contiguous(), "slopes must be contiguous with ", heads, " elements");
  return s->data_ptr<float>();
}

// fp16 0, bf16 1 in every C ABI
int type_of(const Tensor& q) { return q.scalar_type() == at::kBFloat16 ? 1 : 0; }

void check_scores(std::optional<double> scale, double softcap, int64_t window) {
  TORCH_CHECK(!scale.has_value() || (*scale > 0 && std::isfinite(*scale)), "scale must be positive and finite");
  TORCH_CHECK(softcap >= 0 && softcap <= 1000 && (softcap == 0 || (float)softcap > 0), "softcap must be 0 (none) or in (0, 1000]");
  TORCH_CHECK(window >= 0 && window <= INT_MAX, "window must be 0 (none) or positive");
}

void check_groups(int64_t h, int64_t hk) { TORCH_CHECK(hk > 0 && h % hk == 0, "n_heads must be divisible by n_kv_heads (GQA)"); }
void check_head_dim(int64_t d) { TORCH_CHECK(d == 64 || d == 128, "Only head_dim=64 or head_dim=128 is supported"); }

// Whether two tensors of the same sizes and strides share an element: their distance is a
// sum of steps d_i·stride_i with |d_i| < size_i. Strides are taken from the largest, so
// each d_i has two candidates at most; dimensions that do not nest count as apart.
bool share(const Tensor& a, const Tensor& b) {
  const int64_t n = a.dim();
  if (a.numel() == 0 || a.strides() != b.strides() || !a.is_alias_of(b)) return false;
  int64_t order[8], reach[9] = {};
  if (n > 8) return false;
  for (int64_t i = 0; i < n; ++i) order[i] = i;
  std::sort(order, order + n, [&](int64_t x, int64_t y) { return a.stride(x) > a.stride(y); });
  for (int64_t i = n - 1; i >= 0; --i) {
    if (a.size(order[i]) > 1 && reach[i + 1] >= a.stride(order[i])) return false;
    reach[i] = reach[i + 1] + (a.size(order[i]) - 1) * a.stride(order[i]);
  }
  auto meets = [&](auto& self, int64_t dist, int64_t i) -> bool {
    if (std::abs(dist) > reach[i]) return false;
    if (i == n) return true;
    const int64_t s = a.stride(order[i]), most = a.size(order[i]) - 1;
    if (most == 0) return self(self, dist, i + 1);
    const int64_t d = dist / s;   // towards 0: the other candidate is one further
    for (int64_t x : {d, dist < 0 ? d - 1 : d + 1})
      if (std::abs(x) <= most && self(self, dist - x * s, i + 1)) return true;
    return false;
  };
  return meets(meets, b.storage_offset() - a.storage_offset(), 0);
}

// ── autograd ──────────────────────────────────────────────────────────────────
// There is no derivative, so the Autograd key refuses a call that needs one, backward
// (an input that requires a gradient while gradients are recorded) or forward (an input
// with a tangent). It does so for every kind of tensor, before the fake kernels that
// tracing calls in place of these.
void refuse_derivative(const Tensor& x) {
  if (!x.defined()) return;
  TORCH_CHECK(!(x.requires_grad() && at::GradMode::is_enabled()) && !x._fw_grad(/*level=*/0).defined(),
              "forward only: call it under torch.no_grad() or on detached tensors");
}
void refuse_derivative(const Maybe& x) {
  if (x.has_value()) refuse_derivative(*x);
}
template <class T> void refuse_derivative(const T&) {}

template <const char* Name, class F> struct Gate;
template <const char* Name, class R, class... A> struct Gate<Name, R(A...)> {
  static const c10::TypedOperatorHandle<R(A...)>& op() {
    static const auto handle = c10::Dispatcher::singleton().findSchemaOrThrow(Name, "").template typed<R(A...)>();
    return handle;
  }
  static R autograd(c10::DispatchKeySet keys, A... args) {
    (refuse_derivative(args), ...);
    at::AutoDispatchBelowAutograd below;
    return op().redispatch(keys & c10::after_autograd_keyset, args...);
  }
};

}  // namespace
}  // namespace mi355ops

#endif  // MI355_BINDING_H
