// Host path: what its files share (settings, descriptors, checks, the status word).
#pragma once
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <atomic>
#include <mutex>
#include <optional>

#include "../../include/llsa_b200.h"

namespace llsa_host {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::variable_list;

// ------------------------------------------------------------------ settings (mirrored from ops.py)
enum Flag : int {
  kForceGeneric = 1,    // every stage on the scalar kernels
  kNoTcgen05 = 2,       // pooled stages on the mma.sync kernels
  kExactGrad = 4,       // one level: token weight kept in the pooled-key gradients
  kTwoPass = 8,         // long pooled lists: two passes over the keys for every row
  kDeviceChecks = 16,   // read the status word back after every operator
  kNoOverlap = 32,      // index transpose on the main stream
};
inline std::atomic<int> g_flags{0}, g_wait_limit{0};
inline std::atomic<bool> g_has_hook{false};
inline PyObject* g_hook = nullptr;      // guarded by the GIL

inline bool flag(Flag f) { return g_flags.load(std::memory_order_relaxed) & f; }

inline void mark(const char* name) {
  if (!g_has_hook.load(std::memory_order_relaxed)) return;
  pybind11::gil_scoped_acquire gil;
  if (g_hook) pybind11::reinterpret_borrow<pybind11::object>(g_hook)(name);
}

// ------------------------------------------------------------------ descriptors
inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LLSA_F32;
    case at::kBFloat16: return LLSA_BF16;
    case at::kInt: return LLSA_I32;
    case at::kLong: return LLSA_I64;
    default: TORCH_CHECK_TYPE(false, "llsa_b200 supports float32 and bfloat16 tensors, got ", t);
  }
}

inline LlsaTensor desc(const Tensor& t) {
  LlsaTensor d;
  d.ptr = t.data_ptr();
  d.dtype = dtype_code(t.scalar_type());
  d.ndim = (int32_t) t.dim();
  TORCH_CHECK(t.dim() <= 4, "llsa_b200: tensors of at most 4 dimensions, got ", t.dim());
  for (int i = 0; i < d.ndim; ++i) {
    d.shape[i] = t.size(i);
    d.stride[i] = t.stride(i);
  }
  return d;
}

inline LlsaTensor packed(void* p, int dtype, std::initializer_list<int64_t> shape) {
  LlsaTensor d;
  d.ptr = p;
  d.dtype = dtype;
  d.ndim = (int32_t) shape.size();
  int i = 0;
  for (int64_t s : shape) d.shape[i++] = s;
  int64_t st = 1;
  for (i = d.ndim - 1; i >= 0; --i) {
    d.stride[i] = st;
    st *= d.shape[i];
  }
  return d;
}

inline void ok(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "llsa_b200.", what, " failed (code ", rc, "): ", llsa_last_error_string());
}

inline void need_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "llsa_b200 runs on CUDA tensors only (got a ", t.device().type(), " tensor); there is no CPU path");
}

// Operands the caller may leave out are undefined tensors here.  A host pointer in a descriptor would be read by a kernel.
inline void need_cuda(std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    if (t.defined()) need_cuda(t);
}
inline Tensor or_none(const OptTensor& t) { return t.value_or(Tensor()); }

inline void check_float(std::initializer_list<const Tensor*> ts) {
  const at::ScalarType dt = (*ts.begin())->scalar_type();
  TORCH_CHECK_TYPE(dt == at::kFloat || dt == at::kBFloat16, "llsa_b200 supports float32 and bfloat16 tensors, got ", dt);
  for (const Tensor* t : ts) TORCH_CHECK_TYPE(t->scalar_type() == dt, "llsa_b200: all floating-point operands must share one dtype");
}

// Unit channel stride; bf16 rows on 32-byte boundaries (256-bit loads of the tensor-core kernels), fp32 rows on 16-byte ones; no rows that
// overlap, such as those of an expanded tensor: tensor maps are specified for strides that reach past a row.
inline bool rows_ok(const Tensor& t) {
  const int64_t align = t.scalar_type() == at::kBFloat16 ? 32 : 16, per = align / t.element_size();
  if (t.stride(-1) != 1 || (uintptr_t) t.data_ptr() % align) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) != 1 && (t.stride(i) % per || t.stride(i) < t.size(-1))) return false;
  return true;
}
inline Tensor prep(const Tensor& t) { return rows_ok(t) ? t : t.contiguous(); }
inline Tensor cont(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
inline bool table_ok(const Tensor& f) {
  return f.stride(-1) == 1 && (uintptr_t) f.data_ptr() % 16 == 0 && (f.stride(0) * f.element_size()) % 16 == 0;
}

// Blocks carved out of one allocation, every one on a 256-byte boundary.
struct Carver {
  int64_t off = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = off;
    off += (bytes + 255) / 256 * 256;
    return at;
  }
};
inline Tensor byte_buffer(int64_t n, const Tensor& like) {
  return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(like.device()));
}

// ------------------------------------------------------------------ status word
struct Status {
  Tensor word;
  explicit Status(const Tensor& like) {
    if (flag(kDeviceChecks)) word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(like.device()));
  }
  int32_t* ptr() const { return word.defined() ? (int32_t*) word.data_ptr() : nullptr; }
  void check(const char* what) const {
    if (word.defined()) ok(llsa_status_check(word.item<int32_t>()), what);
  }
};

inline OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

}  // namespace llsa_host
