// torch_ops.h -- what the autograd nodes over the C entries share: checks of
// arguments, layouts, workspaces, saved tensors, and the list of what the module
// offers (torch_ops.cpp makes the module).
#pragma once
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <vector>

#include "concord_amd.h"

// What other sources add to the module: each puts a function here before the
// module is made.  (Hidden: two modules of this code in one process keep lists
// of their own.)
namespace concord_ops {
typedef void (*Registrar)(pybind11::module_&);
__attribute__((visibility("hidden"))) inline std::vector<Registrar>& registrars() {
  static std::vector<Registrar> list;
  return list;
}
struct Register {
  explicit Register(Registrar f) { registrars().push_back(f); }
};
}  // namespace concord_ops

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;   // (an autograd node takes no undefined tensor for an argument)

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
Tensor value(const MaybeTensor& t) { return t ? *t : Tensor(); }

// ---- checks -------------------------------------------------------------------
void need_gpu(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.device().is_cuda(), op, ": ", name, " must be a ROCm device tensor (got ", t.device(),
              "); there is no CPU implementation");
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CONCORD_F32;
    case at::kBFloat16: return CONCORD_BF16;
    case at::kHalf: return CONCORD_F16;
    default: return -1;
  }
}

// a C entry's return code
void check(int rc, const char* op) {
  if (rc == CONCORD_OK) return;
  if (rc == CONCORD_EINVAL) TORCH_CHECK_VALUE(false, op, ": ", concord_last_error());
  TORCH_CHECK(false, op, " failed (", rc, "): ", concord_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A dual tensor need not require grad, so the choice of a node by requires_grad
// alone would drop its tangent without a word.
void no_tangent(const char* op, std::initializer_list<const Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op, " has no derivative in forward mode");
}

void only_once(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, " is differentiable once: its backward has no gradient of its own");
}

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

// t as [rows, width] with adjacent columns, and its leading dimension: a view,
// or a copy where the strides allow none
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows rows_of(const Tensor& t, int64_t rows, int64_t width) {
  if (t.is_contiguous()) return {t, width};
  Tensor r = t.reshape({rows, width});
  if ((width > 1 && r.stride(1) != 1) || (rows > 1 && r.stride(0) < width)) r = r.contiguous();
  return {r, rows > 1 ? r.stride(0) : width};
}

// ---- saved tensors ----------------------------------------------------------------
// A saved-tensor hook (offloading to the host, recomputation) may give a saved
// tensor back in another layout: the backwards take strides from what comes
// back and keep none of the forward's.

// a vector or table that the kernels index without strides: its elements
// adjacent, on 16 bytes
Tensor packed(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}

// its type, extent and device have to be what was saved (like: the upstream gradient)
void came_back(const Tensor& t, at::ScalarType type, int64_t numel, const Tensor& like, const char* op,
               const char* name) {
  TORCH_CHECK(t.defined() && t.scalar_type() == type && t.numel() == numel && t.device() == like.device(), op,
              ": the saved ", name, " came back as another tensor");
}

// ---- layouts of heads ---------------------------------------------------------------
// a tensor as [tokens, heads, dim] the way the kernels read it: rows on 16
// bytes, dimensions adjacent; a view, or a copy where it is laid out otherwise
struct Operand {
  Tensor t;
  int64_t token, head;   // strides
};
Operand operand(const Tensor& x) {
  const bool four = x.dim() == 4;
  const int64_t b = four ? x.size(0) : 1, n = x.size(-3), h = x.size(-2), d = x.size(-1);
  // one stride has to step through the tokens of all sequences
  int64_t token = n > 1 || !four ? x.stride(-3) : x.stride(0);
  int64_t head = h > 1 ? x.stride(-2) : d;
  const bool one = b <= 1 || n <= 1 || x.stride(0) == n * token;
  if (b * n <= 1) token = h * d;
  const bool ok = one && x.stride(-1) == 1 && token % 8 == 0 && head % 8 == 0 && token >= d && token < (1 << 24) &&
                  (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0;
  if (ok) return {x, token, head};
  return {x.clone(at::MemoryFormat::Contiguous), h * d, d};
}

}  // namespace
