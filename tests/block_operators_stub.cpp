// block_operators_stub.cpp -- the autograd nodes of csrc/torch_ops_block.cpp on CPU
// tensors, over C entries that launch nothing: the forwards fill what they keep with
// counted values, the backwards record every operand as they were told to read it.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

namespace c10::hip {
struct NoStream {
  void* stream() const { return nullptr; }
};
inline NoStream no_stream(int) { return {}; }
}  // namespace c10::hip

#define is_cuda is_cpu
#define getCurrentHIPStream no_stream
#include "../concord_amd/csrc/torch_ops_block.cpp"
#undef is_cuda
#undef getCurrentHIPStream

namespace {

std::vector<std::pair<std::string, Tensor>> seen;
std::vector<std::string> misaligned;

at::ScalarType type_of(int dtype) {
  return dtype == CONCORD_F32 ? at::kFloat : dtype == CONCORD_BF16 ? at::kBFloat16 : at::kHalf;
}
void record(const char* name, const void* p, at::ScalarType type, std::vector<int64_t> sizes,
            std::vector<int64_t> strides, int align = 1) {
  if ((uintptr_t)p % align) misaligned.push_back(name);
  if (!p) return;
  seen.emplace_back(name, at::from_blob(const_cast<void*>(p), sizes, strides, at::TensorOptions().dtype(type)).clone());
}

}  // namespace

extern "C" {

const char* concord_last_error(void) { return "stub"; }

int concord_embedding_fwd(const void*, int, int64_t, const void*, int64_t, int, int64_t, int64_t, float, void*, int64_t, int,
                          void*) {
  return CONCORD_OK;
}
size_t concord_embedding_workspace_bytes(int64_t, int64_t, int64_t) { return 16; }
int concord_embedding_bwd(const void* tokens, int index64, int64_t n, const void* dy, int64_t ld_dy, int dtype, int64_t, int64_t C,
                          float scale, void*, int64_t, int, void*, size_t, void*) {
  record("tokens", tokens, index64 ? at::kLong : at::kInt, {n}, {1});
  record("dy", dy, type_of(dtype), {n, C}, {ld_dy, 1});
  record("scale", &scale, at::kFloat, {1}, {1});
  return CONCORD_OK;
}

int concord_qk_norm_rope_fwd(const concord_qk_args*, void*) { return CONCORD_OK; }
size_t concord_qk_norm_rope_workspace_bytes(const concord_qk_args*) { return 16; }
int concord_qk_norm_rope_bwd(const concord_qk_args* args, void*, size_t, void*) {
  const concord_qk_args& a = *args;
  auto rows = [&](const char* name, const void* p, int64_t t, int64_t h, int64_t H) {
    record(name, p, type_of(a.dtype), {a.T, H, a.D}, {t, h, 1}, 16);
    if (t % 8 || h % 8) misaligned.push_back(name);
  };
  rows("q", a.q, a.q_t, a.q_h, a.H);
  rows("k", a.k, a.k_t, a.k_h, a.HK);
  rows("dq_out", a.dq_out, a.dq_t, a.dq_h, a.H);
  rows("dk_out", a.dk_out, a.dk_t, a.dk_h, a.HK);
  record("q_weight", a.q_weight, type_of(a.wtype), {a.D}, {1});
  record("k_weight", a.k_weight, type_of(a.wtype), {a.D}, {1});
  record("positions", a.positions, a.pos64 ? at::kLong : at::kInt, {a.pos_seq}, {1});
  double settings[4] = {a.base, a.eps, (double)a.R, (double)a.adjacent};
  record("settings", settings, at::kDouble, {4}, {1});
  return CONCORD_OK;
}

int concord_pack8(const void*, int64_t, int, int64_t, int64_t, int8_t*, uint8_t*, void*) { return CONCORD_OK; }
int concord_unpack8(const int8_t*, const uint8_t*, int64_t, int64_t, void*, int64_t, int, void*) { return CONCORD_OK; }
int concord_gelu8_fwd(const void*, int64_t, int, int64_t rows, int64_t C, int gated, int, void*, int64_t, int8_t* codes,
                      uint8_t* exponents, void*) {
  const int64_t wide = gated ? 2 : 1;
  for (int64_t i = 0; codes && i < rows * wide * C; ++i) codes[i] = (int8_t)(i % 100);
  for (int64_t i = 0; exponents && i < rows * wide * ((C + 31) / 32); ++i) exponents[i] = (uint8_t)(i % 100);
  return CONCORD_OK;
}
int concord_gelu8_bwd(const void* dy, int64_t ld_dy, const int8_t* codes, const uint8_t* exponents, int dtype, int64_t rows,
                      int64_t C, int gated, int tanh_form, void*, int64_t, void*) {
  const int64_t wide = gated ? 2 : 1, nb = (C + 31) / 32;
  record("dy", dy, type_of(dtype), {rows, C}, {ld_dy, 1});
  record("codes", codes, at::kChar, {rows, wide * C}, {wide * C, 1});
  record("exponents", exponents, at::kByte, {rows, wide * nb}, {wide * nb, 1});
  record("tanh", &tanh_form, at::kInt, {1}, {1});
  return CONCORD_OK;
}

}  // extern "C"

// a backward's operands since the last call, and the names of those that lay badly
static std::pair<std::vector<std::pair<std::string, Tensor>>, std::vector<std::string>> recorded() {
  auto r = std::make_pair(seen, misaligned);
  seen.clear();
  misaligned.clear();
  return r;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  for (auto add : concord_ops::registrars()) add(m);
  m.def("recorded", &recorded);
}
