// operators_stub.cpp -- the autograd nodes of csrc/torch_ops.cpp on CPU tensors,
// over C entries that launch nothing: the forwards fill their results with
// counted values, the backwards record every operand as they were told to read
// it (pointer, strides and sizes).  What a backward hands to the kernels can be
// checked this way without a GPU.
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
#include "../concord_amd/csrc/torch_ops.cpp"
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
template <class T>
void count(T* p, int64_t n) {
  for (int64_t i = 0; p && i < n; ++i) p[i] = (T)(i % 100);
}

}  // namespace

extern "C" {

const char* concord_last_error(void) { return "stub"; }

int concord_layernorm_fwd(const void*, int64_t, int, const void*, const void*, int, int64_t M, int64_t, float, void*,
                          int64_t, float* mean, float* rstd, void*) {
  count(mean, M);
  count(rstd, M);
  return CONCORD_OK;
}
size_t concord_layernorm_workspace_bytes(int64_t, int64_t) { return 16; }
int concord_layernorm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype, const void* weight,
                          int wdtype, const float* mean, const float* rstd, int64_t M, int64_t C, void*, int64_t, void*,
                          void*, void*, size_t, void*) {
  record("dy", dy, type_of(dtype), {M, C}, {ld_dy, 1});
  record("x", x, type_of(dtype), {M, C}, {ld_x, 1});
  record("weight", weight, type_of(wdtype), {C}, {1});
  record("mean", mean, at::kFloat, {M}, {1});
  record("rstd", rstd, at::kFloat, {M}, {1});
  return CONCORD_OK;
}

size_t concord_distill_workspace_bytes(int64_t, int64_t) { return 0; }
int concord_distill_fwd(const void*, int64_t, int, int64_t M, int64_t, const float*, int64_t, const int64_t*, int64_t,
                        int32_t, float, float* loss, float* stats, void*, size_t, void*) {
  count(loss, M);
  count(stats, 4 * M);
  return CONCORD_OK;
}
int concord_distill_bwd(const float* dloss, int64_t ld_dloss, const void* logits, int64_t ld_l, int dtype, int64_t M,
                        int64_t V, const float* teacher, int64_t ld_t, const int64_t* index, int64_t ld_i, int32_t K,
                        float, const float* stats, void*, int64_t, void*) {
  record("dloss", dloss, at::kFloat, {M}, {ld_dloss});
  record("logits", logits, type_of(dtype), {M, V}, {ld_l, 1});
  record("teacher", teacher, at::kFloat, {M, K}, {ld_t, 1});
  record("index", index, at::kLong, {M, K}, {ld_i, 1});
  record("stats", stats, at::kFloat, {M, 4}, {4, 1}, 16);
  return CONCORD_OK;
}

size_t concord_attention_fwd_workspace_bytes(const concord_attn_args*) { return 0; }
int concord_attention_fwd(const concord_attn_args* a, void*, size_t, void*) {
  count((int8_t*)a->out_low, a->TQ * a->H * a->D);
  count(a->lse, a->H * a->TQ);
  for (int64_t i = 0; i < a->TQ * a->H * a->D; ++i) ((at::BFloat16*)a->out)[i] = (float)(i % 100);
  return CONCORD_OK;
}
size_t concord_attention_workspace_bytes(const concord_attn_args*) { return 16; }
int concord_attention_bwd(const concord_attn_args* args, void*, size_t, void*) {
  const concord_attn_args& a = *args;
  auto rows = [&](const char* name, const uint16_t* p, int64_t t, int64_t h, int64_t T, int64_t H) {
    record(name, p, at::kBFloat16, {T, H, a.D}, {t, h, 1}, 16);
    if (t % 8 || h % 8) misaligned.push_back(name);
  };
  rows("q", a.q, a.q_t, a.q_h, a.TQ, a.H);
  rows("k", a.k, a.k_t, a.k_h, a.TK, a.HK);
  rows("v", a.v, a.v_t, a.v_h, a.TK, a.HK);
  rows("out", a.out, a.o_t, a.o_h, a.TQ, a.H);
  rows("dout", a.dout, a.do_t, a.do_h, a.TQ, a.H);
  record("lse", a.lse, at::kFloat, {a.H, a.TQ}, {a.TQ, 1});
  record("out_low", a.out_low, at::kChar, {a.TQ, a.H, a.D}, {(int64_t)a.H * a.D, a.D, 1}, 16);
  record("starts", a.starts, at::kInt, {a.B + 1}, {1});
  record("k_starts", a.k_starts, at::kInt, {a.B + 1}, {1});
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

PYBIND11_MODULE(concord_operators_stub, m) {
  m.def("layer_norm", &layer_norm);
  m.def("attention", &attention);
  m.def("distill_loss", &distill_loss);
  m.def("recorded", &recorded);
}
