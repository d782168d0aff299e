// distill.hip -- distillation from a teacher's top logits: the Kullback-
// Leibler divergence of a student's distribution from the teacher's, which is
// known at its K largest logits only, forward and backward.
//
// Per row, with z the student's logits, (t_k, i_k) the teacher's, T the
// temperature and entries outside [0, V) left out:
//   q = softmax(z / T) over the vocabulary, p = softmax(t / T) over the entries
//   loss = T^2 sum_k p_k (log p_k - log q[i_k])
//   dz   = g T (q - p),  p added up at entries that name one place twice
// A row without an entry has loss 0 and gradient 0, and so has the gradient
// of a row whose upstream gradient g is 0, whatever its logits hold.
//
// Bound by memory: forward reads the logits once (running maximum and sum of
// exponentials), backward reads them again and writes the gradient.  All
// statistics are fp32.  A row is one wave's (V <= 1024), one block's, or is
// split over several blocks when the rows are too few to fill the chip.
#include "elem.h"

namespace concord {

constexpr int kTopMax = 1024;      // teacher entries per row
constexpr int kWaveRow = 1024;     // longest row that one wave takes

struct DistillArgs {
  const void* z;
  int64_t ldz, M, V;
  const float* t;           // teacher's logits [M][K]
  int64_t ldt;
  const int64_t* idx;       // their places
  int64_t ldi;
  int K;
  float c;                  // log2(e) / T
  float T;
  float* loss;
  float* stat;              // [M][2]: the row's largest logit, sum exp((z - it) / T)
  float* part;              // [M][splits][2] of split rows
  int splits;
  int64_t seg;              // elements of a split (a multiple of 8)
  const float* g;           // backward: gradient of the loss rows, stride ldg (0: one value for all)
  int64_t ldg;
  void* dz;
  int64_t lddz;
};

// A running maximum and the sum of 2^((z - max) c) under it.
struct MaxSum {
  float m, s;
};
// (an empty part has m = -inf, s = 0; a maximum of -inf gives factor 2^0)
CONCORD_DEV float rel_exp2(float z, float m, float c) { return __builtin_amdgcn_exp2f((z - m) * c); }
CONCORD_DEV MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  // an empty side adds nothing (its factor would be 2^(-inf + inf))
  const float x = a.s == 0.0f ? 0.0f : a.s * rel_exp2(a.m, m, c);
  const float y = b.s == 0.0f ? 0.0f : b.s * rel_exp2(b.m, m, c);
  return MaxSum{m, x + y};
}
// over the wave: the maximum first, then the sums under it
CONCORD_DEV MaxSum wave_join(MaxSum a, float c) {
  const float m = wave_max_f32(a.m);
  return MaxSum{m, wave_sum(a.s == 0.0f ? 0.0f : a.s * rel_exp2(a.m, m, c))};
}

// threads of one row: a wave, or a block of four
template <int W>
struct Lanes {
  static CONCORD_DEV int id() { return W == 1 ? threadIdx.x & 63 : threadIdx.x; }
  static CONCORD_DEV int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
};

// [v0, v1) of a row in `N` elements per thread and round: 16-byte chunks
// where the row's address allows, single elements before and after them.
// f(element index, values[n], count of valid ones) sees each element once.
template <class T>
struct Span {
  static constexpr int VEC = 16 / (int)sizeof(T);
  int64_t head, body;   // elements before the first whole chunk; whole chunks
  CONCORD_DEV Span(const T* p, int64_t n) {
    const int64_t mis = ((uintptr_t)p & 15) / sizeof(T);
    head = mis ? min<int64_t>(VEC - mis, n) : 0;
    body = (n - head) / VEC;
  }
};

// statistics of z[0, n)
template <class T, int W>
CONCORD_DEV MaxSum row_stats(const T* z, int64_t n, float c) {
  constexpr int VEC = Span<T>::VEC, U = 4, TH = W * 64;
  const Span<T> sp(z, n);
  const int lane = Lanes<W>::id();
  MaxSum a{-INFINITY, 0.0f};
  auto add = [&](const float* v, int cnt) {
    float m = a.m;
    for (int i = 0; i < cnt; ++i) m = fmaxf(m, v[i]);
    float s = a.s == 0.0f ? 0.0f : a.s * rel_exp2(a.m, m, c);
    // all of them -inf so far: they add nothing
    if (m != -INFINITY)
      for (int i = 0; i < cnt; ++i) s += rel_exp2(v[i], m, c);
    else
      for (int i = 0; i < cnt; ++i) s += v[i] == v[i] ? 0.0f : v[i];
    a = MaxSum{m, s};
  };
  if (lane < sp.head) {
    const float v = to_f32(z[lane]);
    add(&v, 1);
  }
  const Chunk<T, VEC>* q = (const Chunk<T, VEC>*)(z + sp.head);
  int64_t k = lane;
  for (; k + (U - 1) * TH < sp.body; k += U * TH) {
    Chunk<T, VEC> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = q[k + u * TH];
    float v[U * VEC];
#pragma unroll
    for (int i = 0; i < U * VEC; ++i) v[i] = to_f32(r[i / VEC].v[i % VEC]);
    add(v, U * VEC);
  }
  for (; k < sp.body; k += TH) {
    const Chunk<T, VEC> r = q[k];
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(r.v[i]);
    add(v, VEC);
  }
  const int64_t tail = sp.head + sp.body * VEC;
  if (lane < n - tail) {
    const float v = to_f32(z[tail + lane]);
    add(&v, 1);
  }
  return wave_join(a, c);
}

// join of the block's waves, to every thread
CONCORD_DEV MaxSum block_join(MaxSum a, float (*red)[2], float c) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    red[wave][0] = a.m;
    red[wave][1] = a.s;
  }
  __syncthreads();
  MaxSum t{red[0][0], red[0][1]};
#pragma unroll
  for (int k = 1; k < 4; ++k) t = join(t, MaxSum{red[k][0], red[k][1]}, c);
  return t;
}

// the teacher's side of a row by one wave: its maximum and sum over the
// entries inside the vocabulary (s = 0: none)
CONCORD_DEV MaxSum teacher_stats(const DistillArgs& a, int64_t row) {
  const int lane = threadIdx.x & 63;
  MaxSum s{-INFINITY, 0.0f};
  for (int k = lane; k < a.K; k += 64) {
    const int64_t i = a.idx[row * a.ldi + k];
    const float t = a.t[row * a.ldt + k];
    if (i >= 0 && i < a.V && t != -INFINITY) s = join(s, MaxSum{t, 1.0f}, a.c);
  }
  return wave_join(s, a.c);
}

// loss of a row from its statistics, by one wave
template <class T>
CONCORD_DEV void row_loss(const DistillArgs& a, int64_t row, MaxSum q) {
  const int lane = threadIdx.x & 63;
  const MaxSum t = teacher_stats(a, row);
  const T* z = (const T*)a.z + row * a.ldz;
  constexpr float LN2 = 0.69314718055994531f;
  const float inv_T = a.c * LN2, logs = (__builtin_log2f(q.s) - __builtin_log2f(t.s)) * LN2;
  float sum = 0.0f;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t i = a.idx[row * a.ldi + k];
    const float tk = a.t[row * a.ldt + k];
    if (i >= 0 && i < a.V && tk != -INFINITY) {
      const float p = rel_exp2(tk, t.m, a.c) / t.s;
      // log p - log q; a probability that rounds to zero adds nothing
      if (p != 0.0f) sum += p * (((tk - t.m) - (to_f32(z[i]) - q.m)) * inv_T + logs);
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) {
    a.loss[row] = t.s == 0.0f ? 0.0f : sum * (a.T * a.T);
    if (a.stat) {
      a.stat[2 * row] = q.m;
      a.stat[2 * row + 1] = q.s;
    }
  }
}

template <class T, int W>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillArgs a) {
  __shared__ float red[4][2];
  if (W == 1) {
    const int64_t row = (int64_t)blockIdx.x * 4 + Lanes<W>::wave();
    if (row < a.M) row_loss<T>(a, row, row_stats<T, 1>((const T*)a.z + row * a.ldz, a.V, a.c));
    return;
  }
  const int64_t row = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t v0 = split * a.seg, n = min<int64_t>(a.seg, a.V - v0);
  const MaxSum s = block_join(row_stats<T, 4>((const T*)a.z + row * a.ldz + v0, n, a.c), red, a.c);
  if (a.splits == 1) {
    if (Lanes<W>::wave() == 0) row_loss<T>(a, row, s);
  } else if (threadIdx.x == 0) {
    float* p = a.part + ((int64_t)row * a.splits + split) * 2;
    p[0] = s.m;
    p[1] = s.s;
  }
}

// split rows: the parts joined and the loss, one wave a row
template <class T>
__global__ __launch_bounds__(256) void distill_join_kernel(DistillArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + Lanes<1>::wave();
  if (row >= a.M) return;
  const float* p = a.part + row * a.splits * 2;
  MaxSum s{-INFINITY, 0.0f};
  for (int k = threadIdx.x & 63; k < a.splits; k += 64) s = join(s, MaxSum{p[2 * k], p[2 * k + 1]}, a.c);
  row_loss<T>(a, row, wave_join(s, a.c));
}

// The gradient of [v0, v0 + n) of a row: q written first, then the entries
// that fall there, each place once, by the first entry that names it.
template <class T, int W>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a) {
  constexpr int TH = W * 64, VEC = Span<T>::VEC;
  extern __shared__ int32_t entries[];   // per row: K places in [v0, v0 + n) or -1, then their p
  const int lane = Lanes<W>::id(), slot = W == 1 ? Lanes<W>::wave() : 0;
  int32_t* place = entries + slot * 2 * a.K;
  float* prob = (float*)(place + a.K);
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + slot : blockIdx.x / a.splits;
  if (W == 1 && row >= a.M) return;   // (a wave for itself: no barrier below)
  const int64_t v0 = W == 1 ? 0 : (int64_t)(blockIdx.x % a.splits) * a.seg;
  const int64_t n = W == 1 ? a.V : min<int64_t>(a.seg, a.V - v0);
  const T* z = (const T*)a.z + row * a.ldz + v0;
  T* dz = (T*)a.dz + row * a.lddz + v0;
  const MaxSum t = teacher_stats(a, row);
  const float g = a.g[row * a.ldg] * a.T;
  const float m = a.stat[2 * row], inv = 1.0f / a.stat[2 * row + 1];
  const bool none = g == 0.0f || t.s == 0.0f;
  for (int k = lane; k < a.K; k += TH) {
    const int64_t i = a.idx[row * a.ldi + k] - v0;
    const float tk = a.t[row * a.ldt + k];
    const bool in = i >= 0 && i < n && tk != -INFINITY && !none;
    place[k] = in ? (int32_t)i : -1;
    prob[k] = in ? rel_exp2(tk, t.m, a.c) / t.s : 0.0f;
  }
  auto grad = [&](float v) { return none ? 0.0f : g * (rel_exp2(v, m, a.c) * inv); };
  const Span<T> sp(z, n);
  if (((uintptr_t)dz & 15) == ((uintptr_t)z & 15)) {
    constexpr int U = 2;
    if (lane < sp.head) dz[lane] = from_f32<T>(grad(to_f32(z[lane])));
    const Chunk<T, VEC>* q = (const Chunk<T, VEC>*)(z + sp.head);
    Chunk<T, VEC>* o = (Chunk<T, VEC>*)(dz + sp.head);
    auto chunk = [&](const Chunk<T, VEC>& r) {
      Chunk<T, VEC> w;
#pragma unroll
      for (int i = 0; i < VEC; ++i) w.v[i] = from_f32<T>(grad(to_f32(r.v[i])));
      return w;
    };
    int64_t k = lane;
    for (; k + (U - 1) * TH < sp.body; k += U * TH) {
      Chunk<T, VEC> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = q[k + u * TH];
#pragma unroll
      for (int u = 0; u < U; ++u) o[k + u * TH] = chunk(r[u]);
    }
    for (; k < sp.body; k += TH) o[k] = chunk(q[k]);
    const int64_t tail = sp.head + sp.body * VEC;
    if (lane < n - tail) dz[tail + lane] = from_f32<T>(grad(to_f32(z[tail + lane])));
  } else {
    for (int64_t k = lane; k < n; k += TH) dz[k] = from_f32<T>(grad(to_f32(z[k])));
  }
  // the stores above come before those below, also of other threads
  __threadfence_block();
  if (W > 1) __syncthreads();
  for (int k = lane; k < a.K; k += TH) {
    const int32_t i = place[k];
    if (i < 0) continue;
    float p = 0.0f;
    bool first = true;
    for (int j = 0; j < a.K; ++j)
      if (place[j] == i) {
        p += prob[j];
        first = first && j >= k;
      }
    if (first) dz[i] = from_f32<T>(g * (rel_exp2(to_f32(z[i]), m, a.c) * inv - p));
  }
}

// ---- host -------------------------------------------------------------------
// Blocks a row is split over: none while the rows alone give 1024 blocks; at
// least 4096 elements a block.
static int distill_splits(int64_t M, int64_t V) {
  if (V <= kWaveRow || M >= 1024) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(1024, M), V / 4096));
}
static void distill_split(DistillArgs& a) {
  a.splits = distill_splits(a.M, a.V);
  a.seg = cdiv(cdiv(a.V, a.splits), 8) * 8;
  a.splits = (int)cdiv(a.V, a.seg);
}

template <class T>
static void distill_fwd(const DistillArgs& a, hipStream_t st) {
  if (a.V <= kWaveRow)
    hipLaunchKernelGGL((distill_fwd_kernel<T, 1>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((distill_fwd_kernel<T, 4>), dim3((unsigned)(a.M * a.splits)), dim3(256), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 0, st, a);
}
template <class T>
static void distill_bwd(const DistillArgs& a, hipStream_t st) {
  const size_t lds = (size_t)a.K * 8;   // a row's entries
  if (a.V <= kWaveRow)
    hipLaunchKernelGGL((distill_bwd_kernel<T, 1>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 4 * lds, st, a);
  else
    hipLaunchKernelGGL((distill_bwd_kernel<T, 4>), dim3((unsigned)(a.M * a.splits)), dim3(256), lds, st, a);
}

static int distill_check(const char* what, const DistillArgs& a, int dtype, float temperature) {
  CONCORD_CHECK(a.M >= 0 && a.V >= 1 && a.M < (1LL << 24) && a.V < (1LL << 30), "%s: bad size", what);
  CONCORD_CHECK(a.K >= 0 && a.K <= kTopMax, "%s: at most %d teacher entries a row", what, kTopMax);
  CONCORD_CHECK(dtype == CONCORD_F32 || dtype == CONCORD_BF16 || dtype == CONCORD_F16, "%s: bad type", what);
  CONCORD_CHECK(a.ldz >= a.V && a.ldt >= a.K && a.ldi >= a.K, "%s: leading dimension too small", what);
  CONCORD_CHECK(temperature > 0.0f && temperature < INFINITY, "%s: the temperature must be positive", what);
  CONCORD_CHECK(a.M == 0 || (a.z && ((a.t && a.idx) || a.K == 0)), "%s: NULL argument", what);
  return CONCORD_OK;
}

static DistillArgs distill_args(const void* logits, int64_t ld_l, int64_t M, int64_t V, const float* teacher,
                                int64_t ld_t, const int64_t* index, int64_t ld_i, int32_t K, float temperature) {
  DistillArgs a{};
  a.z = logits, a.ldz = ld_l, a.M = M, a.V = V, a.t = teacher, a.ldt = ld_t, a.idx = index, a.ldi = ld_i, a.K = K;
  a.T = temperature;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  return a;
}

}  // namespace concord

using namespace concord;

extern "C" size_t concord_distill_workspace_bytes(int64_t M, int64_t V) {
  if (M < 1 || V < 1) return 0;
  const int s = distill_splits(M, V);
  return s > 1 ? (size_t)M * s * 2 * sizeof(float) : 0;
}

extern "C" int concord_distill_fwd(const void* logits, int64_t ld_l, int dtype, int64_t M, int64_t V,
                                   const float* teacher, int64_t ld_t, const int64_t* index, int64_t ld_i, int32_t K,
                                   float temperature, float* loss, float* stats, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  DistillArgs a = distill_args(logits, ld_l, M, V, teacher, ld_t, index, ld_i, K, temperature);
  if (const int rc = distill_check("concord_distill_fwd", a, dtype, temperature)) return rc;
  if (M == 0) return CONCORD_OK;
  CONCORD_CHECK(loss, "concord_distill_fwd: NULL argument");
  const size_t need = concord_distill_workspace_bytes(M, V);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("concord_distill_fwd: workspace of %zu bytes needed", need);
    return CONCORD_EWORKSPACE;
  }
  a.loss = loss, a.stat = stats, a.part = (float*)workspace;
  distill_split(a);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CONCORD_F32) distill_fwd<float>(a, st);
  else if (dtype == CONCORD_BF16) distill_fwd<BF16>(a, st);
  else distill_fwd<_Float16>(a, st);
  return launch_status("distill_fwd");
}

extern "C" int concord_distill_bwd(const float* dloss, int64_t ld_dloss, const void* logits, int64_t ld_l, int dtype,
                                   int64_t M, int64_t V, const float* teacher, int64_t ld_t, const int64_t* index,
                                   int64_t ld_i, int32_t K, float temperature, const float* stats, void* dlogits,
                                   int64_t ld_d, void* stream) {
  DistillArgs a = distill_args(logits, ld_l, M, V, teacher, ld_t, index, ld_i, K, temperature);
  if (const int rc = distill_check("concord_distill_bwd", a, dtype, temperature)) return rc;
  CONCORD_CHECK(ld_d >= V && ld_dloss >= 0, "concord_distill_bwd: leading dimension too small");
  if (M == 0) return CONCORD_OK;
  CONCORD_CHECK(dloss && stats && dlogits, "concord_distill_bwd: NULL argument");
  a.g = dloss, a.ldg = ld_dloss, a.stat = (float*)stats, a.dz = dlogits, a.lddz = ld_d;
  distill_split(a);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CONCORD_F32) distill_bwd<float>(a, st);
  else if (dtype == CONCORD_BF16) distill_bwd<BF16>(a, st);
  else distill_bwd<_Float16>(a, st);
  return launch_status("distill_bwd");
}
