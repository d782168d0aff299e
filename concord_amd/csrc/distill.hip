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
// exponentials), backward reads them again and writes the gradient: 166 us (5.0
// TB/s) and 295 us (5.6 TB/s: what the forward read last is still cached) at
// 8192 x 50257 bf16, where a copy moves 5.0 TB/s.  All statistics are fp32.  A
// row is one wave's (V <= 1024), one block's, or is split over several blocks
// when the rows are too few to fill the chip.
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
  float* stat;              // [M][4]: the row's largest logit and sum exp((z - it) / T), the same of the entries
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
// (an empty part has m = -inf, s = 0, and is passed over wherever parts meet: its
// factor would be 2^(-inf + inf), no number)
CONCORD_DEV float rel_exp2(float z, float m, float c) { return __builtin_amdgcn_exp2f((z - m) * c); }
CONCORD_DEV MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  // an empty side adds nothing
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

// A row's elements [0, n) as whole 16-byte chunks where its address allows, and
// the elements before and after them, at most VEC - 1 each, one a lane:
// edge(lane) is the lane's, or -1.
template <class T>
struct Span {
  static constexpr int VEC = 16 / (int)sizeof(T);
  int64_t head, body, n;   // elements before the first whole chunk; whole chunks
  CONCORD_DEV Span(const T* p, int64_t n_) : n(n_) {
    const int64_t mis = ((uintptr_t)p & 15) / sizeof(T);
    head = mis ? min<int64_t>(VEC - mis, n) : 0;
    body = (n - head) / VEC;
  }
  CONCORD_DEV int64_t edge(int lane) const {
    const int64_t tail = head + body * VEC + lane - VEC;
    return lane < head ? lane : lane >= VEC && lane < 2 * VEC && tail < n ? tail : -1;
  }
};

// statistics of z[0, n)
template <class T, int W>
CONCORD_DEV MaxSum row_stats(const T* z, int64_t n, float c) {
  constexpr int VEC = Span<T>::VEC, U = W == 1 ? 2 : 4, TH = W * 64;
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
  const int64_t edge = sp.edge(lane);
  const float last = edge >= 0 ? to_f32(z[edge]) : -INFINITY;
  const Chunk<T, VEC>* q = (const Chunk<T, VEC>*)(z + sp.head);
  for (int64_t k0 = 0; k0 < sp.body; k0 += U * TH) {
    // U chunks in flight; past the end the chunk before it again, not counted
    Chunk<T, VEC> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = q[min<int64_t>(k0 + u * TH + lane, sp.body - 1)];
    if (k0 + U * TH <= sp.body) {
      float v[U * VEC];
#pragma unroll
      for (int i = 0; i < U * VEC; ++i) v[i] = to_f32(r[i / VEC].v[i % VEC]);
      add(v, U * VEC);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = k0 + u * TH + lane < sp.body ? to_f32(r[u].v[i]) : -INFINITY;
        add(v, VEC);
      }
    }
  }
  add(&last, 1);
  return wave_join(a, c);
}

// One of the teacher's entries: its logit (-inf: left out, also where its index
// lies outside the vocabulary) and its place.
struct Entry {
  float t;
  int64_t i;
};
CONCORD_DEV Entry entry(const DistillArgs& a, int64_t row, int k) {
  const int64_t i = a.idx[row * a.ldi + k];
  const float t = a.t[row * a.ldt + k];
  return Entry{i >= 0 && i < a.V ? t : -INFINITY, i};
}
// a set of entries' maximum and sum (s = 0: none)
CONCORD_DEV MaxSum with_entry(MaxSum s, float t, float c) {
  return t == -INFINITY ? s : join(s, MaxSum{t, 1.0f}, c);
}
// an entry's part of the loss, p (log p - log q); q, t: the statistics of the
// logits and of the entries.  A probability that rounds to zero adds nothing.
template <class T>
CONCORD_DEV float entry_loss(const DistillArgs& a, const T* z, Entry e, MaxSum q, MaxSum t) {
  constexpr float LN2 = 0.69314718055994531f;
  const float p = e.t == -INFINITY ? 0.0f : rel_exp2(e.t, t.m, a.c) / t.s;
  if (p == 0.0f) return 0.0f;
  const float logs = __builtin_log2f(q.s) - __builtin_log2f(t.s);
  return p * (((e.t - t.m) - (to_f32(z[e.i]) - q.m)) * (a.c * LN2) + logs * LN2);
}
CONCORD_DEV void store_row(const DistillArgs& a, int64_t row, float sum, MaxSum q, MaxSum t) {
  a.loss[row] = t.s == 0.0f ? 0.0f : sum * (a.T * a.T);
  if (a.stat) *(float4*)(a.stat + 4 * row) = make_float4(q.m, q.s, t.m, t.s);
}

// the loss of a row from its statistics, by one wave
template <class T>
CONCORD_DEV void wave_loss(const DistillArgs& a, int64_t row, MaxSum q) {
  const int lane = threadIdx.x & 63;
  MaxSum t{-INFINITY, 0.0f};
  for (int k = lane; k < a.K; k += 64) t = with_entry(t, entry(a, row, k).t, a.c);
  t = wave_join(t, a.c);
  float sum = 0.0f;
  for (int k = lane; k < a.K; k += 64) sum += entry_loss(a, (const T*)a.z + row * a.ldz, entry(a, row, k), q, t);
  sum = wave_sum(sum);
  if (lane == 0) store_row(a, row, sum, q, t);
}

constexpr int kEntries = kTopMax / 256;   // of a thread of a block

// Statistics and loss of a row by a block.  The entries are read before the
// logits, so that only the last gather and two barriers follow the pass.
template <class T>
CONCORD_DEV void block_loss(const DistillArgs& a, int64_t row) {
  __shared__ float red[2][4][2], part[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const T* z = (const T*)a.z + row * a.ldz;
  Entry e[kEntries];
#pragma unroll
  for (int n = 0; n < kEntries; ++n) {
    e[n] = Entry{-INFINITY, 0};
    if (threadIdx.x + 256 * n < a.K) e[n] = entry(a, row, threadIdx.x + 256 * n);
  }
  const MaxSum q1 = row_stats<T, 4>(z, a.V, a.c);
  MaxSum t1{-INFINITY, 0.0f};
#pragma unroll
  for (int n = 0; n < kEntries; ++n) t1 = with_entry(t1, e[n].t, a.c);
  t1 = wave_join(t1, a.c);
  if (lane == 0) {
    *(float2*)red[0][wave] = make_float2(q1.m, q1.s);
    *(float2*)red[1][wave] = make_float2(t1.m, t1.s);
  }
  __syncthreads();
  MaxSum q{red[0][0][0], red[0][0][1]}, t{red[1][0][0], red[1][0][1]};
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    q = join(q, MaxSum{red[0][k][0], red[0][k][1]}, a.c);
    t = join(t, MaxSum{red[1][k][0], red[1][k][1]}, a.c);
  }
  float sum = 0.0f;
#pragma unroll
  for (int n = 0; n < kEntries; ++n) sum += entry_loss(a, z, e[n], q, t);
  sum = wave_sum(sum);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) store_row(a, row, ((part[0] + part[1]) + part[2]) + part[3], q, t);
}

// SPLIT: a block's part of a row
template <class T, int W, bool SPLIT>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillArgs a) {
  if constexpr (W == 1) {
    const int64_t row = (int64_t)blockIdx.x * 4 + Lanes<W>::wave();
    if (row < a.M) wave_loss<T>(a, row, row_stats<T, 1>((const T*)a.z + row * a.ldz, a.V, a.c));
  } else if constexpr (!SPLIT) {
    block_loss<T>(a, blockIdx.x);
  } else {
    __shared__ float red[4][2];
    const int64_t row = blockIdx.x / a.splits, v0 = (int64_t)(blockIdx.x % a.splits) * a.seg;
    const MaxSum s = row_stats<T, 4>((const T*)a.z + row * a.ldz + v0, min<int64_t>(a.seg, a.V - v0), a.c);
    if ((threadIdx.x & 63) == 0) *(float2*)red[threadIdx.x >> 6] = make_float2(s.m, s.s);
    __syncthreads();
    if (threadIdx.x == 0) {
      MaxSum t{red[0][0], red[0][1]};
      for (int k = 1; k < 4; ++k) t = join(t, MaxSum{red[k][0], red[k][1]}, a.c);
      *(float2*)(a.part + (int64_t)blockIdx.x * 2) = make_float2(t.m, t.s);
    }
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
  wave_loss<T>(a, row, wave_join(s, a.c));
}

// The gradient of [v0, v0 + n) of a row: q written first, then the entries
// that fall there, each place once, by the first entry that names it.
// (Measured at 8192 x 50257 bf16, K 64: entries read, and their logits gathered,
// ahead of the pass, and a search that leaves the sum to the entries that
// share a place, rows in segments of about 16 KB, so that the blocks in flight
// sweep memory in order: 344 -> 293 us.  With the last rows first 282, and the next
// forward, which finds the first rows cached, 175 -> 163.)
template <class T, int W>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a) {
  constexpr int TH = W * 64, VEC = Span<T>::VEC, NE = W == 1 ? 1 : kTopMax / TH;
  // per row: K places in [v0, v0 + n) or -1, padded to a multiple of 4, then their p
  extern __shared__ __attribute__((aligned(16))) int32_t entries[];
  const int lane = Lanes<W>::id(), slot = W == 1 ? Lanes<W>::wave() : 0, kp = (a.K + 3) & ~3;
  int32_t* place = entries + slot * 2 * kp;
  float* prob = (float*)(place + kp);
  // the last rows first: the forward read them last, and they are still cached
  const int64_t nth = W == 1 ? (int64_t)blockIdx.x * 4 + slot : blockIdx.x / a.splits, row = a.M - 1 - nth;
  if (W == 1 && nth >= a.M) return;   // (a wave for itself: no barrier below)
  const int64_t v0 = W == 1 ? 0 : (int64_t)(blockIdx.x % a.splits) * a.seg;
  const int64_t n = W == 1 ? a.V : min<int64_t>(a.seg, a.V - v0);
  const T* z = (const T*)a.z + row * a.ldz + v0;
  T* dz = (T*)a.dz + row * a.lddz + v0;
  const float4 st = *(const float4*)(a.stat + 4 * row);   // maximum and sum of the logits, of the entries
  const float g = a.g[row * a.ldg] * a.T;
  const bool none = g == 0.0f || st.w == 0.0f;
  const float m = st.x, inv = 1.0f / st.y, scale = none ? 0.0f : g * inv;
  // a block's lanes keep their entries: place here or -1, the teacher's logit,
  // the student's (a wave's rows are short and read them after the pass)
  int32_t at[NE];
  float et[NE], ez[NE];
  auto read = [&](int j, int k) {
    at[j] = -1;
    if (k < a.K) {
      const Entry e = entry(a, row, k);
      if (e.t != -INFINITY && e.i >= v0 && e.i < v0 + n && !none) at[j] = (int32_t)(e.i - v0);
      et[j] = e.t;
    }
  };
  auto put = [&](int j, int k) {
    if (k < a.K) {
      place[k] = at[j];
      prob[k] = at[j] >= 0 ? rel_exp2(et[j], st.z, a.c) / st.w : 0.0f;
    } else if (k < kp) {
      place[k] = -1;
    }
  };
  if (W > 1) {
#pragma unroll
    for (int j = 0; j < NE; ++j) read(j, lane + TH * j);
#pragma unroll
    for (int j = 0; j < NE; ++j) ez[j] = at[j] >= 0 ? to_f32(z[at[j]]) : 0.0f;
  }
  auto grad = [&](float v) { return none ? 0.0f : scale * rel_exp2(v, m, a.c); };
  const Span<T> sp(z, n);
  if (((uintptr_t)dz & 15) == ((uintptr_t)z & 15)) {
    constexpr int U = 4;
    const int64_t edge = sp.edge(lane);
    const float last = edge >= 0 ? to_f32(z[edge]) : 0.0f;
    const Chunk<T, VEC>* q = (const Chunk<T, VEC>*)(z + sp.head);
    Chunk<T, VEC>* o = (Chunk<T, VEC>*)(dz + sp.head);
    for (int64_t k0 = lane; k0 < sp.body; k0 += U * TH) {
      Chunk<T, VEC> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = q[min<int64_t>(k0 + u * TH, sp.body - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Chunk<T, VEC> w;
#pragma unroll
        for (int i = 0; i < VEC; ++i) w.v[i] = from_f32<T>(grad(to_f32(r[u].v[i])));
        if (k0 + u * TH < sp.body) store_stream(&o[k0 + u * TH], w);
      }
    }
    if (edge >= 0) dz[edge] = from_f32<T>(grad(last));
  } else {
    for (int64_t k = lane; k < n; k += TH) dz[k] = from_f32<T>(grad(to_f32(z[k])));
  }
  if (W > 1) {
#pragma unroll
    for (int j = 0; j < NE; ++j) put(j, lane + TH * j);
  } else {
    for (int k = lane; k < kp; k += TH) read(0, k), put(0, k);
  }
  // the stores above come before those below, also of other threads
  __threadfence_block();
  if (W > 1) __syncthreads();
  auto fix = [&](int k, int32_t i, float zi) {
    int same = 0;
#pragma unroll 4
    for (int b = 0; b < kp; b += 4) {
      const int4 w = *(const int4*)(place + b);
      same += (w.x == i) + (w.y == i) + (w.z == i) + (w.w == i);
    }
    float p = prob[k];
    bool first = true;
    if (same > 1) {   // one place named more than once: the first adds them up
      p = 0.0f;
      for (int b = 0; b < a.K; ++b)
        if (place[b] == i) {
          p += prob[b];
          first = first && b >= k;
        }
    }
    if (first) dz[i] = from_f32<T>(g * (rel_exp2(zi, m, a.c) * inv - p));
  };
  if (W > 1) {
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (at[j] >= 0) fix(lane + TH * j, at[j], ez[j]);
  } else {
    for (int k = lane; k < a.K; k += TH)
      if (place[k] >= 0) fix(k, place[k], to_f32(z[place[k]]));
  }
}

// ---- host -------------------------------------------------------------------
// Blocks a row is split over in the forward: none while the rows alone give 1024 blocks; at
// least 4096 elements a block.
static int distill_splits(int64_t M, int64_t V) {
  if (V <= kWaveRow || M >= 1024) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(1024, M), V / 4096));
}
static void distill_split(DistillArgs& a, int splits) {
  a.splits = splits;
  a.seg = cdiv(cdiv(a.V, a.splits), 8) * 8;
  a.splits = (int)cdiv(a.V, a.seg);
}
static bool distill_fits(const DistillArgs& a) { return grid_fits(a.M * a.splits, 256); }

template <class T>
static void distill_fwd(const DistillArgs& a, hipStream_t st) {
  if (a.V <= kWaveRow)
    hipLaunchKernelGGL((distill_fwd_kernel<T, 1, false>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 0, st, a);
  else if (a.splits == 1)
    hipLaunchKernelGGL((distill_fwd_kernel<T, 4, false>), dim3((unsigned)a.M), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((distill_fwd_kernel<T, 4, true>), dim3((unsigned)(a.M * a.splits)), dim3(256), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 0, st, a);
}
template <class T>
static void distill_bwd(const DistillArgs& a, hipStream_t st) {
  const size_t lds = (size_t)((a.K + 3) & ~3) * 8;   // a row's entries
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
  CONCORD_CHECK(((uintptr_t)stats & 15) == 0, "concord_distill_fwd: stats must lie on 16 bytes");
  a.loss = loss, a.stat = stats, a.part = (float*)workspace;
  distill_split(a, distill_splits(M, V));
  CONCORD_CHECK(distill_fits(a), "concord_distill_fwd: bad size");
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
  CONCORD_CHECK(dloss && stats && dlogits && ((uintptr_t)stats & 15) == 0,
                "concord_distill_bwd: NULL argument or stats not on 16 bytes");
  a.g = dloss, a.ldg = ld_dloss, a.stat = (float*)stats, a.dz = dlogits, a.lddz = ld_d;
  // (segments of about 16 KB: forward and backward of 8192 x 50257 bf16 444 us; of 24 KB 451)
  distill_split(a, V <= kWaveRow ? 1 : (int)std::max<int64_t>(1, V * (dtype == CONCORD_F32 ? 4 : 2) / 16384));
  CONCORD_CHECK(distill_fits(a), "concord_distill_bwd: bad size");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CONCORD_F32) distill_bwd<float>(a, st);
  else if (dtype == CONCORD_BF16) distill_bwd<BF16>(a, st);
  else distill_bwd<_Float16>(a, st);
  return launch_status("distill_bwd");
}
