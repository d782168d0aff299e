// layernorm.hip -- layer norm of the rows of an activation, forward and
// backward, with the reduction of the weight's and bias's gradients.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
//   y  = h w + b
//   g  = dy w;  dx = r (g - mean(g) - h mean(g h))
//   dw = sum over rows of dy h;  db = sum over rows of dy
//
// Both passes are bound by memory: a row is read once, kept in registers, and
// written once.  A row belongs to W waves (or 16 lanes of one) whose threads hold
// E elements each at fixed columns, so the weight, the bias and the column sums of
// dw and db stay in registers over all rows that a workgroup takes.  All sums
// are fp32.  Kernel times in a trace, 32768 x 4096 bf16: forward 97 us (5.5 TB/s),
// backward 155 us (5.2 TB/s, its second kernel included), where a 1 GiB copy moves
// 5.0 TB/s; 16384 x 384: 7.8 and 15.9 us, near the cost of the launches and their
// latencies.
#include "elem.h"

namespace concord {

struct LnArgs {
  const void* x;
  const void* dy;     // backward
  void* out;          // y, or dx
  int64_t ldx, ldy, ldo;
  const void* w;      // NULL: ones
  const void* b;      // NULL: zeros
  int wtype;
  int64_t M, C;
  float eps;
  float* mean;        // forward: written unless NULL; backward: read
  float* rstd;
  float* part;        // backward: [blocks][2][C] partial dw, db, or NULL
};

// Threads of one row and the columns they hold: chunk i of thread t is the
// VEC columns from (i TH + t) VEC, TH = W L threads: W waves (L = 64), or 16
// lanes of one (L = 16, W = 1) where a row is that short.
template <class T, int VEC, int E, int W, int L>
struct LnRow {
  static constexpr int NV = E / VEC, TH = W * L, SLOTS = W == 1 ? 256 / L : 1, THREADS = W == 1 ? 256 : W * 64;
  // rows a lane takes at once where a wave has rows of its own: their loads and
  // sums overlap, and a short row alone has too few bytes in flight
  static constexpr int R = W > 1 ? 1 : E == 8 ? 4 : 2;
  // with one row at a time the next row's loads are issued before this row's
  // sums; not in a block of 16 waves, whose 128 registers a thread hold one row
  static constexpr bool AHEAD = W > 1 && W < 16;
  // sum over the row's lanes of a wave
  static CONCORD_DEV float sum(float v) { return L == 16 ? row16_sum(v) : wave_sum(v); }
  typedef Chunk<T, VEC> V;
  // the thread's place among its row's threads, and its row in the block
  static CONCORD_DEV int lane() { return W == 1 ? threadIdx.x & (L - 1) : threadIdx.x; }
  static CONCORD_DEV int slot() {
    if (W > 1) return 0;
    return L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x / L;
  }
  static CONCORD_DEV int col(int i) { return (i * TH + lane()) * VEC; }
  // raw row: columns at or past C stay zero (VEC divides C)
  static CONCORD_DEV void load(V (&r)[NV], const void* p, int64_t row, int64_t ld, int C) {
    const T* q = (const T*)p + row * ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      r[i] = V{};
      if (col(i) < C) r[i] = *(const V*)(q + col(i));
    }
  }
  static CONCORD_DEV void store(void* p, int64_t row, int64_t ld, int C, const float (&v)[E]) {
    T* q = (T*)p + row * ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      V r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = from_f32<T>(v[i * VEC + e]);
      if (col(i) < C) store_stream((V*)(q + col(i)), r);
    }
  }
  template <class P>
  static CONCORD_DEV void vector_of(float (&v)[E], const P* p, int C) {
    constexpr int PV = VEC * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : VEC;
#pragma unroll
    for (int i = 0; i < E; i += PV) {
      const int c = col(i / VEC) + i % VEC;
      const Chunk<P, PV> w = *(const Chunk<P, PV>*)(p + (c < C ? c : 0));
#pragma unroll
      for (int e = 0; e < PV; ++e) v[i + e] = to_f32(w.v[e]);
    }
  }
  // the weight or the bias at the thread's columns (any value past C)
  static CONCORD_DEV void vector(float (&v)[E], const void* p, int dtype, int C, float none) {
    if (!p) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = none;
    } else if (dtype == CONCORD_F32) {
      vector_of(v, (const float*)p, C);
    } else if (dtype == CONCORD_BF16) {
      vector_of(v, (const BF16*)p, C);
    } else {
      vector_of(v, (const _Float16*)p, C);
    }
  }
};

template <class T, int VEC, int E, int W, int L>
__global__ __launch_bounds__((LnRow<T, VEC, E, W, L>::THREADS)) void ln_fwd_kernel(LnArgs a) {
  typedef LnRow<T, VEC, E, W, L> R;
  typedef typename R::V V;
  constexpr int NV = R::NV;
  __shared__ float red[2][W][2];
  const int C = (int)a.C, wave = threadIdx.x >> 6;
  float w[E], b[E];
  R::vector(w, a.w, a.wtype, C, 1.0f);
  R::vector(b, a.b, a.wtype, C, 0.0f);
  // columns each wave of the row holds: the weight of its mean among the waves'
  float n[W], inv_n[W];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    n[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) n[k] += (float)min(max(C - (i * W + k) * L * VEC, 0), L * VEC);
    inv_n[k] = n[k] > 0.0f ? 1.0f / n[k] : 0.0f;
  }
  float inv_own = inv_n[0];
#pragma unroll
  for (int k = 1; k < W; ++k) inv_own = wave == k ? inv_n[k] : inv_own;
  const float inv_c = 1.0f / (float)C;
  constexpr int NR = R::R;
  const int64_t step = (int64_t)gridDim.x * R::SLOTS * NR;
  int64_t row = ((int64_t)blockIdx.x * R::SLOTS + R::slot()) * NR;
  V raw[NR][NV];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (NR == 1 || r0 + r < a.M) R::load(raw[r], a.x, r0 + r, a.ldx, C);
  };
  if (R::AHEAD && row < a.M) fetch(row);
  // (a block with W > 1 takes one row at a time: its waves leave together)
  for (int par = 0; row < a.M; row += step, par ^= 1) {
    float x[NR][E];
    if (!R::AHEAD) fetch(row);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < E; ++i) x[r][i] = to_f32(raw[r][i / VEC].v[i % VEC]);
    if (R::AHEAD && row + step < a.M) fetch(row + step);
    // mean, then the squares about it; over several waves each about its own
    // mean, joined as M2 = sum M2_w + n_w (mean_w - mean)^2
    float s[NR], mean[NR], m2[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) s[r] += x[r][i];
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s[r] = R::sum(s[r]);
      mean[r] = s[r] * inv_own;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m2[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float d = x[r][i] - mean[r];
        m2[r] = R::col(i / VEC) < C ? __builtin_fmaf(d, d, m2[r]) : m2[r];
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) m2[r] = R::sum(m2[r]);
    if (W > 1) {
      if ((threadIdx.x & 63) == 0) {
        red[par][wave][0] = s[0];
        red[par][wave][1] = m2[0];
      }
      __syncthreads();
      float tot = 0.0f, tot2 = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) tot += red[par][k][0];
      const float all = tot * inv_c;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float d = red[par][k][0] * inv_n[k] - all;
        tot2 += __builtin_fmaf(n[k] * d, d, red[par][k][1]);
      }
      mean[0] = all;
      m2[0] = tot2;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float rstd = 1.0f / __builtin_sqrtf(m2[r] * inv_c + a.eps);
      float y[E];
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] = __builtin_fmaf((x[r][i] - mean[r]) * rstd, w[i], b[i]);
      if (NR == 1 || row + r < a.M) {
        R::store(a.out, row + r, a.ldo, C, y);
        if (a.mean && R::lane() == 0) {
          a.mean[row + r] = mean[r];
          a.rstd[row + r] = rstd;
        }
      }
    }
  }
}

template <class T, int VEC, int E, int W, int L>
__global__ __launch_bounds__((LnRow<T, VEC, E, W, L>::THREADS)) void ln_bwd_kernel(LnArgs a) {
  typedef LnRow<T, VEC, E, W, L> R;
  typedef typename R::V V;
  constexpr int NV = R::NV;
  __shared__ float red[2][W][2];
  __shared__ float cols[W == 1 ? R::SLOTS : 1][W == 1 ? L * E : 1];
  const int C = (int)a.C, wave = threadIdx.x >> 6;
  float w[E], dw[E], db[E];
  R::vector(w, a.w, a.wtype, C, 1.0f);
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.0f;
  const float inv_c = 1.0f / (float)C;
  constexpr int NR = R::R;
  const int64_t step = (int64_t)gridDim.x * R::SLOTS * NR;
  int64_t row = ((int64_t)blockIdx.x * R::SLOTS + R::slot()) * NR;
  V rx[NR][NV], ry[NR][NV];
  float mean[NR], rstd[NR];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      // (no row there: the first again, its dy taken as zeros)
      // the last rows first: their producer wrote them last, and they are still cached
      const int64_t at = a.M - 1 - (NR == 1 || r0 + r < a.M ? r0 + r : r0);
      R::load(rx[r], a.x, at, a.ldx, C);
      R::load(ry[r], a.dy, at, a.ldy, C);
      mean[r] = a.mean[at];
      rstd[r] = a.rstd[at];
    }
  };
  if (R::AHEAD && row < a.M) fetch(row);
  for (int par = 0; row < a.M; row += step, par ^= 1) {
    if (!R::AHEAD) fetch(row);
    float h[NR][E], dy[NR][E], s1[NR], s2[NR], rs[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      rs[r] = rstd[r];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        // a column past C has dy = 0, so it adds nothing below
        h[r][i] = (to_f32(rx[r][i / VEC].v[i % VEC]) - mean[r]) * rstd[r];
        dy[r][i] = NR == 1 || row + r < a.M ? to_f32(ry[r][i / VEC].v[i % VEC]) : 0.0f;
      }
    }
    if (R::AHEAD && row + step < a.M) fetch(row + step);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s1[r] = s2[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool in = R::col(i / VEC) < C;
        const float hy = in ? dy[r][i] * h[r][i] : 0.0f;
        dw[i] += hy;
        db[i] += dy[r][i];
        s1[r] = in ? __builtin_fmaf(dy[r][i], w[i], s1[r]) : s1[r];
        s2[r] = in ? __builtin_fmaf(hy, w[i], s2[r]) : s2[r];
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s1[r] = R::sum(s1[r]);
      s2[r] = R::sum(s2[r]);
    }
    if (W > 1) {
      if ((threadIdx.x & 63) == 0) {
        red[par][wave][0] = s1[0];
        red[par][wave][1] = s2[0];
      }
      __syncthreads();
      s1[0] = s2[0] = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        s1[0] += red[par][k][0];
        s2[0] += red[par][k][1];
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float m1 = s1[r] * inv_c, m2 = s2[r] * inv_c;
      float dx[E];
#pragma unroll
      for (int i = 0; i < E; ++i) dx[i] = rs[r] * (__builtin_fmaf(dy[r][i], w[i], -m1) - h[r][i] * m2);
      if (NR == 1 || row + r < a.M) R::store(a.out, a.M - 1 - (row + r), a.ldo, C, dx);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
  if (W == 1) {
    // the block's rows hold the same columns: added in their order
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) cols[R::slot()][R::col(i / VEC) + i % VEC] = half ? db[i] : dw[i];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += 256) {
        float v = cols[0][c];
#pragma unroll
        for (int k = 1; k < R::SLOTS; ++k) v += cols[k][c];
        part[half * a.C + c] = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = R::col(i / VEC) + i % VEC;
      if (c < C) {
        part[c] = dw[i];
        part[a.C + c] = db[i];
      }
    }
  }
}

// Rows longer than a block holds in registers: a block of 16 waves reads a row
// once for each of its sums (from the second time on out of the caches).
template <class T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LnArgs a) {
  __shared__ float red[2][16];
  const int wave = threadIdx.x >> 6;
  auto total = [&](float v, int k) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[k][wave] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[k][i];
    return t;
  };
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    T* y = (T*)a.out + row * a.ldo;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < a.C; c += 1024) s += to_f32(x[c]);
    const float mean = total(s, 0) / (float)a.C;
    float m2 = 0.0f;
    for (int64_t c = threadIdx.x; c < a.C; c += 1024) {
      const float d = to_f32(x[c]) - mean;
      m2 = __builtin_fmaf(d, d, m2);
    }
    const float rstd = 1.0f / __builtin_sqrtf(total(m2, 1) / (float)a.C + a.eps);
    for (int64_t c = threadIdx.x; c < a.C; c += 1024)
      y[c] = from_f32<T>(__builtin_fmaf((to_f32(x[c]) - mean) * rstd, a.w ? load_any(a.w, a.wtype, c) : 1.0f,
                                        a.b ? load_any(a.b, a.wtype, c) : 0.0f));
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LnArgs a) {
  __shared__ float red[2][2][16];
  const int wave = threadIdx.x >> 6;
  int par = 0;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, par ^= 1) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* dy = (const T*)a.dy + row * a.ldy;
    T* dx = (T*)a.out + row * a.ldo;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < a.C; c += 1024) {
      const float g = to_f32(dy[c]) * (a.w ? load_any(a.w, a.wtype, c) : 1.0f);
      s1 += g;
      s2 = __builtin_fmaf(g, (to_f32(x[c]) - mean) * rstd, s2);
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if ((threadIdx.x & 63) == 0) {
      red[par][0][wave] = s1;
      red[par][1][wave] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s1 += red[par][0][i];
      s2 += red[par][1][i];
    }
    const float m1 = s1 / (float)a.C, m2 = s2 / (float)a.C;
    for (int64_t c = threadIdx.x; c < a.C; c += 1024) {
      const float g = to_f32(dy[c]) * (a.w ? load_any(a.w, a.wtype, c) : 1.0f);
      dx[c] = from_f32<T>(rstd * ((g - m1) - (to_f32(x[c]) - mean) * rstd * m2));
    }
  }
}

// column partials of dw and db for rows blockIdx.y, + gridDim.y, ... (long rows)
template <class T>
__global__ __launch_bounds__(256) void ln_cols_kernel(LnArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    const float dy = to_f32(((const T*)a.dy)[row * a.ldy + c]);
    dw = __builtin_fmaf(dy, (to_f32(((const T*)a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row], dw);
    db += dy;
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.C;
  part[c] = dw;
  part[a.C + c] = db;
}

// dw and db from the blocks' partials: 64 columns a block, each wave a
// sixteenth of the partial rows in order, then the waves' sums in order.
__global__ __launch_bounds__(1024) void ln_cols_sum_kernel(const float* __restrict__ part, int nb, int64_t C,
                                                           void* dw, void* db, int wtype) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;   // of the 2 C columns
  float v = 0.0f;
  if (c < 2 * C) {
    const int per = (nb + 15) / 16, end = min(nb, (wave + 1) * per);
    int r = wave * per;
    for (; r + 8 <= end; r += 8) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = part[(int64_t)(r + i) * 2 * C + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += t[i];
    }
    for (; r < end; ++r) v += part[(int64_t)r * 2 * C + c];
  }
  s[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < 2 * C) {
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += s[k][lane];
    if (c < C) {
      if (dw) store_any(dw, wtype, c, v);
    } else if (db) {
      store_any(db, wtype, c - C, v);
    }
  }
}

// ---- host -------------------------------------------------------------------
// waves of a row (W), by its length alone: a thread holds 8 or 16 elements;
// 0: longer than a block holds
static int ln_waves(int64_t C) { return C <= 1024 ? 1 : C <= 4096 ? 4 : C <= 8192 ? 8 : C <= 16384 ? 16 : 0; }

// rows a block takes at once (LnRow::SLOTS * LnRow::R)
static int64_t ln_block_rows(int64_t C) { return C <= 128 ? 64 : C <= 512 ? 16 : C <= 1024 ? 8 : 1; }

// blocks of the backward, each with one partial row of dw and db
static int64_t ln_bwd_blocks(int64_t M, int64_t C) {
  const int W = ln_waves(C);
  if (W == 0) return std::min<int64_t>(M, 256);
  return std::min<int64_t>(cdiv(M, ln_block_rows(C)), W >= 8 ? 256 : 512);
}

static size_t elem_size(int dtype) { return dtype == CONCORD_F32 ? 4 : 2; }

static bool chunked(const void* p, int64_t ld, size_t es) {
  return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0;
}

template <class T, int VEC, int E, int W, int L>
static void ln_launch(bool bwd, const LnArgs& a, unsigned grid, hipStream_t st) {
  const dim3 th(LnRow<T, VEC, E, W, L>::THREADS);
  if (!bwd) hipLaunchKernelGGL((ln_fwd_kernel<T, VEC, E, W, L>), dim3(grid), th, 0, st, a);
  else hipLaunchKernelGGL((ln_bwd_kernel<T, VEC, E, W, L>), dim3(grid), th, 0, st, a);
}
template <class T, int VEC>
static void ln_rows(bool bwd, const LnArgs& a, unsigned grid, hipStream_t st) {
  if (a.C <= 128) ln_launch<T, VEC, 8, 1, 16>(bwd, a, grid, st);
  else if (a.C <= 512) ln_launch<T, VEC, 8, 1, 64>(bwd, a, grid, st);
  else if (a.C <= 1024) ln_launch<T, VEC, 16, 1, 64>(bwd, a, grid, st);
  else if (a.C <= 2048) ln_launch<T, VEC, 8, 4, 64>(bwd, a, grid, st);
  else if (a.C <= 4096) ln_launch<T, VEC, 16, 4, 64>(bwd, a, grid, st);
  else if (a.C <= 8192) ln_launch<T, VEC, 16, 8, 64>(bwd, a, grid, st);
  else ln_launch<T, VEC, 16, 16, 64>(bwd, a, grid, st);
}

template <class T>
static void ln_pass(bool bwd, const LnArgs& a, hipStream_t st) {
  const int W = ln_waves(a.C);
  const size_t es = sizeof(T);
  const bool vec = a.C % (16 / es) == 0 && chunked(a.x, a.ldx, es) && chunked(a.out, a.ldo, es) &&
                   (!bwd || chunked(a.dy, a.ldy, es)) && (((uintptr_t)a.w | (uintptr_t)a.b) & 15) == 0;
  const unsigned grid =
      (unsigned)(bwd ? ln_bwd_blocks(a.M, a.C) : std::min<int64_t>(cdiv(a.M, ln_block_rows(a.C)), 2048));
  constexpr int V = 16 / (int)sizeof(T);
  if (W == 0) {
    if (!bwd) hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3(std::min<int64_t>(a.M, 1024)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((ln_bwd_long_kernel<T>), dim3(std::min<int64_t>(a.M, 1024)), dim3(1024), 0, st, a);
    if (bwd && a.part)
      hipLaunchKernelGGL((ln_cols_kernel<T>), dim3((unsigned)cdiv(a.C, 256), grid), dim3(256), 0, st, a);
  } else if (vec) {
    ln_rows<T, V>(bwd, a, grid, st);
  } else {
    ln_rows<T, 1>(bwd, a, grid, st);
  }
}

static void ln_run(bool bwd, int dtype, const LnArgs& a, hipStream_t st) {
  if (dtype == CONCORD_F32) ln_pass<float>(bwd, a, st);
  else if (dtype == CONCORD_BF16) ln_pass<BF16>(bwd, a, st);
  else ln_pass<_Float16>(bwd, a, st);
}

static bool dtype_ok(int t) { return t == CONCORD_F32 || t == CONCORD_BF16 || t == CONCORD_F16; }

}  // namespace concord

using namespace concord;

extern "C" int concord_layernorm_fwd(const void* x, int64_t ld_x, int dtype, const void* weight, const void* bias,
                                     int wdtype, int64_t M, int64_t C, float eps, void* y, int64_t ld_y, float* mean,
                                     float* rstd, void* stream) {
  CONCORD_CHECK(M >= 0 && C >= 1 && M < (1LL << 40) && C < (1LL << 30), "concord_layernorm_fwd: bad size");
  CONCORD_CHECK(dtype_ok(dtype) && dtype_ok(wdtype), "concord_layernorm_fwd: bad type");
  CONCORD_CHECK(ld_x >= C && ld_y >= C, "concord_layernorm_fwd: leading dimension < C");
  CONCORD_CHECK(!mean == !rstd, "concord_layernorm_fwd: mean without rstd");
  if (M == 0) return CONCORD_OK;
  CONCORD_CHECK(x && y, "concord_layernorm_fwd: NULL argument");
  LnArgs a{};
  a.x = x, a.ldx = ld_x, a.out = y, a.ldo = ld_y, a.w = weight, a.b = bias, a.wtype = wdtype;
  a.M = M, a.C = C, a.eps = eps, a.mean = mean, a.rstd = rstd;
  ln_run(false, dtype, a, (hipStream_t)stream);
  return launch_status("layernorm_fwd");
}

extern "C" size_t concord_layernorm_workspace_bytes(int64_t M, int64_t C) {
  if (M < 1 || C < 1) return 0;
  return (size_t)ln_bwd_blocks(M, C) * 2 * (size_t)C * sizeof(float);
}

extern "C" int concord_layernorm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype,
                                     const void* weight, int wdtype, const float* mean, const float* rstd, int64_t M,
                                     int64_t C, void* dx, int64_t ld_dx, void* dweight, void* dbias, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  CONCORD_CHECK(M >= 0 && C >= 1 && M < (1LL << 40) && C < (1LL << 30), "concord_layernorm_bwd: bad size");
  CONCORD_CHECK(dtype_ok(dtype) && dtype_ok(wdtype), "concord_layernorm_bwd: bad type");
  CONCORD_CHECK(ld_x >= C && ld_dy >= C && ld_dx >= C, "concord_layernorm_bwd: leading dimension < C");
  CONCORD_CHECK(M == 0 || (dy && x && dx && mean && rstd), "concord_layernorm_bwd: NULL argument");
  hipStream_t st = (hipStream_t)stream;
  const bool cols = dweight || dbias;
  CONCORD_CHECK(!cols || grid_fits(cdiv(2 * C, 64), 1024), "concord_layernorm_bwd: too many columns for their sums");
  if (M > 0) {
    if (cols && (!workspace || workspace_bytes < concord_layernorm_workspace_bytes(M, C))) {
      set_error("concord_layernorm_bwd: workspace of %zu bytes needed", concord_layernorm_workspace_bytes(M, C));
      return CONCORD_EWORKSPACE;
    }
    LnArgs a{};
    a.x = x, a.ldx = ld_x, a.dy = dy, a.ldy = ld_dy, a.out = dx, a.ldo = ld_dx, a.w = weight, a.wtype = wdtype;
    a.M = M, a.C = C, a.mean = (float*)mean, a.rstd = (float*)rstd, a.part = cols ? (float*)workspace : nullptr;
    ln_run(true, dtype, a, st);
  }
  if (cols)   // (an empty batch: sums over no partials, zero)
    hipLaunchKernelGGL(ln_cols_sum_kernel, dim3((unsigned)cdiv(2 * C, 64)), dim3(1024), 0, st,
                       (const float*)workspace, M > 0 ? (int)ln_bwd_blocks(M, C) : 0, C, dweight, dbias, wdtype);
  return launch_status("layernorm_bwd");
}
