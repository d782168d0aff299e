// qk_rope.hip -- the norm of each head's query and key with the rotation by
// position in the same pass, forward and backward.
//
// A row x of D elements at position p, pairs i < R / 2 of its first R elements:
//   r = 1 / sqrt(mean(x^2) + eps),  h = x r,  u = h w
//   y = u with pair i (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = p base^(-2 i / R)
// backward, from dy:
//   du = dy rotated by -t,  g = du w,  dx = r (g - h mean(g h)),  dw = sum over rows of du h
//
// Bound by memory: every row is read once and written once, its statistics are
// formed again in the backward rather than kept.  A row belongs to L adjacent
// lanes, 8 or 16 elements each, that hold both elements of their pairs, so the rotation
// exchanges nothing; a lane's angles depend on the token alone and serve all heads
// that it takes.  Angles are formed in 64 bits (a far position times a frequency
// loses its fraction in 32) and reduced to an eighth of a turn before the sine and
// cosine, which are 32-bit polynomials.
//
// Kernel times, 32768 tokens of 40 heads of 128, bf16: forward 116 to 130 us (5.8 to 5.2
// TB/s), backward 196 to 213 us (5.1 to 4.7; the longer ones with positions given), where a
// 1 GiB copy moves 5.1 TB/s; fp32 252 and 378 us (5.3); 64 tokens 4.3 us, a chain of a
// position's load, an exponential and the row.
#include "elem.h"

namespace concord {

struct QkArgs {
  const void* x[2];         // q and k; backward too
  const void* dy[2];        // backward
  void* out[2];             // y, or dx: [T][H][D], rows adjacent
  int64_t x_t[2], x_h[2], dy_t[2], dy_h[2];
  const void* w[2];         // NULL: ones
  int wtype;
  const void* pos;          // NULL: the token's place in its sequence
  int pos64;
  uint32_t T, seq, pos_seq; // tokens; tokens of a sequence; period of pos
  int H[2];
  int D, R, adjacent;
  int heads[2];             // heads of a slice
  uint32_t blocks[2];       // blocks of a slice
  uint32_t k_at;            // first block of k's slices
  float eps;
  double log2_base;
  float* part[2];           // backward: [blocks of q's or k's slices][D] partial dw, or NULL
};

// a lane's V pairs: elements (a + j, b + j), or (a + 2 j, a + 2 j + 1) where pairs are adjacent
struct QkLane {
  int a, b;
  bool in, turned;
};
template <int V>
CONCORD_DEV QkLane qk_lane(int l, int D, int R, bool adjacent) {
  QkLane s;
  s.in = l * 2 * V < D;
  s.turned = l * 2 * V < R;
  if (adjacent) s.a = l * 2 * V, s.b = s.a + V;
  else if (s.turned) s.a = l * V, s.b = R / 2 + l * V;
  else s.a = R + (l * 2 * V - R) / 2, s.b = s.a + (D - R) / 2;
  return s;
}

// cosine and sine of pi/2 times a quarter-turn count given in 64 bits.  To the
// nearest quarter turn, then Taylor polynomials of theta = pi/2 (turn - nearest),
// |theta| <= pi/4: the first terms left out are at most theta^12 / 12! = 2^-33 of 1 (cosine) and
// theta^10 / 11! = 2^-28.7 of theta (sine), where a rounding is 2^-24.
CONCORD_DEV void sincos_quarters(double quarters, float& c, float& s) {
  const double n = __builtin_rint(quarters);
  const float th = (float)((quarters - n) * 1.5707963267948966);
  const int q = (int)(int64_t)n & 3;
  const float t = th * th;
  float cs = __builtin_fmaf(t, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  cs = __builtin_fmaf(t, cs, -1.0f / 720.0f);
  cs = __builtin_fmaf(t, cs, 1.0f / 24.0f);
  cs = __builtin_fmaf(t, cs, -0.5f);
  cs = __builtin_fmaf(t, cs, 1.0f);
  float sn = __builtin_fmaf(t, 1.0f / 362880.0f, -1.0f / 5040.0f);
  sn = __builtin_fmaf(t, sn, 1.0f / 120.0f);
  sn = __builtin_fmaf(t, sn, -1.0f / 6.0f);
  sn = __builtin_fmaf(t * th, sn, th);
  const float u = q & 1 ? sn : cs, v = q & 1 ? cs : sn;
  c = (q + 1) & 2 ? -u : u;
  s = q & 2 ? -v : v;
}

// sum over the group of L lanes, to each: lanes 1 and 2 apart, the mirrored half row, the
// mirrored row, the other row
template <int L>
CONCORD_DEV float group_sum(float v) {
#define CONCORD_DPP_ADD(ctrl) \
  v = __fadd_rn(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true)))
  if (L > 1) CONCORD_DPP_ADD(0xB1);
  if (L > 2) CONCORD_DPP_ADD(0x4E);
  if (L > 4) CONCORD_DPP_ADD(0x141);
  if (L > 8) CONCORD_DPP_ADD(0x140);
#undef CONCORD_DPP_ADD
  if (L > 16) v += __shfl_xor(v, 16, 64);
  return v;
}

// A mean square below 2^-96, whose terms 32 bits may have lost, or infinite (or NaN).  Its
// row is taken times k = 2^48 or 2^-48, and the squares of that times k: they lie in range
// for every row there is, and every factor stays a normal number.  (The test costs nothing
// that shows: forward of 32768 x 40 heads of 128 130 us with it and without, backward 213.)
CONCORD_DEV bool out_of_range(float square) { return __float_as_uint(square) - 0x0F800000u >= 0x7F800000u - 0x0F800000u; }

// a lane's share of a row; a lane behind the row's end holds the row's first elements
// and stores nothing
template <class T, int V>
struct QkRow {
  typedef Chunk<T, V> C;
  C a, b;
  CONCORD_DEV void load(const T* p, const QkLane& s) {
    a = *(const C*)(p + (s.in ? s.a : 0));
    b = *(const C*)(p + (s.in ? s.b : 0));
  }
  CONCORD_DEV void get(float (&v)[2 * V], const QkLane& s) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = s.in ? to_f32(a.v[j]) : 0.0f, v[V + j] = s.in ? to_f32(b.v[j]) : 0.0f;
  }
  template <bool PAST>
  CONCORD_DEV void store(T* p, const QkLane& s, const float (&v)[2 * V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = from_f32<T>(v[j]), b.v[j] = from_f32<T>(v[V + j]);
    if (!s.in) return;
    if constexpr (PAST) {
      store_stream((C*)(p + s.a), a);
      store_stream((C*)(p + s.b), b);
    } else {
      *(C*)(p + s.a) = a;
      *(C*)(p + s.b) = b;
    }
  }
};

// v's pairs turned by +t (dir = 1) or -t (dir = -1)
template <bool ADJ, int V>
CONCORD_DEV void turn(float (&v)[2 * V], const float (&c)[V], const float (&s)[V], float dir) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int ia = ADJ ? 2 * j : j, ib = ADJ ? 2 * j + 1 : V + j;
    const float a = v[ia], b = v[ib], sn = s[j] * dir;
    v[ia] = __builtin_fmaf(a, c[j], -(b * sn));
    v[ib] = __builtin_fmaf(a, sn, b * c[j]);
  }
}

// Blocks of a slice of the heads (q's slices, then k's) share the tokens: a group of L
// lanes takes a token's heads of the slice, U at a time.
template <class T, int V, int L, bool ADJ, bool BWD, bool PAST>
__global__ __launch_bounds__(256) void qk_kernel(QkArgs a) {
  constexpr int G = 256 / L, U = BWD ? 2 : 4, E = 2 * V;
  __shared__ float sums[BWD ? G : 1][BWD ? L * E : 1];
  const int l = threadIdx.x & (L - 1), g = threadIdx.x / L;
  const int which = blockIdx.x >= a.k_at;
  const uint32_t bid = blockIdx.x - (which ? a.k_at : 0), slice = bid / a.blocks[which], nb = a.blocks[which];
  const int H = a.H[which], h0 = (int)slice * a.heads[which], h1 = min(h0 + a.heads[which], H);
  const QkLane s = qk_lane<V>(l, a.D, a.R, ADJ);
  const T *x0 = (const T*)a.x[which], *y0 = (const T*)a.dy[which];
  const int64_t x_t = a.x_t[which], x_h = a.x_h[which], dy_t = a.dy_t[which], dy_h = a.dy_h[which];
  float w[E], dw[E];
#pragma unroll
  for (int j = 0; j < E; ++j) dw[j] = 0.0f, w[j] = 1.0f;
  if (const void* wp = a.w[which]) {
#pragma unroll
    for (int j = 0; j < E; ++j) w[j] = load_any(wp, a.wtype, s.in ? (j < V ? s.a : s.b) + j % V : 0);
  }
  // the lane's first frequency, in quarter turns a position, and the step from pair to pair
  const double each = a.R ? -2.0 * a.log2_base / a.R : 0.0;
  const double freq0 = exp2(each * (l * V)) * 0.63661977236758134, ratio = exp2(each);
  const float inv_d = 1.0f / (float)a.D;
  // The group's rows in batches of up to U heads of a token.  The next batch, the next
  // token's included, is loaded before this one is worked on.
  QkRow<T, V> x[2][U], y[2][BWD ? U : 1];
  float c[V], sn[V];
  const uint32_t step = nb * G;
  auto load = [&](int b, uint32_t t, int h) {
    const T *xt = x0 + t * x_t, *yt = y0 + t * dy_t;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hu = min(h + u, h1 - 1);
      x[b][u].load(xt + hu * x_h, s);
      if (BWD) y[b][u].load(yt + hu * dy_h, s);
    }
  };
  auto position = [&](uint32_t t) {
    const uint32_t at = a.pos ? t % a.pos_seq : t % a.seq;
    return !a.pos ? (int64_t)at : a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
  };
  auto angles = [&](int64_t p) {
    double f = freq0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sincos_quarters((double)p * f, c[j], sn[j]);
      if (!s.turned) c[j] = 1.0f, sn[j] = 0.0f;
      f *= ratio;
    }
  };
  auto work = [&](int b, uint32_t t, int h) {
    T* out = (T*)a.out[which] + ((int64_t)t * H + h) * a.D;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;
      float v[E];
      x[b][u].get(v, s);
      float q = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) q = __builtin_fmaf(v[j], v[j], q);
      const float square = __builtin_fmaf(group_sum<L>(q), inv_d, a.eps);
      float r = __builtin_amdgcn_rsqf(square), k = 1.0f;   // (1 / sqrt is r k)
      const bool rescaled = out_of_range(square);
      if (rescaled) {
        k = square < 1.0f ? 0x1p48f : 0x1p-48f;
        q = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          v[j] *= k;
          q = __builtin_fmaf(v[j] * k, v[j] * k, q);
        }
        r = __builtin_amdgcn_rsqf(__builtin_fmaf(group_sum<L>(q), inv_d, a.eps * k * k * k * k)) * k;
      }
      if constexpr (!BWD) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = v[j] * r * w[j];
        turn<ADJ, V>(v, c, sn, 1.0f);
      } else {
        float d[E];
        y[b][u].get(d, s);
        turn<ADJ, V>(d, c, sn, -1.0f);
        float along = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          v[j] *= r;
          dw[j] = __builtin_fmaf(d[j], v[j], dw[j]);
          d[j] *= w[j];
          along = __builtin_fmaf(d[j], v[j], along);
        }
        along = group_sum<L>(along) * inv_d;
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = r * __builtin_fmaf(-v[j], along, d[j]);
        if (rescaled) {
#pragma unroll
          for (int j = 0; j < E; ++j) v[j] *= k;
        }
      }
      x[b][u].template store<PAST>(out + (int64_t)u * a.D, s, v);
    }
  };
  uint32_t t = (bid - slice * nb) * G + g;
  int h = h0;
  if (t < a.T) {
    load(0, t, h);
    int64_t p = position(t);
    // one batch from buffer b; false after the last
    auto batch = [&](int b) {
      if (h == h0) angles(p);
      const bool same = h + U < h1;
      const uint32_t t2 = same ? t : t + step;
      const int h2 = same ? h + U : h0;
      if (t2 < a.T) {
        load(b ^ 1, t2, h2);
        if (!same) p = position(t2);
      }
      work(b, t, h);
      t = t2, h = h2;
      return t < a.T;
    };
    while (batch(0) && batch(1)) {
    }
  }
  if constexpr (BWD) {
    if (!a.part[which]) return;
    // the block's groups in order
    if (s.in) {
#pragma unroll
      for (int j = 0; j < E; ++j) sums[g][(j < V ? s.a : s.b) + j % V] = dw[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += 256) {
      float v = sums[0][i];
#pragma unroll
      for (int k = 1; k < G; ++k) v += sums[k][i];
      a.part[which][(int64_t)bid * a.D + i] = v;
    }
  }
}

// dw from the blocks' partials: 64 columns a block, each wave a sixteenth of the
// rows in order, then the waves' sums in order
__global__ __launch_bounds__(1024) void qk_dw_kernel(const float* p0, const float* p1, int rows0, int rows1, int D,
                                                     void* dw0, void* dw1, int wtype) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, nb = blockIdx.y ? rows1 : rows0;
  const float* p = blockIdx.y ? p1 : p0;
  void* dw = blockIdx.y ? dw1 : dw0;
  if (!dw) return;
  float v = 0.0f;
  if (c < D) {
    const int per = (nb + 15) / 16, end = min(nb, (wave + 1) * per);
    int r = wave * per;
    for (; r + 8 <= end; r += 8) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = p[(int64_t)(r + i) * D + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += t[i];
    }
    for (; r < end; ++r) v += p[(int64_t)r * D + c];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < D) {
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += sums[k][lane];
    store_any(dw, wtype, c, v);
  }
}

// ---- host -------------------------------------------------------------------
struct QkPlan {
  int v, lanes;        // elements of a lane's half, lanes of a row
  int heads[2];        // a slice's
  int parts[2];        // slices of q and of k
  uint32_t blocks[2];  // of a slice
  bool past;           // results past the caches
};
static QkPlan qk_plan(const concord_qk_args& g, bool bwd) {
  QkPlan p{};
  // 16 bytes a load where both halves of the turned and of the other elements are whole
  // chunks of them (adjacent pairs take 16 bytes in two neighbouring loads); the forward of
  // wider rows keeps to 8, whose smaller state leaves more waves (bf16, 32768 x 40 heads,
  // us by 16 bytes and by 8: of 64 forward 64 and 70, backward 94 and 145; of 80 130 and 106,
  // 165 and 244; of 96 126 and 105, 161 and 252; of 112 177 and 115, 185 and 260; of 128 145
  // and 116, 196 and 260.  16384 x 9 heads: of 64 8.1 and 10.1, 11.5 and 13.0; of 80 to 128
  // the two are within a tenth but for the forward of 96, 13.2 and 15.1, and 112, 19.5 and 15.6)
  p.v = g.dtype != CONCORD_F32 && !g.adjacent && g.R % 16 == 0 && g.D % 16 == 0 && (bwd || g.D <= 64) ? 8 : 4;
  p.lanes = 1;
  while (p.lanes * 2 * p.v < g.D) p.lanes *= 2;
  const int64_t groups = 256 / p.lanes;
  // as many heads a slice as leave 512 blocks: the angles are formed once a slice
  for (int most = 16; most >= 1; most /= 2) {
    const int H[2] = {g.H, g.HK};
    for (int i = 0; i < 2; ++i) {
      p.parts[i] = (int)cdiv(H[i], most);
      p.heads[i] = p.parts[i] ? (int)cdiv(H[i], p.parts[i]) : 1;
    }
    if (cdiv(g.T, groups) * (p.parts[0] + p.parts[1]) >= 512) break;
  }
  // Many tokens: a little under two blocks a CU in all, a slice's by its share of the
  // heads, that go on from token to token (forward of 32768 x 40 heads of 128: 122 us, 137
  // with four a CU, 134 with a block for each group's token).  Few: no block takes two.
  const int64_t total = cdiv(g.T, groups), all = g.H + g.HK;
  const bool few = total * (p.parts[0] + p.parts[1]) <= 2048;
  // (16384 x 9 heads of 64 10.5 -> 8.3 us forward, 14.0 -> 11.7 backward; 32768 x 40 of 128
  // 133 -> 124 forward, but 215 -> 228 backward, whose many blocks store as they read)
  p.past = few || !bwd;
  for (int i = 0; i < 2; ++i) {
    const int64_t want = few ? total : std::max<int64_t>(1, 480 * p.heads[i] / all);
    // (an eighth over its share rather than a round of its own for the last few)
    const int64_t rounds = cdiv(std::max<int64_t>(1, total - want / 8), want);
    p.blocks[i] = (uint32_t)cdiv(total, rounds);
  }
  return p;
}

template <class T, int V, int L, bool ADJ>
static void qk_pass(const QkArgs& a, uint32_t blocks, bool bwd, bool past, hipStream_t st) {
  const dim3 grid(blocks);
  if (!bwd) hipLaunchKernelGGL((qk_kernel<T, V, L, ADJ, false, true>), grid, dim3(256), 0, st, a);
  else if (past) hipLaunchKernelGGL((qk_kernel<T, V, L, ADJ, true, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((qk_kernel<T, V, L, ADJ, true, false>), grid, dim3(256), 0, st, a);
}
template <class T, int V, int L>
static void qk_launch(const QkArgs& a, uint32_t blocks, bool bwd, bool past, hipStream_t st) {
  if constexpr (V == 4) {
    if (a.adjacent) return qk_pass<T, V, L, true>(a, blocks, bwd, past, st);
  }
  qk_pass<T, V, L, false>(a, blocks, bwd, past, st);
}
template <class T>
static void qk_lanes(const QkArgs& a, const QkPlan& p, uint32_t blocks, bool bwd, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (p.v == 8) {
      switch (p.lanes) {
        case 1: return qk_launch<T, 8, 1>(a, blocks, bwd, p.past, st);
        case 2: return qk_launch<T, 8, 2>(a, blocks, bwd, p.past, st);
        case 4: return qk_launch<T, 8, 4>(a, blocks, bwd, p.past, st);
        case 8: return qk_launch<T, 8, 8>(a, blocks, bwd, p.past, st);
        default: return qk_launch<T, 8, 16>(a, blocks, bwd, p.past, st);
      }
    }
  }
  switch (p.lanes) {
    case 1: return qk_launch<T, 4, 1>(a, blocks, bwd, p.past, st);
    case 2: return qk_launch<T, 4, 2>(a, blocks, bwd, p.past, st);
    case 4: return qk_launch<T, 4, 4>(a, blocks, bwd, p.past, st);
    case 8: return qk_launch<T, 4, 8>(a, blocks, bwd, p.past, st);
    case 16: return qk_launch<T, 4, 16>(a, blocks, bwd, p.past, st);
    default: return qk_launch<T, 4, 32>(a, blocks, bwd, p.past, st);
  }
}
static uint32_t qk_rows(const QkPlan& p, int i) { return p.blocks[i] * (uint32_t)p.parts[i]; }
static void qk_run(QkArgs& a, const QkPlan& p, int dtype, bool bwd, hipStream_t st) {
  for (int i = 0; i < 2; ++i) a.heads[i] = p.heads[i], a.blocks[i] = p.blocks[i];
  a.k_at = qk_rows(p, 0);
  const uint32_t blocks = a.k_at + qk_rows(p, 1);
  if (dtype == CONCORD_F32) qk_lanes<float>(a, p, blocks, bwd, st);
  else if (dtype == CONCORD_BF16) qk_lanes<BF16>(a, p, blocks, bwd, st);
  else qk_lanes<_Float16>(a, p, blocks, bwd, st);
}

static bool qk_aligned(const void* p, int64_t t, int64_t h) {
  return ((uintptr_t)p & 15) == 0 && t % 8 == 0 && h % 8 == 0;
}

static bool qk_sizes_ok(const concord_qk_args& g) {
  return g.T >= 0 && g.T < (1LL << 31) && g.H >= 0 && g.HK >= 0 && g.H < (1 << 14) && g.HK < (1 << 14) && g.H + g.HK > 0 &&
         g.D >= 8 && g.D <= 256 && g.D % 8 == 0 && g.R >= 0 && g.R <= g.D && g.R % 8 == 0;
}

// checks that both passes share, and their arguments
static int qk_args(const concord_qk_args* args, const char* name, bool bwd, QkArgs& a) {
  CONCORD_CHECK(args, "%s: NULL argument", name);
  const concord_qk_args& g = *args;
  CONCORD_CHECK(qk_sizes_ok(g), "%s: bad size", name);
  for (int t : {g.dtype, g.wtype})
    CONCORD_CHECK(t == CONCORD_F32 || t == CONCORD_BF16 || t == CONCORD_F16, "%s: bad type", name);
  CONCORD_CHECK(g.base > 0 && g.base < 1e300 && g.eps >= 0 && __builtin_isfinite(g.eps), "%s: bad base or eps", name);
  if (g.T == 0) return CONCORD_OK;
  CONCORD_CHECK(g.seq >= 1 && g.seq <= g.T && (!g.positions || (g.pos_seq >= 1 && g.pos_seq <= g.T)), "%s: bad sequence length",
                name);
  CONCORD_CHECK((g.H == 0 || g.q) && (g.HK == 0 || g.k), "%s: NULL argument", name);
  CONCORD_CHECK((g.H == 0 || qk_aligned(g.q, g.q_t, g.q_h)) && (g.HK == 0 || qk_aligned(g.k, g.k_t, g.k_h)),
                "%s: rows must lie on 16 bytes, strides in multiples of 8", name);
  void* const out[2] = {bwd ? g.dq : g.q_out, bwd ? g.dk : g.k_out};
  CONCORD_CHECK((g.H == 0 || out[0]) && (g.HK == 0 || out[1]), "%s: NULL result", name);
  CONCORD_CHECK((((uintptr_t)out[0] | (uintptr_t)out[1]) & 15) == 0, "%s: results must lie on 16 bytes", name);
  if (bwd) {
    CONCORD_CHECK((g.H == 0 || g.dq_out) && (g.HK == 0 || g.dk_out), "%s: NULL gradient", name);
    CONCORD_CHECK((g.H == 0 || qk_aligned(g.dq_out, g.dq_t, g.dq_h)) && (g.HK == 0 || qk_aligned(g.dk_out, g.dk_t, g.dk_h)),
                  "%s: rows must lie on 16 bytes, strides in multiples of 8", name);
  }
  a.x[0] = g.q, a.x[1] = g.k, a.x_t[0] = g.q_t, a.x_h[0] = g.q_h, a.x_t[1] = g.k_t, a.x_h[1] = g.k_h;
  a.dy[0] = g.dq_out, a.dy[1] = g.dk_out, a.dy_t[0] = g.dq_t, a.dy_h[0] = g.dq_h, a.dy_t[1] = g.dk_t, a.dy_h[1] = g.dk_h;
  a.out[0] = out[0], a.out[1] = out[1];
  a.w[0] = g.q_weight, a.w[1] = g.k_weight, a.wtype = g.wtype;
  a.pos = g.positions, a.pos64 = g.pos64;
  a.T = (uint32_t)g.T, a.seq = (uint32_t)g.seq, a.pos_seq = (uint32_t)(g.positions ? g.pos_seq : 1);
  a.H[0] = g.H, a.H[1] = g.HK, a.D = g.D, a.R = g.R, a.adjacent = g.adjacent != 0, a.eps = g.eps;
  a.log2_base = __builtin_log2(g.base);
  return CONCORD_OK;
}

static size_t qk_workspace(const concord_qk_args& g, const QkPlan& p) {
  return ((size_t)qk_rows(p, 0) + qk_rows(p, 1)) * g.D * sizeof(float);
}

}  // namespace concord

using namespace concord;

extern "C" int concord_qk_norm_rope_fwd(const concord_qk_args* args, void* stream) {
  QkArgs a{};
  if (const int rc = qk_args(args, "concord_qk_norm_rope_fwd", false, a)) return rc;
  if (args->T == 0) return CONCORD_OK;
  qk_run(a, qk_plan(*args, false), args->dtype, false, (hipStream_t)stream);
  return launch_status("qk_norm_rope_fwd");
}

extern "C" size_t concord_qk_norm_rope_workspace_bytes(const concord_qk_args* args) {
  if (!args || !qk_sizes_ok(*args) || args->T == 0) return 0;
  return qk_workspace(*args, qk_plan(*args, true));
}

extern "C" int concord_qk_norm_rope_bwd(const concord_qk_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  QkArgs a{};
  if (const int rc = qk_args(args, "concord_qk_norm_rope_bwd", true, a)) return rc;
  const concord_qk_args& g = *args;
  if (g.T == 0 && !g.dq_weight && !g.dk_weight) return CONCORD_OK;
  hipStream_t st = (hipStream_t)stream;
  int rows[2] = {};
  if (g.T > 0) {
    const QkPlan p = qk_plan(g, true);
    if ((g.dq_weight || g.dk_weight) && (!workspace || workspace_bytes < qk_workspace(g, p))) {
      set_error("concord_qk_norm_rope_bwd: workspace of %zu bytes needed", qk_workspace(g, p));
      return CONCORD_EWORKSPACE;
    }
    for (int i = 0; i < 2; ++i) rows[i] = (int)qk_rows(p, i);
    a.part[0] = g.dq_weight ? (float*)workspace : nullptr;
    a.part[1] = g.dk_weight ? (float*)workspace + (int64_t)rows[0] * g.D : nullptr;
    qk_run(a, p, g.dtype, true, st);
  }
  if (g.dq_weight || g.dk_weight)   // (no token: sums over no partials, zero)
    hipLaunchKernelGGL(qk_dw_kernel, dim3((unsigned)cdiv(g.D, 64), 2), dim3(1024), 0, st, (const float*)a.part[0],
                       (const float*)a.part[1], rows[0], rows[1], g.D, g.dq_weight, g.dk_weight, g.wtype);
  return launch_status("qk_norm_rope_bwd");
}
