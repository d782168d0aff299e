// attention_bwd.hip -- the gradients of attention (attention.hip):
//   delta = sum over d of dout out,  dP = dout v^T,  dS = P (dP - delta),
//   dq = scale dS k,  dv = P^T dout,  dk = scale dS^T q
// with P = 2^(scale log2(e) q k^T - lse) formed again from the forward's lse.
//
// Two kernels, each sum in registers in a fixed order (no atomics): one holds
// queries and passes over their keys for dq, and leaves delta for the other,
// which holds keys and passes over the queries of all heads that share them
// for dk and dv.  The price is that both form P and dP: seven products instead
// of five.  dS is rounded to bf16 for its two products.
//
// dq is bound by power as the forward is: 2 x 8192 x 32 / 8 heads of 128 without a
// mask 2800 us (three products, 1178 TFLOP/s), MFMA pipes busy 0.65.  dk / dv
// take 3890 us (four products, 1131 TFLOP/s), busy 0.56: their sums fill the
// registers of two waves per SIMD, which leaves few fragment reads in flight.
#include "attention.h"

namespace concord {

struct AttnBwd {
  const uint16_t *q, *k, *v, *out, *dout;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h, do_t, do_h;
  uint16_t *dq, *dk, *dv;
  int64_t dq_t, dq_h, dk_t, dk_h, dv_t, dv_h;
  const float* lse;
  const int8_t* low;
  float* delta;
  float* part;      // the shares' sums
  AttnSeqs seq;
  int32_t slots, rep, D, causal, heads, rows_h, splits;   // rows_h: key heads
  float c, scale;
};

constexpr int kDqRows = 128, kDkvRows = 128;   // queries of a dq workgroup, keys of a dk / dv one
constexpr int kStep = 64;      // keys (queries) of a step

// dq and delta: the forward's shape.  A lane holds one query's column of the
// transposed scores, so lse and delta are lane-local.
// SPLIT: a share of the key tiles, as in the forward; fp32 sums.
template <int NK, bool SPLIT>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnBwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kStep, 4> T;
  constexpr int ND = DIM::ND;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES];   // two slots of k and v
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lin = attn_xcd(blockIdx.x, gridDim.x), share = 0;
  if (SPLIT) {
    share = lin % a.splits;
    lin /= a.splits;
  }
  const int per = a.rep * a.slots;
  const int hk = lin / per, in = lin - hk * per;
  const int slot = a.slots - 1 - in / a.rep, head = hk * a.rep + in % a.rep;
  AttnPlace p = attn_place<kDqRows, false>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lq) return;

  const int row0 = p.first + wave * 32, rows = p.lq - row0, off = p.lk - p.lq;
  const int last = min(p.first + kDqRows, p.lq) - 1;
  const int keys = a.causal ? max(0, min(p.lk, last + off + 1)) : p.lk;
  int tiles = (keys + kStep - 1) / kStep;
  const int qi = row0 + (lane & 31);
  int jmax = a.causal ? min(p.lk - 1, qi + off) : p.lk - 1;
  int jlo = a.causal ? min(p.lk - 1, row0 + off) : p.lk - 1;
  int jhi = a.causal ? min(p.lk - 1, row0 + 31 + off) : p.lk - 1;
  if (SPLIT) {   // keys count from the share's first
    const int t0 = (int)((int64_t)tiles * share / a.splits), j0 = t0 * kStep;
    tiles = (int)((int64_t)tiles * (share + 1) / a.splits) - t0;
    p.k0 += j0;
    p.lk -= j0;
    jmax -= j0;
    jlo -= j0;
    jhi -= j0;
  }

  Fixed<DIM> q, g;
  q.load(a.q + (p.q0 + row0) * a.q_t + (int64_t)head * a.q_h, rows, a.q_t, a.D, lane);
  g.load(a.dout + (p.q0 + row0) * a.do_t + (int64_t)head * a.do_h, rows, a.do_t, a.D, lane);
  const int64_t at = (int64_t)head * a.seq.TQ + p.q0 + qi;
  const float lse = qi < p.lq ? a.lse[at] : INFINITY;
  float delta;
  {
    Fixed<DIM> o;
    o.load(a.out + (p.q0 + row0) * a.o_t + (int64_t)head * a.o_h, rows, a.o_t, a.D, lane);
    const int64_t low_t = (int64_t)a.heads * a.D;
    delta = row_dot(o, a.low + (p.q0 + row0) * low_t + (int64_t)head * a.D, rows, low_t, a.D, g, lane);
    if (share == 0 && lane < 32 && qi < p.lq) a.delta[at] = delta;
  }
  const uint16_t* kp = a.k + p.k0 * a.k_t + (int64_t)hk * a.k_h;
  const uint16_t* vp = a.v + p.k0 * a.v_t + (int64_t)hk * a.v_h;
  T tk, tv;
  tk.init(a.k_t, a.D, lane);
  tv.init(a.v_t, a.D, lane);
  const uint32_t base = lds_addr(lds);
  Frags<DIM> fr;
  fr.init(base, lane);

  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = zero16();
  auto load = [&](int t) {
    const uint32_t s = base + (uint32_t)((t & 1) * 2 * T::BYTES);
    tk.load(kp + (int64_t)t * kStep * a.k_t, p.lk - t * kStep, s, wave);
    tv.load(vp + (int64_t)t * kStep * a.v_t, p.lk - t * kStep, s + T::BYTES, wave);
  };
  auto step = [&](int j0) {
    constexpr uint32_t kt = 0, vt = T::BYTES;
    const bool masked = j0 + kStep - 1 > jlo;
    const int lim = jmax - j0 - 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < NK; ++k) s = mfma(fr.rows(kt, i, k), q.f[k], s);
#pragma unroll
      for (int k = 0; k < NK; ++k) dp = mfma(fr.rows(vt, i, k), g.f[k], dp);
      if (masked)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 32 * i + 8 * (r >> 2) + (r & 3) > lim ? -INFINITY : s[r];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -lse)) * (dp[r] - delta);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8 ds = round8(s, u);
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = mfma(fr.cols(kt, d, 2 * i + u), ds, dq[d]);
      }
    }
  };
  if (tiles > 0) load(0);
  for (int t = 0; t < tiles; ++t) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    lds_barrier();
    if (t + 1 < tiles) load(t + 1);
    if (t * kStep <= jhi) step(t * kStep);
    fr.move(t & 1 ? -2 * T::BYTES : 2 * T::BYTES);
  }
  if constexpr (SPLIT) {
    if ((lane & 31) < rows)
      store_sums(a.part + (((int64_t)share * a.seq.TQ + p.q0 + qi) * a.heads + head) * a.D, dq, a.D, lane);
    return;
  }
  uint16_t* out = a.dq + (p.q0 + row0) * a.dq_t + (int64_t)head * a.dq_h;
#pragma unroll
  for (int d = 0; d < ND; ++d) store_block(out, a.dq_t, rows, a.D, d, dq[d], a.scale, lane);
}

// dk and dv: a wave holds 32 keys, and the scores untransposed (rows:
// queries), so P and dS are the B operands of dv^T += dout^T P and
// dk^T += q^T dS as they come.  lse and delta of a step's queries lie in LDS.
//
// SPLIT: a workgroup takes one of `splits` equal shares of the steps and leaves
// fp32 sums for attn_sum_kernel.
template <int NK, bool SPLIT>
__global__ __launch_bounds__(256, NK <= 4 ? 3 : 2) void attn_dkv_kernel(AttnBwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kStep, 4> T;
  constexpr int ND = DIM::ND;
  // two slots of q and dout, then two of lse and delta
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES + 2 * 2 * kStep * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lin = attn_xcd(blockIdx.x, gridDim.x), share = 0;
  if (SPLIT) {
    share = lin % a.splits;
    lin /= a.splits;
  }
  const int hk = lin / a.slots, slot = lin - hk * a.slots;   // (the first keys have the most queries)
  const AttnPlace p = attn_place<kDkvRows, true>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lk) return;

  const int key0 = p.first + wave * 32, left = p.lk - key0, off = p.lk - p.lq;
  // the first query that sees any of the workgroup's keys
  const int first = a.causal ? max(0, p.first - off) : 0;
  const int t0 = first / kStep;
  const int per = max(0, (p.lq + kStep - 1) / kStep - t0);   // steps of a head
  const int steps = per * a.rep;
  const int it0 = SPLIT ? (int)((int64_t)steps * share / a.splits) : 0;
  const int it1 = SPLIT ? (int)((int64_t)steps * (share + 1) / a.splits) : steps;

  Fixed<DIM> k, v;
  f32x16 dk[ND], dv[ND];
  const int64_t tok = p.k0 + key0;
  k.load(a.k + tok * a.k_t + (int64_t)hk * a.k_h, left, a.k_t, a.D, lane);
  v.load(a.v + tok * a.v_t + (int64_t)hk * a.v_h, left, a.v_t, a.D, lane);
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
  T tq, tg;
  tq.init(a.q_t, a.D, lane);
  tg.init(a.do_t, a.D, lane);
  const uint32_t base = lds_addr(lds), stats = base + 4 * T::BYTES;
  Frags<DIM> fr;
  fr.init(base, lane);

  auto load = [&](int it, int ring) {
    const int r = it / per, i0 = (t0 + it - r * per) * kStep, head = hk * a.rep + r;
    const uint32_t s = base + (uint32_t)(ring * 2 * T::BYTES);
    tq.load(a.q + (p.q0 + i0) * a.q_t + (int64_t)head * a.q_h, p.lq - i0, s, wave);
    tg.load(a.dout + (p.q0 + i0) * a.do_t + (int64_t)head * a.do_h, p.lq - i0, s + T::BYTES, wave);
    // (a query past the last reads 0, and q = dout = 0: it adds nothing)
    if (wave < 2) {
      const float* src = (wave ? a.delta : a.lse) + (int64_t)head * a.seq.TQ + p.q0 + i0;
      const i32x4 rs = rows_rsrc((const uint16_t*)src, min(p.lq - i0, kStep), 4, 4);
      dma4(rs, (uint32_t)lane * 4, stats + (uint32_t)((ring * 2 + wave) * kStep * 4));
    }
  };
  uint32_t own = stats + (uint32_t)((lane >> 5) * 16);   // lse of the half wave's first row
  auto step = [&](int i0) {
    constexpr uint32_t qt = 0, gt = T::BYTES;
    const bool masked = a.causal && i0 + off < key0 + 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // P and dv, then dP, dS and dk; with wide heads kept in that order
      // (sched_barrier), the fewest values at a time.  A spilled register costs
      // more than its reload here, which waits for the DMA of the next step too
      // (15 packed sequences, 16384 tokens, 32 / 8 x 128: 1197 us with 7 of them, 1050
      // without).
      bf16x8 e[2], es[2];
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) s = mfma(fr.rows(qt, i, kk), k.f[kk], s);
      if (masked) {
        const int lim = key0 + (lane & 31) - off - i0 - 4 * (lane >> 5);   // key j sees queries from j - off on
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 32 * i + 8 * (r >> 2) + (r & 3) < lim ? -INFINITY : s[r];
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const i32x4 lse = *(const lds_i32x4*)(lds_at(own) + (32 * i + 8 * g) * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[4 * g + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + r], a.c, -__int_as_float(lse[r])));
      }
      e[0] = round8(s, 0);
      e[1] = round8(s, 1);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) dv[d] = mfma(fr.cols(gt, d, 2 * i + u), e[u], dv[d]);
      if constexpr (NK > 4) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) dp = mfma(fr.rows(gt, i, kk), v.f[kk], dp);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const i32x4 delta = *(const lds_i32x4*)(lds_at(own) + (kStep + 32 * i + 8 * g) * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) dp[4 * g + r] = s[4 * g + r] * (dp[4 * g + r] - __int_as_float(delta[r]));
      }
      es[0] = round8(dp, 0);
      es[1] = round8(dp, 1);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[d] = mfma(fr.cols(qt, d, 2 * i + u), es[u], dk[d]);
      if constexpr (NK > 4) __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (it0 < it1) load(it0, 0);
  for (int it = it0; it < it1; ++it) {
    const int ring = (it - it0) & 1;
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    lds_barrier();
    if (it + 1 < it1) load(it + 1, ring ^ 1);
    const int i0 = (t0 + it % per) * kStep;
    // (causal: where the step's last query sees none of the wave's keys there is nothing to add)
    if (!a.causal || i0 + kStep - 1 + off >= key0) step(i0);
    const int sign = ring ? -1 : 1;
    fr.move(sign * 2 * T::BYTES);
    own += (uint32_t)(sign * 2 * kStep * 4);
  }
  if constexpr (SPLIT) {
    if ((lane & 31) >= left) return;
    // [share][dk, dv][token][key head][D]
    const int64_t row = (int64_t)a.rows_h * a.D, all = a.seq.TK * row;
    float* to = a.part + (int64_t)share * 2 * all + (tok + (lane & 31)) * row + (int64_t)hk * a.D;
    store_sums(to, dk, a.D, lane);
    store_sums(to + all, dv, a.D, lane);
    return;
  }
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    store_block(a.dk + tok * a.dk_t + (int64_t)hk * a.dk_h, a.dk_t, left, a.D, d, dk[d], a.scale, lane);
    store_block(a.dv + tok * a.dv_t + (int64_t)hk * a.dv_h, a.dv_t, left, a.D, d, dv[d], 1.0f, lane);
  }
}

// Shares' sums added in their order, a thread 8 elements of a row: N outputs of
// tokens x heads x D, part [share][N][token][head][D]
struct AttnSum {
  const float* part;
  int64_t all;       // elements of an output
  int32_t splits, heads, D;
  uint16_t* to[2];
  int64_t t[2], h[2];
  float scale[2];
};
template <int N>
__global__ __launch_bounds__(256) void attn_sum_kernel(AttnSum a) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;   // D is a multiple of 8
  if (e >= a.all) return;
  const int64_t row = e / a.D, tok = row / a.heads;
  const int c = (int)(e - row * a.D), head = (int)(row - tok * a.heads);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float v[8] = {};
    for (int s = 0; s < a.splits; ++s) {
      const float4* p = (const float4*)(a.part + ((int64_t)s * N + n) * a.all + e);
      const float4 x = p[0], y = p[1];
      v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
      v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    const float f = a.scale[n];
    *(uint4*)(a.to[n] + tok * a.t[n] + (int64_t)head * a.h[n] + c) =
        make_uint4(pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f),
                   pack_bf16x2(v[4] * f, v[5] * f), pack_bf16x2(v[6] * f, v[7] * f));
  }
}

// Shares a key tile's steps are split into.  A launch of the key tiles alone may
// leave CUs idle (few tiles: a short batch, few key heads) or wait for the tile
// with the most queries (a causal mask, sequences of different lengths): up to
// four times the workgroups that the chip holds even that out.  A share has four
// steps at least, and the shares' sums cost 16 bytes an element, which must stay
// below a sixth of the launch's time (products at 1 PFLOP/s on a full chip, sums
// at 5 TB/s; lengths are not known here, so the mean stands for them).  2 x 4096
// causal, 32 / 8 heads of 128: the whole backward 1273 us in one share, 957 us.
static int dkv_splits(const concord_attn_args& g) {
  if (g.TQ < 1 || g.TK < 1) return 1;
  AttnSeqs s = attn_seqs(g);
  const double wgs = (double)attn_slots(s, g.TK, kDkvRows) * g.HK, room = g.D <= 64 ? 768.0 : 512.0;
  const double per_seq = (double)g.TQ / (double)std::max<int64_t>(g.B, 1) * (g.causal ? 0.5 : 1.0);
  const double steps = per_seq / kStep * (g.H / g.HK);
  const double time = 8.0 * g.TK * per_seq * g.H * g.D / 1e15 * std::max(1.0, room / wgs);
  const double share = 16.0 * g.TK * g.HK * g.D / 5e12;
  double n = (g.causal || g.starts ? 4.0 : 1.0) * room / wgs;
  n = std::min(std::min(n, steps / 4.0), time / 6.0 / share);
  return n < 2.0 ? 1 : n < 16.0 ? (int)n : 16;
}

// the workspace: delta, then the shares' sums
static size_t delta_bytes(const concord_attn_args& g) {
  return ((size_t)g.TQ * (size_t)g.H * sizeof(float) + 255) / 256 * 256;
}

}  // namespace concord

using namespace concord;

extern "C" size_t concord_attention_workspace_bytes(const concord_attn_args* args) {
  if (!args || attn_sizes("concord_attention_workspace_bytes", *args) || args->TQ < 1) return 0;
  const size_t n = dkv_splits(*args), m = key_splits(*args, 6.0);
  const size_t dkv = n > 1 ? n * 2 * (size_t)args->TK * (size_t)args->HK : 0;
  const size_t dq = m > 1 ? m * (size_t)args->TQ * (size_t)args->H : 0;
  return delta_bytes(*args) + std::max(dkv, dq) * (size_t)args->D * sizeof(float);   // (one after the other)
}

extern "C" int concord_attention_bwd(const concord_attn_args* args, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  CONCORD_CHECK(args, "concord_attention_bwd: NULL argument");
  const concord_attn_args& g = *args;
  const char* what = "concord_attention_bwd";
  if (const int rc = attn_check(what, g)) return rc;
  CONCORD_CHECK(attn_operand(g.dout, g.do_t, g.do_h, g.TQ, g.D) && attn_operand(g.dq, g.dq_t, g.dq_h, g.TQ, g.D) &&
                    attn_operand(g.dk, g.dk_t, g.dk_h, g.TK, g.D) && attn_operand(g.dv, g.dv_t, g.dv_h, g.TK, g.D),
                "%s: NULL, misaligned or badly strided gradient", what);
  CONCORD_CHECK((g.lse && g.out_low && ((uintptr_t)g.out_low & 15) == 0) || g.TQ == 0,
                "%s: lse or out_low is NULL or misaligned", what);
  if (g.TQ == 0 && g.TK == 0) return CONCORD_OK;
  const size_t need = concord_attention_workspace_bytes(args);
  if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes on 16 needed", what, need);
    return CONCORD_EWORKSPACE;
  }
  AttnBwd a{};
  a.q = g.q, a.k = g.k, a.v = g.v, a.out = g.out, a.dout = g.dout, a.dq = g.dq, a.dk = g.dk, a.dv = g.dv;
  a.q_t = g.q_t, a.q_h = g.q_h, a.k_t = g.k_t, a.k_h = g.k_h, a.v_t = g.v_t, a.v_h = g.v_h;
  a.o_t = g.o_t, a.o_h = g.o_h, a.do_t = g.do_t, a.do_h = g.do_h;
  a.dq_t = g.dq_t, a.dq_h = g.dq_h, a.dk_t = g.dk_t, a.dk_h = g.dk_h, a.dv_t = g.dv_t, a.dv_h = g.dv_h;
  a.lse = g.lse, a.low = g.out_low, a.heads = g.H, a.delta = (float*)workspace;
  a.rep = g.H / g.HK, a.D = g.D, a.causal = g.causal != 0, a.c = g.scale * kLog2e, a.scale = g.scale;
  a.seq = attn_seqs(g);
  a.part = (float*)((char*)workspace + delta_bytes(g));
  hipStream_t st = (hipStream_t)stream;
  AttnSum sum{};
  sum.part = a.part, sum.D = g.D;
  AttnSeqs keys = a.seq;
  const int q_splits = key_splits(g, 6.0), k_splits = dkv_splits(g);
  const int64_t q_slots = g.TQ > 0 ? attn_slots(a.seq, g.TQ, kDqRows) : 0;
  const int64_t k_slots = g.TK > 0 ? attn_slots(keys, g.TK, kDkvRows) : 0;
  CONCORD_CHECK(grid_fits(q_slots * g.H * q_splits, 256) && grid_fits(k_slots * g.HK * k_splits, 256),
                "%s: too many tiles", what);
  if (g.TQ > 0) {
    a.splits = q_splits;
    a.slots = (int32_t)q_slots;
    const dim3 grid((unsigned)(q_slots * g.H * a.splits));
    attn_by_dim(g.D, [&](auto nk) {
      constexpr int NK = decltype(nk)::value;
      if (a.splits > 1) hipLaunchKernelGGL((attn_dq_kernel<NK, true>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((attn_dq_kernel<NK, false>), grid, dim3(256), 0, st, a);
    });
    if (a.splits > 1) {
      sum.all = g.TQ * g.H * g.D, sum.splits = a.splits, sum.heads = g.H;
      sum.to[0] = g.dq, sum.t[0] = g.dq_t, sum.h[0] = g.dq_h, sum.scale[0] = g.scale;
      hipLaunchKernelGGL((attn_sum_kernel<1>), dim3((unsigned)cdiv(sum.all, 2048)), dim3(256), 0, st, sum);
    }
  }
  if (g.TK > 0) {
    a.seq = keys;
    a.splits = k_splits;
    a.slots = (int32_t)k_slots;
    a.rows_h = g.HK;
    const dim3 grid((unsigned)(k_slots * g.HK * a.splits));
    attn_by_dim(g.D, [&](auto nk) {
      constexpr int NK = decltype(nk)::value;
      if (a.splits > 1) hipLaunchKernelGGL((attn_dkv_kernel<NK, true>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((attn_dkv_kernel<NK, false>), grid, dim3(256), 0, st, a);
    });
    if (a.splits > 1) {
      sum.all = g.TK * g.HK * g.D, sum.splits = a.splits, sum.heads = g.HK;
      sum.to[0] = g.dk, sum.t[0] = g.dk_t, sum.h[0] = g.dk_h, sum.scale[0] = g.scale;
      sum.to[1] = g.dv, sum.t[1] = g.dv_t, sum.h[1] = g.dv_h, sum.scale[1] = 1.0f;
      hipLaunchKernelGGL((attn_sum_kernel<2>), dim3((unsigned)cdiv(sum.all, 2048)), dim3(256), 0, st, sum);
    }
  }
  return launch_status("attention_bwd");
}
