// attention_bwd.hip -- the gradients of attention (attention.hip):
//   delta = sum over d of dout out,  dP = dout v^T,  dS = P (dP - delta),
//   dq = scale dS k,  dv = P^T dout,  dk = scale dS^T q
// with P = 2^(scale log2(e) q k^T - lse) formed again from the forward's lse.
//
// Two kernels, each sum in registers in a fixed order (no atomics): one holds
// queries and passes over their keys for dq, and leaves delta for the other,
// which holds keys and passes over the queries of all heads that share them
// for dk and dv.  The price is that both form P and dP: seven products instead
// of five.
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
  AttnSeqs seq;
  int32_t slots, rep, D, causal, heads;
  float c, scale;
};

constexpr int kDqRows = 128;   // queries of a dq workgroup
constexpr int kStep = 64;      // keys (queries) of a step

// dq and delta: the forward's shape.  A lane holds one query's column of the
// transposed scores, so lse and delta are lane-local.
template <int NK>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnBwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kStep, 4> T;
  constexpr int ND = DIM::ND;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES];   // two slots of k and v
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lin = attn_xcd(blockIdx.x, gridDim.x);
  const int per = a.rep * a.slots;
  const int hk = lin / per, in = lin - hk * per;
  const int slot = a.slots - 1 - in / a.rep, head = hk * a.rep + in % a.rep;
  const AttnPlace p = attn_place<kDqRows, false>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lq) return;

  const int row0 = p.first + wave * 32, rows = p.lq - row0, off = p.lk - p.lq;
  const int last = min(p.first + kDqRows, p.lq) - 1;
  const int keys = a.causal ? max(0, min(p.lk, last + off + 1)) : p.lk;
  const int tiles = (keys + kStep - 1) / kStep;
  const int qi = row0 + (lane & 31);
  const int jmax = a.causal ? min(p.lk - 1, qi + off) : p.lk - 1;
  const int jlo = a.causal ? min(p.lk - 1, row0 + off) : p.lk - 1;
  const int jhi = a.causal ? min(p.lk - 1, row0 + 31 + off) : p.lk - 1;

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
    if (lane < 32 && qi < p.lq) a.delta[at] = delta;
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
  uint16_t* out = a.dq + (p.q0 + row0) * a.dq_t + (int64_t)head * a.dq_h;
#pragma unroll
  for (int d = 0; d < ND; ++d) store_block(out, a.dq_t, rows, a.D, d, dq[d], a.scale, lane);
}

// dk and dv: a wave holds KB blocks of 32 keys, and the scores untransposed
// (rows: queries), so P and dS are the B operands of dv^T += dout^T P and
// dk^T += q^T dS as they come.  lse and delta of a step's queries lie in LDS.
template <int NK, int KB>
__global__ __launch_bounds__(256, KB == 1 ? 2 : 1) void attn_dkv_kernel(AttnBwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kStep, 4> T;
  constexpr int ND = DIM::ND, KEYS = 128 * KB;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES + 2 * 2 * kStep * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lin = attn_xcd(blockIdx.x, gridDim.x);
  const int hk = lin / a.slots, slot = lin - hk * a.slots;   // (the first keys have the most queries)
  const AttnPlace p = attn_place<KEYS, true>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lk) return;

  const int key0 = p.first + wave * 32 * KB, off = p.lk - p.lq;
  // the first query that sees any of the workgroup's keys
  const int first = a.causal ? max(0, p.first - off) : 0;
  const int t0 = first / kStep;
  const int per = max(0, (p.lq + kStep - 1) / kStep - t0);   // steps of a head
  const int steps = per * a.rep;

  Fixed<DIM> k[KB], v[KB];
  f32x16 dk[KB][ND], dv[KB][ND];
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int64_t tok = p.k0 + key0 + 32 * b;
    k[b].load(a.k + tok * a.k_t + (int64_t)hk * a.k_h, p.lk - key0 - 32 * b, a.k_t, a.D, lane);
    v[b].load(a.v + tok * a.v_t + (int64_t)hk * a.v_h, p.lk - key0 - 32 * b, a.v_t, a.D, lane);
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[b][d] = dv[b][d] = zero16();
  }
  T tq, tg;
  tq.init(a.q_t, a.D, lane);
  tg.init(a.do_t, a.D, lane);
  const uint32_t base = lds_addr(lds), stats = base + 4 * T::BYTES;
  Frags<DIM> fr;
  fr.init(base, lane);

  auto load = [&](int it) {
    const int r = it / per, i0 = (t0 + it - r * per) * kStep, head = hk * a.rep + r;
    const uint32_t s = base + (uint32_t)((it & 1) * 2 * T::BYTES);
    tq.load(a.q + (p.q0 + i0) * a.q_t + (int64_t)head * a.q_h, p.lq - i0, s, wave);
    tg.load(a.dout + (p.q0 + i0) * a.do_t + (int64_t)head * a.do_h, p.lq - i0, s + T::BYTES, wave);
    // (a query past the last reads 0, and q = dout = 0: it adds nothing)
    if (wave < 2) {
      const float* src = (wave ? a.delta : a.lse) + (int64_t)head * a.seq.TQ + p.q0 + i0;
      const i32x4 rs = rows_rsrc((const uint16_t*)src, min(p.lq - i0, kStep), 4, 4);
      dma4(rs, (uint32_t)lane * 4, stats + (uint32_t)(((it & 1) * 2 + wave) * kStep * 4));
    }
  };
  uint32_t own = stats + (uint32_t)((lane >> 5) * 16);   // lse of the half wave's first row
  auto step = [&](int i0) {
    constexpr uint32_t qt = 0, gt = T::BYTES;
    const bool masked = a.causal && i0 + off < key0 + 32 * KB - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bf16x8 pb[KB][2], ds[KB][2];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) s = mfma(fr.rows(qt, i, kk), k[b].f[kk], s);
        if (masked) {
          // key j sees queries from j - off on
          const int lim = key0 + 32 * b + (lane & 31) - off - i0 - 4 * (lane >> 5);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 32 * i + 8 * (r >> 2) + (r & 3) < lim ? -INFINITY : s[r];
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 lse = *(const lds_i32x4*)(lds_at(own) + (32 * i + 8 * g) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[4 * g + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + e], a.c, -__int_as_float(lse[e])));
        }
        pb[b][0] = round8(s, 0);
        pb[b][1] = round8(s, 1);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) dp = mfma(fr.rows(gt, i, kk), v[b].f[kk], dp);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 delta = *(const lds_i32x4*)(lds_at(own) + (kStep + 32 * i + 8 * g) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * g + e] = s[4 * g + e] * (dp[4 * g + e] - __int_as_float(delta[e]));
        }
        ds[b][0] = round8(dp, 0);
        ds[b][1] = round8(dp, 1);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const bf16x8 x = fr.cols(gt, d, 2 * i + u), y = fr.cols(qt, d, 2 * i + u);
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            dv[b][d] = mfma(x, pb[b][u], dv[b][d]);
            dk[b][d] = mfma(y, ds[b][u], dk[b][d]);
          }
        }
    }
  };
  if (steps > 0) load(0);
  for (int it = 0; it < steps; ++it) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    lds_barrier();
    if (it + 1 < steps) load(it + 1);
    const int i0 = (t0 + it % per) * kStep;
    // (causal: where the step's last query sees none of the wave's keys there is nothing to add)
    if (!a.causal || i0 + kStep - 1 + off >= key0) step(i0);
    const int sign = it & 1 ? -1 : 1;
    fr.move(sign * 2 * T::BYTES);
    own += (uint32_t)(sign * 2 * kStep * 4);
  }
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int64_t tok = p.k0 + key0 + 32 * b;
    const int left = p.lk - key0 - 32 * b;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      store_block(a.dk + tok * a.dk_t + (int64_t)hk * a.dk_h, a.dk_t, left, a.D, d, dk[b][d], a.scale, lane);
      store_block(a.dv + tok * a.dv_t + (int64_t)hk * a.dv_h, a.dv_t, left, a.D, d, dv[b][d], 1.0f, lane);
    }
  }
}

}  // namespace concord

using namespace concord;

extern "C" size_t concord_attention_workspace_bytes(const concord_attn_args* args) {
  if (!args || args->TQ < 1 || args->H < 1) return 0;
  return (size_t)args->TQ * (size_t)args->H * sizeof(float);   // delta
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
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes needed", what, need);
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
  hipStream_t st = (hipStream_t)stream;
  if (g.TQ > 0) {
    const int64_t slots = attn_slots(a.seq, g.TQ, kDqRows);
    CONCORD_CHECK(slots * g.H < (1LL << 31), "%s: too many tiles", what);
    a.slots = (int32_t)slots;
    attn_by_dim(g.D, [&](auto nk) {
      hipLaunchKernelGGL((attn_dq_kernel<decltype(nk)::value>), dim3((unsigned)(slots * g.H)), dim3(256), 0, st, a);
    });
  }
  if (g.TK > 0) {
    constexpr int KB = 1;
    const int64_t slots = attn_slots(a.seq, g.TK, 128 * KB);
    CONCORD_CHECK(slots * g.HK < (1LL << 31), "%s: too many tiles", what);
    a.slots = (int32_t)slots;
    attn_by_dim(g.D, [&](auto nk) {
      hipLaunchKernelGGL((attn_dkv_kernel<decltype(nk)::value, KB>), dim3((unsigned)(slots * g.HK)), dim3(256), 0, st,
                         a);
    });
  }
  return launch_status("attention_bwd");
}
