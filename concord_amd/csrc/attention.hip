// attention.hip -- attention over whole sequences, forward:
//   out = softmax(scale q k^T) v, each query over the keys of its sequence.
//
// A workgroup of four waves holds 128 queries of one head, 32 a wave, and
// passes once over their keys, 64 at a time, with the running maximum and sum
// of each query's softmax.  Everything is transposed: a wave forms the scores
// as k q^T, so a lane holds one query's column and the maximum, the sum and
// the rescaling are lane-local (one exchange between the half waves for the
// maximum); the probabilities, rounded to bf16 (off by up to 2^-8 of themselves,
// as out is by its own rounding; the matrix core takes no wider operand at this
// rate), are the B operand of out^T += v^T p without leaving the lane.
//
// Bound by power: with every CU in MFMAs the clock falls to 1.7 - 1.75 GHz (a
// small launch runs at 2.1).  2 x 8192 x 32 / 8 heads of 128 without a mask 1985
// us, 1108 TFLOP/s, MFMA pipes busy 0.62 of the time; a library's 16384^3
// product reaches 1341 TFLOP/s here.  Heads of 64 have half the MFMAs to the
// same exponentials: 2 x 4096 x 64 heads 580 - 610 us, 900 - 950 TFLOP/s, busy 0.52.
#include "attention.h"

namespace concord {

struct AttnFwd {
  const uint16_t *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  uint16_t* out;
  int64_t o_t, o_h;
  float* lse;
  int8_t* low;
  float* part;      // split keys: [share][token][head][D] sums, then [share][token][head] (m, l)
  AttnSeqs seq;
  int32_t slots, rep, D, causal, heads, splits;   // rep: query heads of a key head
  float c;                         // scale log2(e)
};

constexpr int kAttnQ = 128;   // queries of a workgroup
constexpr int kAttnK = 64;    // keys of a step

// SPLIT: a workgroup takes one of `splits` equal shares of the key tiles and
// leaves its sums, unnormalised, with their m and l for attn_join_kernel.
template <int NK, bool SPLIT>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnFwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kAttnK, 4> T;
  constexpr int ND = DIM::ND;
  constexpr bool PIPE = NK > 4;
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
  AttnPlace p = attn_place<kAttnQ, false>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lq) return;

  const int row0 = p.first + wave * 32;                  // the wave's first query
  const int rows = p.lq - row0;                          // (may be <= 0: it still loads tiles)
  const int off = p.lk - p.lq;                           // causal: query i sees keys <= i + off
  // keys of the workgroup's last query
  const int last = min(p.first + kAttnQ, p.lq) - 1;
  const int keys = a.causal ? max(0, min(p.lk, last + off + 1)) : p.lk;
  int tiles = (keys + kAttnK - 1) / kAttnK;
  // the wave's first and last queries' last keys
  const int qi = row0 + (lane & 31);
  int jlo_raw = row0 + off, jlo = a.causal ? min(p.lk - 1, jlo_raw) : p.lk - 1;
  int jhi = a.causal ? min(p.lk - 1, row0 + 31 + off) : p.lk - 1;
  if (SPLIT) {   // keys count from the share's first
    const int t0 = (int)((int64_t)tiles * share / a.splits), j0 = t0 * kAttnK;
    tiles = (int)((int64_t)tiles * (share + 1) / a.splits) - t0;
    p.k0 += j0;
    p.lk -= j0;
    jlo_raw -= j0;
    jlo -= j0;
    jhi -= j0;
  }

  Fixed<DIM> q;
  q.load(a.q + (p.q0 + row0) * a.q_t + (int64_t)head * a.q_h, rows, a.q_t, a.D, lane);
  const uint16_t* kp = a.k + p.k0 * a.k_t + (int64_t)hk * a.k_h;
  const uint16_t* vp = a.v + p.k0 * a.v_t + (int64_t)hk * a.v_h;
  T tk, tv;
  tk.init(a.k_t, a.D, lane);
  tv.init(a.v_t, a.D, lane);
  const uint32_t base = lds_addr(lds);   // two slots of k, then two of v
  Frags<DIM> fr;
  fr.init(base, lane);

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = zero16();
  float m = -3.4028235e38f, l = 0.0f;   // of the scaled scores, in powers of two; l: this half wave's keys

  auto load_k = [&](int t) {
    tk.load(kp + (int64_t)t * kAttnK * a.k_t, p.lk - t * kAttnK, base + (uint32_t)((t & 1) * T::BYTES), wave);
  };
  auto load_v = [&](int t) {
    tv.load(vp + (int64_t)t * kAttnK * a.v_t, p.lk - t * kAttnK, base + (uint32_t)((2 + (t & 1)) * T::BYTES), wave);
  };
  auto lane_max = [&](const f32x16 (&s)[2]) CONCORD_INLINE_LAMBDA {
    float x = s[0][0];
#pragma unroll
    for (int r = 1; r < 32; ++r) x = fmaxf(x, s[r >> 4][r & 15]);
    return x;
  };
  auto masked = [&](int t) CONCORD_INLINE_LAMBDA { return (t + 1) * kAttnK - 1 > jlo; };
  auto mask = [&](int t, f32x16 (&s)[2]) CONCORD_INLINE_LAMBDA {
    // (the lane's last key: from the first query's, so that no register holds it meanwhile)
    uint32_t in_wave = lane & 31;
    pin(in_wave);
    const int end = a.causal ? min(jlo_raw + (int)in_wave, p.lk - 1) : p.lk - 1;
    const int lim = end - t * kAttnK - 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] = 32 * i + 8 * (r >> 2) + (r & 3) > lim ? -INFINITY : s[i][r];
  };
  // The sums are relative to m, which follows the maximum only when that has
  // grown by more than 2^8: the factor of out and l is then nearly never
  // applied, and the probabilities' rounding is relative to each.
  // mx: the largest of the lane's scores.
  auto raise = [&](float mx) CONCORD_INLINE_LAMBDA {
    const Halves both = halves(mx);
    const float top = fmaxf(both.lo, both.hi) * a.c;
    if (__builtin_amdgcn_ballot_w64(top > m + 8.0f)) {
      const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
  };
  // before the exponentials of tile t; mx: the largest of the lane's scores, unmasked
  auto settle = [&](int t, f32x16 (&s)[2], float mx) CONCORD_INLINE_LAMBDA {
    if (masked(t)) {
      mask(t, s);
      mx = lane_max(s);
    }
    raise(mx);
  };
  // Tile t's exponentials and product with v, and (NEXT) the scores of tile
  // t + 1.  A wave issues in order and an MFMA holds the matrix core for 32
  // clocks, so the step is laid out by hand: unit j is one MFMA (first those of
  // the scores, then those with v), the fragment read of unit j + AHEAD, and
  // its share of the exponentials and of the next maximum; nothing moves
  // between units.
  auto step = [&](auto nextc, auto slotc, f32x16 (&s)[2], f32x16 (&next)[2], float& mx) CONCORD_INLINE_LAMBDA {
    constexpr bool NEXT = decltype(nextc)::value;
    constexpr int SLOT = decltype(slotc)::value, AHEAD = 2;
    constexpr int NS = NEXT ? 2 * NK : 0, NU = NS + 4 * ND;          // units of the scores, of the step
    constexpr uint32_t kt = (1 - SLOT) * T::BYTES, vt = (2 + SLOT) * T::BYTES;
    bf16x8 frag[AHEAD + 1], e[4];
    auto read = [&](auto jc) CONCORD_INLINE_LAMBDA {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < NS) frag[j % (AHEAD + 1)] = fr.rows(kt, j & 1, j >> 1);
      else if constexpr (j < NU) frag[j % (AHEAD + 1)] = fr.cols(vt, (j - NS) % ND, (j - NS) / ND);
    };
    // exponentials done after n units: all before the last quarter of the
    // products with v, and each quarter's before its products
    constexpr auto done = [](int n) constexpr {
      const int even = (32 * n + NS + 3 * ND - 1) / (NS + 3 * ND);
      const int need = n >= NS ? 8 * ((n - NS) / ND + 1) : 0;
      const int v = even > need ? even : need;
      return v < 32 ? v : 32;
    };
    auto exps = [&](auto fromc, auto toc) CONCORD_INLINE_LAMBDA {
      constexpr int from = decltype(fromc)::value, to = decltype(toc)::value;
      static_for<to - from>([&](auto rc) CONCORD_INLINE_LAMBDA {
        constexpr int r = from + decltype(rc)::value;
        float& x = reinterpret_cast<float*>(&s[r >> 4])[r & 15];
        x = __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.c, -m));
        l += x;
        if constexpr (r % 8 == 7) e[r / 8] = round8(s[r >> 4], (r >> 3) & 1);
      });
    };
    static_for<AHEAD>([&](auto jc) CONCORD_INLINE_LAMBDA { read(jc); });
    exps(std::integral_constant<int, 0>(), std::integral_constant<int, done(0)>());
    __builtin_amdgcn_sched_barrier(0);
    static_for<NU>([&](auto jc) CONCORD_INLINE_LAMBDA {
      constexpr int j = decltype(jc)::value;
      read(std::integral_constant<int, j + AHEAD>());
      if constexpr (j < NS) {
        constexpr int i = j & 1, k = j >> 1;
        next[i] = mfma(frag[j % (AHEAD + 1)], q.f[k], k == 0 ? zero16() : next[i]);
      } else {
        constexpr int d = (j - NS) % ND, u = (j - NS) / ND;
        o[d] = mfma(frag[j % (AHEAD + 1)], e[u], o[d]);
        if constexpr (NEXT) {
          // 32 scores over the 4 ND units
          constexpr int from = 32 * (j - NS) / (4 * ND), to = 32 * (j - NS + 1) / (4 * ND);
#pragma unroll
          for (int r = from; r < to; ++r) mx = r == 0 ? next[0][0] : fmaxf(mx, next[r >> 4][r & 15]);
        }
      }
      exps(std::integral_constant<int, done(j)>(), std::integral_constant<int, done(j + 1)>());
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  const int own = jhi < 0 ? 0 : min(tiles, jhi / kAttnK + 1);   // tiles with a key for any of the wave's queries
  typedef std::integral_constant<int, 0> S0;
  typedef std::integral_constant<int, 1> S1;
  auto scores = [&](f32x16 (&s)[2]) CONCORD_INLINE_LAMBDA {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = zero16();
#pragma unroll
      for (int k = 0; k < NK; ++k) s[i] = mfma(fr.rows(0, i, k), q.f[k], s[i]);
    }
  };
  if constexpr (!PIPE) {
    // Narrow heads have few MFMAs to an exponential, so past the first tile the
    // maximum is not even formed: m stays until a lane's 32 probabilities add up
    // to more than 2^20 (or to no number).  The scores are then formed again from
    // the tile, which still lies in LDS, and m is raised.  (2 x 4096 x 10 heads of
    // 64: 112 -> 109.5 us; 64 heads: 600 us before, 582 and 609 in two runs since.)
    auto exps = [&](f32x16 (&s)[2]) CONCORD_INLINE_LAMBDA {
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 32; ++r) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 4][r & 15], a.c, -m));
        s[r >> 4][r & 15] = e;
        sum += e;
      }
      return sum;
    };
    if (tiles > 0) load_k(0), load_v(0);
    for (int t = 0; t < tiles; ++t) {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // this wave's part of tile t has landed
      lds_barrier();                              // everyone's has, and tile t - 1 has been read
      if (t + 1 < tiles) load_k(t + 1), load_v(t + 1);
      if (t < own) {
        f32x16 s[2];
        scores(s);
        if (masked(t)) mask(t, s);
        if (t == 0) raise(lane_max(s));
        float sum = exps(s);
        if (__builtin_amdgcn_ballot_w64(!(sum <= 0x1p20f))) {
          scores(s);
          if (masked(t)) mask(t, s);
          raise(lane_max(s));
          sum = exps(s);
        }
        l += sum;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bf16x8 e = round8(s[u >> 1], u & 1);
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] = mfma(fr.cols(2 * T::BYTES, d, u), e, o[d]);
        }
      }
      fr.move(t & 1 ? -T::BYTES : T::BYTES);
    }
  } else if (tiles > 0) {
    // before tile t: its values and tile t + 1's keys have landed, and those of
    // the slots to fill next have been read
    auto turn = [&](int t) CONCORD_INLINE_LAMBDA {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      lds_barrier();
      if (t + 2 < tiles) load_k(t + 2);
      if (t + 1 < tiles) load_v(t + 1);
    };
    f32x16 sa[2], sb[2];
    load_k(0);
    load_v(0);
    if (tiles > 1) load_k(1);
    if (tiles > 1) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * T::PER));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::PER));
    lds_barrier();
    scores(sa);
    float mx = lane_max(sa);
    int t = 0;
    for (; t + 2 < own; t += 2) {
      turn(t);
      settle(t, sa, mx);
      step(std::true_type(), S0(), sa, sb, mx);
      turn(t + 1);
      settle(t + 1, sb, mx);
      step(std::true_type(), S1(), sb, sa, mx);
    }
    if (t + 1 < own) {
      turn(t);
      settle(t, sa, mx);
      step(std::true_type(), S0(), sa, sb, mx);
      turn(t + 1);
      settle(t + 1, sb, mx);
      step(std::false_type(), S1(), sb, sa, mx);
      t += 2;
    } else if (t < own) {
      turn(t);
      settle(t, sa, mx);
      step(std::false_type(), S0(), sa, sb, mx);
      ++t;
    }
    for (; t < tiles; ++t) turn(t);
  }

  const Halves both = halves(l);
  l = both.lo + both.hi;
  if constexpr (SPLIT) {
    if ((lane & 31) >= rows) return;
    const int64_t row = (p.q0 + qi) * a.heads + head, all = a.seq.TQ * a.heads;
    store_sums(a.part + ((int64_t)share * all + row) * a.D, o, a.D, lane);
    if (lane < 32)
      *(float2*)(a.part + (int64_t)a.splits * all * a.D + ((int64_t)share * all + row) * 2) = make_float2(m, l);
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = a.out + (p.q0 + row0) * a.o_t + (int64_t)head * a.o_h;
  const int64_t low_t = (int64_t)a.heads * a.D;
  int8_t* low = a.low ? a.low + (p.q0 + row0) * low_t + (int64_t)head * a.D : nullptr;
#pragma unroll
  for (int d = 0; d < ND; ++d) store_block(out, a.o_t, rows, a.D, d, o[d], inv, lane, low, low_t);
  if (a.lse && lane < 32 && lane < rows)
    a.lse[(int64_t)head * a.seq.TQ + p.q0 + qi] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// out, lse and out_low of split keys: a thread 8 elements of a row
__global__ __launch_bounds__(256) void attn_join_kernel(AttnFwd a) {
  const int64_t all = a.seq.TQ * a.heads, e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= all * a.D) return;
  const int64_t row = e / a.D, tok = row / a.heads;
  const int c = (int)(e - row * a.D), head = (int)(row - tok * a.heads);
  const float2* ml = (const float2*)(a.part + (int64_t)a.splits * all * a.D);
  float m = -3.4028235e38f, l = 0.0f, v[8] = {};
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[(int64_t)s * all + row].x);
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[(int64_t)s * all + row];
    const float f = __builtin_amdgcn_exp2f(x.x - m);   // (a share without keys has l = 0 and sums of 0)
    l = __builtin_fmaf(x.y, f, l);
    const float4* p = (const float4*)(a.part + ((int64_t)s * all + row) * a.D + c);
    const float4 y = p[0], z = p[1];
    const float w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(w[i], f, v[i]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t hi[4], lo[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = v[2 * i] * inv, y = v[2 * i + 1] * inv;
    hi[i] = pack_bf16x2(x, y);
    lo[i >> 1] |= (uint32_t)(left_over(x, hi[i] & 0xFFFF) | left_over(y, hi[i] >> 16) << 8) << (16 * (i & 1));
  }
  *(uint4*)(a.out + tok * a.o_t + (int64_t)head * a.o_h + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  if (a.low) *(uint2*)(a.low + e) = make_uint2(lo[0], lo[1]);
  if (a.lse && c == 0) a.lse[(int64_t)head * a.seq.TQ + tok] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

}  // namespace concord

using namespace concord;

extern "C" size_t concord_attention_fwd_workspace_bytes(const concord_attn_args* args) {
  if (!args || attn_sizes("concord_attention_fwd_workspace_bytes", *args) || args->TQ < 1) return 0;
  const int n = key_splits(*args, 4.0);
  return n > 1 ? (size_t)n * (size_t)args->TQ * (size_t)args->H * (size_t)(args->D + 2) * sizeof(float) : 0;
}

extern "C" int concord_attention_fwd(const concord_attn_args* args, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  CONCORD_CHECK(args, "concord_attention_fwd: NULL argument");
  const concord_attn_args& g = *args;
  if (const int rc = attn_check("concord_attention_fwd", g)) return rc;
  CONCORD_CHECK(!g.lse == !g.out_low && ((uintptr_t)g.out_low & 15) == 0,
                "concord_attention_fwd: lse and out_low come together, out_low on 16 bytes");
  if (g.TQ == 0) return CONCORD_OK;
  const size_t need = concord_attention_fwd_workspace_bytes(args);
  if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) {
    set_error("concord_attention_fwd: workspace of %zu bytes on 16 needed", need);
    return CONCORD_EWORKSPACE;
  }
  AttnFwd a{};
  a.splits = key_splits(g, 4.0);
  a.part = (float*)workspace;
  a.q = g.q, a.k = g.k, a.v = g.v, a.out = g.out, a.lse = g.lse, a.low = g.out_low, a.heads = g.H;
  a.q_t = g.q_t, a.q_h = g.q_h, a.k_t = g.k_t, a.k_h = g.k_h, a.v_t = g.v_t, a.v_h = g.v_h;
  a.o_t = g.o_t, a.o_h = g.o_h;
  a.seq = attn_seqs(g);
  const int64_t slots = attn_slots(a.seq, g.TQ, kAttnQ);
  CONCORD_CHECK(grid_fits(slots * g.H * a.splits, 256), "concord_attention_fwd: too many tiles");
  a.slots = (int32_t)slots;
  a.rep = g.H / g.HK, a.D = g.D, a.causal = g.causal != 0, a.c = g.scale * kLog2e;
  const dim3 grid((unsigned)(slots * g.H * a.splits));
  hipStream_t st = (hipStream_t)stream;
  attn_by_dim(g.D, [&](auto nk) {
    constexpr int NK = decltype(nk)::value;
    if (a.splits > 1) hipLaunchKernelGGL((attn_fwd_kernel<NK, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_fwd_kernel<NK, false>), grid, dim3(256), 0, st, a);
  });
  if (a.splits > 1)
    hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)cdiv(g.TQ * g.H * g.D, 2048)), dim3(256), 0, st, a);
  return launch_status("attention_fwd");
}
