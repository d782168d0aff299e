// attention.hip -- attention over whole sequences, forward:
//   out = softmax(scale q k^T) v, each query over the keys of its sequence.
//
// A workgroup of four waves holds 128 queries of one head, 32 a wave, and
// passes once over their keys, 64 at a time, with the running maximum and sum
// of each query's softmax.  Everything is transposed: a wave forms the scores
// as k q^T, so a lane holds one query's column and the maximum, the sum and
// the rescaling are lane-local (one exchange between the half waves for the
// maximum); the probabilities, rounded to bf16, are the B operand of
// out^T += v^T p without leaving the lane.
#include "attention.h"

namespace concord {

struct AttnFwd {
  const uint16_t *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  uint16_t* out;
  int64_t o_t, o_h;
  float* lse;
  int8_t* low;
  AttnSeqs seq;
  int32_t slots, rep, D, causal, heads;   // rep: query heads of a key head
  float c;                         // scale log2(e)
};

constexpr int kAttnQ = 128;   // queries of a workgroup
constexpr int kAttnK = 64;    // keys of a step

template <int NK>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnFwd a) {
  typedef Dim<NK> DIM;
  typedef Tile<DIM, kAttnK, 4> T;
  constexpr int ND = DIM::ND;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES];   // two slots of k and v
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lin = attn_xcd(blockIdx.x, gridDim.x);
  const int per = a.rep * a.slots;
  const int hk = lin / per, in = lin - hk * per;
  const int slot = a.slots - 1 - in / a.rep, head = hk * a.rep + in % a.rep;
  const AttnPlace p = attn_place<kAttnQ, false>(a.seq, slot);
  if (p.first < 0 || p.first >= p.lq) return;

  const int row0 = p.first + wave * 32;                  // the wave's first query
  const int rows = p.lq - row0;                          // (may be <= 0: it still loads tiles)
  const int off = p.lk - p.lq;                           // causal: query i sees keys <= i + off
  // keys of the workgroup's last query
  const int last = min(p.first + kAttnQ, p.lq) - 1;
  const int keys = a.causal ? max(0, min(p.lk, last + off + 1)) : p.lk;
  const int tiles = (keys + kAttnK - 1) / kAttnK;
  // the lane's last key, and the wave's first and last queries' last keys
  const int qi = row0 + (lane & 31);
  const int jmax = a.causal ? min(p.lk - 1, qi + off) : p.lk - 1;
  const int jlo = a.causal ? min(p.lk - 1, row0 + off) : p.lk - 1;
  const int jhi = a.causal ? min(p.lk - 1, row0 + 31 + off) : p.lk - 1;

  Fixed<DIM> q;
  q.load(a.q + (p.q0 + row0) * a.q_t + (int64_t)head * a.q_h, rows, a.q_t, a.D, lane);
  const uint16_t* kp = a.k + p.k0 * a.k_t + (int64_t)hk * a.k_h;
  const uint16_t* vp = a.v + p.k0 * a.v_t + (int64_t)hk * a.v_h;
  T tk, tv;
  tk.init(a.k_t, a.D, lane);
  tv.init(a.v_t, a.D, lane);
  const uint32_t base = lds_addr(lds);
  Frags<DIM> fr;
  fr.init(base, lane);

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = zero16();
  float m = -3.4028235e38f, l = 0.0f;   // of the scaled scores, in powers of two; l: this half wave's keys

  auto load = [&](int t) {
    const uint32_t s = base + (uint32_t)((t & 1) * 2 * T::BYTES);
    tk.load(kp + (int64_t)t * kAttnK * a.k_t, p.lk - t * kAttnK, s, wave);
    tv.load(vp + (int64_t)t * kAttnK * a.v_t, p.lk - t * kAttnK, s + T::BYTES, wave);
  };
  auto step = [&](int j0) {
    constexpr uint32_t kt = 0, vt = T::BYTES;
    f32x16 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = zero16();
#pragma unroll
      for (int k = 0; k < NK; ++k) s[i] = mfma(fr.rows(kt, i, k), q.f[k], s[i]);
    }
    if (j0 + kAttnK - 1 > jlo) {
      const int lim = jmax - j0 - 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = 32 * i + 8 * (r >> 2) + (r & 3) > lim ? -INFINITY : s[i][r];
    }
    float mx = s[0][0];
#pragma unroll
    for (int r = 1; r < 32; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
    const Halves both = halves(mx);
    mx = fmaxf(both.lo, both.hi) * a.c;
    // The sums are relative to m, which follows the maximum only when that has
    // grown by more than 2^8: the factor of out and l is then nearly never
    // applied, and the probabilities stay within 2^8, exact in their type as
    // those below 1 are.
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.0f)) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 4][r & 15], a.c, -m));
      s[r >> 4][r & 15] = e;
      l += e;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bf16x8 e = round8(s[u >> 1], u & 1);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = mfma(fr.cols(vt, d, u), e, o[d]);
    }
  };
  if (tiles > 0) load(0);
  for (int t = 0; t < tiles; ++t) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // this wave's part of tile t has landed
    lds_barrier();                              // everyone's has, and tile t - 1 has been read
    if (t + 1 < tiles) load(t + 1);
    // (past jhi no key is left for any of the wave's queries)
    if (t * kAttnK <= jhi) step(t * kAttnK);
    fr.move(t & 1 ? -2 * T::BYTES : 2 * T::BYTES);
  }

  const Halves both = halves(l);
  l = both.lo + both.hi;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = a.out + (p.q0 + row0) * a.o_t + (int64_t)head * a.o_h;
  const int64_t low_t = (int64_t)a.heads * a.D;
  int8_t* low = a.low ? a.low + (p.q0 + row0) * low_t + (int64_t)head * a.D : nullptr;
#pragma unroll
  for (int d = 0; d < ND; ++d) store_block(out, a.o_t, rows, a.D, d, o[d], inv, lane, low, low_t);
  if (a.lse && lane < 32 && lane < rows)
    a.lse[(int64_t)head * a.seq.TQ + p.q0 + qi] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

}  // namespace concord

using namespace concord;

extern "C" int concord_attention_fwd(const concord_attn_args* args, void* stream) {
  CONCORD_CHECK(args, "concord_attention_fwd: NULL argument");
  const concord_attn_args& g = *args;
  if (const int rc = attn_check("concord_attention_fwd", g)) return rc;
  CONCORD_CHECK(!g.lse == !g.out_low && ((uintptr_t)g.out_low & 15) == 0,
                "concord_attention_fwd: lse and out_low come together, out_low on 16 bytes");
  if (g.TQ == 0) return CONCORD_OK;
  AttnFwd a{};
  a.q = g.q, a.k = g.k, a.v = g.v, a.out = g.out, a.lse = g.lse, a.low = g.out_low, a.heads = g.H;
  a.q_t = g.q_t, a.q_h = g.q_h, a.k_t = g.k_t, a.k_h = g.k_h, a.v_t = g.v_t, a.v_h = g.v_h;
  a.o_t = g.o_t, a.o_h = g.o_h;
  a.seq = attn_seqs(g);
  const int64_t slots = attn_slots(a.seq, g.TQ, kAttnQ);
  CONCORD_CHECK(slots * g.H < (1LL << 31), "concord_attention_fwd: too many tiles");
  a.slots = (int32_t)slots;
  a.rep = g.H / g.HK, a.D = g.D, a.causal = g.causal != 0, a.c = g.scale * kLog2e;
  const dim3 grid((unsigned)(slots * g.H));
  attn_by_dim(g.D, [&](auto nk) {
    hipLaunchKernelGGL((attn_fwd_kernel<decltype(nk)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
  });
  return launch_status("attention_fwd");
}
